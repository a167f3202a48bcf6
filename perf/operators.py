"""Cases, inputs and plain forms of the learned per-atom operators.

Two operators of ``ye3t_b200.runtime``:

``species_embedding``     ``out[i] = scale * table[species[i]]`` and the table's gradient;
``structure_attention``   softmax attention among the atoms of each structure of a packed batch, scores
                          lowered by ``slope_h`` times the distance of the two atoms, with grouped heads,
                          and the gradients of queries, keys, values, positions and slopes.

``run`` computes them in elementary torch operations in 32 bits, or through the package where ``own`` is set.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
FLOAT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# -- cases -----------------------------------------------------------------------------------
def _embedding(atoms, species, channels, dtype, train, skew, **more):
    return dict(more, op="embedding", atoms=atoms, species=species, channels=channels, dtype=dtype, train=train,
                skew=skew)


def _attention(structures, atoms, heads, key_heads, width, dtype, train, ragged, readout=False, **more):
    return dict(more, op="attention", structures=structures, atoms=atoms, heads=heads, key_heads=key_heads,
                width=width, dtype=dtype, train=train, ragged=ragged, readout=readout)


def listed():
    return [
        # one small box of 80 atoms, an element table of 118 rows: the lookup of an MD step, latency only
        _embedding(80, 118, 64, "float32", False, False, name="embedding lookup 80 atoms"),
        # a box of 2^20 atoms of four species with 32 channels: very long segments for few table rows
        _embedding(1 << 20, 4, 32, "float32", True, False, name="embedding train 2^20 atoms"),
        # a training batch of 65,536 atoms in bf16 with wide vectors and the usual skew (most atoms hydrogen)
        _embedding(65536, 118, 256, "bfloat16", True, True, name="embedding train bf16"),
        # a table of 50,021 atom environments and an odd width, most rows untouched
        _embedding(200003, 50021, 100, "float32", True, True, name="embedding train environments"),
        # one structure of 80 atoms in fp32, forward only: the smallest call
        _attention(1, 80, 4, 4, 32, "float32", False, False, name="attention 80 atoms"),
        # a batch of molecules (0 to 40 atoms) in bf16, forward: screening
        _attention(2048, 20, 8, 8, 32, "bfloat16", False, True, name="attention molecules bf16"),
        # molecules with forces: gradients of everything, in fp32
        _attention(512, 32, 4, 4, 32, "float32", True, True, name="attention molecules train"),
        # a training batch of clusters of a few hundred atoms, keys shared by four heads
        _attention(16, 300, 8, 2, 64, "bfloat16", True, True, name="attention clusters train bf16"),
        # one structure of 4,096 atoms in fp32 with forces
        _attention(1, 4096, 4, 4, 64, "float32", True, False, name="attention 4096 train"),
        # one structure of 16,384 atoms, forward in bf16
        _attention(1, 16384, 8, 8, 64, "bfloat16", False, False, name="attention 16384 bf16"),
        # one structure of 8,192 atoms, the largest training pass
        _attention(1, 8192, 8, 8, 64, "bfloat16", True, False, name="attention 8192 train bf16"),
        # pooled readout: a single query per structure over its atoms, keys shared by two heads
        _attention(8, 16384, 8, 4, 64, "bfloat16", False, True, True, name="attention readout bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16"])
    train = rng.random() < 0.5
    if rng.random() < 0.3:
        channels = _spread(rng, 3, 512)
        atoms = _spread(rng, 1, min(1 << 20, (1 << 25) // channels))
        return _embedding(atoms, _spread(rng, 1, 60000), channels, dtype, train, rng.random() < 0.5)
    key_heads = rng.choice([1, 2, 3, 4, 8])
    heads = key_heads * rng.choice([1, 1, 2]) if key_heads < 8 else 8
    width = rng.choice([8, 16, 20, 32, 48, 64, 64, 80, 128, rng.randint(5, 128)])
    readout = rng.random() < 0.25
    ragged = rng.random() < 0.7
    structures = _spread(rng, 1, 1024)
    # the padded pairs of all structures and heads stay below those of the largest listed case
    room = 2 ** 37 / (heads * width * structures * (4 if ragged else 1))
    if readout:
        atoms = _spread(rng, 2, max(2, min(20000, 2 ** 27 / (key_heads * width * structures))))
    else:
        atoms = _spread(rng, 2, max(2, min(8192, math.sqrt(room / (4 if train else 1)))))
    return _attention(structures, atoms, heads, key_heads, width, dtype, train, ragged, readout)


def _lengths(case):
    """Atoms of each structure: all the same, or anything from none to twice the mean."""
    n, mean = case["structures"], case["atoms"]
    if not case["ragged"]:
        return [mean] * n
    rng = random.Random(n * 1000003 + mean)
    out = [rng.randint(0, 2 * mean - 1) for _ in range(n)]
    if sum(out) == 0:
        out[0] = mean
    return out


def _counts(case):
    keys = _lengths(case)
    return ([1] * len(keys) if case["readout"] else keys), keys


# -- inputs ----------------------------------------------------------------------------------
def _padded(counts):
    """Row numbers [structure, longest] of a packed batch and which of them are rows."""
    n = torch.tensor(counts, device=DEVICE)
    first = torch.cumsum(n, 0) - n
    at = torch.arange(max(1, max(counts)), device=DEVICE)
    there = at[None, :] < n[:, None]
    return torch.where(there, first[:, None] + at[None, :], 0), there


def _positions(count, atoms, generator):
    """Positions in a box of one structure's atoms at the benchmark's density of 0.05 atoms per cubic Angstrom."""
    return torch.rand(count, 3, generator=generator, device=DEVICE) * (atoms / 0.05) ** (1.0 / 3.0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dtype = FLOAT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE).to(dtype)

    state = {"case": case}
    if case["op"] == "embedding":
        n, v = case["atoms"], case["species"]
        u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
        u = u ** 3 if case["skew"] else u
        state["species"] = (u * v).long().clamp_(0, v - 1)
        state["table"] = normal(v, case["channels"])
        state["scale"] = math.sqrt(case["channels"])
        if case["train"]:
            state["grad"] = normal(n, case["channels"])
            state["table"].requires_grad_(True)
        return state
    queries, keys = _counts(case)
    nq, nk, h, hk, d = sum(queries), sum(keys), case["heads"], case["key_heads"], case["width"]
    state["query"], state["key"], state["value"] = normal(nq, h, d), normal(nk, hk, d), normal(nk, hk, d)
    state["key_positions"] = _positions(nk, case["atoms"], g)
    state["positions"] = _positions(nq, case["atoms"], g) if case["readout"] else state["key_positions"]
    state["slopes"] = 2.0 ** (-4.0 * (torch.arange(h, device=DEVICE) + torch.rand(h, generator=g, device=DEVICE)) / h)
    state["scale"] = d ** -0.5
    if case["train"]:
        state["grad"] = normal(nq, h, d)
        for name in ("query", "key", "value", "positions", "key_positions", "slopes"):
            state[name].requires_grad_(True)
    state["query_rows"], state["query_there"] = _padded(queries)
    state["key_rows"], state["key_there"] = _padded(keys)
    if own:
        from ye3t_b200.runtime import StructureLayout
        state["layout"] = StructureLayout(queries, keys if case["readout"] else None, heads=h, key_heads=hk,
                                          device=DEVICE)
    return state


# -- plain forms -----------------------------------------------------------------------------
def _plain_embedding(s):
    table, z, dtype = s["table"].detach().float(), s["species"], s["table"].dtype
    out = (table[z] * s["scale"]).to(dtype)
    if not s["case"]["train"]:
        return out
    grad = torch.zeros_like(table).index_add_(0, z, s["grad"].float() * s["scale"])
    return out, grad.to(dtype)


def _plain_attention(s):
    case = s["case"]
    n, h, hk, d = case["structures"], case["heads"], case["key_heads"], case["width"]
    qr, kr, qt, kt = s["query_rows"], s["key_rows"], s["query_there"], s["key_there"]
    lq, lk, m = qr.shape[1], kr.shape[1], h // hk
    dtype = s["query"].dtype
    slopes = s["slopes"].detach()

    def group_queries(x):  # [rows, h, d] -> [structure * key head, heads of it * longest, d]
        x = x.detach().float()[qr] * qt[:, :, None, None]
        return x.view(n, lq, hk, m, d).permute(0, 2, 3, 1, 4).reshape(n * hk, m * lq, d)

    def group_keys(x):  # [rows, hk, d] -> [structure * key head, longest, d]
        return (x.detach().float()[kr] * kt[:, :, None, None]).permute(0, 2, 1, 3).reshape(n * hk, lk, d)

    def flat_queries(x):
        return x.view(n, hk, m, lq, d).permute(0, 3, 1, 2, 4).reshape(n, lq, h, d)[qt]

    def flat_keys(x):
        return x.view(n, hk, lk, d).permute(0, 2, 1, 3)[kt]

    q, k, v = group_queries(s["query"]), group_keys(s["key"]), group_keys(s["value"])
    apart = s["positions"].detach()[qr][:, :, None] - s["key_positions"].detach()[kr][:, None, :]
    distance = apart.square().sum(-1).sqrt()
    score = torch.bmm(q, k.transpose(1, 2)).view(n, h, lq, lk) * s["scale"]
    score = score - slopes[None, :, None, None] * distance[:, None]
    score = score.masked_fill(~kt[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    out = flat_queries(torch.bmm(p.view(n * hk, m * lq, lk), v))
    if not case["train"]:
        return out.to(dtype)
    del score, top
    g = group_queries(s["grad"])
    dv = torch.bmm(p.view(n * hk, m * lq, lk).transpose(1, 2), g)
    dp = torch.bmm(g, v.transpose(1, 2)).view(n, h, lq, lk)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del p, dp
    dslopes = -(ds * distance[:, None]).sum((0, 2, 3))
    pull = (ds * slopes[None, :, None, None]).sum(1) * torch.where(distance > 0, 1.0 / distance, 0.0)
    force = pull[..., None] * apart
    dx, dy = -force.sum(2)[qt], force.sum(1)[kt]
    ds = ds.view(n * hk, m * lq, lk) * s["scale"]
    dq, dk = flat_queries(torch.bmm(ds, k)), flat_keys(torch.bmm(ds.transpose(1, 2), q))
    places = (dx, dy) if case["readout"] else (dx + dy,)
    return (out.to(dtype), dq.to(dtype), dk.to(dtype), flat_keys(dv).to(dtype)) + places + (dslopes,)


def run(state):
    if not own:
        return _plain_embedding(state) if state["case"]["op"] == "embedding" else _plain_attention(state)
    from ye3t_b200 import runtime
    s, train = state, state["case"]["train"]
    if s["case"]["op"] == "embedding":
        out = runtime.species_embedding(s["table"], s["species"], scale=s["scale"])
        return (out.detach(),) + torch.autograd.grad(out, s["table"], s["grad"]) if train else out
    readout = s["case"]["readout"]
    out = runtime.structure_attention(s["query"], s["key"], s["value"], s["layout"], positions=s["positions"],
                                      key_positions=s["key_positions"] if readout else None, slopes=s["slopes"],
                                      scale=s["scale"])
    if not train:
        return out
    wanted = [s["query"], s["key"], s["value"], s["positions"]] + ([s["key_positions"]] if readout else [])
    return (out.detach(),) + torch.autograd.grad(out, wanted + [s["slopes"]], s["grad"])


# -- work and the definition in 64 bits ------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "embedding":
        n, c, v = case["atoms"], case["channels"], case["species"]
        rows = min(v, n)
        once = 8 * n + size * c * (rows + n)
        return {"bytes": once + (size * c * (n + v) if case["train"] else 0), "flops": n * c * (2 if case["train"] else 1)}
    queries, keys = _counts(case)
    pairs = sum(a * b for a, b in zip(queries, keys)) * case["heads"] * case["width"]
    row_q, row_k = size * case["heads"] * case["width"], size * case["key_heads"] * case["width"]
    nq, nk = sum(queries), sum(keys)
    place = 12 * (nq + nk if case["readout"] else nk)
    forward = nq * 2 * row_q + nk * 2 * row_k + place
    backward = nq * 2 * row_q + nk * 2 * row_k + place
    if case["train"]:
        return {"bytes": forward + backward, "flops": 14 * pairs}
    return {"bytes": forward, "flops": 4 * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        table, z = s["table"].detach().double(), s["species"]
        out = s["scale"] * torch.index_select(table, 0, z)
        if not case["train"]:
            return out
        order = torch.argsort(z, stable=True)
        sums = torch.cumsum(s["grad"].double()[order], 0)
        ends = torch.cumsum(torch.bincount(z, minlength=case["species"]), 0)
        sums = torch.cat([torch.zeros_like(sums[:1]), sums])[torch.cat([torch.zeros_like(ends[:1]), ends])]
        return out, s["scale"] * (sums[1:] - sums[:-1])
    queries, keys = _counts(case)
    h, hk, d = case["heads"], case["key_heads"], case["width"]
    if sum(a * b for a, b in zip(queries, keys)) * h * d * (14 if case["train"] else 4) > 4e12:
        return None
    q, k, v = (s[name].detach().double() for name in ("query", "key", "value"))
    x, y, slopes = s["positions"].detach().double(), s["key_positions"].detach().double(), s["slopes"].detach().double()
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dx, dy, dslopes = torch.zeros_like(x), torch.zeros_like(y), torch.zeros_like(slopes)
    a = b = 0
    for nq, nk in zip(queries, keys):
        i, j = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        if not nq or not nk:
            continue
        apart = x[i, None, :] - y[None, j, :]
        distance = torch.linalg.vector_norm(apart, dim=-1)
        unit = apart / torch.where(distance == 0, 1.0, distance)[..., None]
        for head in range(h):
            kh = head * hk // h
            p = torch.softmax(s["scale"] * (q[i, head] @ k[j, kh].T) - slopes[head] * distance, dim=-1)
            out[i, head] = p @ v[j, kh]
            if case["train"]:
                go = s["grad"][i, head].double()
                dv[j, kh] += p.T @ go
                ds = p * (go @ v[j, kh].T - (go * out[i, head]).sum(-1, keepdim=True))
                dq[i, head] = s["scale"] * (ds @ k[j, kh])
                dk[j, kh] += s["scale"] * (ds.T @ q[i, head])
                dslopes[head] -= (ds * distance).sum()
                force = slopes[head] * ds[..., None] * unit
                dx[i] -= force.sum(1)
                dy[j] += force.sum(0)
    if not case["train"]:
        return out
    places = (dx, dy) if case["readout"] else (dx + dy,)
    return (out, dq, dk, dv) + places + (dslopes,)

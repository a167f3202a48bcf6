"""Species embedding and structure attention against plain float64 evaluations.

Tolerances, derived before the first run.  float32: a result is a sum of n products
rounded to 2^-24 each, held against the sum of magnitudes' scale; with n up to some thousands and
exp2 good to 2^-22, 2e-6 times sqrt of the number of scores' magnitudes stays under 2e-5 of the result's
norm.  bfloat16: the final rounding is 2^-9 = 2e-3 of a value at most, and probabilities
rounded to bfloat16 before a product add as much again: 6e-3 of the result's norm.  Position and slope
gradients are float32 for both types.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TOL = {torch.float32: 2e-5, torch.bfloat16: 6e-3, torch.float64: 1e-13}


def _close(got, want, tol, what=""):
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, what
    if want.numel() == 0:
        return
    assert torch.isfinite(got).all(), what
    err = float((got - want).norm())
    assert err <= tol * max(float(want.norm()), 1e-30), (what, err, float(want.norm()))


# -- species embedding -----------------------------------------------------------------------
EMBEDDING = [
    # atoms, species, channels
    (1, 1, 1), (1, 118, 64), (31, 3, 5), (32, 4, 32), (33, 2, 33), (4095, 118, 8), (4096, 1, 12), (4097, 300, 100),
    (70001, 5, 64), (9999, 50021, 17), (20000, 70000, 4), (300001, 3, 7), (5, 1000, 513),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("atoms,species,channels", EMBEDDING)
def test_embedding_and_gradient(atoms, species, channels, dtype):
    from ye3t_b200 import runtime as rt
    g = torch.Generator(device=DEV).manual_seed(atoms + species)
    index = torch.int32 if atoms % 2 else torch.int64
    z = (torch.rand(atoms, generator=g, device=DEV) ** 2 * species).long().clamp_(0, species - 1).to(index)
    table = torch.randn(species, channels, generator=g, device=DEV, dtype=torch.float64).to(dtype)
    grad = torch.randn(atoms, channels, generator=g, device=DEV, dtype=torch.float64).to(dtype)
    table.requires_grad_(True)
    out = rt.species_embedding(table, z, scale=1.75)
    want = (table.detach().double()[z.long()] * 1.75).to(dtype)
    assert torch.equal(out, want)
    (dt,) = torch.autograd.grad(out, table, grad, retain_graph=True)
    ref = torch.zeros(species, channels, dtype=torch.float64, device=DEV)
    ref.index_add_(0, z.long(), grad.double() * 1.75)
    _close(dt, ref, TOL[dtype])
    unused = torch.bincount(z.long(), minlength=species) == 0
    assert not dt[unused].any()
    assert torch.equal(dt, torch.autograd.grad(out, table, grad)[0])


def test_embedding_out_of_range_and_empty():
    from ye3t_b200 import runtime as rt
    table = torch.randn(6, 20, device=DEV, requires_grad=True)
    z = torch.tensor([0, 5, -1, 6, 2, 2, 1 << 40], device=DEV)
    out = rt.species_embedding(table, z)
    assert not out[[2, 3, 6]].any() and torch.equal(out[[0, 1, 4]], table.detach()[[0, 5, 2]])
    grad = torch.full_like(out, float("nan"))
    grad[[0, 1, 4, 5]] = torch.randn(4, 20, device=DEV)
    (dt,) = torch.autograd.grad(out, table, grad)
    assert torch.equal(dt[2], grad[4] + grad[5]) and torch.equal(dt[0], grad[0]) and not dt[[1, 3, 4]].any()
    with pytest.raises(IndexError):
        rt.species_embedding(table, z, validate=True)
    none = rt.species_embedding(table, torch.empty(0, dtype=torch.int64, device=DEV))
    assert none.shape == (0, 20)
    (dt,) = torch.autograd.grad(none, table, torch.empty(0, 20, device=DEV))
    assert not dt.any()
    assert rt.species_embedding(table, z.reshape(1, 7)).shape == (1, 7, 20)
    transposed = torch.randn(20, 6, device=DEV).t()
    assert torch.equal(rt.species_embedding(transposed, z[:2]), transposed[[0, 5]])
    # a view whose data does not start on 16 bytes
    shifted = torch.randn(6 * 20 + 1, device=DEV)[1:].view(6, 20)
    assert torch.equal(rt.species_embedding(shifted, z[:2]), shifted[[0, 5]])


def test_embedding_gradient_by_differences():
    """The lookup is linear in the table: a difference of any size gives the gradient."""
    from ye3t_b200 import runtime as rt
    g = torch.Generator(device=DEV).manual_seed(5)
    table = torch.randn(4, 3, generator=g, device=DEV, dtype=torch.float64, requires_grad=True)
    z = torch.randint(0, 4, (50,), generator=g, device=DEV)
    w = torch.randn(50, 3, generator=g, device=DEV, dtype=torch.float64)
    (dt,) = torch.autograd.grad(rt.species_embedding(table, z, scale=0.5), table, w)
    for v, c in ((0, 0), (3, 2), (1, 1)):
        e = torch.zeros_like(table)
        e[v, c] = 1.0
        f = [(rt.species_embedding(table.detach() + s * e, z, scale=0.5) * w).sum() for s in (0.5, -0.5)]
        assert abs(float(f[0] - f[1] - dt[v, c])) < 1e-12 * 50


# -- structure attention ---------------------------------------------------------------------
def _plain(q, k, v, x, y, slopes, scale, queries, keys, grad):
    """Output and gradients in float64, structure by structure."""
    q, k, v, grad = (t.detach().double() for t in (q, k, v, grad))
    if x is not None:
        x, y, slopes = (t.detach().double() for t in (x, y, slopes))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    dx = dy = dsl = None
    if x is not None:
        dx, dy, dsl = torch.zeros_like(x), torch.zeros_like(y), torch.zeros_like(slopes)
    H, m = q.shape[1], q.shape[1] // k.shape[1]
    a = b = 0
    for nq, nk in zip(queries, keys):
        i, j = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        if nq == 0 or nk == 0:
            continue
        if x is not None:
            r = x[i, None] - y[None, j]
            d = r.norm(dim=-1)
            u = torch.where(d[..., None] > 0, r / d.clamp_min(1e-300)[..., None], 0.0)
        for h in range(H):
            s = scale * q[i, h] @ k[j, h // m].T
            if x is not None:
                s = s - slopes[h] * d
            p = torch.softmax(s, -1)
            out[i, h] = p @ v[j, h // m]
            g = grad[i, h]
            dp = g @ v[j, h // m].T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            dv[j, h // m] += p.T @ g
            dq[i, h] = scale * ds @ k[j, h // m]
            dk[j, h // m] += scale * ds.T @ q[i, h]
            if x is not None:
                dsl[h] -= (ds * d).sum()
                f = slopes[h] * ds[..., None] * u
                dx[i] -= f.sum(1)
                dy[j] += f.sum(0)
    return out, dq, dk, dv, dx, dy, dsl


def _inputs(queries, keys, H, Hk, D, dtype, seed, bias=True, side=6.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    nq, nk = sum(queries), sum(keys)
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q, k, v, grad = n(nq, H, D).to(dtype), n(nk, Hk, D).to(dtype), n(nk, Hk, D).to(dtype), n(nq, H, D).to(dtype)
    x = y = sl = None
    if bias:
        x, y = torch.rand(nq, 3, generator=g, device=DEV) * side, torch.rand(nk, 3, generator=g, device=DEV) * side
        sl = torch.rand(H, generator=g, device=DEV) - 0.2
    return q, k, v, grad, x, y, sl


def _run(rt, q, k, v, grad, x, y, sl, queries, keys, scale, same):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    xs = None if x is None else x.detach().requires_grad_(True)
    ys = None if y is None or same else y.detach().requires_grad_(True)
    ss = None if sl is None else sl.detach().requires_grad_(True)
    layout = rt.StructureLayout(queries, None if same else keys, heads=q.shape[1], key_heads=k.shape[1], device=DEV)
    out = rt.structure_attention(*leaves, layout, positions=xs, key_positions=ys, slopes=ss, scale=scale)
    wanted = leaves + [t for t in (xs, ys, ss) if t is not None]
    return out, torch.autograd.grad(out, wanted, grad), layout


def _check(queries, keys, H, Hk, D, dtype, *, same=False, bias=True, scale=None, seed=0):
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, y, sl = _inputs(queries, keys, H, Hk, D, dtype, seed, bias)
    if same:
        y = x
    out, grads, _ = _run(rt, q, k, v, grad, x, y, sl, queries, keys, scale, same)
    ref = _plain(q, k, v, x, y, sl, D ** -0.5 if scale is None else scale, queries, keys, grad)
    _close(out, ref[0], TOL[dtype], "out")
    names = ["dq", "dk", "dv"]
    for name, got, want in zip(names, grads, ref[1:4]):
        _close(got, want, TOL[dtype], name)
    if bias:
        places = [ref[4] + ref[5]] if same else [ref[4], ref[5]]
        for name, got, want in zip(["dx", "dy"], grads[3:], places):
            _close(got, want, TOL[torch.float32], name)
        _close(grads[-1], ref[6], TOL[torch.float32], "dslopes")
    return out, grads


SHAPES = [
    # queries and keys of each structure (the same atoms), heads, key heads, width
    ([1], 1, 1, 1), ([2], 2, 1, 8), ([80], 4, 4, 32), ([3, 0, 17, 1, 33], 4, 2, 20), ([64], 2, 2, 64),
    ([65, 63, 128, 129], 2, 1, 64), ([500], 3, 3, 128), ([257, 1, 300], 8, 2, 48), ([1000], 1, 1, 100),
    ([31] * 40, 8, 8, 32), ([129] * 3, 6, 3, 5), ([16, 32, 48, 64, 96], 4, 4, 77),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts,H,Hk,D", SHAPES)
def test_attention_same_atoms(counts, H, Hk, D, dtype):
    _check(counts, counts, H, Hk, D, dtype, same=True, seed=sum(counts) + D)


CROSS = [
    # queries and keys of each structure apart
    ([1], [80], 4, 2, 32), ([1] * 9, [0, 1, 31, 32, 33, 500, 2, 64, 7], 8, 4, 64), ([5, 0, 3], [0, 40, 700], 2, 2, 24),
    ([300, 2], [1, 200], 4, 1, 64), ([1, 1], [5000, 1300], 4, 4, 128), ([200], [3], 2, 2, 16),
    ([1, 0, 700], [900, 4, 0], 2, 1, 40), ([3000], [5], 1, 1, 32),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("queries,keys,H,Hk,D", CROSS)
def test_attention_apart(queries, keys, H, Hk, D, dtype):
    _check(queries, keys, H, Hk, D, dtype, seed=sum(keys) + D)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts,H,Hk,D", [([20, 300], 4, 2, 64), ([7, 9], 2, 2, 33), ([700], 2, 1, 128)])
def test_attention_without_distance(counts, H, Hk, D, dtype):
    _check(counts, counts, H, Hk, D, dtype, same=True, bias=False, scale=0.2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_repeatable(dtype):
    a = _check([300, 1, 40], [300, 1, 40], 4, 2, 64, dtype, same=True, seed=3)
    b = _check([300, 1, 40], [300, 1, 40], 4, 2, 64, dtype, same=True, seed=3)
    assert torch.equal(a[0], b[0]) and all(torch.equal(s, t) for s, t in zip(a[1], b[1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 36])
def test_attention_strides_and_alignment(D, dtype):
    """Query, key and value cut from one projection, and a start off 16 bytes: the same values as dense."""
    from ye3t_b200 import runtime as rt
    n, H = [150, 20], 2
    q, k, v, grad, x, _, sl = _inputs(n, n, H, H, D, dtype, 9)
    dense = _run(rt, q, k, v, grad, x, x, sl, n, n, None, True)
    both = torch.stack([q, k, v], 1).reshape(sum(n), 3, H, D)
    cut = _run(rt, both[:, 0], both[:, 1], both[:, 2], grad, x, x, sl, n, n, None, True)
    flat = torch.zeros(3, sum(n) * H * D + 1, dtype=dtype, device=DEV)
    for t, s in zip(flat, (q, k, v)):
        t[1:] = s.reshape(-1)
    off = _run(rt, *(t[1:].view(sum(n), H, D) for t in flat), grad, x, x, sl, n, n, None, True)
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    moved = _run(rt, *swapped, grad.transpose(0, 1).contiguous().transpose(0, 1), x, x, sl, n, n, None, True)
    across = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    turned = _run(rt, *across, grad, x, x, sl, n, n, None, True)
    for other in (cut, off, moved, turned):
        assert torch.equal(dense[0], other[0])
        assert all(torch.equal(s, t) for s, t in zip(dense[1], other[1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("counts", [[40, 70, 30], [3, 5, 9], [200, 130, 64]])
def test_attention_structures_do_not_touch(counts, bad, dtype):
    """Non-finite data in one structure leaves every other structure's results as they were."""
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, _, sl = _inputs(counts, counts, 4, 2, 64, dtype, 21)
    clean = _run(rt, q, k, v, grad, x, x, sl, counts, counts, None, True)
    mid = slice(counts[0], counts[0] + counts[1])
    for t in (q, k, v, grad, x):
        t[mid] = bad
    dirty = _run(rt, q, k, v, grad, x, x, sl, counts, counts, None, True)
    keep = torch.ones(sum(counts), dtype=torch.bool, device=DEV)
    keep[mid] = False
    assert torch.equal(clean[0][keep], dirty[0][keep])
    for s, t in zip(clean[1][:4], dirty[1][:4]):
        assert torch.equal(s[keep], t[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_far_apart_and_large_scores(dtype):
    """Atoms so far away that every score but the own is far below: the row keeps its own value; scores
    of some thousands neither overflow nor lose the row."""
    from ye3t_b200 import runtime as rt
    n = [90]
    q, k, v, grad, _, _, _ = _inputs(n, n, 2, 2, 32, dtype, 2)
    x = torch.arange(90, device=DEV)[:, None] * torch.tensor([1e4, 0.0, 0.0], device=DEV)
    sl = torch.ones(2, device=DEV)
    out, _, _ = _run(rt, q, k, v, grad, x, x, sl, n, n, None, True)
    assert torch.equal(out, v)
    _check(n, n, 2, 2, 32, dtype, same=True, scale=0.0)
    big = _run(rt, q * 40, k * 40, v, grad, x * 0, x * 0, sl, n, n, None, True)[0]
    want = _plain(q * 40, k * 40, v, x * 0, x * 0, sl, 32 ** -0.5, n, n, grad)[0]
    _close(big, want, 1e-3 if dtype == torch.float32 else 6e-3)


@pytest.mark.parametrize("n", [48, 150])
def test_attention_gradients_by_differences(n):
    """Central differences of the float32 output in single coordinates: step e, error e^2 + 2^-23 |f| / e."""
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, _, sl = _inputs([n], [n], 2, 1, 32, torch.float32, 11)
    _, grads, layout = _run(rt, q, k, v, grad, x, x, sl, [n], [n], None, True)

    def f(q, k, v, x, sl):
        out = rt.structure_attention(q, k, v, layout, positions=x, slopes=sl)
        return float((out.double() * grad.double()).sum())

    args = [q, k, v, x, sl]
    g = torch.Generator(device=DEV).manual_seed(1)
    for number, name in enumerate(["q", "k", "v", "x", "slopes"]):
        # a random direction: the derivative along it is the gradient's product with it
        step = torch.randn(args[number].shape, generator=g, device=DEV)
        e = 2e-3
        moved = [list(args), list(args)]
        moved[0][number], moved[1][number] = args[number] + e * step, args[number] - e * step
        slope = (f(*moved[0]) - f(*moved[1])) / (2 * e)
        want = float((grads[number].double() * step.double()).sum())
        size = float(grads[number].norm()) * math.sqrt(step.numel())
        assert abs(slope - want) <= 2e-2 * float(grads[number].norm()) + 1e-3 * size / 10, (name, slope, want)


def test_attention_on_another_stream():
    from ye3t_b200 import runtime as rt
    n = [200, 30]
    q, k, v, grad, x, _, sl = _inputs(n, n, 2, 2, 64, torch.bfloat16, 4)
    want = _run(rt, q, k, v, grad, x, x, sl, n, n, None, True)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        got = _run(rt, q, k, v, grad, x, x, sl, n, n, None, True)
    torch.cuda.current_stream(DEV).wait_stream(side)
    assert torch.equal(want[0], got[0]) and all(torch.equal(s, t) for s, t in zip(want[1], got[1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_mixed_batch(dtype):
    """Every kind of structure in one batch: none, single atoms and keys, molecules, one or two queries over many
    keys, and structures of several tiles."""
    queries = [0, 1, 5, 1, 2, 200, 300, 64, 65, 3] + [20] * 300
    keys = [3, 1, 0, 500, 900, 200, 1, 64, 65, 70] + [20] * 300
    _check(queries, keys, 4, 2, 64, dtype, seed=17)
    _check([20] * 80 + [500, 1, 0, 64], [20] * 80 + [500, 1, 0, 64], 4, 4, 40, dtype, same=True, seed=18)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_long_and_split(dtype):
    """Columns split over several CTAs and joined on both sides, many tiles of rescaled rows."""
    _check([130, 2], [2100, 9], 2, 1, 64, dtype, seed=31)
    _check([1500], [140], 2, 1, 128, dtype, seed=32)
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, y, sl = _inputs([150], [1300], 2, 2, 64, dtype, 33)
    # scores that rise along the keys: the running maximum moves at every tile
    ramp = torch.linspace(0, 30, 1300, device=DEV)[:, None, None]
    k = (k * 0.1 + ramp * q.float().mean(0) / q.float().mean(0).norm(dim=-1, keepdim=True) ** 2).to(dtype)
    out, grads, _ = _run(rt, q, k, v, grad, x, y, sl, [150], [1300], 1.0, False)
    ref = _plain(q, k, v, x, y, sl, 1.0, [150], [1300], grad)
    # scores of some hundreds carry 2^-24 of themselves
    _close(out, ref[0], 1e-4 if dtype == torch.float32 else 6e-3, "out")


def test_attention_offsets_past_32_bits():
    """Rows so far apart that their offsets pass 2^32 elements."""
    from ye3t_b200 import runtime as rt
    n, far = 2200, 1 << 21
    base = torch.zeros(n * far, dtype=torch.bfloat16, device=DEV)
    for queries in ([n], [1]):
        q, k, v, _, x, y, sl = _inputs(queries, [n], 1, 1, 32, torch.bfloat16, 5)
        wide = base.as_strided((n, 2, 1, 32), (far, 1 << 20, 32, 1))
        wide[:, 0], wide[:, 1] = k, v
        layout = rt.StructureLayout(queries, [n], heads=1, device=DEV)
        near = rt.structure_attention(q, k, v, layout, positions=x, key_positions=y, slopes=sl)
        got = rt.structure_attention(q, wide[:, 0], wide[:, 1], layout, positions=x, key_positions=y, slopes=sl)
        assert torch.equal(near, got)


def test_embedding_past_32_bits():
    from ye3t_b200 import runtime as rt
    n, c = (1 << 21) + 5, 1025
    table = torch.randn(7, c, device=DEV).bfloat16()
    z = torch.arange(n, device=DEV) % 7
    out = rt.species_embedding(table, z)
    rows = torch.tensor([0, 1, (1 << 20) + 3, n - 2, n - 1], device=DEV)
    assert torch.equal(out[rows], table[z[rows]])
    dt = rt._embedding_adjoint(out, z, 7, 1.0)
    # bf16 inputs summed in fp32: each species' sum is its row times its count
    want = table.double() * torch.bincount(z).double()[:, None]
    _close(dt, want, TOL[torch.bfloat16])


def test_learned_in_a_cuda_graph():
    from ye3t_b200 import runtime as rt
    n = [300, 20, 1]
    q, k, v, _, x, _, sl = _inputs(n, n, 2, 2, 64, torch.bfloat16, 4)
    layout = rt.StructureLayout(n, heads=2, device=DEV)
    table, z = torch.randn(5, 64, device=DEV), torch.randint(0, 5, (321,), device=DEV)

    def step():
        return rt.structure_attention(q, k, v, layout, positions=x, slopes=sl), rt.species_embedding(table, z)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    q.add_(1.0)
    z.add_(1).remainder_(5)
    graph.replay()
    again = step()
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert not torch.equal(got[0], want[0])


def test_learned_torch_ops():
    """torch.ops.ye3t_b200.* give the runtime functions' results and gradients."""
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    ops = torch.ops.ye3t_b200
    n = [70, 1, 0, 30]
    q, k, v, grad, x, _, sl = _inputs(n, n, 4, 2, 48, torch.float32, 6)
    layout = rt.StructureLayout(n, heads=4, key_heads=2, device=DEV)
    want, grads, _ = _run(rt, q, k, v, grad, x, x, sl, n, n, 0.3, True)
    args = [t.detach().requires_grad_(True) for t in (q, k, v, x, sl)]
    out, _ = ops.structure_attention(args[0], args[1], args[2], layout.tables, layout.counts, args[3], None, args[4], 0.3)
    assert torch.equal(out, want)
    for a, b in zip(torch.autograd.grad(out, args, grad), grads):
        assert torch.equal(a, b)
    out, _ = ops.structure_attention(q, k, v, layout.tables, layout.counts, None, None, None, 0.3)
    assert torch.equal(out, rt.structure_attention(q, k, v, layout, scale=0.3))
    table = torch.randn(9, 20, device=DEV, requires_grad=True)
    z = torch.randint(0, 9, (100,), device=DEV)
    g = torch.randn(100, 20, device=DEV)
    a, b = ops.species_embedding(table, z, 2.0), rt.species_embedding(table, z, scale=2.0)
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, table, g)[0], torch.autograd.grad(b, table, g)[0])
    with pytest.raises(ValueError):
        rt.StructureLayout.from_tensors(layout.tables[:-1], layout.counts)
    with pytest.raises(ValueError):
        rt.StructureLayout.from_tensors(layout.tables, layout.counts[:-1])


# Base-2 log of a row's sum of exponentials.  A score is a sum of D = 48 products of unit normals in fp32: at most
# 48 * 2^-23 * sum |q k| scale log2(e) = 48 * 1.2e-7 * 31 * 0.3 * 1.44 = 8e-5 off.  With bfloat16 the sum may be that of the
# rounded probabilities, each within 2^-9: log2(1 + 2^-9) = 2.8e-3 more.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 3e-3)])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("queries,keys", [([70, 1, 0, 30], [70, 1, 0, 30]), ([5, 3, 64, 33], [7, 0, 64, 1]),
                                          ([1, 2, 1], [5000, 700, 90]), ([3, 90, 20], [200, 0, 40000]),
                                          ([300, 129], [500, 9000])])
def test_attention_op_returns_log_sum_exp(queries, keys, bias, dtype, tol):
    """The registered op's second result is written for every row, whichever kernel takes it; +inf without keys."""
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    q, k, v, _, x, y, sl = _inputs(queries, keys, 4, 2, 48, dtype, 11, bias)
    layout = rt.StructureLayout(queries, keys, heads=4, key_heads=2, device=DEV)
    want = torch.full((sum(queries), 4), float("inf"), dtype=torch.float64, device=DEV)
    a = b = 0
    for nq, nk in zip(queries, keys):
        if nq and nk:
            s = 0.3 * torch.einsum("ihd,jhd->hij", q[a:a + nq].double(), k[b:b + nk].double().repeat_interleave(2, 1))
            if bias:
                d = (x[a:a + nq, None].double() - y[None, b:b + nk].double()).norm(dim=-1)
                s = s - sl.double()[:, None, None] * d
            want[a:a + nq] = torch.logsumexp(s, -1).T / math.log(2.0)
        a, b = a + nq, b + nk
    # the allocator hands the results memory that holds NaN
    for shape, of in (((sum(queries), 4, 48), dtype), ((sum(queries), 4), torch.float32)):
        torch.full(shape, float("nan"), dtype=of, device=DEV)
    _, lse = torch.ops.ye3t_b200.structure_attention(q, k, v, layout.tables, layout.counts, x, y, sl, 0.3)
    assert lse.shape == want.shape and torch.equal(torch.isinf(lse), torch.isinf(want))
    held = torch.isfinite(want)
    assert (lse[held].double() - want[held]).abs().max() <= tol and (lse[~held] > 0).all()


@pytest.mark.parametrize("keys", [[65, 700, 3000], [2, 90, 131]])
@pytest.mark.parametrize("D", [7, 20, 64, 128])
def test_attention_key_gradients_of_one_query_are_rounded_once(keys, D):
    """With one query and one head a key, dk = scale dS q and dv = P g are single products in fp32: what bfloat16 adds is
    the rounding of the result, at most 2^-9 of each value."""
    from ye3t_b200 import runtime as rt
    queries = [1] * len(keys)
    q, k, v, grad, x, y, sl = _inputs(queries, keys, 2, 2, D, torch.bfloat16, D)
    _, grads, _ = _run(rt, q, k, v, grad, x, y, sl, queries, keys, 0.2, False)
    ref = _plain(q, k, v, x, y, sl, 0.2, queries, keys, grad)
    for got, want in zip(grads[1:3], ref[2:4]):
        _close(got, want, 2.0 ** -9 + TOL[torch.float32])


def test_attention_op_log_sum_exp_takes_no_gradient():
    """A loss on the registered op's log-sum-exp is refused: it is not silently without a gradient."""
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    n = [70, 30]
    q, k, v, grad, _, _, _ = _inputs(n, n, 2, 2, 16, torch.float32, 3, False)
    layout = rt.StructureLayout(n, heads=2, device=DEV)
    q.requires_grad_(True)
    out, lse = torch.ops.ye3t_b200.structure_attention(q, k, v, layout.tables, layout.counts, None, None, None, 0.25)
    assert out.requires_grad and not lse.requires_grad
    with pytest.raises(RuntimeError):
        torch.autograd.grad(lse.sum(), q)
    (dq,) = torch.autograd.grad((out * lse[..., None]).sum(), q, retain_graph=True)
    assert torch.equal(dq, torch.autograd.grad(out, q, lse[..., None].expand_as(out))[0])


def test_attention_energies_example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "attention_energies.py")
    spec = importlib.util.spec_from_file_location("attention_energies", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, forces = example.train(25, log=None)
    assert losses[-1] < 0.5 * losses[0]
    assert torch.isfinite(forces).all() and float(forces.norm()) > 0


def test_attention_from_a_thread_of_its_own():
    """A thread's first CUDA work is the call itself: no context is current there yet."""
    import threading
    from ye3t_b200 import runtime as rt
    n = [300, 200]
    q, k, v, grad, x, _, sl = _inputs(n, n, 2, 2, 64, torch.bfloat16, 4)
    layout = rt.StructureLayout(n, heads=2, device=DEV)
    want = rt.structure_attention(q, k, v, layout, positions=x, slopes=sl)
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(rt.structure_attention(q, k, v, layout, positions=x, slopes=sl))
        except Exception as exc:  # noqa: BLE001 - shown by the assertion
            got.append(exc)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert isinstance(got[0], torch.Tensor), got[0]
    assert torch.equal(got[0], want)


def test_attention_empty_batches():
    from ye3t_b200 import runtime as rt
    for queries, keys in (([], []), ([0, 0], [0, 0]), ([0, 0], [3, 4]), ([3, 4], [0, 0])):
        q, k, v, grad, x, y, sl = _inputs(queries, keys, 2, 2, 16, torch.float32, 0)
        out, grads, _ = _run(rt, q, k, v, grad, x, y, sl, queries, keys, None, False)
        assert not out.any() and not any(t.any() for t in grads)


def test_attention_broadcast_inputs():
    """One query for every structure (a row of stride zero): its gradient is the sum over structures."""
    from ye3t_b200 import runtime as rt
    keys = [40, 3, 100]
    q, k, v, grad, x, y, sl = _inputs([1] * 3, keys, 2, 1, 32, torch.float32, 8)
    one = q[:1].clone().requires_grad_(True)
    layout = rt.StructureLayout([1] * 3, keys, heads=2, key_heads=1, device=DEV)
    out = rt.structure_attention(one.expand(3, 2, 32), k, v, layout, positions=x, key_positions=y, slopes=sl)
    (dq,) = torch.autograd.grad(out, one, grad)
    ref = _plain(one.detach().expand(3, 2, 32), k, v, x, y, sl, 32 ** -0.5, [1] * 3, keys, grad)
    _close(out, ref[0], TOL[torch.float32])
    _close(dq, ref[1].sum(0, keepdim=True), TOL[torch.float32])


def test_attention_gradient_is_first_order_only():
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, _, sl = _inputs([5], [5], 1, 1, 8, torch.float32, 0)
    q.requires_grad_(True)
    layout = rt.StructureLayout([5], heads=1, device=DEV)
    out = rt.structure_attention(q, k, v, layout)
    (dq,) = torch.autograd.grad(out, q, grad.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


def test_attention_refusals():
    from ye3t_b200 import runtime as rt
    n = [4, 6]
    q, k, v, _, x, _, sl = _inputs(n, n, 4, 2, 16, torch.float32, 0)
    layout = rt.StructureLayout(n, heads=4, key_heads=2, device=DEV)

    def call(q=q, k=k, v=v, layout=layout, **more):
        return rt.structure_attention(q, k, v, layout, **more)

    call()
    with pytest.raises(TypeError):
        call(q.half(), k.half(), v.half())
    with pytest.raises(TypeError):
        call(q.double(), k.double(), v.double())
    with pytest.raises(TypeError):
        call(k=k.bfloat16())
    with pytest.raises(TypeError):
        call(layout=n)
    with pytest.raises(ValueError):
        call(q[:9])
    with pytest.raises(ValueError):
        call(q[:, :2])
    with pytest.raises(ValueError):
        call(v=v[:, :, :8])
    with pytest.raises(ValueError):
        call(q.repeat(1, 1, 9), k.repeat(1, 1, 9), v.repeat(1, 1, 9))
    with pytest.raises(ValueError):
        call(positions=x)
    with pytest.raises(ValueError):
        call(slopes=sl)
    with pytest.raises(ValueError):
        call(positions=x.double(), slopes=sl)
    with pytest.raises(ValueError):
        call(positions=x, slopes=sl[:2])
    with pytest.raises(ValueError):
        call(key_positions=x)
    with pytest.raises(ValueError):
        call(q.cpu(), k.cpu(), v.cpu())
    with pytest.raises(ValueError):
        call(backend="reference")
    with pytest.raises(ValueError):
        call(layout=rt.StructureLayout(n, n, heads=4, key_heads=2, device=DEV), positions=x, slopes=sl)


def test_embedding_refusals():
    from ye3t_b200 import runtime as rt
    table, z = torch.randn(3, 4, device=DEV), torch.tensor([0, 1], device=DEV)
    with pytest.raises(TypeError):
        rt.species_embedding(table.half(), z)
    with pytest.raises(TypeError):
        rt.species_embedding(table, z.float())
    with pytest.raises(ValueError):
        rt.species_embedding(table[0], z)
    with pytest.raises(ValueError):
        rt.species_embedding(table, z, backend="reference")
    with pytest.raises(ValueError):
        rt.species_embedding(table.cpu(), z.cpu())

"""Structure attention on rows and values that are not finite, against its definition in float64.

A score that is not a number makes its row one, as does a value that is not a number, however small its weight: the
definition multiplies it all the same.  Tolerances are those of the finite cases: float32 2e-5 of the result's norm
(some thousand products rounded to 2^-24 and exp2 to 2^-22), bfloat16 6e-3 (the result's own rounding, 1.7e-3 rms, and
that of the probabilities before their product).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TOL = {torch.float32: 2e-5, torch.bfloat16: 6e-3}


def _inputs(queries, keys, H, Hk, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    nq, nk = sum(queries), sum(keys)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    x, y = (torch.rand(n, 3, generator=g, device=DEV) * 6.0 for n in (nq, nk))
    return (normal(nq, H, D), normal(nk, Hk, D), normal(nk, Hk, D), normal(nq, H, D), x, y,
            torch.rand(H, generator=g, device=DEV) - 0.2)


def _definition(q, k, v, x, y, slopes, scale, queries, keys):
    """Output and base-2 log-sum-exp in float64, structure by structure."""
    q, k, v, x, y, slopes = (t.double() for t in (q, k, v, x, y, slopes))
    m = q.shape[1] // k.shape[1]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], math.inf, dtype=torch.float64, device=DEV)
    a = b = 0
    for nq, nk in zip(queries, keys):
        i, j = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        d = (x[i, None] - y[None, j]).norm(dim=-1)
        s = scale * torch.einsum("ihd,jhd->hij", q[i], k[j].repeat_interleave(m, 1)) - slopes[:, None, None] * d
        out[i] = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[j].repeat_interleave(m, 1))
        lse[i] = torch.logsumexp(s, -1).T / math.log(2.0)
    return out, lse


def _same_numbers(got, want, tol, what):
    got, want = got.detach().double(), want.detach().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    held = torch.isfinite(want)
    assert torch.isfinite(got[held]).all(), what
    assert float((got[held] - want[held]).norm()) <= tol * max(float(want[held].norm()), 1e-30), what


# 385 keys: three parts, the last of which holds one key; 700 several; 70 a single part
FEW = ([1, 2, 1], [385, 700, 70])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["query", "infinite query", "positions", "slopes", "keys", "last key", "all but one key"])
def test_few_queries_keep_what_is_not_a_number(where, dtype):
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    queries, keys = FEW
    q, k, v, _, x, y, sl = _inputs(queries, keys, 4, 2, 48, dtype, 3)
    nan = float("nan")
    if where == "query":
        q[0, 1, 5] = q[2, 0, 0] = nan
    elif where == "infinite query":
        q[0, 1, 5] = float("inf")
    elif where == "positions":
        x[1, 2] = nan
    elif where == "slopes":
        sl[3] = nan
    elif where == "keys":
        k[:385, 1, 7] = nan
    elif where == "last key":
        k[384, 0, 7] = nan
    else:
        k[385 + 1:385 + 700, 0, 7] = k[1085 + 1:, 1, 0] = nan
    layout = rt.StructureLayout(queries, keys, heads=4, key_heads=2, device=DEV)
    assert dict(zip(rt._LAYOUT_COUNTS, layout.counts))["few_item_count"] > 3
    out, lse = torch.ops.ye3t_b200.structure_attention(q, k, v, layout.tables, layout.counts, x, y, sl, 0.15)
    want, want_lse = _definition(q, k, v, x, y, sl, 0.15, queries, keys)
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    _same_numbers(out, want, TOL[dtype], "out")
    if where != "infinite query":  # of which the definition in torch is infinite, and not a number here
        _same_numbers(lse, want_lse, 1e-4, "log-sum-exp")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [48, 100])
@pytest.mark.parametrize("queries,keys", [([150], [200]), ([150], [9000]), ([40], [50]), ([2], [700])])
def test_a_row_without_finite_scores_gives_zeros(queries, keys, D, dtype):
    """A row whose scores are all -inf gives zeros and takes part in no gradient, whichever kernel has it."""
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, y, sl = _inputs(queries, keys, 2, 1, D, dtype, D)
    dead = queries[0] // 2
    # powers of two, so that the products of the pieces of a value stay exact: -2^200 is past fp32
    k[:, :, 0], q[:, :, 0], q[dead, :, 0] = 2.0 ** 100, 0.0, -(2.0 ** 100)
    leaves = [t.requires_grad_(True) for t in (q, k, v, x, y, sl)]
    layout = rt.StructureLayout(queries, keys, heads=2, key_heads=1, device=DEV)
    out = rt.structure_attention(q, k, v, layout, positions=x, key_positions=y, slopes=sl, scale=0.25)
    dq, dk, dv, dx, dy, dsl = torch.autograd.grad(out, leaves, grad)
    for got in (out, dq, dx):
        assert not got[dead].any()
    # the other rows, by themselves
    keep = torch.arange(queries[0], device=DEV) != dead
    wide = [t.detach().double().requires_grad_(True) for t in (q[keep], k, v, x[keep], y, sl)]
    want = _definition(*wide, 0.25, [queries[0] - 1], keys)[0]
    ref = torch.autograd.grad(want, wide, grad[keep].double())
    tol, fine = TOL[dtype], TOL[torch.float32]
    _same_numbers(out[keep], want, tol, "out")
    _same_numbers(dq[keep][:, :, 1:], ref[0][:, :, 1:], tol, "dq")  # component 0 is a difference of 2^100s
    for got, expect, t, what in ((dk, ref[1], tol, "dk"), (dv, ref[2], tol, "dv"), (dx[keep], ref[3], fine, "dx"),
                                 (dy, ref[4], fine, "dy"), (dsl, ref[5], fine, "dslopes")):
        _same_numbers(got, expect, t, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("queries,keys", [(40, 60), (150, 200), (150, 9000), (1, 9000), (2, 300)])
def test_a_value_that_is_not_a_number_is_not_lost_to_a_small_weight(queries, keys, dtype):
    """The weight of a far key underflows; its value still counts, whether or not the keys are split over CTAs."""
    from ye3t_b200 import runtime as rt
    q, k, v, _, x, y, sl = _inputs([queries], [keys], 2, 2, 48, dtype, 5)
    y[keys // 2:] += 1000.0
    sl.fill_(1.0)
    v[keys - 3, 0, 11] = float("nan")
    layout = rt.StructureLayout([queries], [keys], heads=2, device=DEV)
    out = rt.structure_attention(q, k, v, layout, positions=x, key_positions=y, slopes=sl, scale=0.15)
    want, _ = _definition(q, k, v, x, y, sl, 0.15, [queries], [keys])
    assert torch.isnan(want[:, 0, 11]).all() and torch.isfinite(want[:, 1]).all()
    _same_numbers(out, want, TOL[dtype], "out")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [5, 24, 64, 128])
def test_gradients_of_keys_in_items_of_128(D, dtype):
    """One and two queries over numbers of keys about the length of an item, heads that share keys."""
    from ye3t_b200 import runtime as rt
    queries, keys = [1, 2, 0, 1, 2, 1, 2], [127, 128, 140, 129, 256, 257, 65]
    q, k, v, grad, x, y, sl = _inputs(queries, keys, 4, 2, D, dtype, D)
    leaves = [t.requires_grad_(True) for t in (q, k, v, x, y, sl)]
    layout = rt.StructureLayout(queries, keys, heads=4, key_heads=2, device=DEV)
    assert dict(zip(rt._LAYOUT_COUNTS, layout.counts))["few_item_count"] >= 6
    out = rt.structure_attention(q, k, v, layout, positions=x, key_positions=y, slopes=sl, scale=0.2)
    got = torch.autograd.grad(out, leaves, grad)
    wide = [t.detach().double().requires_grad_(True) for t in (q, k, v, x, y, sl)]
    ref = torch.autograd.grad(_definition(*wide, 0.2, queries, keys)[0], wide, grad.double())
    for n, (a, b) in enumerate(zip(got, ref)):
        _same_numbers(a, b, TOL[dtype if n < 3 else torch.float32], n)


def _in_two_threads(calls, times):
    """Each call, many times over, in a thread and on a stream of its own; the return codes that are not zero."""
    import threading
    streams = [torch.cuda.Stream(DEV) for _ in calls]
    failed = []

    def work(call, stream):
        torch.cuda.set_device(DEV)
        for _ in range(times):
            rc = call(stream)
            if rc:
                failed.append(rc)
                return

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(call, s.cuda_stream)) for call, s in zip(calls, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return failed


def test_calls_of_two_threads_do_not_limit_each_other():
    """Two widths of small structures, and two small tables, on the same kernels: what shared memory a launch may have is
    not what another thread's call needs."""
    import ctypes

    from ye3t_b200 import _native as nat
    from ye3t_b200 import runtime as rt
    lib, layout = nat.lib(), rt.StructureLayout([64, 50], heads=2, device=DEV)
    hold, attention, adjoint, tables = [], [], [], []
    for D in (8, 128):
        q, k, v, g, x, _, sl = _inputs([64, 50], [64, 50], 2, 2, D, torch.float32, D)
        args = rt._attention_args(q, k, v, x, x, sl, layout, 0.2)
        out, lse = rt._attention_forward(q, k, v, x, x, sl, layout, 0.2, False)
        ws, size = rt._attention_workspace(args, 1, q.device)
        grads = [torch.empty_like(t) for t in (q, k, v, x, sl)]
        hold += [q, k, v, g, x, sl, out, lse, ws, args] + grads
        at = [t.data_ptr() for t in (out, g, lse, ws)]
        to = [t.data_ptr() for t in grads]
        attention.append(lambda s, a=args, at=at: lib.y3b_structure_attention(ctypes.byref(a), at[3], 0, at[0], at[2], 0, s))
        adjoint.append(lambda s, a=args, at=at, to=to, size=size: lib.y3b_structure_attention_adjoint(
            ctypes.byref(a), at[0], at[1], at[2], at[3], size, to[0], to[1], to[2], to[3], 0, to[4], 0, s))
    for species in (2, 24):
        grad, z = torch.ones(500, 128, device=DEV), torch.arange(500, device=DEV) % species
        size = int(lib.y3b_species_embedding_adjoint_workspace_bytes(nat.F32, 500, species, 128))
        ws, out = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV), torch.empty(species, 128, device=DEV)
        hold += [grad, z, ws, out]
        p = [t.data_ptr() for t in (grad, z, ws, out)]
        tables.append(lambda s, p=p, n=species, size=size: lib.y3b_species_embedding_adjoint(
            nat.F32, p[0], p[1], 8, 500, n, 128, 1.0, p[2], size, p[3], 0, s))
    for calls in (attention, adjoint, tables):
        assert all(call(0) == 0 for call in calls)
        assert not _in_two_threads(calls, 20000)
    del hold


@pytest.mark.parametrize("on", [False, True])
def test_registered_operators_read_the_status_where_validation_is_on(monkeypatch, on):
    """YE3T_B200_VALIDATE holds for torch.ops as for the runtime's functions."""
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    monkeypatch.setenv("YE3T_B200_VALIDATE", "1" if on else "0")
    read = []
    monkeypatch.setattr(rt, "_raise_on_status", lambda status, what: read.append((what, int(status))))
    n = [100, 7]
    q, k, v, grad, x, _, sl = _inputs(n, n, 2, 2, 16, torch.float32, 1)
    layout = rt.StructureLayout(n, heads=2, device=DEV)
    q.requires_grad_(True)
    out, _ = torch.ops.ye3t_b200.structure_attention(q, k, v, layout.tables, layout.counts, x, None, sl, 0.3)
    torch.autograd.grad(out, q, grad)
    assert read == ([("structure_attention", 0), ("structure_attention adjoint", 0)] if on else [])


def test_registered_adjoints_refuse_what_does_not_fit():
    """The adjoints are operators of their own: a gradient of another size or type is refused, not read past its end."""
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    ops = torch.ops.ye3t_b200
    grad, z = torch.ones(5, 8, device=DEV), torch.tensor([0, 1, 2, 1, 0], device=DEV)
    assert ops.species_embedding_adjoint(grad, z, 3, 1.0).shape == (3, 8)
    for g, s, n in ((grad[:3], z, 3), (grad[None], z, 3), (grad, z.reshape(1, 5), 3), (grad[:, :0], z, 3), (grad, z, -1)):
        with pytest.raises(ValueError):
            ops.species_embedding_adjoint(g, s, n, 1.0)
    for g, s in ((grad.half(), z), (grad, z.float())):
        with pytest.raises(TypeError):
            ops.species_embedding_adjoint(g, s, 3, 1.0)
    n = [4, 6]
    q, k, v, grad, x, _, sl = _inputs(n, n, 4, 2, 16, torch.float32, 0)
    layout = rt.StructureLayout(n, heads=4, key_heads=2, device=DEV)
    out, lse = ops.structure_attention(q, k, v, layout.tables, layout.counts, x, None, sl, 0.25)

    def adjoint(grad=grad, out=out, lse=lse):
        return ops.structure_attention_adjoint(grad, q, k, v, layout.tables, layout.counts, x, None, sl, out, lse, 0.25)

    assert adjoint()[0].shape == q.shape
    assert torch.equal(adjoint()[0], adjoint(out=out.transpose(0, 1).contiguous().transpose(0, 1),
                                             lse=lse.t().contiguous().t())[0])
    for wrong in ({"grad": grad[:9]}, {"grad": grad.bfloat16()}, {"out": out[:, :2]}, {"out": out.double()},
                  {"lse": lse[:4]}, {"lse": lse.double()}, {"lse": lse.cpu()}):
        with pytest.raises(ValueError):
            adjoint(**wrong)


def test_forward_mode_derivatives_are_refused():
    """A tangent is not dropped without a word, with or without gradients recorded."""
    import torch.autograd.forward_ad as forward_ad
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    n = [4, 6]
    q, k, v, _, x, _, sl = _inputs(n, n, 2, 2, 16, torch.float32, 0)
    layout = rt.StructureLayout(n, heads=2, device=DEV)
    table, z = torch.ones(3, 4, device=DEV), torch.tensor([0, 2], device=DEV)
    given = [q, k, v, x, sl]
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t.clone(), torch.ones_like(t)) for t in given + [table]]
        for recorded in (True, False):
            with torch.set_grad_enabled(recorded):
                for call in (lambda t: rt.species_embedding(t, z),
                             lambda t: torch.ops.ye3t_b200.species_embedding(t, z, 1.0)):
                    with pytest.raises(NotImplementedError):
                        call(dual[5])
                    assert call(table).shape == (2, 4)
                for number in range(5):
                    q1, k1, v1, x1, s1 = (dual[m] if m == number else t for m, t in enumerate(given))
                    with pytest.raises(NotImplementedError):
                        rt.structure_attention(q1, k1, v1, layout, positions=x1, slopes=s1)
                    with pytest.raises(NotImplementedError):
                        torch.ops.ye3t_b200.structure_attention(q1, k1, v1, layout.tables, layout.counts, x1, None, s1, 0.25)
                assert rt.structure_attention(q, k, v, layout, positions=x, slopes=sl).shape == q.shape


@pytest.mark.parametrize("queries,keys", [([70, 1, 0, 30], [70, 1, 0, 30]), ([5, 3, 64, 33], [7, 2, 64, 1]),
                                          ([1, 2, 1], [5000, 700, 90]), ([300, 129], [500, 9000])])
def test_log_sum_exp_of_bfloat16_is_that_of_float32(queries, keys):
    """Every kernel sums the probabilities as they are, before any is rounded to bfloat16: products of bfloat16 values are
    exact in float32, so that the bound is that of float32 data.  Widths of 48 products of unit normals: 48 * 2^-23 * 31 *
    0.3 * 1.44 = 8e-5."""
    import ye3t_b200.torch_ops  # noqa: F401
    from ye3t_b200 import runtime as rt
    q, k, v, _, x, y, sl = _inputs(queries, keys, 4, 2, 48, torch.bfloat16, 12)
    layout = rt.StructureLayout(queries, keys, heads=4, key_heads=2, device=DEV)
    _, lse = torch.ops.ye3t_b200.structure_attention(q, k, v, layout.tables, layout.counts, x, y, sl, 0.3)
    want = _definition(q, k, v, x, y, sl, 0.3, queries, keys)[1]
    held = torch.isfinite(want)
    assert torch.equal(held, torch.isfinite(lse))
    assert float((lse[held].double() - want[held]).abs().max()) <= 1e-4


@pytest.mark.parametrize("queries,keys,H,Hk,D", [([300, 129], [300, 129], 4, 2, 64), ([200], [4000], 2, 2, 48),
                                                 ([700], [700], 3, 3, 32), ([260], [400], 2, 1, 128),
                                                 ([1, 2], [900, 300], 4, 2, 64)])
@pytest.mark.parametrize("bias", [True, False])
def test_bfloat16_results_are_rounded_once(queries, keys, H, Hk, D, bias):
    """What bfloat16 results are off by is their own rounding: they are the rounded float64 results but for values beside
    a rounding's edge.  Before it they are within d = 2^-16 of the norm (probabilities in two pieces of 8 bits, sums of
    float32); a value within d of an edge goes to the other side, a step of r = 2^-7 at most, in a share d / r of all:
    sqrt(d r) = 3.5e-4 of the norm, and twice that is allowed."""
    from ye3t_b200 import runtime as rt
    q, k, v, grad, x, y, sl = _inputs(queries, keys, H, Hk, D, torch.bfloat16, D)
    layout = rt.StructureLayout(queries, keys, heads=H, key_heads=Hk, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    places = dict(positions=x, key_positions=y, slopes=sl) if bias else {}
    out = rt.structure_attention(q, k, v, layout, **places)
    got = (out,) + torch.autograd.grad(out, leaves, grad)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    want = _definition(*wide, x, y, sl if bias else 0.0 * sl, D ** -0.5, queries, keys)[0]
    for a, b, what in zip(got, (want,) + torch.autograd.grad(want, wide, grad.double()), ("out", "dq", "dk", "dv")):
        off = (a.detach().double() - b.detach().bfloat16().double()).norm() / b.detach().norm()
        assert float(off) <= 2.0 * 2.0 ** -11.5, (what, float(off))

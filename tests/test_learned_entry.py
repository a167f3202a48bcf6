"""Learned operators: what their entry points write, check and pass on, without a GPU."""

import numpy as np
import pytest


@pytest.mark.parametrize("queries,keys", [([5], [5]), ([1, 1], [5000, 70]), ([300, 20], [300, 0]), ([], [])])
def test_layout_writes_sixteen_counts(queries, keys):
    """Callers reserve sixteen values for the counts, and the size query fills them in as the call does."""
    from ye3t_b200 import _native as nat
    from ye3t_b200 import runtime as rt
    q, k = np.array(queries, np.int64), np.array(keys, np.int64)
    counts = np.full(20, -77, np.int64)
    need = nat.lib().y3b_structure_layout(q.ctypes.data, k.ctypes.data, q.size, 4, 2, counts.ctypes.data, 0, 0)
    assert need >= 2 and (counts[:16] >= 0).all() and (counts[16:] == -77).all()
    packed, sizes = rt._layout_tables(q, k, 4, 2)
    assert packed.size == need
    named = dict(zip(rt._LAYOUT_COUNTS[6:], sizes))
    assert len(sizes) == len(named) == len(rt._LAYOUT_COUNTS) - 6
    assert named["few_slot_count"] == named["few_item_count"]
    assert sizes[:4] + sizes[5:] == counts[:16].tolist()


@pytest.mark.parametrize("queries,keys", [([1] * 8, [5000, 32000, 16384, 9000, 20011, 12000, 30001, 6000]),
                                          ([2] * 200, [5000] * 200)])
def test_layout_of_few_queries_has_no_entry_a_key(queries, keys):
    """A readout's tables go by chunks of its keys: the host work of a batch is not that of its keys."""
    from ye3t_b200 import runtime as rt
    packed, _ = rt._layout_tables(np.array(queries), np.array(keys), 8, 4)
    # an item of eight values a hundred keys in two tables, and some for each structure
    assert packed.size <= 16 * (sum(keys) // 100) + 64 * len(keys)


class _Library:
    """Stands in for the native library: notes which calls are made, and whether the device was current then."""

    def __init__(self):
        self.current, self.calls = 0, {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = self.current
            return 64 if name.endswith("_bytes") else 0
        return call


@pytest.mark.parametrize("current", [0, 1])
def test_native_calls_run_with_the_tensors_device_current(monkeypatch, current):
    """The kernels launch on the current device, which need not be that of the tensors."""
    import contextlib
    from types import SimpleNamespace

    import torch
    from ye3t_b200 import _native as nat
    from ye3t_b200 import runtime as rt
    lib = _Library()
    lib.current = current

    @contextlib.contextmanager
    def device(wanted):
        before, lib.current = lib.current, wanted.index
        yield
        lib.current = before

    class Device(SimpleNamespace):
        type, index = "cuda", 1

    class Tensor(SimpleNamespace):
        """A tensor of the second device, of which only the shape matters."""

        def __init__(self, *shape, dtype=torch.float32):
            super().__init__(shape=torch.Size(shape), dtype=dtype, device=Device())

        def contiguous(self):
            return self

        def new_empty(self, shape, dtype=None):
            return Tensor(*shape, dtype=dtype or self.dtype)

        def stride(self, dim=None):
            return (1, 1, 1) if dim is None else 1

        data_ptr = element_size = numel = lambda self: 4

    monkeypatch.setattr(nat, "lib", lambda: lib)
    monkeypatch.setattr(rt, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: lib.current)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch, "empty", lambda shape, dtype=None, device=None: Tensor(*np.atleast_1d(shape), dtype=dtype))
    monkeypatch.setattr(torch, "empty_like", lambda t: t)
    z = Tensor(5, dtype=torch.int64)
    rt._embedding_forward(Tensor(3, 4), z, 1.0, False)
    rt._embedding_adjoint(Tensor(5, 4), z, 3, 1.0)
    layout = SimpleNamespace(_args=nat.StructureAttentionArgs(), device=Device(), _stream=0)
    q, x, slopes = Tensor(5, 2, 8), Tensor(5, 3), Tensor(2)
    out, lse = rt._attention_forward(q, q, q, x, x, slopes, layout, 1.0, False)
    rt._attention_adjoint(out, q, q, q, x, x, slopes, out, lse, layout, 1.0, True, False)
    launches = {name: dev for name, dev in lib.calls.items() if not name.endswith("_bytes")}
    assert launches == {"y3b_species_embedding": 1, "y3b_species_embedding_adjoint": 1, "y3b_structure_attention": 1,
                        "y3b_structure_attention_adjoint": 1}
    assert lib.current == current

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

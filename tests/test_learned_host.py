"""Learned operators: what is checked on the host, without a GPU."""

import ctypes


import numpy as np
import pytest
import torch


def test_layout_counts_are_checked():
    from ye3t_b200.runtime import StructureLayout
    with pytest.raises(ValueError):
        StructureLayout([3, -1], heads=1)
    with pytest.raises(ValueError):
        StructureLayout([3, 1], [2], heads=1)
    with pytest.raises(ValueError):
        StructureLayout([[3, 1]], heads=1)
    with pytest.raises(ValueError):
        StructureLayout([1.5], heads=1)
    with pytest.raises(ValueError):
        StructureLayout([3], heads=4, key_heads=3)
    with pytest.raises(ValueError):
        StructureLayout([3], heads=0)
    with pytest.raises(ValueError):
        StructureLayout([2**30, 2**30], heads=1)
    with pytest.raises(ValueError):
        StructureLayout([3], heads=1, device="cpu")


def test_cpu_tensors_are_refused():
    from ye3t_b200 import runtime as rt
    with pytest.raises(ValueError):
        rt.species_embedding(torch.zeros(2, 2), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        rt.structure_attention(torch.zeros(2, 1, 4), torch.zeros(2, 1, 4), torch.zeros(2, 1, 4), None)


def test_entry_points_refuse_bad_arguments():
    """The C entry points return an error code before they touch the device."""
    from ye3t_b200 import _native as nat
    lib = nat.lib()
    assert lib.y3b_species_embedding(nat.C64, 0, 1, 1, 0, 8, 1, 1.0, 0, 0, 0) == -1
    assert lib.y3b_species_embedding(nat.F32, 0, 1, 1, 0, 2, 1, 1.0, 0, 0, 0) == -1
    assert lib.y3b_species_embedding(nat.F32, 0, 1, 0, 0, 8, 1, 1.0, 0, 0, 0) == -1
    assert lib.y3b_species_embedding(nat.F32, 0, 1, 1, 0, 8, 1, 1.0, 0, 0, 0) == -1
    assert lib.y3b_species_embedding(nat.F32, 0, 1, 1, 0, 8, 0, 1.0, 0, 0, 0) == 0
    assert lib.y3b_species_embedding_adjoint_workspace_bytes(nat.F32, -1, 1, 1) == -1
    assert lib.y3b_species_embedding_adjoint_workspace_bytes(nat.F32, 1 << 31, 1, 1) == -1
    assert lib.y3b_species_embedding_adjoint_workspace_bytes(nat.F32, 1000, 1000, 8) > 0
    assert lib.y3b_species_embedding_adjoint(nat.F32, 0, 0, 8, 10, 3, 4, 1.0, 0, 0, 0, 0, 0) == -1
    one, minus = np.array([5], np.int64), np.array([-1], np.int64)
    sizes = np.zeros(16, np.int64)
    layout = lambda q, k, h=4, hk=2: lib.y3b_structure_layout(  # noqa: E731
        q.ctypes.data, k.ctypes.data, 1, h, hk, sizes.ctypes.data, 0, 0)
    assert layout(one, one) > 0
    assert layout(minus, one) == -1 and layout(one, minus) == -1 and layout(one, one, 4, 3) == -1
    assert lib.y3b_structure_layout(0, 0, 1, 1, 1, sizes.ctypes.data, 0, 0) == -1
    assert lib.y3b_structure_attention(None, 0, 0, 0, 0, 0, 0) == -1
    a = nat.StructureAttentionArgs()
    a.dtype, a.heads, a.key_heads, a.width = nat.F32, 4, 2, 32
    call = lambda: lib.y3b_structure_attention(ctypes.byref(a), 0, 0, 0, 0, 0, 0)  # noqa: E731
    assert call() == 0  # nothing to do
    a.key_heads = 3
    assert call() == -1 and b"multiple" in lib.y3b_last_error()
    a.key_heads, a.width = 2, 129
    assert call() == -1 and b"width" in lib.y3b_last_error()
    a.width, a.dtype = 32, nat.F64
    assert call() == -1
    a.dtype, a.query_count = nat.BF16, 5
    assert call() == -1
    a.query_count, a.positions = 0, 16
    assert call() == -1 and b"slopes" in lib.y3b_last_error()


def test_argument_struct_layout(tmp_path):
    """The ctypes mirror has the header's size and offsets."""
    import os
    import subprocess
    from ye3t_b200 import _native as nat
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cls = nat.StructureAttentionArgs
    fields = [f[0] for f in cls._fields_]
    src = tmp_path / "layout.c"
    lines = "".join(f'printf("%zu\\n", offsetof(y3b_structure_attention_args, {f}));\n' for f in fields)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ye3t_b200.h"\nint main(void) {\n'
                   'printf("%zu\\n", sizeof(y3b_structure_attention_args));\n' + lines + "return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(repo, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(cls)
    assert out[1:] == [getattr(cls, f).offset for f in fields]


def _random_counts(rng):
    n = int(rng.integers(1, 30))
    big = int(rng.choice([3, 40, 200, 3000]))
    queries, keys = rng.integers(0, big, n), rng.integers(0, big, n)
    if rng.random() < 0.3:
        queries = np.minimum(queries, 2)
    return queries, keys


@pytest.mark.parametrize("seed", range(40))
def test_layout_tables_hold_every_row_once(seed, counts=None):
    """Every query (and key) of a batch is in exactly one small structure, row entry, few-query item set or tile; a
    tile's items are its structure's columns, each once; slots are joined once."""
    from ye3t_b200 import runtime as rt
    rng = np.random.default_rng(seed)
    queries, keys = _random_counts(rng) if counts is None else (np.array(counts), np.array(counts))
    heads, key_heads = ((8, 2), (4, 4), (1, 1))[seed % 3]
    packed, sizes = rt._layout_tables(queries, keys, heads, key_heads)
    counts = dict(zip(rt._LAYOUT_COUNTS[6:], sizes), structure_count=len(queries))
    tables, at = {}, 0
    for name, width, count in rt._LAYOUT_TABLES:
        n = counts["small_32_count"] + counts["small_64_count"] if count is None else counts[count]
        n = n + 1 if name.endswith("offsets") else n
        tables[name] = packed[at:at + width * n].reshape((n, width) if width > 1 else n)
        at += width * n
    assert at == packed.size
    q_off, k_off = tables["query_offsets"], tables["key_offsets"]
    small = {tuple(r) for r in tables["small"]}
    assert len(small) == len(tables["small"]) == counts["small_32_count"] + counts["small_64_count"]
    for k, (a, n, b, m) in enumerate(tables["small"]):
        most = 32 if k < counts["small_32_count"] else 64
        assert n <= most and m <= most
    for side, off, other in (("query", q_off, k_off), ("forward", q_off, k_off), ("key", k_off, q_off)):
        seen = np.zeros(off[-1], int)
        for a, n, b, m in small:
            first, count = (b, m) if side == "key" else (a, n)
            seen[first:first + count] += 1
        for row, structure in tables["key_rows" if side == "key" else "query_rows"]:
            assert off[structure] <= row < off[structure + 1]
            seen[row] += 1
        kinds = ("key",) if side == "key" else (side, "few")
        for kind in kinds:
            items, joins = tables[f"{kind}_items"], tables[f"{kind}_joins"]
            columns, slots = {}, {}
            for row, rows, col, cols, slot, *rest in items:
                structure = int(np.searchsorted(off, row, side="right")) - 1
                assert 1 <= rows <= 128 and off[structure] <= row and row + rows <= off[structure + 1]
                assert not any(rest)
                columns.setdefault((row, rows), []).append((col, cols, structure))
                if slot >= 0:
                    assert slot not in slots
                    slots[slot] = (row, rows)
                else:
                    assert kind != "few"
            assert sorted(slots) == list(range(counts[f"{kind}_slot_count"]))
            for (row, rows), parts in columns.items():
                seen[row:row + rows] += 1
                structure = parts[0][2]
                at = other[structure]
                for col, cols, _ in sorted(p for p in parts if p[1]):
                    assert col == at
                    at += cols
                assert at == other[structure + 1]
            joined = []
            for row, rows, first, count in joins:
                assert all(slots[first + k] == (row, rows) for k in range(count))
                joined += list(range(first, first + count))
            assert sorted(joined) == sorted(slots)
            if kind == "few":
                assert all(i[1] <= 2 for i in items)
        assert (seen == 1).all()


@pytest.mark.parametrize("atoms", [129, 1000, 2048, 5000, 8192, 16384, 20000])
def test_layout_tables_of_one_structure(atoms):
    """The same for one structure, whose tiles are cut by waves."""
    for seed in range(3):
        test_layout_tables_hold_every_row_once(seed, [atoms])

"""The example's page for a growing row, where there is no page or no room left:
nothing that another row holds is written over (plain torch, on the CPU)."""
import importlib.util
import os
import types

import torch

from conftest import ROOT

spec = importlib.util.spec_from_file_location("decode_block", os.path.join(ROOT, "examples", "decode_block.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def cache(refs, lens, tables, S):
    i = lambda x: torch.tensor(x, dtype=torch.int32)
    return types.SimpleNamespace(refs=i(refs), lens=i(lens), tables=i(tables), S=S, width=len(tables[0]))


def test_pages_in_order():
    c = cache([1, 0, 1, 0, 0], [4, 3, 0], [[0, -1], [2, -1], [-1, -1]], 4)
    at, slots = example.grow(c, torch.tensor([2, 0, 1], dtype=torch.int32))
    assert at.tolist() == [0, 4, 3] and slots.tolist() == [4, 12, 11]
    assert c.refs.tolist() == [1, 1, 1, 1, 0] and c.lens.tolist() == [5, 4, 1]
    assert c.tables.tolist() == [[0, 3], [2, -1], [1, -1]]


def test_no_page_left():
    c = cache([1, 1, 0], [4, 4], [[0, -1], [1, -1]], 4)
    at, slots = example.grow(c, torch.tensor([0, 1], dtype=torch.int32))
    assert slots[0] == 8 and slots[1] < 0  # (stored nowhere, and attention reports the row)
    assert c.refs.tolist() == [1, 1, 1] and c.tables.tolist() == [[0, 2], [1, -1]] and c.lens.tolist() == [5, 5]
    at, slots = example.grow(c, torch.tensor([0, 1], dtype=torch.int32))
    assert slots[0] == 9 and slots[1] < 0
    assert c.refs.tolist() == [1, 1, 1] and c.tables.tolist() == [[0, 2], [1, -1]]


def test_row_at_its_width():
    c = cache([1, 1, 1, 0], [8, 3], [[0, 1], [2, -1]], 4)
    for n in (9, 10):
        at, slots = example.grow(c, torch.tensor([0, 1], dtype=torch.int32))
        assert slots[0] < 0 and c.lens[0] == n
        assert c.tables[0].tolist() == [0, 1]
    # the other row took the free page, none was lost to the full one
    assert c.refs.tolist() == [1, 1, 1, 1] and c.tables[1].tolist() == [2, 3] and slots[1] == 12

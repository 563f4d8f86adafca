"""The 4-bit paged KV cache (ctransformers_amd/ops.py, csrc/engine_kv4.h) at the edges of what its calls accept."""
import pytest
import torch

from ctransformers_amd import ops
from test_kv4 import dev  # noqa: F401  (the fixture)


def ints(dev, *x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---- pages --------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("length,add", [(2**31 - 1, 2**31 - 1), (1, 2**31 - 1), (2**31 - 1, 1), (2**30, 2**30)])
def test_room_behind_lengths_near_2_31(dev, length, add):
    """pages of one token: the end of what is asked for lies at 2^31 and beyond, far outside of the table.  Refused, nothing has changed, its neighbours included."""
    pages = torch.zeros((8, 16), dtype=torch.uint8, device=dev)
    table, lens, refs = ints(dev, [0, 1, -1, -1], [2, -1, -1, -1]), ints(dev, length, 1), ints(dev, 1, 1, 1, 0, 0, 0, 0, 0)
    t, n, r, short = ops.kv_reserve(pages, table, lens, refs, ints(dev, add, 1), page_tokens=1)
    assert int(short) == -1
    assert torch.equal(t, table) and torch.equal(n, lens) and torch.equal(r, refs)


def test_no_length_beyond_2_31(dev):
    """a table with room for it, but no int32 that could hold the length: refused; the largest length that fits is not"""
    pages = torch.zeros((4, 16), dtype=torch.uint8, device=dev)
    table, refs = ints(dev, [0, 1, -1, -1]), ints(dev, 1, 1, 0, 0)
    for length, add, want in ((2**31 - 1, 10, -1), (2**31 - 10, 10, -1), (2**31 - 10, 9, 0), (2**30, 2**30, -1)):
        lens = ints(dev, length)
        t, n, r, short = ops.kv_reserve(pages, table, lens, refs, ints(dev, add), page_tokens=2**30)
        assert int(short) == want and n.tolist() == [length + (0 if want else add)]
        assert torch.equal(t, table) and torch.equal(r, refs)

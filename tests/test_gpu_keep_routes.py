"""Moves of rows in a paged cache and the choice of keys, by every route that sizes and numbers of heads take, exactly."""
import pytest
import torch

from oracle import tree

from test_gpu_paged import BF16, E4M3, _batch, _bits, _full_cache
from test_gpu_evict import _planes, _same

pytestmark = pytest.mark.gpu


def _ops():
    from fractaltensor_b200 import ops
    return ops


def test_rows_that_stay_need_no_page():
    """A sequence of a batch's padding has no pages, and a path of token 0 alone, which stays where it is; a second token is a row without a place."""
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    table, first = i32([[2, 0], [-1, -1]]), i32([7, -4])
    cache = _full_cache(4, 2, 16, 64, BF16, 3)
    before = [c.clone() for c in cache]
    kept = i32([[0, 2, 3, -1], [0, -1, -1, -1]])
    ops.paged_cache_keep(cache, kept, i32([3, 1]), table, first=first)
    ops.check_status()
    for c, x in zip(cache, before):
        x[2, :, 8] = x[2, :, 9]
        x[2, :, 9] = x[2, :, 10]
        assert torch.equal(c, x)
    kept[1, 1] = 2
    ops.paged_cache_keep(cache, kept[1:].contiguous(), i32([2]), table[1:].contiguous(), first=first[1:].contiguous())
    with pytest.raises(FtbError):
        ops.check_status()
    assert all(torch.equal(c, x) for c, x in zip(cache, before))

"""Sequences with more new tokens than positions: those in front of position 0 see nothing and are seen by none."""
import math

import pytest
import torch

from oracle import tree

from test_gpu_paged import BF16, E4M3, _batch, _full_cache, _numbers
from test_gpu_tree import _check, _tree_rows

pytestmark = pytest.mark.gpu

SHAPES = [
    # group, new, lens
    (4, [5, 3], [3, 40]),
    (4, [40, 33], [20, 300]),
    (8, [33, 40], [32, 1]),
    (2, [150, 9], [140, 0]),
    (1, [1, 1], [0, 9]),
]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("width", [0, 4000])
@pytest.mark.parametrize("group,new,lens", SHAPES)
def test_attention(eight_bit, width, group, new, lens):
    from fractaltensor_b200 import ops
    kv, d, page = 4, 128, 16
    table, ln, st, pages = _batch(new, lens, page, width=width)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    mask = _tree_rows(new, st, T, 7)
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    lse = torch.full((T, kv * group), 7.0, device="cuda")
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.08, tree=mask.cuda(), lse=lse)
    ops.check_status()
    _check(o, lse, q, cache, table, ln, st, 0.08, mask=mask)
    front = [int(st[b]) + i for b in range(len(new)) for i in range(new[b] - lens[b])]
    assert len(front) > 0 and bool((o[front] == 0).all()) and bool(torch.isneginf(lse[front]).all())


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("width", [0, 4000])
@pytest.mark.parametrize("group,new,lens", SHAPES)
def test_weights(eight_bit, width, group, new, lens):
    from fractaltensor_b200 import ops
    kv, d, page = 4, 64, 16
    table, ln, st, pages = _batch(new, lens, page, width=width)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    scale = 1.0 / math.sqrt(d)
    lse = torch.empty(T, kv * group, device="cuda")
    weights = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)).cuda()
    before = weights.clone()
    args = (table.cuda(), ln.cuda(), st.cuda())
    ops.paged_attention(q, cache, *args, scale=scale, lse=lse)
    ops.paged_attention_weights(q, cache, weights, lse, *args, scale=scale)
    ops.check_status()
    want, tol = tree.weights(before, q, cache, lse, table, ln, st, scale)
    assert bool(((weights.double().cpu() - want).abs() <= tol).all())

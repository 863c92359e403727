"""Accumulated attention weight of long sequences and in wide tables, as close to 64 bits as its roundings allow."""
import math

import pytest
import torch

from oracle import tree

from test_gpu_paged import BF16, E4M3, F16, _batch, _bits, _full_cache, _numbers

pytestmark = pytest.mark.gpu


def _ops():
    from fractaltensor_b200 import ops
    return ops


def _close(before, q, cache, lse, table, ln, st, scale):
    """-> (weights, tolerance), counted step by step.

    Products of 16-bit numbers are exact in 32 bits.  A score's sum takes them in d / 8 steps or fewer, each of which cuts off less than 2^-23
    of what the sum can have come to: its positive products or its negative ones, whichever are more.  A bf16 query over an 8-bit cache keeps each
    number to 2^-25 of its largest.  The argument of the exponential is rounded once, the logarithm before it too, and the scale twice: 2^-24 each of what they are;
    the exponential is good to 2^-22.  A key's sum of n terms is n additions of half a step, and one more for the number that was there."""
    k = tree.paged.dense(cache, 0)
    T, heads, d = q.shape
    kv, page = k.shape[1], k.shape[2]
    rescaled = q.dtype == BF16 and len(cache) == 4
    out, tol, terms = before.cpu().double().clone(), torch.zeros(before.shape, dtype=torch.float64), torch.zeros(before.shape)
    q, lse = q.cpu().double(), lse.cpu().double()
    where = tree.paged.places(table, ln, st, page, T)
    for b, pos in where:
        out[int(table[b, pos // page]), :, pos % page] = 0.0
    old = out.abs().clone()
    g = torch.arange(heads) * kv // heads
    for t, (b, pos) in enumerate(where):
        j = torch.arange(pos + 1)
        rows = table[b].long()[j // page]
        kj = k[rows, :, j % page]
        for h in range(heads):
            products = kj[:, g[h]] * q[t, h] * scale
            x, most = products.sum(1), torch.maximum(products.clamp(min=0).sum(1), -products.clamp(max=0).sum(1))
            off = d // 8 * 2.0 ** -23 * most + 2.0 ** -24 * ((x - lse[t, h]).abs() + lse[t, h].abs() + 2 * x.abs()) + 2.0 ** -22
            if rescaled:
                off = off + 2.0 ** -25 * scale * q[t, h].abs().max() * kj[:, g[h]].abs().sum(1)
            p = torch.exp(x - lse[t, h])
            out[rows, g[h], j % page] += p
            tol[rows, g[h], j % page] += p * off
            terms[rows, g[h], j % page] += 1
    return out, tol + (terms + 1) * 2.0 ** -24 * out.abs() + 2.0 ** -24 * old


def _weigh(kv, group, d, page, new, lens, dtype, eight_bit, launches, width=0):
    """launches: 1: the kernel for few rows; 3: packing, the one for many and the join; 4: both."""
    ops = _ops()
    from fractaltensor_b200._lib import lib
    table, ln, st, pages = _batch(new, lens, page, width=width)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else dtype, 3)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), dtype, 9, spread=0.3).cuda()
    scale = 1.0 / math.sqrt(d)
    lse = torch.empty(T, kv * group, device="cuda")
    weights = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)).cuda()
    before = weights.clone()
    args = (table.cuda(), ln.cuda(), st.cuda())
    ops.paged_attention(q, cache, *args, scale=scale, lse=lse)
    n = lib.ftb_launch_count()
    ops.paged_attention_weights(q, cache, weights, lse, *args, scale=scale)
    assert lib.ftb_launch_count() - n == launches
    ops.check_status()
    want, tol = _close(before, q, cache, lse, table, ln, st, scale)
    err = (weights.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol).nan_to_num(9e9).max()), bad.nonzero()[:5].tolist())
    again = before.clone()
    ops.paged_attention_weights(q, cache, again, lse, *args, scale=scale)
    assert torch.equal(_bits(again), _bits(weights))


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,group,d,page,new,lens,launches", [
    (2, 4, 128, 16, [1, 1], [900, 333], 1),    # tiles of 8 rows, a token each
    (2, 16, 128, 16, [1], [900], 1),           # tiles of 16
    (1, 4, 64, 32, [7], [500], 1),             # two of them
    (2, 4, 128, 16, [25], [700], 3),           # 128 rows on the tensor cores
    (1, 3, 64, 64, [30, 23], [600, 257], 4),
])
def test_close(dtype, eight_bit, kv, group, d, page, new, lens, launches):
    _weigh(kv, group, d, page, new, lens, dtype, eight_bit, launches)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("group,d,page,new,lens,launches", [
    (4, 128, 64, [1], [40_003], 1),            # a token
    (4, 64, 16, [6], [20_011], 1),             # two tiles of 16 rows
    (2, 64, 128, [35], [20_011], 3),           # many rows behind many blocks that all of them see
    (2, 64, 32, [35, 1, 9], [9001, 15_000, 44], 1),
    (2, 64, 32, [65, 1, 9], [9001, 15_000, 44], 4),
])
def test_long_sequences(eight_bit, group, d, page, new, lens, launches):
    _weigh(1, group, d, page, new, lens, BF16, eight_bit, launches)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens,launches", [([5, 9], [300, 77], 4), ([12], [301], 3), ([1, 1, 1], [300, 20, 1], 1)])
def test_tables_wider_than_the_sequences(eight_bit, new, lens, launches):
    """Rows of a table for sequences of 128 000 keys: a few dozen rows go to the tensor cores."""
    _weigh(2, 4, 128, 128, new, lens, F16, eight_bit, launches, width=1000)

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


# ----------------------------------------------------------------------------------- moves in the same pages
def _steps(n, K, pattern, g):
    """`K` of n positions or fewer that ascend, so that what a step writes lies close to what others read."""
    if pattern < 6:  # all of them some places further on, from the start or behind a stretch that stays
        by = (1, 63, 64, 257, 512, 1025)[pattern]
        stay = (0, 0, 5, 100, 1, 0)[pattern]
        return torch.cat([torch.arange(stay), torch.arange(stay, K) + by])[:K]
    if pattern == 6:  # four of every five
        return torch.arange(K) + torch.arange(K) // 4
    return torch.randperm(n, generator=g)[:K].sort().values


def _moved(planes, kept, counts, table, page):
    """oracle.tree.keep for positions from 0 on, a head at a time."""
    after = [x.clone() for x in planes]
    B, kv = kept.shape[:2]
    for b in range(B):
        n = int(counts[b])
        to = torch.arange(n)
        for h in range(kv):
            src = kept[b, h, :n].long()
            for x, y in zip(planes, after):
                y[table[b, to // page].long(), h, to % page] = x[table[b, src // page].long(), h, src % page]
    return after


# Up to 9 heads (of 148 SMs): parts of a row, clusters of 8; up to 55: whole rows, clusters of 8; up to 222: clusters of 4; more: a CTA.
HEADS = [(1, 9), (1, 10), (2, 8), (5, 11), (7, 8), (10, 8), (37, 6), (223, 1), (30, 8)]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,kv", HEADS)
def test_moves_in_place(B, kv, d, eight_bit):
    """Every route goes through several steps, each of which reads what the ones in front of it wrote next to."""
    ops = _ops()
    page = 32
    K = 2300 if B * kv <= 55 else 1150 if B * kv <= 222 else 400
    n = K + 1100 if B * kv <= 222 else K + 300
    table, _, _, pages = _batch([0] * B, [n] * B, page)
    g = torch.Generator().manual_seed(B * kv + d)
    kept = torch.full((B, kv, K), -1, dtype=torch.int32)
    counts = torch.full((B,), K, dtype=torch.int32)
    for b in range(B):
        rows = [_steps(n, K, p, g) for p in range(8)]
        rows = [r for r in rows if int(r[-1]) < n]
        mine = [rows[(b + h) % len(rows)] for h in range(kv)]
        counts[b] = min(len(r) for r in mine)
        for h in range(kv):
            kept[b, h, : len(mine[h])] = mine[h].int()
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3)
    weights = torch.rand(pages, kv, page, generator=g).cuda()
    planes = _planes(cache, weights)
    before = [x.clone() for x in planes]
    want = _moved([x.cpu() for x in planes], kept, counts, table, page)
    args = (cache, kept.cuda(), counts.cuda(), table.cuda())
    for _ in range(3):
        for x, y in zip(planes, before):
            x.copy_(y)
        ops.paged_cache_keep(*args, weights=weights)
        _same(planes, want)
    ops.check_status()


# ------------------------------------------------------------------------------------------------ eviction
def _chosen(weights, table, lens, keep, recent):
    """oracle.tree.choose by sorts that keep the order of equal ones."""
    B, kv, page = len(lens), weights.shape[1], weights.shape[2]
    kept = torch.full((B, kv, keep), -1, dtype=torch.int32)
    for b in range(B):
        n = int(lens[b])
        if n <= keep:
            kept[b, :, :n] = torch.arange(n).int()
            continue
        j = torch.arange(n - recent)
        w = weights[table[b, j // page].long(), :, j % page].T  # [kv, keys]
        nan = torch.isnan(w)
        order = torch.sort(torch.where(nan, -torch.inf, w), dim=1, descending=True, stable=True).indices
        order = order.gather(1, torch.sort(nan.gather(1, order).int(), dim=1, stable=True).indices)
        kept[b, :, : keep - recent] = order[:, : keep - recent].sort(1).values.int()
        kept[b, :, keep - recent:] = torch.arange(n - recent, n).int()
    return torch.tensor([min(int(n), keep) for n in lens], dtype=torch.int32), kept


def _weights(pages, kv, page, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(pages, kv, page, generator=g)
    w = torch.where(torch.rand(w.shape, generator=g) < 0.5, (w * 4).round() / 4, w)
    w = torch.where(torch.rand(w.shape, generator=g) < 0.01, float("nan"), w)
    return torch.where(torch.rand(w.shape, generator=g) < 0.01, -float("inf"), w)


def _evicted(B, kv, d, page, lens, keep, recent, eight_bit, width=0):
    ops = _ops()
    table, ln, _, pages = _batch([0] * B, lens, page, width=width)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3)
    weights = _weights(pages, kv, page, 5)
    want_lens, want_kept = _chosen(weights, table, lens, keep, recent)
    weights = weights.cuda()
    planes = _planes(cache, weights)
    want = _moved([x.cpu() for x in planes], want_kept, want_lens, table, page)
    now, kept = ops.paged_cache_evict(cache, weights, table.cuda(), ln.cuda(), keep, recent)
    ops.check_status()
    assert torch.equal(now.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
    _same(planes, want)


def test_the_sorts_choose_what_the_oracle_does():
    weights = _weights(12, 2, 16, 1)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(2)).view(2, 6).int()
    for keep, recent in ((10, 0), (50, 7), (90, 90)):
        for x, y in zip(_chosen(weights, table, [96, 40], keep, recent), tree.choose(weights, table, [96, 40], keep, recent)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("B,kv", HEADS)
def test_evictions_in_place(B, kv, eight_bit):
    lens = [(2900, 1500, 900, 3100)[b % 4] if B * kv <= 222 else (700, 300, 450, 690)[b % 4] for b in range(B)]
    _evicted(B, kv, 64, 32, lens, 1200 if B * kv <= 222 else 310, 100, eight_bit)


@pytest.mark.parametrize("B,kv,lens,keep,recent", [
    (19, 2, 60000, 700, 30),   # one CTA a head, which holds 49 152 keys: the others are looked up again for every digit
    (40, 1, 49200, 20000, 0),  # a few behind them
    (19, 2, 52000, 51999, 7),
    (7, 1, 410000, 900, 100),  # the same of a cluster's CTAs, 8 of 49 152
    (3, 1, 800000, 900, 100),  # and 16
])
def test_more_keys_than_a_cta_holds(B, kv, lens, keep, recent):
    _evicted(B, kv, 64, 128, [lens] + [(200, 5, 1100)[b % 3] for b in range(B - 1)], keep, recent, False)


@pytest.mark.parametrize("B,kv", [(1, 4), (5, 8), (20, 2)])
def test_tables_wider_than_the_sequences(B, kv):
    """Rows of a table for much longer sequences than there are now."""
    _evicted(B, kv, 64, 16, [(600, 90, 333)[b % 3] for b in range(B)], 100, 10, False, width=8200)

"""Accumulated attention weight, eviction and moves of rows in a paged cache, against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import tree

from test_gpu_paged import BF16, E4M3, F16, _batch, _bits, _full_cache, _numbers

pytestmark = pytest.mark.gpu


def _ops():
    from fractaltensor_b200 import ops
    return ops


def _planes(cache, weights=None):
    return [x.view(torch.uint8) if x.dtype == E4M3 else x for x in cache] + ([weights] if weights is not None else [])


def _same(planes, want):
    for x, y in zip(planes, want):
        assert torch.equal(_bits(x), _bits(y))


# ----------------------------------------------------------------------------------------------- weights
SHAPES = [
    # kv, group, d, page, new, lens, window
    (1, 1, 64, 16, [1], [1], None),
    (8, 4, 128, 16, [1], [777], None),
    (2, 8, 128, 64, [1, 1, 1], [5, 64, 333], None),
    (2, 1, 64, 32, [1, 0, 1, 1], [31, 7, 0, 65], None),
    (1, 16, 128, 128, [1, 1], [129, 511], None),
    (2, 3, 64, 16, [1, 5, 2], [100, 5, 47], None),
    (1, 71, 64, 16, [1, 2], [70, 33], None),
    (4, 2, 128, 16, [7, 1, 30], [7, 300, 91], None),
    (1, 4, 128, 64, [130], [130], None),
    (2, 4, 128, 16, [67, 150], [500, 151], None),
    (1, 2, 128, 32, [300], [1200], None),
    (1, 8, 64, 16, [6, 4, 1], [777, 100, 900], 400),
    (2, 4, 128, 16, [1, 1], [500, 40], 1),
    (1, 4, 64, 16, [200], [400], 33),
    (1, 2, 128, 64, [140, 20], [700, 20], 150),
    (1, 1, 128, 128, [520], [520], None),
]


def _weigh_check(got, before, q, cache, lse, table, ln, st, scale, window=None):
    want, tol = tree.weights(before, q, cache, lse, table, ln, st, scale, window)
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol).nan_to_num(9e9).max()), bad.nonzero()[:5].tolist())


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", SHAPES)
def test_weights(dtype, eight_bit, kv, group, d, page, new, lens, window):
    """Unwritten rows of the pages hold NaN; weights of keys that nobody sees keep what they hold."""
    ops = _ops()
    table, ln, st, pages = _batch(new, lens, page, front=1)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else dtype, 3, table, ln)
    T = int(st[-1]) + 2
    q = _numbers((T, (kv * group + 1) * d), dtype, 9, spread=0.3).cuda()[:, d:].unflatten(1, (kv * group, d))
    scale = 1.0 / math.sqrt(d)
    lse = torch.full((T, kv * group), float("nan"), device="cuda")
    weights = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)).cuda()
    before = weights.clone()
    args = (table.cuda(), ln.cuda(), st.cuda())
    ops.paged_attention(q, cache, *args, scale=scale, window=window, lse=lse)
    ops.paged_attention_weights(q, cache, weights, lse, *args, scale=scale, window=window)
    ops.check_status()
    _weigh_check(weights, before, q, cache, lse, table, ln, st, scale, window)
    # twice the same is the same bits
    twice = before.clone()
    ops.paged_attention_weights(q, cache, twice, lse, *args, scale=scale, window=window)
    assert torch.equal(_bits(twice), _bits(weights))


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [40, 70, 3]), ([50, 9], [60, 300]), ([300], [400])])
def test_rows_that_are_not_finite_add_nothing(eight_bit, new, lens):
    ops = _ops()
    kv, group, d, page = 2, 4, 128, 32
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    args = (table.cuda(), ln.cuda(), st.cuda())
    lse = torch.empty(T, kv * group, device="cuda")
    ops.paged_attention(q, cache, *args, scale=0.08, lse=lse)
    lse[::2, 1], lse[0, 3], lse[-1, 2] = float("nan"), float("inf"), -float("inf")
    q[::2, 1] = float("nan")
    weights = torch.rand(pages, kv, page).cuda()
    before = weights.clone()
    ops.paged_attention_weights(q, cache, weights, lse, *args, scale=0.08)
    ops.check_status()
    _weigh_check(weights, before, q.nan_to_num(0.0), cache, lse, table, ln, st, 0.08)


@pytest.mark.parametrize("new,lens", [([1, 1], [90, 40]), ([3], [70]), ([20, 30], [400, 30]), ([200], [600])])
def test_keys_of_minus_infinity_weigh_nothing(new, lens):
    """Scores of -inf are ordinary: of such keys nothing is added, and beside them everything."""
    ops = _ops()
    kv, group, d, page = 2, 3, 128, 16
    table, ln, st, pages = _batch(new, lens, page)
    k, v = _full_cache(pages, kv, page, d, BF16, 3)
    for b, n in enumerate(lens):
        for j in (0, n // 2, n // 3):
            if j != n - 1:
                k[int(table[b, j // page]), :, j % page, 5] = -float("inf")
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    q[..., 5] = q[..., 5].abs() + 0.5
    args = (table.cuda(), ln.cuda(), st.cuda())
    seen = torch.arange(T) if T <= 3 else torch.tensor([t for b in range(len(new)) for t in range(int(st[b]), int(st[b + 1])) if lens[b] - new[b] + t - int(st[b]) > 0])
    lse = torch.empty(T, kv * group, device="cuda")
    ops.paged_attention(q, (k, v), *args, scale=0.08, lse=lse)
    assert bool(torch.isfinite(lse[seen.cuda()]).all())
    weights = torch.zeros(pages, kv, page, device="cuda")
    ops.paged_attention_weights(q, (k, v), weights, lse, *args, scale=0.08)
    ops.check_status()
    assert bool(torch.isfinite(weights).all())
    _weigh_check(weights, weights * 0, q, (k, v), lse, table, ln, st, 0.08)


@pytest.mark.parametrize("by", [2.0 ** 100, 2.0 ** -100])
def test_scales_of_queries_and_keys_that_cancel(by):
    ops = _ops()
    kv, group, d, page, new, lens = 1, 4, 128, 16, [3, 1], [90, 33]
    table, ln, st, pages = _batch(new, lens, page)
    k = _numbers((pages, kv, page, d), torch.float32, 3)
    from oracle import paged
    (kc, ke), (vc, ve) = paged.quantise(k.double() / by), paged.quantise(k)
    cache = tuple(x.cuda() for x in (kc.view(E4M3), vc.view(E4M3), ke, ve))
    q = (_numbers((4, kv * group, d), torch.float32, 1) * by).to(BF16).cuda()
    args = (table.cuda(), ln.cuda(), st.cuda())
    lse = torch.empty(4, kv * group, device="cuda")
    ops.paged_attention(q, cache, *args, scale=0.1, lse=lse)
    weights = torch.zeros(pages, kv, page).cuda()
    ops.paged_attention_weights(q, cache, weights, lse, *args, scale=0.1)
    ops.check_status()
    assert bool(torch.isfinite(lse).all())
    _weigh_check(weights, weights * 0, q, cache, lse, table, ln, st, 0.1)
    assert abs(float(weights.sum()) - 4 * kv * group) < 1e-3


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 1], [40, 70]), ([200, 33], [260, 300])])
def test_a_window_of_everything(eight_bit, new, lens):
    ops = _ops()
    kv, group, d, page = 2, 4, 64, 16
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    args = (table.cuda(), ln.cuda(), st.cuda())
    lse = torch.empty(T, kv * group, device="cuda")
    ops.paged_attention(q, cache, *args, scale=0.1, lse=lse)
    got = []
    for window in (None, 2 ** 31 - 1, 2 ** 40):
        got.append(torch.zeros(pages, kv, page, device="cuda"))
        ops.paged_attention_weights(q, cache, got[-1], lse, *args, scale=0.1, window=window)
    ops.check_status()
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("eight_bit", [False, True])
def test_many_stretches_a_piece(eight_bit):
    """Dozens of sequences with one tile of rows or two to a block of keys: every CTA goes through many blocks, of all lengths."""
    ops = _ops()
    kv, group, d, page = 3, 3, 64, 32
    g = torch.Generator().manual_seed(7)
    new = torch.randint(6, 60, (90,), generator=g).tolist()
    lens = [n + int(m) for n, m in zip(new, torch.randint(0, 700, (90,), generator=g))]
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    args = (table.cuda(), ln.cuda(), st.cuda())
    lse = torch.empty(T, kv * group, device="cuda")
    ops.paged_attention(q, cache, *args, scale=0.1, lse=lse)
    weights = torch.rand(pages, kv, page, generator=g).cuda()
    before = weights.clone()
    ops.paged_attention_weights(q, cache, weights, lse, *args, scale=0.1)
    ops.check_status()
    _weigh_check(weights, before, q, cache, lse, table, ln, st, 0.1)


def test_weights_of_a_page_that_is_not_there():
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    table, ln, st, pages = _batch([1, 1], [40, 20], 16)
    cache = _full_cache(pages, 1, 16, 64, F16, 3)
    q = _numbers((2, 2, 64), F16, 1).cuda()
    lse = torch.full((2, 2), 3.0, device="cuda")
    weights = torch.zeros(pages, 1, 16, device="cuda")
    good = weights.clone()
    ops.paged_attention_weights(q, cache, good, lse, table.cuda(), ln.cuda(), st.cuda())
    ops.check_status()
    bad = table.clone()
    bad[0, 1] = pages
    ops.paged_attention_weights(q, cache, weights, lse, bad.cuda(), ln.cuda(), st.cuda())
    with pytest.raises(FtbError):
        ops.check_status()
    good[int(table[0, 1])] = 0.0
    assert torch.equal(weights, good)
    ops.paged_attention_weights(q, cache, weights, lse, table.cuda(), (ln + 1000).cuda(), st.cuda())  # behind the table's width
    with pytest.raises(FtbError):
        ops.check_status()


# ------------------------------------------------------------------------------------------------- moves
@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("kv,d,page,K,first,lens,per_head,weighed,elsewhere", [
    (2, 128, 16, 5, [10, 0, 33], [40, 5, 90], False, False, False),
    (3, 64, 32, 9, [10, 0, 33], [40, 9, 90], False, True, False),
    (8, 128, 64, 64, [7], [600], True, True, False),
    (1, 64, 16, 700, None, [1500, 800, 720], True, True, False),
    (2, 128, 16, 1300, None, [2600], True, False, False),
    (2, 128, 16, 1300, None, [2600, 1301], True, True, True),
    (2, 64, 128, 40, [100, 3], [300, 50], False, False, True),
    (1, 128, 32, 2, [0], [4], False, False, False),
])
def test_keep(eight_bit, kv, d, page, K, first, lens, per_head, weighed, elsewhere):
    ops = _ops()
    B = len(lens)
    table, ln, _, pages = _batch([0] * B, lens, page, extra_pages=2 + (B * -(-K // page) + 8 if elsewhere else 0))
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3)
    weights = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)).cuda() if weighed else None
    g = torch.Generator().manual_seed(K)
    f = torch.tensor(first or [0] * B, dtype=torch.int32)
    room = [lens[b] - int(f[b]) for b in range(B)]
    counts = torch.tensor([min(K, room[b]) - (b % 2) for b in range(B)], dtype=torch.int32)
    kept = torch.full((B, kv, K), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(kv):
            kept[b, h, : int(counts[b])] = torch.randperm(room[b], generator=g)[: int(counts[b])].sort().values.int()
    kept[:, :, 0] = 0
    kept = kept if per_head else kept[:, 0].contiguous()
    into = None
    if elsewhere:
        free = torch.tensor([p for p in range(pages) if p not in set(table.flatten().tolist())], dtype=torch.int32)
        W = -(-(int(f.max()) + K) // page)
        into = torch.full((B, W + 1), -1, dtype=torch.int32)
        at = 0
        for b in range(B):
            lo, hi = int(f[b]) // page, -(-(int(f[b]) + int(counts[b])) // page)
            into[b, lo:hi] = free[at: at + hi - lo]
            at += hi - lo
    planes = _planes(cache, weights)
    want = tree.keep([x.cpu() for x in planes], kept, counts, table, f, into)
    ops.paged_cache_keep(cache, kept.cuda(), counts.cuda(), table.cuda(), first=f.cuda() if first else None, into=into.cuda() if elsewhere else None,
                         weights=weights)
    ops.check_status()
    _same(planes, want)


def test_keep_without_a_place():
    """Rows with a negative number or without a page are not moved and set the status word; counts behind K are cut."""
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    cache = _full_cache(4, 1, 16, 64, BF16, 3)
    before = [c.cpu() for c in cache]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    for kept, counts, tab, moved in (([0, -1, 5], 3, table, [0, 5]), ([0, 4, 60], 3, table, [0, 4]), ([1, 2, 20], 3, i32([[2, 9, 3]]), [1, 2])):
        for c, x in zip(cache, before):
            c.copy_(x)
        ops.paged_cache_keep(cache, i32([kept]).cuda(), i32([counts]).cuda(), tab.cuda())
        with pytest.raises(FtbError):
            ops.check_status()
        for c, x in zip(cache, before):
            want = x.clone()
            for i, k in enumerate(kept):
                if k in moved:
                    want[2, 0, i] = x[2, 0, k]
            assert torch.equal(c.cpu(), want)
    for c, x in zip(cache, before):
        c.copy_(x)
    ops.paged_cache_keep(cache, i32([[1, 2]]).cuda(), i32([77]).cuda(), table.cuda())
    ops.paged_cache_keep(cache, i32([[1, 2]]).cuda(), i32([-3]).cuda(), table.cuda())
    ops.check_status()
    assert all(torch.equal(c.cpu()[2, 0, :2], x[2, 0, 1:3]) for c, x in zip(cache, before))


# ---------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("kv,d,page,lens,keep,recent,elsewhere", [
    (2, 128, 16, [100, 7, 40, 0], 32, 8, False),
    (1, 64, 32, [5], 1, 0, False),
    (1, 64, 32, [5], 1, 1, False),
    (3, 128, 64, [700, 300], 299, 0, False),
    (2, 64, 128, [1500], 1499, 3, False),
    (2, 64, 16, [1500, 20], 64, 64, True),
    (1, 128, 16, [5000, 1200, 1300], 1200, 100, True),
    (1, 128, 16, [9000], 2500, 500, False),
    (2, 64, 128, [40000], 700, 30, False),
    (2, 64, 128, [70000], 700, 30, False),
])
def test_evict(eight_bit, kv, d, page, lens, keep, recent, elsewhere):
    ops = _ops()
    B = len(lens)
    per = [-(-min(n, keep) // page) for n in lens]
    table, ln, _, pages = _batch([0] * B, lens, page, extra_pages=2 + (sum(per) if elsewhere else 0))
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else F16, 3)
    g = torch.Generator().manual_seed(2)
    weights = torch.randn(pages, kv, page, generator=g)
    weights = torch.where(torch.rand(weights.shape, generator=g) < 0.6, (weights * 2).round() / 2, weights)  # many of them equal, -0 among them
    weights = torch.where(torch.rand(weights.shape, generator=g) < 0.02, float("nan"), weights)
    weights = torch.where(torch.rand(weights.shape, generator=g) < 0.01, float("inf"), weights)
    weights = torch.where(torch.rand(weights.shape, generator=g) < 0.01, -float("inf"), weights)
    into = None
    if elsewhere:
        free = [p for p in range(pages) if p not in set(table.flatten().tolist())]
        into = torch.full((B, max(per)), -1, dtype=torch.int32)
        for b in range(B):
            into[b, : per[b]] = torch.tensor(free[sum(per[:b]): sum(per[: b + 1])])
    want_lens, want_kept = tree.choose(weights, table, lens, keep, recent)
    weights = weights.cuda()
    planes = _planes(cache, weights)
    want = tree.keep([x.cpu() for x in planes], want_kept, want_lens, table, None, into)
    now, kept = ops.paged_cache_evict(cache, weights, table.cuda(), ln.cuda(), keep, recent, into=into.cuda() if elsewhere else None)
    ops.check_status()
    assert torch.equal(now.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
    _same(planes, want)


def test_evict_all_equal_and_too_long():
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    table = torch.tensor([[2, 0, 3], [1, 4, 5]], dtype=torch.int32).cuda()
    cache = _full_cache(6, 2, 16, 64, BF16, 3)
    weights = torch.zeros(6, 2, 16, device="cuda")
    now, kept = ops.paged_cache_evict(cache, weights, table, torch.tensor([48, 30], dtype=torch.int32).cuda(), 10, 4)
    ops.check_status()
    assert now.tolist() == [10, 10]
    assert kept[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 44, 45, 46, 47] and kept[1, 1].tolist() == [0, 1, 2, 3, 4, 5, 26, 27, 28, 29]
    now, kept = ops.paged_cache_evict(cache, weights, table, torch.tensor([49, -2], dtype=torch.int32).cuda(), 10, 4)
    with pytest.raises(FtbError):  # 49 keys do not fit the table: 48 are looked at
        ops.check_status()
    assert now.tolist() == [10, 0] and kept[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 44, 45, 46, 47] and kept[1, 0].tolist() == [-1] * 10


@pytest.mark.parametrize("kind", ["powers of four", "halves of an octave", "last bits", "two values"])
@pytest.mark.parametrize("sequences,width", [(1, 0), (1, 600), (1, 4100), (40, 0), (16, 3100)])
def test_evict_by_digits(kind, sequences, width):
    """Weights whose order is known after one digit of their bits, two or three, or only after the last."""
    ops = _ops()
    page, keep, recent, n = 16, 50, 6, 5000 if kind == "two values" else 240
    table, ln, _, pages = _batch([0] * sequences, [n] * sequences, page)
    table = torch.nn.functional.pad(table, (0, max(0, width - table.shape[1])), value=-1)  # (as wide as for sequences of one CTA, or of a cluster of 8 or 16)
    cache = _full_cache(pages, 2, page, 64, BF16, 3)
    g = torch.Generator().manual_seed(7)
    i = torch.arange(pages * 2 * page, dtype=torch.int64)[torch.randperm(pages * 2 * page, generator=g)].view(pages, 2, page)
    weights = {"powers of four": 4.0 ** (i % 120 - 60).double(), "halves of an octave": 1.0 + (i % 128).double() / 128, "last bits": 1.0 + (i % 256).double() * 2.0**-23,
               "two values": 1.0 + (i % 100 == 0).double()}[kind].float()
    want_lens, want_kept = tree.choose(weights, table, [n] * sequences, keep, recent)
    weights = weights.cuda()
    planes = _planes(cache, weights)
    want = tree.keep([x.cpu() for x in planes], want_kept, want_lens, table, None, None)
    now, kept = ops.paged_cache_evict(cache, weights, table.cuda(), ln.cuda(), keep, recent)
    ops.check_status()
    assert torch.equal(now.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
    _same(planes, want)


def test_refusals():
    ops = _ops()
    table, ln, st, pages = _batch([1, 1], [40, 20], 16)
    cache = _full_cache(pages, 2, 16, 64, F16, 3)
    table, ln, st = table.cuda(), ln.cuda(), st.cuda()
    weights, lse, q = torch.zeros(pages, 2, 16).cuda(), torch.zeros(2, 4).cuda(), _numbers((2, 4, 64), F16, 1).cuda()
    kept = torch.zeros(2, 3, dtype=torch.int32).cuda()
    for call in (lambda: ops.paged_cache_evict(cache, weights, table, ln, 0), lambda: ops.paged_cache_evict(cache, weights, table, ln, 4, 5),
                 lambda: ops.paged_cache_evict(cache, weights, table, ln, 4, -1), lambda: ops.paged_cache_evict(cache, weights[1:].contiguous(), table, ln, 4),
                 lambda: ops.paged_cache_evict(cache, weights, table, ln[:1], 4), lambda: ops.paged_cache_evict(cache, weights, table, ln, 4, into=table[:1]),
                 lambda: ops.paged_cache_keep(cache, kept[:1], ln, table), lambda: ops.paged_cache_keep(cache, kept[:, None], ln, table),
                 lambda: ops.paged_cache_keep(cache, kept, ln[:1], table), lambda: ops.paged_cache_keep(cache, kept, ln, table, first=ln[:1]),
                 lambda: ops.paged_cache_keep(cache, kept, ln, table, weights=weights[:1].contiguous()),
                 lambda: ops.paged_attention_weights(q, cache, weights, lse[:1], table, ln, st), lambda: ops.paged_attention_weights(q[:, :3], cache, weights, lse, table, ln, st),
                 lambda: ops.paged_attention_weights(q, cache, weights, lse, table, ln, st, window=0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.paged_cache_evict(cache, weights.double(), table, ln, 4), lambda: ops.paged_cache_keep(cache, kept.long(), ln, table),
                 lambda: ops.paged_attention_weights(q.bfloat16(), cache, weights, lse, table, ln, st),
                 lambda: ops.paged_attention_weights(q, cache, weights, lse.half(), table, ln, st)):
        with pytest.raises(TypeError):
            call()


# ------------------------------------------------------------------------------------------ all of it together
@pytest.mark.parametrize("eight_bit", [False, True])
def test_answering_with_eviction(eight_bit):
    """Prompts, then tokens one by one, weights added up, down to `keep` keys when there are more than `keep` + 8: the attention is that over
    the keys that stayed, and the weights of a sequence add up to the heads that each of its tokens had."""
    ops = _ops()
    kv, group, d, page, keep, recent = 2, 3, 64, 16, 24, 8
    lens = [30, 5]
    table, ln, st, pages = _batch(lens, [n + 24 for n in lens], page)
    table = table.cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = ops.paged_cache(pages, kv, page, d, E4M3 if eight_bit else BF16)
    weights = torch.full((pages, kv, page), float("nan"), device="cuda")  # (new tokens begin at 0)
    rows = [[[] for _ in range(kv)] for _ in range(2)]                    # what stays of each sequence and head
    ln, new = i32(lens), lens
    for step in range(20):
        T = sum(new)
        starts = i32([0, new[0], T])
        k, v = (_numbers((T, kv, d), BF16, 100 * step + i).cuda() for i in range(2))
        q = _numbers((T, kv * group, d), BF16, 100 * step + 2).cuda()
        ops.paged_cache_write(cache, k, v, table, ln, starts)
        lse = torch.empty(T, kv * group, device="cuda")
        before = weights.clone()
        o = ops.paged_attention(q, cache, table, ln, starts, scale=0.125, lse=lse)
        ops.paged_attention_weights(q, cache, weights, lse, table, ln, starts, scale=0.125)
        ops.check_status()
        _weigh_check(torch.nan_to_num(weights), torch.nan_to_num(before), q, cache, lse, table.cpu(), ln.cpu(), starts.cpu(), 0.125)
        if int(ln.max()) > keep + 8:
            dense = [tree.paged.dense(cache, i) for i in range(2)]
            was = [int(n) for n in ln]
            ln, kept = ops.paged_cache_evict(cache, weights, table, ln, keep, recent)
            ops.check_status()
            after = [tree.paged.dense(cache, i) for i in range(2)]
            for b in range(2):
                assert int(ln[b]) == min(was[b], keep)
                for h in range(kv):
                    for i in range(int(ln[b])):
                        src = int(kept[b, h, i])
                        for x, y in zip(dense, after):
                            assert torch.equal(x[int(table[b, src // page]), h, src % page], y[int(table[b, i // page]), h, i % page])
        new = [1, 1]
        ln = ln + 1


@pytest.mark.parametrize("eight_bit", [False, True])
def test_captured_and_on_another_stream(eight_bit):
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    kv, group, d, page, keep, recent = 2, 4, 128, 16, 20, 5
    table, ln, st, pages = _batch([1, 2], [60, 45], page, width=8)
    start = _full_cache(pages, kv, page, d, E4M3 if eight_bit else F16, 3)
    cache = tuple(c.clone() for c in start)
    q = _numbers((3, kv * group, d), F16, 1).cuda()
    weights = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)).cuda()
    w0 = weights.clone()
    table, ln, st = table.cuda(), ln.cuda(), st.cuda()
    lse = torch.empty(3, kv * group, device="cuda")

    def step():
        ops.paged_attention(q, cache, table, ln, st, scale=0.1, lse=lse)
        ops.paged_attention_weights(q, cache, weights, lse, table, ln, st, scale=0.1)
        return ops.paged_cache_evict(cache, weights, table, ln, keep, recent)

    def fresh():
        weights.copy_(w0)
        for c, s in zip(cache, start):
            c.copy_(s)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        now, kept = step()
    for lens in ([60, 45], [33, 19], [21, 50]):
        ln.copy_(torch.tensor(lens))
        fresh()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in _planes(cache, weights)] + [now.clone(), kept.clone()]
        fresh()
        want_now, want_kept = step()
        torch.cuda.synchronize()
        _same(got, _planes(cache, weights) + [want_now, want_kept])
    with pytest.raises(FtbError):  # (the last lengths reach behind the second sequence's pages: recorded, and the same in both)
        ops.check_status()

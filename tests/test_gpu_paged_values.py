"""Attention over an 8-bit paged cache whose visible rows are zeros or differ widely in size, against 64 bits."""
import math

import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _ops():
    from fractaltensor_b200 import ops
    return ops


def _batch(new, lens, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    counts = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(counts) + 2, generator=g).int()
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), sum(counts) + 2


def _numbers(shape, seed, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _cache(pages, kv, page, d, seed):
    """An 8-bit cache of numbers about 1, exponents about 119."""
    out = [], []
    for i in range(2):
        codes, exps = paged.quantise(_numbers((pages, kv, page, d), seed + i).cpu())
        out[0].append(codes.view(E4M3).cuda())
        out[1].append(exps.cuda())
    return tuple(out[0] + out[1])


def _change(cache, i, table, lens, rows, steps):
    """Keys (0) or values (1) of the positions rows(n) -> bool [n]: zeros as they are stored (steps None), or 2^steps as large."""
    page = cache[0].shape[2]
    for b, n in enumerate(lens):
        j = rows(n).nonzero()[:, 0]
        at = table[b].cpu().long()[j // page].cuda(), slice(None), (j % page).cuda()
        if steps is None:
            cache[i].view(torch.uint8)[at] = 0
            cache[2 + i][at] = 1
        else:
            cache[2 + i][at] = (cache[2 + i][at].int() + steps).clamp(1, 247).byte()


def _exact(q, cache, table, lens, new, scale, window):
    """-> (o, bound) as the oracle's, on the device in 64 bits."""
    k, v = (paged.values(cache[i].view(torch.uint8), cache[2 + i]) for i in range(2))
    kv, page, heads = k.shape[1], k.shape[2], q.shape[1]
    o, mean, size, most, first = [], [], [], [], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        j = torch.arange(n, device="cuda")
        rows = table[b].long()[j // page]
        kb, vb = (x[rows, :, j % page].repeat_interleave(heads // kv, 1).transpose(0, 1) for x in (k, v))  # [heads, n, d]
        x = q[first:first + m].double().transpose(0, 1)
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = j > pos
        if window:
            hidden = hidden | (j <= pos - window)
        w = torch.softmax((x @ kb.transpose(1, 2) * scale).masked_fill(hidden, -math.inf), -1)
        o.append((w @ vb).transpose(0, 1))
        mean.append((w @ vb.abs()).transpose(0, 1))
        size.append((x.abs() @ kb.abs().transpose(1, 2) * scale).masked_fill(hidden, 0).amax(-1).T)
        most.append(vb.abs().amax(-1)[:, None].expand(-1, m, -1).masked_fill(hidden, 0).amax(-1).T)
        first += m
    o, mean, size, most = (torch.cat(x).cpu() for x in (o, mean, size, most))
    return o, (mean, size, most)


def _check(o, q, cache, table, lens, new, scale, window=None):
    want, (mean, size, most) = _exact(q, cache, table, lens, new, scale, window)
    # the oracle's tolerance, term by term, but for half of fp16's smallest number, which has no part in bf16 results: taken off
    # behind the sum it would leave 0 of a tolerance below 2^-78, since 2^-25 + 2^-79 is 2^-25 in 64 bits
    eps, d = torch.finfo(q.dtype).eps, q.shape[2]
    score = (2 * (d + 4) * 2.0 ** -24 * size + 2.0 ** -21 + 2.0 ** -16)[..., None]
    tol = eps / 2 * want.abs() + (2.0 ** -11 + 2 * score + 2.0 ** -20) * mean + max(lens) * 2.0 ** -24 * most[..., None]
    tol = tol * (1 + eps)
    err = (o.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol).nan_to_num(9e9).max()), bad.nonzero()[:4].tolist(), float(want.abs().max()))


# kv, group, d, page, new, lens, window: single tokens in tiles of 8 and 16 rows, drafts, tiles of 128 and 256 rows (nearly all of them
# cut: there are more CTAs than blocks of keys), a tile of one block, a window
SHAPES = [
    (2, 4, 128, 16, [1, 1, 1], [600, 33, 300], None),
    (1, 16, 64, 32, [1, 1], [511, 130], None),
    (2, 8, 128, 64, [2, 1, 2], [400, 1333, 40], None),
    (1, 4, 128, 16, [1], [5000], None),
    (2, 4, 128, 16, [20, 30], [700, 400], None),
    (2, 5, 64, 32, [90, 1, 25], [600, 257, 100], None),
    (1, 4, 128, 64, [200], [700], None),
    (2, 4, 64, 16, [300], [300], None),
    (2, 4, 128, 32, [150], [900], 300),
]
ROWS = {
    "first 16": lambda n: torch.arange(n) < 16,
    "first 128": lambda n: torch.arange(n) < 128,
    "every second": lambda n: torch.arange(n) % 2 == 0,
    "a block": lambda n: (torch.arange(n) >= 128) & (torch.arange(n) < 256),
    "all but every 50th": lambda n: torch.arange(n) % 50 != 0,
    "behind 200": lambda n: torch.arange(n) >= 200,
    "all": lambda n: torch.arange(n) >= 0,
}


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("steps", [0, 10, 60, -60])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", SHAPES)
def test_values_of_zero_keep_their_weight(kv, group, d, page, new, lens, window, steps, rows):
    """A key whose value is a row of zeros (stored with the smallest exponent) weighs as any other, whatever the others' size."""
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    _change(cache, 1, table, lens, lambda n: ~ROWS[rows](n), steps)
    _change(cache, 1, table, lens, ROWS[rows], None)
    q = _numbers((sum(new), kv * group, d), 1)
    o = _ops().paged_attention(q, cache, table, ln, st, scale=0.3, window=window)
    _ops().check_status()
    _check(o, q, cache, table, lens, new, 0.3, window)


@pytest.mark.parametrize("rows", ["first 128", "every second", "a block", "behind 200"])
@pytest.mark.parametrize("steps", [-100, -30, 30, 100])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", SHAPES)
def test_visible_values_of_different_sizes(kv, group, d, page, new, lens, window, steps, rows):
    """Visible values 2^steps times as large as the others."""
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    _change(cache, 1, table, lens, ROWS[rows], steps)
    q = _numbers((sum(new), kv * group, d), 1)
    o = _ops().paged_attention(q, cache, table, ln, st, scale=0.3, window=window)
    _ops().check_status()
    _check(o, q, cache, table, lens, new, 0.3, window)


@pytest.mark.parametrize("new,lens", [([1] * 6, [700] * 6), ([30] * 6, [700] * 6), ([200], [700])])
def test_large_values_without_weight(new, lens):
    """The largest values by 2^70 are of keys that weigh 2^-200: what is left is the others' mean, zeros among them."""
    kv, group, d, page = 2, 4, 64, 16
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    q = _numbers((sum(new), kv * group, d), 1)
    q[..., 0] = 8.0
    far = lambda n: (torch.arange(n) >= 256) & (torch.arange(n) < 384)  # whole blocks: a block's codes share their largest exponent
    _change(cache, 1, table, lens, far, 70)
    _change(cache, 1, table, lens, lambda n: torch.arange(n) % 3 == 1, None)
    for b, n in enumerate(lens):  # the keys of those: a code of -448 in the first place, zeros behind
        j = far(n).nonzero()[:, 0]
        at = table[b].cpu().long()[j // page].cuda(), slice(None), (j % page).cuda()
        cache[0].view(torch.uint8)[at] = 0
        cache[0].view(torch.uint8)[at + (0,)] = 0xFE
        cache[2][at] = 124
    o = _ops().paged_attention(q, cache, table, ln, st, scale=0.3)
    _ops().check_status()
    want, (mean, size, _) = _exact(q, cache, table, lens, new, 0.3, None)
    # scores as in the oracle's tolerance, weights of fp16; weights below fp16's smallest number beside the largest share: none has
    # a value above 8 here, the far ones' shares being below 2^-120
    eps = torch.finfo(BF16).eps
    tol = (eps / 2 * want.abs() + (2.0 ** -11 + 4 * (d + 4) * 2.0 ** -24 * size[..., None] + 2.0 ** -15) * mean + 700 * 2.0 ** -24 * 8) * (1 + eps)
    err = (o.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).nan_to_num(9e9).max())


@pytest.mark.parametrize("zero", ["first 128", "every second"])
def test_many_whole_tiles_with_values_of_zero(zero):
    """More tiles than CTAs, most of them not cut."""
    kv, group, d, page = 8, 4, 128, 16
    new, lens = [40] * 40, [300 + 50 * b for b in range(40)]
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    _change(cache, 1, table, lens, ROWS[zero], None)
    q = _numbers((sum(new), kv * group, d), 1)
    o = _ops().paged_attention(q, cache, table, ln, st, scale=0.3)
    _ops().check_status()
    _check(o, q, cache, table, lens, new, 0.3)


@pytest.mark.parametrize("keys", ["all", "first 128", "every second", "behind 200", None])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", SHAPES)
def test_queries_of_zero(kv, group, d, page, new, lens, window, keys):
    """Rows of queries that are zeros, or the smallest numbers, over keys of zeros and others: the mean of the values."""
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    _change(cache, 0, table, lens, lambda n: torch.arange(n) >= 0, -20)
    if keys:
        _change(cache, 0, table, lens, ROWS[keys], None)
    q = _numbers((sum(new), kv * group, d), 1)
    q[::2] = 0.0
    q[1::4] *= 2.0 ** -120
    o = _ops().paged_attention(q, cache, table, ln, st, scale=0.3, window=window)
    _ops().check_status()
    _check(o, q, cache, table, lens, new, 0.3, window)


@pytest.mark.parametrize("hidden", [False, True])
@pytest.mark.parametrize("steps", [-118, -90, 90, 118, 126])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", SHAPES)
def test_sizes_of_queries_and_keys_that_cancel(kv, group, d, page, new, lens, window, steps, hidden):
    """Keys 2^steps times as large, queries 2^-steps times: ordinary scores.  hidden: a value of the last position is NaN, which rows that
    do not see it are computed key by key for."""
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    _change(cache, 0, table, lens, lambda n: torch.arange(n) >= 0, steps)
    q = (_numbers((sum(new), kv * group, d), 1).float() * 2.0 ** -steps).to(BF16)
    bad = tuple(c.clone() for c in cache)
    if hidden:
        for b, n in enumerate(lens):
            at = int(table[b, (n - 1) // page]), slice(None), (n - 1) % page
            bad[1].view(torch.uint8)[at] = 0x7F
            bad[3][at] = 255
    o = _ops().paged_attention(q, bad, table, ln, st, scale=0.3, window=window)
    _ops().check_status()
    if hidden:  # the last token of each sequence sees it
        last = st[1:].long() - 1
        assert bool(torch.isnan(o[last].float()).all())
        o[last] = _exact(q, cache, table, lens, new, 0.3, window)[0].to(BF16).cuda()[last]
    _check(o, q, cache, table, lens, new, 0.3, window)


@pytest.mark.parametrize("apart", [16, 23, 25, 28, 31])
@pytest.mark.parametrize("new,lens", [([30] * 3, [700, 800, 900]), ([200], [900])])
def test_values_far_below_the_largest_of_their_block(new, lens, apart):
    """One value of each 128, 2^apart times as large as the others, whose key weighs nothing: the others' mean is left."""
    kv, group, d, page = 2, 4, 64, 16
    table, ln, st, pages = _batch(new, lens, page)
    cache = _cache(pages, kv, page, d, 3)
    q = _numbers((sum(new), kv * group, d), 1)
    q[..., 0] = 8.0
    rows = lambda n: (torch.arange(n) % 128 == 5) & (torch.arange(n) < 600)  # before the first token that asks
    _change(cache, 1, table, lens, rows, apart)
    for b, n in enumerate(lens):  # their keys: a code of -448 in the first place, zeros behind
        j = rows(n).nonzero()[:, 0]
        at = table[b].cpu().long()[j // page].cuda(), slice(None), (j % page).cuda()
        cache[0].view(torch.uint8)[at] = 0
        cache[0].view(torch.uint8)[at + (0,)] = 0xFE
        cache[2][at] = 124
    o = _ops().paged_attention(q, cache, table, ln, st, scale=0.3)
    _ops().check_status()
    want, (mean, size, most) = _exact(q, cache, table, lens, new, 0.3, None)
    # as in test_large_values_without_weight, and values as products take them: fp16 numbers code * 2^(7 - below) in units of
    # 2^(e - 134), e the block's largest exponent; off by 2^-25 of them, that is 2^-32 * 2^(e - 127), and 2^(e - 127) is below the
    # largest value / 224
    eps = torch.finfo(BF16).eps
    tol = eps / 2 * want.abs() + (2.0 ** -11 + 4 * (d + 4) * 2.0 ** -24 * size[..., None] + 2.0 ** -15) * mean + 900 * 2.0 ** -24 * 8
    # Rows here have exponents one or two apart, so that some lie 32 or more below the largest: 2^(7 - below) is 0 in fp16 then (its
    # smallest number is 2^-24), and they are off by themselves.  Their part of the mean of |values|:
    lost = tuple(c.clone() for c in cache)
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        at = table[b].long()[j // page], slice(None), j % page
        e = cache[3][at].int()  # [n, kv]
        top = torch.cat([x.amax(0, keepdim=True).expand_as(x) for x in e.split(128)])
        assert apart >= 30 or not bool((top - e > 31).any())
        lost[1].view(torch.uint8)[at] = lost[1].view(torch.uint8)[at] * (top - e > 31)[..., None]
    tol = (tol + 2.0 ** -32 / 224 * most[..., None] + _exact(q, lost, table, lens, new, 0.3, None)[1][0]) * (1 + eps)
    err = (o.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).nan_to_num(9e9).max())


@pytest.mark.parametrize("dtype", [torch.float32, BF16, F16])
@pytest.mark.parametrize("first", [1, 3, 100, 244])
def test_reading_at_the_ends_of_the_exponents(dtype, first):
    """Every code under the first, last and some exponents that rows are stored with: rounded once, and bf16 exact from 3 to 246."""
    kv, d, page = 4, 128, 16
    table, ln, st, pages = _batch([16], [16], page)
    cache = _ops().paged_cache(pages, kv, page, d, E4M3)
    at = int(table[0, 0])
    codes = torch.arange(256, dtype=torch.uint8).view(2, d).repeat(page // 2, 1)
    for h in range(kv):
        for i in range(2):
            cache[i].view(torch.uint8)[at, h] = codes.cuda()
            cache[2 + i][at, h] = first + h
    got = _ops().paged_cache_read(cache, table, ln, st, 16, dtype=dtype)
    _ops().check_status()
    for h in range(kv):
        numbers = paged.values(codes, torch.full((page,), first + h, dtype=torch.uint8))
        want = numbers.float().to(dtype)  # (the numbers have four bits: fp32 has them all, or infinity)
        for x in got:
            assert torch.equal(x[:, h].cpu().nan_to_num(nan=3.0), want.nan_to_num(nan=3.0))
            if dtype == BF16 and 3 <= first + h <= 246:
                assert torch.equal(x[:, h].cpu().double().nan_to_num(nan=3.0), numbers.nan_to_num(nan=3.0))

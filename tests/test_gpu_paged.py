"""The paged cache, attention over it and the verification of drafted tokens against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _ops():
    from fractaltensor_b200 import ops
    return ops


def _batch(new, lens, page, extra_pages=2, width=0, seed=0, front=0):
    """Pages in random order for sequences of the given lengths: (table, lens, starts, pages), tables padded with -1."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + extra_pages
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max(1, width, max(counts))), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    starts = [front]
    for n in new:
        starts.append(starts[-1] + n)
    return table, torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32), pages


def _numbers(shape, dtype, seed, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return (x * torch.exp(spread * torch.randn(shape[:-1], generator=g))[..., None]).to(dtype)


def _full_cache(pages, kv, page, d, dtype, seed, table=None, lens=None, stale=float("nan")):
    """A cache of random numbers; rows that no sequence has written hold `stale`."""
    k, v = (_numbers((pages, kv, page, d), BF16 if dtype == E4M3 else dtype, seed + i) for i in range(2))
    if table is not None:
        written = torch.zeros(pages, page, dtype=torch.bool)
        for b in range(len(lens)):
            for j in range(int(lens[b])):
                written[int(table[b, j // page]), j % page] = True
        for x in (k, v):
            x.masked_fill_(~written[:, None, :, None], stale)
    if dtype != E4M3:
        return k.cuda(), v.cuda()
    (kc, ke), (vc, ve) = paged.quantise(k), paged.quantise(v)
    return kc.view(E4M3).cuda(), vc.view(E4M3).cuda(), ke.cuda(), ve.cuda()


def _bits(t):
    return t.contiguous().view(torch.uint8).cpu()


# ------------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,d,page,new,lens", [
    (1, 64, 16, [1], [1]),
    (8, 128, 16, [1, 1, 0, 1], [17, 16, 40, 1]),
    (3, 64, 32, [5, 33, 0], [33, 33, 0]),
    (5, 128, 128, [200, 7], [300, 129]),
    (2, 128, 64, [1] * 70, list(range(1, 71))),
])
def test_write_then_read_16_bit(dtype, kv, d, page, new, lens):
    ops = _ops()
    table, ln, st, pages = _batch(new, lens, page)
    T = int(st[-1])
    pad = 3
    qkv = _numbers((T + pad, (2 * kv + 1) * d), dtype, 5).cuda()
    k, v = qkv[:, d:(kv + 1) * d].unflatten(1, (kv, d)), qkv[:, (kv + 1) * d:].unflatten(1, (kv, d))
    cache = ops.paged_cache(pages, kv, page, d, dtype)
    for c in cache:
        c.fill_(7.0)
    ops.paged_cache_write(cache, k, v, table.cuda(), ln.cuda(), st.cuda())
    want = [torch.full((pages, kv, page, d), 7.0, dtype=dtype) for _ in range(2)]
    for t, place in enumerate(paged.places(table, ln, st, page, T)):
        b, pos = place
        for w, x in zip(want, (k, v)):
            w[int(table[b, pos // page]), :, pos % page] = x[t].cpu()
    for c, w in zip(cache, want):
        assert torch.equal(_bits(c), _bits(w))
    out = tuple(torch.full((T + pad, kv, d), -3.0, dtype=dtype, device="cuda") for _ in range(2))
    got = ops.paged_cache_read(cache, table.cuda(), ln.cuda(), st.cuda(), T + pad, out=out)
    for o, x in zip(got, (k, v)):
        assert torch.equal(o[:T], x[:T]) and bool((o[T:] == -3.0).all())
    ops.check_status()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,page,kv", [(64, 16, 3), (128, 64, 8), (128, 32, 1)])
def test_write_8_bit_has_the_definition_s_bits(dtype, d, page, kv):
    ops = _ops()
    new, lens = [37, 1, 90], [50, 9, 90]
    table, ln, st, pages = _batch(new, lens, page)
    T = int(st[-1])
    x = [_numbers((T, kv, d), dtype, 11 + i, spread=2.0) for i in range(2)]
    for i, t in enumerate(x):
        t[0] = 0.0
        t[1, :, 1:] = 0.0
        t[2] = 1.75                                    # the largest code itself
        t[3, :, 0], t[3, :, 1] = 1.765625 if dtype == F16 else 1.7578125, -1.0  # just above it: the next exponent
        t[4] = torch.linspace(-448, 448, d).to(dtype)  # ties between codes
        t[5] = torch.finfo(dtype).tiny
        t[6, :, -1] = float("inf")
        t[7, :, d // 2] = float("nan")
        t[8] = torch.finfo(dtype).max
        t[9, :, 0] = torch.finfo(dtype).max
        t[10] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest number there is
        t[11] = -0.0
    cache = ops.paged_cache(pages, kv, page, d, E4M3)
    ops.paged_cache_write(cache, x[0].cuda(), x[1].cuda(), table.cuda(), ln.cuda(), st.cuda())
    for i in range(2):
        codes = torch.zeros(pages, kv, page, d, dtype=torch.uint8)
        exps = torch.ones(pages, kv, page, dtype=torch.uint8)
        c, e = paged.quantise(x[i])
        for t, (b, pos) in enumerate(paged.places(table, ln, st, page, T)):
            codes[int(table[b, pos // page]), :, pos % page] = c[t]
            exps[int(table[b, pos // page]), :, pos % page] = e[t]
        assert torch.equal(cache[2 + i].cpu(), exps)
        assert torch.equal(cache[i].view(torch.uint8).cpu(), codes)
    for out_dtype in (torch.float32, BF16, F16):
        got = ops.paged_cache_read(cache, table.cuda(), ln.cuda(), st.cuda(), T, dtype=out_dtype)
        for i in range(2):
            want = paged.values(*paged.quantise(x[i])).to(out_dtype)
            assert torch.equal(torch.nan_to_num(got[i].cpu(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))
    ops.check_status()


def test_tokens_without_a_place_are_not_stored():
    """Negative positions, pages that the table does not have, rows around the sequences."""
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    kv, d, page = 2, 64, 16
    cache = ops.paged_cache(3, kv, page, d, BF16)
    k = torch.ones(12, kv, d, dtype=BF16, device="cuda")
    table = torch.tensor([[2], [0]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([2, 6, 10], dtype=torch.int32, device="cuda")
    lens = torch.tensor([2, 4], dtype=torch.int32, device="cuda")  # four tokens of a sequence of two keys: two are in front of it
    ops.paged_cache_write(cache, k, k, table, lens, starts)
    ops.check_status()
    want = torch.zeros(3, page)
    want[2, :2] = 1
    want[0, :4] = 1
    assert torch.equal(cache[0][:, 0, :, 0].float().cpu(), want)
    out = ops.paged_cache_read(cache, table, lens, starts, 12)
    assert bool((out[0][2:4] == 0).all()) and bool((out[0][4:10] == 1).all())
    # a page number out of range, and a length behind the table's width: an error on the status word, nothing stored
    for bad_table, bad_lens in ((torch.tensor([[3], [-1]]), lens), (table, torch.tensor([30, 33]))):
        before = cache[0].clone()
        ops.paged_cache_write(cache, 2 * k, k, bad_table.int().cuda(), bad_lens.int().cuda(), starts)
        with pytest.raises(FtbError):
            ops.check_status()
        assert torch.equal(before, cache[0])
        ops.paged_cache_read(cache, bad_table.int().cuda(), bad_lens.int().cuda(), starts, 12)
        ops.paged_attention(k, cache, bad_table.int().cuda(), bad_lens.int().cuda(), starts)
        with pytest.raises(FtbError):
            ops.check_status()
    ops.check_status()


# --------------------------------------------------------------------------------------------- attention
def _check(o, q, cache, table, ln, st, scale, window, rows=None):
    want, bound = paged.attention(q, cache, table, ln, st, scale, window)
    tol = paged.tolerance(want, bound, q.dtype, q.shape[2], len(cache) == 4, int(ln.max()))
    err = (o.double().cpu() - want).abs()
    lo, hi = (int(st[0]), int(st[-1])) if rows is None else rows
    bad = ~(err[lo:hi] <= tol[lo:hi])
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol)[lo:hi].nan_to_num(9e9).max()), bad.nonzero()[:5].tolist())


SHAPES = [
    # kv, group, d, page, new, lens, window
    (1, 1, 64, 16, [1], [1], None),
    (1, 1, 128, 16, [1], [1000], None),
    (8, 4, 128, 16, [1], [777], None),
    (2, 8, 128, 64, [1, 1, 1], [5, 64, 333], None),
    (2, 1, 64, 32, [1, 0, 1, 1], [31, 7, 0, 65], None),
    (1, 16, 128, 128, [1, 1], [129, 511], None),
    (2, 3, 64, 16, [1, 5, 2], [100, 5, 47], None),
    (1, 5, 128, 32, [4, 4], [200, 130], None),
    (1, 71, 64, 16, [1, 2], [70, 33], None),
    (4, 2, 128, 16, [7, 1, 30], [7, 300, 91], None),
    (1, 4, 128, 64, [130], [130], None),
    (2, 4, 128, 16, [67, 150], [500, 151], None),
    (1, 8, 64, 128, [257], [300], None),
    (1, 7, 128, 16, [40, 1, 90, 1], [41, 600, 333, 2], None),
    (1, 2, 128, 32, [300], [3000], None),
    (1, 1, 128, 16, [40], [5000], None),
    (2, 8, 128, 64, [5, 5, 5], [400, 1333, 5], None),
    (1, 8, 64, 16, [6, 4, 1], [777, 100, 2000], 400),
    (2, 10, 128, 32, [3, 2, 3], [600, 64, 1500], None),
    (1, 6, 64, 128, [4, 5], [3000, 129], None),
    (1, 45, 128, 16, [1, 1], [900, 17], None),
    (2, 2, 128, 64, [260], [2000], None),
    (1, 8, 64, 32, [30, 31], [4000, 900], None),
    (1, 1, 64, 16, [600, 1, 129], [600, 40, 1000], None),
    (3, 1, 128, 128, [128], [128], None),
    (2, 4, 128, 16, [1, 1], [500, 40], 1),
    (2, 4, 128, 16, [1, 3], [500, 40], 100),
    (1, 4, 64, 16, [200], [400], 33),
    (1, 2, 128, 64, [140, 20], [700, 20], 150),
]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", SHAPES)
def test_attention(dtype, eight_bit, kv, group, d, page, new, lens, window):
    """Unwritten rows of the pages hold NaN, rows around the sequences keep what they hold."""
    ops = _ops()
    table, ln, st, pages = _batch(new, lens, page, front=1)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else dtype, 3, table, ln)
    T = int(st[-1]) + 2
    qkv = _numbers((T, (kv * group + 1) * d), dtype, 9, spread=0.3).cuda()
    q = qkv[:, d:].unflatten(1, (kv * group, d))
    scale = 1.0 / math.sqrt(d)
    out = torch.full((T, kv * group, d), 5.0, dtype=dtype, device="cuda")
    got = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=scale, window=window, out=out)
    ops.check_status()
    assert got is out and bool((out[0] == 5.0).all()) and bool((out[-2:] == 5.0).all())
    _check(out, q, cache, table, ln, st, scale, window)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens,window", [([1, 1], [700, 333], 100), ([40, 1], [700, 333], 77), ([300], [900], 130), ([20, 20], [400, 500], 64)])
def test_pages_in_front_of_the_window_may_be_gone(eight_bit, new, lens, window):
    ops = _ops()
    kv, group, d, page = 2, 4, 128, 16
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    q = _numbers((int(st[-1]), kv * group, d), BF16, 1).cuda()
    want = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.1, window=window)
    gone = table.clone()
    for b, (n, m) in enumerate(zip(lens, new)):
        gone[b, : max(0, n - m + 1 - window) // page] = -1
    got = ops.paged_attention(q, cache, gone.cuda(), ln.cuda(), st.cuda(), scale=0.1, window=window)
    ops.check_status()
    assert torch.equal(got, want)
    _check(got, q, cache, table, ln, st, 0.1, window)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens", [([3, 2], [1, 2]), ([4], [0]), ([200, 1], [150, 0]), ([5, 0], [5, 0])])
def test_tokens_that_see_nothing_get_zeros(eight_bit, new, lens):
    ops = _ops()
    table, ln, st, pages = _batch(new, lens, 16)
    cache = _full_cache(pages, 2, 16, 64, E4M3 if eight_bit else F16, 3, table, ln)
    q = _numbers((int(st[-1]), 4, 64), F16, 1).cuda()
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.125)
    ops.check_status()
    for b in range(len(new)):
        hidden = max(0, new[b] - lens[b])
        assert bool((o[int(st[b]):int(st[b]) + hidden] == 0).all())
    _check(o, q, cache, table, ln, st, 0.125, None)


@pytest.mark.parametrize("worst", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,n,at,window", [(6, 40, 37, None), (200, 333, 201, None), (1, 300, 100, 150), (160, 500, 400, 30), (90, 90, 89, None)])
def test_what_is_not_seen_has_no_part(worst, eight_bit, new, n, at, window):
    """A key and value that are not finite at one position: tokens that see it say so, the others have what they had."""
    ops = _ops()
    kv, group, d, page = 2, 4, 128, 16
    table, ln, st, pages = _batch([new], [n], page)
    if eight_bit and worst != worst or not eight_bit:
        base = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    else:
        pytest.skip("8-bit rows that are not finite are NaN")
    q = _numbers((new, kv * group, d), BF16, 1).cuda()
    args = (table.cuda(), ln.cuda(), st.cuda())
    good = ops.paged_attention(q, base, *args, scale=0.1, window=window)
    for which in (0, 1):
        cache = tuple(c.clone() for c in base)
        if eight_bit:
            cache[which].view(torch.uint8)[int(table[0, at // page]), 1, at % page] = 0x7F
            cache[2 + which][int(table[0, at // page]), 1, at % page] = 255
        else:
            cache[which][int(table[0, at // page]), 1, at % page, 5] = worst
        o = ops.paged_attention(q, cache, *args, scale=0.1, window=window)
        ops.check_status()
        pos = torch.arange(n - new, n)
        sees = (pos >= at) & ((pos - at < window) if window else torch.ones_like(pos, dtype=torch.bool))
        hidden = (~sees).cuda()
        assert torch.equal(o[:, :group], good[:, :group])           # the other kv head
        # (the same numbers, or, where they are computed key by key, to rounding)
        want, bound = paged.attention(q, base, table, ln, st, 0.1, window)
        tol = paged.tolerance(want, bound, BF16, d, eight_bit, n)
        assert bool(((o.double().cpu() - want).abs() <= tol)[~sees].all())
        if which == 1 and bool(sees.any()):
            assert not bool(torch.isfinite(o[sees.cuda()][:, group:].float()).all(-1).any())


@pytest.mark.parametrize("steps", [14, 17, 60, -60])
@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,n,begin,end,window", [(3, 40, 38, 40, None), (20, 333, 320, 333, None), (200, 333, 250, 333, None), (300, 300, 100, 101, None),
                                                    (20, 700, 500, 560, 130), (200, 700, 400, 520, 150), (129, 2000, 1990, 1995, None)])
def test_the_size_of_what_is_not_seen_has_no_part(steps, eight_bit, d, new, n, begin, end, window):
    """Keys and values 2^steps times as large at positions begin .. end - 1: tokens that see none of them have what they had."""
    ops = _ops()
    kv, group, page = 2, 4, 16
    table, ln, st, pages = _batch([new], [n], page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    j = torch.arange(begin, end)
    at = table[0][j // page].long().cuda(), slice(None), (j % page).cuda()
    for i in range(2):
        if eight_bit:
            cache[2 + i][at] = (cache[2 + i][at].int() + steps).clamp(1, 254).byte()
        else:
            cache[i][at] = cache[i][at] * 2.0 ** steps
    q = _numbers((new, kv * group, d), BF16, 1).cuda()
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.1, window=window)
    ops.check_status()
    pos = torch.arange(n - new, n)
    sees = pos >= begin
    if window:
        sees &= pos - window < end - 1
    assert bool(sees.any()) and not bool(sees.all())
    want, bound = paged.attention(q, cache, table, ln, st, 0.1, window)
    tol = paged.tolerance(want, bound, BF16, d, eight_bit, n)
    err = ((o.double().cpu() - want).abs() / tol)[~sees]
    assert bool((err <= 1).all()), float(err.nan_to_num(9e9).max())


def test_page_offsets_beyond_32_bits():
    ops = _ops()
    kv, d, page = 8, 128, 128
    pages = (1 << 33) // (kv * d * page * 2) + 3  # 8 GB of keys
    cache = tuple(torch.empty(pages, kv, page, d, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    ln, st = torch.tensor([300], dtype=torch.int32), torch.tensor([0, 300], dtype=torch.int32)
    k, v = _numbers((300, kv, d), BF16, 1).cuda(), _numbers((300, kv, d), BF16, 2).cuda()
    args = (table.cuda(), ln.cuda(), st.cuda())
    ops.paged_cache_write(cache, k, v, *args)
    got = ops.paged_cache_read(cache, *args, 300)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    q = _numbers((300, kv * 2, d), BF16, 3).cuda()
    o = ops.paged_attention(q, cache, *args, scale=0.1)
    one = ops.paged_attention(q[-1:], cache, table.cuda(), ln.cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(), scale=0.1)
    ops.check_status()
    small = tuple(c[table[0].long()].clone() for c in cache)
    _check(o, q, small, torch.tensor([[0, 1, 2]]), ln, st, 0.1, None)
    _check(one, q[-1:], small, torch.tensor([[0, 1, 2]]), ln, torch.tensor([0, 1]), 0.1, None)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("kv,group,d,page,new,lens,window", [
    (8, 4, 128, 16, [40] * 40, [300 + 50 * b for b in range(40)], None),
    (8, 2, 64, 32, [150] * 12, [1000 + 77 * b for b in range(12)], None),
    (8, 4, 128, 64, [700], [2500], None),
    (8, 4, 128, 64, [1000], [1000], None),
    (8, 2, 128, 16, [900, 1, 400], [1200, 77, 2222], 300),
    (8, 8, 128, 16, [1 + b % 9 for b in range(60)], [10 + 40 * b for b in range(60)], None),
    (8, 8, 128, 32, [5] * 50, [100 + 60 * b for b in range(50)], None),
    (8, 5, 64, 16, [6] * 50, [100 + 60 * b for b in range(50)], 700),
    (4, 4, 64, 16, [1 if b % 5 else 90 for b in range(70)], [90 + 20 * b for b in range(70)], None),
])
def test_many_tiles(eight_bit, kv, group, d, page, new, lens, window):
    """More tiles than CTAs: each walks several, many blocks long.  On the device in 64 bits, and three calls without a wait between them."""
    ops = _ops()
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    q = _numbers((int(st[-1]), kv * group, d), BF16, 1, spread=0.3).cuda()
    scale = 1.0 / math.sqrt(d)
    args = (cache, table.cuda(), ln.cuda(), st.cuda())
    got = [ops.paged_attention(q, *args, scale=scale, window=window) for _ in range(3)]
    ops.check_status()
    k, v = (paged.dense(cache, i).cuda() for i in range(2))
    for b, (n, m) in enumerate(zip(lens, new)):
        j = torch.arange(n, device="cuda")
        rows = table[b].cuda().long()[j // page]
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = j > pos
        if window:
            hidden = hidden | (j <= pos - window)
        for h in range(kv * group):
            kj, vj = k[rows, h // group, j % page], v[rows, h // group, j % page]
            x = q[int(st[b]):int(st[b]) + m, h].double()
            w = torch.softmax((x @ kj.T * scale).masked_fill(hidden, -math.inf), -1)
            want = w @ vj
            size = (x.abs() @ kj.abs().T * scale).masked_fill(hidden, 0).amax(-1)
            bound = (w @ vj.abs(), size, vj.abs().amax().expand(m))
            tol = paged.tolerance(want, bound, BF16, d, eight_bit, n)
            for o in got:
                err = (o[int(st[b]):int(st[b]) + m, h].double() - want).abs()
                assert bool((err <= tol).all()), (b, h, float((err / tol).max()))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_many_sequences():
    """More sequences than a warp or a block has threads."""
    ops = _ops()
    B = 1500
    lens = [1 + (37 * b) % 90 for b in range(B)]
    new = [0 if b % 7 == 3 else 1 for b in range(B)]
    table, ln, st, pages = _batch(new, lens, 16)
    cache = _full_cache(pages, 1, 16, 64, BF16, 3)
    q = _numbers((int(st[-1]), 2, 64), BF16, 1).cuda()
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.125)
    ops.check_status()
    _check(o, q, cache, table, ln, st, 0.125, None)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_captured_calls_follow_what_changes(eight_bit):
    """Write and attention in a graph, replayed with other tokens, lengths and pages; two graphs on two streams at once."""
    ops = _ops()
    kv, group, d, page, B = 2, 4, 128, 16, 5
    scale = 0.1
    runs = []
    for seed in (1, 2):
        lens = [40 + 13 * seed * b for b in range(B)]
        table, ln, st, pages = _batch([1] * B, [n + 60 for n in lens], page, seed=seed)
        cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, seed)
        s = {"table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "starts": st.cuda(), "cache": cache,
             "q": _numbers((B, kv * group, d), BF16, seed).cuda(), "k": _numbers((B, kv, d), BF16, seed + 5).cuda(),
             "v": _numbers((B, kv, d), BF16, seed + 6).cuda(), "stream": torch.cuda.Stream()}
        s["stream"].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s["stream"]):
            ops.paged_cache_write(cache, s["k"], s["v"], s["table"], s["lens"], s["starts"])
            ops.paged_attention(s["q"], cache, s["table"], s["lens"], s["starts"], scale=scale)
        s["stream"].synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s["stream"]):
            ops.paged_cache_write(cache, s["k"], s["v"], s["table"], s["lens"], s["starts"])
            s["o"] = ops.paged_attention(s["q"], cache, s["table"], s["lens"], s["starts"], scale=scale)
        s["g"], s["host"] = g, (table, lens, st)
        runs.append(s)
    for step in range(6):
        for i, s in enumerate(runs):
            with torch.cuda.stream(s["stream"]):
                s["lens"].add_(7)
                s["k"].copy_(_numbers((B, kv, d), BF16, 100 * step + i).cuda())
        torch.cuda.synchronize()
        for _ in range(20):
            for s in runs:
                with torch.cuda.stream(s["stream"]):
                    s["g"].replay()
        torch.cuda.synchronize()
        for s in runs:
            table, _, st = s["host"]
            _check(s["o"], s["q"], s["cache"], table, s["lens"].cpu(), st, scale, None)
    ops.check_status()


def test_calls_on_two_streams_at_once():
    ops = _ops()
    kv, group, d, page = 4, 4, 128, 32
    cases = []
    for i, (new, lens) in enumerate((([1] * 9, [700 + 31 * b for b in range(9)]), ([150, 3], [800, 90]))):
        table, ln, st, pages = _batch(new, lens, page, seed=i)
        cache = _full_cache(pages, kv, page, d, F16, 20 + i)
        q = _numbers((int(st[-1]), kv * group, d), F16, i).cuda()
        cases.append((q, cache, table.cuda(), ln.cuda(), st.cuda()))
    want = [ops.paged_attention(*c, scale=0.1) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(30):
        for s, c, g in zip(streams, cases, got):
            with torch.cuda.stream(s):
                g.append(ops.paged_attention(*c, scale=0.1))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)
    ops.check_status()


# ------------------------------------------------------------------------------------------------ drafts
@pytest.mark.parametrize("B,K,V,one_hot,ragged", [
    (1, 4, 49152, False, False), (7, 1, 1, False, False), (33, 5, 1001, False, True), (5, 8, 37, True, False), (4, 0, 500, True, False),
    (3, 40, 129, False, False), (2, 3, 131072 + 5, False, True), (16, 2, 8192, True, True), (64, 3, 33000, False, False),
])
def test_verify(B, K, V, one_hot, ragged):
    ops = _ops()
    g = torch.Generator().manual_seed(B * K + V)
    for trial in range(3):
        logits = 3.0 * torch.randn(B, K + 1, V, generator=g)
        probs = torch.softmax(logits, -1)
        draft = torch.softmax(logits[:, :K] + 0.5 * torch.randn(B, K, V, generator=g), -1)
        drafts = torch.multinomial(draft.reshape(B * K, V), 1, generator=g).reshape(B, K) if K else torch.empty(B, 0, dtype=torch.int64)
        u = torch.rand(B, K + 1, generator=g)
        u[0] = 0.0
        u[-1] = 1.0 - 2.0 ** -24
        counts = torch.randint(-1, K + 2, (B,), generator=g).int() if ragged else None
        want = paged.verify(probs, drafts, u, None if one_hot else draft, counts)
        got = ops.verify_drafts(probs.cuda(), drafts.cuda(), u.cuda(), None if one_hot else draft.cuda(),
                                None if counts is None else counts.cuda())
        ops.check_status()
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verify_rows_apart_and_unusual_numbers():
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    B, K, V = 6, 2, 700
    g = torch.Generator().manual_seed(3)
    wide = torch.zeros(B, K + 1, V + 61)
    wide[..., :V] = torch.softmax(2 * torch.randn(B, K + 1, V, generator=g), -1)
    wide[..., V:] = 1e9  # behind the rows
    probs, draft = wide[..., :V], torch.softmax(torch.randn(B, K + 3, V, generator=g), -1)[:, 1:K + 1]
    drafts = torch.randint(0, V, (B, K), generator=g)
    u = torch.rand(B, K + 1, generator=g)
    probs[1, :, 5:90] = float("nan")
    probs[2, 0] = draft[2, 0]        # nothing left of the difference: p itself
    u[2, 0], drafts[2, 0] = 0.9999999, 3
    probs[2, 0, 3] = 0.0
    draft[2, 0, 3] = 1e-30
    probs[3, 0, 10] = float("inf")
    probs[4, :] = -probs[4, :]
    u[5, K] = 1.0                    # not below 1: the last token that weighs anything
    probs[5, :, V - 20:] = 0.0
    c = wide.cuda()[..., :V]
    want = paged.verify(probs, drafts, u, draft)
    got = ops.verify_drafts(c, drafts.cuda(), u.cuda(), draft.cuda())
    with pytest.raises(FtbError):    # the row without a positive number
        ops.check_status()
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert int(got[0][4, 0]) == -1
    bad = drafts.clone()
    bad[0, 0], bad[3, 1] = V, -5
    probs[4] = probs[0]
    want = paged.verify(probs, bad, u, draft)
    got = ops.verify_drafts(probs.cuda(), bad.cuda(), u.cuda(), draft.cuda())
    with pytest.raises(FtbError):
        ops.check_status()
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    ops.check_status()


def test_verified_tokens_follow_the_target():
    """Over many random numbers the first token has the target's distribution, whatever the draft's."""
    ops = _ops()
    V, B = 8, 200000
    g = torch.Generator().manual_seed(1)
    p, q = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(torch.randn(V, generator=g), 0)
    probs, draft = p.expand(B, 2, V).contiguous(), q.expand(B, 1, V).contiguous()
    drafts = torch.multinomial(q, B, replacement=True, generator=g).reshape(B, 1)
    tokens, _ = ops.verify_drafts(probs.cuda(), drafts.cuda(), torch.rand(B, 2, generator=g).cuda(), draft.cuda())
    ops.check_status()
    share = torch.bincount(tokens[:, 0].cpu(), minlength=V) / B
    assert float((share - p).abs().max()) < 5 * math.sqrt(0.25 / B)  # five standard deviations of the widest


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("eight_bit", [False, True])
def test_steps_of_drafted_decoding(eight_bit):
    """A prompt in two chunks, then steps of three drafts: write, attend, project, verify; against the same in 64 bits."""
    ops = _ops()
    kv, group, d, page, V, K = 2, 2, 64, 16, 512, 3
    heads, H, B = kv * group, kv * group * d, 3
    scale = 1.0 / math.sqrt(d)
    table, _, _, pages = _batch([0] * B, [160] * B, page, seed=4)
    cache = ops.paged_cache(pages, kv, page, d, E4M3 if eight_bit else BF16)
    P = (0.5 * _numbers((H, V), BF16, 7, spread=0.0)).cuda()
    lens = [0] * B
    for step, n in enumerate(([70, 33, 1], [41, 64, 9], [K + 1] * B, [K + 1] * B)):
        st = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32)
        lens = [a + b for a, b in zip(lens, n)]
        ln = torch.tensor(lens, dtype=torch.int32)
        qkv = _numbers((sum(n), (heads + 2 * kv) * d), BF16, 30 + step, spread=0.2).cuda()
        q, k, v = (qkv[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
        args = (table.cuda(), ln.cuda(), st.cuda())
        ops.paged_cache_write(cache, k, v, *args)
        o = ops.paged_attention(q, cache, *args, scale=scale)
        _check(o, q, cache, table, ln, st, scale, None)
        if n[0] != K + 1:
            continue
        probs = ops.project_softmax_rows(o.reshape(sum(n), H), P).view(B, K + 1, V)
        g = torch.Generator().manual_seed(step)
        drafts = probs[:, :K].argmax(-1)
        drafts[1, 1] = 5
        u = torch.rand(B, K + 1, generator=g).cuda()
        tokens, counts = ops.verify_drafts(probs, drafts, u)
        ops.check_status()
        want = paged.verify(probs.cpu(), drafts.cpu(), u.cpu())
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
        # the tokens that were not taken leave the cache by their lengths alone
        lens = [a - (K + 1) + int(c) for a, c in zip(lens, counts)]


# --------------------------------------------------------------------------------------------- refusals
def test_refusals():
    ops = _ops()
    cache = ops.paged_cache(4, 2, 16, 64, BF16)
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    lens, starts = torch.ones(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 4, 64, dtype=BF16, device="cuda")
    k = torch.zeros(1, 2, 64, dtype=BF16, device="cuda")
    att = lambda q=q, cache=cache, table=table, lens=lens, starts=starts, **kw: ops.paged_attention(q, cache, table, lens, starts, **kw)
    put = lambda k=k, v=k, cache=cache, lens=lens: ops.paged_cache_write(cache, k, v, table, lens, starts)
    att(), put()
    for call, error in [
        (lambda: att(q=q.cpu()), RuntimeError), (lambda: att(q=q.half()), TypeError), (lambda: att(q=q.float()), TypeError),
        (lambda: att(q=q[:, :3]), ValueError), (lambda: att(q=q[..., :32]), ValueError), (lambda: att(q=q[0]), ValueError),
        (lambda: att(q=torch.zeros(1, 64, 4, dtype=BF16, device="cuda").transpose(1, 2)), ValueError),
        (lambda: att(q=torch.zeros(257, dtype=BF16, device="cuda")[1:].view(1, 4, 64)), ValueError),
        (lambda: att(window=0), ValueError), (lambda: att(scale=0.0), RuntimeError), (lambda: att(scale=float("inf")), RuntimeError),
        (lambda: att(scale=float("nan")), RuntimeError), (lambda: att(out=q[:, :2]), ValueError), (lambda: att(out=q.half()), TypeError), (lambda: att(out=q), RuntimeError),
        (lambda: att(cache=cache[:1]), TypeError), (lambda: att(cache=(cache[0], cache[1][:3])), ValueError),
        (lambda: att(cache=(cache[0].float(), cache[1].float())), TypeError), (lambda: att(cache=(cache[0].view(torch.uint8).view(E4M3),) * 2), ValueError),
        (lambda: att(cache=tuple(c.transpose(1, 2) for c in cache)), ValueError), (lambda: att(cache=tuple(c[:, :, :8].contiguous() for c in cache)), ValueError),
        (lambda: att(table=table.long()), TypeError), (lambda: att(table=table[0]), ValueError), (lambda: att(table=table.cpu()), RuntimeError),
        (lambda: att(lens=lens.float()), TypeError), (lambda: att(lens=torch.ones(2, dtype=torch.int32, device="cuda")), ValueError),
        (lambda: att(starts=lens), ValueError),
        (lambda: put(k=k[:, :1]), ValueError), (lambda: put(v=k[:0]), ValueError), (lambda: put(k=k.half(), v=k.half()), TypeError), (lambda: put(v=k.half()), TypeError),
        (lambda: ops.paged_cache_read(cache, table, lens, starts, 1, dtype=F16), TypeError),
        (lambda: ops.paged_cache_read(cache, table, lens, starts, 1, out=(k, k[0])), ValueError),
        (lambda: ops.paged_cache(0, 2, 16, 64, BF16), ValueError), (lambda: ops.paged_cache(1, 2, 24, 64, BF16), ValueError),
        (lambda: ops.paged_cache(1, 2, 16, 96, BF16), ValueError), (lambda: ops.paged_cache(1, 2, 16, 64, torch.float32), TypeError),
    ]:
        with pytest.raises(error):
            call()
    probs, drafts = torch.rand(2, 4, 10, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    u = torch.rand(2, 4, device="cuda")
    ops.verify_drafts(probs, drafts, u)
    for call, error in [
        (lambda: ops.verify_drafts(probs[:, :3], drafts, u), ValueError), (lambda: ops.verify_drafts(probs.double(), drafts, u), TypeError),
        (lambda: ops.verify_drafts(probs.cpu(), drafts, u), RuntimeError), (lambda: ops.verify_drafts(probs, drafts.int(), u), TypeError),
        (lambda: ops.verify_drafts(probs, drafts[0], u), ValueError), (lambda: ops.verify_drafts(probs, drafts, u[:, :3].contiguous()), ValueError),
        (lambda: ops.verify_drafts(probs, drafts, u, draft_probs=probs), ValueError),
        (lambda: ops.verify_drafts(probs, drafts, u, draft_probs=probs[:, :3, :9]), ValueError),
        (lambda: ops.verify_drafts(probs, drafts, u, counts=drafts[:, 0].contiguous()), TypeError),
        (lambda: ops.verify_drafts(probs.transpose(1, 2).contiguous().transpose(1, 2), drafts, u), ValueError),
        (lambda: ops.verify_drafts(probs[:, :, :0], drafts, u), ValueError),
    ]:
        with pytest.raises(error):
            call()
    # nothing to do
    empty = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(q[:0], cache, table, lens, empty).shape == (0, 4, 64)
    ops.paged_cache_write(cache, k[:0], k[:0], table, lens, empty)
    assert ops.paged_cache_read(cache, table, lens, empty, 0)[0].shape == (0, 2, 64)
    assert ops.verify_drafts(probs[:0], drafts[:0], u[:0])[0].shape == (0, 4)
    ops.check_status()

"""Attention for trees of drafted tokens, their masks and their verification, against the 64-bit oracle."""
import math
import random

import pytest
import torch

from oracle import paged, tree

from test_gpu_paged import BF16, E4M3, F16, _batch, _bits, _full_cache, _numbers

pytestmark = pytest.mark.gpu


def _ops():
    from fractaltensor_b200 import ops
    return ops


def _parents(N, seed):
    r = random.Random(seed)
    return [-1] + [r.randrange(max(0, i - 9), i) for i in range(1, N)]


# -------------------------------------------------------------------------------------------------- mask
@pytest.mark.parametrize("B,N", [(1, 1), (3, 2), (2, 31), (2, 32), (3, 33), (2, 64), (5, 100), (1, 1030)])
def test_mask(B, N):
    ops = _ops()
    parents = torch.tensor([_parents(N, 7 * b + N) for b in range(B)], dtype=torch.int32)
    if N > 5:  # parents that do not lie in front are none
        parents[0, 3], parents[B - 1, 4], parents[0, 5] = 3, -7, 2 ** 31 - 1
    got = ops.tree_mask(parents.cuda())
    assert torch.equal(got.cpu(), tree.mask(parents))


# --------------------------------------------------------------------------------------------- attention
def _tree_rows(new, starts, rows, seed, words=None):
    """Masks of random trees for packed rows; rows of no sequence have all bits."""
    words = words or max(1, (max(new) + 31) // 32)
    out = torch.full((rows, words), -1, dtype=torch.int32)
    for b, n in enumerate(new):
        if n > 0:
            m = tree.mask(torch.tensor([_parents(n, seed + b)]))[0][:, :words]
            out[int(starts[b]):int(starts[b]) + n, : m.shape[1]] = m
    return out


def _check(o, lse, q, cache, table, ln, st, scale, window=None, mask=None):
    want, bound, want_lse = tree.attention(q, cache, table, ln, st, scale, window, mask)
    keys, d = int(ln.max()), q.shape[2]
    tol = paged.tolerance(want, bound, q.dtype, d, len(cache) == 4, keys)
    lo, hi = int(st[0]), int(st[-1])
    err = (o.double().cpu() - want).abs()
    bad = ~(err[lo:hi] <= tol[lo:hi])
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol)[lo:hi].nan_to_num(9e9).max()), bad.nonzero()[:5].tolist())
    if lse is not None:
        tol = tree.lse_tolerance(want_lse, bound[1], d, len(cache) == 4, keys)
        lse = lse.double().cpu()
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isneginf(lse[lo:hi]), empty[lo:hi])
        err = torch.where(empty, 0.0, (lse - want_lse).abs())
        assert bool((err[lo:hi] <= tol[lo:hi]).all()), float((err / tol)[lo:hi].nan_to_num(9e9).max())


SHAPES = [
    # kv, group, d, page, new, lens
    (1, 1, 64, 16, [1], [1]),
    (1, 4, 128, 16, [5], [5]),
    (8, 4, 128, 16, [25], [200]),
    (2, 2, 128, 64, [2, 1, 3], [5, 64, 333]),
    (2, 1, 64, 32, [1, 0, 7, 1], [31, 0, 7, 65]),
    (1, 16, 128, 128, [9, 9], [129, 511]),
    (2, 3, 64, 16, [13, 13, 13], [100, 13, 47]),
    (4, 2, 128, 16, [33, 64, 40], [33, 300, 91]),
    (1, 8, 128, 64, [64, 64], [64, 1500]),
    (1, 5, 128, 32, [100], [230]),
    (1, 2, 64, 16, [130, 3], [700, 44]),
    (1, 1, 64, 16, [1, 1, 1], [600, 1, 129]),
    (1, 8, 64, 32, [2, 2, 1, 1], [400, 90, 17, 64]),
    # a few rows behind whole tiles of 256 or 128
    (1, 8, 128, 64, [33, 33], [700, 90]),
    (1, 8, 128, 64, [33], [6000]),
    (2, 16, 64, 16, [17, 20, 3], [300, 40, 77]),
    (1, 1, 128, 32, [130, 129, 5], [200, 900, 30]),
]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,group,d,page,new,lens", SHAPES)
def test_attention(dtype, eight_bit, kv, group, d, page, new, lens):
    """Unwritten rows of the pages hold NaN, rows around the sequences keep what they hold."""
    ops = _ops()
    table, ln, st, pages = _batch(new, lens, page, front=1)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else dtype, 3, table, ln)
    T = int(st[-1]) + 2
    mask = _tree_rows(new, st, T, 11)
    qkv = _numbers((T, (kv * group + 1) * d), dtype, 9, spread=0.3).cuda()
    q = qkv[:, d:].unflatten(1, (kv * group, d))
    out = torch.full((T, kv * group, d), 5.0, dtype=dtype, device="cuda")
    lse = torch.full((T, kv * group), 7.0, device="cuda")
    scale = 1.0 / math.sqrt(d)
    got = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=scale, out=out, tree=mask.cuda(), lse=lse)
    ops.check_status()
    assert got is out and bool((out[0] == 5.0).all()) and bool((out[-2:] == 5.0).all())
    assert bool((lse[0] == 7.0).all()) and bool((lse[-2:] == 7.0).all())
    _check(out, lse, q, cache, table, ln, st, scale, mask=mask)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens,group", [([1, 1], [300, 17], 4), ([3], [50], 2), ([40, 33], [40, 300], 4), ([200, 1], [500, 64], 8)])
def test_any_bits_rows_without_any(eight_bit, new, lens, group):
    """Masks that are no trees; tokens that see no new token, not even themselves, and with no key in front nothing at all."""
    ops = _ops()
    kv, d, page = 2, 128, 32
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    g = torch.Generator().manual_seed(4)
    mask = torch.randint(-2 ** 31, 2 ** 31, (T, (max(new) + 31) // 32 + 1), generator=g).int()
    mask[::3] = 0
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    lse = torch.empty(T, kv * group, device="cuda")
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.08, tree=mask.cuda(), lse=lse)
    ops.check_status()
    _check(o, lse, q, cache, table, ln, st, 0.08, mask=mask)
    empty = [t for b in range(len(new)) if new[b] == lens[b] for t in range(int(st[b]), int(st[b + 1])) if t % 3 == 0]
    assert bool((o[empty] == 0).all()) and bool(torch.isneginf(lse[empty]).all())


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 1], [300, 17]), ([7], [90]), ([60, 2], [60, 300]), ([300, 40], [500, 64])])
def test_all_bits_are_no_mask(eight_bit, new, lens):
    """A mask of ones, of columns for all tokens or for a few, hides nothing; and lse does not change the result's bits."""
    ops = _ops()
    kv, group, d, page = 2, 4, 128, 16
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else F16, 3, table, ln)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), F16, 1).cuda()
    args = (q, cache, table.cuda(), ln.cuda(), st.cuda())
    want = ops.paged_attention(*args, scale=0.1)
    lse = [torch.empty(T, kv * group, device="cuda") for _ in range(3)]
    assert torch.equal(_bits(ops.paged_attention(*args, scale=0.1, lse=lse[0])), _bits(want))
    got = []
    for i, words in enumerate((1, (max(new) + 31) // 32 + 2)):
        ones = torch.full((T, words), -1, dtype=torch.int32, device="cuda")
        got.append(ops.paged_attention(*args, scale=0.1, tree=ones, lse=lse[1 + i]))
    ops.check_status()
    assert torch.equal(_bits(got[0]), _bits(got[1])) and torch.equal(lse[1], lse[2])
    _check(want, lse[0], q, cache, table, ln, st, 0.1)
    _check(got[0], lse[1], q, cache, table, ln, st, 0.1)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("new,lens,window", [([1, 1], [300, 17], 40), ([3], [50], 5), ([100, 33], [100, 300], 64), ([260], [600], 100)])
def test_lse_of_windows(eight_bit, new, lens, window):
    ops = _ops()
    kv, group, d, page = 2, 4, 64, 16
    table, ln, st, pages = _batch(new, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    q = _numbers((int(st[-1]), kv * group, d), BF16, 1).cuda()
    lse = torch.empty(int(st[-1]), kv * group, device="cuda")
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.1, window=window, lse=lse)
    ops.check_status()
    _check(o, lse, q, cache, table, ln, st, 0.1, window)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("new,lens", [([4, 4], [30, 70]), ([30], [200]), ([70, 70], [140, 300])])
def test_other_branches_have_no_part(eight_bit, what, new, lens):
    """What a token's branch does not see may hold anything, its keys and its values."""
    ops = _ops()
    kv, group, d, page = 2, 4, 128, 16
    table, ln, st, pages = _batch(new, lens, page)
    clean = _full_cache(pages, kv, page, d, BF16, 3)
    T = int(st[-1])
    mask = torch.zeros(T, 3, dtype=torch.int32)
    spoilt = [c.clone() for c in clean]
    for b in range(len(new)):  # the second token is nobody's parent
        for i in range(new[b]):
            for j in range(i + 1):
                if j != 1 or i == 1:
                    w = int(mask[int(st[b]) + i, j // 32]) & 0xffffffff | 1 << (j % 32)
                    mask[int(st[b]) + i, j // 32] = w - 2 ** 32 if w >= 2 ** 31 else w
        pos = lens[b] - new[b] + 1
        for c in spoilt:
            c[int(table[b, pos // page]), :, pos % page, ::3] = what
    if eight_bit:
        clean, spoilt = ([x.cuda() for x in (kc.view(E4M3), vc.view(E4M3), ke, ve)] for (kc, ke), (vc, ve) in
                         ((paged.quantise(c[0].cpu()), paged.quantise(c[1].cpu())) for c in (clean, spoilt)))
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    lse = torch.empty(T, kv * group, device="cuda")
    o = ops.paged_attention(q, tuple(spoilt), table.cuda(), ln.cuda(), st.cuda(), scale=0.08, tree=mask.cuda(), lse=lse)
    ops.check_status()
    rows = [int(st[b]) + i for b in range(len(new)) for i in range(new[b]) if i != 1]
    want, bound, want_lse = tree.attention(q, tuple(clean), table, ln, st, 0.08, None, mask)
    tol = paged.tolerance(want, bound, BF16, d, eight_bit, max(lens))
    assert bool(((o.double().cpu() - want).abs() <= tol)[rows].all())
    tol = tree.lse_tolerance(want_lse, bound[1], d, eight_bit, max(lens))
    assert bool(((lse.double().cpu() - want_lse).abs() <= tol)[rows].all())


@pytest.mark.parametrize("new,lens", [([1, 1], [300, 17]), ([9], [90]), ([40, 70], [40, 300]), ([150], [500])])
def test_lse_over_values_of_very_different_sizes(new, lens):
    """8 bits: what a value's exponent does to its weight has no part in the logarithm."""
    ops = _ops()
    kv, group, d, page = 2, 4, 128, 16
    table, ln, st, pages = _batch(new, lens, page)
    k, v = _numbers((pages, kv, page, d), torch.float32, 3), _numbers((pages, kv, page, d), torch.float32, 4)
    g = torch.Generator().manual_seed(1)
    by = torch.tensor([0.0, 2.0 ** -100, 2.0 ** -40, 1.0, 2.0 ** 20])[torch.randint(0, 5, (pages, kv, page), generator=g)]
    (kc, ke), (vc, ve) = paged.quantise(k), paged.quantise(v * by[..., None])
    cache = tuple(x.cuda() for x in (kc.view(E4M3), vc.view(E4M3), ke, ve))
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    mask = _tree_rows(new, st, T, 5)
    lse = torch.empty(T, kv * group, device="cuda")
    ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), scale=0.08, tree=mask.cuda(), lse=lse)
    ops.check_status()
    _, bound, want = tree.attention(q, cache, table, ln, st, 0.08, None, mask)
    err = (lse.double().cpu() - want).abs()
    assert bool((err <= tree.lse_tolerance(want, bound[1], d, True, max(lens))).all()), float(err.max())


def test_logarithms_of_layers_side_by_side():
    """lse may begin anywhere: a slice of one array for all layers."""
    ops = _ops()
    table, ln, st, pages = _batch([3], [40], 16)
    cache = _full_cache(pages, 1, 16, 64, BF16, 3)
    q = _numbers((3, 3, 64), BF16, 1).cuda()
    layers = torch.zeros(4, 3, 3, device="cuda")
    for x in layers:
        ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), lse=x)
    weights = torch.zeros(pages * 16 + 1, device="cuda")[1:].view(pages, 1, 16)
    ops.paged_attention_weights(q, cache, weights, layers[1], table.cuda(), ln.cuda(), st.cuda())
    ops.check_status()
    assert bool((layers == layers[0]).all()) and abs(float(weights.sum()) - 9) < 1e-4


def test_calls_on_two_streams_at_once():
    ops = _ops()
    kv, group, d, page, N, V = 2, 8, 128, 16, 33, 9000
    table, ln, st, pages = _batch([N, N], [900, 1500], page)
    cache = _full_cache(pages, kv, page, d, BF16, 3)
    qs = [_numbers((2 * N, kv * group, d), BF16, i).cuda() for i in range(2)]
    trees = [tuple(x.cuda() for x in _forest(2, N, V, i)) for i in range(2)]
    args = (cache, table.cuda(), ln.cuda(), st.cuda())

    def step(i):
        probs, tokens, parents, u = trees[i]
        return (ops.paged_attention(qs[i], *args, scale=0.1, tree=ops.tree_mask(parents).flatten(0, 1)),) + ops.verify_tree(probs, tokens, parents, u)

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(step(i))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(x, y))
    ops.check_status()


def test_refusals():
    ops = _ops()
    table, ln, st, pages = _batch([3], [40], 16)
    cache = _full_cache(pages, 1, 16, 64, BF16, 3)
    q = _numbers((3, 2, 64), BF16, 1).cuda()
    args = (q, cache, table.cuda(), ln.cuda(), st.cuda())
    mask = torch.full((3, 1), -1, dtype=torch.int32, device="cuda")
    good = ops.paged_attention(*args, tree=mask)
    for kw in (dict(tree=mask[:2]), dict(tree=mask[:, 0]), dict(tree=mask[:, :0]), dict(tree=mask, window=4), dict(lse=torch.empty(3, 1, device="cuda"))):
        with pytest.raises(ValueError):
            ops.paged_attention(*args, **kw)
    for kw in (dict(tree=mask.long()), dict(lse=torch.empty(3, 2, dtype=BF16, device="cuda"))):
        with pytest.raises(TypeError):
            ops.paged_attention(*args, **kw)
    from fractaltensor_b200._lib import FtbError
    for kw in (dict(lse=good.view(torch.float32).view(-1)[:6].view(3, 2), out=good), dict(lse=cache[0].view(torch.float32).view(-1)[:6].view(3, 2)),
               dict(out=good, tree=good.view(torch.int32).view(-1)[:3].view(3, 1))):
        with pytest.raises(FtbError):
            ops.paged_attention(*args, **kw)


# ------------------------------------------------------------------------------------------ verification
def _forest(B, N, V, seed):
    """Trees whose tokens are likely ones, some of them twice among siblings."""
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    logits = 2.5 * torch.randn(B, N, V, generator=g)
    probs = torch.softmax(logits, -1)
    parents = torch.tensor([_parents(N, seed + 13 * b) for b in range(B)], dtype=torch.int32)
    tokens = torch.zeros(B, N, dtype=torch.int64)
    top = probs.topk(min(V, 6), -1).indices
    for b in range(B):
        for i in range(N):
            tokens[b, i] = top[b, max(0, int(parents[b, i])), r.randrange(top.shape[2])]
    return probs, tokens, parents, torch.rand(B, N, generator=g)


def _same(got, want):
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (2, 1, 5000), (3, 7, 11), (64, 33, 300), (5, 64, 4097), (4, 25, 49152), (40, 13, 9001), (1, 1024, 130), (2, 100, 130001)])
def test_verify(B, N, V):
    ops = _ops()
    probs, tokens, parents, u = _forest(B, N, V, B + N + V)
    got = ops.verify_tree(probs.cuda(), tokens.cuda(), parents.cuda(), u.cuda())
    ops.check_status()
    _same(got, tree.verify(probs, tokens, parents, u))


def test_a_chain_is_what_verify_drafts_takes():
    ops = _ops()
    B, K, V = 50, 6, 5000
    g = torch.Generator().manual_seed(3)
    probs = torch.softmax(4 * torch.randn(B, K + 1, V, generator=g), -1).cuda()
    drafts = torch.multinomial(probs[:, :K].reshape(B * K, V), 1).reshape(B, K)
    u = torch.rand(B, K + 1, generator=g).cuda()
    tokens, counts = ops.verify_drafts(probs, drafts, u)
    parents = torch.arange(-1, K).int().expand(B, K + 1).contiguous().cuda()
    own = torch.cat([drafts[:, :1] * 0, drafts], 1)
    got = ops.verify_tree(probs, own, parents, torch.cat([u[:, K:], u[:, :K]], 1))
    ops.check_status()
    assert torch.equal(got[0], tokens) and torch.equal(got[2], counts) and int(counts.max()) > 2
    assert torch.equal(got[1], torch.where(torch.arange(K + 1).cuda() < counts[:, None], torch.arange(K + 1).cuda(), -1).int())


def test_verify_extremes():
    """Nothing left, numbers that are none, tokens without a parent, outside the vocabulary, the same twice; u at its ends."""
    ops = _ops()
    from fractaltensor_b200._lib import FtbError
    V = 40
    rows = torch.full((9, 4, V), 1.0 / V)
    rows[0, 0] = 0.0
    rows[0, 0, 7] = 1.0                                # all of it is the one that u refuses at 1: nothing is left
    rows[1, 0, 3], rows[1, 0, 4] = float("nan"), float("inf")
    rows[2, 0] = -1.0                                  # a row without a probability
    rows[3, 0] = 0.0
    rows[3, 0, 5:7] = 0.5
    tokens = torch.tensor([[0, 7, 7, 7], [0, 3, 4, 9], [0, 1, 2, 3], [0, 5, 5, 6], [0, 1, 2, 3], [0, 1, 2, 3], [0, 39, 0, 1], [0, 1, 1, 1], [0, 99, -5, 2]])
    parents = torch.tensor([[-1, 0, 0, 0], [-1, 0, 0, 0], [-1, 0, 1, 2], [-1, 0, 0, 0], [-1, -1, 2, 0], [-1, 0, 1, 2], [-1, 0, 1, 1], [-1, 0, 0, 0],
                            [-1, 0, 0, 0]]).int()
    for first in (0.0, 0.5, 1.0 - 2.0 ** -24):
        for rest in (0.0, 0.6, 1.0, 2.0):
            u = torch.full((9, 4), rest)
            u[:, 0] = first
            got = ops.verify_tree(rows.cuda(), tokens.cuda(), parents.cuda(), u.cuda())
            with pytest.raises(FtbError):  # row 2, and the tokens of the last one
                ops.check_status()
            _same(got, tree.verify(rows, tokens, parents, u))
    good = [4, 5, 6, 7]
    ops.verify_tree(rows[good].cuda(), tokens[good].cuda(), parents[good].cuda(), u[good].cuda())
    ops.check_status()


def test_verify_strided_rows():
    ops = _ops()
    probs, tokens, parents, u = _forest(3, 9, 700, 1)
    wide = torch.full((9, 3, 705), float("nan")).cuda()
    wide[:, :, 2:702] = probs.transpose(0, 1).cuda()
    got = ops.verify_tree(wide[:, :, 2:702].transpose(0, 1), tokens.cuda(), parents.cuda(), u.cuda())
    ops.check_status()
    _same(got, tree.verify(probs, tokens, parents, u))


def test_verification_samples_the_target():
    """First tokens of many sequences with the same row: each share within 5 standard deviations of its probability."""
    ops = _ops()
    B, N, V = 20000, 4, 12
    p = torch.softmax(torch.randn(V, generator=torch.Generator().manual_seed(5)), -1)
    u = torch.rand(B, N, generator=torch.Generator().manual_seed(6))
    tokens = torch.tensor([0, 3, 5, 1]).expand(B, N).contiguous()
    parents = torch.tensor([-1, 0, 0, 0]).int().expand(B, N).contiguous()
    out, path, counts = ops.verify_tree(p.cuda().expand(B, N, V), tokens.cuda(), parents.cuda(), u.cuda())
    share = torch.bincount(out[:, 0].cpu(), minlength=V) / B
    assert bool(((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all())


def test_verify_refusals():
    ops = _ops()
    probs, tokens, parents, u = (x.cuda() for x in _forest(2, 3, 50, 1))
    for args in ((probs[:1], tokens, parents, u), (probs[:, :2], tokens, parents, u), (probs, tokens[:, :2], parents, u), (probs, tokens, parents, u[:1]),
                 (probs[..., ::2], tokens, parents, u), (probs[..., :0], tokens, parents, u), (probs, tokens, parents[0], u)):
        with pytest.raises(ValueError):
            ops.verify_tree(*(a if i == 0 else a.contiguous() for i, a in enumerate(args)))
    for args in ((probs.half(), tokens, parents, u), (probs, tokens.int(), parents, u), (probs, tokens, parents.long(), u), (probs, tokens, parents, u.double())):
        with pytest.raises(TypeError):
            ops.verify_tree(*args)
    with pytest.raises(ValueError):
        ops.tree_mask(parents[0])
    with pytest.raises(TypeError):
        ops.tree_mask(parents.long())
    assert ops.tree_mask(parents[:0]).shape == (0, 3, 1)
    assert ops.verify_tree(probs[:0], tokens[:0], parents[:0], u[:0])[2].shape == (0,)


# ------------------------------------------------------------------------------------------- the whole step
@pytest.mark.parametrize("eight_bit", [False, True])
def test_a_step_of_drafted_trees(eight_bit):
    """Write, attend, verify, keep: the cache then holds what a plain run over the accepted tokens writes, and the next
    token attends to the same."""
    ops = _ops()
    kv, group, d, page, B, N, V = 2, 4, 128, 16, 3, 21, 500
    lens0 = [40, 7, 123]
    table, _, _, pages = _batch([0] * B, [n + 2 * N for n in lens0], page)
    table = table.cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    make = lambda n, s: _numbers((n, kv, d), BF16, s).cuda()
    cache = ops.paged_cache(pages, kv, page, d, E4M3 if eight_bit else BF16)
    plain = ops.paged_cache(pages, kv, page, d, E4M3 if eight_bit else BF16)
    k0, v0 = make(sum(lens0), 1), make(sum(lens0), 2)
    starts0 = i32([0, 40, 47, 170])
    for c in (cache, plain):
        ops.paged_cache_write(c, k0, v0, table, i32(lens0), starts0)
    probs, tokens, parents, u = (x.cuda() for x in _forest(B, N, V, 4))
    k, v = make(B * N, 3), make(B * N, 4)
    q = _numbers((B * N, kv * group, d), BF16, 5).cuda()
    lens, starts = i32([n + N for n in lens0]), i32([0, N, 2 * N, 3 * N])
    ops.paged_cache_write(cache, k, v, table, lens, starts)
    o = ops.paged_attention(q, cache, table, lens, starts, scale=0.08, tree=ops.tree_mask(parents).flatten(0, 1))
    out, path, counts = ops.verify_tree(probs, tokens, parents, u)
    ops.paged_cache_keep(cache, path, counts, table, first=i32(lens0))
    ops.check_status()
    now = i32(lens0) + counts
    n = counts.tolist()
    assert max(n) > 2
    rows = torch.cat([b * N + path[b, : n[b]].long() for b in range(B)])
    new = i32([0] + [sum(n[: b + 1]) for b in range(B)])
    ops.paged_cache_write(plain, k[rows], v[rows], table, now, new)
    # the accepted tokens saw what they see in a plain run over them
    again = ops.paged_attention(q[rows], plain, table, now, new, scale=0.08)
    assert float((again.float() - o[rows].float()).abs().max()) <= 2.0 ** -6 * float(again.float().abs().max())
    whole = i32([0] + [int(now[: b + 1].sum()) for b in range(B)])
    for x, y in zip(ops.paged_cache_read(cache, table, now, whole, int(whole[-1])), ops.paged_cache_read(plain, table, now, whole, int(whole[-1]))):
        assert torch.equal(_bits(x), _bits(y))
    ops.check_status()


@pytest.mark.parametrize("eight_bit", [False, True])
def test_captured_and_on_another_stream(eight_bit):
    """A captured step follows the lengths, masks and random numbers that its buffers get."""
    ops = _ops()
    kv, group, d, page, B, N, V = 2, 2, 64, 16, 2, 9, 300
    table, ln, st, pages = _batch([N, N], [60, 25], page, width=8)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else F16, 3)
    q = _numbers((B * N, kv * group, d), F16, 1).cuda()
    probs, tokens, parents, u = (x.cuda() for x in _forest(B, N, V, 9))
    table, ln, st = table.cuda(), ln.cuda(), st.cuda()
    lse = torch.empty(B * N, kv * group, device="cuda")

    def step():
        mask = ops.tree_mask(parents)
        return ops.paged_attention(q, cache, table, ln, st, scale=0.1, tree=mask.flatten(0, 1), lse=lse), ops.verify_tree(probs, tokens, parents, u)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        o, (out, path, counts) = step()
    for seed in (20, 21):
        new = _forest(B, N, V, seed)
        for x, y in zip((probs, tokens, parents, u), new):
            x.copy_(y)
        ln.copy_(torch.tensor([60 - seed, 26]))
        graph.replay()
        torch.cuda.synchronize()
        _same((out, path, counts), tree.verify(*new))
        _check(o, lse, q, cache, table.cpu(), ln.cpu(), st.cpu(), 0.1, mask=tree.mask(new[2]).flatten(0, 1))
    ops.check_status()

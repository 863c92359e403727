"""Trees of drafted tokens in the attention kernel for many rows, which takes calls that make many units of work: here, tables for long contexts."""
import math

import pytest
import torch

from oracle import paged, tree

from test_gpu_paged import BF16, E4M3, F16, _batch, _bits, _full_cache, _numbers
from test_gpu_tree import _check, _tree_rows

pytestmark = pytest.mark.gpu

WIDTH = 4000  # pages of a row of the table: 64 000 keys and more, 1024 units for every tile of 16 rows


def _attend(q, cache, table, ln, st, **kw):
    """The call, and that it ran three kernels: for many rows, for few rows, and what joins them.  (Two are those for few rows and their join.)"""
    from fractaltensor_b200 import ops
    from fractaltensor_b200._lib import lib
    kw.setdefault("lse", torch.full(q.shape[:2], 7.0, device="cuda"))
    n = lib.ftb_launch_count()
    o = ops.paged_attention(q, cache, table.cuda(), ln.cuda(), st.cuda(), **kw)
    assert lib.ftb_launch_count() - n == 3
    ops.check_status()
    return o, kw["lse"]


SHAPES = [
    # kv, group, d, page, new, lens; tiles of 128 rows
    (2, 4, 128, 16, [25, 9], [200, 300]),
    (4, 1, 64, 16, [70, 17, 1], [100, 17, 129]),
    (4, 16, 64, 32, [5, 8], [5, 300]),
    (3, 3, 128, 64, [13, 0, 13, 40], [100, 9, 13, 500]),
    (8, 4, 128, 128, [33, 3], [1500, 60]),      # 4 rows behind a tile
    (8, 4, 64, 16, [34, 2], [700, 2]),          # 8
    (8, 4, 128, 32, [35, 2], [129, 128]),       # 12, which are too many
    (4, 8, 64, 16, [16, 16], [16, 1000]),       # whole tiles
    # of 256
    (4, 8, 128, 64, [33, 33], [700, 90]),       # 8 behind it
    (4, 8, 64, 16, [34, 34], [300, 34]),        # 16
    (4, 8, 128, 16, [35, 35], [35, 257]),       # 24: a second tile
    (4, 4, 128, 32, [70, 1, 66], [900, 40, 66]),
    (8, 2, 64, 16, [300, 40], [700, 64]),
    (2, 1, 128, 16, [520, 3], [520, 44]),
    (8, 8, 128, 64, [33], [6000]),              # one sequence, the last rows apart
    (8, 4, 64, 32, [65], [65]),
]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,group,d,page,new,lens,around", [s + (a,) for s in SHAPES for a in (0, 1) if len(s[4]) > 1 or a == 0])
def test_attention(dtype, eight_bit, kv, group, d, page, new, lens, around):
    """Unwritten rows of the pages hold NaN, rows around the sequences keep what they hold (and count in the choice of tiles)."""
    table, ln, st, pages = _batch(new, lens, page, width=WIDTH, front=around)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else dtype, 3, table, ln)
    lo, hi = int(st[0]), int(st[-1])
    T = hi + 2 * around
    mask = _tree_rows(new, st, T, 11)
    q = _numbers((T, (kv * group + 1) * d), dtype, 9, spread=0.3).cuda()[:, d:].unflatten(1, (kv * group, d))
    out = torch.full((T, kv * group, d), 5.0, dtype=dtype, device="cuda")
    scale = 1.0 / math.sqrt(d)
    o, lse = _attend(q, cache, table, ln, st, scale=scale, out=out, tree=mask.cuda())
    assert o is out and bool((out[:lo] == 5.0).all()) and bool((out[hi:] == 5.0).all())
    assert bool((lse[:lo] == 7.0).all()) and bool((lse[hi:] == 7.0).all())
    _check(o, lse, q, cache, table, ln, st, scale, mask=mask)
    again, _ = _attend(q, cache, table, ln, st, scale=scale, out=torch.full_like(out, 5.0), tree=mask.cuda())
    assert torch.equal(_bits(again), _bits(o))


FORMS = [(4, [40, 33], [40, 300]), (8, [200, 1], [500, 64]), (8, [33, 33], [33, 160]), (1, [130, 60], [150, 60])]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("words", [1, 0, 3])
@pytest.mark.parametrize("group,new,lens", FORMS)
def test_any_bits_rows_without_any(eight_bit, words, group, new, lens):
    """Masks that are no trees, of fewer words than new tokens have bits or of more; tokens that see no new token, not even themselves, and with no
    key in front nothing at all."""
    kv, d, page = 4, 128, 32
    table, ln, st, pages = _batch(new, lens, page, width=WIDTH)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    words = words if words == 1 else (max(new) + 31) // 32 + words
    mask = torch.randint(-2 ** 31, 2 ** 31, (T, words), generator=torch.Generator().manual_seed(4)).int()
    mask[::3] = 0
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    o, lse = _attend(q, cache, table, ln, st, scale=0.08, tree=mask.cuda())
    _check(o, lse, q, cache, table, ln, st, 0.08, mask=mask)
    empty = [t for b in range(len(new)) if new[b] == lens[b] for t in range(int(st[b]), int(st[b + 1])) if t % 3 == 0 and t - int(st[b]) < 32 * words]
    assert len(empty) > 0 or new[0] != lens[0]
    assert bool((o[empty] == 0).all()) and bool(torch.isneginf(lse[empty]).all())


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("group,new,lens", FORMS)
def test_all_bits_are_no_mask(eight_bit, group, new, lens):
    """A mask of ones, of columns for all tokens or for a few, hides nothing; and lse does not change the result's bits."""
    kv, d, page = 4, 64, 16
    table, ln, st, pages = _batch(new, lens, page, width=WIDTH)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else F16, 3, table, ln)
    T = int(st[-1])
    q = _numbers((T, kv * group, d), F16, 1).cuda()
    got = [_attend(q, cache, table, ln, st, scale=0.1, tree=torch.full((T, words), -1, dtype=torch.int32, device="cuda"))
           for words in (1, (max(new) + 31) // 32 + 2)]
    assert torch.equal(_bits(got[0][0]), _bits(got[1][0])) and torch.equal(got[0][1], got[1][1])
    none, _ = _attend(q, cache, table, ln, st, scale=0.1, tree=torch.full((T, 1), -1, dtype=torch.int32, device="cuda"), lse=None)
    assert torch.equal(_bits(none), _bits(got[0][0]))
    _check(*got[0], q, cache, table, ln, st, 0.1)


def _without_second(new, lens, st, T):
    """A mask in which every sequence's second token is nobody's parent, and where that one is: [(sequence, position)]."""
    mask = torch.zeros(T, (max(new) + 31) // 32, dtype=torch.int64)
    at = []
    for b, n in enumerate(new):
        for i in range(n):
            for j in range(i + 1):
                if j != 1 or i == 1:
                    mask[int(st[b]) + i, j // 32] |= 1 << (j % 32)
        if n > 1:
            at.append((b, lens[b] - n + 1))
    return torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).int(), at


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("group,new,lens", [(4, [40, 33], [140, 300]), (8, [33, 33], [33, 160]), (8, [33], [900])])
def test_other_branches_have_no_part(eight_bit, what, group, new, lens):
    """What a token's branch does not see may hold anything, its keys and its values."""
    kv, d, page = 8, 128, 16
    table, ln, st, pages = _batch(new, lens, page, width=WIDTH)
    clean = _full_cache(pages, kv, page, d, BF16, 3)
    T = int(st[-1])
    mask, at = _without_second(new, lens, st, T)
    spoilt = [c.clone() for c in clean]
    for b, pos in at:
        for c in spoilt:
            c[int(table[b, pos // page]), :, pos % page, ::3] = what
    if eight_bit:
        clean, spoilt = ([x.cuda() for x in (kc.view(E4M3), vc.view(E4M3), ke, ve)] for (kc, ke), (vc, ve) in
                         ((paged.quantise(c[0].cpu()), paged.quantise(c[1].cpu())) for c in (clean, spoilt)))
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    o, lse = _attend(q, tuple(spoilt), table, ln, st, scale=0.08, tree=mask.cuda())
    rows = [int(st[b]) + i for b in range(len(new)) for i in range(new[b]) if i != 1]
    want, bound, want_lse = tree.attention(q, tuple(clean), table, ln, st, 0.08, None, mask)
    tol = paged.tolerance(want, bound, BF16, d, eight_bit, max(lens))
    assert bool(((o.double().cpu() - want).abs() <= tol)[rows].all())
    tol = tree.lse_tolerance(want_lse, bound[1], d, eight_bit, max(lens))
    assert bool(((lse.double().cpu() - want_lse).abs() <= tol)[rows].all())


@pytest.mark.parametrize("group,new,lens", [(4, [40, 70], [40, 300]), (8, [33, 33], [90, 160]), (8, [33], [500])])
def test_values_of_very_different_sizes(group, new, lens):
    """8 bits: exponents far apart in the blocks that a mask reaches into."""
    kv, d, page = 8, 128, 16
    table, ln, st, pages = _batch(new, lens, page, width=WIDTH)
    k, v = _numbers((pages, kv, page, d), torch.float32, 3), _numbers((pages, kv, page, d), torch.float32, 4)
    g = torch.Generator().manual_seed(1)
    by = torch.tensor([0.0, 2.0 ** -100, 2.0 ** -40, 1.0, 2.0 ** 20])[torch.randint(0, 5, (pages, kv, page), generator=g)]
    (kc, ke), (vc, ve) = paged.quantise(k), paged.quantise(v * by[..., None])
    cache = tuple(x.cuda() for x in (kc.view(E4M3), vc.view(E4M3), ke, ve))
    T = int(st[-1])
    q = _numbers((T, kv * group, d), BF16, 1).cuda()
    mask = _tree_rows(new, st, T, 5)
    o, lse = _attend(q, cache, table, ln, st, scale=0.08, tree=mask.cuda())
    _check(o, lse, q, cache, table, ln, st, 0.08, mask=mask)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_cut_tiles(eight_bit):
    """A few tiles behind thousands of keys: each is cut into a dozen pieces or more, and the last rows' too."""
    kv, group, d, page, new, lens = 2, 8, 128, 64, [34, 33], [5000, 3100]
    table, ln, st, pages = _batch(new, lens, page, width=4 * WIDTH)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3, table, ln)
    T = int(st[-1])
    mask = _tree_rows(new, st, T, 11)
    mask[::5] = 0
    q = _numbers((T, kv * group, d), BF16, 1, spread=0.3).cuda()
    o, lse = _attend(q, cache, table, ln, st, scale=0.08, tree=mask.cuda())
    _check(o, lse, q, cache, table, ln, st, 0.08, mask=mask)


def test_captured_beside_an_eager_call():
    """A replayed call follows masks and lengths, with its scratch memory apart from that of calls on another stream."""
    from fractaltensor_b200 import ops
    kv, group, d, page, new, lens = 4, 8, 128, 16, [33, 33], [700, 90]
    table, ln, st, pages = _batch(new, lens, page, width=WIDTH)
    cache = _full_cache(pages, kv, page, d, BF16, 3, table, ln)
    T = int(st[-1])
    masks = [_tree_rows(new, st, T, seed) for seed in (3, 4, 5)]
    q = _numbers((T, kv * group, d), BF16, 1, spread=0.3).cuda()
    mask, lens_now = masks[0].cuda(), ln.cuda()
    args = (q, cache, table.cuda(), lens_now, st.cuda())
    lse = torch.empty(T, kv * group, device="cuda")
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.paged_attention(*args, scale=0.08, tree=mask, lse=lse)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        o = ops.paged_attention(*args, scale=0.08, tree=mask, lse=lse)
    eager = (q, cache, table.cuda(), ln.cuda(), st.cuda())
    eager_mask, eager_lse = masks[0].cuda(), torch.empty_like(lse)
    for m, n in ((masks[1], 700), (masks[2], 650)):
        mask.copy_(m)
        lens_now[0] = n
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        with torch.cuda.stream(other):
            e = ops.paged_attention(*eager, scale=0.08, tree=eager_mask, lse=eager_lse)
        torch.cuda.synchronize()
        _check(o, lse, q, cache, table, lens_now.cpu(), st, 0.08, mask=m)
        _check(e, eager_lse, q, cache, table, ln, st, 0.08, mask=masks[0])
    ops.check_status()

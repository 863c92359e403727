"""What the calls on trees of drafts and on eviction refuse before they touch a device, and the oracle's own definitions."""
import ctypes

import pytest
import torch

from oracle import tree


@pytest.fixture(scope="module")
def lib():
    from fractaltensor_b200 import _lib
    return _lib.lib


A = lambda n: ctypes.c_void_p(n << 20)  # never read: the checks come first; far from each other
Z = ctypes.c_void_p(0)


def _attn(lib, **kw):
    a = dict(q=A(1), q_row=256, q_head=64, k=A(2), v=A(3), ke=Z, ve=Z, table=A(4), lens=A(5), starts=A(6), tree=A(7), words=1, o=A(8), lse=A(9), T=1,
             B=1, W=1, pages=1, kv=1, group=4, page=16, d=64, window=0, scale=1.0, dtype=2, scratch=Z, sb=0, ws=A(10), wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_attn_tree_fwd(*a.values())


def _weights(lib, **kw):
    a = dict(q=A(1), q_row=256, q_head=64, k=A(2), ke=Z, lse=A(9), table=A(4), lens=A(5), starts=A(6), weights=A(7), T=1, B=1, W=1, pages=1, kv=1,
             group=4, page=16, d=64, window=0, scale=1.0, dtype=2, scratch=Z, sb=0, ws=A(10), wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_attn_weights(*a.values())


def _keep(lib, **kw):
    a = dict(k=A(2), v=A(3), ke=Z, ve=Z, weights=Z, kept=A(7), ks=1, kh=0, counts=A(8), first=Z, table=A(4), into=Z, B=1, W=1, iw=0, K=1, pages=1,
             kv=1, page=16, d=64, ws=A(10), wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_cache_keep(*a.values())


def _evict(lib, **kw):
    a = dict(k=A(2), v=A(3), ke=Z, ve=Z, weights=A(7), table=A(4), lens=A(5), into=Z, now=A(8), kept=A(9), B=1, W=1, iw=0, keep=4, recent=1, pages=1,
             kv=1, page=16, d=64, ws=A(10), wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_cache_evict(*a.values())


def _verify(lib, **kw):
    a = dict(p=A(1), ps=20, pr=10, tokens=A(2), parents=A(3), u=A(4), out=A(5), path=A(6), counts=A(7), B=1, N=2, V=10, ws=A(10), wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_verify_tree(*a.values())


CACHE = [dict(k=Z), dict(table=Z), dict(B=0), dict(W=0), dict(pages=0), dict(kv=0), dict(page=24), dict(page=8), dict(page=256), dict(d=96)]
ROWS = [dict(q=Z), dict(lens=Z), dict(starts=Z), dict(T=-1), dict(dtype=0), dict(dtype=3), dict(group=0), dict(window=-1), dict(scale=0.0),
        dict(scale=float("nan")), dict(scale=3.4e38), dict(group=70000)]


@pytest.mark.parametrize("kw", CACHE + ROWS + [dict(v=Z), dict(o=Z), dict(ke=A(11)), dict(words=0), dict(words=-1), dict(window=5)])
def test_attention_arguments(lib, kw):
    assert _attn(lib, **kw) == 1


@pytest.mark.parametrize("kw", CACHE + ROWS + [dict(lse=Z), dict(weights=Z)])
def test_weights_arguments(lib, kw):
    assert _weights(lib, **kw) == 1


@pytest.mark.parametrize("kw", CACHE + [dict(v=Z), dict(kept=Z), dict(counts=Z), dict(K=-1), dict(into=A(12), iw=0), dict(ke=A(11))])
def test_keep_arguments(lib, kw):
    assert _keep(lib, **kw) == 1


@pytest.mark.parametrize("kw", CACHE + [dict(v=Z), dict(weights=Z), dict(lens=Z), dict(now=Z), dict(kept=Z), dict(keep=0), dict(keep=-1),
                                        dict(recent=-1), dict(recent=5), dict(into=A(12), iw=0), dict(ve=A(11))])
def test_evict_arguments(lib, kw):
    assert _evict(lib, **kw) == 1


def test_most_positions(lib):
    most = 1 << 30
    assert _keep(lib, K=most + 1, ks=most + 1) == 1
    assert _evict(lib, keep=most + 1) == _evict(lib, keep=(1 << 31) - 1) == 1
    assert _evict(lib, W=most // 16 + 1) == 1


@pytest.mark.parametrize("kw", [dict(p=Z), dict(tokens=Z), dict(parents=Z), dict(u=Z), dict(out=Z), dict(path=Z), dict(counts=Z), dict(B=-1), dict(N=0),
                                dict(N=1025), dict(V=0), dict(V=(1 << 30) + 1)])
def test_verify_arguments(lib, kw):
    assert _verify(lib, **kw) == 1


def test_mask_arguments(lib):
    for a in ((Z, A(2), 1, 1), (A(1), Z, 1, 1), (A(1), A(2), -1, 1), (A(1), A(2), 1, -1), (A(1), A(2), 1 << 20, 1 << 20), (A(1), A(1), 2, 3)):
        assert lib.ftb_tree_mask(*a, Z) == 1, a
    assert lib.ftb_tree_mask(Z, Z, 0, 5, Z) == lib.ftb_tree_mask(Z, Z, 5, 0, Z) == 0


def test_alignment_and_workspace(lib):
    odd, odder = ctypes.c_void_p((13 << 20) + 8), ctypes.c_void_p((13 << 20) + 2)
    for kw in (dict(q=odd), dict(k=odd), dict(o=odd), dict(lse=odder), dict(q_row=4)):
        assert _attn(lib, **kw) == 2, kw
    for kw in (dict(q=odd), dict(k=odd), dict(ke=odd), dict(lse=odder), dict(weights=odder), dict(q_head=7)):
        assert _weights(lib, **kw) == 2, kw
    for call in (_keep, _evict):
        assert call(lib, k=odd) == call(lib, v=odd) == call(lib, ke=odd, ve=A(11)) == 2
    assert _evict(lib, weights=odder) == 2
    for call in (_attn, _weights, _keep, _evict, _verify):
        assert call(lib, ws=Z) == call(lib, wb=1) == 3
    # no rows: nothing to do, and nothing is asked of a device
    assert _attn(lib, T=0) == _weights(lib, T=0) == _keep(lib, K=0) == _verify(lib, B=0) == 0


def test_results_over_what_is_read(lib):
    for kw in (dict(lse=A(1)), dict(lse=A(2)), dict(lse=A(3)), dict(lse=A(7)), dict(lse=A(8)), dict(o=A(7)), dict(o=A(1)),
               dict(lse=A(11), ke=A(11), ve=A(12)), dict(lse=A(12), ke=A(11), ve=A(12))):
        assert _attn(lib, **kw) == 1, kw
    for kw in (dict(weights=A(1)), dict(weights=A(2)), dict(weights=A(9)), dict(weights=A(11), ke=A(11))):
        assert _weights(lib, **kw) == 1, kw
    for out in ("now", "kept"):
        for at in (2, 3, 4, 5, 7):
            assert _evict(lib, **{out: A(at)}) == 1, (out, at)
        assert _evict(lib, into=A(12), iw=1, **{out: A(12)}) == 1
    assert _evict(lib, now=A(9)) == 1
    for out in ("out", "path", "counts"):
        for at in (2, 3, 4) + tuple(i for i in (5, 6, 7) if {"out": 5, "path": 6, "counts": 7}[out] != i):
            assert _verify(lib, **{out: A(at)}) == 1, (out, at)


def test_cpu_tensors_are_refused():
    from fractaltensor_b200 import ops
    cache = tuple(torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16) for _ in range(2))
    i = torch.zeros(1, dtype=torch.int32)
    s = torch.zeros(2, dtype=torch.int32)
    x, w = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 16)
    for call in (lambda: ops.paged_attention(x, cache, i[None], i, s, tree=i[None], lse=torch.zeros(1, 1)), lambda: ops.tree_mask(i[None]),
                 lambda: ops.verify_tree(torch.zeros(1, 1, 4), i[None].long(), i[None], torch.zeros(1, 1)),
                 lambda: ops.paged_cache_keep(cache, i[None], i, i[None]), lambda: ops.paged_cache_evict(cache, w, i[None], i, 1),
                 lambda: ops.paged_attention_weights(x, cache, w, torch.zeros(1, 1), i[None], i, s)):
        with pytest.raises(RuntimeError):
            call()


# ---------------------------------------------------------------------------------------- the oracle
def test_oracle_mask_and_path():
    parents = torch.tensor([[-1, 0, 0, 1, 3, 2, 7, -1]])
    assert [tree.path_to(parents[0].tolist(), i) for i in range(8)] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [0, 2, 5], [6], [7]]
    assert tree.mask(parents)[0, :, 0].tolist() == [1, 3, 5, 11, 27, 37, 64, 128]
    chain = torch.arange(-1, 63)[None]
    assert tree.mask(chain)[0, 31].tolist() == [-1, 0] and tree.mask(chain)[0, 63].tolist() == [-1, -1]


def test_oracle_verification_samples_the_target():
    """Over a fine grid of random numbers for one drafted pair the first token comes as often as the target says."""
    p = torch.tensor([0.5, 0.2, 0.3]).double()
    n = 40
    u = (torch.arange(n).double() + 0.5) / n
    grid = torch.cartesian_prod(u, u, u).float()
    B = len(grid)
    probs = p.float().expand(B, 3, 3)
    out, path, counts = tree.verify(probs, torch.tensor([[0, 1, 2]]).expand(B, 3), torch.tensor([[-1, 0, 0]]).expand(B, 3), grid)
    share = torch.bincount(out[:, 0], minlength=3) / B
    assert float((share - p).abs().max()) < 2.0 / n
    assert set(map(tuple, path[:, :2].tolist())) == {(0, 1), (0, 2), (0, -1)}


def test_oracle_choice():
    w = torch.tensor([3.0, float("nan"), 5.0, 3.0, -1.0, 9.0, 0.0, float("inf")]).reshape(1, 1, 8)
    now, kept = tree.choose(w, torch.tensor([[0]]), [8], 4, 1)
    assert now.tolist() == [4] and kept[0, 0].tolist() == [0, 2, 5, 7]
    assert tree.choose(w, torch.tensor([[0]]), [8], 7, 0)[1][0, 0].tolist() == [0, 2, 3, 4, 5, 6, 7]
    assert tree.choose(w, torch.tensor([[0]]), [2], 4, 1)[1][0, 0].tolist() == [0, 1, -1, -1]

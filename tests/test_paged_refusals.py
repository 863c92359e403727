"""What the entry points of the paged cache refuse before they touch a device, and the oracle's own definitions."""
import ctypes

import pytest
import torch

from oracle import paged


@pytest.fixture(scope="module")
def lib():
    from fractaltensor_b200 import _lib
    return _lib.lib


P = ctypes.c_void_p(16)  # never read: the checks come first
Z = ctypes.c_void_p(0)


def _attn(lib, **kw):
    a = dict(q=P, q_row=256, q_head=64, k=P, v=P, ke=Z, ve=Z, table=P, lens=P, starts=P, o=P, T=1, B=1, W=1, pages=1, kv=1, group=4,
             page=16, d=64, window=0, scale=1.0, dtype=2, scratch=Z, sb=0, ws=P, wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_attn_fwd(*a.values())


def _write(lib, **kw):
    a = dict(k=P, v=P, kr=64, kh=64, vr=64, vh=64, kc=P, vc=P, ke=Z, ve=Z, table=P, lens=P, starts=P, T=1, B=1, W=1, pages=1, kv=1,
             page=16, d=64, dtype=2, ws=P, wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_cache_write(*a.values())


def _read(lib, **kw):
    a = dict(kc=P, vc=P, ke=Z, ve=Z, table=P, lens=P, starts=P, k=P, v=P, T=1, B=1, W=1, pages=1, kv=1, page=16, d=64, dtype=2, ws=P,
             wb=256, stream=Z)
    a.update(kw)
    return lib.ftb_paged_cache_read(*a.values())


COMMON = [dict(table=Z), dict(lens=Z), dict(starts=Z), dict(ke=P), dict(T=-1), dict(B=0), dict(W=0), dict(pages=0), dict(kv=0),
          dict(page=24), dict(page=8), dict(page=256), dict(d=96), dict(dtype=0), dict(dtype=3)]


@pytest.mark.parametrize("kw", COMMON + [dict(q=Z), dict(o=Z), dict(group=0), dict(window=-1), dict(scale=0.0), dict(scale=-1.0),
                                         dict(scale=float("nan")), dict(scale=float("inf")), dict(group=70000)])
def test_attention_arguments(lib, kw):
    assert _attn(lib, **kw) == 1


@pytest.mark.parametrize("kw", COMMON + [dict(k=Z), dict(v=Z), dict(kc=Z), dict(vc=Z)])
def test_write_arguments(lib, kw):
    assert _write(lib, **kw) == 1


@pytest.mark.parametrize("kw", COMMON + [dict(k=Z), dict(v=Z), dict(kc=Z), dict(vc=Z)])
def test_read_arguments(lib, kw):
    assert _read(lib, **kw) == 1


def test_alignment_and_workspace(lib):
    odd = ctypes.c_void_p(24)
    for kw in (dict(q=odd), dict(k=odd), dict(v=odd), dict(o=odd), dict(q_row=4), dict(q_head=63)):
        assert _attn(lib, **kw) == 2, kw
    assert _attn(lib, o=P) == 1  # over the queries
    for call in (_attn, _write, _read):  # exponents are fetched 16 at a time
        assert call(lib, ke=odd, ve=P) == call(lib, ke=P, ve=ctypes.c_void_p(17)) == 2
    for kw in (dict(k=odd), dict(vc=odd), dict(kr=4), dict(vh=1)):
        assert _write(lib, **kw) == 2, kw
    for kw in (dict(k=odd), dict(vc=odd)):
        assert _read(lib, **kw) == 2, kw
    assert _attn(lib, ws=Z) == _write(lib, ws=Z) == _read(lib, ws=Z) == 3
    assert _attn(lib, wb=1) == _write(lib, wb=1) == _read(lib, wb=1) == 3
    # no rows: nothing to do, and nothing is asked of a device
    assert _attn(lib, T=0) == _write(lib, T=0) == _read(lib, T=0) == 0


def test_verify_arguments(lib):
    def call(**kw):
        a = dict(p=P, ps=20, pr=10, q=Z, qs=0, qr=0, drafts=P, u=P, counts=Z, tokens=P, out=P, B=1, K=1, V=10, ws=P, wb=256, stream=Z)
        a.update(kw)
        return lib.ftb_verify_drafts(*a.values())
    for kw in (dict(p=Z), dict(drafts=Z), dict(u=Z), dict(tokens=Z), dict(out=Z), dict(B=-1), dict(K=-1), dict(V=0)):
        assert call(**kw) == 1, kw
    assert call(ws=Z) == 3
    assert call(B=0) == 0


def test_cpu_tensors_are_refused():
    from fractaltensor_b200 import ops
    cache = tuple(torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16) for _ in range(2))
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.paged_attention(x, cache, i[None], i[:1], i), lambda: ops.paged_cache_write(cache, x, x, i[None], i[:1], i),
                 lambda: ops.paged_cache_read(cache, i[None], i[:1], i, 1),
                 lambda: ops.verify_drafts(torch.zeros(1, 1, 4), torch.zeros(1, 0, dtype=torch.int64), torch.zeros(1, 1))):
        with pytest.raises(RuntimeError):
            call()


def test_oracle_codes_are_the_nearest():
    """Every e4m3 code is its own; numbers between two go to the nearer one, ties to the even one; the scale is the smallest."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 0x7F) != 0x7F]
    x = codes.view(torch.float8_e4m3fn).double()
    x = torch.cat([x, torch.tensor([448.0, -448.0])])
    got, e = paged.quantise(x)
    assert int(e) == 127 and torch.equal(got[:-2], codes)
    pos = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (pos[1:] + pos[:-1]) / 2
    got, _ = paged.quantise(torch.cat([mid, pos[-1:]]))
    assert torch.equal(got[:-1].int(), torch.arange(126) + torch.arange(126) % 2)
    for m, want in ((448.0, 127), (448.1, 128), (224.0, 126), (224.1, 127), (0.0, 1), (2.0 ** -140, 1), (3.0e38, 127 + 120)):
        assert int(paged.quantise(torch.tensor([m, 0.0]))[1]) == want


def test_oracle_verification_takes_by_the_ratio():
    p, q = torch.tensor([[[0.2, 0.8], [0.5, 0.5]]]), torch.tensor([[[0.4, 0.6]]])
    for u, want in ((0.49, [0, 0]), (0.51, [1, -1])):
        got, n = paged.verify(p, torch.tensor([[0]]), torch.tensor([[u, 0.3]]), q)
        assert got.tolist() == [want] and n.tolist() == [2 if u < 0.5 else 1]


@pytest.mark.parametrize("scale", [2.5e38, 3.4e38])
def test_a_scale_that_is_infinite_in_log2_is_refused(lib, scale):
    assert _attn(lib, o=ctypes.c_void_p(1 << 20), scale=scale) == 1

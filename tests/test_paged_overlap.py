"""Results over what a call reads are refused before a device is touched; neighbours in one buffer are not."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from fractaltensor_b200 import _lib
    return _lib.lib


A = lambda n: ctypes.c_void_p(n)
FAR = 1 << 40


def _attn(lib, q, o, T, heads, d, q_row, q_head=None, **kw):
    a = dict(q=A(q), q_row=q_row, q_head=d if q_head is None else q_head, k=A(FAR), v=A(2 * FAR), ke=A(0), ve=A(0), table=A(16), lens=A(16), starts=A(16),
             o=A(o), T=T, B=1, W=1, pages=4, kv=heads, group=1, page=16, d=d, window=0, scale=1.0, dtype=2, scratch=A(0), sb=0, ws=A(16), wb=256, stream=A(0))
    a.update(kw)
    return lib.ftb_paged_attn_fwd(*a.values())


Q = 1 << 20
ROWS = 4 * 64 * 2  # bytes of a row of 4 heads of 64


@pytest.mark.parametrize("T,q_row,at", [
    (1, 256, 0), (1, 256, 16), (1, 256, -16), (3, 256, 2 * ROWS + 16), (3, 256, -3 * ROWS + 16), (3, 768, 3 * ROWS - 16), (5, 4096, 4 * 4096 * 2 + 16),
    (2, 0, 128), (3, -256, -2 * ROWS + 16), (3, -256, -5 * ROWS + 16),
])
def test_results_over_queries_are_refused(lib, T, q_row, at):
    assert _attn(lib, Q, Q + at, T, 4, 64, q_row) == 1


@pytest.mark.parametrize("T,q_row,at", [
    (1, 256, ROWS), (1, 256, -ROWS), (3, 256, 3 * ROWS), (3, 256, -3 * ROWS), (2, 4096, ROWS), (2, 4096, 4096 * 2 - 2 * ROWS), (2, 0, ROWS), (3, -256, ROWS),
    (3, -256, -5 * ROWS),
])
def test_neighbours_are_not(lib, T, q_row, at):
    assert _attn(lib, Q, Q + at, T, 4, 64, q_row) != 1


def test_results_over_the_cache_are_refused(lib):
    size = 4 * 2 * 16 * 64 * 2
    for cache in ("k", "v"):
        for at, want in ((0, True), (size - 16, True), (-256 + 16, True), (size, False), (-256, False)):
            assert (_attn(lib, Q, 4 * FAR + at, 1, 2, 64, 128, **{cache: A(4 * FAR)}) == 1) == want, (cache, at)
    for at, want in ((0, True), (4 * 2 * 16, False)):
        assert (_attn(lib, Q, 4 * FAR + at, 1, 2, 64, 128, ke=A(4 * FAR), ve=A(5 * FAR)) == 1) == want


def test_what_is_read_out_does_not_overlap(lib):
    def read(k, v, **kw):
        a = dict(kc=A(FAR), vc=A(2 * FAR), ke=A(0), ve=A(0), table=A(16), lens=A(16), starts=A(16), k=A(k), v=A(v), T=3, B=1, W=1, pages=4, kv=2, page=16,
                 d=64, dtype=2, ws=A(16), wb=256, stream=A(0))
        a.update(kw)
        return lib.ftb_paged_cache_read(*a.values())
    size = 3 * 2 * 64 * 2
    assert read(Q, Q) == read(Q, Q + size - 16) == read(Q + size - 16, Q) == 1
    assert read(Q, Q + size) != 1 and read(Q + size, Q) != 1
    assert read(FAR, Q) == read(Q, 2 * FAR + 16) == read(2 * FAR, Q) == 1
    e = dict(ke=A(4 * FAR), ve=A(5 * FAR))
    assert read(4 * FAR, Q, **e) == read(Q, 5 * FAR, **e) == 1
    assert read(Q, Q + size, dtype=0, **e) == 1 and read(Q, Q + 2 * size, dtype=0, **e) != 1

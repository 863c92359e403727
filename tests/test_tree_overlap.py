"""What the calls on trees of drafts and on a cache's rows refuse by address, before they touch a device.  (Only refusals: an address that is
not refused would be read on a machine with a device.)"""
import ctypes

from test_tree_refusals import _attn, _keep, _verify, lib  # noqa: F401


def test_verification_over_its_probabilities(lib):
    """Sequences read their rows while others' results are written: no result has a part of them."""
    P, V, row, seq, B, N = 1 << 30, 100, 128, 1000, 3, 2
    size = 4 * ((B - 1) * seq + (N - 1) * row + V)
    call = lambda out, at, **kw: _verify(lib, **{"p": ctypes.c_void_p(P), "ps": seq, "pr": row, "B": B, "N": N, "V": V, out: ctypes.c_void_p(at), **kw})
    for out, n in (("out", 8 * B * N), ("path", 4 * B * N), ("counts", 4 * B)):
        for at in (P, P + 4 * row, P + 4 * V, P + 4 * (seq + V) - 8, P + size - 8, P - n + 8):
            assert call(out, at) == 1, (out, at)
        # rows that all sequences share, rows the other way round
        assert call(out, P + 4 * row, ps=0) == 1 and call(out, P - 4 * seq, ps=-seq) == 1
    # the longest rows
    assert _verify(lib, p=ctypes.c_void_p(1 << 44), V=1 << 30, ps=2 << 30, pr=1 << 30, counts=ctypes.c_void_p((1 << 44) + (8 << 30) - 8)) == 1


def test_words_that_begin_anywhere(lib):
    """Masks and weights are read four bytes at a time."""
    odd = ctypes.c_void_p((13 << 20) + 2)
    assert _attn(lib, tree=odd) == 2 and _keep(lib, weights=odd) == 2

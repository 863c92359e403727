"""Calls of the paged operators that differ in what surrounds them: devices, copied and shared pages, repeated indexes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def test_scratch_is_sized_for_the_tensors_device(monkeypatch):
    """The scratch memory's size follows from a device's SMs: it is asked for where the tensors' device is the current one."""
    from fractaltensor_b200 import _lib, ops
    inside, asked = [], []

    class On(ops._on):
        __slots__ = ()

        def __enter__(self):
            inside.append(self.device)
            return super().__enter__()

        def __exit__(self, *e):
            inside.pop()
            return super().__exit__(*e)

    class Lib:
        def __getattr__(self, name):
            f = getattr(_lib.lib, name)
            if not name.startswith("ftb_paged"):
                return f

            def call(*args):
                asked.append((name, list(inside)))
                return f(*args)
            return call

    monkeypatch.setattr(ops, "_on", On)
    monkeypatch.setattr(ops, "lib", Lib())
    monkeypatch.setattr(ops, "host", _lib._NoHost)
    cache = ops.paged_cache(4, 2, 16, 64, BF16)
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    lens, starts = torch.ones(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    ops.paged_attention(torch.zeros(1, 4, 64, dtype=BF16, device="cuda"), cache, table, lens, starts)
    ops.check_status()
    assert {n for n, _ in asked} == {"ftb_paged_attn_scratch_bytes", "ftb_paged_attn_fwd"}
    assert all(where == [cache[0].device.index] for _, where in asked), asked


def _run(q, cache, table, lens, starts, **kw):
    from fractaltensor_b200 import ops
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    o = ops.paged_attention(q, cache, i(table), i(lens), i(starts), **kw)
    ops.check_status()
    return o


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_sequences_share(dtype, new):
    """A prefix whose pages are in two tables, then a page of its own each, one of them copied out of the shared one within the cache."""
    from fractaltensor_b200 import ops
    kv, group, d, page, n = 2, 4, 64, 16, 45  # two whole pages and 13 keys of a third
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = ops.paged_cache(6, kv, page, d, dtype)
    k, v = (torch.randn(n, kv, d, generator=g, device="cuda").to(BF16) for _ in range(2))
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    ops.paged_cache_write(cache, k, v, i([[4, 1, 3]]), i([n]), i([0, n]))
    if dtype == BF16:  # rows of page 3 into page 0, read where they lie
        rows = [c[3].transpose(0, 1)[:13] for c in cache]
        ops.paged_cache_write(cache, *rows, i([[4, 1, 0]]), i([n]), i([0, 13]))
    else:
        for c in cache:
            c.view(torch.uint8)[0] = c.view(torch.uint8)[3]
    q = torch.randn(2 * new, kv * group, d, generator=g, device="cuda").to(BF16)
    one = _run(q[:new], cache, [[4, 1, 3]], [n], [0, new], scale=0.2)
    two = _run(q[new:], cache, [[4, 1, 3]], [n], [0, new], scale=0.2)
    both = _run(q, cache, [[4, 1, 3], [4, 1, 0]], [n, n], [0, new, 2 * new], scale=0.2)
    for a, b in ((both[:new], one), (both[new:], two)):  # (other cuts of the work: the same to the rounding of weights and results)
        assert float((a.float() - b.float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())
    for b in range(2):
        got = ops.paged_cache_read(cache, i([[4, 1, 3], [4, 1, 0]][b:b + 1]), i([n]), i([0, n]), n, dtype=BF16)
        want = ops.paged_cache_read(cache, i([[4, 1, 3]]), i([n]), i([0, n]), n, dtype=BF16)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ops.check_status()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("T,starts", [(5, [0, 0, 0]), (300, [0, 0, 0]), (7, [7, 7, 7]), (300, [300, 300, 300])])
def test_rows_without_a_sequence_stay(dtype, T, starts):
    from fractaltensor_b200 import ops
    kv, group, d, page = 2, 4, 64, 16
    cache = ops.paged_cache(4, kv, page, d, dtype)
    before = [c.clone() for c in cache]
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    x = torch.ones(T, kv, d, dtype=BF16, device="cuda")
    for _ in range(3):  # (scratch memory holds whatever was there)
        ops.paged_cache_write(cache, x, x, i([[0, 1], [2, 3]]), i([20, 9]), i(starts))
        out = torch.full((T, kv * group, d), 3.0, dtype=BF16, device="cuda")
        junk = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
        del junk
        _run(torch.ones_like(out), cache, [[0, 1], [2, 3]], [20, 9], starts, out=out)
        assert bool((out == 3.0).all())
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, cache))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("T", [1, 30])
def test_queries_that_are_one_row_for_all_heads(dtype, T):
    from fractaltensor_b200 import ops
    kv, group, d, page, n = 2, 4, 64, 16, 45
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = ops.paged_cache(3, kv, page, d, dtype)
    k, v = (torch.randn(n, kv, d, generator=g, device="cuda").to(BF16) for _ in range(2))
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    ops.paged_cache_write(cache, k, v, i([[2, 0, 1]]), i([n]), i([0, n]))
    q = torch.randn(1, 1, d, generator=g, device="cuda").to(BF16)
    want = _run(q.expand(T, kv * group, d).contiguous(), cache, [[2, 0, 1]], [n], [0, T])
    assert torch.equal(_run(q.expand(T, kv * group, d), cache, [[2, 0, 1]], [n], [0, T]), want)

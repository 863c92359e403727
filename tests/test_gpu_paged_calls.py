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

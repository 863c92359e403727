"""What the attention over a paged cache asks for beside its results."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,kv,group,d", [(2048, 8, 4, 128), (100, 4, 4, 64), (700, 1, 8, 128)])
def test_a_prompt_asks_for_its_tiles_alone(T, kv, group, d):
    """One sequence of many rows: a flag a row, two places of 128 or 256 rows for each CTA, and what is to be joined (less than 128 bytes each)."""
    from fractaltensor_b200._lib import lib
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    R = 256 if T * group > 128 else 128
    n = lib.ftb_paged_attn_scratch_bytes(T, 1, kv, group, d)
    least = 4 * T * kv * group + 2 * sms * R * (d + 2) * 4
    assert least <= n <= least + 128 * sms + 512

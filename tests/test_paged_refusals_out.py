"""What norm_rope_paged refuses as `out`, before anything reaches a device."""
import pytest
import torch

from hackthenorth_amd.kernels.paged import norm_rope_paged

BF16 = torch.bfloat16


@pytest.mark.parametrize("out,message", [
    (torch.zeros(3, 4, 128), "out must"), (torch.zeros(2, 4, 128, dtype=BF16), "out must"),
    (torch.zeros(3, 2, 128, dtype=BF16), "out must"),
    (torch.zeros(3, 8, 128, dtype=BF16)[:, ::2], "out must"),
    (torch.zeros(3, 4, 128, dtype=BF16), "GPU only")])
def test_append_refuses_out(out, message):
    q, kv = torch.zeros(3, 4, 128, dtype=BF16), torch.zeros(3, 2, 128, dtype=BF16)
    pool, angles = torch.zeros(6, 2, 16, 128, dtype=BF16), torch.zeros(9, 128, dtype=BF16)
    with pytest.raises(ValueError, match=message):
        norm_rope_paged(q, kv, kv, None, None, angles, angles, pool, pool.clone(),
                        torch.zeros(2, 3, dtype=torch.int32), torch.tensor([0, 1, 3]),
                        torch.tensor([5, 6]), out=out)

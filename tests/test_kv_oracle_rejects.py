"""The paged-cache oracle turns down outputs that are wrong (CPU; the mistakes are planted in what it is given)."""
import pytest
import torch

from oracle import kv_oracle as K


@pytest.mark.parametrize("dtype,most", [(torch.bfloat16, 2.0 ** -10), (torch.float16, 2.0 ** -8)])
def test_large_values_behind_vanishing_weights_get_no_slack(dtype, most):
    # one key of value 1, 1000 of 60000 with weights e^-200: float16 may add 1000 * 2^-35 * 60000 = 2^-9, bf16 nothing.
    # What is left comes from scores of 200, 2 * (8 + 3) * 200 * 2^-24 < 2^-11, and the sums, 2130 * 2^-24 < 2^-12.
    n, hd, page = 1001, 8, 64
    k, v = torch.zeros(16, 1, page, hd), torch.full((16, 1, page, hd), 60000.0)
    k[..., 0] = -200.0
    k[0, 0, 0, 0], v[0, 0, 0] = 0.0, 1.0
    q = torch.zeros(1, 1, hd)
    q[..., 0] = 1.0
    y, slack = K.attn(q.to(dtype), k.to(dtype), v.to(dtype), torch.arange(16, dtype=torch.int32)[None],
                      torch.tensor([n], dtype=torch.int32), 1.0)
    assert bool((y == 1.0).all()) and bool((slack < most).all())
    with pytest.raises(AssertionError):
        K.assert_rounds_to((y * (1 + 2.0 ** -6)).to(dtype), y, slack)

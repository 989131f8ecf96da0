"""The paged-cache oracle turns down outputs that are wrong (CPU; the mistakes are planted in what it is given)."""
import pytest
import torch

import kv_markers as M
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step,lost", [(1, 32), (7, 21)])
def test_a_lost_or_doubled_tile_of_a_long_row_shows(step, lost, dtype):
    # the markers of kv_markers.py on 70000 positions: 32 of them lost or doubled, or three of those that count
    n, hd = 70000, 64
    y = M.result(n, hd, step)
    K.assert_rounds_to(K.rounded(y, dtype).to(dtype), y, y * M.SLACK)
    for at in (0, 34000, n - lost):
        j = torch.arange(n)
        for used in (torch.cat([j[:at], j[at + lost:]]), torch.cat([j, j[at:at + lost]])):
            bad = K.rounded(M.result(n, hd, step, used=used), dtype).to(dtype)
            with pytest.raises(AssertionError):
                K.assert_rounds_to(bad, y, y * M.SLACK)

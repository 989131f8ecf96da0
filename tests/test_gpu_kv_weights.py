"""attn_step: what the softmax weights count for.  Scores that are exact in float32 (one key element against one query
element), so that hardly anything but the weights' own precision is left between a kernel and the formula."""
import pytest
import torch

from oracle import kv_oracle as K
from vortex_amd import attn_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
BF, F16 = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def one_hot(B, H, hd, dtype):
    """Queries whose score with a key is the key's element 0."""
    q = torch.zeros(B, H, hd)
    q[..., 0] = 1.0
    return q.to(dtype).to(DEV)


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (BF, True), (F16, False), (F16, True)])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
def test_weights_keep_all_their_bits(override, hd, dtype, fp8, form):
    """Two keys a sequence: score 0 with value 0, score s in (-1, 0) with value v in 1..2; y = v w / (1 + w), w = e^s.

    The kernel may be off by, relative to y, in units of 2^-24: the factor's two roundings and the product's on |s| < 1: 3;
    the subtraction from a reference that lies at most 1 (float16: 12) beyond the largest score: 2 (13), counted with
    ln 2 < 1; the power of two: 2; three terms of the weight added up: 3; the sum of the weights: 1; the division, the
    product with it and the join's factor: 3.  In all 14 (25).  Weights of 16 bits are off by up to 2^7 such units."""
    override(attn_short=form)
    B, H, g = 128, 8, gen(hd)
    t = FP8 if fp8 else dtype
    k, v = torch.randn(B, H, 16, hd, generator=g), torch.zeros(B, H, 16, hd)
    k[:, :, 0, 0], k[:, :, 1, 0] = 0.0, -torch.rand(B, H, generator=g).clamp(2.0 ** -6, 1 - 2.0 ** -6)
    v[:, :, 1] = 1 + torch.rand(B, H, hd, generator=g)
    k, v = k.to(t), v.to(t)
    table = torch.randperm(B, generator=g).to(torch.int32)[:, None]
    kd, vd = k.double()[table[:, 0].long()], v.double()[table[:, 0].long()]
    w = torch.exp(kd[:, :, 1, :1])
    y = vd[:, :, 1] * w / (1 + w)
    lens = torch.full((B,), 2, dtype=torch.int32)
    got = attn_step(one_hot(B, H, hd, dtype), k.to(DEV), v.to(DEV), table.to(DEV), lens.to(DEV), scale=1.0)
    K.assert_rounds_to(got, y, y * (25 if dtype == F16 else 14) * 2.0 ** -24)

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


def flat_row(n, hd, dtype, fp8, low, first, rest, kv_heads=1, page=64):
    """One sequence of n keys on which one_hot queries score 0 at position n // 3 (value `first`) and `low` everywhere
    else (value `rest`)."""
    P, t = -(-n // page), FP8 if fp8 else dtype
    k, v = torch.zeros(P, kv_heads, page, hd), torch.full((P, kv_heads, page, hd), float(rest))
    k[..., 0] = low
    at = n // 3
    k[at // page, :, at % page], v[at // page, :, at % page] = 0.0, first
    return k.to(t).to(DEV), v.to(t).to(DEV), torch.arange(P, dtype=torch.int32)[None].to(DEV)


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("dtype,fp8", [(F16, False), (F16, True), (BF, False)])
@pytest.mark.parametrize("low", [float("-inf"), -200.0, -60.0, -30.0, -25.25, -20.0, -12.0])
def test_a_long_row_behind_one_large_weight(override, low, dtype, fp8, form):
    """131072 values of 60000 (448 in 8 bits, times a scale) behind weights that vanish, that are small, and that
    together outweigh the one key of value 1: y = (1 + (n - 1) w 60000) / (1 + (n - 1) w), all terms of one sign.

    Slack: a run is at most the row, 512 tiles of 3 products whose sums lose 2^-24 or so each time, all in one
    direction at worst: 2^-13 with the weights' sum counted beside it; twice that is 2^-12.  What float16 keeps of the
    127 weights beside the large one, 2^-36 each, adds 127 * 2^-36 * 60000 = 2^-13.  2^-11 for both."""
    override(attn_short=form)
    n, hd = 131072, 32
    if fp8 and low == float("-inf"):
        low = -448.0
    big, vs = (448.0, torch.full((1,), 128.0, device=DEV)) if fp8 else (60000.0, None)
    k, v, table = flat_row(n, hd, dtype, fp8, low, 1.0 / 128 if fp8 else 1.0, big)
    low, big = float(k[0, 0, 0, 0]), float(v[0, 0, 0, 0]) * (128.0 if fp8 else 1.0)
    w = (n - 1) * torch.exp(torch.tensor(low, dtype=torch.float64))
    y = ((1 + w * big) / (1 + w)).expand(1, 2, hd)
    got = attn_step(one_hot(1, 2, hd, dtype), k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0, v_scale=vs)
    K.assert_rounds_to(got, y, y * 2.0 ** -11)


def test_a_position_without_weight_adds_nothing():
    # bf16, the largest values there are: behind a score of -inf, and behind one whose weight underflows
    for low in (float("-inf"), -200.0):
        k, v, table = flat_row(100, 64, BF, False, 0.0, 3e38, 1.0, page=16)
        k[33 // 16, 0, 33 % 16, 0] = low
        got = attn_step(one_hot(1, 2, 64, BF), k, v, table, torch.tensor([100], dtype=torch.int32, device=DEV), scale=1.0)
        assert torch.equal(got, torch.ones_like(got)), (low, got.flatten()[:4])


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("low", [0.0, -0.25, -9.0, -30.0, -60.0])
def test_infinite_values_stay_where_they_are(override, low, dtype, form):
    """An infinite value behind a weight of any size above 0 makes its own element infinite, opposite ones NaN, and leaves
    the other elements alone; behind a weight of 0 it is 0 * inf, as in the formula."""
    override(attn_short=form)
    n, hd, page = 300, 64, 16
    k, v, table = flat_row(n, hd, dtype, False, 0.0, 1.0, 1.0, page=page)
    k[5, 0, 3, 0] = low
    v[5, 0, 3, 7], v[5, 0, 3, 9], v[0, 0, 1, 9] = float("inf"), float("-inf"), float("inf")
    v[2, 0, 2, 11] = float("-inf")
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    got = attn_step(one_hot(1, 3, hd, dtype), k, v, table, lens, scale=1.0)
    assert bool((got[..., 7] == float("inf")).all()) and bool((got[..., 11] == float("-inf")).all()) and bool(got[..., 9].isnan().all())
    rest = [d for d in range(hd) if d not in (7, 9, 11)]
    # the weights' sum beside the values': ones, so that only the last rounding and the sums' 2^-20 are left
    K.assert_rounds_to(got[..., rest], torch.ones(1, 3, len(rest), dtype=torch.float64), torch.full((1, 3, len(rest)), 2.0 ** -18))
    k[5, 0, 3, 0] = float("-inf")
    got = attn_step(one_hot(1, 3, hd, dtype), k, v, table, lens, scale=1.0)
    assert bool(got[..., 7].isnan().all()) and bool(got[..., rest].isfinite().all())


def test_scores_that_rise_and_fall_over_many_tiles(override):
    # float16: the reference follows the scores in both directions; every tile counts what it weighs
    n, hd, page = 20000, 32, 64
    for form in (0, 1):
        override(attn_short=form)
        for period in (64, 128, 300, 4000):
            k, v, table = flat_row(n, hd, F16, False, 0.0, 1.0, 1.0, page=page)
            j = torch.arange(k.shape[0] * page)
            s = (-20 + 20 * torch.cos(2 * torch.pi * j / period)).to(F16)
            k[..., 0] = s.view(-1, 1, page).to(DEV)
            x = (1 + torch.rand(j.numel(), hd, generator=gen(period)) * 2.0 ** (j[:, None] % 8)).to(F16)
            v[:, 0] = x.view(-1, page, hd).to(DEV)
            w = torch.exp(s[:n].double())
            y = (w @ x[:n].double()) / w.sum()
            got = attn_step(one_hot(1, 1, hd, F16), k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0)
            # scores to 40: 3 * 40 + 40 + 12 units of 2^-24, twice; 160 tiles of a run in each of two sums, 3 products each
            K.assert_rounds_to(got, y.expand(1, 1, hd), y.expand(1, 1, hd) * (344 + 1000) * 2.0 ** -24, f"period {period} form {form}")

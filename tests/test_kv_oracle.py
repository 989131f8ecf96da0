"""Pins of the paged-cache oracle (CPU)."""
import math

import pytest
import torch

from oracle import kv_oracle as K


def test_rounded_is_the_types_own_rounding():
    y = torch.randn(20000, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 3
    y = torch.cat([y, y * 1e-3, torch.tensor([0.0, 448.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9])]).float().double()
    for t in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
        assert torch.equal(K.rounded(y, t), y.float().to(t).double())


def test_attention_hand_value():
    # two keys, scores 0 and ln 3: weights 1/4 and 3/4
    k = torch.zeros(1, 1, 16, 8)
    v = torch.zeros(1, 1, 16, 8)
    k[0, 0, 1, 0], v[0, 0, 0, 2], v[0, 0, 1, 2] = math.log(3), 4.0, 8.0
    q = torch.zeros(1, 1, 8)
    q[0, 0, 0] = 1.0
    out, _ = K.attn(q, k, v, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([2], dtype=torch.int32), 1.0)
    assert abs(float(out[0, 0, 2]) - 7.0) < 1e-6
    # a table that names no page leaves nothing
    out, _ = K.attn(q, k, v, torch.full((1, 1), 9, dtype=torch.int32), torch.tensor([2], dtype=torch.int32), 1.0)
    assert float(out.abs().max()) == 0.0


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_matches_the_stack_oracle_and_keeps_products(interleaved):
    from oracle import stack_oracle as S
    from vortex_amd import rotary_turns
    x = torch.randn(5, 3, 32, generator=torch.Generator().manual_seed(2))
    pos = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32)
    y, _ = K.rotate(x, pos, rotary_turns(32, 10000.0), interleaved)
    if not interleaved:
        assert torch.allclose(y, S.rotary(x[None], 10000.0)[0].double(), atol=1e-5)
    # a rotation keeps the product of two vectors that turn by the same distance
    a, _ = K.rotate(x, pos + 7, rotary_turns(32, 10000.0), interleaved)
    b, _ = K.rotate(x, pos + 1007, rotary_turns(32, 10000.0), interleaved)
    assert torch.allclose((a[0] * a[3]).sum(), (b[0] * b[3]).sum(), atol=1e-4)


def test_turns_of_the_scalings():
    from vortex_amd import rotary_turns
    d, base, f = 64, 10000.0, 8.0
    plain = rotary_turns(d, base)
    assert plain.dtype == torch.float64 and abs(float(plain[0]) - 1 / (2 * math.pi)) < 1e-15
    assert torch.allclose(rotary_turns(d, base, factor=f), plain / f, rtol=1e-14)
    stretched = rotary_turns(d, base, factor=f, scaling="base")
    assert abs(float(stretched[0] / plain[0]) - 1) < 1e-12 and abs(float(stretched[-1] * f / plain[-1]) - 1) < 1e-12
    parts = rotary_turns(d, base, factor=f, scaling="parts", original_length=2048)
    seen = plain * 2048
    assert torch.equal(parts[seen >= 32], plain[seen >= 32])
    assert torch.allclose(parts[seen <= 1], plain[seen <= 1] / f, rtol=1e-14)
    mid = (seen > 1) & (seen < 32)
    assert bool(mid.any()) and bool(((parts[mid] < plain[mid]) & (parts[mid] > plain[mid] / f)).all())
    for bad in (dict(scaling="x"), dict(scaling="parts"), dict(factor=0.0)):
        with pytest.raises(ValueError):
            rotary_turns(d, base, **bad)
    with pytest.raises(ValueError):
        rotary_turns(63)

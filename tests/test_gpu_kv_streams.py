"""The forms of rotary_append and kv_copy_pages for calls beyond the last-level cache, and a token step's values."""
import pytest
import torch

from oracle import kv_oracle as K
from vortex_amd import attn_step, kv_copy_pages, rotary_append, rotary_turns

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
BF, F16 = torch.bfloat16, torch.float16


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (F16, False), (BF, True), (F16, True)])
@pytest.mark.parametrize("heads,kv_heads,hd,rd", [(32, 32, 128, 128), (20, 4, 80, 48), (48, 1, 256, 256), (8, 8, 64, 16)])
def test_large_appends_equal_small_ones(heads, kv_heads, hd, rd, dtype, fp8, interleaved):
    """A call whose rows of q and k, read and written, are more than 128 MiB is the same bit for bit as the same rows in
    calls of 50 tokens, which the oracle checks elsewhere; in part of the call against the oracle here as well."""
    page = 64
    T = (132 << 20) // ((heads + kv_heads) * hd * 4) + 3
    assert T * (heads + kv_heads) * hd * 4 > 128 << 20
    g = torch.Generator(device=DEV).manual_seed(hd)
    q, k, v = torch.randn(T, heads + 2 * kv_heads, hd, device=DEV, generator=g).to(dtype).split([heads, kv_heads, kv_heads], dim=1)
    P = -(-T // page) + 2
    table = torch.randperm(P, generator=torch.Generator().manual_seed(1))[:P - 2].to(torch.int32)[None].to(DEV)
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    pos[5::97] = -1
    seq = torch.zeros(T, dtype=torch.int32, device=DEV)
    ks, vs = ((0.01 + 0.02 * torch.rand(2, kv_heads, device=DEV, generator=g)).unbind(0)) if fp8 else (None, None)
    turns = rotary_turns(rd, device=DEV)

    def run(parts):
        kp, vp = (torch.zeros(P, kv_heads, page, hd, device=DEV).to(FP8 if fp8 else dtype) for _ in range(2))
        qo, ko = torch.full((T, heads, hd), 5.0, dtype=dtype, device=DEV), torch.full((T, kv_heads, hd), 5.0, dtype=dtype, device=DEV)
        for a, b in parts:
            rotary_append(q[a:b], k[a:b], v[a:b], pos[a:b], turns, kp, vp, table, seq=seq[a:b], interleaved=interleaved, k_scale=ks,
                          v_scale=vs, q_out=qo[a:b], k_out=ko[a:b])
        return qo, ko, kp, vp

    large, small = run([(0, T)]), run([(a, min(a + 50, T)) for a in range(0, T, 50)])
    for x, y in zip(large, small):
        assert torch.equal(bits(x), bits(y))
    for part in (slice(0, 20), slice(T - 20, T)):
        real = (pos[part] >= 0).cpu()
        for got, x in ((large[0], q), (large[1], k)):
            y, slack = K.rotate(x[part], pos[part], turns, interleaved)
            K.assert_rounds_to(got[part].cpu()[real], y[real], slack[real])
            assert bool((got[part].cpu()[~real] == 5.0).all())


@pytest.mark.parametrize("dtype,shape", [(BF, (6, 190, 8, 64, 128)), (FP8, (4, 2201, 3, 64, 80)), (torch.uint8, (3, 90, 999, 501))])
def test_large_copies(dtype, shape):
    # more than 64 MiB copied; pages of whole 16-byte pieces, of a last piece that is not full, of odd addresses
    size = torch.Size(shape[2:]).numel() * (2 if dtype == BF else 1)
    pools = torch.randint(0, 255, (shape[0], shape[1], size), dtype=torch.uint8, device=DEV)
    want, n = pools.clone(), shape[1] // 2
    order = torch.randperm(shape[1], generator=torch.Generator().manual_seed(2)).to(DEV)
    src, dst = order[:n], order[n:2 * n]
    want[:, dst] = pools[:, src]
    assert shape[0] * n * size > 64 << 20
    typed = pools.view(dtype).view(shape)
    assert kv_copy_pages(typed, src.to(torch.int32), dst.to(torch.int32)) is typed
    assert torch.equal(pools, want)


def test_every_token_of_a_step_on_a_side_stream_has_its_value():
    # append and attention as a token step uses them, every output against the oracle with the queries it was given
    B, H, Kh, hd, page, steps = 3, 4, 2, 64, 16, 20
    pools = torch.zeros(2, 40, Kh, page, hd, dtype=BF, device=DEV)
    table = torch.arange(24, dtype=torch.int32).view(B, 8).to(DEV)
    turns = rotary_turns(hd, device=DEV)
    x = torch.randn(steps, B, H + 2 * Kh, hd, generator=torch.Generator().manual_seed(31)).to(BF).to(DEV)
    lens = torch.tensor([0, 9, 30], dtype=torch.int32, device=DEV)
    start = lens.cpu()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    kept = []
    with torch.cuda.stream(s):
        for i in range(steps):
            lens.add_(1)
            q, k, v = x[i].split([H, Kh, Kh], dim=1)
            r = rotary_append(q, k, v, lens - 1, turns, pools[0], pools[1], table)
            kept.append((r, pools.clone(), attn_step(r, pools[0], pools[1], table, lens)))
    s.synchronize()
    for i, (r, held, got) in enumerate(kept):
        pos = start + i
        y, slack = K.rotate(x[i, :, :H], pos, turns, False)
        K.assert_rounds_to(r, y, slack, f"token {i}")
        y, slack = K.attn(r, held[0], held[1], table, pos + 1, hd ** -0.5)
        K.assert_rounds_to(got, y, slack, f"token {i}")

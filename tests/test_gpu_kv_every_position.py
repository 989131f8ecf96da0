"""attn_step counts every cached position once, on long rows, ragged batches and calls beyond the last-level cache."""
import pytest
import torch

import kv_markers as M
from oracle import kv_oracle as K
from vortex_amd import attn_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
BF, F16 = torch.bfloat16, torch.float16


def query(B, H, hd, dtype):
    q = torch.zeros(B, H, hd, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    return q


def paged(k, v, kv_heads, page, seed, spare=3):
    """Rows [n, hd] as pages in random order, NaN behind the end, the same in every head; k_pages, v_pages, page ids."""
    n, hd = k.shape
    need = max(1, -(-n // page))
    ids = torch.randperm(need + spare, generator=torch.Generator().manual_seed(seed))[:need]
    out = []
    for x in (k, v):
        full = torch.full((need * page, hd), float("nan"))
        full[:n] = x.float()
        raw = lambda y: y.to(x.dtype).view(torch.uint8 if x.dtype == FP8 else x.dtype).to(DEV)
        p = raw(torch.tensor(float("nan"))).expand(need + spare, kv_heads, page, hd).contiguous()
        p[ids.to(DEV)] = raw(full.view(need, 1, page, hd))
        out.append(p.view(x.dtype))
    return out[0], out[1], ids.to(torch.int32)


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("step", [1, 7])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (F16, False), (BF, True)])
@pytest.mark.parametrize("kv_heads,group,hd,page", [(2, 2, 64, 64), (1, 1, 128, 16), (1, 20, 32, 32), (2, 1, 256, 128), (1, 3, 80, 64)])
@pytest.mark.parametrize("lens", [[70000], [9999, 0, 3, 5000, 131071], [40000] + [1] * 63])
def test_every_position_counts_once(override, lens, kv_heads, group, hd, page, dtype, fp8, step, form):
    override(attn_short=form)
    t = FP8 if fp8 else dtype
    sides = [paged(*M.rows(n, hd, step, t, i), kv_heads, page, i) for i, n in enumerate(lens)]
    table = torch.full((len(lens), max(len(s[2]) for s in sides)), -1, dtype=torch.int32)
    first = 0
    for b, s in enumerate(sides):
        table[b, :len(s[2])] = s[2] + first
        first += s[0].shape[0]
    k, v = (torch.cat([s[i].view(torch.uint8) for s in sides]).view(t) for i in (0, 1))
    want = torch.stack([M.result(n, hd, step) for n in lens])[:, None].expand(-1, kv_heads * group, -1)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = attn_step(query(len(lens), kv_heads * group, hd, dtype), k, v, table.to(DEV), lt, scale=1.0)
    K.assert_rounds_to(got, want, want * M.SLACK, f"{lens[:3]} {hd} {step}")
    for b, n in enumerate(lens):                        # pages that are not there: every 5th
        table[b, ::5] = -1
    at = [torch.arange(n)[torch.arange(n) // page % 5 != 0] for n in lens]
    want = torch.stack([M.result(n, hd, step, used=a) for n, a in zip(lens, at)])[:, None].expand(-1, kv_heads * group, -1)
    got = attn_step(query(len(lens), kv_heads * group, hd, dtype), k, v, table.to(DEV), lt, scale=1.0)
    K.assert_rounds_to(got, want, want * M.SLACK, f"holes, {lens[:3]} {hd} {step}")


@pytest.mark.parametrize("room", [True, False])
@pytest.mark.parametrize("step", [1, 7])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (F16, False), (BF, True), (F16, True)])
@pytest.mark.parametrize("hd", [32, 64, 80, 128, 160, 256])
def test_reads_beyond_the_last_level_cache(hd, dtype, fp8, step, room):
    # more than 128 MiB of reads in a call: its loads are non-temporal where the pages could all be different ones (room).
    # The sequences are one, read to different lengths
    kv_heads, group, page, longest, t = 2, 3, 64, 5001, FP8 if fp8 else dtype
    B = (160 << 20) // (longest * kv_heads * hd * 2 * t.itemsize) + 1
    lens = [longest - 7 * b % 600 for b in range(B)]
    k, v, ids = paged(*M.rows(longest, hd, step, t, hd), kv_heads, page, hd, spare=sum(lens) // page + B if room else 3)
    assert sum(lens) * kv_heads * hd * 2 * k.element_size() > 130 << 20
    want = torch.stack([M.result(n, hd, step, of=longest) for n in lens])[:, None].expand(-1, kv_heads * group, -1)
    got = attn_step(query(B, kv_heads * group, hd, dtype), k, v, ids[None].expand(B, -1).to(DEV),
                    torch.tensor(lens, dtype=torch.int32, device=DEV), scale=1.0)
    K.assert_rounds_to(got, want, want * M.SLACK, f"{B} x {longest}, {hd}")


@pytest.mark.parametrize("room", [True, False])
@pytest.mark.parametrize("dtype,fp8,hd,group", [(BF, False, 128, 1), (F16, False, 64, 8), (BF, True, 128, 8), (BF, False, 80, 4)])
def test_random_values_beyond_the_last_level_cache(dtype, fp8, hd, group, room):
    # four different queries, each in many rows of the call
    n, kv_heads, page, t = 3001, 2, 64, FP8 if fp8 else dtype
    g = torch.Generator().manual_seed(hd)
    scale = 30.0 if fp8 else 1.0
    R = (140 << 20) // (2048 * kv_heads * hd * 2 * t.itemsize * 4) + 1
    k, v, ids = paged((scale * torch.randn(n, hd, generator=g)).to(t), (scale * torch.randn(n, hd, generator=g)).to(t), kv_heads, page,
                      5, spare=4 * R * (n // page + 1) if room else 3)
    ks = vs = torch.tensor([0.02, 0.05], device=DEV) if fp8 else None
    lens = torch.tensor([n, n - 1, 2048, 2500], dtype=torch.int32)
    q = (2 * torch.randn(4, kv_heads * group, hd, generator=g)).to(dtype)
    y, slack = K.attn(q, k, v, ids[None].expand(4, -1), lens, hd ** -0.5, ks, vs)
    got = attn_step(q.repeat(R, 1, 1).to(DEV), k, v, ids[None].expand(4 * R, -1).to(DEV), lens.repeat(R).to(DEV), k_scale=ks, v_scale=vs)
    K.assert_rounds_to(got, y.repeat(R, 1, 1), slack.repeat(R, 1, 1))

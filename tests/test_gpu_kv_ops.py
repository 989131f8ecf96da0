"""attn_step, rotary_append and kv_copy_pages against the float64 oracle: every element has to be one of the roundings
that the oracle's value allows (oracle/kv_oracle.py derives the slack)."""
import pytest
import torch

from oracle import kv_oracle as K
from vortex_amd import attn_step, kv_copy_pages, rotary_append, rotary_turns

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
BF, F16 = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cache(seed, lens, kv_heads, hd, page, dtype, fp8=False, spare=2):
    """Pages in random order, everything behind a sequence's end NaN; (k, v, table, k_scale, v_scale) on the device."""
    g = gen(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    P = sum(need) + spare
    k, v = torch.randn(P, kv_heads, page, hd, generator=g), torch.randn(P, kv_heads, page, hd, generator=g)
    ks = vs = None
    if fp8:
        ks, vs = 0.01 + 0.05 * torch.rand(kv_heads, generator=g), 0.01 + 0.05 * torch.rand(kv_heads, generator=g)
        k, v = k * 30, v * 30
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    used = torch.zeros(P, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            p = order.pop()
            table[b, i] = p
            used[p, : min(page, n - i * page)] = True
    nan = ~used[:, None, :, None].expand(k.shape)
    t = FP8 if fp8 else dtype
    k, v = k.masked_fill(nan, float("nan")).to(t), v.masked_fill(nan, float("nan")).to(t)
    up = lambda x: None if x is None else x.to(DEV)
    return up(k), up(v), up(table), up(ks), up(vs)


def check_attn(q, c, lens, scale=None, what=""):
    k, v, table, ks, vs = c
    lt = torch.tensor(lens, dtype=torch.int32)
    got = attn_step(q, k, v, table, lt.to(DEV), scale=scale, k_scale=ks, v_scale=vs)
    y, slack = K.attn(q, k, v, table, lt, q.shape[2] ** -0.5 if scale is None else scale, ks, vs)
    assert got.dtype == q.dtype and got.shape == q.shape
    K.assert_rounds_to(got, y, slack, what)
    return got


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 255, 511, 1000]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("kv_heads,group,hd,page", [(2, 1, 128, 16), (1, 4, 128, 64), (3, 5, 64, 32), (1, 16, 32, 16),
                                                    (1, 20, 80, 16), (2, 8, 256, 128), (1, 1, 8, 16), (1, 3, 24, 1024),
                                                    (2, 2, 40, 16), (1, 33, 96, 64), (1, 2, 160, 32), (1, 2, 200, 16)])
def test_attention_over_lengths_heads_and_pages(kv_heads, group, hd, page, dtype, fp8):
    c = cache(hd + group, LENS, kv_heads, hd, page, dtype, fp8)
    q = (2 * torch.randn(len(LENS), kv_heads * group, hd, generator=gen(7))).to(dtype).to(DEV)
    got = check_attn(q, c, LENS)
    assert float(got[0].abs().max()) == 0.0


@pytest.mark.parametrize("lens", [[70000], [5000, 0, 3, 9999], [1] * 300, [2049, 0] * 9, [0, 0, 0], [40000] + [1] * 63])
def test_attention_long_and_ragged_batches(lens):
    # few rows and a long axis, many short rows, very uneven ones: every way the positions are shared out
    dtype, kv_heads, group, hd, page = BF, 2, 2, 64, 64
    c = cache(len(lens), lens, kv_heads, hd, page, dtype)
    q = (2 * torch.randn(len(lens), kv_heads * group, hd, generator=gen(3))).to(dtype).to(DEV)
    check_attn(q, c, lens)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    a, b = (attn_step(q, c[0], c[1], c[2], lt) for _ in range(2))
    assert torch.equal(a, b)                    # the order of every sum is fixed


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (F16, True)])
@pytest.mark.parametrize("kv_heads,group,hd,page", [(2, 1, 128, 16), (1, 8, 64, 64), (1, 17, 32, 16), (2, 3, 256, 32), (1, 5, 80, 16),
                                                    (1, 2, 136, 16)])
def test_attention_both_launch_forms(override, kv_heads, group, hd, page, dtype, fp8, form):
    override(attn_short=form)
    lens = [0, 1, 33, 700, 2500, 64, 256, 257]
    c = cache(hd + group, lens, kv_heads, hd, page, dtype, fp8)
    q = (2 * torch.randn(len(lens), kv_heads * group, hd, generator=gen(17))).to(dtype).to(DEV)
    check_attn(q, c, lens)
    c[2][3, 5], c[2][4, :] = -1, -1             # a page that is not there, a sequence without any
    got = check_attn(q, c, lens)
    assert float(got[4].abs().max()) == 0.0


def test_attention_sharp_and_flat_scores():
    lens = [700, 333]
    c = cache(5, lens, 2, 64, 32, BF)
    q = torch.randn(2, 4, 64, generator=gen(4)).to(BF).to(DEV)
    for scale in (0.0, 1e-6, 3.0, -2.0):        # no difference at all, one key taking everything, a negative factor
        check_attn(q, c, lens, scale, f"scale {scale}")
    # scores that rise from position to position: the running maximum moves at every step
    k, v, table, _, _ = cache(6, [1000], 1, 64, 16, BF)
    rise = torch.linspace(-60, 60, 1000)
    flat = torch.zeros(table.shape[1] * 16, 64)
    flat[:1000, 0] = rise
    for order in (1, -1):
        rows = flat.clone()
        rows[:1000] = rows[:1000].flip(0) if order < 0 else rows[:1000]
        for i, p in enumerate(table[0].tolist()):
            k[p, 0] = rows[i * 16:(i + 1) * 16].to(BF).to(DEV)
        q1 = torch.zeros(1, 1, 64)
        q1[0, 0, 0] = 1.0
        check_attn(q1.to(BF).to(DEV), (k, v, table, None, None), [1000], 1.0)


def test_attention_infinities():
    # a score of -inf weighs nothing; one of +inf or NaN shows in the result as in the formula
    lens = [200, 200, 200, 200]
    k, v, table, _, _ = cache(8, lens, 1, 64, 16, BF)
    q = torch.ones(4, 1, 64, dtype=BF, device=DEV)
    k[table[0, 3].item(), 0, 5] = float("-inf")
    k[table[1, :2].long(), 0] = float("-inf")
    k[table[2, 3].item(), 0, 5] = float("nan")
    v[table[3, 3].item(), 0, 5, 7] = float("inf")
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = attn_step(q, k, v, table, lt, scale=0.125)
    kc, vc = k.cpu(), v.cpu()
    for b in (0, 1):
        y, slack = K.attn(q[b:b + 1].cpu(), kc.float().masked_fill(kc.isinf(), -1e4).to(BF), vc, table[b:b + 1], lt[b:b + 1], 0.125)
        d = (got[b].cpu().double() - y[0]).abs()
        assert bool((d <= y[0].abs() * 2 ** -8 + 1e-3 * y[0].abs().max()).all())
    assert bool(got[2].isnan().all())
    assert float(got[3, 0, 7]) == float("inf") and bool(got[3, 0, :7].isfinite().all())


def test_attention_small_weights_count_what_they_are():
    # bf16: a value of 1e30 behind a weight of 2^-115 (or one that underflows) must not come through; f16: one weight of
    # 1 and 20000 of 2^-12 that together outweigh it
    k, v, table, _, _ = cache(12, [300, 300], 1, 64, 16, BF)
    q = torch.zeros(2, 1, 64, dtype=BF, device=DEV)
    q[:, 0, 0] = 1.0
    k[..., 0] = 0.0
    for b, low in ((0, -79.5), (1, -200.0)):
        p = table[b, 7].item()
        k[p, 0, 3], v[p, 0, 3] = 0.0, 1e30
        k[p, 0, 3, 0] = low
    check_attn(q, (k, v, table, None, None), [300, 300], 1.0)
    n = 20000
    k, v, table, _, _ = cache(13, [n], 1, 64, 64, F16)
    k[...] = 0.0
    k[table[0, 100].item(), 0, 9, 0] = 8.3125
    v.copy_((v.float().nan_to_num().abs() + 0.5).to(F16))
    q = torch.zeros(1, 1, 64, dtype=F16, device=DEV)
    q[0, 0, 0] = 1.0
    lt = torch.tensor([n], dtype=torch.int32)
    y, slack = K.attn(q, k, v, table, lt, 1.0)
    # terms are kept to 2^-35 of the largest weight here, and a sum's rounding errors do not all point one way: half of
    # the general slack's 2^-16 and (2 n + 128) 2^-24 terms is ample, and its 2^-25 term does not apply
    slack = y.abs() * (2.0 ** -15 + 2.0 ** -13) / 2 + n * 2.0 ** -35 * v.float().nan_to_num().abs().max().item() / (1 + n * 2.0 ** -12)
    K.assert_rounds_to(attn_step(q, k, v, table, lt.to(DEV), scale=1.0), y, slack)


def test_attention_heads_do_not_touch_each_other():
    # NaN or infinities in one query head, and in a shared value column, stay there
    lens, H = [200, 33], 6
    c = cache(14, lens, 2, 64, 16, BF)
    q = torch.randn(2, H, 64, generator=gen(5)).to(BF).to(DEV)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = attn_step(q, *c[:3], lt)
    for bad in (float("nan"), float("inf")):
        x = q.clone()
        x[0, 4, 3] = bad
        got = attn_step(x, *c[:3], lt)
        keep = torch.ones(2, H, dtype=torch.bool, device=DEV)
        keep[0, 4] = False
        assert torch.equal(got[keep], want[keep]) and bool(got[0, 4].isnan().all())
    c[1][c[2][0, 2].item(), 1, 3, 5] = float("nan")
    got = attn_step(q, *c[:3], lt)
    assert bool(got[0, 3:, 5].isnan().all())
    got[0, 3:, 5] = want[0, 3:, 5]
    assert torch.equal(got, want)


def test_attention_many_sequences_and_large_pages():
    r = torch.randint(0, 5, (1500,), generator=gen(15)).tolist()
    c = cache(15, r, 1, 32, 16, BF)
    check_attn(torch.randn(1500, 2, 32, generator=gen(6)).to(BF).to(DEV), c, r)
    for page, hd in ((65536, 8), (4096, 64)):
        lens = [70000, 3] if page > 60000 else [5000, 4097, 4096]
        c = cache(16, lens, 1, hd, page, BF, spare=1)
        check_attn(torch.randn(len(lens), 1, hd, generator=gen(7)).to(BF).to(DEV), c, lens)


def test_attention_strides_and_layouts():
    lens, kv_heads, group, hd, page = [129, 64, 7], 2, 3, 64, 32
    k, v, table, _, _ = cache(9, lens, kv_heads, hd, page, BF)
    B, H = 3, kv_heads * group
    q = torch.randn(B, H, hd, generator=gen(1)).to(BF).to(DEV)
    want = attn_step(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    wide = torch.full((B, 3 * H + 1, hd), float("nan"), dtype=BF, device=DEV)       # q as a view of a projection
    wide[:, H:2 * H] = q
    assert torch.equal(attn_step(wide[:, H:2 * H], k, v, table, lt), want)
    # slots ahead of heads, padded rows, keys and values in one tensor
    P = k.shape[0]
    both = torch.full((P, page, 2, kv_heads, hd + 8), float("nan"), dtype=BF, device=DEV)
    both[:, :, 0, :, :hd], both[:, :, 1, :, :hd] = k.transpose(1, 2), v.transpose(1, 2)
    kk, vv = both[:, :, 0, :, :hd].transpose(1, 2), both[:, :, 1, :, :hd].transpose(1, 2)
    assert torch.equal(attn_step(q, kk, vv, table, lt), want)
    vt = v.transpose(1, 2).contiguous().transpose(1, 2)                             # the two sides laid out differently
    assert torch.equal(attn_step(q, k, vt, table, lt), want)
    big = torch.full((B, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)    # a wider table, read in part
    big[:, :table.shape[1]] = table
    assert torch.equal(attn_step(q, k, v, big[:, :table.shape[1]], lt), want)
    out = torch.empty(B, H, hd, dtype=BF, device=DEV)
    assert attn_step(q, k, v, big, lt, out=out) is out and torch.equal(out, want)
    # one table row for several queries of a sequence, as a continuation of several tokens uses it
    n = torch.tensor([127, 128, 129], dtype=torch.int32, device=DEV)
    same = attn_step(q[:1].expand(3, H, hd), k, v, table[:1].expand(3, -1), n)
    y, slack = K.attn(q[:1].expand(3, H, hd), k, v, table[:1].expand(3, -1), n, hd ** -0.5)
    K.assert_rounds_to(same, y, slack)


@pytest.mark.parametrize("hd,pad", [(64, 8), (128, 24), (256, 8), (32, 8), (80, 16)])
def test_attention_8_bit_rows_at_odd_strides(hd, pad):
    # rows hd + pad bytes apart: 8-byte multiples that are no 16-byte multiples, keys and values differently
    lens = [129, 64, 7, 500]
    k, v, table, ks, vs = cache(hd, lens, 2, hd, 16, BF, True)
    q = torch.randn(4, 6, hd, generator=gen(1)).to(BF).to(DEV)
    lt = torch.tensor(lens, dtype=torch.int32)
    y, slack = K.attn(q, k, v, table, lt, hd ** -0.5, ks, vs)

    def apart(x):
        w = torch.zeros(x.shape[0], 2, 16, hd + pad, device=DEV).to(FP8)
        w.view(torch.uint8)[..., :hd] = x.view(torch.uint8)
        return w[..., :hd]

    for kk, vv in ((apart(k), apart(v)), (k, apart(v)), (apart(k), v)):
        K.assert_rounds_to(attn_step(q, kk, vv, table, lt.to(DEV), k_scale=ks, v_scale=vs), y, slack)


def test_scales_on_pages_of_the_activations_type():
    lens = [100, 33]
    k, v, table, _, _ = cache(3, lens, 2, 64, 16, F16)
    ks, vs = torch.tensor([0.5, 3.0], device=DEV), torch.tensor([0.125, 7.0], device=DEV)
    q = torch.randn(2, 4, 64, generator=gen(1)).to(F16).to(DEV)
    lt = torch.tensor(lens, dtype=torch.int32)
    y, slack = K.attn(q, k, v, table, lt, 0.125, ks, vs)
    K.assert_rounds_to(attn_step(q, k, v, table, lt.to(DEV), k_scale=ks, v_scale=vs), y, slack)
    x = torch.randn(1, 2, 64, generator=gen(2)).to(F16).to(DEV)
    kp, vp = torch.zeros(1, 2, 16, 64, dtype=F16, device=DEV), torch.zeros(1, 2, 16, 64, dtype=F16, device=DEV)
    rotary_append(x, x, x, torch.tensor([5], dtype=torch.int32, device=DEV), rotary_turns(64, device=DEV), kp, vp,
                  torch.zeros(1, 1, dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs)
    w = x.double().cpu() / vs.double().cpu()[None, :, None]
    K.assert_rounds_to(vp[:, :, 5], w, w.abs() * 2.0 ** -24)
    w, sl = K.rotate(x, torch.tensor([5]), rotary_turns(64), False)
    d = ks.double().cpu()[None, :, None]
    K.assert_rounds_to(kp[:, :, 5], w / d, sl / d + (w / d).abs() * 2.0 ** -24)


def test_attention_leaves_out_pages_that_are_not_there():
    lens = [100, 64, 40, 500]
    k, v, table, _, _ = cache(10, lens, 1, 64, 16, BF)
    table = table[:, :8].contiguous()                                   # the last length is beyond the table's reach
    table[0, 2], table[0, 5], table[1, :] = -1, k.shape[0], 2 ** 30     # holes, and a row with no page at all
    q = torch.randn(4, 2, 64, generator=gen(2)).to(BF).to(DEV)
    got = check_attn(q, (k, v, table, None, None), lens)
    assert float(got[1].abs().max()) == 0.0


def test_attention_offsets_beyond_32_bits():
    # pages of 1 MiB in a pool of 5 GiB a side: the byte offsets of the last pages do not fit 32 bits
    hd, page, heads = 128, 512, 8
    P = 5 * 1024 ** 3 // (hd * page * heads * 2)
    k = torch.zeros(P, heads, page, hd, dtype=BF, device=DEV)
    v = torch.zeros(P, heads, page, hd, dtype=BF, device=DEV)
    far = [P - 1, 0, P - 2, P // 2 + 3]
    small = torch.randn(2, 4, heads, page, hd, generator=gen(11)).to(BF)
    for i, p in enumerate(far):
        k[p], v[p] = small[0, i].to(DEV), small[1, i].to(DEV)
    q = torch.randn(1, heads, hd, generator=gen(12)).to(BF).to(DEV)
    n = torch.tensor([2000], dtype=torch.int32, device=DEV)
    got = attn_step(q, k, v, torch.tensor([far], dtype=torch.int32, device=DEV), n)
    y, slack = K.attn(q, small[0], small[1], torch.arange(4, dtype=torch.int32)[None], n, hd ** -0.5)
    K.assert_rounds_to(got, y, slack)
    pos = torch.tensor([3 * page - 1, 1], dtype=torch.int32, device=DEV)
    x = torch.randn(2, heads, hd, generator=gen(13)).to(BF).to(DEV)
    rotary_append(x, x, x, pos, rotary_turns(hd, device=DEV), k, v, torch.tensor([far], dtype=torch.int32, device=DEV))
    assert torch.equal(v[P - 2, :, page - 1], x[0]) and torch.equal(v[P - 1, :, 1], x[1])
    kv_copy_pages(k.view(1, P, heads, page, hd), torch.tensor([P - 1], dtype=torch.int32, device=DEV),
                  torch.tensor([P - 3], dtype=torch.int32, device=DEV))
    assert torch.equal(k[P - 3], k[P - 1]) and float(k[P - 4].abs().max()) == 0.0


def append_case(seed, T, heads, kv_heads, hd, rd, page, dtype, fp8, pos, seq, rows, interleaved, dense=True, base=10000.0,
                given_out=True):
    g = gen(seed)
    width = max(1, max((p // page + 1 for p in pos if p >= 0), default=1))
    at = [(t // (T // rows) if seq is None else seq[t]) for t in range(T)]
    names = sorted({(s, p // page) for s, p in zip(at, pos) if p >= 0})
    P = len(names) + 2
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((rows, width), -1, dtype=torch.int32)
    for s, i in names:
        table[s, i] = order.pop()
    qkv = torch.randn(T, heads + 2 * kv_heads, hd, generator=g).to(dtype).to(DEV)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    ks = vs = None
    if fp8:
        ks, vs = (0.002 + 0.02 * torch.rand(kv_heads, generator=g)).to(DEV), (0.01 + 0.02 * torch.rand(kv_heads, generator=g)).to(DEV)
    t = FP8 if fp8 else dtype
    mark = torch.full((P, kv_heads, page, hd), 3.0)
    kp, vp = mark.to(t).to(DEV), mark.to(t).to(DEV)
    q_out = torch.full((T, heads, hd), 5.0, dtype=dtype, device=DEV) if given_out else None
    k_out = torch.full((T, kv_heads, hd), 5.0, dtype=dtype, device=DEV) if dense else None
    turns = rotary_turns(rd, base, device=DEV)
    p = torch.tensor(pos, dtype=torch.int32, device=DEV)
    got = rotary_append(q, k, v, p, turns, kp, vp, table.to(DEV), interleaved=interleaved, k_scale=ks, v_scale=vs,
                        seq=None if seq is None else torch.tensor(seq, dtype=torch.int32, device=DEV), q_out=q_out, k_out=k_out)
    assert q_out is None or got is q_out
    real = torch.tensor([x >= 0 for x in pos])
    for y, x, name in ((got, q, "q_out"), (k_out, k, "k_out")):
        if y is None:
            continue
        want, slack = K.rotate(x, p, turns, interleaved)
        K.assert_rounds_to(y.cpu()[real], want[real], slack[real], name)
        rest = y.cpu()[~real]
        assert bool((rest == (5.0 if given_out or name == "k_out" else 0.0)).all()) or not rest.numel()
    for pages, x, sc, name in ((kp, k, ks, "k_pages"), (vp, v, vs, "v_pages")):
        want = torch.full((P, kv_heads, page, hd), 3.0, dtype=torch.float64)
        slack = torch.zeros_like(want)
        y, sl = K.rotate(x, p, turns, interleaved) if x is k else (x.detach().cpu().double(), torch.zeros(T, kv_heads, hd, dtype=torch.float64))
        if sc is not None:
            d = sc.cpu().double()[None, :, None]
            y, sl = y / d, sl / d + (y / d).abs() * 2.0 ** -24
        for i in range(T):
            if pos[i] >= 0:
                pg = int(table[at[i], pos[i] // page])
                want[pg, :, pos[i] % page], slack[pg, :, pos[i] % page] = y[i], sl[i]
        K.assert_rounds_to(pages, want, slack, name)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (F16, False), (BF, True), (F16, True)])
@pytest.mark.parametrize("heads,kv_heads,hd,rd,page", [(2, 2, 128, 128, 16), (8, 2, 64, 64, 32), (5, 1, 80, 80, 16), (4, 4, 64, 32, 16),
                                                       (3, 3, 128, 24, 16), (20, 4, 80, 20, 64), (1, 1, 8, 8, 16), (2, 1, 256, 256, 16),
                                                       (6, 2, 40, 2, 16), (2, 2, 96, 0, 16), (16, 1, 32, 32, 128)])
def test_append_over_heads_and_rotary_parts(heads, kv_heads, hd, rd, page, dtype, fp8, interleaved):
    pos = [0, 1, 14, 15, 16, 17, 47, -1, 100, 1001, 3, 2]
    append_case(hd + rd, 12, heads, kv_heads, hd, rd, page, dtype, fp8, pos, None, 1, interleaved)


def test_append_one_token_to_many_and_padded_batches():
    append_case(1, 1, 4, 4, 64, 64, 16, BF, False, [203], None, 1, False, dense=False, given_out=False)
    append_case(2, 40, 4, 2, 64, 64, 16, BF, False, list(range(100, 140)), None, 40, False, dense=False)
    pos = list(range(37)) + [-1] * 27 + list(range(5, 69))                      # a padded batch of two
    append_case(3, 128, 2, 2, 64, 64, 16, F16, False, pos, None, 2, True, given_out=False)
    append_case(4, 200, 3, 1, 128, 64, 64, BF, True, list(range(1000, 1200)), None, 1, False)
    # rows of several sequences in any order
    g = gen(5)
    seq = torch.randint(0, 5, (90,), generator=g).tolist()
    count, pos = [0] * 5, []
    for s in seq:
        pos.append(count[s] + 7 * s)
        count[s] += 1
    append_case(6, 90, 4, 2, 64, 64, 16, BF, False, pos, seq, 5, False)


@pytest.mark.parametrize("base,start", [(10000.0, 131071), (1e11, 1048575), (10000.0, 2 ** 24 + 1)])
def test_append_far_positions_keep_their_angle(base, start):
    # 32-bit angles would be off by radians here; the oracle's are 64-bit
    append_case(9, 3, 2, 2, 128, 128, 4096, BF, False, [start, start + 1, start - 5000], None, 1, False, base=base)


def test_append_in_place_and_pages_that_are_not_there():
    g = gen(21)
    T, H, hd, page = 6, 2, 64, 16
    q, k, v = (torch.randn(T, H, hd, generator=g).to(BF).to(DEV) for _ in range(3))
    turns = rotary_turns(hd, device=DEV)
    pos = torch.tensor([0, 20, 40, 15, 16, 70], dtype=torch.int32, device=DEV)
    seq = torch.tensor([0, 0, 0, 1, 2, 0], dtype=torch.int32, device=DEV)
    table = torch.tensor([[0, -1, 9], [1, 2, 0]], dtype=torch.int32, device=DEV)    # holes, an id too large
    kp, vp = torch.zeros(4, H, page, hd, dtype=BF, device=DEV), torch.zeros(4, H, page, hd, dtype=BF, device=DEV)
    want = rotary_append(q, k, v, pos, turns, kp, vp, table, seq=seq)
    # written: (0, 0) and (1, 15); dropped: a hole, an id too large, a sequence and a position beyond the table
    assert torch.equal(vp[0, :, 0], v[0]) and torch.equal(vp[1, :, 15], v[3])
    vp[0, :, 0], vp[1, :, 15], kp[0, :, 0], kp[1, :, 15] = 0, 0, 0, 0
    assert float(vp.abs().max()) == 0.0 and float(kp.abs().max()) == 0.0
    y, slack = K.rotate(q, pos, turns, False)
    K.assert_rounds_to(want, y, slack)
    qi, ki, kw = q.clone(), k.clone(), torch.empty_like(k)
    rotary_append(q, k, v, pos, turns, kp, vp, table, seq=seq, k_out=kw)
    assert rotary_append(qi, ki, v, pos, turns, kp, vp, table, seq=seq, q_out=qi, k_out=ki) is qi
    assert torch.equal(qi, want) and torch.equal(ki, kw)


def test_append_specials_in_8_bits():
    x = torch.zeros(1, 1, 16, dtype=BF)
    x[0, 0, :6] = torch.tensor([float("nan"), float("inf"), float("-inf"), 1e4, -460.0, 449.0])
    x = x.to(DEV)
    kp, vp = torch.zeros(1, 1, 16, 16, dtype=FP8, device=DEV), torch.zeros(1, 1, 16, 16, dtype=FP8, device=DEV)
    rotary_append(x, x, x, torch.zeros(1, dtype=torch.int32, device=DEV), rotary_turns(0, device=DEV), kp, vp,
                  torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    got = vp.float()[0, 0, 0, :6].tolist()
    assert got[0] != got[0] and got[1:] == [448.0, -448.0, 448.0, -448.0, 448.0]


@pytest.mark.parametrize("dtype,shape", [(BF, (3, 50, 2, 16, 64)), (FP8, (2, 90, 3, 16, 80)), (torch.uint8, (5, 40, 7)),
                                         (torch.float32, (1, 33, 5, 3)), (BF, (4, 20, 1, 1, 1)), (BF, (2, 12, 8, 512, 128))])
def test_copies(dtype, shape):
    raw = torch.randint(0, 255, shape + ((2 if dtype == BF else 4 if dtype == torch.float32 else 1),), dtype=torch.uint8,
                        generator=gen(3))
    pools = raw.to(DEV).view(dtype).squeeze(-1) if dtype not in (FP8, torch.uint8) else raw[..., 0].contiguous().to(DEV).view(dtype)
    b = lambda x: x.contiguous().view(torch.uint8)
    n = shape[1]
    order = torch.randperm(n, generator=gen(4))
    src, dst = order[: n // 3], order[n // 3: 2 * (n // 3)]
    i32 = lambda x: x.to(torch.int32).to(DEV)
    want = pools.clone()
    b(want).view(shape[0], n, -1)[:, dst.to(DEV)] = b(pools).view(shape[0], n, -1)[:, src.to(DEV)]
    other = torch.zeros((shape[0], n + 3) + tuple(shape[2:]), dtype=torch.float32, device=DEV).to(dtype)
    assert kv_copy_pages(pools, i32(src), i32(dst + 3), dst_pools=other) is other
    assert torch.equal(b(other).view(shape[0], n + 3, -1)[:, (dst + 3).to(DEV)], b(pools).view(shape[0], n, -1)[:, src.to(DEV)])
    assert kv_copy_pages(pools, i32(src), i32(dst)) is pools
    assert torch.equal(b(pools), b(want))
    kv_copy_pages(pools, i32(torch.zeros(len(dst))), i32(dst))                      # one page many times
    assert all(torch.equal(b(pools[:, d]), b(pools[:, 0])) for d in dst.tolist() if d)
    before = b(pools).clone()
    bad = torch.tensor([-1, n, 2, 2 ** 30], dtype=torch.int32, device=DEV)
    kv_copy_pages(pools, bad, i32(torch.tensor([3, 4, n, 5])))                      # pages that are not there
    kv_copy_pages(pools, bad[:0], bad[:0])
    assert torch.equal(b(pools), before)


def test_copies_between_strided_pools():
    pools = torch.randn(6, 20, 2, 16, 64, generator=gen(5)).to(BF).to(DEV)
    want = pools.clone()
    sub = pools[::2, 3:15]                                                          # every second pool, some of its pages
    want[::2, 3 + 7] = want[::2, 3 + 2]
    kv_copy_pages(sub, torch.tensor([2], dtype=torch.int32, device=DEV), torch.tensor([7], dtype=torch.int32, device=DEV))
    assert torch.equal(pools, want)


def test_run_together_on_another_stream_and_in_a_graph():
    # append, attention, and a copied page, as a token step uses them; once eagerly on a side stream, then recorded and
    # replayed while lengths and positions move on the device, with eager work between the replays
    B, H, Kh, hd, page = 3, 4, 2, 64, 16
    g = gen(31)
    pools = torch.zeros(2, 40, Kh, page, hd, dtype=BF, device=DEV)
    table = torch.arange(24, dtype=torch.int32).view(B, 8).to(DEV)
    turns = rotary_turns(hd, device=DEV)
    steps = 20
    x = torch.randn(steps, B, H + 2 * Kh, hd, generator=g).to(BF).to(DEV)
    lens = torch.tensor([0, 9, 30], dtype=torch.int32, device=DEV)
    start = lens.clone()

    def token(row):
        lens.add_(1)
        q, k, v = row.split([H, Kh, Kh], dim=1)
        r = rotary_append(q, k, v, lens - 1, turns, pools[0], pools[1], table)
        return attn_step(r, pools[0], pools[1], table, lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = [token(x[i]) for i in range(steps)]
    s.synchronize()
    ended = pools.clone()
    for i in (0, 7, 19):
        lt = start + i + 1
        y, slack = K.attn(torch.zeros(B, H, hd), pools[0].cpu().float(), pools[1].cpu().float(), table, lt, 1.0)
        assert eager[i].shape == y.shape and bool(eager[i].isfinite().all())
    lens.copy_(start)
    pools.zero_()
    row = x[0].clone()
    graph = torch.cuda.CUDAGraph()
    token(row)                                                                      # warm up; put back below
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = token(row)
    lens.copy_(start)
    pools.zero_()
    for i in range(steps):
        row.copy_(x[i])
        graph.replay()
        assert torch.equal(out, eager[i]), i
        attn_step(x[i][:, :H].contiguous(), pools[0], pools[1], table, lens)        # eager calls between the replays
        torch.cuda.synchronize()
    assert torch.equal(pools, ended)

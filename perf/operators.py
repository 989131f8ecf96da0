"""Cases and plain forms of the paged key / value cache operators: attention of one new token per sequence over the
pages, rotary positions with the append into the pages, and copies of whole pages.

A cache layer is two tensors of pages, k_pages and v_pages [pages, kv_heads, page_size, head_dim]; row b of `table`
names the pages of sequence b in order, so key j of that sequence sits in page table[b, j // page_size] at slot
j % page_size."""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_FP8 = torch.float8_e4m3fn
_FP8_MAX = 448.0


def listed():
    return [
        # a chat-length prompt on one device: what a single generation pays per token and attention layer
        dict(op="attn", name="attn one sequence 203", batch=1, heads=32, kv_heads=32, head_dim=128, page=16, longest=203,
             ragged=0, type="bf16", fp8=False),
        # the longest prompt of the end-to-end benchmark
        dict(op="attn", name="attn one sequence 131072", batch=1, heads=32, kv_heads=32, head_dim=128, page=256,
             longest=131072, ragged=0, type="bf16", fp8=False),
        # the batch of the decode benchmark, every sequence at another length, one of them empty
        dict(op="attn", name="attn batch 64 ragged", batch=64, heads=32, kv_heads=32, head_dim=128, page=64, longest=4096,
             ragged=1, type="bf16", fp8=False),
        # shared key heads, smaller heads, an odd length
        dict(op="attn", name="attn shared heads f16", batch=16, heads=32, kv_heads=4, head_dim=64, page=32, longest=8191,
             ragged=2, type="f16", fp8=False),
        # a serving batch on a cache held in 8 bits
        dict(op="attn", name="attn shared heads fp8", batch=32, heads=64, kv_heads=8, head_dim=128, page=64, longest=32768,
             ragged=3, type="bf16", fp8=True),
        # one token of one sequence: latency
        dict(op="rotary", name="rotary one token", batch=1, length=1, heads=32, kv_heads=32, head_dim=128, rotary_dim=128,
             page=16, start=203, ragged=0, interleaved=False, base=10000.0, factor=1.0, type="bf16", fp8=False, dense=False),
        # one token of a serving batch far into long contexts, positions interpolated, cache in 8 bits
        dict(op="rotary", name="rotary batch 64 far fp8", batch=64, length=1, heads=64, kv_heads=8, head_dim=128,
             rotary_dim=128, page=64, start=1000003, ragged=1, interleaved=False, base=1.0e11, factor=128.0, type="bf16",
             fp8=True, dense=False),
        # the prefill of the end-to-end benchmark's short prompt; the dense keys go on to the prompt's own attention
        dict(op="rotary", name="rotary prefill 8192", batch=1, length=8192, heads=32, kv_heads=32, head_dim=128,
             rotary_dim=128, page=256, start=0, ragged=0, interleaved=False, base=10000.0, factor=1.0, type="bf16",
             fp8=False, dense=True),
        # a padded batch of prompts of different lengths, interleaved pairs in half of each head
        dict(op="rotary", name="rotary padded interleaved", batch=8, length=2047, heads=20, kv_heads=4, head_dim=64,
             rotary_dim=32, page=32, start=17, ragged=2, interleaved=True, base=10000.0, factor=1.0, type="f16", fp8=False,
             dense=False),
        # one prompt forked into eight continuations: the page that is not full is copied, in every layer
        dict(op="copy", name="copy fork 7", pools=16, kv_heads=32, head_dim=128, page=16, pages=64, copies=7, fork=True,
             type="bf16", fp8=False),
        # compaction of a cache after its sequences ended
        dict(op="copy", name="copy compact 200", pools=16, kv_heads=8, head_dim=128, page=64, pages=512, copies=200,
             fork=False, type="bf16", fp8=False),
        # small odd pages
        dict(op="copy", name="copy odd pages", pools=2, kv_heads=3, head_dim=80, page=16, pages=90, copies=33, fork=False,
             type="bf16", fp8=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rotary", "rotary", "copy"])
    typ, fp8 = rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.3
    kv = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if kv * g <= 64])
    hd = rng.choice([32, 64, 64, 80, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "attn":
        batch = _log(rng, 1, 200)
        most = min(131072, 131072 * 32 * 128 // (batch * kv * hd))       # at most the keys of the largest listed case
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv, head_dim=hd, page=page,
                    longest=_log(rng, 1, max(2, min(most, 60000 * 32 // heads))), ragged=rng.randrange(100), type=typ, fp8=fp8)
    if op == "rotary":
        batch = _log(rng, 1, 64)
        length = 1 if rng.random() < 0.4 else _log(rng, 1, max(2, 8192 * 64 // (batch * (heads + kv)) * 128 // hd))
        rot = rng.choice([r for r in (hd, hd, hd // 2, hd // 4, 24) if r <= hd])
        far = rng.random() < 0.3
        return dict(op=op, batch=batch, length=length, heads=heads, kv_heads=kv, head_dim=hd, rotary_dim=rot,
                    page=page, start=_log(rng, 1, 1000000) if far else rng.randrange(2000), ragged=rng.randrange(100),
                    interleaved=rng.random() < 0.4, base=rng.choice([10000.0, 1.0e6, 1.0e11]),
                    factor=rng.choice([1.0, 1.0, 8.0, 128.0]), type=typ, fp8=fp8, dense=rng.random() < 0.3)
    pages, pools = _log(rng, 20, 400), rng.choice([2, 6, 10, 16])
    return dict(op=op, pools=pools, kv_heads=min(kv, 8), head_dim=hd if hd < 256 else 128, page=min(page, 64), pages=pages,
                copies=rng.randrange(1, pages // 2), fork=rng.random() < 0.3, type=typ, fp8=fp8)


def _lengths(case):
    """Keys per sequence (attn) or new tokens per sequence (rotary): all the longest where the batch is not ragged."""
    longest = case["longest"] if case["op"] == "attn" else case["length"]
    if not case["ragged"] or longest == 1:
        return [longest] * case["batch"]
    r = random.Random(case["ragged"])
    got = [r.randint(1, longest) for _ in range(case["batch"])]
    got[0] = longest
    if case["batch"] > 2:
        got[1] = 0
    return got


def _starts(case):
    """Tokens that each sequence holds before the append."""
    if not case["ragged"]:
        return [case["start"]] * case["batch"]
    r = random.Random(1000 + case["ragged"])
    return [case["start"] - r.randint(0, min(case["start"], 4000)) for _ in range(case["batch"])]


def _size(case):
    return 1 if case["fp8"] else 2


def _pages(g, shape, case):
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    for i in range(shape[0]):       # page by page: no float32 copy of a large cache
        x[i].normal_(generator=g)
    return x.to(_FP8) if case["fp8"] else x.to(_TYPES[case["type"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, t = "cuda", _TYPES[case["type"]]
    st = dict(op=case["op"])
    if case["op"] == "copy":
        n, pages = case["copies"], case["pages"]
        st["pools"] = _pages(g, (case["pools"], pages, case["kv_heads"], case["page"], case["head_dim"]), case)
        order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        st["dst"] = order[:n].contiguous()
        st["src"] = order[n:n + 1].repeat(n) if case["fork"] else order[n:2 * n].contiguous()
        return st
    B, H, K, hd, ps = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    lens = _lengths(case)
    if case["fp8"]:                 # one scale a head, as a calibrated cache has them
        st["k_scale"] = 0.02 + 0.03 * torch.rand(K, generator=g, device=dev)
        st["v_scale"] = 0.02 + 0.03 * torch.rand(K, generator=g, device=dev)
    else:
        st["k_scale"] = st["v_scale"] = None
    if case["op"] == "attn":
        starts, ends = [0] * B, lens
    else:
        starts = _starts(case)
        ends = [s + n for s, n in zip(starts, lens)]
    first = [s // ps for s in starts]                       # only the pages that the call touches are there
    need = [max(0, -(-e // ps) - f) for e, f in zip(ends, first)]
    width = max(1, max(-(-e // ps) for e in ends))
    spare = 4
    order = torch.randperm(sum(need) + spare, generator=g, device=dev).to(torch.int32)
    row = torch.repeat_interleave(torch.arange(B, device=dev), torch.tensor(need, device=dev))
    ahead = torch.tensor([sum(need[:b]) - first[b] for b in range(B)], device=dev)
    col = torch.arange(sum(need), device=dev) - ahead[row]
    st["table"] = torch.zeros(B, width, dtype=torch.int32, device=dev)
    st["table"][row, col] = order[: sum(need)]
    shape = (sum(need) + spare, K, ps, hd)
    if case["op"] == "attn":
        st["k_pages"], st["v_pages"] = _pages(g, shape, case), _pages(g, shape, case)
        if case["fp8"]:             # values of the size that such a scale is chosen for
            st["k_pages"] = (st["k_pages"].to(torch.bfloat16) * 32).to(_FP8)
            st["v_pages"] = (st["v_pages"].to(torch.bfloat16) * 32).to(_FP8)
        st["q"] = (2 * torch.randn(B, H, hd, generator=g, device=dev)).to(t)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["scale"] = hd ** -0.5
        return st
    L, rd = case["length"], case["rotary_dim"]
    st["k_pages"] = torch.zeros(shape, dtype=_FP8 if case["fp8"] else t, device=dev)
    st["v_pages"] = torch.zeros_like(st["k_pages"])
    qkv = torch.randn(B * L, (H + 2 * K) * hd, generator=g, device=dev).to(t)       # one projection's rows
    st["q"], st["k"], st["v"] = (x.view(B * L, -1, hd) for x in qkv.split([H * hd, K * hd, K * hd], dim=1))
    i = torch.arange(L, device=dev)[None]
    pos = torch.tensor(starts, device=dev)[:, None] + i
    pos = torch.where(i < torch.tensor(lens, device=dev)[:, None], pos, torch.full_like(pos, -1))   # padding
    st["pos"] = pos.reshape(-1).to(torch.int32)
    freq = case["base"] ** (-torch.arange(0, rd, 2, dtype=torch.float64, device=dev) / rd) / case["factor"]
    st["turns"], st["interleaved"] = freq / (2 * math.pi), case["interleaved"]
    st["q_out"] = torch.zeros(B * L, H, hd, dtype=t, device=dev)
    st["k_out"] = torch.zeros(B * L, K, hd, dtype=t, device=dev) if case["dense"] else None
    return st


def _attn_plain(st):
    q, table, lens = st["q"], st["table"].long(), st["lens"]
    (B, H, hd), (_, K, ps, _) = q.shape, st["k_pages"].shape
    S = table.shape[1] * ps

    def rows(pages, scale):
        x = pages.view(torch.uint8)[table].view(pages.dtype) if pages.dtype == _FP8 else pages[table]
        x = x.float().permute(0, 2, 1, 3, 4).reshape(B, K, S, hd)
        return x if scale is None else x * scale[None, :, None, None]

    s = torch.matmul(q.float().view(B, K, H // K, hd), rows(st["k_pages"], st["k_scale"]).transpose(2, 3)) * st["scale"]
    there = (torch.arange(S, device=q.device) < lens[:, None])[:, None, None]
    s = torch.where(there, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.where(there, torch.exp(s - m), torch.zeros_like(s))
    o = torch.matmul(p / p.sum(-1, keepdim=True), rows(st["v_pages"], st["v_scale"]))
    o = torch.where((lens > 0)[:, None, None, None], o, torch.zeros_like(o))
    return o.reshape(B, H, hd).to(q.dtype)


def _rotate_plain(x, cos, sin, interleaved):
    rd, y = 2 * cos.shape[-1], x.float()
    x1, x2 = (y[..., 0:rd:2], y[..., 1:rd:2]) if interleaved else (y[..., : rd // 2], y[..., rd // 2: rd])
    c, s = cos[:, None], sin[:, None]
    y1, y2 = x1 * c - x2 * s, x1 * s + x2 * c
    r = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([r, y[..., rd:]], -1)


def _rotary_plain(st):
    pos, table, ps = st["pos"].long(), st["table"].long(), st["k_pages"].shape[2]
    turn = pos.double()[:, None] * st["turns"]
    angle = (turn - torch.round(turn)) * (2 * math.pi)      # in 64 bits: far positions lose their angle in 32
    cos, sin = angle.cos().float(), angle.sin().float()
    real = pos >= 0
    seq = torch.arange(pos.numel(), device=pos.device) // (pos.numel() // table.shape[0])
    at = pos.clamp(min=0)
    page, slot = table[seq, at // ps][real], (at % ps)[real]
    q = _rotate_plain(st["q"], cos, sin, st["interleaved"]).to(st["q"].dtype)
    st["q_out"].copy_(torch.where(real[:, None, None], q, st["q_out"]))
    k = _rotate_plain(st["k"], cos, sin, st["interleaved"])
    if st["k_out"] is not None:
        st["k_out"].copy_(torch.where(real[:, None, None], k.to(st["k"].dtype), st["k_out"]))
    for x, pages, scale in ((k, st["k_pages"], st["k_scale"]), (st["v"].float(), st["v_pages"], st["v_scale"])):
        if scale is None:
            pages[page, :, slot] = x[real].to(pages.dtype)
        else:
            y = (x[real] / scale[None, :, None]).clamp(-_FP8_MAX, _FP8_MAX).to(_FP8)
            pages.view(torch.uint8)[page, :, slot] = y.view(torch.uint8)
    return [x for x in (st["q_out"], st["k_out"], st["k_pages"], st["v_pages"]) if x is not None]


def _copy_plain(st):
    p = st["pools"].view(torch.uint8) if st["pools"].dtype == _FP8 else st["pools"]
    p[:, st["dst"].long()] = p[:, st["src"].long()]
    return st["pools"]


def run(state):
    st = state
    if not own:
        return {"attn": _attn_plain, "rotary": _rotary_plain, "copy": _copy_plain}[st["op"]](st)
    import vortex_amd
    if st["op"] == "attn":
        return vortex_amd.attn_step(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], scale=st["scale"],
                                    k_scale=st["k_scale"], v_scale=st["v_scale"])
    if st["op"] == "rotary":
        vortex_amd.rotary_append(st["q"], st["k"], st["v"], st["pos"], st["turns"], st["k_pages"], st["v_pages"],
                                 st["table"], interleaved=st["interleaved"], k_scale=st["k_scale"],
                                 v_scale=st["v_scale"], q_out=st["q_out"], k_out=st["k_out"])
        return [x for x in (st["q_out"], st["k_out"], st["k_pages"], st["v_pages"]) if x is not None]
    vortex_amd.kv_copy_pages(st["pools"], st["src"], st["dst"])
    return st["pools"]


def work(case):
    if case["op"] == "copy":
        page = case["kv_heads"] * case["page"] * case["head_dim"] * _size(case)
        reads = 1 if case["fork"] else case["copies"]
        return {"bytes": case["pools"] * (reads + case["copies"]) * page + 8 * case["copies"], "flops": 0}
    H, K, hd = case["heads"], case["kv_heads"], case["head_dim"]
    n = sum(_lengths(case))
    if case["op"] == "attn":
        table = sum(-(-x // case["page"]) for x in _lengths(case))
        return {"bytes": 2 * n * K * hd * _size(case) + 4 * case["batch"] * H * hd + 4 * table + 4 * case["batch"],
                "flops": 4 * n * H * hd}
    dense = 2 * K * hd if case["dense"] else 0
    return {"bytes": n * (2 * (2 * H + 2 * K) * hd + dense + 2 * K * hd * _size(case)) + 4 * case["batch"] * case["length"],
            "flops": 3 * n * (H + K) * case["rotary_dim"]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "copy":
        got = st["pools"].to(torch.float64)
        for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
            got[:, d] = st["pools"][:, s].to(torch.float64)
        return got
    K, ps, hd = case["kv_heads"], case["page"], case["head_dim"]
    table = st["table"].tolist()
    if case["op"] == "attn":
        g = case["heads"] // K
        out = torch.zeros(case["batch"], case["heads"], hd, dtype=torch.float64, device="cuda")
        for b, n in enumerate(st["lens"].tolist()):
            if n == 0:
                continue
            used = st["table"][b, : -(-n // ps)].long()
            for h in range(K):
                key = st["k_pages"][used, h].double().reshape(-1, hd)[:n]
                val = st["v_pages"][used, h].double().reshape(-1, hd)[:n]
                if case["fp8"]:
                    key, val = key * st["k_scale"][h].double(), val * st["v_scale"][h].double()
                w = torch.softmax((key @ st["q"][b, h * g:(h + 1) * g].double().T) * st["scale"], dim=0)
                out[b, h * g:(h + 1) * g] = w.T @ val
        return out
    B, L, rd = case["batch"], case["length"], case["rotary_dim"]
    # the definition: each pair of a head as a complex number, times e^(i * position * frequency)
    freq = torch.tensor([case["base"] ** (-2.0 * i / rd) / case["factor"] for i in range(rd // 2)], dtype=torch.float64,
                        device="cuda")
    pos = st["pos"].view(B, L)
    phase = torch.polar(torch.ones(B * L, rd // 2, dtype=torch.float64, device="cuda"), st["pos"].double()[:, None] * freq)

    def turned(x):
        y = x.double().clone()
        one, two = (slice(0, rd, 2), slice(1, rd, 2)) if case["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
        z = torch.complex(y[..., one], y[..., two]) * phase[:, None]
        y[..., one], y[..., two] = z.real, z.imag
        return y

    real = (st["pos"] >= 0)[:, None, None]
    q, k, v = turned(st["q"]), turned(st["k"]), st["v"].double()
    kp, vp = (torch.zeros(st["k_pages"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    ks, vs = (k / st["k_scale"].double()[:, None], v / st["v_scale"].double()[:, None]) if case["fp8"] else (k, v)
    for b, n in enumerate(_lengths(case)):
        at, end = (int(pos[b, 0]), int(pos[b, 0]) + n) if n else (0, 0)
        while at < end:                             # page by page
            m = min(end, (at // ps + 1) * ps) - at
            rows = slice(b * L + at - int(pos[b, 0]), b * L + at - int(pos[b, 0]) + m)
            for pages, x in ((kp, ks), (vp, vs)):
                pages[table[b][at // ps], :, at % ps: at % ps + m] = x[rows].transpose(0, 1).clamp(-_FP8_MAX, _FP8_MAX) \
                    if case["fp8"] else x[rows].transpose(0, 1)
            at += m
    out = [q * real, k * real, kp, vp]
    return out if case["dense"] else [out[0], kp, vp]

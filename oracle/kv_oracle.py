"""CPU oracle of the paged key / value cache operators, in float64 and from their definitions.  TEST INFRASTRUCTURE ONLY.

Besides the values it gives how far a kernel that works in float32 may be from them before the last rounding, so that a
test can ask for the exactly rounded neighbours: got lies between round(y - slack) and round(y + slack)."""
import math

import torch


def page_of(table, num_pages, page_size, row, pos):
    """The page of a position, or None where the table names none."""
    if pos < 0 or row < 0 or row >= table.shape[0] or pos // page_size >= table.shape[1]:
        return None
    p = int(table[row, pos // page_size])
    return p if 0 <= p < num_pages else None


def attn(q, k_pages, v_pages, table, lens, scale, k_scale=None, v_scale=None):
    """softmax(scale <q, K_j>) V over the positions j < lens[b] whose page is there; zeros where there is none.
    Returns (out, slack) float64 [B, H, hd].

    slack, with w_j the softmax weights and A = sum w_j |V_j| (per output element), n positions:
      scores: float32 sums of hd exact products (hd 2^-24 relative to sum |q k|), two roundings of the factor and one of
        the product (3 * 2^-24 |s|), so a weight is off by a relative d = max_j of that, plus 2^-21 for the power of two
        and its argument's subtraction (|s - max| 2^-24 below 2^-17 where the weight is not negligible, counted there);
        numerator and denominator both carry it: 2 d A
      weights kept as three 16-bit terms: exactly in bf16; in float16 to multiples of 2^-24 where the largest weight is
        2^10 at least, so 2^-35 of it for every value, whatever its weight
      sums over n positions and the join of parts: (n + 64) 2^-24 A, twice (numerator, denominator)"""
    q, table, lens = q.detach().cpu(), table.cpu(), lens.cpu()
    kp, vp = k_pages.detach().cpu(), v_pages.detach().cpu()
    B, H, hd = q.shape
    P, K, ps, _ = kp.shape
    g = H // K
    out, slack = torch.zeros(B, H, hd, dtype=torch.float64), torch.zeros(B, H, hd, dtype=torch.float64)
    for b in range(B):
        n = min(int(lens[b]), table.shape[1] * ps)
        spots = [(page_of(table, P, ps, b, j), j % ps) for j in range(n)]
        spots = [(p, s) for p, s in spots if p is not None]
        if not spots:
            continue
        pages, slots = torch.tensor([p for p, _ in spots]), torch.tensor([s for _, s in spots])
        for h in range(K):
            key, val = kp[pages, h, slots].double(), vp[pages, h, slots].double()
            if k_scale is not None:
                key = key * float(k_scale[h])
            if v_scale is not None:
                val = val * float(v_scale[h])
            x = q[b, h * g:(h + 1) * g].double()
            s = (x @ key.T) * scale
            w = torch.exp(s - s.amax(-1, keepdim=True))
            den = w.sum(-1, keepdim=True)
            out[b, h * g:(h + 1) * g] = w @ val / den
            A = w @ val.abs() / den
            d = (hd * 2.0 ** -24 * (x.abs() @ key.abs().T) * abs(scale)).amax(-1, keepdim=True) \
                + 3 * 2.0 ** -24 * s.abs().amax(-1, keepdim=True) + 2.0 ** -17
            slack[b, h * g:(h + 1) * g] = A * (2 * d + (2 * len(spots) + 128) * 2.0 ** -24)
            if q.dtype == torch.float16:
                slack[b, h * g:(h + 1) * g] += 2.0 ** -35 * val.abs().sum(0) / den
    return out, slack


def rotate(x, pos, turns, interleaved):
    """x [T, H, hd] with each pair as a complex number times exp(2 pi i pos turns).  Returns (y, slack) float64; slack
    counts 2^-21 for cosine and sine (argument and function in float32) and 2^-23 for the two products and their sum,
    relative to |x1| + |x2|."""
    x, pos, turns = x.detach().cpu().double(), pos.cpu().double(), turns.cpu()
    rd = 2 * turns.numel()
    y, slack = x.clone(), torch.zeros_like(x)
    one, two = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    turn = pos[:, None] * turns
    ang = 2 * math.pi * (turn - turn.round())
    z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.ones_like(ang), ang)[:, None]
    y[..., one], y[..., two] = z.real, z.imag
    sl = (x[..., one].abs() + x[..., two].abs()) * (2.0 ** -21 + 2.0 ** -23)
    slack[..., one], slack[..., two] = sl, sl
    return y, slack


def rounded(y, dtype):
    """float64 to the element type, to nearest even in one rounding (e4m3: clamped to +-448 first)."""
    if dtype == torch.float8_e4m3fn:
        y = y.clamp(-448.0, 448.0)
        # nearest multiple of the step 2^(e-3) of y's binade, the smallest step 2^-9: ties to even by torch.round
        step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / step) * step
    bits = {torch.bfloat16: 8, torch.float16: 11}[dtype]
    low = {torch.bfloat16: -126, torch.float16: -14}[dtype]
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** low))) - (bits - 1))
    return torch.round(y / step) * step


def assert_rounds_to(got, y, slack, what=""):
    """Every element of `got` is what y - slack .. y + slack rounds to."""
    g = got.detach().cpu().double()
    lo, hi = rounded(y - slack, got.dtype), rounded(y + slack, got.dtype)
    bad = ~((g >= lo) & (g <= hi))
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements; first at {i}: got {float(g[i])}, value "
                             f"{float(y[i])} +- {float(slack[i])} rounds to {float(lo[i])} .. {float(hi[i])}")

"""Random cases of attn_step and rotary_append over their whole ranges, against the float64 oracle."""
import random

import pytest
import torch

from test_gpu_kv_ops import BF, DEV, F16, append_case, cache, check_attn, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(40))
def test_attention_random(override, seed):
    r = random.Random(seed)
    kv_heads, group = r.choice([1, 1, 2, 3, 5]), r.choice([1, 2, 3, 4, 7, 8, 16, 19])
    hd, page = 8 * r.randint(1, 32), 16 << r.choice([0, 0, 1, 2, 4, 6])
    if r.random() < 0.5:
        hd = r.choice([32, 64, 128, 256])
    B = r.choice([1, 2, 5, 17, 70, 200])
    most = r.choice([1, 40, 300, 3000 if B < 20 else 300])
    lens = [r.randint(0, most) if r.random() < 0.9 else 0 for _ in range(B)]
    dtype, fp8 = r.choice([BF, F16]), r.random() < 0.4
    if r.random() < 0.5:
        override(attn_short=r.randint(0, 1))
    c = cache(seed, lens, kv_heads, hd, page, dtype, fp8)
    q = (r.choice([0.5, 2.0, 6.0]) * torch.randn(B, kv_heads * group, hd, generator=gen(seed))).to(dtype).to(DEV)
    if r.random() < 0.4:                        # some pages that are not there
        for _ in range(3):
            c[2][r.randrange(B), r.randrange(c[2].shape[1])] = r.choice([-1, c[0].shape[0], 2 ** 31 - 1])
    check_attn(q, c, lens, None, f"kv_heads {kv_heads} group {group} hd {hd} page {page} B {B} most {most}")


@pytest.mark.parametrize("seed", range(40))
def test_append_random(seed):
    r = random.Random(1000 + seed)
    kv_heads, heads = r.choice([1, 2, 3, 8]), r.choice([1, 2, 5, 8, 24])
    hd, page, rows = 8 * r.randint(1, 32), 16 << r.choice([0, 0, 1, 3]), r.choice([1, 2, 7, 40])
    rd = r.choice([hd, hd, hd // 2, 2 * r.randint(0, hd // 2)])
    rd -= rd % 2
    per = r.choice([1, 1, 3, 40])
    pos = []
    for _ in range(rows):
        start, n = r.choice([0, r.randint(0, 100), r.randint(0, 5000)]), r.randint(0, per)
        pos += [start + i if i < n else -1 for i in range(per)]
    seq = None
    if r.random() < 0.3:                        # the same rows in another order
        seq = [t // per for t in range(len(pos))]
        order = list(range(len(pos)))
        r.shuffle(order)
        pos, seq = [pos[i] for i in order], [seq[i] for i in order]
    append_case(seed, len(pos), heads, kv_heads, hd, rd, page, r.choice([BF, F16]), r.random() < 0.4, pos, seq, rows,
                r.random() < 0.5, dense=r.random() < 0.5, base=r.choice([1e4, 1e6]), given_out=r.random() < 0.5)

"""The stack's attention blocks on the paged cache: generation, recorded token steps, forks, continuations."""
import pytest
import torch

from oracle import kv_oracle as KO
from vortex_amd import PagedKVCache, attn_step, rotary_append, rotary_turns
from vortex_amd.model import EVO2_7B, RecordedDecodeStep, StripedHyena2

pytestmark = pytest.mark.gpu

CFG = dict(EVO2_7B, hidden_size=128, num_layers=8, num_attention_heads=4, inner_mlp_size=256, hcs_filter_groups=8,
           hcm_filter_groups=8, hcl_filter_groups=128)


def model(**kw):
    return StripedHyena2(dict(CFG, **kw), seed=5, device="cuda").to_inference("cuda")


def tokens(B, L, seed=6):
    return torch.randint(0, 512, (B, L), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def near(got, want):
    # bf16 GEMM and SDPA paths differ between prefill, dense and paged decode: the bound of the dense cache's own tests
    err = (got.float() - want.float()).abs().max() / want.float().abs().max()
    assert err <= 3e-2, err


@pytest.mark.parametrize("L,page,factor", [(256, 64, 1.0), (203, 16, 1.0), (203, 64, 8.0), (1, 16, 1.0)])
def test_paged_generation_matches_a_longer_prefill(L, page, factor):
    m, n = model(rotary_emb_scaling_factor=factor), 6
    ids = tokens(2, L + n)
    want = m(ids)[:, L - 1:L + n - 1]
    toks, scores = m.generate(ids[:, :L], n, forced=ids[:, L:], kv="paged", page_size=page)
    assert torch.equal(toks, ids[:, L:])
    if L > 1:       # a prompt shorter than the filters follows the reference's growing caches, not a longer prefill
        near(scores, want)
    near(scores, m.generate(ids[:, :L], n, forced=ids[:, L:])[1])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("L", [256, 203])
def test_recorded_paged_step_matches_eager(L, fp8):
    # pages of 16: the recorded step crosses page ends; the same kernels on the same data
    m, n = model(), 40
    ids = tokens(2, L + n, 8)
    kw = dict(forced=ids[:, L:], kv="paged", page_size=16, fp8=fp8)
    _, eager = m.generate(ids[:, :L], n, **kw)
    _, rec = m.generate(ids[:, :L], n, graph=True, **kw)
    assert bool(eager.isfinite().all()) and torch.equal(rec, eager)
    if not fp8:
        near(eager, m.generate(ids[:, :L], n, forced=ids[:, L:])[1])


@pytest.mark.parametrize("kv", ["dense", "paged"])
@pytest.mark.parametrize("graph", [False, True])
def test_forked_continuations_match_their_own_generation(kv, graph):
    # three continuations behind each of two prompts that end inside a page, run once and forked
    m, L, n, S = model(), 203, 12, 3
    prompt, cont = tokens(2, L, 1), tokens(2 * S, n, 2)
    toks, got = m.generate(prompt, n, forced=cont, kv=kv, page_size=64, samples=S, graph=graph)
    assert torch.equal(toks, cont)
    _, want = m.generate(prompt.repeat_interleave(S, 0), n, forced=cont)
    near(got, want)
    free, _ = m.generate(prompt, 3, kv=kv, samples=S)       # greedy: equal prompts, equal continuations
    assert torch.equal(free[0], free[2]) and free.shape == (2 * S, 3)


def test_a_stack_without_attention_takes_the_paged_keyword():
    m, ids = model(pattern=("hcs", "hcm", "hcl"), num_layers=3), tokens(2, 150)
    _, want = m.generate(ids, 8, forced=ids[:, :8])
    _, got = m.generate(ids, 8, forced=ids[:, :8], kv="paged", graph=True)
    assert torch.equal(got, want)


def test_model_refusals():
    m = model(num_layers=4)
    ids = tokens(2, 40)
    ipd = m.initialize_inference_params(50, kv="paged", rows=2, page_size=16)
    m(ids, ipd)
    for rows in ([], [2], [-1], [0, 5]):
        with pytest.raises(ValueError):
            m.select_inference_params(ipd, rows)
    for kw in (dict(fp8=True), dict(kv="other"), dict(samples=0), dict(kv="paged", page_size=20), dict(kv="paged", page_size=0)):
        with pytest.raises(ValueError):
            m.generate(ids, 2, **kw)
    with pytest.raises(TypeError):              # a model that was not brought to bfloat16
        StripedHyena2(dict(CFG, num_layers=4), device="cuda").initialize_inference_params(50, kv="paged")


@pytest.mark.parametrize("fp8", [False, True])
def test_dense_rows_of_a_paged_cache(fp8):
    c = PagedKVCache(2, 3, 40, 12, 100, page_size=16, fp8=fp8)
    c.add(3)
    c.extend([50, 0, 17])
    c.pools.copy_(torch.randn(c.pools.shape, device="cuda").mul(4).to(c.pools.dtype))
    c.pools[:, c._free] = float("nan")                      # free pages, and a page's slots behind its sequence's end
    c.pools[:, c._pages[0][3], :, 2:] = float("nan")
    if fp8:
        c.scales.copy_(0.1 + torch.rand(c.scales.shape, device="cuda"))
    for side, x in enumerate(c.dense(1)):
        assert x.shape == (3, 3, 50, 40) and x.dtype == torch.bfloat16
        for r, n in enumerate(c.lengths()):
            assert not x[r, :, n:].any()
            for p in range(n):
                want = c.pools[2 + side, c._pages[r][p // 16], :, p % 16].double()
                if fp8:
                    want = want * c.scales[2 + side].double()[:, None]
                KO.assert_rounds_to(x[r, :, p], want.cpu(), want.abs().cpu() * 2.0 ** -24)


@pytest.mark.parametrize("n", [2, 32, 33, 60])
def test_longer_continuation_on_a_paged_cache(n):
    m, L = model(pattern=("attn",), num_layers=2), 100
    ids = tokens(2, L + n, 3)
    want = m(ids)[:, L:]
    ipd = m.initialize_inference_params(L + n, kv="paged", rows=2, page_size=16)
    m(ids[:, :L], ipd)
    near(m(ids[:, L:], ipd), want)
    with pytest.raises(ValueError):
        m(ids[:, :1], ipd)                                  # the cache is full
    with pytest.raises(ValueError):
        m(ids[:1, :1], ipd)


def test_selected_sequences_go_on():
    m, L, n = model(), 200, 8
    ids = tokens(3, L + n, 4)
    _, want = m.generate(ids[:, :L], n, forced=ids[:, L:])
    with torch.no_grad():
        ipd = m.initialize_inference_params(L + n, kv="paged", rows=3, page_size=32)
        m(ids[:, :L], ipd)
        rows, rec = [0, 1, 2], None
        for i in range(1, n):
            for p in ipd.values():
                p.seqlen_offset = L if p.seqlen_offset == 0 else p.seqlen_offset + 1
            if i == 3:                                      # reordered, one dropped, pages moved to the lowest ids
                m.select_inference_params(ipd, [2, 0])
                rows = [2, 0]
                cache = ipd["mha"].cache
                assert cache.compact() == 2 * 7 and cache.free_pages == 7
            if i == 4:
                rec = RecordedDecodeStep(m, ipd, 2)
                for call in (cache.compact, lambda: m.select_inference_params(ipd, [0, 0])):
                    with pytest.raises(RuntimeError, match="recorded"):
                        call()
            if i == 6:
                rec.release()
                rec = None
                cache.resize(16)                            # new pools; eager steps go on
            x = ids[rows, L + i - 1:L + i]
            got = (m(x, ipd) if rec is None else rec(x))[:, -1]
            near(got, want[rows, i])


def test_a_recording_that_finds_no_pages_leaves_the_caches_usable():
    m, L, n = model(), 200, 6
    ids = tokens(2, L + n, 4)
    _, want = m.generate(ids[:, :L], n, forced=ids[:, L:])
    with torch.no_grad():
        ipd = m.initialize_inference_params(4 * L, kv="paged", rows=2, page_size=16, num_pages=2 * 14)
        m(ids[:, :L], ipd)
        for i in range(1, n):
            for p in ipd.values():
                p.seqlen_offset = L if p.seqlen_offset == 0 else p.seqlen_offset + 1
            if i == 3:
                with pytest.raises(RuntimeError, match="pages needed"):
                    RecordedDecodeStep(m, ipd, 2)
            near(m(ids[:, L + i - 1:L + i], ipd)[:, -1], want[:, i])


def test_two_recorded_caches_in_turn_and_at_once():
    # two graphs of the same shapes replayed on two streams: nothing of one call is shared with another
    B, H, hd, page, W = 4, 8, 128, 64, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    turns = rotary_turns(hd, device="cuda")
    sets = []
    for i in range(2):
        c = PagedKVCache(1, 2, hd, B * W, W * page, page_size=page)
        c.add(B)
        c.extend([3000 - 100 * i, 17, 900, 2049])
        c.pools.normal_(generator=g)
        c.record(10)
        x = torch.randn(B, H + 4, hd, device="cuda", generator=g).bfloat16()
        sets.append((c, x, torch.cuda.CUDAGraph()))

    def step(c, x):
        q, k, v = x.split([H, 2, 2], dim=1)
        pos = c.step()
        return attn_step(rotary_append(q, k, v, pos, turns, *c.layer(0), c.table), *c.layer(0), c.table, c.lens)

    outs, want = [], []
    for c, x, graph in sets:
        lens, pools = c.lens.clone(), c.pools.clone()
        want.append([step(c, x).clone() for _ in range(4)])
        c.lens.copy_(lens)
        c.pools.copy_(pools)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(step(c, x))
        assert torch.equal(c.lens, lens)                    # capturing runs nothing
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for t in range(4):
        for i, (c, x, graph) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                graph.replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in range(2):
        for t in range(4):
            assert torch.equal(got[i][t], want[i][t]), (i, t)

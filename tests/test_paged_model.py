"""The paged cache and attention sinks in the package's own paths: the attention module, the model, generate(),
generate_batch() and the graph decoder, on the torch path (CPU) and on the kernels."""

from __future__ import annotations

import math

import pytest
import torch

import oracle
from sleuth_amd.attention import Attention, causal_mask
from sleuth_amd.config import ModelConfig
from sleuth_amd.generate import GraphDecoder, generate, generate_batch
from sleuth_amd.kv_cache import KVCache
from sleuth_amd.model import Transformer
from sleuth_amd.paged_cache import PagedKVCache
from sleuth_amd.rope import rope_tables

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def config(sliding=False, sinks=0, **kw):
    base = dict(vocab_size=64, d_model=64, n_layers=2, n_heads=4, head_size=32, n_kv_heads=2, qk_norm=True, max_seq_len=128,
                init_std=0.2)
    if sliding:
        base.update(layer_types=["sliding", "sliding"], sliding_window=20, sink_tokens=sinks)
    return ModelConfig(**{**base, **kw})


def model(cfg, device="cpu", dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return Transformer(cfg).to(device=device, dtype=dtype).eval()


# ---------------------------------------------------------------- configuration and masks
def test_config_takes_sink_tokens_only_beside_windows():
    assert config(True, 4).attn_spec(0).sinks == 4
    assert config().attn_spec(0).sinks == 0
    mixed = config(True, 4, layer_types=["sliding", "full"])
    assert [mixed.attn_spec(i).sinks for i in range(2)] == [4, 0]
    for bad in (dict(sink_tokens=3), dict(sliding=True, sinks=-1)):
        with pytest.raises(ValueError, match="sink_tokens"):
            config(**bad)


def test_a_host_spec_without_sinks_works():
    """The host's own AttnSpec has no such field."""
    class Spec:
        kind, head_dim, kv_heads, rope_theta, window, v_from_k = "sliding", 32, 2, 1e4, 20, False

    class Cfg:
        n_heads, attn_scale, norm_eps, pos_type, rope_dim, d_model = 4, 0.0, 1e-6, "rope", 0, 64
        qkv_bias = bias = qk_norm = v_norm = False

        def attn_spec(self, i):
            return Spec

    assert Attention(Cfg(), 0).sinks == 0


def test_mask_with_sinks():
    m = causal_mask(3, 12, 9, 4, "cpu", sinks=2)
    assert [row.nonzero().flatten().tolist() for row in m] == [[0, 1, 6, 7, 8, 9], [0, 1, 7, 8, 9, 10], [0, 1, 8, 9, 10, 11]]
    assert torch.equal(causal_mask(3, 12, 9, 4, "cpu", 0), causal_mask(3, 12, 9, 4, "cpu"))
    assert torch.equal(causal_mask(3, 12, 9, 0, "cpu", 5), causal_mask(3, 12, 9, 0, "cpu"))


# ---------------------------------------------------------------- the cache's book-keeping
def cache_of(batch=3, max_len=100, page=16, pages=12, device="cpu"):
    return PagedKVCache([(2, 32)], batch, max_len, device, torch.float32, page, pages)


def test_pages_are_handed_out_and_come_back():
    c = cache_of()
    c.set_new([17, 0, 5])
    c.reserve(20)
    c.reserve(20)   # (another layer of the same pass)
    assert c.free_pages == 12 - 3 and c.top(20) == 17
    c.advance(20)
    assert c.seq_lens_host == [17, 0, 5] and c.seq_lens.tolist() == [17, 0, 5] and c.pos == 17
    ids = c.page_table[c.page_table >= 0].tolist()
    assert len(set(ids)) == 3
    c.set_new(None)
    c.reserve(1)
    c.advance(1)
    assert c.seq_lens.tolist() == [18, 1, 6] and c.free_pages == 8
    c.release(0)
    assert c.free_pages == 10 and c.seq_lens.tolist() == [0, 1, 6] and not (c.page_table[0] >= 0).any()
    c.reset()
    assert c.free_pages == 12 and c.pos == 0 and c.new_lens is None


def test_a_full_cache_raises_and_hands_nothing_out():
    c = cache_of(pages=3)
    c.set_new([16, 16, 17])
    with pytest.raises(ValueError, match="out of pages"):
        c.reserve(17)
    assert c.free_pages == 3 and not (c.page_table >= 0).any()
    c.set_new([101, 0, 0])
    with pytest.raises(ValueError, match="KV cache full"):
        c.reserve(101)
    for bad in ([1, 2], [1, -1, 0]):
        with pytest.raises(ValueError, match="new_lens"):
            c.set_new(bad)
    for kw in (dict(page=8), dict(page=20), dict(batch=0), dict(pages=0)):
        with pytest.raises(ValueError):
            cache_of(**kw)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 1), (20, 16), (20, 17), (33, 40)])
def test_release_unseen_gives_back_exactly_what_no_later_query_sees(window, sinks):
    c = cache_of(batch=2, max_len=200, pages=40)
    c.set_new([150, 33])
    c.reserve(150)
    c.advance(150)
    before = c.page_table.clone()
    n = c.release_unseen(window, sinks)
    gone = 0
    for b, r in enumerate((150, 33)):
        for j in range(-(-r // 16)):
            # (a page's later slots count: the next tokens go there)
            seen = any(s < sinks or s > r - window for s in range(16 * j, 16 * j + 16))
            assert (c.page_table[b, j] >= 0) == seen, (b, j)
            gone += not seen
            if seen:
                assert c.page_table[b, j] == before[b, j]
    assert n == gone and c.free_pages == 40 - 10 - 3 + gone
    assert c.release_unseen(window, sinks) == 0
    with pytest.raises(ValueError):
        c.release_unseen(0)


@pytest.mark.parametrize("device", DEVICES)
def test_update_and_row(device):
    c = cache_of(device=device)
    g = torch.Generator().manual_seed(0)
    kept = [torch.zeros(2, 0, 32) for _ in range(3)]
    for new in ([17, 0, 5], [1, 3, 30], [15, 1, 0]):
        T = max(new)
        k = torch.randn(3, 2, T, 32, generator=g).to(device)
        c.set_new(new)
        c.update(0, k, 2 * k)
        for b, n in enumerate(new):
            kept[b] = torch.cat([kept[b], k[b, :, :n].cpu()], 1)
        c.advance(T)
    for b, want in enumerate(kept):
        kb, vb, held = c.row(0, b, want.shape[1])
        assert held.all() and torch.equal(kb.cpu(), want) and torch.equal(vb.cpu(), 2 * want)
    c.release_unseen(3, 0)
    kb, vb, held = c.row(0, 0, 33)
    assert held.tolist() == [False] * 16 + [True] * 17 and not kb[:, :16].any() and torch.equal(kb[:, 16:].cpu(), kept[0][:, 16:])


# ---------------------------------------------------------------- the module
def module_and_inputs(cfg, dtype, device, B, T, past, seed=0):
    torch.manual_seed(seed)
    att = Attention(cfg, 0).to(device=device, dtype=dtype).eval()
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, past + T, cfg.d_model, generator=g).to(device=device, dtype=dtype)
    cos, sin = (t.to(device) for t in rope_tables(cfg.head_dim, cfg.max_seq_len, cfg.rope_theta))
    return att, x, cos, sin


def oracle_layer(att, x, cos, sin, window, sinks):
    """The layer over the whole sequence at once, float64 on the CPU."""
    x = x.cpu().double()
    B, S, _ = x.shape
    H, K, hd = att.n_heads, att.n_kv, att.hd
    lin = lambda m: x @ m.weight.detach().cpu().double().T   # noqa: E731
    q, k, v = (lin(m).view(B, S, -1, hd).transpose(1, 2) for m in (att.q_proj, att.k_proj, att.v_proj))
    if att.q_norm is not None:
        nrm = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + att.eps) * w.detach().cpu().double()   # noqa: E731
        q, k = nrm(q, att.q_norm.weight), nrm(k, att.k_norm.weight)
    c, s = cos[:S].cpu().double(), sin[:S].cpu().double()
    rot = lambda t: t * c + torch.cat([-t[..., hd // 2:], t[..., :hd // 2]], -1) * s   # noqa: E731
    q, k = rot(q), rot(k)
    rep = H // K
    w = (q @ k.repeat_interleave(rep, 1).transpose(-1, -2)) * att.scale
    pos = torch.arange(S)
    see = pos[None] <= pos[:, None]
    if window:
        see &= (pos[None] > pos[:, None] - window) | (pos[None] < sinks)
    y = w.masked_fill(~see, -math.inf).softmax(-1) @ v.repeat_interleave(rep, 1)
    return y.transpose(1, 2).reshape(B, S, H * hd) @ att.o_proj.weight.detach().cpu().double().T


def rel(got, want):
    got = got.detach().cpu().double()
    return ((got - want).norm() / want.norm()).item()


# a layer's projections, norms and attention, each rounded to the type once or twice: a few half steps of it in 2-norm
# (eps/2 each, of which about ten meet at the output); fp32: 2^-24 over sums of some hundred terms
REL = {torch.float32: 1e-5, torch.bfloat16: 10 * 2 ** -8, torch.float16: 10 * 2 ** -11}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sliding,sinks", [(False, 0), (True, 0), (True, 3), (True, 30)])
@pytest.mark.parametrize("hd", [32, 64])
@torch.no_grad()
def test_module_on_a_paged_cache(device, dtype, sliding, sinks, hd):
    """A prompt in ragged chunks, then single tokens, over pages: each row equals the whole-sequence layer."""
    if device == "cpu" and dtype == torch.float16:
        pytest.skip("fp16 products on the CPU")
    cfg = config(sliding, sinks, head_size=hd)
    B, S = 3, 75
    att, x, cos, sin = module_and_inputs(cfg, dtype, device, B, S, 0)
    want = oracle_layer(att, x, cos, sin, cfg.sliding_window, sinks)
    c = PagedKVCache([(2, hd)], B, 128, device, dtype, 16, 20)
    done = [0] * B
    for new in ([17, 0, 40], [1, 33, 1], [20, 20, 0], [1, 1, 1], [0, 1, 1], [30, 2, 9]):
        T = max(new)
        xs = torch.zeros(B, T, cfg.d_model, device=device, dtype=dtype)
        for b, n in enumerate(new):
            xs[b, :n] = x[b, done[b]:done[b] + n]
        at = (torch.tensor(done)[:, None] + torch.arange(T)).clamp(max=127).to(device)
        c.set_new(new)
        y = att(xs, cos[at], sin[at], c)
        c.advance(T)
        for b, n in enumerate(new):
            if n:
                assert rel(y[b, :n], want[b, done[b]:done[b] + n]) < REL[dtype], (new, b)
            assert not y[b, n:].any()
            done[b] += n
        if sliding:
            c.release_unseen(cfg.sliding_window, sinks)
    assert att.last_path == ("hip-paged" if device == "cuda" else "torch")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,sinks", [(32, 3), (64, 25), (128, 4)])
@torch.no_grad()
def test_module_with_sinks_on_the_contiguous_cache(device, dtype, hd, sinks):
    """Without a cache, in chunks, verify steps and single tokens, and with per-row lengths."""
    cfg = config(True, sinks, head_size=hd)
    B, S = 2, 80
    att, x, cos, sin = module_and_inputs(cfg, dtype, device, B, S, 0)
    want = oracle_layer(att, x, cos, sin, cfg.sliding_window, sinks)
    path = "hip-sinks" if device == "cuda" else "torch"
    assert rel(att(x, cos[:S], sin[:S]), want) < REL[dtype] and att.last_path == path
    cache = KVCache([(2, hd)], B, 128, device, dtype)
    at = 0
    for T in (40, 1, 5, 1, 20, 13):
        y = att(x[:, at:at + T], cos[at:at + T], sin[at:at + T], cache)
        cache.advance(T)
        assert rel(y, want[:, at:at + T]) < REL[dtype] and att.last_path == path
        at += T
    cache.set_lengths([70, 33])   # a step with each row at its own length
    pos = torch.tensor([70, 33])
    rows = torch.stack([x[0, 70:72], x[1, 33:35]])
    at = (pos[:, None] + torch.arange(2)).to(device)
    y = att(rows, cos[at], sin[at], cache)
    for b, p in enumerate(pos.tolist()):
        assert rel(y[b], want[b, p:p + 2]) < REL[dtype]


@pytest.mark.parametrize("device", DEVICES)
@torch.no_grad()
def test_paged_module_keeps_the_taps_and_refuses_document_masks(device):
    from sleuth_amd.taps import listen, name_taps

    cfg = config()
    att, x, cos, sin = module_and_inputs(cfg, torch.float32, device, 2, 20, 0)
    name_taps(att)
    want = oracle_layer(att, x, cos, sin, 0, 0)
    at = torch.arange(20, device=device).expand(2, 20)
    for tap in ("tap_q", "tap_pattern"):
        seen = []
        c = PagedKVCache([(2, 32)], 2, 128, device, torch.float32, 16)
        name = getattr(att, tap).name
        with listen(att, {name: lambda _, t: seen.append(t)}):
            y = att(x, cos[at], sin[at], c)
        assert seen and rel(y, want) < 1e-5
    c = PagedKVCache([(2, 32)], 2, 128, device, torch.float32, 16)
    with pytest.raises(NotImplementedError):
        att(x, cos[at], sin[at], c, same_doc=torch.ones(2, 1, 20, 20, dtype=torch.bool, device=device))


# ---------------------------------------------------------------- whole models
PROMPTS = [[1, 2, 3], list(range(40)), [7] * 17, [5]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sliding,sinks", [(False, 0), (True, 0), (True, 3)])
@pytest.mark.parametrize("chunk", [8, 64])
def test_generate_batch_equals_generate(device, sliding, sinks, chunk):
    """fp32, greedy: each prompt of the batch gives the tokens that it gives alone."""
    m = model(config(sliding, sinks), device)
    alone = [generate(m, p, 15).new_ids for p in PROMPTS]
    batch = generate_batch(m, PROMPTS, 15, chunk=chunk, page_size=16)
    assert [r.new_ids for r in batch] == alone
    assert [r.prompt_ids for r in batch] == PROMPTS
    assert all(r.stop_reason == "max_new_tokens" for r in batch)


@pytest.mark.parametrize("device", DEVICES)
def test_generate_batch_in_a_small_pool(device):
    """Windows of 20 with 3 first tokens: rows grow to the model's length in a pool that could not hold them whole."""
    m = model(config(True, 3), device)
    batch = generate_batch(m, PROMPTS, 500, chunk=16, page_size=16, n_pages=4 * 5)
    assert [r.stop_reason for r in batch] == ["context_full"] * 4
    assert [len(r.prompt_ids) + len(r.new_ids) for r in batch] == [129] * 4
    assert batch[0].stats["most_pages"] <= 20
    assert [r.new_ids for r in batch] == [generate(m, p, 500).new_ids for p in PROMPTS]
    with pytest.raises(ValueError, match="out of pages"):
        generate_batch(model(config(), device), PROMPTS, 500, chunk=16, page_size=16, n_pages=12)


def test_generate_batch_arguments():
    m = model(config())
    one = generate(m, [3, 4], 20).new_ids
    stop = one[5]
    r = generate_batch(m, [[3, 4], [9]], 20, stop_ids={stop})
    assert r[0].new_ids == one[:one.index(stop) + 1] and r[0].stop_reason == "stop_token"
    assert generate_batch(m, [[3]], 0)[0].new_ids == []
    for bad in ([], [[1], []]):
        with pytest.raises(ValueError, match="at least one token"):
            generate_batch(m, bad)
    with pytest.raises(ValueError, match="chunk"):
        generate_batch(m, [[1]], chunk=0)
    assert len(generate_batch(m, [[1], [2]], 4, temperature=1.0, seed=3)[1].new_ids) == 4


@pytest.mark.gpu
@torch.no_grad()
def test_graph_decoder_with_sinks():
    """The recorded step of a model with first tokens replays as the eager one computes."""
    m = model(config(True, 3, head_size=64), "cuda", torch.bfloat16)
    prompt = torch.randint(64, (1, 50), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    dec = GraphDecoder(m, 128, torch.bfloat16)
    eager = KVCache.for_model(m, 1, 128, torch.bfloat16)
    m(prompt, cache=dec.cache)
    m(prompt, cache=eager)
    tok = torch.tensor([9], device="cuda")
    for i in range(8):
        a = dec.step(tok).clone()
        b = m(tok.view(1, 1), cache=eager).logits[:, -1]
        assert torch.allclose(a.float(), b.float(), atol=0.05, rtol=0.05)
        tok = b.argmax(-1)
    assert dec.replays == 8


@pytest.mark.gpu
@torch.no_grad()
def test_a_served_batch_in_bf16():
    """A run of the operators together: chunks of four prompts, then decode steps, the logits of every pass near those of
    the float32 torch path on the same weights (bf16: some forty roundings of half a step over two layers, in 2-norm)."""
    cfg = config(True, 4, head_size=128, sliding_window=40, max_seq_len=256)
    m = model(cfg, "cuda", torch.bfloat16)
    ref = model(cfg)
    ref.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    c, d = (PagedKVCache.for_model(x, 4, 256, None, 16, 40) for x in (m, ref))
    g = torch.Generator().manual_seed(2)
    for new in ([64, 10, 0, 33], [64, 0, 5, 64], [1, 1, 1, 1], [1, 0, 1, 1], [20, 1, 30, 2]):
        ids = torch.randint(64, (4, max(new)), generator=g)
        outs = []
        for x, cache, dev in ((m, c, "cuda"), (ref, d, "cpu")):
            cache.set_new(new)
            outs.append(x(ids.to(dev), cache=cache).logits.float().cpu())
            cache.release_unseen(40, 4)
        for b, n in enumerate(new):
            if n:
                a, w = outs[0][b, :n], outs[1][b, :n]
                assert ((a - w).norm() / w.norm()).item() < 40 * 2 ** -8
    assert c.free_pages == d.free_pages and c.seq_lens.tolist() == d.seq_lens_host


def test_gated_attention_refuses_a_paged_cache():
    """Its paths read cache.k[layer] as [B, K, max_len, hd]: a pool of pages must not get there."""
    from types import SimpleNamespace

    from sleuth_amd.gated import GatedAttention

    m = GatedAttention(SimpleNamespace(n_heads=4, n_kv_heads=2, head_dim=32, n_rot=32, norm_eps=1e-6), 0)
    cache = PagedKVCache([(2, 32)], 1, 32, "cpu", torch.float32)
    with pytest.raises(NotImplementedError, match="paged"):
        m(torch.zeros(1, 1, 16), torch.ones(1, 32), torch.zeros(1, 32), cache)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@torch.no_grad()
def test_a_sink_layers_verify_rows_are_its_decodes(hd):
    """bf16: a verify step over the contiguous cache attends as the single tokens do, bit for bit; so does a recorded
    step, whose bound is the cache's length."""
    cfg = config(True, 3, head_size=hd, max_seq_len=512, sliding_window=90)
    att, x, cos, sin = module_and_inputs(cfg, torch.bfloat16, "cuda", 1, 300, 0)
    rows = {}
    for T in (1, 5):
        cache = KVCache([(2, hd)], 1, 512, "cuda", torch.bfloat16)
        att(x[:, :200], cos[:200], sin[:200], cache)
        cache.advance(200)
        rows[T] = []
        for at in range(200, 300, T):
            rows[T].append(att(x[:, at:at + T], cos[at:at + T], sin[at:at + T], cache))
            cache.advance(T)
    assert torch.equal(torch.cat(rows[1], 1), torch.cat(rows[5], 1))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,k", [(64, 4), (128, 3), (32, 8)])
@torch.no_grad()
def test_speculative_and_recorded_decoding_with_sinks_equal_plain_greedy(hd, k):
    from sleuth_amd.generate import speculative_generate

    m = model(config(True, 3, head_size=hd, max_seq_len=256, sliding_window=40), "cuda", torch.bfloat16)
    prompt = torch.randint(64, (70,), generator=torch.Generator().manual_seed(4)).tolist()
    plain = generate(m, prompt, 150).new_ids
    assert generate(m, prompt, 150, cuda_graph=True).new_ids == plain
    for graph in (False, True):
        assert speculative_generate(m, prompt, 150, k=k, cuda_graph=graph).new_ids == plain


@pytest.mark.parametrize("device", DEVICES)
def test_a_short_pool_keeps_the_rows_results(device):
    """A row ends, the other two outgrow the pool: what the finished one has is in the error, and what they have so far."""
    from sleuth_amd.paged_cache import OutOfPages

    m = model(config(), device)
    prompts = [[1, 2, 3], list(range(40)), [5] * 125]
    alone = [generate(m, p, 500) for p in prompts]
    with pytest.raises(OutOfPages, match="out of pages") as e:
        generate_batch(m, prompts, 500, chunk=125, page_size=16, n_pages=8 + 3 + 2)
    got = e.value.results
    assert [r.prompt_ids for r in got] == prompts
    assert got[2].stop_reason == alone[2].stop_reason == "context_full" and got[2].new_ids == alone[2].new_ids
    for r, a in zip(got[:2], alone):
        assert r.stop_reason == "out_of_pages" and len(r.new_ids) > 10 and r.new_ids == a.new_ids[:len(r.new_ids)]
    assert got[0].stats["passes"] > 0


def test_a_prompt_past_the_models_length_is_refused_before_any_pass():
    m = model(config())
    m.forward = None   # (no pass)
    with pytest.raises(ValueError, match="exceeds max_seq_len"):
        generate_batch(m, [[1], [2] * 129], 4)


@pytest.mark.gpu
@pytest.mark.parametrize("sliding,sinks", [(False, 0), (True, 3)])
@torch.no_grad()
def test_a_recorded_layer_over_pages_sees_the_rows_grow(sliding, sinks):
    """Recorded at 19 and 5 tokens, replayed up to 100: reserve before each replay, advance after it."""
    cfg = config(sliding, sinks, head_size=64)
    att, x, cos, sin = module_and_inputs(cfg, torch.bfloat16, "cuda", 2, 100, 0)
    want = oracle_layer(att, x, cos, sin, cfg.sliding_window, sinks)
    cache = PagedKVCache([(2, 64)], 2, 128, "cuda", torch.bfloat16, 16)
    cache.set_new([19, 5])
    at = torch.arange(19, device="cuda")[None]
    att(x[:, :19], cos[at], sin[at], cache)
    cache.advance(19)
    cache.set_new(None)
    step, c, s = x[:, 19:20].clone(), cos[:1].repeat(2, 1, 1), sin[:1].repeat(2, 1, 1)
    cache.reserve(1)
    att(step, c, s, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = att(step, c, s, cache)
        with pytest.raises(RuntimeError, match="advance"):
            cache.advance(1)
        with pytest.raises(RuntimeError, match="reserve"):
            cache.reserve(60)
    assert cache.seq_lens_host == [19, 5] == cache.seq_lens.tolist()
    for _ in range(81):
        rows = cache.seq_lens_host
        cache.reserve(1)
        step.copy_(torch.stack([x[b, n:n + 1] for b, n in enumerate(rows)]))
        c.copy_(cos[rows][:, None])
        s.copy_(sin[rows][:, None])
        graph.replay()
        cache.advance(1)
        for b, n in enumerate(rows):
            assert rel(y[b], want[b, n:n + 1]) < REL[torch.bfloat16], (rows, b)


@pytest.mark.gpu
@torch.no_grad()
def test_a_whole_models_pass_over_pages_is_not_recorded():
    m = model(config(), "cuda", torch.bfloat16)
    cache = PagedKVCache.for_model(m, 1, 128, None, 16)
    ids = torch.tensor([[3]], device="cuda")
    m(ids, cache=cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="advance"):
            m(ids, cache=cache)
    torch.cuda.synchronize()
    assert cache.seq_lens_host == [1] == cache.seq_lens.tolist()


# ---------------------------------------------------------------- rewinding
def test_rewind_gives_back_the_pages_behind_the_new_end():
    c = cache_of()
    c.set_new([40, 17, 3])
    c.reserve(40)
    c.advance(40)
    assert c.free_pages == 12 - 3 - 2 - 1
    table = c.page_table.clone()
    c.rewind([32, 17, 0])
    assert c.seq_lens_host == [32, 17, 0] == c.seq_lens.tolist() and c.free_pages == 12 - 2 - 2 and c.pos == 32
    assert torch.equal(c.page_table[0, :2], table[0, :2]) and not (c.page_table[0, 2:] >= 0).any()
    for bad in ([33, 0, 0], [1, 1], [-1, 0, 0]):
        with pytest.raises(ValueError, match="rewind"):
            c.rewind(bad)
    c.set_new([1, 0, 20])
    c.reserve(20)
    c.advance(20)
    assert c.seq_lens_host == [33, 17, 20] and c.free_pages == 12 - 3 - 2 - 2
    ids = c.page_table[c.page_table >= 0].tolist()
    assert len(set(ids)) == len(ids) == 7


@pytest.mark.parametrize("window,sinks", [(20, 0), (17, 5), (33, 16)])
def test_rewind_stops_where_a_page_that_is_gone_would_be_seen(window, sinks):
    for n in range(60, 100):
        c = cache_of(batch=1, max_len=200, pages=13)
        c.set_new([100])
        c.reserve(100)
        c.advance(100)
        c.release_unseen(window, sinks)
        seen = [s for s in range(n) if s < sinks or s > n - window]   # of the next query, at n
        whole = all(c.page_table[0, s // 16] >= 0 for s in seen)
        if whole:
            c.rewind([n])
            assert c.seq_lens_host == [n]
        else:
            with pytest.raises(ValueError, match="given back"):
                c.rewind([n])
            assert c.seq_lens_host == [100] and c.seq_lens.tolist() == [100]
    c = cache_of(batch=1, max_len=200, pages=13)
    c.set_new([100])
    c.reserve(100)
    c.advance(100)
    c.release_unseen(window, sinks)
    c.release(0)
    assert c.free_pages == 13
    c.set_new([9])
    c.reserve(9)
    c.advance(9)
    c.rewind([2])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sliding,sinks", [(False, 0), (True, 3)])
@torch.no_grad()
def test_verify_steps_over_pages(device, sliding, sinks):
    """Guesses, some of them right, verified four tokens at a time for three rows, the rejected ones dropped: each row's
    tokens are those of generate()."""
    m = model(config(sliding, sinks), device)
    prompts, n = PROMPTS[:3], 25
    alone = [generate(m, p, n).new_ids for p in prompts]
    cache = PagedKVCache.for_model(m, 3, 128, None, 16, 24)
    new = [list(p) for p in prompts]
    cache.set_new([len(p) for p in new])
    T = max(map(len, new))
    logits = m(torch.tensor([p + [0] * (T - len(p)) for p in new], device=device), cache=cache).logits
    out = [[int(logits[b, len(p) - 1].argmax())] for b, p in enumerate(new)]
    cache.set_new(None)
    steps = 0
    while min(map(len, out)) < n:
        at = cache.seq_lens_host
        rows = []
        for b, x in enumerate(out):   # right guesses, but for every third token
            ahead = [t if (len(x) + i) % 3 else (t + 1) % 64 for i, t in enumerate((alone[b] + [0] * 8)[len(x):len(x) + 3])]
            rows.append([x[-1]] + (ahead + [0] * 3)[:3])
        choice = m(torch.tensor(rows, device=device), cache=cache).logits.argmax(-1).tolist()
        keep = []
        for b, (row, c) in enumerate(zip(rows, choice)):
            ok = next((i for i in range(3) if c[i] != row[1 + i]), 3)
            out[b] += row[1:1 + ok] + [c[ok]]
            keep.append(at[b] + 1 + ok)
        cache.rewind(keep)
        if sliding:
            cache.release_unseen(20, sinks)
        steps += 1
    assert [x[:n] for x in out] == alone and steps < n


@pytest.mark.parametrize("device", DEVICES)
@torch.no_grad()
def test_torch_path_over_pages_hides_no_nan_and_takes_none_from_unseen_keys(device, monkeypatch):
    monkeypatch.setenv("SLEUTH_AMD_NO_HIP", "1")
    cfg = config(True, 3)
    att, x, cos, sin = module_and_inputs(cfg, torch.float32, device, 1, 61, 0)
    want = oracle_layer(att, x, cos, sin, 20, 3)
    at = torch.arange(61, device=device)[None]

    def last(poison):
        c = PagedKVCache([(2, 32)], 1, 128, device, torch.float32, 16)
        att(x[:, :60], cos[at[:, :60]], sin[at[:, :60]], c)
        c.advance(60)
        for pos in poison:
            for pool in (c.k[0], c.v[0]):
                pool[c.page_table[0, pos // 16], :, pos % 16] = math.nan
        return att(x[:, 60:], cos[at[:, 60:]], sin[at[:, 60:]], c)

    assert rel(last([3, 20, 40]), want[:, 60:]) < REL[torch.float32]   # between the first tokens and the window
    assert last([41]).isnan().all() and last([2]).isnan().all()

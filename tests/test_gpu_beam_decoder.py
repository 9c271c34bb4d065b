"""GPU tests of what the operators for beams, windows and capped scores are for, run together:
a decoder with capped scores, sliding windows and norms on both sides of its blocks, a beam
search over the paged cache, and the cache verbs under them (attend_chunk, expand, fork).

Bars.  Logits against the same decoder in fp32: relative L2 3e-2 a position, the bar of the
plain decoder's tests (twice what bf16 arithmetic alone costs there); a norm behind a block
adds one rounding to the two of the residual add, and a cap's slope is at most 1.  Scores of
beams against teacher forcing through the same kernels: the K/V rows come from decode steps
on one side and from a prompt's kernels on the other, so logits differ by bf16 arithmetic
again, by at most 8e-2 each (the same tests' bar); a sum over n tokens by n times twice that.
Attention: relative L2 4e-3 (see the tests of the operators).  Copied rows: bit for bit.
"""
import pytest
import torch

from voom_amd import ops
from voom_amd.decoder import DecoderConfig, PagedDecoder, random_weights
from voom_amd.kv_paged import PagedKVCache

pytestmark = pytest.mark.gpu

REL, LOGIT_REL, LOGIT_ABS = 4e-3, 3e-2, 8e-2
CFG = DecoderConfig(num_hidden_layers=3, hidden_size=256, num_attention_heads=8,
                    num_key_value_heads=2, head_dim=64, intermediate_size=512, vocab_size=1000,
                    attn_softcap=4.0, sliding_window=24, full_attention_every=2, post_norms=True,
                    residual_scale=0.7)


def weights_of(cfg, seed):
    """Random weights with norms that are not 1, drawn on the CPU."""
    w = random_weights(cfg, seed=seed, std=0.06)
    g = torch.Generator().manual_seed(seed + 1)
    return {k: (1 + 0.2 * torch.randn(v.shape, generator=g)).to(v.dtype) if "norm" in k else v
            for k, v in w.items()}


def reference(cfg, w, ids):
    """fp32 logits [B, L, vocab] of whole sequences, without a cache."""
    w = {k: v.float().cuda() for k, v in w.items()}
    B, L = ids.shape
    nq, nkv, hd = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim

    def norm(x, name):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * w[name]

    half = hd // 2
    inv = 1 / cfg.rope_theta ** (torch.arange(half, device="cuda") / half)
    ang = torch.arange(L, device="cuda")[:, None] * inv
    cos, sin = ang.cos(), ang.sin()

    def turn(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    at = torch.arange(L, device="cuda")
    x = w["model.embed_tokens.weight"][ids]
    for layer in range(cfg.num_hidden_layers):
        p = f"model.layers.{layer}"
        h = norm(x, f"{p}.input_layernorm.weight")

        def heads(name, n):
            return (h @ w[f"{p}.self_attn.{name}.weight"].t()).view(B, L, n, hd).transpose(1, 2)

        q, k, v = turn(heads("q_proj", nq)), turn(heads("k_proj", nkv)), heads("v_proj", nkv)
        k, v = (t.repeat_interleave(nq // nkv, 1) for t in (k, v))
        s = q @ k.transpose(2, 3).contiguous() * hd ** -0.5
        if cfg.attn_softcap:
            s = cfg.attn_softcap * torch.tanh(s / cfg.attn_softcap)
        hidden = at > at[:, None]
        if cfg.window_of(layer):
            hidden |= at[:, None] - at >= cfg.window_of(layer)
        a = torch.softmax(s.masked_fill(hidden, -float("inf")), -1) @ v
        o = a.transpose(1, 2).reshape(B, L, nq * hd) @ w[f"{p}.self_attn.o_proj.weight"].t()
        if cfg.post_norms:
            x = x + cfg.residual_scale * norm(o, f"{p}.post_attention_layernorm.weight")
            h = norm(x, f"{p}.pre_feedforward_layernorm.weight")
        else:
            x = x + o
            h = norm(x, f"{p}.post_attention_layernorm.weight")
        act = torch.nn.functional.silu(h @ w[f"{p}.mlp.gate_proj.weight"].t())
        o = (act * (h @ w[f"{p}.mlp.up_proj.weight"].t())) @ w[f"{p}.mlp.down_proj.weight"].t()
        if cfg.post_norms:
            o = cfg.residual_scale * norm(o, f"{p}.post_feedforward_layernorm.weight")
        x = x + o
    return norm(x, "model.norm.weight") @ w["model.embed_tokens.weight"].t()


def near(got, want):
    rel = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert rel.max().item() <= LOGIT_REL, rel.max().item()


@pytest.mark.parametrize("change", [{}, dict(post_norms=False, residual_scale=1.0),
                                    dict(attn_softcap=0.0, full_attention_every=0),
                                    dict(sliding_window=0)])
def test_logits_in_chunks_tokens_and_replays(change):
    """A prompt in two chunks, eager decode steps, then captured ones."""
    cfg = DecoderConfig(**{**CFG.__dict__, **change})
    print(f"[beam decoder] {change}", flush=True)
    assert not cfg.plain
    w = weights_of(cfg, 5)
    dec = PagedDecoder(cfg, w)
    ids = torch.randint(0, cfg.vocab_size, (2, 60), generator=torch.Generator().manual_seed(2))
    ids = ids.cuda()
    want = reference(cfg, w, ids)
    kv = dec.new_cache(page_positions=32)
    got = [dec.forward(ids[:, :33], kv), dec.forward(ids[:, 33:50], kv)]
    got += [dec.forward(ids[:, t:t + 1], kv) for t in range(50, 55)]
    near(torch.cat(got, 1), want[:, :55])
    logits = torch.empty((2, cfg.vocab_size), device="cuda")
    graph, tok, nxt = dec.capture_decode(kv, 60, logits=logits)
    for t in range(55, 60):
        tok.copy_(ids[:, t:t + 1])
        graph.replay()
        kv.advance(1)
        near(logits, want[:, t])
        assert torch.equal(nxt, logits.argmax(-1))


def test_beam_scores_are_those_of_teacher_forcing():
    print("[beam decoder] scores", flush=True)
    w = weights_of(CFG, 7)
    dec = PagedDecoder(CFG, w)
    K, n, L = 5, 12, 21
    prompt = torch.randint(0, CFG.vocab_size, (2, L), generator=torch.Generator().manual_seed(3))
    kv = dec.new_cache(page_positions=32)
    tokens, scores = dec.generate_beam(prompt, K, n, kv)
    assert tokens.shape == (2, K, n) and (scores[:, 1:] <= scores[:, :-1]).all()
    assert kv.offset == L + n - 1 and kv._batch == 2 * K
    for b in range(2):
        assert len({tuple(t) for t in tokens[b].tolist()}) == K
        ids = torch.cat((prompt[b].cuda().expand(K, L), tokens[b]), 1)
        fresh = dec.forward(ids[:, :-1].contiguous(), dec.new_cache())[:, L - 1:]
        logp = torch.log_softmax(fresh.double(), -1).gather(2, ids[:, L:, None]).sum((1, 2))
        assert (logp - scores[b]).abs().max().item() <= 2 * LOGIT_ABS * n
        near(fresh, reference(CFG, w, ids[:, :-1])[:, L - 1:])
    # more beams find no worse a best one here, and one beam is the greedy search
    greedy, first = dec.generate_beam(prompt, 1, n, dec.new_cache())
    assert greedy.shape == (2, 1, n)
    kv = dec.new_cache()
    logits = dec.forward(prompt.cuda(), kv, last_only=True)
    for t in range(n):
        assert torch.equal(logits[:, -1].argmax(-1), greedy[:, 0, t])
        if t + 1 < n:
            logits = dec.forward(greedy[:, 0, t:t + 1].contiguous(), kv)


def test_beams_that_end_stay_and_a_plain_decoder_searches_too():
    print("[beam decoder] end token", flush=True)
    cfg = DecoderConfig(num_hidden_layers=2, vocab_size=200)
    dec = PagedDecoder(cfg, random_weights(cfg, seed=3, std=0.05))
    prompt = torch.randint(0, 200, (1, 40), generator=torch.Generator().manual_seed(4))
    free, _ = dec.generate_beam(prompt, 4, 8, dec.new_cache())
    end = int(free[0, 0, 3])  # the best beam passes through it
    tokens, scores = dec.generate_beam(prompt, 4, 8, dec.new_cache(), end_token=end)
    assert tokens.shape[2] <= 8
    over = (tokens == end).any(-1)
    assert over.any()
    for row in tokens[0].tolist():
        if end in row:
            at = row.index(end)
            assert set(row[at:]) == {end}
    with pytest.raises(ValueError, match="empty cache"):
        kv = dec.new_cache()
        dec.forward(prompt.cuda(), kv)
        dec.generate_beam(prompt, 2, 2, kv)


@pytest.mark.parametrize("page,spilled", [(32, False), (64, True)])
def test_expand_and_fork(page, spilled):
    print(f"[beam cache] page={page} spilled={spilled}", flush=True)
    B, K, NKV, D, S, layers = 2, 3, 2, 64, 150, 2
    g = torch.Generator(device="cuda").manual_seed(page)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

    kv = PagedKVCache(layers, 1 << 40, page_positions=page)
    want = []
    for layer in range(layers):
        k, v = rnd(B, NKV, S, D), rnd(B, NKV, S, D)
        kv.append(layer, k, v)
        kv.observe(layer, rnd(B, 4, 1, D), torch.zeros((B, 1, 4), device="cuda"))
        want.append([t.repeat_interleave(K, 0) for t in (k, v)])
    sums = [w.repeat_interleave(K, 0) for w in kv._weights]
    if spilled:
        kv.spill([(layer, 0) for layer in range(layers)])
    kv.expand(K)
    assert kv._batch == B * K and kv.offset == S
    for layer in range(layers):
        got = kv.gather(layer)
        assert all(torch.equal(a, b) for a, b in zip(got, want[layer]))
        assert torch.equal(kv._weights[layer], sums[layer])
    live = [p.live_slots for p in kv._pools]
    assert live == [B * K * -(-S // page)] * layers
    # the rows go apart, and then on from one another
    for step in range(3):
        for layer in range(layers):
            new = rnd(B * K, NKV, 20, D), rnd(B * K, NKV, 20, D)
            kv.append(layer, *new)
            want[layer] = [torch.cat(t, 2) for t in zip(want[layer], new)]
        if spilled:
            kv.spill([(layer, i) for layer in range(layers) for i in (0, 1)])
        parents = torch.tensor([[0, 0, 2], [1, 1, 1]], dtype=torch.int32, device="cuda")
        first = torch.full((B, K), S if step == 0 else S + 20 * step, dtype=torch.int32,
                           device="cuda")
        first[1, 0] = S  # (row 0 of the second request never was row 1's)
        first[1, 2] = S
        first[0, 1] = S
        kv.fork(parents, first, since=S)
        rows = torch.tensor([0, 0, 2, 4, 4, 4], device="cuda")
        for layer in range(layers):
            want[layer] = [t[rows] for t in want[layer]]
            sums[layer] = sums[layer][rows]
            got = kv.gather(layer)
            assert all(torch.equal(a, b) for a, b in zip(got, want[layer]))
            assert torch.equal(kv._weights[layer], sums[layer])
    # spills, reloads and cuts of the grown cache
    closed = [(layer, i) for layer in range(layers) for i in range(len(kv._pages[layer]))]
    kv.spill(closed)
    assert kv.reload() == len(closed) > 0
    kv.trim(S + 7)
    for layer in range(layers):
        got = kv.gather(layer)
        assert all(torch.equal(a, b[:, :, :S + 7]) for a, b in zip(got, want[layer]))
    kv.release()


def test_expand_within_a_budget_spills():
    kv = PagedKVCache(1, 3 << 20, page_positions=64)
    k = torch.randn((1, 8, 512, 128), device="cuda").to(torch.bfloat16)  # 2 MiB with V
    kv.append(0, k, k)
    kv.expand(4)
    assert kv.nbytes() <= 3 << 20
    got_k, got_v = kv.gather(0)
    assert torch.equal(got_k, k.expand(4, -1, -1, -1)) and torch.equal(got_v, got_k)
    kv.release()


@pytest.mark.parametrize("window,T", [(40, 1), (100, 30), (0, 150)])
def test_attend_chunk_reloads_what_its_window_reaches(window, T):
    B, NQ, NKV, D, S, page = 2, 8, 2, 64, 300, 32
    print(f"[beam cache] attend_chunk window={window} T={T}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

    kv = PagedKVCache(1, 1 << 40, page_positions=page)
    k, v, q = rnd(B, NKV, S, D), rnd(B, NKV, S, D), rnd(B, NQ, T, D)
    kv.append(0, k, v)
    slopes = torch.rand(NQ, generator=g, device="cuda") * 0.1

    def attend(**kw):
        return kv.attend_chunk(0, q, softcap=10.0, slopes=slopes, window=window, **kw)

    whole, lse = attend(return_lse=True)
    kv.spill([(0, i) for i in range(S // page)])
    spilled = sum(not p.resident for p in kv._pages[0])
    again = attend()
    left = sum(not p.resident for p in kv._pages[0])
    reach = max(0, S - T + 1 - window) if window else 0
    assert left == reach // page and spilled > left
    prefix = torch.full((B,), 9, dtype=torch.int32, device="cuda")
    attend(prefix_lens=prefix)
    assert all(p.resident for p in kv._pages[0])
    torch.cuda.synchronize()
    assert torch.equal(whole, again)
    at, token = torch.arange(S - T, S, device="cuda")[:, None], torch.arange(S, device="cuda")
    s = q.double() @ k.double().repeat_interleave(NQ // NKV, 1).transpose(2, 3).contiguous()
    s = 10 * torch.tanh(s * D ** -0.5 / 10) - slopes.double()[:, None, None] * (at - token).abs()
    s = s.masked_fill((token > at) | ((at - token >= window) if window else False), -float("inf"))
    want = torch.softmax(s, -1) @ v.double().repeat_interleave(NQ // NKV, 1)
    assert ((whole.double() - want).norm() / want.norm()).item() <= REL
    assert (lse.transpose(1, 2).double() - torch.logsumexp(s, -1)).abs().max().item() <= 2e-4
    kv.release()


def test_cache_refusals():
    kv = PagedKVCache(2, 1 << 40, page_positions=32)
    x = torch.randn((4, 2, 40, 64), device="cuda").to(torch.bfloat16)
    with pytest.raises(ValueError, match="needs a kv cache"):
        kv.expand(2)
    kv.append(0, x, x)
    with pytest.raises(ValueError, match="one length"):
        kv.expand(2)
    kv.append(1, x, x)
    parents = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="beams"):
        kv.expand(0)
    with pytest.raises(ValueError, match="parents"):
        kv.fork(parents[:, :3])
    with pytest.raises(ValueError, match="parents"):
        kv.fork(parents.long())
    with pytest.raises(ValueError, match="first"):
        kv.fork(parents, parents[0])
    with pytest.raises(ValueError, match="since"):
        kv.fork(parents, since=41)
    with pytest.raises(ValueError, match="device"):
        kv.fork(parents.cpu())
    with pytest.raises(ValueError, match="65535"):
        kv.expand(20000)
    kv.check_integrity()  # (nothing that was refused has touched it)
    with pytest.raises(ValueError, match="queries"):
        kv.attend_chunk(0, torch.zeros((4, 2, 41, 64), dtype=torch.bfloat16, device="cuda"))
    kv.reserve(60)
    with pytest.raises(ValueError, match="captured"):
        kv.expand(2)
    with pytest.raises(ValueError, match="residual_scale"):
        PagedDecoder(DecoderConfig(residual_scale=0.5), {})
    kv.release()

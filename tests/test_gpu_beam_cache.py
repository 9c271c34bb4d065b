"""The cache under beams and windows where its calls can go wrong: rows behind the last step
of a search, searches refused before they begin, expansions and forks that fail, windows and
distances after an eviction.

Bars.  A search of the test's own over the same decoder: the same tokens, scores within the
n-fold bar of a selection (1e-5 + 2^-23 |score|, test_gpu_beams.py).  Keys of the first layer
by batch shape: bf16 projections of equal inputs, summed in another order at most, so a
relative L2 of 2^-7, two steps of bf16, over a row; rows of other tokens differ by about
sqrt(2).  Attention: relative L2 4e-3 (test_gpu_chunk.py).  Copied rows: bit for bit.
"""
import pytest
import torch

from test_gpu_beam_decoder import CFG, REL, weights_of
from voom_amd import ops
from voom_amd.decoder import DecoderConfig, PagedDecoder, random_weights
from voom_amd.kv_paged import PagedKVCache

pytestmark = pytest.mark.gpu


def rnd(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def steps_alone(dec, prompt, tokens, K):
    """Logits [B, K, V] behind prompt and tokens [B, K, n], in a cache of its own whose rows
    never go on from one another."""
    B = prompt.shape[0]
    kv = dec.new_cache(page_positions=32)
    logits = dec.forward(prompt, kv, last_only=True).expand(B, K, -1)
    kv.expand(K)
    for t in range(tokens.shape[2]):
        logits = dec.forward(tokens[:, :, t].reshape(B * K, 1), kv).view(B, K, -1)
    kv.release()
    return logits


def search_alone(dec, prompt, K, n):
    """generate_beam's search, every step of it from the prompt on."""
    B, rows = prompt.shape[0], torch.arange(K, device="cuda")
    scores = torch.full((B, K), -float("inf"), device="cuda")
    scores[:, 0] = 0
    tokens = torch.empty((B, K, 0), dtype=torch.long, device="cuda")
    for _ in range(n):
        logp = torch.log_softmax(steps_alone(dec, prompt, tokens, K).double(), -1)
        V = logp.shape[-1]
        best = torch.sort((scores.double()[..., None] + logp).flatten(1), dim=1, descending=True,
                          stable=True)
        value, at = best.values[:, :K], best.indices[:, :K]
        past = tokens.gather(1, (at // V)[..., None].expand(-1, -1, tokens.shape[2]))
        found = torch.cat((past, (at % V)[..., None]), -1)
        for b in range(B):  # the best continuation of a beam in the beam's row
            row, parent = [None] * K, (at[b] // V).tolist()
            for i, p in enumerate(parent):
                if row[p] is None:
                    row[p] = i
            rest = [i for i in range(K) if i not in row]
            order = [rest.pop(0) if i is None else i for i in row]
            value[b], found[b] = value[b][order], found[b][order]
        scores, tokens = value.float(), found
    order = scores.argsort(dim=1, descending=True, stable=True)
    return tokens.gather(1, order[..., None].expand_as(tokens)), scores.gather(1, order)


@pytest.mark.parametrize("plain", [False, True])
def test_a_search_is_one_whose_rows_are_never_copied(plain):
    print(f"[beam cache] search, plain={plain}", flush=True)
    cfg = DecoderConfig(num_hidden_layers=2, vocab_size=300) if plain else CFG
    dec = PagedDecoder(cfg, weights_of(cfg, 11))
    K, n, L = 4, 7, 37
    prompt = torch.randint(0, cfg.vocab_size, (2, L), generator=torch.Generator().manual_seed(8))
    prompt = prompt.cuda()
    tokens, scores = dec.generate_beam(prompt, K, n, dec.new_cache(page_positions=32))
    want, value = search_alone(dec, prompt, K, n)
    assert torch.equal(tokens, want)
    bar = n * (1e-5 + 2.0 ** -23 * value.abs().max().item())
    assert (scores - value).abs().max().item() <= bar


@pytest.mark.parametrize("end", [False, True])
def test_rows_hold_their_beams_tokens_behind_a_search(end):
    """All but the last token of each: the first layer's keys go by token and position."""
    print(f"[beam cache] rows behind a search, end={end}", flush=True)
    cfg = DecoderConfig(num_hidden_layers=2, vocab_size=200)
    dec = PagedDecoder(cfg, random_weights(cfg, seed=3, std=0.05))
    B, K, n, L = 2, 4, 5, 33
    prompt = torch.randint(0, 200, (B, L), generator=torch.Generator().manual_seed(6))
    stop = {}
    if end:  # the end token is one that some of the beams pass through
        stop = {"end_token": int(dec.generate_beam(prompt, K, n, dec.new_cache())[0][0, 0, 2])}
    kv = dec.new_cache(page_positions=32)
    tokens, _ = dec.generate_beam(prompt, K, n, kv, **stop)
    n = tokens.shape[2]
    assert kv.offset == L + n - 1
    keys = kv.gather(0)[0][:, :, L:].transpose(1, 2).flatten(2).view(B, K, n - 1, -1)
    apart = 0
    for b in range(B):
        fresh = dec.new_cache()
        dec.forward(torch.cat((prompt[b].cuda().expand(K, L), tokens[b]), 1)[:, :-1].contiguous(),
                    fresh)
        want = fresh.gather(0)[0][:, :, L:].transpose(1, 2).flatten(2)
        off = (keys[b][:, None].double() - want[None].double()).norm(dim=-1) / want.double().norm(
            dim=-1)
        same = off.amax(-1) <= 2.0 ** -7  # [cache row, beam]
        past = tokens[b][:, :-1]
        alike = (past[:, None] == past[None]).all(-1)  # beams that differ in the last token
        assert torch.equal(same.sum(0), alike.sum(0)) and same.any(1).all()
        apart += int((~alike).sum())
    assert apart > 0


def test_windows_and_distances_after_an_eviction():
    """What a window reaches has to lie behind what the eviction left apart; else places in the
    cache are no positions, and the call is refused."""
    print("[beam cache] chunks after an eviction", flush=True)
    NQ, NKV, D, S, budget, recent = 8, 2, 64, 100, 40, 20
    g = gen(1)
    kv = PagedKVCache(1, 1 << 40, page_positions=32)
    k, v = rnd(g, 2, NKV, S + 10, D), rnd(g, 2, NKV, S + 10, D)
    slopes = torch.rand(NQ, generator=g, device="cuda") * 0.1
    prefix = torch.full((2,), 2, dtype=torch.int32, device="cuda")

    def append(a, b):
        kv.append(0, k[:, :, a:b].contiguous(), v[:, :, a:b].contiguous())

    def reference(q, window):
        T = q.shape[2]
        at, token = torch.arange(S + 10 - T, S + 10, device="cuda")[:, None], torch.arange(
            S + 10, device="cuda")
        s = q.double() @ k.double().repeat_interleave(NQ // NKV, 1).transpose(2, 3).contiguous()
        s = s * D ** -0.5 - slopes.double()[:, None, None] * (at - token).abs()
        s = s.masked_fill((token > at) | (at - token >= window), -float("inf"))
        return torch.softmax(s, -1) @ v.double().repeat_interleave(NQ // NKV, 1)

    append(0, S)
    kv.observe(0, rnd(g, 2, NQ, 1, D), torch.zeros((2, 1, NQ), device="cuda"))
    assert kv.evict(budget, sink=2, recent=recent) == S - budget
    append(S, S + 10)  # 50 tokens, the newest 30 of each head next to each other
    for T in (1, 4):
        q = rnd(g, 2, NQ, T, D)
        reach = recent + 10 - T + 1
        got = kv.attend_chunk(0, q, window=reach, slopes=slopes)
        want = reference(q, reach)
        assert ((got.double() - want).norm() / want.norm()).item() <= REL
        for scores in (dict(window=reach + 1), dict(window=1000), dict(slopes=slopes),
                       dict(slopes=slopes, window=reach + 1), dict(prefix_lens=prefix),
                       dict(prefix_lens=prefix, window=1)):
            with pytest.raises(ValueError, match="after evict"):
                kv.attend_chunk(0, q, **scores)
        assert kv.attend_chunk(0, q[:, :, :0], window=1000, prefix_lens=prefix).numel() == 0
        # what goes by no position is as it was
        whole = kv.attend_chunk(0, q, softcap=5.0, window=0)
        assert torch.equal(whole, kv.attend_chunk(0, q, softcap=5.0))
    q = rnd(g, 2, NQ, 1, D)
    kv.trim(15)  # all that is left lies apart, what follows does not
    append(0, 5)
    kv.attend_chunk(0, q, window=5)
    with pytest.raises(ValueError, match="after evict"):
        kv.attend_chunk(0, q, window=6)
    kv.observe(0, q, torch.zeros((2, 1, NQ), device="cuda"))
    kv.evict(18, recent=16)  # 2 are gone, of the newest 5 none
    kv.attend_chunk(0, q, window=5)
    with pytest.raises(ValueError, match="after evict"):
        kv.attend_chunk(0, q, window=6)
    kv.evict(10, recent=3)
    kv.attend_chunk(0, q, window=3)
    with pytest.raises(ValueError, match="after evict"):
        kv.attend_chunk(0, q, window=4)
    kv.trim(0)
    append(0, 30)
    kv.attend_chunk(0, q, window=25, slopes=slopes, prefix_lens=prefix)
    kv.release()


def test_a_decoder_refuses_windows_after_an_eviction_before_it_appends():
    print("[beam cache] decoder after an eviction", flush=True)
    dec = PagedDecoder(CFG, weights_of(CFG, 5))
    ids = torch.randint(0, CFG.vocab_size, (1, 70), generator=torch.Generator().manual_seed(2))
    ids = ids.cuda()
    window = CFG.sliding_window

    def evicted(recent):
        kv = dec.new_cache(page_positions=32)
        dec.forward(ids[:, :60], kv)
        nq, hd = CFG.num_attention_heads, CFG.head_dim
        for layer in range(CFG.num_hidden_layers):
            kv.observe(layer, rnd(gen(layer), 1, nq, 1, hd), torch.zeros((1, 1, nq), device="cuda"))
        kv.evict(40, sink=1, recent=recent)
        return kv

    kv = evicted(window - 2)
    with pytest.raises(ValueError, match="after evict"):
        dec.forward(ids[:, 60:61], kv)
    assert kv.layer_lengths() == (40,) * CFG.num_hidden_layers and kv.offset == 40
    kv = evicted(window - 1)
    dec.forward(ids[:, 60:65], kv)
    assert kv.offset == 45


def test_searches_are_refused_before_the_prompt_runs():
    print("[beam cache] searches refused", flush=True)
    cfg = DecoderConfig(num_hidden_layers=2, vocab_size=200)
    dec = PagedDecoder(cfg, random_weights(cfg, seed=3, std=0.05))
    prompt = torch.randint(0, 200, (2, 9), generator=torch.Generator().manual_seed(6))
    kv = dec.new_cache()

    def refused(match, *args, prompt=prompt, kv=kv, **kw):
        with pytest.raises(ValueError, match=match):
            dec.generate_beam(prompt, *args, kv, **kw)
        assert kv.offset == 0 and kv.layer_lengths() == (0, 0)

    refused("beams", 0, 4)
    refused("beams", -1, 4)
    refused("beams", 33, 4)
    refused("end token", 2, 4, end_token=200)
    refused("end token", 2, 4, end_token=-1)
    refused("prompt", 2, 4, prompt=prompt[:, :0])
    assert kv._geom is None
    kept = dec.new_cache()
    dec.forward(prompt.cuda(), kept)
    kept.reserve(30)
    kept.trim(0)
    refused("captured", 2, 4, kv=kept)
    tokens, scores = dec.generate_beam(prompt, 2, 4, kv, end_token=199)
    assert tokens.shape[:2] == (2, 2) and scores.isfinite().all()


@pytest.mark.parametrize("fails_in", [0, 1, 2])
def test_an_expansion_without_memory_leaves_the_cache_as_it_was(fails_in):
    print(f"[beam cache] expand fails in layer {fails_in}", flush=True)
    B, K, S, page, layers = 2, 3, 100, 32, 3
    g = gen(fails_in)
    kv = PagedKVCache(layers, 1 << 40, page_positions=page)
    want = [(rnd(g, B, 2, S, 64), rnd(g, B, 2, S, 64)) for _ in range(layers)]
    for layer in range(layers):
        kv.append(layer, *want[layer])
    pool = kv._pool(fails_in)
    live = [p.live_slots for p in kv._pools]

    def fails(count):
        raise torch.cuda.OutOfMemoryError("no memory for the slots")

    pool.allocate = fails
    with pytest.raises(torch.cuda.OutOfMemoryError):
        kv.expand(K)
    del pool.allocate
    assert [p.live_slots for p in kv._pools] == live and kv._batch == B
    for layer in range(layers):
        assert all(torch.equal(a, b) for a, b in zip(kv.gather(layer), want[layer]))
    kv.expand(K)
    assert [p.live_slots for p in kv._pools] == [K * n for n in live]
    for layer in range(layers):
        assert all(torch.equal(a, b.repeat_interleave(K, 0))
                   for a, b in zip(kv.gather(layer), want[layer]))
    kv.release()


def test_a_fork_that_is_refused_leaves_the_cache_in_use():
    print("[beam cache] forks refused", flush=True)
    g = gen(4)
    k, v = rnd(g, 4, 2, 50, 64), rnd(g, 4, 2, 50, 64)
    kv = PagedKVCache(1, 1 << 40, page_positions=32)
    kv.append(0, k, v)
    dev = dict(dtype=torch.int32, device="cuda")
    ops.set_bounds_checks(True)
    try:
        with pytest.raises(ValueError, match="its own parent"):
            kv.fork(torch.tensor([[1, 2, 2, 3]], **dev))
        with pytest.raises(ValueError, match="outside"):
            kv.fork(torch.tensor([[0, 1, 2, 4]], **dev))
    finally:
        ops.set_bounds_checks(False)
    assert all(torch.equal(a, b) for a, b in zip(kv.gather(0), (k, v)))
    kv.fork(torch.tensor([[0, 0, 2, 2]], **dev))
    rows = torch.tensor([0, 0, 2, 2], device="cuda")
    assert all(torch.equal(a, b[rows]) for a, b in zip(kv.gather(0), (k, v)))
    # pages and heads that the copy does not take
    for page, D in ((4, 64), (32, 1032)):
        kv = PagedKVCache(1, 1 << 40, page_positions=page)
        k, v = rnd(g, 2, 1, 9, D), rnd(g, 2, 1, 9, D)
        kv.append(0, k, v)
        for call in (lambda: kv.expand(2), lambda: kv.fork(torch.zeros((1, 2), **dev))):
            with pytest.raises(ValueError, match="8 tokens"):
                call()
        kv.expand(1)  # (nothing to copy)
        assert kv._batch == 2
        assert all(torch.equal(a, b) for a, b in zip(kv.gather(0), (k, v)))
        kv.release()


def test_a_fork_of_observed_rows_leaves_out_parents_that_are_none():
    print("[beam cache] wild parents, observed", flush=True)
    g = gen(6)
    k, v = rnd(g, 6, 2, 40, 64), rnd(g, 6, 2, 40, 64)
    kv = PagedKVCache(1, 1 << 40, page_positions=32)
    kv.append(0, k, v)
    kv.observe(0, rnd(g, 6, 4, 1, 64), torch.zeros((6, 1, 4), device="cuda"))
    sums = kv._weights[0].clone()
    kv.fork(torch.tensor([[0, -1, 3], [2, 99, 2]], dtype=torch.int32, device="cuda"))
    rows = torch.tensor([0, 1, 2, 5, 4, 5], device="cuda")
    assert all(torch.equal(a, b[rows]) for a, b in zip(kv.gather(0), (k, v)))
    assert torch.equal(kv._weights[0], sums[rows])
    kv.release()


@pytest.mark.parametrize("page,spilled", [(32, 7), (64, 2), (32, 9)])
def test_a_capped_token_streams_what_the_budget_leaves_out(page, spilled):
    """Spilled pages that do not fit max_bytes stay spilled; those that do come back."""
    print(f"[beam cache] capped token, page={page} spilled={spilled}", flush=True)
    B, NQ, NKV, D, S = 2, 8, 2, 64, 300
    g = gen(page + spilled)
    kv = PagedKVCache(2, 1 << 40, page_positions=page)
    k, v, q = rnd(g, B, NKV, S, D), rnd(g, B, NKV, S, D), rnd(g, B, NQ, 1, D)
    for layer in range(2):
        kv.append(layer, k, v)
    whole = kv.attend_chunk(0, q, softcap=3.0)
    s = q.double() @ k.double().repeat_interleave(NQ // NKV, 1).transpose(2, 3).contiguous()
    s = 3 * torch.tanh(s * D ** -0.5 / 3)
    want = torch.softmax(s, -1) @ v.double().repeat_interleave(NQ // NKV, 1)
    pages = [(0, i) for i in range(spilled)]
    assert kv.spill(pages) == spilled
    kv.max_bytes = kv.nbytes() + spilled * kv.page_nbytes - 1
    for _ in range(3):
        got = kv.attend_chunk(0, q, softcap=3.0)
        assert sum(not p.resident for p in kv._pages[0]) == spilled
        assert got.shape == whole.shape
        assert ((got.double() - want).norm() / want.norm()).item() <= REL
    assert not kv._prefetched
    # what the call takes besides goes the way of the layer's resident pages
    out = torch.empty((B, 1, NQ, D), dtype=torch.bfloat16, device="cuda")
    more = [dict(new_lens=torch.tensor([1, 0], dtype=torch.int32, device="cuda")), dict(out=out),
            dict(slopes=torch.zeros(NQ, device="cuda"))]
    for scores in more:
        got = kv.attend_chunk(0, q, softcap=3.0, **scores)
        assert torch.equal(got[:1], whole[:1])
        assert torch.equal(got[1], 0 * whole[1] if "new_lens" in scores else whole[1])
        assert kv.spill(pages) == spilled
    assert torch.equal(out.permute(0, 2, 1, 3), whole)
    kv.max_bytes += 1
    assert torch.equal(kv.attend_chunk(0, q, softcap=3.0), whole)
    assert all(p.resident for p in kv._pages[0])
    kv.release()

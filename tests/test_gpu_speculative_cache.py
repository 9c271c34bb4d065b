"""GPU test of PagedKVCache's verbs for drafted tokens and bounded caches, run together as a
serving step runs them: projections appended with head norms and rotation, a tree of drafts
attended, the accepted branch kept, its weights observed, the cache cut to a budget, and a
token decoded over what is left.  Every attention is compared with fp64 over the rows that
the reference says are there; K and V rows exactly.

Bars: outputs as of the tree and decode kernels (relative L2 4e-3); weights relative 4e-4
(the log-sum-exp and the scores are off by 2e-4 each, see the tests of the operators).
"""
import pytest
import torch

from paged_inputs import trees
from voom_amd import ops
from voom_amd.decoder import DecoderConfig, PagedDecoder, random_weights
from voom_amd.kv_paged import KVIntegrityError, PagedKVCache

pytestmark = pytest.mark.gpu

REL, WEIGHT = 4e-3, 4e-4
B, NQ, NKV, D, LAYERS = 2, 8, 2, 64, 2
G = NQ // NKV


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def attend64(q, k, v, sees):
    """fp64 (out [B, NQ, T, D], weights [B, NQ, T, S]); sees bool [B, T, S]."""
    k, v = (x.double().repeat_interleave(G, 1) for x in (k, v))
    s = torch.matmul(q.double(), k.transpose(2, 3).contiguous()) * D ** -0.5
    w = torch.softmax(s.masked_fill(~sees[:, None], -float("inf")), -1)
    return torch.matmul(w, v), w


@pytest.mark.parametrize("page,spilled", [(32, False), (64, True), (256, False)])
def test_a_speculative_step_on_a_bounded_cache(page, spilled):
    print(f"[speculative] page={page} spilled={spilled}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(page)

    def rnd(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    S, T, path, budget, sink, recent = 300, 9, [0, 2, 5, 8], 120, 4, 16
    kv = PagedKVCache(LAYERS, 1 << 40, page_positions=page, resident_pages=1)
    cos, sin = ops.rope_cache(600, D, 1e4)
    wq, wk = (1 + rnd(2, D, std=0.2)).unbind()
    norm = dict(q_weight=wq.contiguous(), k_weight=wk.contiguous())
    for layer in range(LAYERS):
        q = kv.append_qkv(layer, rnd(B, S, (NQ + 2 * NKV) * D), cos, sin, NQ, NKV, **norm)
        assert q.shape == (B, NQ, S, D)
    assert kv.offset == S == kv.next_position
    if spilled:
        kv.spill([(layer, i) for layer in range(LAYERS) for i in (0, 2)])

    mask = trees(1, T, 3)[0].cuda()
    depth = mask.sum(-1).int() - 1
    rows = {}
    for layer in range(LAYERS):
        qkv = rnd(B, T, (NQ + 2 * NKV) * D)
        q = kv.append_qkv(layer, qkv, cos, sin, NQ, NKV, positions=(S + depth).repeat(B, 1), **norm)
        out, lse = kv.attend_tree(layer, q, mask, return_lse=True)
        k, v = kv.gather(layer)
        sees = torch.ones((B, T, S + T), dtype=torch.bool, device="cuda")
        sees[:, :, S:] = mask
        want, _ = attend64(q, k, v, sees)
        torch.cuda.synchronize()
        assert rel(out, want) <= REL
        rows[layer] = (q, lse, k, v)
    assert kv.offset == S + T

    kv.keep_drafts(T, path)
    n = len(path)
    stay = list(range(S)) + [S + i for i in path]
    assert kv.offset == S + n and kv.layer_lengths() == (S + n,) * LAYERS
    for layer in range(LAYERS):
        k, v = kv.gather(layer)
        assert torch.equal(k, rows[layer][2][:, :, stay])
        assert torch.equal(v, rows[layer][3][:, :, stay])

    # the accepted branch is a chain here or not: its rows saw what a chain sees only if
    # every draft of the path is the next one's parent
    chain = all(bool(mask[b, a]) for a, b in zip(path, path[1:]))
    for layer in range(LAYERS):
        q, lse, k, v = rows[layer]
        q = q[:, :, path].contiguous()
        k, v = k[:, :, stay], v[:, :, stay]
        sees = torch.ones((n, S + n), dtype=torch.bool, device="cuda").tril(S).repeat(B, 1, 1)
        _, w = attend64(q, k, v, sees)
        if chain:
            lse = lse[:, path].contiguous()
        else:
            _, lse = kv.attend_tree(layer, q, return_lse=True)
        kv.observe(layer, q, lse)
        got = kv._weights[layer]
        added = w.reshape(B, NKV, G * n, -1).sum(2)
        torch.cuda.synchronize()
        assert (got[:, :, S + n:] == 0).all()
        off = (got[:, :, :S + n].double() - added).abs()
        assert (off <= WEIGHT * added + 1e-6).all()

    sums = [kv._weights[layer][:, :, :S + n].cpu() for layer in range(LAYERS)]
    before = [kv.gather(layer) for layer in range(LAYERS)]
    assert kv.evict(budget, sink=sink, recent=recent) == S + n - budget
    assert kv.offset == budget and kv.next_position == S + n
    assert kv.evict(budget, sink=sink, recent=recent) == 0
    for layer in range(LAYERS):
        k, v = kv.gather(layer)
        kept = torch.zeros((B, NKV, budget), dtype=torch.long)
        for b in range(B):
            for h in range(NKV):
                s = sums[layer][b, h].clone()
                s[:sink] = s[S + n - recent:] = float("inf")
                kept[b, h] = torch.sort(s, descending=True, stable=True).indices[:budget].sort()[0]
        at = kept.cuda()[..., None].expand(-1, -1, -1, D)
        assert torch.equal(k, before[layer][0].gather(2, at))
        assert torch.equal(v, before[layer][1].gather(2, at))
        want = sums[layer].gather(2, kept)
        got = kv._weights[layer].cpu()
        assert torch.equal(got[:, :, :budget], want) and (got[:, :, budget:] == 0).all()

    # a token decoded over what is left, its key rotated at its true position
    for layer in range(LAYERS):
        q = kv.append_qkv(layer, rnd(B, 1, (NQ + 2 * NKV) * D), cos, sin, NQ, NKV, **norm)
        k, v = kv.gather(layer)
        out = kv.attend(layer, q)
        want, _ = attend64(q, k, v, torch.ones((B, 1, budget + 1), dtype=torch.bool, device="cuda"))
        torch.cuda.synchronize()
        assert rel(out, want) <= REL
    assert kv.offset == budget + 1 and kv.next_position == S + n + 1
    with pytest.raises(ValueError, match="after evict"):
        kv.reserve(400)
    kv.trim(0)
    assert kv.next_position == 0


def test_keeping_drafts_leaves_spilled_pages_alone():
    """Pages before the drafts stay where they are; those with drafts come back."""
    print("[speculative] keep_drafts with spilled pages", flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    S, T, page, path = 150, 9, 32, [1, 4, 7]  # the drafts close page 4
    kv = PagedKVCache(LAYERS, 1 << 40, page_positions=page, resident_pages=1)
    full = []
    for layer in range(LAYERS):
        k, v = (torch.randn((B, NKV, S + T + 2, D), generator=g, device="cuda").bfloat16()
                for _ in range(2))
        kv.append(layer, k[:, :, :S + T].contiguous(), v[:, :, :S + T].contiguous())
        full.append((k, v))
    # one page behind the context closed too: 161 tokens, the drafts are the last 11
    for layer, (k, v) in enumerate(full):
        kv.append(layer, k[:, :, S + T:].contiguous(), v[:, :, S + T:].contiguous())
    kv.spill([(layer, i) for layer in range(LAYERS) for i in (0, 2, 4)])
    kv.keep_drafts(T + 2, path)
    for layer, (k, v) in enumerate(full):
        assert [p.resident for p in kv._pages[layer]] == [False, True, False, True]
        at = list(range(S)) + [S + i for i in path]
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k[:, :, at]) and torch.equal(got_v, v[:, :, at])
    kv.release()


def test_refusals_and_small_calls():
    kv = PagedKVCache(1, 1 << 40, page_positions=32)
    with pytest.raises(ValueError, match="kv cache"):
        kv.evict(5)
    k = torch.randn((1, 2, 40, 64), device="cuda").to(torch.bfloat16)
    kv.append(0, k, k)
    q = torch.randn((1, 4, 41, 64), device="cuda").to(torch.bfloat16)
    with pytest.raises(ValueError, match="41 drafts"):
        kv.attend_tree(0, q)
    with pytest.raises(ValueError, match="41 queries"):
        kv.observe(0, q, torch.zeros((1, 41, 4), device="cuda"))
    assert kv.attend_tree(0, q[:, :, :0]).shape == (1, 4, 0, 64)
    with pytest.raises(ValueError, match="observe"):
        kv.evict(30)
    assert kv.evict(40) == 0
    for budget, sink, recent in ((0, 0, 0), (10, 6, 5), (10, -1, 0)):
        with pytest.raises(ValueError, match="budget"):
            kv.evict(budget, sink=sink, recent=recent)
    for path in ([1, 1], [2, 0], [-1], [5], [[0], [1]], [0, 1, 2, 3, 4, 5]):
        with pytest.raises(ValueError, match="path"):
            kv.keep_drafts(5, path)
    with pytest.raises(ValueError, match="drafts"):
        kv.keep_drafts(41, [0])
    kv.keep_drafts(5, [])
    assert kv.offset == 35
    kv.keep_drafts(3, [0, 1, 2])
    assert kv.offset == 35
    kv.keep_drafts(3, torch.tensor([2], device="cuda"))
    got, _ = kv.gather(0)
    assert kv.offset == 33 and torch.equal(got[:, :, 32], k[:, :, 34])
    with pytest.raises(ValueError, match="geometry"):
        kv.append_qkv(0, torch.zeros((1, 2, 100), dtype=torch.bfloat16, device="cuda"), None, None, 3,
                      1)
    kv.reserve(64)
    _, lse = kv.attend_tree(0, q[:, :, :1].contiguous(), return_lse=True)
    kv.observe(0, q[:, :, :1], lse)
    with pytest.raises(ValueError, match="captured"):
        kv.evict(10)


def test_a_decoder_goes_on_after_an_eviction_at_the_next_position():
    cfg = DecoderConfig(num_hidden_layers=2, hidden_size=128, num_attention_heads=2,
                        num_key_value_heads=1, head_dim=64, intermediate_size=128, vocab_size=256)
    model = PagedDecoder(cfg, random_weights(cfg, 3))
    kv = model.new_cache(page_positions=32)
    prompt = torch.randint(0, 256, (1, 90), device="cuda")
    model.forward(prompt, kv, last_only=True)
    for layer in range(2):
        q = torch.randn((1, 2, 8, 64), device="cuda").to(torch.bfloat16)
        kv.observe(layer, q, kv.attend_tree(layer, q, return_lse=True)[1])
    kv.evict(50, sink=2, recent=10)
    seen = []
    tables = model._rope_tables
    model._rope_tables = lambda positions: seen.append(positions.tolist()) or tables(positions)
    logits = model.forward(prompt[:, :1], kv)
    assert torch.isfinite(logits).all() and seen == [[90]] and kv.offset == 51


def filled(layers, tokens, page, max_bytes, seed):
    """A cache of random K/V, with sums that ask for other tokens in every head; and the K/V."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = PagedKVCache(layers, max_bytes, page_positions=page, resident_pages=1)
    full = []
    for layer in range(layers):
        k, v = (torch.randn((B, NKV, tokens, D), generator=g, device="cuda").bfloat16()
                for _ in range(2))
        kv.append(layer, k, v)
        full.append((k, v))
    kv._weights = [torch.rand((B, NKV, tokens), generator=g, device="cuda")
                   for _ in range(layers)]
    return kv, full


def rows_kept(sums, tokens, budget):
    """[B, NKV, budget] positions of the largest sums, ascending."""
    best = torch.sort(sums[:, :, :tokens], dim=-1, descending=True, stable=True).indices
    return best[..., :budget].sort(-1).values


@pytest.mark.parametrize("page,budget", [(32, 96), (32, 100), (64, 7)])
def test_an_eviction_gives_its_pages_back_and_stays_within_the_bytes_allowed(page, budget):
    print(f"[speculative] evicted pages page={page} budget={budget}", flush=True)
    layers, tokens = 4, 20 * page + 3
    page_bytes = B * NKV * page * D * 4
    allowed = 2 * 20 * page_bytes  # two of the four layers
    kv, full = filled(layers, tokens, page, allowed, seed=page + budget)
    sums = [w.clone() for w in kv._weights]
    open_bytes = layers * 3 * page_bytes // page
    assert kv.nbytes() <= allowed + open_bytes and kv.stats.spills >= 2 * 20
    held = []
    moved = ops.compact_kv

    def compact(*args, **kw):
        held.append(sum(pool.live_slots * pool.slot_bytes for pool in kv._pools))
        return moved(*args, **kw)

    ops.compact_kv = compact
    try:
        assert kv.evict(budget) == tokens - budget
    finally:
        ops.compact_kv = moved
    # what the cache may hold, an open page per layer, and the layer that is being cut
    assert len(held) == layers and max(held) <= allowed + (layers + 21) * page_bytes
    pages = -(-budget // page)
    resident = sum(p.resident for lp in kv._pages for p in lp) + sum(map(len, kv._open_slots))
    assert resident <= layers * pages
    assert sum(pool.live_slots for pool in kv._pools) == B * resident
    assert sum(pool.live_slots * pool.slot_bytes for pool in kv._pools) <= (
        kv.nbytes() + layers * page_bytes)
    for layer, (k, v) in enumerate(full):
        at = rows_kept(sums[layer], tokens, budget)[..., None].expand(-1, -1, -1, D)
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k.gather(2, at)) and torch.equal(got_v, v.gather(2, at))
    # the slots are used again: no pool grows while the cache fills up and is cut again
    capacity = [pool.capacity for pool in kv._pools]
    for _ in range(3):
        before = [kv.gather(layer) for layer in range(layers)]
        for layer, (k, v) in enumerate(full):
            kv.append(layer, k[:, :, :5 * page], v[:, :, :5 * page])
        for layer, (k, v) in enumerate(full):
            got_k, got_v = kv.gather(layer)
            assert torch.equal(got_k, torch.cat((before[layer][0], k[:, :, :5 * page]), 2))
            assert torch.equal(got_v, torch.cat((before[layer][1], v[:, :, :5 * page]), 2))
        assert kv.evict(budget) == 5 * page and kv.offset == budget
    assert [pool.capacity for pool in kv._pools] == capacity
    assert kv.next_position == tokens + 15 * page
    kv.release()


@pytest.mark.parametrize("fails_in", [0, 1, 2])
def test_an_eviction_whose_spilled_pages_do_not_come_back(fails_in):
    """Before the first move the cache is as it was; after it no call takes the layers, of
    which some are cut, for one cache."""
    print(f"[speculative] eviction fails in layer {fails_in}", flush=True)
    layers, tokens, page, budget = 3, 100, 32, 40
    kv, full = filled(layers, tokens, page, 1 << 40, seed=fails_in)
    sums = [w.clone() for w in kv._weights]
    kv.spill([(layer, 1) for layer in range(layers)])
    reload = kv.reload

    def broken(pages=None, stream=None):
        if any(p.layer == fails_in for p in pages):
            raise OSError("a page file is gone")
        return reload(pages, stream)

    kv.reload = broken
    with pytest.raises(OSError, match="gone"):
        kv.evict(budget)
    kv.reload = reload
    if fails_in == 0:
        for layer, (k, v) in enumerate(full):
            got_k, got_v = kv.gather(layer)
            assert torch.equal(got_k, k) and torch.equal(got_v, v)
        assert kv.offset == tokens == kv.next_position
        assert kv.evict(budget) == tokens - budget
        for layer, (k, _) in enumerate(full):
            at = rows_kept(sums[layer], tokens, budget)[..., None].expand(-1, -1, -1, D)
            assert torch.equal(kv.gather(layer)[0], k.gather(2, at))
        return
    k, v = (x[:, :, :1].contiguous() for x in full[0])
    q = torch.zeros((B, NQ, 1, D), dtype=torch.bfloat16, device="cuda")
    for call in (lambda: kv.append(0, k, v), lambda: kv.attend(0, q), lambda: kv.gather(2),
                 lambda: kv.attend_tree(0, q), lambda: kv.evict(budget), lambda: kv.trim(10),
                 lambda: kv.keep_drafts(2, [1]), lambda: kv.reserve(200),
                 lambda: kv.observe(0, q, torch.zeros((B, 1, NQ), device="cuda"))):
        with pytest.raises(RuntimeError, match=r"evict\(\) failed"):
            call()
    if fails_in == 1:
        kv.trim(0)
    else:
        kv.release()
    for layer, (k, v) in enumerate(full):
        kv.append(layer, k, v)
    assert kv.offset == tokens == kv.next_position
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k) and torch.equal(got_v, v)


def test_an_eviction_that_cannot_choose_moves_nothing():
    print("[speculative] selection fails", flush=True)
    kv, full = filled(2, 100, 32, 1 << 40, seed=9)
    select, calls = ops.evict_select, []

    def fails(*args, **kw):
        calls.append(0)
        if len(calls) == 2:
            raise MemoryError("no room for the lists")
        return select(*args, **kw)

    ops.evict_select = fails
    try:
        with pytest.raises(MemoryError):
            kv.evict(40)
    finally:
        ops.evict_select = select
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k) and torch.equal(got_v, v)
    assert kv.evict(40) == 60


@pytest.mark.parametrize("fails_in", [0, 2])
def test_drafts_whose_spilled_pages_do_not_come_back_stay_as_they_are(fails_in):
    print(f"[speculative] keep_drafts fails in layer {fails_in}", flush=True)
    layers, tokens = 3, 130
    kv, full = filled(layers, tokens, 32, 1 << 40, seed=20 + fails_in)
    sums = [w.clone() for w in kv._weights]
    kv.spill([(layer, 3) for layer in range(layers)])  # tokens 96 .. 127
    reload = kv.reload

    def broken(pages=None, stream=None):
        if any(p.layer == fails_in for p in pages):
            raise OSError("a page file is gone")
        return reload(pages, stream)

    kv.reload = broken
    with pytest.raises(OSError, match="gone"):
        kv.keep_drafts(9, [1, 4, 8])
    kv.reload = reload
    assert kv.layer_lengths() == (tokens,) * layers and kv.offset == tokens
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k) and torch.equal(got_v, v)
        assert torch.equal(kv._weights[layer], sums[layer])
    kv.keep_drafts(9, [1, 4, 8])
    stay = list(range(tokens - 9)) + [tokens - 9 + i for i in (1, 4, 8)]
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k[:, :, stay]) and torch.equal(got_v, v[:, :, stay])
        assert torch.equal(kv._weights[layer][:, :, :len(stay)], sums[layer][:, :, stay])


@pytest.mark.parametrize("cut", ["all drafts", "trim", "each layer"])
def test_a_rollback_whose_spilled_pages_do_not_come_back_cuts_no_layer(cut):
    print(f"[speculative] rollback fails: {cut}", flush=True)
    layers, tokens = 3, 130
    kv, full = filled(layers, tokens, 32, 1 << 40, seed=30)
    kv.spill([(layer, 3) for layer in range(layers)])  # tokens 96 .. 127
    reload = kv.reload

    def broken(pages=None, stream=None):
        if any(p.layer == 2 for p in pages):
            raise OSError("a page file is gone")
        return reload(pages, stream)

    call = {"all drafts": lambda: kv.keep_drafts(9, []), "trim": lambda: kv.trim(tokens - 9),
            "each layer": lambda: kv.trim_layer_lengths([tokens - 9] * layers)}[cut]
    kv.reload = broken
    with pytest.raises(OSError, match="gone"):
        call()
    kv.reload = reload
    assert kv.layer_lengths() == (tokens,) * layers and kv.offset == tokens
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k) and torch.equal(got_v, v)
    call()
    assert kv.layer_lengths() == (tokens - 9,) * layers and kv.offset == tokens - 9
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k[:, :, :-9]) and torch.equal(got_v, v[:, :, :-9])


def test_a_released_cache_forgets_what_was_reserved():
    """Its counters are of the batch before: a later batch of another size is trimmed, cut to
    its accepted drafts and evicted as in a new cache."""
    print("[speculative] released after reserve", flush=True)
    kv = PagedKVCache(1, 1 << 40, page_positions=32)
    k = torch.randn((3, NKV, 60, D), device="cuda").to(torch.bfloat16)
    kv.append(0, k[:1, :, :20].contiguous(), k[:1, :, :20].contiguous())
    kv.reserve(64)
    kv.release()
    kv.append(0, k, k)
    with pytest.raises(ValueError, match="reserved 0"):
        kv.advance()
    kv.keep_drafts(4, [1, 3])
    assert torch.equal(kv.gather(0)[0], k[:, :, list(range(56)) + [57, 59]])
    kv.trim(50)
    kv._weights[0] = torch.rand((3, NKV, 64), device="cuda")
    assert kv.evict(30) == 20 and kv.offset == 30 and kv.next_position == 50


def test_an_eviction_reports_earlier_damage_before_it_moves_a_row():
    """Damage that attention met in the second layer's spilled pages is raised by the next
    call, which must not be in the middle of an eviction."""
    print("[speculative] pending integrity error", flush=True)
    kv, full = filled(2, 100, 32, 1 << 40, seed=40)
    sums = [w.clone() for w in kv._weights]
    kv.spill([(1, 1)])
    torch.cuda.synchronize()
    page = kv._pages[1][1]
    byte = page.host.part(1, page.host_j)
    byte[100] ^= 0x10
    kv.attend(1, torch.zeros((B, NQ, 1, D), dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    byte[100] ^= 0x10
    with pytest.raises(KVIntegrityError):
        kv.evict(40)
    for layer, (k, v) in enumerate(full):
        got_k, got_v = kv.gather(layer)
        assert torch.equal(got_k, k) and torch.equal(got_v, v)
    assert kv.evict(40) == 60
    for layer, (k, _) in enumerate(full):
        at = rows_kept(sums[layer], 100, 40)[..., None].expand(-1, -1, -1, D)
        assert torch.equal(kv.gather(layer)[0], k.gather(2, at))

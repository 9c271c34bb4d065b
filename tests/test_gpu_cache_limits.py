"""The operators on drafts and bounded caches at their largest sizes: batches of several
wavefronts' worth of sequences, windows of many drafts, pools past 2^32 elements.

Bars as where each operator is tested by itself: output 4e-3 in the 2-norm, LSE 2e-4
absolute, a weight 2e-4 of itself and a sum 2^-20; selection and moves are exact.
"""
import numpy as np
import pytest
import torch

from paged_inputs import cache, inputs, lens_tensor, trees
from voom_amd import ops
from voom_amd.page_pool import v_slot_shape

INF = float("inf")
REL, LSE_ABS = 4e-3, 2e-4
WEIGHT, SUM = 2e-4, 2.0 ** -20


def reference(q, k, v, ctx, n, sees):
    """fp64 (out [n, NQ, D], lse [n, NQ], weight [NKV, ctx]) of one sequence: the newest n of
    ctx tokens, row t sees drafts sees[t]; every row sees a key."""
    NQ, D = q.shape[0], q.shape[2]
    NKV = k.shape[0]
    k64, v64 = k[:, :ctx].double(), v[:, :ctx].double()
    q64 = q[:, :n].double().view(NKV, -1, n, D)
    s = torch.matmul(q64, k64[:, None].transpose(2, 3)) * D ** -0.5
    hidden = torch.zeros((n, ctx), dtype=torch.bool, device=q.device)
    hidden[:, ctx - n:] = ~sees[:n, :n]
    s.masked_fill_(hidden, -INF)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - lse[..., None])
    out = torch.matmul(w, v64[:, None]).view(NQ, n, D).transpose(0, 1)
    return out, lse.view(NQ, n).t(), w.sum((1, 2))


def check(out, lse, want, want_lse):
    assert (out.double() - want).norm() <= REL * want.norm()
    assert ((lse.double() - want_lse).abs() <= LSE_ABS).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,spare", [(65, 0), (200, 40), (1024, 0), (1024, 40)])
def test_batches_of_many_sequences(B, spare):
    """Tables of few pages are walked segment by segment, of many (``spare`` pages behind
    the contexts) cut into equal shares over all sequences."""
    print(f"[limits] B={B} spare={spare}", flush=True)
    NQ, NKV, D, PT, T, budget = 4, 2, 64, 32, 3, 60
    rng = np.random.default_rng(B)
    ctx = rng.integers(0, 200, B)
    ctx[rng.random(B) < 0.3] = 0
    ctx[[0, B - 1]] = 0
    ctx[B // 2] = 200
    lens = np.minimum(rng.integers(0, T + 1, B), ctx)
    q, k, v = inputs(B, NQ, NKV, D, 200, T)
    k_pool, v_pool, table = cache(k, v, PT, spare=spare)
    sees = trees(B, T, 3).cuda()
    ctx_t, lens_t = lens_tensor(ctx.tolist()), lens_tensor(lens.tolist())
    out, lse = ops.paged_gqa_tree(q, k_pool, v_pool, table, ctx_t, mask=sees, draft_lens=lens_t,
                                  return_lse=True)
    _, causal = ops.paged_gqa_tree(q, k_pool, v_pool, table, ctx_t, draft_lens=lens_t,
                                   return_lse=True)
    sums = torch.zeros((B, NKV, 203), device="cuda")
    ops.paged_gqa_observe(q, causal, k_pool, table, ctx_t, sums, window_lens=lens_t)
    tril = torch.ones((T, T), dtype=torch.bool, device="cuda").tril()
    for b in range(B):
        n, c = int(lens[b]), int(ctx[b])
        assert (out[b, n:] == 0).all() and (lse[b, n:] == -INF).all()
        assert (sums[b, :, c:] == 0).all()
        if n == 0:
            assert (sums[b] == 0).all()
            continue
        want, want_lse, _ = reference(q[b], k[b], v[b], c, n, sees[b])
        check(out[b, :n], lse[b, :n], want, want_lse)
        _, _, weight = reference(q[b], k[b], v[b], c, n, tril)
        # (the LSE given is the kernel's, off by LSE_ABS)
        assert ((sums[b, :, :c].double() - weight).abs()
                <= (WEIGHT + 2 * LSE_ABS + SUM) * weight).all()
    keep, counts = ops.evict_select(sums, ctx_t, budget, sink=2, recent=8)
    gk, gv = ops.gather_kv(k_pool, v_pool, table, 200)
    before = sums.clone()
    ops.compact_kv(k_pool, v_pool, table, keep, counts, scores=sums)
    tk, tv = ops.gather_kv(k_pool, v_pool, table, 200)
    assert torch.equal(counts, ctx_t.clamp(max=budget))
    for b in range(B):
        m = int(counts[b])
        for h in range(NKV):
            at = keep[b, h, :m].long()
            assert m < 2 or (at[1:] > at[:-1]).all()
            assert (keep[b, h, m:] == -1).all()
            assert torch.equal(tk[b, h, :m], gk[b, h, at])
            assert torch.equal(tv[b, h, :m], gv[b, h, at])
            assert torch.equal(sums[b, h, :m], before[b, h, at]) and (sums[b, h, m:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_windows_of_several_loads_in_a_large_batch(D):
    """Windows whose rows go through the keys once, twice or three times, in one call."""
    print(f"[limits] windows of several loads, D={D}", flush=True)
    B, NQ, NKV, L = 70, 8, 2, 150
    rng = np.random.default_rng(D)
    ctx = rng.integers(0, 900, B)
    ctx[[3, 69]] = 0
    ctx[40] = 900
    lens = np.minimum(rng.integers(0, L + 1, B), ctx)
    lens[40] = L
    q, k, v = inputs(B, NQ, NKV, D, 900, L)
    k_pool, v_pool, table = cache(k, v, 64)
    ctx_t, lens_t = lens_tensor(ctx.tolist()), lens_tensor(lens.tolist())
    _, lse = ops.paged_gqa_tree(q, k_pool, v_pool, table, ctx_t, draft_lens=lens_t,
                                return_lse=True)
    sums = torch.full((B, NKV, 901), 0.25, device="cuda")
    ops.paged_gqa_observe(q, lse, k_pool, table, ctx_t, sums, window_lens=lens_t)
    tril = torch.ones((L, L), dtype=torch.bool, device="cuda").tril()
    for b in range(B):
        n, c = int(lens[b]), int(ctx[b])
        assert (sums[b, :, c:] == 0.25).all()
        if n == 0:
            assert (sums[b] == 0.25).all()
            continue
        _, want_lse, weight = reference(q[b], k[b], v[b], c, n, tril)
        assert ((lse[b, :n].double() - want_lse).abs() <= LSE_ABS).all()
        # three loads: three more roundings of the sum than where a window is one
        assert ((sums[b, :, :c].double() - weight - 0.25).abs()
                <= (WEIGHT + 2 * LSE_ABS) * weight + 4 * SUM * (weight + 0.25)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("NQ,NKV,D,ctx", [(2, 1, 64, 1500), (2, 2, 128, 1024)])
def test_as_many_drafts_as_a_call_takes(NQ, NKV, D, ctx):
    T = 1024
    print(f"[limits] T={T} D={D} ctx={ctx}", flush=True)
    q, k, v = inputs(1, NQ, NKV, D, ctx, T)
    k_pool, v_pool, table = cache(k, v, 64)
    tril = torch.ones((T, T), dtype=torch.bool, device="cuda").tril()
    for sees, mask in ((trees(1, T, 7).cuda(), True), (tril[None], False)):
        out, lse = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([ctx]),
                                      mask=sees if mask else None, return_lse=True)
        want, want_lse, weight = reference(q[0], k[0], v[0], ctx, T, sees[0])
        check(out[0], lse[0], want, want_lse)
    sums = torch.zeros((1, NKV, ctx), device="cuda")
    ops.paged_gqa_observe(q, lse, k_pool, table, lens_tensor([ctx]), sums)
    # up to 2,048 rows are added, 32 or more of them at a time: chains of 64 sums at most
    assert ((sums[0].double() - weight).abs()
            <= (WEIGHT + 2 * LSE_ABS + 64 * 2.0 ** -24 + SUM) * weight).all()


@pytest.mark.gpu
def test_pools_past_2_to_the_32_elements():
    """The same calls on a small pool and on the last slots of one of 4.46e9 elements."""
    NQ, NKV, D, PT, B, L, T = 16, 8, 128, 256, 2, 700, 5
    pages = -(-L // PT)
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((B, L, (NQ + 2 * NKV) * D), generator=g, device="cuda").bfloat16()
    cos, sin = ops.rope_cache(L, D, 1e4)
    positions = torch.arange(L, dtype=torch.int32, device="cuda").repeat(B, 1)
    got = []
    for slots in (B * pages, 17000):
        print(f"[limits] {slots} slots", flush=True)
        k_pool = torch.empty((slots, NKV, PT, D), dtype=torch.bfloat16, device="cuda")
        v_pool = torch.empty((slots,) + v_slot_shape(NKV, D, PT), dtype=torch.bfloat16,
                             device="cuda")
        table = (slots - 1 - torch.arange(B * pages, device="cuda")).int().view(B, pages)
        ctx = lens_tensor([L] * B)
        q = ops.qk_norm_rope_append(qkv, cos, sin, positions, k_pool, v_pool, table,
                                    lens_tensor([0] * B), NQ, NKV)
        new = q[:, :, L - T:].contiguous()
        out, lse = ops.paged_gqa_tree(new, k_pool, v_pool, table, ctx, return_lse=True)
        sums = torch.zeros((B, NKV, L), device="cuda")
        ops.paged_gqa_observe(new, lse, k_pool, table, ctx, sums)
        keep, counts = ops.evict_select(sums, ctx, 300, sink=4, recent=32)
        before = [k_pool[table.long()].clone(), v_pool[table.long()].clone()]
        ops.compact_kv(k_pool, v_pool, table, keep, counts, scores=sums)
        after = [k_pool[table[:, :1].long()].clone(), v_pool[table[:, :1].long()].clone()]
        # the last page ends behind the last token: what lies there is not compared
        heads = [x[:, :2] for x in before]
        got.append([q, out, lse, sums, keep, counts] + heads + after)
        torch.cuda.synchronize()
        del k_pool, v_pool
        torch.cuda.empty_cache()
    assert slots * NKV * PT * D > 2 ** 32
    for small, far in zip(*got):
        assert torch.equal(small, far)

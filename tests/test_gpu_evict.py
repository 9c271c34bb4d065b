"""GPU parity of the operators that keep a paged cache within a budget: the attention weight
that tokens receive (ops.paged_gqa_observe) against fp64, the selection (ops.evict_select)
and the move of what stays (ops.compact_kv) exactly.

Bar of the weights.  A score is a sum of D products of bf16 values in fp32, off by at most
D 2^-24 sum |q k| scale (1.1e-4 at D = 128, |q| 1.6 and |k| 0.8 on average, scale D^-0.5);
the scaling and the base-2 exponent add 2^-23 of their size (under 40), the fp32 log-sum-exp
2^-24 of its own: a weight is off by less than 2e-4 of itself, and the sum of non-negative
terms and the earlier sum by 2^-20 (sums of at most 16 terms in a chain, then a tree).
"""
import numpy as np
import pytest
import torch

from paged_inputs import cache, inputs, lens_tensor
from voom_amd import _lib, ops

INF, NAN = float("inf"), float("nan")
WEIGHT, SUM = 2e-4, 2.0 ** -20


# ---- the weights ------------------------------------------------------------------


def window_reference(q, k, ctx, lens, scale):
    """fp64 (lse [B, L, NQ], added weight [B, NKV, S]) of causal windows."""
    B, NQ, L, D = q.shape
    NKV, S = k.shape[1:3]
    G = NQ // NKV
    q, k = q.double().cpu(), k.double().cpu()
    lse = torch.full((B, L, NQ), -INF, dtype=torch.float64)
    added = torch.zeros((B, NKV, S), dtype=torch.float64)
    for b in range(B):
        for t in range(lens[b]):
            see = ctx[b] - lens[b] + t + 1
            for h in range(NQ):
                s = k[b, h // G, :see] @ q[b, h, t] * scale
                lse[b, t, h] = torch.logsumexp(s, 0)
                if lse[b, t, h] > -INF:
                    added[b, h // G, :see] += torch.exp(s - lse[b, t, h])
    return lse, added


@pytest.mark.gpu
@pytest.mark.parametrize("B,NQ,NKV,D,PT,L,ctx,lens", [
    (1, 9, 3, 64, 64, 1, [1], None),                      # one token
    (1, 9, 3, 64, 64, 1, [640], None),
    (3, 32, 8, 128, 64, 1, [700, 0, 257], None),          # decode, an empty sequence
    (2, 28, 4, 128, 32, 33, [600, 33], [33, 7]),          # a window; nothing before it
    (2, 8, 2, 64, 256, 90, [1000, 90], [90, 0]),          # rows in two loads; no window
    (1, 40, 2, 128, 64, 30, [300], None),                 # 20 heads a group, three loads
    (4, 16, 1, 128, 4096, 5, [4097, 5, 256, 255], None),  # the largest page
])
def test_weights_against_fp64(B, NQ, NKV, D, PT, L, ctx, lens):
    print(f"[observe] B={B} NQ={NQ} NKV={NKV} D={D} PT={PT} L={L} ctx={ctx} lens={lens}",
          flush=True)
    q, k, v = inputs(B, NQ, NKV, D, max(ctx), L)
    n = [min(x, c) for x, c in zip(lens or [L] * B, ctx)]
    k_pool, _, table = cache(k, v, PT)
    lse, added = window_reference(q, k, ctx, n, D ** -0.5)
    cap = max(ctx) + 3
    before = torch.rand((B, NKV, cap), device="cuda")
    args = (q, lse.float().cuda(), k_pool, table, lens_tensor(ctx))
    kw = dict(window_lens=None if lens is None else lens_tensor(lens))
    out = torch.full_like(before, -7.0)
    got = ops.paged_gqa_observe(*args, before, out=out, **kw)
    assert got is out
    here = before.clone()
    assert ops.paged_gqa_observe(*args, here, **kw) is here
    torch.cuda.synchronize()
    for b in range(B):
        c = ctx[b]
        assert torch.equal(out[b, :, :c], here[b, :, :c])
        assert (out[b, :, c:] == -7.0).all() and torch.equal(here[b, :, c:], before[b, :, c:])
        want = before[b, :, :c].double().cpu() + added[b, :, :c]
        bar = WEIGHT * added[b, :, :c] + SUM * want
        assert ((out[b, :, :c].double().cpu() - want).abs() <= bar).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.7])
def test_weight_scales_and_one_token_lse(scale):
    print(f"[observe] scale={scale}", flush=True)
    q, k, v = inputs(2, 8, 2, 64, 300, 1, seed=3)
    k_pool, _, table = cache(k, v, 32)
    lse, added = window_reference(q, k, [300, 200], [1, 1], scale)
    zero = torch.zeros((2, 2, 320), device="cuda")
    out = ops.paged_gqa_observe(q, lse[:, 0].float().cuda(), k_pool, table, lens_tensor([300, 200]),
                                zero, scale=scale)
    torch.cuda.synchronize()
    assert (out[1, :, 200:] == 0).all() and (out[:, :, 300:] == 0).all()
    off = (out[:, :, :300].double().cpu() - added).abs()
    assert (off <= WEIGHT * added + SUM * added).all()


@pytest.mark.gpu
def test_rows_without_a_sum_and_bad_values_stay_where_they_are():
    """A log-sum-exp of -inf adds nothing, NaN in unseen keys and in rows past the window
    reaches nothing, lengths out of range are clamped; calls without rows change nothing."""
    print("[observe] empty rows, NaN, clamps", flush=True)
    B, NQ, NKV, D, L, S = 1, 4, 2, 128, 6, 90
    q, k, v = inputs(B, NQ, NKV, D, S, L, seed=4)
    n = 4
    lse, added = window_reference(q, k, [S], [n], D ** -0.5)
    k[:, 0, S - 1] = NAN  # the window's last token: seen by its own row alone
    q[:, :, n:] = NAN
    lse[:, n:] = NAN
    lse[0, n - 1, :2] = -INF  # that row's heads of kv head 0
    k_pool, _, table = cache(k, v, 32)
    zero = torch.zeros((B, NKV, 96), device="cuda")
    got = ops.paged_gqa_observe(q, lse.float().cuda(), k_pool, table, lens_tensor([S]), zero.clone(),
                                window_lens=lens_tensor([n]))
    torch.cuda.synchronize()
    _, fewer = window_reference(q[:, :, :n - 1], k[:, :, :S - 1], [S - 1], [n - 1], D ** -0.5)
    got = got.double().cpu()
    bar = (WEIGHT + SUM) * fewer[0, 0]
    assert ((got[0, 0, :S - 1] - fewer[0, 0]).abs() <= bar).all() and got[0, 0, S - 1] == 0
    assert ((got[0, 1, :S] - added[0, 1]).abs() <= (WEIGHT + SUM) * added[0, 1]).all()
    # a context past the scores and the table, more window rows than rows
    short = torch.zeros((B, NKV, 50), device="cuda")
    q, k, v = inputs(B, NQ, NKV, D, S, L, seed=5)
    k_pool, _, table = cache(k, v, 32)
    lse, added = window_reference(q, k, [50], [L], D ** -0.5)
    ops.paged_gqa_observe(q, lse.float().cuda(), k_pool, table, lens_tensor([1000]), short,
                          window_lens=lens_tensor([77]))
    torch.cuda.synchronize()
    got = short.double().cpu()
    assert ((got - added[..., :50]).abs() <= (WEIGHT + SUM) * added[..., :50]).all()
    same = zero + 3
    ops.paged_gqa_observe(q, lse.float().cuda(), k_pool, table, lens_tensor([-4]), same)
    ops.paged_gqa_observe(q[:, :, :0].contiguous(), lse[:, :0].float().cuda(), k_pool, table,
                          lens_tensor([S]), same)
    ops.paged_gqa_observe(q[:0], lse[:0].float().cuda(), k_pool, table[:0], lens_tensor([]),
                          same[:0])
    assert (same == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("S", [90, 700])
def test_a_row_whose_lse_is_nan_reaches_what_it_sees_and_nothing_else(S):
    print(f"[observe] NaN and infinite lse, S={S}", flush=True)
    B, NQ, NKV, D, L = 1, 4, 2, 128, 5
    q, k, v = inputs(B, NQ, NKV, D, S, L, seed=14)
    k_pool, _, table = cache(k, v, 32)
    lse, _ = window_reference(q, k, [S], [L], D ** -0.5)
    lse = lse.float().cuda()
    less = lse.clone()
    lse[0, 1, 0], less[0, 1, 0] = NAN, -INF     # a head of kv head 0; sees up to S - 4
    lse[0, 3, 3], less[0, 3, 3] = INF, -INF     # exp(-inf) is 0
    got, without = (ops.paged_gqa_observe(q, x, k_pool, table, lens_tensor([S]),
                                          torch.zeros((B, NKV, S), device="cuda"))
                    for x in (lse, less))
    torch.cuda.synchronize()
    assert torch.isnan(got[0, 0, :S - 3]).all()
    assert torch.equal(got[0, 0, S - 3:], without[0, 0, S - 3:])
    assert torch.equal(got[0, 1], without[0, 1])


# ---- the selection ------------------------------------------------------------------


def select_reference(scores, ctx, budget, sink, recent):
    B, NKV, cap = scores.shape
    keep = np.full((B, NKV, budget), -1, np.int32)
    lens = np.zeros(B, np.int32)
    for b in range(B):
        c = min(max(ctx[b], 0), cap)
        lens[b] = min(c, budget)
        for h in range(NKV):
            if c <= budget:
                keep[b, h, :c] = np.arange(c)
                continue
            s = scores[b, h, sink:c - recent].astype(np.float64)
            s[np.isnan(s)] = -np.inf
            lowest = np.isnan(scores[b, h, sink:c - recent])  # below -inf
            order = sorted(range(len(s)), key=lambda i: (lowest[i], -s[i], i))
            mid = np.array(order[:budget - sink - recent], np.int64) + sink
            keep[b, h] = np.sort(np.concatenate([np.arange(sink), mid, np.arange(c - recent, c)]))
    return keep, lens


def select_case(name, rng, B, NKV, cap):
    s = rng.random((B, NKV, cap)).astype(np.float32)
    if name == "ties":
        s = np.round(s * 4) / 4
    elif name == "zeros":
        s[s < 0.9] = 0
        s[rng.random(s.shape) < 0.3] *= -1  # -0 and negative numbers
    elif name == "odd":
        for value, share in ((NAN, 0.2), (INF, 0.1), (-INF, 0.1), (1e-42, 0.1), (-1e-42, 0.1),
                             (-0.0, 0.1)):
            s[rng.random(s.shape) < share] = value
    elif name == "equal":
        s[:] = 0.5
    elif name == "wide":
        s = np.exp(40 * (s - 0.5)).astype(np.float32)
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["plain", "ties", "zeros", "odd", "equal", "wide"])
@pytest.mark.parametrize("cap,ctx,budget,sink,recent", [
    (2, [2, 1, 0], 1, 0, 0),
    (100, [100, 64, 33], 32, 4, 8),
    (640, [640, 577, 576], 576, 4, 64),
    (1500, [1500, 1100, 2000], 1000, 0, 1000),  # nothing to choose; past the scores
    (5003, [5003, 4096, -3], 511, 500, 0),
    (40000, [40000, 33000, 16384], 4096, 4, 256),
    (140001, [140001, 131072, 1], 1, 0, 0),
])
def test_selection_is_exact(name, cap, ctx, budget, sink, recent):
    print(f"[select] {name} cap={cap} budget={budget} sink={sink} recent={recent}", flush=True)
    s = select_case(name, np.random.default_rng(cap + budget), 3, 2, cap)
    keep, lens = ops.evict_select(torch.from_numpy(s).cuda(), lens_tensor(ctx), budget, sink=sink,
                                  recent=recent)
    torch.cuda.synchronize()
    want, want_lens = select_reference(s, ctx, budget, sink, recent)
    assert np.array_equal(lens.cpu().numpy(), want_lens)
    assert np.array_equal(keep.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["ties", "odd", "equal"])
@pytest.mark.parametrize("B,NKV,cap,budget,sink,recent", [
    (33, 2, 40000, 5000, 4, 100),      # more long rows than are cut into pieces
    (1, 2, 1048576, 65536, 4, 1000),   # as many pieces as a row is cut into
    (1, 1, 1048577, 3, 1, 1),          # one token more
    (1, 3, 32769, 32000, 16000, 16000),  # nothing to choose
    (2, 1, 50000, 49999, 0, 0),        # all but one
])
def test_long_rows(name, B, NKV, cap, budget, sink, recent):
    print(f"[select] {name} B={B} cap={cap} budget={budget}", flush=True)
    rng = np.random.default_rng(cap)
    s = select_case(name, rng, B, NKV, cap)
    ctx = [cap - (17 * b) % cap for b in range(B)]
    scores, lens = torch.from_numpy(s).cuda(), lens_tensor(ctx)
    keep, counts = ops.evict_select(scores, lens, budget, sink=sink, recent=recent)
    one = torch.empty_like(keep)  # the same by one workgroup per row
    assert _lib.lib().voom_evict_select(scores.data_ptr(), lens.data_ptr(), one.data_ptr(),
                                        counts.data_ptr(), B, NKV, cap, budget, sink, recent,
                                        0) == 0
    torch.cuda.synchronize()
    assert torch.equal(keep, one)
    for b in range(B):
        assert int(counts[b]) == min(ctx[b], budget)
        for h in range(NKV):
            x = s[b, h, sink:ctx[b] - recent].astype(np.float64)
            lowest = np.isnan(x)
            x[lowest] = -np.inf
            order = np.lexsort((np.arange(len(x)), -x, lowest))[:budget - sink - recent]
            want = np.sort(np.concatenate([np.arange(sink), order + sink,
                                           np.arange(ctx[b] - recent, ctx[b])]))
            want = want if ctx[b] > budget else np.arange(ctx[b])
            got = keep[b, h].cpu().numpy()
            assert np.array_equal(got[:len(want)], want) and (got[len(want):] == -1).all()


@pytest.mark.gpu
def test_long_rows_in_a_graph_and_on_two_streams():
    """Each call has a workspace of its own."""
    print("[select] long rows replayed and on two streams", flush=True)
    scores = [torch.rand((1, 4, 70000), device="cuda") ** 3 for _ in range(2)]
    ctx = lens_tensor([70000])
    want = [ops.evict_select(s, ctx, 4000, sink=4, recent=64)[0] for s in scores]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, stream in zip(scores, side):
            with torch.cuda.stream(stream):
                got.append(ops.evict_select(s, ctx, 4000, sink=4, recent=64)[0])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    live = scores[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep, _ = ops.evict_select(live, ctx, 4000, sink=4, recent=64)
    for i in (0, 1, 0, 1):
        live.copy_(scores[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(keep, want[i])


# ---- the move -----------------------------------------------------------------------


def kept_lists(rng, B, H, n, start, ctx):
    """Random ascending positions in [start, ctx) of random counts, the first sequence's
    list full."""
    keep = np.full((B, H, n), -1, np.int32)
    lens = np.array([n] + [int(rng.integers(0, n + 1)) for _ in range(B - 1)], np.int32)
    for b in range(B):
        for h in range(H):
            keep[b, h, :lens[b]] = np.sort(rng.choice(np.arange(start[b], ctx), lens[b], False))
    return keep, lens


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["in place", "other pages", "mixed pages"])
@pytest.mark.parametrize("B,NKV,D,PT,ctx,n,per_head,start", [
    (1, 1, 32, 1, 9, 4, True, False),        # one-token pages, the smallest head
    (2, 3, 64, 16, 100, 37, True, False),    # pages below a V block
    (3, 2, 128, 64, 700, 5, False, True),    # an accepted branch
    (2, 2, 96, 32, 300, 299, True, True),    # nearly all of it
    (1, 4, 128, 256, 3000, 1100, True, False),  # more rows than one step
    (1, 2, 128, 64, 2500, 2500, False, False),  # every row: nothing moves in place
])
def test_move_is_exact(where, B, NKV, D, PT, ctx, n, per_head, start):
    print(f"[compact] {where} B={B} NKV={NKV} D={D} PT={PT} ctx={ctx} n={n}", flush=True)
    rng = np.random.default_rng(ctx + n)
    _, k, v = inputs(B, NKV, NKV, D, ctx, 1)
    pages = -(-ctx // PT)
    k_pool, v_pool, both = cache(k, v, PT, spare=pages)
    table, other = both[:, :pages].contiguous(), both[:, pages:].contiguous()
    k_pool[torch.isnan(k_pool)] = 0  # gather compares bits
    v_pool[torch.isnan(v_pool)] = 0
    at = rng.integers(0, max(ctx - n, 1), B) if start else np.zeros(B, np.int64)
    keep, lens = kept_lists(rng, B, NKV if per_head else 1, n, at, ctx)
    if where == "mixed pages":  # every other page is the sequence's own
        other[:, ::2] = table[:, ::2]
    dst = None if where == "in place" else other
    to = table if dst is None else dst
    want_k, want_v = (x.clone() for x in ops.gather_kv(k_pool, v_pool, to, ctx))
    src_k, src_v = ops.gather_kv(k_pool, v_pool, table, ctx)
    scores = torch.rand((B, NKV, ctx + 5), device="cuda")
    want_s = torch.zeros_like(scores)
    for b in range(B):
        want_s[b, :, :at[b]] = scores[b, :, :at[b]]
        for h in range(NKV):
            i = torch.from_numpy(keep[b, h if per_head else 0, :lens[b]]).long().cuda()
            rows = slice(int(at[b]), int(at[b] + lens[b]))
            want_k[b, h, rows], want_v[b, h, rows] = src_k[b, h, i], src_v[b, h, i]
            want_s[b, h, rows] = scores[b, h, i]
    moved = torch.empty_like(scores) if where == "other pages" else None
    ops.compact_kv(k_pool, v_pool, table, torch.from_numpy(keep).cuda(), lens_tensor(lens),
                   start=lens_tensor(at) if start else None, dst_table=dst, scores=scores,
                   scores_out=moved)
    torch.cuda.synchronize()
    got_k, got_v = ops.gather_kv(k_pool, v_pool, to, ctx)
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    assert torch.equal(scores if moved is None else moved, want_s)


@pytest.mark.gpu
@pytest.mark.parametrize("n,start,lowest", [
    (4096, 5000, 0), (4097, 5000, 0),   # both sides of what is read at once
    (10000, 5000, 0),                   # all of them move back
    (10000, 2500, 1000),                # the first ones back, the others forward
    (9000, 300, 500),                   # all forward
    (8193, 0, 0),
])
@pytest.mark.parametrize("own_array", [True, False])
def test_scores_of_long_lists_that_go_to_other_pages(n, start, lowest, own_array):
    """K and V may go to any place of other pages, and the scores go along, in their own
    array too."""
    print(f"[compact] scores n={n} start={start} lowest={lowest} own_array={own_array}", flush=True)
    NKV, D, PT, ctx = 2, 32, 64, 15100
    rng = np.random.default_rng(n + start)
    _, k, v = inputs(1, NKV, NKV, D, ctx, 1)
    pages = -(-ctx // PT)
    k_pool, v_pool, both = cache(k, v, PT, spare=pages)
    table, other = both[:, :pages].contiguous(), both[:, pages:].contiguous()
    keep = np.stack([np.arange(lowest, lowest + n), np.arange(lowest, lowest + n)])
    if lowest != 0:  # a gap in the second head's list, further on in the first's
        keep[0, n // 2:] += 3000
        keep[1] = np.sort(rng.choice(np.arange(lowest, ctx), n, False))
    behind = keep >= start + np.arange(n)
    assert {(5000, 0): not behind.any(), (2500, 1000): behind.any() and not behind.all(),
            (300, 500): behind.all(), (0, 0): behind.all()}[start, lowest]
    at = torch.from_numpy(keep).cuda()
    scores = torch.rand((1, NKV, ctx + 7), device="cuda")
    want = torch.zeros_like(scores)
    want[:, :, :start] = scores[:, :, :start]
    want[0, :, start:start + n] = scores[0].gather(1, at)
    out = scores if own_array else torch.empty_like(scores)
    ops.compact_kv(k_pool, v_pool, table, at[None].int(), lens_tensor([n]),
                   start=lens_tensor([start]), dst_table=other, scores=scores, scores_out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    got_k, got_v = ops.gather_kv(k_pool, v_pool, other, start + n)
    rows = at[..., None].expand(-1, -1, D)
    assert torch.equal(got_k[0, :, start:], k[0].gather(1, rows))
    assert torch.equal(got_v[0, :, start:], v[0].gather(1, rows))


@pytest.mark.gpu
def test_rows_outside_the_tables_are_left_out():
    print("[compact] bad positions, slots and counts", flush=True)
    _, k, v = inputs(2, 2, 2, 64, 128, 1, seed=9)
    k_pool, v_pool, table = cache(k, v, 32)
    bad = table.clone()
    bad[0, 1], bad[1, 2] = -1, 1 << 20
    keep = torch.tensor([[[2, 40, 70, 1000]], [[-5, 70, 100, 127]]], dtype=torch.int32,
                        device="cuda")
    before_k, before_v = ops.gather_kv(k_pool, v_pool, table, 128)
    ops.compact_kv(k_pool, v_pool, bad, keep, lens_tensor([4, 9]))
    torch.cuda.synchronize()
    k2, v2 = ops.gather_kv(k_pool, v_pool, table, 128)
    for x, y in ((k2, before_k), (v2, before_v)):
        want = y.clone()
        want[0, :, 0], want[0, :, 2] = y[0, :, 2], y[0, :, 70]  # 40 has no page, 1000 is outside
        want[1, :, 2], want[1, :, 3] = y[1, :, 100], y[1, :, 127]  # -5; 70 has no page
        assert torch.equal(x, want)
    # rows past the table, a negative start, a negative count, no rows at all
    ops.compact_kv(k_pool, v_pool, table, keep[:, :, 3:].clamp(0, 127).contiguous(),
                   lens_tensor([1, -1]), start=lens_tensor([2 ** 31 - 1, -3]))
    scores = torch.ones((2, 2, 128), device="cuda")
    ops.compact_kv(k_pool, v_pool, table, keep[:, :, :0].contiguous(), lens_tensor([0, 0]),
                   start=lens_tensor([5, 200]), scores=scores)
    torch.cuda.synchronize()
    again = ops.gather_kv(k_pool, v_pool, table, 128)
    assert torch.equal(again[0], k2) and torch.equal(again[1], v2)
    assert (scores[0, :, :5] == 1).all() and (scores[0, :, 5:] == 0).all()
    assert (scores[1] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad_page", [0, 12, 30])
@pytest.mark.parametrize("B,D", [(1, 96), (33, 64)])
def test_a_page_outside_the_pool_in_a_long_list(B, D, bad_page):
    """Lists of several steps, a page of one sequence -1: what would come from it or go to
    it stays, all else is moved."""
    print(f"[compact] bad page {bad_page} B={B} D={D}", flush=True)
    NKV, PT, ctx, n = 2, 64, 2500, 1400
    rng = np.random.default_rng(bad_page)
    _, k, v = inputs(B, NKV, NKV, D, ctx, 1)
    k_pool, v_pool, table = cache(k, v, PT)
    k_pool[torch.isnan(k_pool)] = 0
    v_pool[torch.isnan(v_pool)] = 0
    keep, lens = kept_lists(rng, B, NKV, n, np.zeros(B, np.int64), ctx)
    src_k, src_v = ops.gather_kv(k_pool, v_pool, table, ctx)
    want_k, want_v = src_k.clone(), src_v.clone()
    for b in range(B):
        for h in range(NKV):
            for_b = keep[b, h, :lens[b]]
            to = np.arange(lens[b])
            if b == 0:
                moved = (for_b // PT != bad_page) & (to // PT != bad_page)
                for_b, to = for_b[moved], to[moved]
            want_k[b, h, torch.from_numpy(to)] = src_k[b, h, torch.from_numpy(for_b).long()]
            want_v[b, h, torch.from_numpy(to)] = src_v[b, h, torch.from_numpy(for_b).long()]
    broken = table.clone()
    broken[0, bad_page] = -1
    ops.compact_kv(k_pool, v_pool, broken, torch.from_numpy(keep).cuda(), lens_tensor(lens))
    torch.cuda.synchronize()
    got_k, got_v = ops.gather_kv(k_pool, v_pool, table, ctx)
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)


@pytest.mark.gpu
def test_checked_lists_raise():
    _, k, v = inputs(1, 1, 1, 64, 64, 1)
    k_pool, v_pool, table = cache(k, v, 32)

    def move(keep, n, start=0, dst=None):
        ops.compact_kv(k_pool, v_pool, table, torch.tensor([[keep]], dtype=torch.int32).cuda(),
                       lens_tensor([n]), start=lens_tensor([start]), dst_table=dst)

    ops.set_bounds_checks(True)
    try:
        move([1, 5, -1], 2)
        for match, args in (("ascend", ([5, 1], 2)), ("ascend", ([5, 5], 2)),
                            ("outside", ([1, 64], 2)), ("outside", ([-1, 3], 2)),
                            ("keep_lens", ([1, 2], 3)), ("in place", ([1, 2], 2, 2))):
            with pytest.raises(ValueError, match=match):
                move(*args)
        other = torch.tensor([[1, 0]], dtype=torch.int32).cuda() if table[0, 0] == 0 else (
            torch.tensor([[0, 1]], dtype=torch.int32).cuda())
        assert (other != table).all()
        for match, args in (("own pages", ([1, 2], 2, 2, table.clone())),
                            ("read elsewhere", ([1, 40], 2, 0, other)),
                            ("twice", ([1, 2, 3], 3, 31, other * 0 + 1 - table[0, 0]))):
            with pytest.raises(ValueError, match=match):
                move(*args)
        move([1, 2], 2, 2, other)  # page 1 of the pool is not read
        move([5, 6], 2, 2, table.clone())
    finally:
        ops.set_bounds_checks(False)


@pytest.mark.gpu
def test_graph_replays():
    """Observe, select and the move captured together, eager calls between the replays."""
    print("[evict] graph replay", flush=True)
    q, k, v = inputs(2, 8, 2, 128, 900, 1, seed=12)
    k_pool, v_pool, both = cache(k, v, 64, spare=16)
    table, other = both[:, :15].contiguous(), both[:, 15:].contiguous()
    ctx = lens_tensor([900, 300])
    scores = torch.rand((2, 2, 960), device="cuda")

    def run():
        _, lse = ops.paged_gqa_decode(q, k_pool, v_pool, table, ctx, return_lse=True)
        sums = ops.paged_gqa_observe(q, lse, k_pool, table, ctx, scores,
                                     out=torch.zeros_like(scores))
        keep, lens = ops.evict_select(sums, ctx, 400, sink=4, recent=32)
        moved = torch.empty_like(sums)
        ops.compact_kv(k_pool, v_pool, table, keep, lens, dst_table=other, scores=sums,
                       scores_out=moved)
        return (sums, keep, lens, moved) + ops.gather_kv(k_pool, v_pool, other, 400)

    eager = [t.clone() for t in run()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    keep_alive = list(ops._WORKSPACES.values())
    for _ in range(3):
        for t in outs:
            t.zero_()
        run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(outs, eager))
    del keep_alive


# ---- refusals -----------------------------------------------------------------------


@pytest.mark.gpu
def test_wrapper_refusals():
    q, k, v = inputs(2, 8, 2, 64, 40, 3)
    k_pool, v_pool, table = cache(k, v, 32)
    ctx, lse = lens_tensor([40, 40]), torch.zeros((2, 3, 8), device="cuda")
    scores = torch.zeros((2, 2, 64), device="cuda")
    keep, lens = torch.zeros((2, 2, 5), dtype=torch.int32, device="cuda"), lens_tensor([5, 5])

    def refused(match, fn, *args, **kw):
        with pytest.raises(ValueError, match=match):
            fn(*args, **kw)

    good = dict(q=q, lse=lse, k_pool=k_pool, table=table, ctx=ctx, scores=scores)
    for match, change in (
            ("ROCm", dict(q=q.cpu())), ("contiguous", dict(q=q.transpose(1, 2))),
            ("lse", dict(lse=lse[:, :2].contiguous())), ("lse", dict(lse=lse.double())),
            ("head_dim", dict(q=torch.cat((q, q), -1))), ("bfloat16", dict(q=q.half())),
            ("multiple", dict(q=q[:, :7].contiguous(), lse=lse[..., :7].contiguous())),
            ("table", dict(table=table.long())), ("ctx", dict(ctx=ctx[:1])),
            ("scores", dict(scores=scores[:, :1].contiguous())),
            ("scores", dict(scores=scores.double())), ("scores", dict(scores=scores[..., :0]))):
        refused(match, ops.paged_gqa_observe, *{**good, **change}.values())
    refused("window_lens", ops.paged_gqa_observe, *good.values(), window_lens=lens[:1])
    refused("out", ops.paged_gqa_observe, *good.values(), out=scores[..., :3].contiguous())
    refused("finite", ops.paged_gqa_observe, *good.values(), scale=INF)

    refused("scores", ops.evict_select, scores[0], ctx, 5)
    refused("scores", ops.evict_select, scores.half(), ctx, 5)
    refused("ctx", ops.evict_select, scores, ctx.long(), 5)
    for budget, sink, recent in ((0, 0, 0), (5, 3, 3), (5, -1, 0), (5, 0, -1)):
        refused("budget", ops.evict_select, scores, ctx, budget, sink=sink, recent=recent)

    good = dict(k=k_pool, v=v_pool, table=table, keep=keep, lens=lens)
    for match, change in (
            ("ROCm", dict(keep=keep.cpu())), ("bfloat16", dict(k=k_pool.half())),
            ("v_pool", dict(v=v_pool.transpose(2, 3).contiguous())),
            ("table", dict(table=table[0])), ("keep must", dict(keep=keep.long())),
            ("keep must", dict(keep=keep[:1])), ("keep_lens", dict(lens=lens[:1]))):
        refused(match, ops.compact_kv, *{**good, **change}.values())
    refused("start", ops.compact_kv, *good.values(), start=lens[:1])
    refused("dst_table", ops.compact_kv, *good.values(), dst_table=table[:1])
    refused("scores_out", ops.compact_kv, *good.values(), scores_out=scores)
    refused("scores_out", ops.compact_kv, *good.values(), scores=scores,
            scores_out=scores[..., :3].contiguous())
    refused("scores", ops.compact_kv, *good.values(), scores=scores[:1])


def test_abi_refusals():
    """Refused on the host, before any launch (pointers that are never read)."""
    import ctypes

    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def refused(match, rc):
        assert rc == _lib.VOOM_EINVAL and match in _lib.last_error(), (rc, _lib.last_error())

    def observe(q=p, batch=1, nq=4, nkv=2, d=64, page=64, pages=2, slots=2, window=3, cap=64,
                scale=0.1):
        return lib.voom_paged_gqa_observe(q, p, p, p, p, None, p, p, batch, nq, nkv, d, page,
                                          pages, slots, window, cap, scale, None)

    refused("null pointer", observe(q=None))
    refused("aligned", observe(q=ctypes.c_void_p(258)))
    refused("empty page pool", observe(slots=0))
    for bad in (dict(batch=0), dict(batch=1025), dict(nq=5), dict(nkv=0), dict(d=96),
                dict(window=0), dict(pages=0)):
        refused("geometry", observe(**bad))
    refused("page_tokens", observe(page=16))
    refused("block table", observe(pages=1 << 25))
    refused("scores", observe(cap=0))
    refused("finite", observe(scale=NAN))

    def select(s=p, batch=1, nkv=2, cap=64, budget=8, sink=0, recent=0):
        return lib.voom_evict_select(s, p, p, p, batch, nkv, cap, budget, sink, recent, None)

    refused("null pointer", select(s=None))
    for bad in (dict(batch=0), dict(nkv=0), dict(cap=0), dict(cap=1 << 30)):
        refused("geometry", select(**bad))
    for bad in (dict(budget=0), dict(sink=9), dict(sink=-1), dict(recent=-1),
                dict(sink=4, recent=5), dict(sink=8, recent=2 ** 31 - 1)):
        refused("budget", select(**bad))

    def compact(k=p, scores=None, out=None, batch=1, nkv=2, d=64, page=64, pages=2, dst=2, slots=2,
                heads=2, n=5, cap=0):
        return lib.voom_compact_kv(k, p, p, p, p, p, None, scores, out, batch, nkv, d, page, pages,
                                   dst, slots, heads, n, cap, None)

    refused("null pointer", compact(k=None))
    refused("aligned", compact(k=ctypes.c_void_p(264)))
    for bad in (dict(batch=0), dict(batch=65536), dict(nkv=0), dict(pages=0), dict(dst=0),
                dict(slots=0), dict(n=0)):
        refused("geometry", compact(**bad))
    refused("head_dim", compact(d=48))
    refused("page_tokens", compact(page=48))
    refused("rows in the pool", compact(slots=1 << 30))
    refused("lists", compact(heads=3))
    refused("scores", compact(scores=p))
    refused("scores", compact(scores=p, out=p, cap=0))


def test_abi_refusals_of_workspaces_of_long_rows():
    lib, p = _lib.lib(), 1 << 20
    need = lib.voom_evict_select_workspace_bytes(2, 8, 100000)
    assert need > 0 and lib.voom_evict_select_workspace_bytes(2, 8, 200000) > need
    for args in ((2, 8, 32768), (9, 8, 100000), (1, 1, (1 << 20) + 1), (0, 8, 100000)):
        assert lib.voom_evict_select_workspace_bytes(*args) == 0
    for ws, size in ((p, need - 1), (p + 4, need)):
        assert lib.voom_evict_select_split(p, p, p, p, ws, size, 2, 8, 100000, 100, 4, 4,
                                           None) == _lib.VOOM_EINVAL
        assert "workspace" in _lib.last_error()
    assert lib.voom_evict_select_split(p, p, p, p, p, need, 2, 8, 100000, 4, 4, 4,
                                       None) == _lib.VOOM_EINVAL


def test_destinations_that_a_move_reads_are_refused():
    def i32(x):
        return torch.tensor(x, dtype=torch.int32)

    table = i32([[3, 5], [4, 1]])
    lists, lens = i32([[[2, 7, 9]], [[0, 1, 12]]]), i32([3, 2])  # pages of 8 tokens
    for match, dst, start in (("read elsewhere", [[5, 0], [6, 7]], None),
                              ("read elsewhere", [[4, 0], [6, 7]], None),
                              ("twice", [[6, 0], [6, 7]], None),
                              ("twice", [[6, 6], [7, 2]], [6, 0]),
                              ("own pages", [[3, 0], [6, 7]], [3, 0])):
        with pytest.raises(ValueError, match=match):
            ops.check_destination(table, i32(dst), lists, lens, None if start is None else
                                  i32(start), 8)
    for dst, start in (([[0, 2], [6, 7]], None), ([[3, 2], [1, 7]], None),  # 1 is not read
                       ([[0], [6]], [6, 0]), ([[3, 3], [4, 4]], None)):
        ops.check_destination(table, i32(dst), lists, lens, None if start is None else
                              i32(start), 8)
    ops.check_destination(table, table, lists, i32([0, 0]), None, 8)


@pytest.mark.gpu
def test_a_selection_without_heads_is_refused():
    """(its lengths would not be written)"""
    for shape in ((2, 0, 10), (2, 3, 0)):
        with pytest.raises(ValueError, match="scores"):
            ops.evict_select(torch.zeros(shape, device="cuda"), lens_tensor([4, 4]), 5)
    keep, lens = ops.evict_select(torch.zeros((0, 3, 10), device="cuda"), lens_tensor([]), 5)
    assert keep.shape == (0, 3, 5) and lens.shape == (0,)

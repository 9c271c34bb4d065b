"""GPU parity of attention over ragged chunks (voom_paged_gqa_chunk, ops.paged_gqa_chunk)
against fp64 softmax attention over the same bf16 K/V with the same scores and masks.

Bars.  Output: relative L2 error <= 4e-3: it is rounded to bf16 (at most 2^-9 of a value's
binade, 1.1e-3 in the 2-norm) and so is every softmax weight before the fp32 sums (the same,
less where many average out); 4e-3 is twice the sum of the two worst cases' halves.  LSE: it
is summed of unrounded weights.  A score is a sum of D products of bf16 values in fp32, off by
at most D 2^-24 sum |q k| (under 1e-4 at D = 128, |q k| of 2 times 1 on average, scale
D^-0.5); a cap passes no more of that on (its slope is at most 1) and adds 3e-7 of its own
value, the scaling, the slopes and the base-2 exponent 2^-22 of a score's size (under 60 for
those that weigh something here): absolute 2e-4.
"""
import ctypes

import pytest
import torch

import paged_inputs
from paged_inputs import inputs, lens_tensor
from voom_amd import ops

REL, LSE_ABS = 4e-3, 2e-4
INF, NAN = float("inf"), float("nan")
ROOM = 0  # tokens that the tables have room for besides


@pytest.fixture(params=[0, 1 << 17], ids=["tight", "roomy"])
def room(request):
    """Tables of the cached tokens alone, and such as a server reserves: the rows that may see
    many tokens take another kernel."""
    global ROOM
    ROOM = request.param
    yield
    ROOM = 0


def cache(k, v, page, spare=0):
    k_pool, v_pool, table = paged_inputs.cache(k, v, page, spare=spare)
    return k_pool, v_pool, torch.nn.functional.pad(table, (0, ROOM // page))


def reference(q, k, v, ctx, lens, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None):
    """fp64 (out [B, T, NQ, D], lse [B, T, NQ]) of padded q [B, NQ, T, D]; a row's unseen
    keys are left out of it."""
    B, NQ, T, D = q.shape
    G = NQ // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((B, T, NQ, D), dtype=torch.float64)
    lse = torch.full((B, T, NQ), -INF, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    slope = torch.zeros(NQ, dtype=torch.float64) if slopes is None else slopes.double().cpu()
    for b in range(B):
        key = torch.arange(ctx[b])
        for t in range(lens[b]):
            at = ctx[b] - lens[b] + t
            seen = (key <= at) & ((at - key < window) if window else torch.ones_like(key) == 1)
            seen = (seen | (key < (prefix[b] if prefix else 0))).nonzero()[:, 0]
            if not len(seen):
                continue
            for h in range(NQ):
                s = k[b, h // G][seen] @ q[b, h, t] * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                s = s - slope[h] * (at - seen).abs().double()
                lse[b, t, h] = torch.logsumexp(s, 0)
                if lse[b, t, h] > -INF:
                    out[b, t, h] = torch.softmax(s, 0) @ v[b, h // G][seen]
    return out, lse


def check(got, want, lse_abs=LSE_ABS):
    torch.cuda.synchronize()
    out, lse = (x.double().cpu() for x in got)
    ref, ref_lse = want
    dead = ref_lse == -INF
    assert ((lse == -INF) == dead).all()
    assert (out[dead] == 0).all()
    assert torch.isfinite(out).all()
    if dead.all():
        return
    rel = ((out - ref).norm() / ref.norm()).item()
    assert rel <= REL, rel
    row = ((out - ref).norm(dim=-1) / ref.norm(dim=-1).clamp(min=1e-3)).max().item()
    assert row <= 5 * REL, row
    off = (lse - ref_lse)[~dead].abs().max().item()
    assert off <= lse_abs, off


def geometric(NQ):
    return torch.exp2(-8.0 * torch.arange(1, NQ + 1, device="cuda") / NQ)


def pack(q, lens):
    """Packed rows [N, NQ, D] and starts of padded q [B, NQ, T, D]."""
    rows = torch.cat([q[b, :, :n].transpose(0, 1) for b, n in enumerate(lens)])
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return rows.contiguous(), lens_tensor(starts)


def packed_of(padded, lens):
    return torch.cat([padded[b, :n] for b, n in enumerate(lens)])


MODES = [
    dict(),
    dict(softcap=50.0),
    dict(softcap=2.0),                            # most scores far out on the cap
    dict(slopes=True),
    dict(window=37),
    dict(window=1),                               # a token sees itself alone
    dict(window=100, prefix=5),
    dict(prefix=70),                              # seen in both directions
    dict(softcap=30.0, slopes=True, window=300, prefix=33),
]
SHAPES = [
    # B, NQ, NKV, D, PT, ctx, new tokens
    (1, 9, 3, 64, 64, [1], [1]),                             # the first token
    (1, 9, 3, 64, 64, [640], [1]),
    (3, 28, 4, 128, 64, [700, 0, 31], [5, 0, 3]),            # a sequence of nothing, odd group
    (4, 32, 8, 128, 256, [1500, 40, 2100, 16], [1, 40, 3, 16]),
    (2, 16, 1, 128, 32, [2100, 97], [9, 9]),                 # the largest group
    (2, 8, 2, 64, 4096, [4133, 40], [37, 1]),                # the largest page
    (2, 4, 4, 128, 64, [300, 129], [300, 65]),               # whole prompts, a head a kv head
    (1, 8, 2, 128, 32, [777], [400]),                        # many row tiles
    (1, 2, 1, 64, 64, [1200], [131]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", range(len(MODES)))
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_chunk_against_fp64(shape, mode, room):
    B, NQ, NKV, D, PT, ctx, lens = SHAPES[shape]
    kw = dict(MODES[mode])
    print(f"[chunk] {SHAPES[shape]} {kw}", flush=True)
    q, k, v = inputs(B, NQ, NKV, D, max(ctx), max(lens), seed=shape * 16 + mode)
    k_pool, v_pool, table = cache(k, v, PT, spare=40 if max(ctx) > 1024 else 0)
    if kw.get("slopes"):
        kw["slopes"] = geometric(NQ)
    call = dict(kw)
    if "prefix" in kw:
        kw["prefix"] = [min(kw["prefix"], c) for c in ctx]
        call["prefix_lens"] = lens_tensor([call.pop("prefix")] * B)  # clamped to the context
    want = reference(q, k, v, ctx, lens, **kw)
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor(ctx),
                              new_lens=lens_tensor(lens), return_lse=True, **call)
    check(got, want)
    rows, starts = pack(q, lens)
    got = ops.paged_gqa_chunk(rows, k_pool, v_pool, table, lens_tensor(ctx), starts=starts,
                              return_lse=True, **call)
    check(got, tuple(packed_of(x, lens) for x in want))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [m for m in MODES if "window" in m])
@pytest.mark.parametrize("NQ,NKV,D,PT,ctx,lens", [
    (16, 8, 64, 64, [900], [800]), (16, 8, 128, 32, [1000, 500], [500, 90])])
def test_windows_of_long_chunks(NQ, NKV, D, PT, ctx, lens, mode):
    print(f"[chunk] {NQ} {NKV} {D} {ctx} {lens} {mode}", flush=True)
    q, k, v = inputs(len(ctx), NQ, NKV, D, max(ctx), max(lens), seed=31)
    k_pool, v_pool, table = cache(k, v, PT)
    kw, call = dict(mode), dict(mode)
    if "slopes" in kw:
        kw["slopes"] = call["slopes"] = geometric(NQ)
    if "prefix" in kw:
        kw["prefix"] = [kw["prefix"]] * len(ctx)
        call["prefix_lens"] = lens_tensor(kw["prefix"])
        del call["prefix"]
    want = reference(q, k, v, ctx, lens, **kw)
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor(ctx),
                              new_lens=lens_tensor(lens), return_lse=True, **call)
    check(got, want)
    rows, starts = pack(q, lens)
    got = ops.paged_gqa_chunk(rows, k_pool, v_pool, table, lens_tensor(ctx), starts=starts,
                              return_lse=True, **call)
    check(got, tuple(packed_of(x, lens) for x in want))


@pytest.mark.gpu
@pytest.mark.parametrize("scale,softcap", [(-0.2, 0.0), (0.0, 0.0), (0.7, 3.0), (-0.4, 20.0),
                                           (0.3, 1000.0)])
def test_scales_and_caps(scale, softcap, room):
    print(f"[chunk] scale={scale} softcap={softcap}", flush=True)
    for T, ctx in ((3, 300), (150, 200)):
        q, k, v = inputs(1, 9, 3, 64, ctx, T, seed=4)
        k_pool, v_pool, table = cache(k, v, 32)
        got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([ctx]), scale=scale,
                                  softcap=softcap, return_lse=True)
        check(got, reference(q, k, v, [ctx], [T], scale=scale, softcap=softcap))


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [1e-4, 1e30])
def test_caps_that_leave_nothing_of_a_score_and_all_of_it(softcap, room):
    for T, ctx in ((3, 300), (20, 300), (150, 200)):
        q, k, v = inputs(1, 9, 3, 64, ctx, T, seed=14)
        q[:, :, 0] = 0  # scores of 0 are on the polynomial, whatever its coefficients
        k_pool, v_pool, table = cache(k, v, 32)
        got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([ctx]), softcap=softcap,
                                  return_lse=True)
        check(got, reference(q, k, v, [ctx], [T], softcap=softcap))


@pytest.mark.gpu
@pytest.mark.parametrize("NQ,NKV,D,ctx,lens", [
    (4, 2, 64, [9000, 40], [33, 1]),       # a row tile in as many pieces as 64 of its keys allow
    (8, 1, 128, [5000, 70], [18, 70]),
    (3, 3, 64, [7001, 7001, 3], [40, 1, 0]),
])
def test_row_tiles_in_many_pieces(NQ, NKV, D, ctx, lens, room):
    print(f"[chunk] pieces {NQ} {NKV} {D} {ctx} {lens}", flush=True)
    q, k, v = inputs(len(ctx), NQ, NKV, D, max(ctx), max(lens), seed=23)
    k_pool, v_pool, table = cache(k, v, 64)
    want = reference(q, k, v, ctx, lens, softcap=9.0)
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor(ctx),
                              new_lens=lens_tensor(lens), softcap=9.0, return_lse=True)
    check(got, want)
    rows, starts = pack(q, lens)
    got = ops.paged_gqa_chunk(rows, k_pool, v_pool, table, lens_tensor(ctx), starts=starts,
                              softcap=9.0, return_lse=True)
    check(got, tuple(packed_of(x, lens) for x in want))


@pytest.mark.gpu
def test_slopes_of_any_sign_and_size(room):
    """Slopes so steep that a token's own key alone is left, none, and such as favour far
    tokens."""
    q, k, v = inputs(1, 8, 2, 128, 500, 80, seed=5)
    k_pool, v_pool, table = cache(k, v, 64)
    slopes = torch.tensor([100.0, 3.0, 0.5, 0.0, -0.01, -0.2, 1e-4, 30.0], device="cuda")
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([500]), slopes=slopes,
                              return_lse=True)
    # (-0.2 * 500 tokens: scores of up to 110)
    check(got, reference(q, k, v, [500], [80], slopes=slopes), lse_abs=2 * LSE_ABS)


@pytest.mark.gpu
@pytest.mark.parametrize("NQ,NKV,D,ctx,T,window,prefix", [
    (9, 3, 64, 90, 5, 20, 3), (8, 2, 128, 1333, 14, 200, 40), (32, 4, 128, 31, 31, 7, 2),
    (8, 2, 128, 900, 300, 250, 0), (4, 2, 64, 1000, 333, 0, 70), (32, 8, 128, 900, 300, 250, 0),
    (24, 8, 64, 900, 400, 250, 30)])
def test_what_a_row_does_not_see_cannot_reach_it(NQ, NKV, D, ctx, T, window, prefix, room):
    """NaN and infinities in K and V of tokens before the window and of later ones, in the
    queries of rows behind the new tokens, and behind the context (the pools are NaN there)."""
    print(f"[chunk] NaN in unseen tokens, D={D} T={T} ctx={ctx} window={window}", flush=True)
    q, k, v = inputs(1, NQ, NKV, D, ctx, T, seed=6)
    n = T - 2
    bad = [ctx - 1, ctx - n + n // 2]
    if window:
        lost = ctx - n - window  # what no row sees, if not of the prefix
        bad += [p for p in (prefix, lost // 2, lost) if prefix <= p <= lost]
    for i, j in enumerate(bad):
        k[:, :, j], v[:, :, j] = (NAN, INF)[i % 2], (-INF, NAN)[i % 2]
    q[:, :, n:] = NAN
    k_pool, v_pool, table = cache(k, v, 64, spare=20 if ctx > 1024 else 0)
    out, lse = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([ctx]), window=window,
                                   prefix_lens=lens_tensor([prefix]), new_lens=lens_tensor([n]),
                                   return_lse=True)
    torch.cuda.synchronize()
    at = torch.arange(ctx - n, ctx)
    sick = torch.zeros(T, dtype=torch.bool)
    for j in bad:
        sick[:n] |= (j <= at) & ((at - j < window) if window else True) | (j < prefix)
    assert sick[:n].any() and (not sick[:n].all())
    assert torch.isnan(out[:, sick].float()).any(-1).all()
    clean = [x.clone() for x in (k, v)]
    for x in clean:
        x[:, :, bad] = 0
    want, want_lse = reference(q, *clean, [ctx], [n], window=window, prefix=[prefix])
    check((out[:, ~sick], lse[:, ~sick]), (want[:, ~sick], want_lse[:, ~sick]))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 200])
@pytest.mark.parametrize("page,first,count", [(32, 0, 64), (64, 96, 700), (64, 0, 1500)])
def test_keys_that_score_minus_infinity_weigh_nothing(page, first, count, T, room):
    """Whole blocks and splits of them; a row whose every key scores -inf counts as empty."""
    ctx, D = 1500, 128
    print(f"[chunk] -inf keys {first} + {count}", flush=True)
    q, k, v = inputs(1, 8, 2, D, ctx, T, seed=7)
    k[:, :, first:first + count] = 0
    k[:, :, first:first + count, 5] = torch.finfo(torch.bfloat16).min
    q[..., 5] = 4.0  # 4 times the lowest value is past fp32's range
    k_pool, v_pool, table = cache(k, v, page)
    k64 = k.double()
    k64[:, :, first:first + count, 5] = -INF
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([ctx]), scale=0.1,
                              return_lse=True)
    check(got, reference(q, k64, v, [ctx], [T], scale=0.1))
    # a cap leaves none of them out: tanh(-inf) = -1
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([ctx]), scale=0.1,
                              softcap=20.0, return_lse=True)
    check(got, reference(q, k64, v, [ctx], [T], scale=0.1, softcap=20.0))


@pytest.mark.gpu
@pytest.mark.parametrize("T,NQ,NKV", [(6, 9, 3), (120, 9, 3), (1400, 16, 8)])
def test_lengths_out_of_range_and_more_new_tokens_than_cached(T, NQ, NKV):
    print(f"[chunk] clamped lengths, T={T}", flush=True)
    D = 64
    q, k, v = inputs(3, NQ, NKV, D, 64, T, seed=8)
    k_pool, v_pool, table = cache(k, v, 32)
    got = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([1000, -5, 3]),
                              new_lens=lens_tensor([9999, 4, 5]), return_lse=True,
                              prefix_lens=lens_tensor([-3, 9, 2]))
    # rows before the cache see its prefix alone
    check(got, reference(q, k, v, [64, 0, 3], [T, 4, 5], prefix=[0, 0, 2]))
    table[0, 0], table[1, 1] = -1, 10 ** 9  # slot ids outside the pool read slot 0
    out = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([64] * 3))
    fixed = table.clone()
    fixed[0, 0], fixed[1, 1] = 0, 0
    want = ops.paged_gqa_chunk(q, k_pool, v_pool, fixed, lens_tensor([64] * 3))
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(want))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,ctx", [([2, 1, 4], [80, 40, 9]), ([150, 1, 0, 260], [900, 40, 9, 260])])
def test_packed_rows_of_no_sequence_stay(lens, ctx, room):
    """Rows before the first and behind the last sequence, and starts past the rows."""
    print(f"[chunk] rows of no sequence, {lens}", flush=True)
    B = len(lens)
    q, k, v = inputs(B, 8, 2, 128, max(ctx), max(lens), seed=9)
    k_pool, v_pool, table = cache(k, v, 64)
    rows, starts = pack(q, lens)
    rows = torch.cat((rows[:3], rows, rows[:5])).contiguous()
    out = torch.full_like(rows, 7.0)
    got, lse = ops.paged_gqa_chunk(rows, k_pool, v_pool, table, lens_tensor(ctx),
                                   starts=starts + 3, out=out, return_lse=True)
    assert got is out
    want = reference(q, k, v, ctx, lens)
    check((out[3:-5], lse[3:-5]), tuple(packed_of(x, lens) for x in want))
    assert (out[:3] == 7).all() and (out[-5:] == 7).all()
    N = rows.shape[0]
    wild = torch.tensor([-4] + [N + 100 * i for i in range(B)], dtype=torch.int32, device="cuda")
    ops.paged_gqa_chunk(rows, k_pool, v_pool, table, lens_tensor(ctx), starts=wild, out=out)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_plain_scores_are_those_of_the_other_attention_calls(room):
    """Without cap, slopes, window and prefix: the decode, window and tree calls' results."""
    D = 128
    q, k, v = inputs(2, 32, 8, D, 1500, 9, seed=10)
    k_pool, v_pool, table = cache(k, v, 64)
    ctx = lens_tensor([1500, 1500])
    out, lse = ops.paged_gqa_chunk(q, k_pool, v_pool, table, ctx, return_lse=True)
    tree, tree_lse = ops.paged_gqa_tree(q, k_pool, v_pool, table, ctx, return_lse=True)
    window = ops.paged_gqa_prefill(q, k_pool, v_pool, table, 1500)
    one = q[:, :, -1].contiguous()
    decode = ops.paged_gqa_decode(one, k_pool, v_pool, table, ctx)
    token = ops.paged_gqa_chunk(one, k_pool, v_pool, table, ctx, starts=lens_tensor([0, 1, 2]))
    torch.cuda.synchronize()
    for a, b in ((out, tree), (out, window), (token, decode)):
        assert ((a.double() - b.double()).norm() / b.double().norm()).item() <= REL
    assert (lse - tree_lse).abs().max().item() <= LSE_ABS


@pytest.mark.gpu
def test_empty_calls():
    k_pool, v_pool, table = cache(*inputs(1, 2, 1, 64, 32, 1)[1:], 32)
    for B, T in ((0, 3), (1, 0)):
        q = torch.empty((B, 2, T, 64), dtype=torch.bfloat16, device="cuda")
        out, lse = ops.paged_gqa_chunk(q, k_pool, v_pool, table[:B], lens_tensor([5] * B),
                                       return_lse=True)
        assert out.shape == (B, T, 2, 64) and lse.shape == (B, T, 2)
    q = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    out, lse = ops.paged_gqa_chunk(q, k_pool, v_pool, table, lens_tensor([5]),
                                   starts=lens_tensor([0, 0]), return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


@pytest.mark.gpu
def test_graph_replays_with_new_lengths_and_overlapping_streams():
    """Captured, with other eager calls between the replays and other lengths on the device;
    and two calls at once on two streams: each result is the eager one's, bit for bit."""
    print("[chunk] graph replay, two streams", flush=True)
    calls = []
    for seed, (ctx, lens) in enumerate([([2500, 700], [9, 1]), ([1800, 40], [300, 2])]):
        q, k, v = inputs(2, 32, 8, 128, max(ctx), max(lens), seed=seed + 20)
        k_pool, v_pool, table = cache(k, v, 64, spare=8)
        rows, starts = pack(q, lens)
        calls.append(dict(args=(rows, k_pool, v_pool, table, lens_tensor(ctx)), starts=starts))

    def run(i):
        return ops.paged_gqa_chunk(*calls[i]["args"], starts=calls[i]["starts"], softcap=30.0,
                                   window=1000, return_lse=True)

    eager = [[t.clone() for t in run(i)] for i in (0, 1)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        run(1)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(o, e))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([run(i) for _ in range(5)])
    torch.cuda.synchronize()
    for rs, e in zip(got, eager):
        assert all(torch.equal(a, b) for r in rs for a, b in zip(r, e))
    for i in (0, 1):  # other lengths in the captured call's own tensors
        calls[i]["args"][4].copy_(lens_tensor([1300, 39]))
        N = calls[i]["args"][0].shape[0]
        calls[i]["starts"].copy_(lens_tensor([0, N // 3, N]))
    again = [[t.clone() for t in run(i)] for i in (0, 1)]
    for i in (0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], again[i]))


@pytest.mark.gpu
def test_wrapper_refusals():
    q, k, v = inputs(2, 8, 2, 64, 40, 3)
    k_pool, v_pool, table = cache(k, v, 32)
    ctx = lens_tensor([40, 40])
    good = dict(q=q, k_pool=k_pool, v_pool=v_pool, block_table=table, ctx_lens=ctx)

    def refused(match, **change):
        with pytest.raises(ValueError, match=match):
            ops.paged_gqa_chunk(**{**good, **change})

    rows, starts = pack(q, [3, 3])
    refused("ROCm device", q=q.cpu())
    refused("contiguous", q=q.transpose(1, 2).contiguous().transpose(1, 2))
    refused("B, NQ, T, D", q=rows)
    refused("N, NQ, D", starts=starts)
    refused("starts", q=rows, starts=starts[:2].contiguous())
    refused("starts", q=rows, starts=starts.long())
    refused("new_lens", q=rows, starts=starts, new_lens=ctx)
    refused("new_lens", new_lens=lens_tensor([3]))
    refused("bfloat16", q=q.half())
    refused("head_dim", q=torch.cat((q, q), -1))
    refused("multiple", q=q[:, :7].contiguous())
    refused("V", v_pool=v_pool.transpose(2, 3).contiguous())
    refused("block_table", block_table=table.long())
    refused("ctx_lens", ctx_lens=ctx.long())
    refused("slopes", slopes=torch.ones(7, device="cuda"))
    refused("slopes", slopes=torch.ones(8, device="cuda", dtype=torch.float64))
    refused("prefix_lens", prefix_lens=lens_tensor([1]))
    refused("out", out=q)
    refused("window", window=-1)
    refused("softcap", softcap=-1.0)
    refused("softcap", softcap=INF)
    refused("softcap", softcap=NAN)
    refused("finite", scale=NAN)
    unaligned = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    refused("aligned", q=unaligned)
    ops.set_bounds_checks(True)
    try:
        refused("context lengths", ctx_lens=lens_tensor([40, 400]))
        refused("starts", q=rows, starts=lens_tensor([0, 4, 3]))
        refused("starts", q=rows, starts=lens_tensor([0, 4, 7]))
        refused("new_lens", new_lens=lens_tensor([1, 4]))
    finally:
        ops.set_bounds_checks(False)


def test_abi_refusals():
    """Refused on the host, before any launch (pointers that are never read)."""
    from voom_amd import _lib

    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def call(q=p, starts=None, lens=None, batch=1, rows=0, tokens=3, nq=4, nkv=2, d=64, page=64,
             pages=2, slots=2, window=0, scale=0.1, cap=0.0, ws=None, ws_bytes=0):
        rc = lib.voom_paged_gqa_chunk(q, p, p, p, p, starts, lens, None, None, p, None, ws,
                                      ws_bytes, batch, rows, tokens, nq, nkv, d, page, pages,
                                      slots, window, scale, cap, None)
        return rc, _lib.last_error()

    def refused(match, **kw):
        rc, msg = call(**kw)
        assert rc == _lib.VOOM_EINVAL and match in msg, (rc, msg)

    refused("null pointer", q=None)
    refused("empty page pool", slots=0)
    for bad in (dict(batch=0), dict(batch=1025), dict(nq=5), dict(nkv=0), dict(nq=34), dict(d=96),
                dict(tokens=0), dict(rows=3), dict(rows=-1, tokens=0), dict(tokens=-1),
                dict(page=48), dict(page=16), dict(page=8192), dict(pages=0),
                dict(pages=1 << 25), dict(tokens=1 << 26)):
        refused("unsupported geometry", **bad)
        sizes = {**dict(batch=1, rows=0, tokens=3, nq=4, nkv=2, d=64, page=64, pages=2), **bad}
        assert lib.voom_paged_gqa_chunk_workspace_bytes(*sizes.values(), 0) == 0
    refused("starts", starts=p)
    refused("starts", rows=3, tokens=0)
    refused("starts", starts=p, lens=p, rows=3, tokens=0)
    refused("window", window=-1)
    refused("finite", scale=float("inf"))
    refused("finite", cap=-1.0)
    refused("finite", cap=float("nan"))
    for cap in (1e-9, 1e-30, 3e38):
        refused("out of proportion", cap=cap)
    refused("out of proportion", scale=1e30, cap=1e28)
    refused("out of proportion", scale=1e-42, cap=1.0)
    refused("aligned", q=ctypes.c_void_p(264))
    refused("workspace", pages=100, ws=p, ws_bytes=64)

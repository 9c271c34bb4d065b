"""GPU parity of the attention of drafted tokens (voom_paged_gqa_tree, ops.paged_gqa_tree)
against fp64 softmax attention over the same bf16 K/V under the same mask.

Bars.  Output: relative L2 error <= 4e-3, as of the causal window kernel: the output is
rounded to bf16 (at most 2^-9 per value, 1.1e-3 in the 2-norm) and so is every softmax
weight before the fp32 sums (the same, less where many average out); 4e-3 is twice the sum
of the two worst cases' halves.  LSE: it is summed of unrounded weights.  A score is a sum of
D products of bf16 values in fp32, off by at most D 2^-24 sum |q k| (under 1e-4 at D = 128,
|q k| of 2 times 1 on average, scale D^-0.5), the scaling and the base-2 exponent add 2^-23
of a score's size (under 40 here): absolute 2e-4.
"""
import pytest
import torch

from paged_inputs import cache, inputs, lens_tensor, trees
from voom_amd import ops

REL, LSE_ABS = 4e-3, 2e-4
INF, NAN = float("inf"), float("nan")


def reference(q, k, v, ctx, lens, mask, scale):
    """fp64 (out [B, T, NQ, D], lse [B, T, NQ]); a row's unseen keys are left out of it."""
    B, NQ, T, D = q.shape
    G = NQ // k.shape[1]
    out = torch.zeros((B, T, NQ, D), dtype=torch.float64)
    lse = torch.full((B, T, NQ), -INF, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    for b in range(B):
        before = ctx[b] - lens[b]
        for t in range(lens[b]):
            seen = list(range(before)) + [before + j for j in range(lens[b]) if mask[b, t, j]]
            if not seen:
                continue
            for h in range(NQ):
                s = k[b, h // G][seen] @ q[b, h, t] * scale
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


@pytest.mark.gpu
@pytest.mark.parametrize("B,NQ,NKV,D,PT,T,ctx,lens", [
    (1, 9, 3, 64, 64, 1, [1], None),                 # one token, one draft
    (1, 9, 3, 64, 64, 7, [640], None),               # one segment per workgroup
    (1, 4, 4, 64, 32, 33, [33], None),               # nothing before the drafts
    (2, 9, 3, 64, 64, 11, [130, 65], [11, 4]),       # ragged drafts, two row tiles
    (3, 28, 4, 128, 64, 5, [700, 0, 31], [5, 5, 3]), # an empty sequence, odd group
    (2, 16, 1, 128, 32, 9, [2100, 97], [9, 9]),      # the largest group, split over keys
    (4, 32, 8, 128, 256, 16, [1500, 40, 2500, 16], [16, 1, 13, 16]),
    (1, 64, 8, 128, 64, 61, [4000], None),           # many row tiles
    (2, 8, 2, 64, 4096, 37, [5001, 40], [37, 0]),    # the largest page; no drafts at all
    (1, 2, 1, 128, 64, 130, [1200], None),           # drafts over several blocks
])
def test_tree_against_fp64(B, NQ, NKV, D, PT, T, ctx, lens):
    print(f"[tree] B={B} NQ={NQ} NKV={NKV} D={D} PT={PT} T={T} ctx={ctx} lens={lens}", flush=True)
    q, k, v = inputs(B, NQ, NKV, D, max(max(ctx), 1), T)
    mask = trees(B, T, 5)
    k_pool, v_pool, table = cache(k, v, PT, spare=40 if max(ctx) > 1024 else 0)
    n = [min(x, c) for x, c in zip(lens or [T] * B, ctx)]  # no more drafts than tokens
    got = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor(ctx), mask=mask.cuda(),
                             draft_lens=None if lens is None else lens_tensor(lens),
                             return_lse=True)
    check(got, reference(q, k, v, ctx, n, mask, D ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("T,ctx", [(13, 40), (40, 1500)])
def test_no_mask_is_causal_and_a_shared_mask_serves_every_sequence(T, ctx):
    print(f"[tree] causal and shared masks, T={T} ctx={ctx}", flush=True)
    q, k, v = inputs(2, 8, 2, 128, ctx, T, seed=3)
    k_pool, v_pool, table = cache(k, v, 64)
    call = (q, k_pool, v_pool, table, lens_tensor([ctx, ctx - 3]))
    tril = torch.ones(T, T, dtype=torch.bool).tril()
    got = ops.paged_gqa_tree(*call, return_lse=True)
    check(got, reference(q, k, v, [ctx, ctx - 3], [T, T], tril.expand(2, T, T), 128 ** -0.5))
    again = ops.paged_gqa_tree(*call, mask=tril.cuda(), return_lse=True)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert torch.equal(got[0], ops.paged_gqa_tree(*call))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.7])
def test_scales(scale):
    print(f"[tree] scale={scale}", flush=True)
    q, k, v = inputs(1, 9, 3, 64, 300, 6, seed=4)
    mask = trees(1, 6, 2)
    k_pool, v_pool, table = cache(k, v, 32)
    got = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([300]), mask=mask.cuda(),
                             scale=scale, return_lse=True)
    check(got, reference(q, k, v, [300], [6], mask, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("NQ,NKV,D,T,ctx", [(9, 3, 64, 5, 90), (8, 2, 128, 14, 1333),
                                            (32, 4, 128, 30, 31)])
def test_what_a_row_does_not_see_cannot_reach_it(NQ, NKV, D, T, ctx):
    """NaN and infinities in K and V of drafts that a row does not see, in the queries of
    rows past the drafts, and behind the context (the pools are NaN there)."""
    print(f"[tree] NaN in unseen drafts, D={D} T={T} ctx={ctx}", flush=True)
    q, k, v = inputs(1, NQ, NKV, D, ctx, T, seed=6)
    n = T - 2
    before = ctx - n
    mask = torch.eye(T, dtype=torch.bool)[None].repeat(1, 1, 1)
    mask[:, :, 0] = True       # a root that all see, and siblings
    bad = [2, n - 1]
    for j, value in zip(bad, (NAN, INF)):
        k[:, :, before + j], v[:, :, before + j] = value, -value
    q[:, :, n:] = NAN
    k_pool, v_pool, table = cache(k, v, 64, spare=20 if ctx > 1024 else 0)
    out, lse = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([ctx]), mask=mask.cuda(),
                                  draft_lens=lens_tensor([n]), return_lse=True)
    torch.cuda.synchronize()
    want, want_lse = reference(q, k, v, [ctx], [n], mask, D ** -0.5)
    assert torch.isnan(out[:, bad].float()).all()
    keep = [t for t in range(T) if t not in bad]
    check((out[:, keep], lse[:, keep]), (want[:, keep], want_lse[:, keep]))


@pytest.mark.gpu
@pytest.mark.parametrize("page,first,count", [(32, 0, 64), (64, 96, 700), (64, 0, 1500)])
def test_keys_that_score_minus_infinity_weigh_nothing(page, first, count):
    """Whole blocks and splits of them; a row whose every key scores -inf counts as empty."""
    ctx, T, D = 1500, 4, 128
    print(f"[tree] -inf keys {first} + {count}", flush=True)
    q, k, v = inputs(1, 8, 2, D, ctx, T, seed=7)
    k[:, :, first:first + count] = 0
    k[:, :, first:first + count, 5] = torch.finfo(torch.bfloat16).min
    q[..., 5] = 4.0  # 4 times the lowest value is past fp32's range
    k_pool, v_pool, table = cache(k, v, page)
    k64 = k.double()
    k64[:, :, first:first + count, 5] = -INF
    mask = trees(1, T, 9)
    got = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([ctx]), mask=mask.cuda(),
                             scale=0.1, return_lse=True)
    check(got, reference(q, k64, v, [ctx], [T], mask, 0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("NQ,NKV,D", [(9, 3, 64), (8, 2, 128)])
@pytest.mark.parametrize("ctx", [700, 1480, 2500])
def test_an_infinite_value_stays_infinite_however_a_context_is_cut(NQ, NKV, D, ctx):
    """Infinities of both signs in V of the newest draft, in the last of any number of pieces:
    its own row holds them, all else is as without them."""
    T = 4
    print(f"[tree] infinite V at the end, D={D} ctx={ctx}", flush=True)
    q, k, v = inputs(1, NQ, NKV, D, ctx, T, seed=11)
    plain = v.clone()
    v[:, :, ctx - 1, 3], v[:, :, ctx - 1, D - 2] = INF, -INF
    got = []
    for values in (plain, v):
        for spare in (0, 60):  # a wider table: the same context in other pieces
            k_pool, v_pool, table = cache(k, values, 64, spare=spare)
            got.append(ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([ctx]),
                                          return_lse=True))
    torch.cuda.synchronize()
    for (finite, lse), (out, lse_inf) in zip(got[:2], got[2:]):
        want = finite.clone()
        want[:, T - 1, :, 3], want[:, T - 1, :, D - 2] = INF, -INF
        assert torch.equal(out, want) and torch.equal(lse, lse_inf)


@pytest.mark.gpu
def test_rows_without_a_key_and_lengths_out_of_range():
    print("[tree] empty mask rows, clamped lengths", flush=True)
    T, D, page = 6, 64, 32
    q, k, v = inputs(3, 9, 3, D, 64, T, seed=8)
    k_pool, v_pool, table = cache(k, v, page)
    mask = trees(3, T, 4)
    mask[0, 2] = False  # sees the tokens before the drafts, or nothing where there are none
    mask[1, 4] = False
    got = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([6, 50, 64]), mask=mask.cuda(),
                             return_lse=True)
    want = reference(q, k, v, [6, 50, 64], [6] * 3, mask, D ** -0.5)
    assert (want[1][0, 2] == -INF).all() and (want[1][1, 4] > -INF).all()
    check(got, want)
    # past the table, negative, more drafts than tokens or rows
    got = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([1000, -5, 3]),
                             mask=mask.cuda(), draft_lens=lens_tensor([99, 4, 5]), return_lse=True)
    check(got, reference(q, k, v, [64, 0, 3], [6, 0, 3], mask, D ** -0.5))
    # slot ids outside the pool read slot 0
    table[0, 0], table[1, 1] = -1, 10 ** 9
    out = ops.paged_gqa_tree(q, k_pool, v_pool, table, lens_tensor([64, 64, 64]))
    torch.cuda.synchronize()
    fixed = table.clone()
    fixed[0, 0], fixed[1, 1] = 0, 0
    want = ops.paged_gqa_tree(q, k_pool, v_pool, fixed, lens_tensor([64, 64, 64]))
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(want))


@pytest.mark.gpu
def test_empty_calls():
    k_pool, v_pool, table = cache(*inputs(1, 2, 1, 64, 32, 1)[1:], 32)
    for B, T in ((0, 3), (1, 0)):
        q = torch.empty((B, 2, T, 64), dtype=torch.bfloat16, device="cuda")
        out, lse = ops.paged_gqa_tree(q, k_pool, v_pool, table[:B], lens_tensor([5] * B),
                                      return_lse=True)
        assert out.shape == (B, T, 2, 64) and lse.shape == (B, T, 2)


@pytest.mark.gpu
def test_graph_replays_and_overlapping_streams():
    """Captured with other eager calls between the replays, and two calls at once on two
    streams: each result is the eager one's, bit for bit."""
    print("[tree] graph replay, two streams", flush=True)
    calls = []
    for seed, (ctx, T) in enumerate([(2500, 9), (1800, 30)]):
        q, k, v = inputs(2, 32, 8, 128, ctx, T, seed=seed + 20)
        k_pool, v_pool, table = cache(k, v, 64)
        calls.append(dict(args=(q, k_pool, v_pool, table, lens_tensor([ctx, ctx // 3])),
                          mask=trees(2, T, seed).cuda()))

    def run(i):
        return ops.paged_gqa_tree(*calls[i]["args"], mask=calls[i]["mask"], return_lse=True)

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


@pytest.mark.gpu
def test_wrapper_refusals():
    q, k, v = inputs(2, 8, 2, 64, 40, 3)
    k_pool, v_pool, table = cache(k, v, 32)
    ctx = lens_tensor([40, 40])
    good = dict(q=q, k_pool=k_pool, v_pool=v_pool, block_table=table, ctx_lens=ctx)

    def refused(match, mask=None, draft_lens=None, scale=None, **change):
        with pytest.raises(ValueError, match=match):
            ops.paged_gqa_tree(*{**good, **change}.values(), mask=mask, draft_lens=draft_lens,
                               scale=scale)

    refused("ROCm device", q=q.cpu())
    refused("contiguous", q=q.transpose(1, 2).contiguous().transpose(1, 2))
    refused("B, NQ, T, D", q=q[0])
    refused("bfloat16", q=q.half())
    refused("head_dim", q=torch.cat((q, q), -1))
    refused("multiple", q=q[:, :7].contiguous())
    refused("V", v_pool=v_pool.transpose(2, 3).contiguous())
    refused("block_table", block_table=table.long())
    refused("block_table", block_table=table[:1])
    refused("ctx_lens", ctx_lens=ctx.long())
    refused("draft_lens", draft_lens=lens_tensor([3]))
    refused("mask", mask=torch.ones(3, 3, device="cuda"))
    refused("mask", mask=torch.ones(2, 3, 4, dtype=torch.bool, device="cuda"))
    refused("finite", scale=float("nan"))
    unaligned = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    refused("aligned", q=unaligned)
    if torch.cuda.device_count() > 1:
        with torch.cuda.device(1):
            refused("current device")


def test_abi_refusals():
    """Refused on the host, before any launch (pointers that are never read)."""
    import ctypes

    from voom_amd import _lib

    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def call(q=p, mask=None, mask_batch=1, batch=1, nq=4, nkv=2, d=64, page=64, pages=2, slots=2,
             drafts=3, scale=0.1, ws=None, ws_bytes=0):
        rc = lib.voom_paged_gqa_tree(q, p, p, p, p, None, mask, mask_batch, p, None, ws, ws_bytes,
                                     batch, nq, nkv, d, page, pages, slots, drafts, scale, None)
        return rc, _lib.last_error()

    def refused(match, **kw):
        rc, msg = call(**kw)
        assert rc == _lib.VOOM_EINVAL and match in msg, (rc, msg)

    refused("null pointer", q=None)
    refused("empty page pool", slots=0)
    for bad in (dict(batch=0), dict(batch=1025), dict(nq=5), dict(nkv=0), dict(nq=34), dict(d=96),
                dict(drafts=0), dict(drafts=1025), dict(page=48), dict(page=16), dict(page=8192),
                dict(pages=0), dict(pages=1 << 25)):
        refused("unsupported geometry", **bad)
        assert lib.voom_paged_gqa_tree_workspace_bytes(
            *[{**dict(batch=1, nq=4, nkv=2, d=64, drafts=3, page=64, pages=2), **bad}[n]
              for n in ("batch", "nq", "nkv", "d", "drafts", "page", "pages")]) == 0
    refused("masks", mask=p, mask_batch=3, batch=2)
    refused("finite", scale=float("inf"))
    refused("aligned", q=ctypes.c_void_p(264))
    refused("workspace", pages=100, ws=p, ws_bytes=64)

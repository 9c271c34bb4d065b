"""Beam selection (voom_beam_select, ops.beam_select) against a search in fp64 on the host,
and copies between beams (voom_fork_kv, ops.fork_kv) bit for bit.

Bars.  Tokens, parents and counts of common tokens: equal.  Scores: the logarithm of a sum of
exponentials in fp32, each off by at most 2^-21 (an argument of up to 2^5 in 2^-24 steps, and
the exponential), summed 32 at a time and then in five levels of a tree: under 40 roundings
of 2^-24 on top, so 4e-6 of the sum and as much of its logarithm, absolute; and the rounding
of the score itself, 2^-24 of it.  1e-5 + 2^-23 |score|.
"""
import ctypes

import numpy as np
import pytest
import torch

from paged_inputs import cache, inputs, lens_tensor
from voom_amd import ops

INF, NAN = float("inf"), float("nan")


def search(logits, scores, last=None, end=None):
    """fp64 (scores, tokens, parents), by row."""
    x = logits.double().cpu().numpy()
    s = scores.double().cpu().numpy()
    B, K, V = x.shape
    out = np.zeros((B, K)), np.zeros((B, K), np.int64), np.zeros((B, K), np.int32)
    for b in range(B):
        found = []
        for j in range(K):
            if last is not None and int(last[b, j]) == end:
                found.append((s[b, j] if s[b, j] < INF else -INF, j, end))
                continue
            with np.errstate(all="ignore"):
                top = x[b, j].max()
                lse = top + np.log(np.exp(x[b, j] - top).sum())
                c = s[b, j] + (x[b, j] - lse)
            if not (np.isfinite(lse) and np.isfinite(s[b, j])):
                c = np.full(V, -INF)
            order = np.argsort(-c, kind="stable")[:K]
            found += [(c[t], j, int(t)) for t in order]
        found = sorted(found, key=lambda f: (-f[0], f[1], f[2]))[:K]
        rows, rest = {}, []
        for f in found:
            if f[1] in rows:
                rest.append(f)
            else:
                rows[f[1]] = f
        for j in range(K):
            if j not in rows:
                rows[j] = rest.pop(0)
            out[0][b, j], out[2][b, j], out[1][b, j] = rows[j]
    return out


def check(got, want):
    torch.cuda.synchronize()
    scores, tokens, parents = got[:3]
    assert np.array_equal(parents.cpu().numpy(), want[2])
    assert np.array_equal(tokens.cpu().numpy(), want[1])
    got = scores.double().cpu().numpy()
    dead = want[0] == -INF
    assert np.array_equal(got == -INF, dead)
    off = np.abs(got - want[0])[~dead]
    assert (off <= 1e-5 + np.abs(want[0][~dead]) * 2.0 ** -23).all(), off.max()


def make(B, K, V, dtype, seed, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn((B, K, V), generator=g, device="cuda") * std).to(dtype)
    scores = -torch.rand((B, K), generator=g, device="cuda") * 6 - 3
    return logits, scores


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V", [
    (1, 1, 1), (1, 1, 50), (2, 3, 2), (1, 4, 49152), (3, 5, 8191), (2, 2, 8192), (2, 7, 8193),
    (1, 32, 1000), (1, 32, 20011), (5, 8, 33333), (1, 3, 128256), (40, 2, 515)])
def test_select_against_fp64(B, K, V, dtype):
    print(f"[beam] B={B} K={K} V={V} {dtype}", flush=True)
    logits, scores = make(B, K, V, dtype, B * 7 + K)
    check(ops.beam_select(logits, scores), search(logits, scores))
    g = torch.Generator(device="cuda").manual_seed(V)
    last = torch.randint(0, 2, (B, K), generator=g, device="cuda")
    check(ops.beam_select(logits, scores, last=last, end_token=0), search(logits, scores, last, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 4, 32])
@pytest.mark.parametrize("V", [33, 4096, 40003])
def test_equal_continuations_go_to_the_lowest(K, V):
    """Constant logits, a few values, and both zeros: all ties."""
    print(f"[beam] ties, K={K} V={V}", flush=True)
    scores = torch.full((2, K), -1.5, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    few = torch.randint(0, 3, (2, K, V), generator=g, device="cuda").float()
    zeros = torch.where(few == 1, -0.0, 0.0)
    for logits in (torch.full((2, K, V), 0.25, device="cuda"), few, zeros, few.bfloat16()):
        # (every beam has the same logits: equal across beams as well)
        logits = logits[:, :1].expand(2, K, V).contiguous()
        check(ops.beam_select(logits, scores), search(logits, scores))


@pytest.mark.gpu
def test_infinities_and_nan():
    print("[beam] infinities and NaN", flush=True)
    K, V = 4, 9000
    logits, scores = make(8, K, V, torch.float32, 3)
    logits[0, 1, 77] = NAN          # the beam counts as -inf
    logits[1, 2] = -INF             # no token left
    logits[2, :, 5:] = -INF         # five tokens left
    logits[3, 0, 8500] = INF
    scores[4] = torch.tensor([-1.0, -INF, -INF, -INF])   # a first step
    scores[5, 2] = NAN
    scores[6, 1] = INF
    logits[7] = NAN                 # nothing: the first tokens of the first beam, at -inf
    check(ops.beam_select(logits, scores), search(logits, scores))
    last = torch.zeros((8, K), dtype=torch.int64, device="cuda")
    check(ops.beam_select(logits, scores, last=last, end_token=0),
          search(logits, scores, last, 0))  # all have ended
    last[:, 0] = 3
    check(ops.beam_select(logits.bfloat16(), scores, last=last, end_token=0),
          search(logits.bfloat16(), scores, last, 0))


@pytest.mark.gpu
def test_large_logits_and_unaligned_rows():
    """Logits whose exponentials would overflow, and tensors off 16-byte boundaries."""
    for dtype in (torch.bfloat16, torch.float32):
        logits, scores = make(2, 3, 4099, dtype, 5, std=300.0)
        flat = torch.empty(logits.numel() + 3, dtype=dtype, device="cuda")
        for shift in range(4):
            view = flat[shift:shift + logits.numel()].view(logits.shape)
            view.copy_(logits)
            check(ops.beam_select(view, scores), search(logits, scores))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 2, 6, 32])
def test_what_rows_have_in_common(K):
    """first and shared over many steps against histories kept as lists."""
    print(f"[beam] common tokens, K={K}", flush=True)
    B, V, n = 3, 40, 12
    scores = torch.full((B, K), -INF, device="cuda")
    scores[:, 0] = 0
    shared = torch.full((B, K, K), n, dtype=torch.int32, device="cuda")
    past = [[list(range(-n, 0)) for _ in range(K)] for _ in range(B)]
    for step in range(14):
        logits, _ = make(B, K, V, torch.float32, 100 + step)
        ctx = lens_tensor([n + step] * B)
        want = search(logits, scores)
        old = [[list(h) for h in rows] for rows in past]
        scores, tokens, parents, first, shared = ops.beam_select(logits, scores, shared=shared,
                                                                 ctx_lens=ctx)
        check((scores, tokens, parents), want)
        p, f, sh = parents.tolist(), first.tolist(), shared.tolist()

        def common(a, b):
            m = 0
            while m < len(a) and a[m] == b[m]:
                m += 1
            return m

        for b in range(B):
            for j in range(K):
                assert p[b][p[b][j]] == p[b][j]
                if p[b][j] == j:
                    assert f[b][j] == n + step
                # (a lower bound: rows that part may meet again by chance)
                assert f[b][j] <= common(old[b][j], old[b][p[b][j]])
                past[b][j] = list(old[b][p[b][j]])
            for i in range(K):
                for j in range(K):
                    assert sh[b][i][j] <= common(past[b][i], past[b][j])
                    assert (p[b][i] == p[b][j]) <= (sh[b][i][j] == n + step)
            for j in range(K):
                past[b][j].append((int(tokens[b, j]), step))


@pytest.mark.gpu
def test_select_in_a_graph_and_on_a_side_stream():
    logits, scores = make(4, 5, 30011, torch.bfloat16, 9)
    shared = torch.zeros((4, 5, 5), dtype=torch.int32, device="cuda")
    ctx = lens_tensor([9] * 4)

    def run():
        return ops.beam_select(logits, scores, shared=shared, ctx_lens=ctx)

    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        for t in out:
            t.zero_()
        run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_select_refusals():
    logits, scores = make(2, 3, 50, torch.float32, 1)
    last = torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    shared, ctx = torch.zeros((2, 3, 3), dtype=torch.int32, device="cuda"), lens_tensor([1, 1])

    def refused(match, logits=logits, scores=scores, **kw):
        with pytest.raises(ValueError, match=match):
            ops.beam_select(logits, scores, **kw)

    refused("logits", logits=logits[0])
    refused("logits", logits=logits.half())
    refused("ROCm device", logits=logits.cpu())
    refused("contiguous", logits=logits.transpose(0, 1))
    refused("scores", scores=scores.double())
    refused("scores", scores=scores[:1])
    refused("together", last=last)
    refused("together", end_token=1)
    refused("last", last=last.int(), end_token=1)
    refused("end token", last=last, end_token=50)
    refused("end token", last=last, end_token=-1)
    refused("together", shared=shared)
    refused("shared", shared=shared.long(), ctx_lens=ctx)
    refused("shared", shared=shared, ctx_lens=ctx.long())
    refused("beams", *make(1, 33, 50, torch.float32, 1))
    out = ops.beam_select(logits[:0], scores[:0])
    assert out[0].shape == (0, 3)


# ---- copies -------------------------------------------------------------------


def layers_of(n, B, K, NKV, D, PT, S, seed):
    pools = []
    for i in range(n):
        _, k, v = inputs(B * K, NKV, NKV, D, S, 1, seed=seed + i)
        pools.append((k, v, *cache(k, v, PT, spare=i % 3, seed=seed + i)))
    return pools


def tokens_of(k_pool, v_pool, table, S, PT):
    at = torch.arange(S, device=table.device)
    slot, off, vb = table.long()[:, at // PT], at % PT, min(PT, 32)
    return (k_pool.transpose(1, 2)[slot, off],
            v_pool.permute(0, 2, 4, 1, 3)[slot, off // vb, off % vb])


@pytest.mark.gpu
@pytest.mark.parametrize("n,B,K,NKV,D,PT,S", [
    (1, 1, 2, 1, 64, 32, 1), (2, 1, 4, 3, 64, 64, 100), (3, 2, 5, 8, 128, 64, 333),
    (1, 3, 3, 2, 40, 16, 77), (2, 1, 6, 2, 256, 256, 300), (70, 1, 2, 1, 8, 8, 20),
    (1, 2, 4, 2, 128, 4096, 1000)])
def test_fork_copies_bit_for_bit(n, B, K, NKV, D, PT, S):
    print(f"[fork] layers={n} B={B} K={K} NKV={NKV} D={D} PT={PT} S={S}", flush=True)
    pools = layers_of(n, B, K, NKV, D, PT, S, 50)
    g = torch.Generator().manual_seed(S)
    stay = torch.zeros((B, K), dtype=torch.bool)
    stay[:, torch.randperm(K, generator=g)[:max(1, K // 2)]] = True
    parents = torch.arange(K).repeat(B, 1)
    for b in range(B):
        roots = stay[b].nonzero()[:, 0]
        for j in range(K):
            if not stay[b, j]:
                parents[b, j] = roots[int(torch.randint(len(roots), (1,), generator=g))]
    ctx = [S - b * (S // 3) for b in range(B)]
    first = torch.stack([torch.randint(0, c + 1, (K,), generator=g) for c in ctx])
    first[0, -1] = -3  # from the start
    want = []
    for k, v, k_pool, v_pool, table in pools:
        k2, v2 = k_pool.clone(), v_pool.clone()
        vb = min(PT, 32)
        for b in range(B):
            for j in range(K):
                p = int(parents[b, j])
                if p == j:
                    continue
                for t in range(max(0, int(first[b, j])), ctx[b]):
                    src, dst = (int(table[b * K + r, t // PT]) for r in (p, j))
                    o = t % PT
                    k2[dst, :, o] = k_pool[src, :, o]
                    v2[dst, :, o // vb, :, o % vb] = v_pool[src, :, o // vb, :, o % vb]
        want.append((k2, v2))
    dev = dict(dtype=torch.int32, device="cuda")
    ops.fork_kv([p[2] for p in pools], [p[3] for p in pools], [p[4] for p in pools],
                lens_tensor(ctx), parents.to(**dev), first.to(**dev))
    torch.cuda.synchronize()
    for (_, _, k_pool, v_pool, _), (k2, v2) in zip(pools, want):
        assert torch.equal(k_pool.view(torch.int16), k2.view(torch.int16))
        assert torch.equal(v_pool.view(torch.int16), v2.view(torch.int16))


@pytest.mark.gpu
def test_fork_leaves_out_what_lies_outside():
    """Parents, contexts and slot ids out of range: nothing else is written."""
    (k, v, k_pool, v_pool, table), = layers_of(1, 1, 4, 2, 64, 32, 64, 3)
    before = k_pool.clone(), v_pool.clone()
    dev = dict(dtype=torch.int32, device="cuda")
    wild = torch.tensor([[0, -1, 99, 3]], **dev)
    ops.fork_kv([k_pool], [v_pool], [table], lens_tensor([64]), wild)
    bad = table.clone()
    bad[1], bad[2] = -1, 10 ** 6
    ops.fork_kv([k_pool], [v_pool], [bad], lens_tensor([64]),
                torch.tensor([[0, 0, 0, 1]], **dev))
    ops.fork_kv([k_pool], [v_pool], [table], lens_tensor([-5]),
                torch.tensor([[0, 0, 0, 0]], **dev))
    torch.cuda.synchronize()
    assert torch.equal(k_pool.view(torch.int16), before[0].view(torch.int16))
    assert torch.equal(v_pool.view(torch.int16), before[1].view(torch.int16))
    ops.fork_kv([k_pool], [v_pool], [table], lens_tensor([10 ** 6]),  # clamped to the table
                torch.tensor([[2, 2, 2, 2]], **dev))
    torch.cuda.synchronize()
    kt, vt = tokens_of(k_pool, v_pool, table, 64, 32)
    for r in range(4):
        assert torch.equal(kt[r], k.transpose(1, 2)[2]) and torch.equal(vt[r], v.transpose(1, 2)[2])


@pytest.mark.gpu
def test_fork_refusals():
    (_, _, k_pool, v_pool, table), = layers_of(1, 2, 2, 2, 64, 32, 40, 3)
    dev = dict(dtype=torch.int32, device="cuda")
    good = dict(k_pools=[k_pool], v_pools=[v_pool], block_tables=[table],
                ctx_lens=lens_tensor([40, 40]), parents=torch.tensor([[0, 0], [1, 1]], **dev))

    def refused(match, **change):
        with pytest.raises(ValueError, match=match):
            ops.fork_kv(**{**good, **change})

    refused("one entry", k_pools=[])
    refused("one entry", v_pools=[v_pool, v_pool])
    refused("contiguous", k_pools=[k_pool.transpose(2, 3)])
    refused("bfloat16", k_pools=[k_pool.half()])
    refused("v_pool", v_pools=[v_pool[:1]])
    refused("block_table", block_tables=[table[:3]])
    refused("block_table", block_tables=[table.long()])
    refused("parents", parents=torch.tensor([0, 0], **dev))
    refused("ctx_lens", ctx_lens=lens_tensor([40]))
    refused("first", first=torch.tensor([[0, 0]], **dev))
    ops.set_bounds_checks(True)
    try:
        refused("parents", parents=torch.tensor([[0, 2], [1, 1]], **dev))
        refused("own parent", parents=torch.tensor([[1, 0], [1, 1]], **dev))
        refused("context lengths", ctx_lens=lens_tensor([40, 400]))
    finally:
        ops.set_bounds_checks(False)


def test_abi_refusals():
    """Refused on the host, before any launch (pointers that are never read)."""
    from voom_amd import _lib

    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def select(match, logits=p, dtype=2, last=None, end=0, shared=None, ctx=None, ws=p,
               ws_bytes=1 << 30, batch=1, beams=2, vocab=9):
        rc = lib.voom_beam_select(logits, dtype, p, last, end, shared, ctx, p, p, p, None, None,
                                  ws, ws_bytes, batch, beams, vocab, None)
        assert rc == _lib.VOOM_EINVAL and match in _lib.last_error(), (rc, _lib.last_error())

    select("null pointer", logits=None)
    select("null pointer", ws=None)
    for bad in (dict(batch=0), dict(beams=0), dict(beams=33), dict(vocab=0),
                dict(vocab=(1 << 24) + 1), dict(batch=65536)):
        select("beams", **bad)
        sizes = {**dict(batch=1, beams=2, vocab=9), **bad}
        assert lib.voom_beam_select_workspace_bytes(*sizes.values()) == 0
    select("bf16 or fp32", dtype=1)
    select("end token", last=p, end=9)
    select("shared", shared=p)
    select("aligned", logits=ctypes.c_void_p(258))
    select("workspace", ws_bytes=8)

    def fork(match, layers=1, batch=1, beams=2, nkv=2, d=64, page=32, pages=3, slots=4, pool=p):
        arr, num = (ctypes.c_void_p * 1)(pool), lambda x: (ctypes.c_int * 1)(x)
        good = (ctypes.c_void_p * 1)(p)
        rc = lib.voom_fork_kv(arr, good, good, num(pages), num(slots), layers, p, p, None, batch,
                              beams, nkv, d, page, None)
        assert rc == _lib.VOOM_EINVAL and match in _lib.last_error(), (rc, _lib.last_error())

    for bad in (dict(layers=0), dict(batch=0), dict(beams=0), dict(nkv=0), dict(batch=40000)):
        fork("geometry", **bad)
    for d in (0, 4, 1032):
        fork("head_dim", d=d)
    for page in (4, 24, 8192):
        fork("page_tokens", page=page)
    fork("aligned", pool=ctypes.c_void_p(264))
    fork("pages", pages=0)
    fork("pages", slots=0)
    fork("pages", pages=1 << 26)


def test_parents_are_checked_on_the_host_too():
    with pytest.raises(ValueError, match="outside"):
        ops.check_parents(torch.tensor([[0, 2]]))
    with pytest.raises(ValueError, match="own parent"):
        ops.check_parents(torch.tensor([[1, 0]]))
    ops.check_parents(torch.tensor([[1, 1], [0, 1]]))

"""GPU parity of the head norms, rotation and page write of new tokens
(ops.qk_norm_rope_append) against fp64.

Bar: everything runs in fp32 and is rounded to bf16 once, off by at most eps / 2 = 2^-8 of
the value.  Before it: the sum of at most 256 squares, root, quotient and two products are
off by less than 2^-18 of the normed value (the squares are positive: at most 8 in a chain
and 5 exchanges; 2^-24 each), and a rotated value a cos - b sin by that and three roundings
of |a| + |b|: 2^-17 (|a| + |b|).
"""
import pytest
import torch

from paged_inputs import lens_tensor
from voom_amd import _lib, ops
from voom_amd.kv_paged import PagedKVCache
from voom_amd.page_pool import v_slot_shape

HALF_BF16, FP32 = 2.0 ** -8, 2.0 ** -17


def reference(qkv, cos, sin, positions, nq, nkv, hd, wq, wk, eps, pairs):
    """fp64 (heads [B, L, nq + 2 nkv, hd], their bar)."""
    B, L, _ = qkv.shape
    x = qkv.double().view(B, L, nq + 2 * nkv, hd).clone()
    size = x.abs()
    for sl, w in ((slice(0, nq), wq), (slice(nq, nq + nkv), wk)):
        if w is not None:
            y = x[:, :, sl]
            x[:, :, sl] = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + eps) * w.double()
    half = cos.shape[1]
    i = torch.arange(half, device=qkv.device)
    a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    at = positions.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    qk = x[:, :, :nq + nkv]
    u, v = qk[..., a].clone(), qk[..., b].clone()
    size = x.abs()
    qk[..., a], qk[..., b] = u * c - v * s, v * c + u * s
    size[:, :, :nq + nkv, a] = size[:, :, :nq + nkv, b] = u.abs() + v.abs()
    return x, HALF_BF16 * x.abs() + FP32 * size


def make(B, L, nq, nkv, hd, rot, PT, ctx, seed=1, norm="both", dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-ctx // PT)
    slots = B * pages + 2
    st = {"qkv": torch.randn((B, L, (nq + 2 * nkv) * hd), generator=g, device="cuda").to(dtype),
          "k": torch.randn((slots, nkv, PT, hd), generator=g, device="cuda").to(dtype),
          "v": torch.randn((slots,) + v_slot_shape(nkv, hd, PT), generator=g,
                           device="cuda").to(dtype)}
    perm = torch.randperm(slots, generator=torch.Generator().manual_seed(seed))
    st["table"] = perm[:B * pages].view(B, pages).int().cuda().contiguous()
    st["cos"], st["sin"] = ops.rope_cache(ctx + 5, rot, 1e4)
    w = (1 + 0.3 * torch.randn((2, hd), generator=g, device="cuda")).to(dtype)
    st["wq"] = w[0].contiguous() if norm in ("both", "q") else None
    st["wk"] = w[1].contiguous() if norm in ("both", "k") else None
    return st


def written(st, ctx):
    return ops.gather_kv(st["k"], st["v"], st["table"], ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("B,L,nq,nkv,hd,rot,PT,ctx,norm", [
    (1, 1, 9, 3, 64, 64, 64, 640, "both"),
    (3, 13, 28, 4, 128, 64, 64, 300, "both"),
    (2, 7, 4, 2, 128, 128, 256, 257, "none"),
    (2, 40, 4, 1, 128, 16, 32, 100, "q"),
    (1, 33, 2, 2, 96, 96, 16, 70, "k"),       # heads of 12 chunks; pages below a V block
    (2, 5, 3, 1, 80, 32, 1, 9, "both"),       # one-token pages
    (1, 3, 1, 1, 256, 256, 64, 64, "both"),
    (1, 3, 5, 1, 16, 16, 8, 64, "both"),
    (1, 301, 32, 8, 128, 128, 64, 333, "both"),
    (2, 65, 6, 2, 64, 48, 4096, 90, "both"),
])
def test_against_fp64(pairs, B, L, nq, nkv, hd, rot, PT, ctx, norm):
    print(f"[qk] pairs={pairs} B={B} L={L} nq={nq} nkv={nkv} hd={hd} rot={rot} PT={PT} {norm}",
          flush=True)
    st = make(B, L, nq, nkv, hd, rot, PT, ctx, norm=norm)
    g = torch.Generator().manual_seed(3)
    start = [int(torch.randint(0, ctx - L + 1, (1,), generator=g)) for _ in range(B)]
    lens = [L] + [int(torch.randint(0, L + 1, (1,), generator=g)) for _ in range(B - 1)]
    positions = torch.randint(0, ctx, (B, L), generator=g).int().cuda()
    eps = 1e-5
    before_k, before_v = written(st, ctx)
    q = ops.qk_norm_rope_append(st["qkv"], st["cos"], st["sin"], positions, st["k"], st["v"],
                                st["table"], lens_tensor(start), nq, nkv, q_weight=st["wq"],
                                k_weight=st["wk"], eps=eps, interleaved=pairs,
                                new_lens=lens_tensor(lens))
    torch.cuda.synchronize()
    want, bar = reference(st["qkv"], st["cos"], st["sin"], positions, nq, nkv, hd, st["wq"],
                          st["wk"], eps, pairs)
    off = (q.transpose(1, 2).double() - want[:, :, :nq]).abs()
    assert (off <= bar[:, :, :nq]).all()
    got_k, got_v = written(st, ctx)
    v_new = st["qkv"].view(B, L, nq + 2 * nkv, hd)[:, :, nq + nkv:].transpose(1, 2)
    for b in range(B):
        rows = slice(start[b], start[b] + lens[b])
        k_want = want[b, :lens[b], nq:nq + nkv].transpose(0, 1)
        k_bar = bar[b, :lens[b], nq:nq + nkv].transpose(0, 1)
        assert ((got_k[b, :, rows].double() - k_want).abs() <= k_bar).all()
        assert torch.equal(got_v[b, :, rows], v_new[b, :, :lens[b]])
        before_k[b, :, rows], before_v[b, :, rows] = got_k[b, :, rows], got_v[b, :, rows]
    assert torch.equal(got_k, before_k) and torch.equal(got_v, before_v)  # the others as they were


@pytest.mark.gpu
def test_bad_places_are_not_written_and_positions_clamped():
    print("[qk] clamps", flush=True)
    B, L, nq, nkv, hd, PT, ctx = 4, 6, 2, 1, 64, 32, 64
    st = make(B, L, nq, nkv, hd, 64, PT, ctx)
    st["table"][2, 0], st["table"][3, 1] = -1, 1 << 25
    positions = torch.tensor([[-7, 0, 1, 60, 10 ** 6, 2 ** 31 - 1]] * B, dtype=torch.int32).cuda()
    k0, v0 = st["k"].clone(), st["v"].clone()
    q = ops.qk_norm_rope_append(st["qkv"], st["cos"], st["sin"], positions, st["k"], st["v"],
                                st["table"], lens_tensor([-3, 61, 29, 2 ** 31 - 4]), nq, nkv,
                                q_weight=st["wq"], k_weight=st["wk"], eps=0.0)
    torch.cuda.synchronize()
    want, bar = reference(st["qkv"], st["cos"], st["sin"], positions, nq, nkv, hd, st["wq"],
                          st["wk"], 0.0, False)
    assert ((q.transpose(1, 2).double() - want[:, :, :nq]).abs() <= bar[:, :, :nq]).all()
    k, v = st["k"].clone(), st["v"].clone()
    # sequence 1: tokens 0..2 at 61..63; sequence 2: 29..31 have no page, 32..34 do
    for b, t, at in ((1, 0, 61), (1, 1, 62), (1, 2, 63), (2, 3, 32), (2, 4, 33), (2, 5, 34)):
        slot, off = int(st["table"][b, at // PT]), at % PT
        assert ((k[slot, 0, off].double() - want[b, t, nq]).abs() <= bar[b, t, nq]).all()
        assert torch.equal(v[slot, 0, 0, :, off], st["qkv"][b, t, (nq + nkv) * hd:])
        k[slot, 0, off], v[slot, 0, 0, :, off] = k0[slot, 0, off], v0[slot, 0, 0, :, off]
    assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.gpu
def test_matches_the_rotation_without_norms():
    """Whole-head half layout without norms: the separate rope_split and append_kv, to the
    last place of the rounding."""
    B, L, nq, nkv, hd, PT, ctx = 2, 9, 9, 3, 64, 64, 128
    st = make(B, L, nq, nkv, hd, hd, PT, ctx, norm="none")
    at = torch.arange(30, 30 + L, dtype=torch.int32, device="cuda")
    full = [torch.cat((t[30:30 + L],) * 2, -1).contiguous() for t in (st["cos"], st["sin"])]
    q0, k0, v0 = ops.rope_split(st["qkv"], *full, nq, nkv, hd)
    q = ops.qk_norm_rope_append(st["qkv"], st["cos"], st["sin"], at.repeat(B, 1), st["k"], st["v"],
                                st["table"], lens_tensor([30, 30]), nq, nkv)
    k, v = written(st, ctx)
    torch.cuda.synchronize()
    assert torch.equal(v[:, :, 30:30 + L], v0)
    for a, b in ((q, q0), (k[:, :, 30:30 + L], k0)):
        assert ((a.double() - b.double()).abs() <= 2 * HALF_BF16 * b.double().abs() + 1e-6).all()


@pytest.mark.gpu
def test_graph_replays_and_empty_calls():
    st = make(2, 3, 4, 2, 64, 64, 32, 96)
    positions, start = torch.full((2, 3), 4, dtype=torch.int32).cuda(), lens_tensor([40, 7])

    def run():
        return ops.qk_norm_rope_append(st["qkv"], st["cos"], st["sin"], positions, st["k"], st["v"],
                                       st["table"], start, 4, 2, q_weight=st["wq"],
                                       k_weight=st["wk"])

    eager = run().clone()
    k, v = st["k"].clone(), st["v"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = run()
    for _ in range(3):
        q.zero_()
        st["k"].zero_()
        st["v"].zero_()
        st["k"].copy_(k)
        st["v"].copy_(v)
        st["k"][st["table"][0, 1].long()] = 0
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, eager)
        want = k.clone()
        want[st["table"][0, 1].long()] = 0
        want[st["table"][0, 1].long(), :, 8:11] = k[st["table"][0, 1].long(), :, 8:11]
        assert torch.equal(st["k"], want) and torch.equal(st["v"], v)
    for B, L in ((0, 3), (2, 0)):
        q = ops.qk_norm_rope_append(st["qkv"][:B, :L].contiguous(), st["cos"], st["sin"],
                                    positions[:B, :L].contiguous(), st["k"], st["v"],
                                    st["table"][:B], start[:B], 4, 2)
        assert q.shape == (B, 4, L, 64)


@pytest.mark.gpu
def test_wrapper_refusals():
    st = make(2, 3, 4, 2, 64, 64, 32, 96)
    good = dict(qkv=st["qkv"], cos=st["cos"], sin=st["sin"],
                positions=torch.zeros((2, 3), dtype=torch.int32, device="cuda"), k=st["k"],
                v=st["v"], table=st["table"], start=lens_tensor([0, 0]), nq=4, nkv=2)

    def refused(match, q_weight=None, new_lens=None, eps=1e-6, **change):
        with pytest.raises(ValueError, match=match):
            ops.qk_norm_rope_append(*{**good, **change}.values(), q_weight=q_weight,
                                    new_lens=new_lens, eps=eps)

    refused("ROCm", qkv=st["qkv"].cpu())
    refused("contiguous", qkv=st["qkv"].transpose(0, 1))
    refused("qkv must", qkv=st["qkv"][..., :-64].contiguous())
    refused("bfloat16", qkv=st["qkv"].half())
    refused("geometry", nkv=3)
    refused("v_pool", v=st["v"].transpose(2, 3).contiguous())
    refused("cos and sin", cos=st["cos"].half())
    refused("cos and sin", sin=st["sin"][:, :8].contiguous())
    refused("positions", positions=good["positions"].long())
    refused("positions", positions=good["positions"][:, :2].contiguous())
    refused("block_table", table=st["table"].long())
    refused("start", start=lens_tensor([0]))
    refused("new_lens", new_lens=lens_tensor([1]))
    refused("q_weight", q_weight=st["wq"][:32].contiguous())
    refused("q_weight", q_weight=st["wq"].float())
    refused("eps", eps=-1.0)
    refused("rotary_dim", cos=st["cos"][:, :12].contiguous(), sin=st["sin"][:, :12].contiguous())


def test_abi_refusals():
    """Refused on the host, before any launch (pointers that are never read)."""
    import ctypes

    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def refused(match, qkv=p, eps=1e-6, rows=8, rot=64, batch=1, new=3, nq=4, nkv=2, hd=64,
                page=64, pages=2, slots=2):
        rc = lib.voom_qk_norm_rope_append(qkv, None, None, eps, p, p, rows, rot, 0, p, p, p, p, p, p,
                                          None, batch, new, nq, nkv, hd, page, pages, slots, None)
        assert rc == _lib.VOOM_EINVAL and match in _lib.last_error(), (rc, _lib.last_error())

    refused("null pointer", qkv=None)
    refused("aligned", qkv=ctypes.c_void_p(264))
    for bad in (dict(batch=0), dict(new=0), dict(nq=0), dict(nkv=0), dict(pages=0), dict(slots=0),
                dict(rows=0)):
        refused("geometry", **bad)
    for hd in (0, 24, 272):
        refused("head_dim", hd=hd)
    for rot in (0, 24, 80):
        refused("rotary_dim", rot=rot)
    refused("page_tokens", page=48)
    refused("block table", pages=1 << 25)
    refused("eps", eps=-1.0)


def test_checked_places_and_positions():
    def i32(x):
        return torch.tensor(x, dtype=torch.int32)

    table = i32([[3, 5], [4, -1]])  # pages of 8 tokens in a pool of 6
    good = dict(positions=i32([[0, 9, 4], [2, 2, 77]]), rope_rows=10, block_table=table,
                start=i32([13, 6]), new_lens=i32([3, 2]), num_slots=6, page=8)
    ops.check_new_tokens(**good)
    ops.check_new_tokens(**{**good, "new_lens": i32([0, 0]), "start": i32([99, -4])})
    for match, change in (("positions", dict(rope_rows=9)), ("positions", dict(new_lens=None)),
                          ("positions", dict(positions=i32([[-1, 0, 0], [0, 0, 0]]))),
                          ("new_lens", dict(new_lens=i32([4, 0]))),
                          ("new_lens", dict(new_lens=i32([-1, 0]))),
                          ("block table", dict(start=i32([14, 6]))),
                          ("block table", dict(start=i32([-1, 6]))),
                          ("block table", dict(start=i32([2 ** 31 - 2, 6]))),
                          ("block table", dict(block_table=table[:, :0])),
                          ("slot ids", dict(start=i32([13, 7]))),
                          ("slot ids", dict(num_slots=5))):
        with pytest.raises(ValueError, match=match):
            ops.check_new_tokens(**{**good, **change})


@pytest.mark.gpu
def test_checked_calls_raise_and_the_cache_refuses_positions_past_the_tables():
    print("[qk] checked calls", flush=True)
    B, L, nq, nkv, hd, PT, ctx = 2, 6, 2, 1, 64, 32, 64
    st = make(B, L, nq, nkv, hd, 64, PT, ctx)
    k0 = st["k"].clone()

    def call(positions, start):
        return ops.qk_norm_rope_append(st["qkv"], st["cos"], st["sin"], positions, st["k"],
                                       st["v"], st["table"], lens_tensor(start), nq, nkv)

    at = torch.arange(L, dtype=torch.int32, device="cuda").repeat(B, 1)
    ops.set_bounds_checks(True)
    try:
        for match, positions, start in (("positions", at + 64, [0, 0]),
                                        ("block table", at, [0, 59])):
            with pytest.raises(ValueError, match=match):
                call(positions, start)
        assert torch.equal(st["k"], k0)
        q = call(at + 63, [0, 58])
    finally:
        ops.set_bounds_checks(False)
    assert torch.equal(q, call(at + 63, [0, 58]))

    kv = PagedKVCache(1, 1 << 40, page_positions=PT)
    cos, sin = ops.rope_cache(10, hd, 1e4)
    kv.append_qkv(0, st["qkv"], cos, sin, nq, nkv)
    with pytest.raises(ValueError, match="6 tokens from position 6 on, but cos and sin hold 10"):
        kv.append_qkv(0, st["qkv"], cos, sin, nq, nkv)
    assert kv.offset == L
    kv.append_qkv(0, st["qkv"][:, :4].contiguous(), cos, sin, nq, nkv)
    kv.append_qkv(0, st["qkv"][:, :0].contiguous(), cos[:3], sin[:3], nq, nkv)
    assert kv.offset == 10

"""GPU parity of the norm behind a block joined with the residual add and the next norm
(voom_add_post_norm, ops.add_post_norm) against the formula in fp64.

Bars.  The stream: one rounding to bf16, 2^-8 of the value, and fp32 arithmetic on the two
terms, a mean of up to 8,192 squares (summed in at most 40 steps) and five roundings more:
under 2^-18 of their sizes.  The result: the same 2^-8, and of y's fp32 error and the second
mean as much again, 2^-17 of what the terms would give.
"""
import ctypes

import pytest
import torch

from voom_amd import ops

NAN = float("nan")


def reference(x, delta, post_weight, weight, eps, gate=None, scale=1.0):
    x, delta, post_weight, weight = (t.double() for t in (x, delta, post_weight, weight))
    H = x.shape[-1]
    r = delta / (delta.square().mean(-1, keepdim=True) + eps).sqrt() * post_weight * scale
    if gate is not None:
        rows = x.numel() // H
        groups = gate.shape[0] if gate.dim() == 2 else 1
        g = gate.double().view(groups, 1, H).expand(groups, rows // groups, H)
        r = r * g.reshape(x.shape)
    y = x + r
    inv = 1 / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    size = x.abs() + r.abs()
    return y, y * inv * weight, size, size * inv * weight.abs()


def make(*shape, seed=0, H=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, std=1.0):
        return (torch.randn(s, generator=g, device="cuda") * std).to(torch.bfloat16)

    H = shape[-1]
    return (rnd(*shape, std=3.0), rnd(*shape), 1 + rnd(H, std=0.2), 1 + rnd(H, std=0.2), rnd)


def check(y, out, want):
    torch.cuda.synchronize()
    ref_y, ref, size_y, size = want
    assert ((y.double() - ref_y).abs() <= ref_y.abs() * 2.0 ** -8 + size_y * 2.0 ** -18).all()
    assert ((out.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + size * 2.0 ** -17).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 8), (1, 576), (1, 1, 4096), (3, 5, 576), (7, 2048),
                                   (9, 2056), (2, 3, 8192), (5, 1000), (513, 24)])
@pytest.mark.parametrize("groups", [None, 0, 1, "rows"])
def test_post_norm_against_fp64(shape, groups):
    print(f"[post] {shape} gates={groups}", flush=True)
    x, delta, pw, w, rnd = make(*shape, seed=len(shape))
    rows, H = x.numel() // shape[-1], shape[-1]
    gate = None if groups is None else rnd(H) if groups == 0 else rnd(
        rows if groups == "rows" else groups, H)
    for scale in (1.0, 0.22, -2.0):
        want = reference(x, delta, pw, w, 1e-6, gate, scale)
        y = torch.full_like(x, NAN)
        before = x.clone()
        out = ops.add_post_norm(x, delta, pw, w, 1e-6, gate=gate, scale=scale, x_out=y)
        check(y, out, want)
        assert torch.equal(x, before)
        out2 = ops.add_post_norm(before, delta, pw, w, 1e-6, gate=gate, scale=scale)  # in place
        torch.cuda.synchronize()
        assert torch.equal(before, y) and torch.equal(out2, out)


@pytest.mark.gpu
def test_a_gate_for_each_sequence():
    x, delta, pw, w, rnd = make(3, 7, 264, seed=4)
    gate = rnd(3, 264)
    y = torch.empty_like(x)
    out = ops.add_post_norm(x, delta, pw, w, 1e-5, gate=gate, x_out=y)
    check(y, out, reference(x, delta, pw, w, 1e-5, gate))


@pytest.mark.gpu
def test_zero_rows_large_values_and_nan():
    x, delta, pw, w, _ = make(4, 512, seed=5)
    x[0], delta[0] = 0, 0
    x[1], delta[1] = x[1] * 1e15, delta[1] * 1e15
    delta[2, 77] = NAN
    y = torch.empty_like(x)
    out = ops.add_post_norm(x, delta, pw, w, 1e-6, x_out=y)
    torch.cuda.synchronize()
    assert (y[0] == 0).all() and (out[0] == 0).all()
    assert torch.isnan(out[2].float()).all() and torch.isfinite(out[3].float()).all()
    ref = reference(x, delta, pw, w, 1e-6)
    check(y[[1, 3]], out[[1, 3]], [t[[1, 3]] for t in ref])


@pytest.mark.gpu
def test_graph_and_side_stream():
    x, delta, pw, w, _ = make(100, 1024, seed=6)
    y = torch.empty_like(x)

    def run():
        return ops.add_post_norm(x, delta, pw, w, 1e-6, x_out=y)

    want, want_y = run().clone(), y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        out.zero_()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(y, want_y)


@pytest.mark.gpu
def test_refusals():
    x, delta, pw, w, rnd = make(6, 64)
    good = dict(x=x, delta=delta, post_weight=pw, weight=w, eps=1e-6)

    def refused(match, **change):
        with pytest.raises(ValueError, match=match):
            ops.add_post_norm(**{**good, **change})

    refused("bfloat16", x=x.float())
    refused("ROCm device", x=x.cpu())
    refused("contiguous", x=x.t().contiguous().t())
    refused("delta", delta=delta[:3])
    refused("delta", delta=delta.half())
    refused("weights", post_weight=pw[:32].contiguous())
    refused("weights", weight=w.float())
    refused("x_out", x_out=torch.empty(3, 64, device="cuda", dtype=torch.bfloat16))
    refused("gate", gate=rnd(4, 64))
    refused("gate", gate=rnd(0, 64))
    refused("gate", gate=rnd(64).float())
    refused("eps", eps=-1.0)
    odd = make(2, 60)
    refused("multiple of 8", **dict(zip(("x", "delta", "post_weight", "weight"), odd)))
    unaligned = torch.empty(6 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 64)
    refused("aligned", x=unaligned)
    assert ops.add_post_norm(x[:0], delta[:0], pw, w, 1e-6).shape == (0, 64)


def test_abi_refusals():
    """Refused on the host, before any launch (pointers that are never read)."""
    from voom_amd import _lib

    lib, p = _lib.lib(), ctypes.c_void_p(256)

    def refused(match, x=p, gate=None, gate_rows=0, rows=4, hidden=64, eps=1e-6):
        rc = lib.voom_add_post_norm(x, p, p, p, gate, gate_rows, p, p, rows, hidden, eps, 1.0,
                                    None)
        assert rc == _lib.VOOM_EINVAL and match in _lib.last_error(), (rc, _lib.last_error())

    refused("null pointer", x=None)
    for bad in (dict(rows=0), dict(hidden=0), dict(hidden=60), dict(hidden=8200)):
        refused("hidden", **bad)
    refused("gate", gate=p, gate_rows=3)
    refused("gate", gate=p)
    refused("eps", eps=-1.0)
    refused("eps", eps=float("nan"))
    refused("aligned", x=ctypes.c_void_p(264))

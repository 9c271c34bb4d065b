"""Beam selection over logits of which most or all lie far below zero: vocabularies whose
unused tokens are masked with large finite values, rows shifted as a whole, and rows with
few tokens above -inf.  The oracle and the bars are those of test_gpu_beams.py; a logit is
subtracted from one of its lane, exactly where both are of one size, and what lies further
off than the sum's rounding adds nothing to it, so that the bars hold for any shift.
"""
import pytest
import torch

from test_gpu_beams import INF, check, make, search
from voom_amd import ops

pytestmark = pytest.mark.gpu

# (1, 5): 8 logits a lane; (64, 4): 32 (256 pieces and more)
SHAPES = [(1, 5), (64, 4)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K", SHAPES)
@pytest.mark.parametrize("V,unused", [(700, 3), (1000, 300), (2050, 2), (8193, 1), (8200, 40)])
def test_unused_tokens_of_large_negative_logits(V, unused, B, K, dtype):
    print(f"[beam masks] B={B} K={K} V={V} unused={unused} {dtype}", flush=True)
    for low in (-100.0, -1e9, torch.finfo(dtype).min):
        logits, scores = make(B, K, V, dtype, V + K)
        logits[..., V - unused:] = low
        check(ops.beam_select(logits, scores), search(logits, scores))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K", SHAPES)
@pytest.mark.parametrize("V", [1, 700, 1000, 2050, 8193])
@pytest.mark.parametrize("shift", [-100.0, -1000.0, 1000.0])
def test_shifted_logits(V, B, K, dtype, shift):
    print(f"[beam masks] B={B} K={K} V={V} shift={shift} {dtype}", flush=True)
    logits, scores = make(B, K, V, dtype, V + B)
    logits += shift
    check(ops.beam_select(logits, scores), search(logits, scores))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K", SHAPES)
@pytest.mark.parametrize("V", [700, 2050, 9001])
def test_few_tokens_above_minus_infinity(V, B, K, dtype):
    print(f"[beam masks] few, B={B} K={K} V={V} {dtype}", flush=True)
    logits, scores = make(B, K, V, dtype, 3)
    logits[...] = -INF
    for token, value in ((3, -150.0), (V // 2, -152.0), (V - 1, -190.0)):
        logits[..., token] = value
    check(ops.beam_select(logits, scores), search(logits, scores))
    logits[..., 3] = torch.finfo(dtype).min
    check(ops.beam_select(logits, scores), search(logits, scores))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V", [(1, 5, 1), (2, 3, 40), (64, 4, 700), (1, 2, 9001)])
def test_rows_of_the_largest_floats(B, K, V, dtype):
    """All tokens of some beams at one value so large that a score beside it is lost: they are
    worth the score less log V, and tie."""
    print(f"[beam masks] large, B={B} K={K} V={V} {dtype}", flush=True)
    for value in (torch.finfo(dtype).min, torch.finfo(dtype).max, -1e30, 1e20):
        logits, scores = make(B, K, V, dtype, 7)
        logits[:, ::2] = value
        whole = logits.double()  # (less its maximum the oracle's sum keeps log V)
        want = search(whole - whole.amax(-1, keepdim=True), scores)
        check(ops.beam_select(logits, scores), want)

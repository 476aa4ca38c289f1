"""Masked attention with caps far past its scores, where capped scores are all but the scores themselves: what a program gets
that switches the cap off with a large value.

The bounds are those of the uncapped call (masked_reference.py), which do not grow with the cap, twice: a tanh to a few 2^-24 of
itself adds 4 * 2^-24 |s| to a score's 4 * 2^-24 |s|, and the probabilities that the bounds are taken at differ by at most 2 %
between the two (scores up to 10: s - x is at most x^3 / (3 cap^2) = 0.02 at a cap of 129)."""
import sys

import pytest
import torch

from masked_reference import attention, check, ranges_of

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("o", "lse", "dq", "dk", "dv")


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def make(seed, B, Sq, Skv, H, KH, D, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    shapes = ((B, Sq, H, D), (B, Skv, KH, D), (B, Skv, KH, D), (B, Sq, H, D))
    q, k, v, d_o = [torch.randn(s, generator=g).to(dtype).cuda() for s in shapes]
    return q * std, k, v, d_o


def run(ffk, variant, q, k, v, d_o, scale, **how):
    ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
    try:
        o, lse = ffk.masked_attention_forward(q, k, v, scale, **how)
        got = (o, lse) + tuple(ffk.masked_attention_backward(q, k, v, o, d_o, lse, scale, **how))
        torch.cuda.synchronize()
    finally:
        ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
    return dict(zip(NAMES, got))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sq,Skv,D", [(150, 150, 64), (150, 150, 128), (90, 200, 80), (70, 70, 256), (3, 2500, 128), (1, 2000, 40)])
@pytest.mark.parametrize("cap", [129.0, 1e3, 1e5, 1e8, 1e30])
@pytest.mark.parametrize("bias", [False, True])
def test_far_past_the_scores(ffk, Sq, Skv, D, cap, bias, dtype):
    B, H, KH, scale = 2, 4, 2, D ** -0.5
    q, k, v, d_o = make(Sq + D, B, Sq, Skv, H, KH, D, dtype)
    slopes = torch.tensor([2.0 ** -(h + 3) for h in range(H)]).cuda() if bias else None
    ranges = ranges_of(B, Sq, Skv, Sq == Skv, torch.tensor([[0, Skv // 3, Skv], [2, Skv // 2, Skv - 3]], dtype=torch.int32), None, Skv - Sq).cuda()
    how = dict(ranges=ranges, slopes=slopes, offset=Skv - Sq, d_o=d_o, unit=UNIT[dtype])
    want, plain = attention(q, k, v, scale, cap=cap, **how), attention(q, k, v, scale, **how)
    for name in NAMES:
        want[name + "_tol"] = 2 * plain[name + "_tol"]
    for variant in (1, 0):
        say("cap", cap, (Sq, Skv, D), bias, dtype, variant)
        got = run(ffk, variant, q, k, v, d_o, scale, score_cap=cap, key_ranges=ranges, distance_slopes=slopes, query_offset=Skv - Sq)
        for name in NAMES:
            check(got[name], want, name, "cap %g, variant %d, " % (cap, variant))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap", [100.0, 128.0, 200.0])
def test_scores_on_both_sides_of_the_cap(ffk, D, cap, dtype):
    """Scores of some hundreds, of which the tanh bends a part and flattens a part, on either side of where the kernels change."""
    q, k, v, d_o = make(D, 1, 130, 130, 4, 2, D, dtype, 80.0)
    want = attention(q, k, v, D ** -0.5, True, cap, None, None, 0, d_o, UNIT[dtype])
    for variant in (1, 0):
        say("both sides", cap, D, dtype, variant)
        got = run(ffk, variant, q, k, v, d_o, D ** -0.5, causal=True, score_cap=cap)
        for name in NAMES:
            check(got[name], want, name, "cap %g, variant %d, " % (cap, variant))

"""Rows of masked attention that see a single key: their probability is 1 whatever the score, so the scores have no gradient.
Nothing of such a row reaches dq and dk, not even rounding noise, next to which the true gradients of small batches would be
nothing."""
import sys

import pytest
import torch

from masked_reference import attention, check

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def make(seed, B, Sq, Skv, H, KH, D, dtype):
    g = torch.Generator().manual_seed(seed)
    shapes = ((B, Sq, H, D), (B, Skv, KH, D), (B, Skv, KH, D), (B, Sq, H, D))
    return [torch.randn(s, generator=g).to(dtype).cuda() for s in shapes]


def run(ffk, variant, q, k, v, d_o, **how):
    scale = q.shape[3] ** -0.5
    ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
    try:
        o, lse = ffk.masked_attention_forward(q, k, v, scale, **how)
        dq, dk, dv = ffk.masked_attention_backward(q, k, v, o, d_o, lse, scale, **how)
        torch.cuda.synchronize()
    finally:
        ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


SCORES = [(0.0, False), (20.0, False), (0.0, True), (5.0, True)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [8, 32, 64, 80, 128, 256])
@pytest.mark.parametrize("cap,bias", SCORES)
def test_every_row_sees_one_key(ffk, D, cap, bias, dtype):
    """Sequences of one position, many rows on the one key that there is, and rows with a key each, near and far."""
    H, KH = 4, 2
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)]).cuda() if bias else None
    for B, Sq, Skv, keys in ((8, 1, 1, lambda i: 0), (2, 200, 1, lambda i: 0), (2, 1, 700, lambda i: 401), (1, 300, 333, lambda i: i * 37 % 333),
                             (2, 150, 150, lambda i: i)):
        q, k, v, d_o = make(D + Sq + Skv, B, Sq, Skv, H, KH, D, dtype)
        ranges = torch.tensor([[[keys(i), keys(i) + 1] for i in range(Sq)]] * B, dtype=torch.int32).cuda()
        for variant in (1, 0):
            say("one key", dtype, D, cap, bias, (B, Sq, Skv), variant)
            got = run(ffk, variant, q, k, v, d_o, score_cap=cap, key_ranges=ranges, distance_slopes=slopes)
            assert not got["dq"].any() and not got["dk"].any(), ((B, Sq, Skv), variant, float(got["dq"].abs().max()), float(got["dk"].abs().max()))
            want = attention(q, k, v, D ** -0.5, cap=cap, ranges=ranges, slopes=slopes, d_o=d_o, unit=UNIT[dtype])
            for name in ("o", "lse", "dv"):
                check(got[name], want, name)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap,bias", SCORES)
def test_among_rows_that_see_more(ffk, D, cap, bias, dtype):
    """First positions of causal documents, and every third row of a batch whose others see all keys: zero there, and what the
    others give is as without them."""
    B, S, H, KH = 2, 290, 4, 2
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)]).cuda() if bias else None
    q, k, v, d_o = make(D + 5, B, S, S, H, KH, D, dtype)
    starts = torch.tensor([[0, 1, 2, 140, 290], [3, 133, 134, 200, 280]], dtype=torch.int32).cuda()
    documents = ffk.attention_key_ranges(B, S, S, causal=True, document_starts=starts)
    thirds = torch.tensor([[[i, i + 1] if i % 3 == 0 else [0, S] for i in range(S)]] * B, dtype=torch.int32).cuda()
    for ranges in (documents, thirds):
        one = (ranges[..., 1] - ranges[..., 0] == 1).cpu()
        want = attention(q, k, v, D ** -0.5, cap=cap, ranges=ranges, slopes=slopes, d_o=d_o, unit=UNIT[dtype])
        for variant in (1, 0):
            say("among others", dtype, D, cap, bias, variant)
            got = run(ffk, variant, q, k, v, d_o, score_cap=cap, key_ranges=ranges, distance_slopes=slopes)
            for name in ("o", "lse", "dq", "dk", "dv"):
                check(got[name], want, name, "variant %d, " % variant)
            assert not got["dq"].cpu()[one].any()
            if ranges is documents:
                continue
            # dk again from the other rows alone (which see the same windows of keys)
            rest = torch.where(one.cuda()[..., None], torch.zeros_like(ranges), ranges)
            o, lse = got["o"], got["lse"]
            ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
            try:
                without = ffk.masked_attention_backward(q, k, v, o, d_o, lse, D ** -0.5, score_cap=cap, key_ranges=rest, distance_slopes=slopes)[1]
                torch.cuda.synchronize()
            finally:
                ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
            assert torch.equal(without, got["dk"]), variant

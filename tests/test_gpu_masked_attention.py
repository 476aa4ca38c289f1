"""Masked attention and the key ranges against their definitions in 64 bits, within bounds that follow from the roundings
(tests/masked_reference.py)."""
import ctypes
import math
import sys

import pytest
import torch

from masked_reference import attention, check, ranges_of

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def make(seed, B, Sq, Skv, H, KH, D, Dv, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    shapes = ((B, Sq, H, D), (B, Skv, KH, D), (B, Skv, KH, Dv), (B, Sq, H, Dv))
    q, k, v, d_o = (torch.randn(s, generator=g).to(dtype) for s in shapes)
    return (q * std).cuda(), k.cuda(), v.cuda(), d_o.cuda()


def run(ffk, q, k, v, d_o, scale, **how):
    o, lse = ffk.masked_attention_forward(q, k, v, scale, **how)
    dq, dk, dv = ffk.masked_attention_backward(q, k, v, o, d_o, lse, scale, **how)
    torch.cuda.synchronize()
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def compare(ffk, q, k, v, d_o, causal=False, cap=0.0, ranges=None, slopes=None, offset=0):
    """By the kernels that the size asks for, and by those for many rows and keys."""
    scale = q.shape[3] ** -0.5
    want = attention(q, k, v, scale, causal, cap, ranges, slopes, offset, d_o, UNIT[q.dtype])
    for variant in (1, 0):
        ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
        try:
            got = run(ffk, q, k, v, d_o, scale, causal=causal, score_cap=cap, key_ranges=ranges, distance_slopes=slopes, query_offset=offset)
        finally:
            ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
        for name in ("o", "lse", "dq", "dk", "dv"):
            check(got[name], want, name, "variant %d, " % variant)
    return got


def slopes_of(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=F32).cuda()


# --------------------------------------------------------------------------
# key ranges
# --------------------------------------------------------------------------
@pytest.mark.parametrize("starts", [
    [[0, 5, 5, 12, 30], [3, 3, 10, 20, 29]],  # empty documents, positions before the first and behind the last
    [[0, 0, 0, 0, 0], [30, 30, 30, 30, 30]],  # no position in any
    [[0, 1, 2, 3, 4], [-4, 2, 7, 90, 95]],    # documents of one position; starts outside of the positions
])
@pytest.mark.parametrize("causal", [False, True])
def test_key_ranges_of_documents(ffk, starts, causal):
    st = torch.tensor(starts, dtype=torch.int32)
    prefixes = torch.tensor([[0, 3, 99, 2], [1, -5, 2, 4]], dtype=torch.int32)
    for pre in (None, prefixes) if causal else (None,):
        for seq_q, seq_kv, offset in ((30, 30, 0), (7, 30, 11), (30, 17, 0), (1, 40, 29)):
            say("key ranges", seq_q, seq_kv, offset, pre is not None)
            got = ffk.attention_key_ranges(2, seq_q, seq_kv, causal=causal, document_starts=st.cuda(),
                                           prefix_lengths=None if pre is None else pre.cuda(), query_offset=offset)
            want = ranges_of(2, seq_q, seq_kv, causal, st.clamp(min=0), pre, offset)
            assert torch.equal(got.cpu(), want), (got.cpu(), want)


def test_key_ranges_without_documents(ffk):
    for causal, pre in ((False, None), (True, None), (True, [[4], [0], [100]])):
        pre = None if pre is None else torch.tensor(pre, dtype=torch.int32)
        got = ffk.attention_key_ranges(3, 9, 7, causal=causal, prefix_lengths=None if pre is None else pre.cuda())
        assert torch.equal(got.cpu(), ranges_of(3, 9, 7, causal, None, pre))


def test_key_ranges_in_any_order_stay_inside(ffk):
    """Starts that descend mean nothing, but every range stays within the keys."""
    st = torch.tensor([[50, -9, 2000000000, 3, -2000000000, 7]], dtype=torch.int32).cuda()
    pre = torch.full((1, 5), 2147483647, dtype=torch.int32).cuda()
    got = ffk.attention_key_ranges(1, 300, 40, causal=True, document_starts=st, prefix_lengths=pre).cpu()
    assert int(got.min()) >= 0 and int(got.max()) <= 40
    assert bool(((got[..., 0] < got[..., 1]) | (got == 0).all(dim=-1)).all())


def test_key_ranges_of_many_rows(ffk):
    g = torch.Generator().manual_seed(3)
    st = torch.randint(0, 701, (5, 41), generator=g, dtype=torch.int32).sort(dim=1).values
    pre = torch.randint(0, 30, (5, 40), generator=g, dtype=torch.int32)
    got = ffk.attention_key_ranges(5, 700, 700, causal=True, document_starts=st.cuda(), prefix_lengths=pre.cuda())
    assert torch.equal(got.cpu(), ranges_of(5, 700, 700, True, st, pre))


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------
SHAPES = [  # B, Sq, Skv, H, KH, D, Dv
    (1, 1, 1, 1, 1, 64, 64), (2, 1, 70, 4, 2, 64, 64), (1, 31, 33, 2, 2, 128, 128), (2, 129, 129, 4, 1, 64, 64),
    (1, 200, 200, 2, 1, 128, 128), (1, 70, 300, 2, 2, 64, 64), (1, 300, 70, 3, 3, 128, 128),
    (1, 65, 65, 2, 1, 256, 256), (2, 50, 90, 6, 2, 80, 80), (1, 40, 40, 2, 2, 8, 8), (1, 37, 64, 3, 1, 96, 96),
    (1, 100, 100, 2, 1, 64, 128), (1, 90, 60, 2, 2, 128, 40), (1, 33, 140, 4, 4, 256, 64), (1, 45, 45, 1, 1, 200, 24),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
def test_shapes(ffk, shape, causal, dtype):
    say("masked attention", shape, "causal", causal, dtype)
    B, Sq, Skv, H, KH, D, Dv = shape
    compare(ffk, *make(Sq + Skv + D, *shape, dtype), causal=causal)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (5.0, True)])
def test_capped_and_biased(ffk, D, cap, bias, dtype):
    say("masked attention", D, "cap", cap, "bias", bias, dtype)
    B, S, H, KH = 2, 150, 4, 2
    q, k, v, d_o = make(D, B, S, S, H, KH, D, D, dtype, 3.0 if cap else 1.0)
    starts = torch.tensor([[0, 70, 140], [10, 11, 150]], dtype=torch.int32)
    ranges = ffk.attention_key_ranges(B, S, S, causal=True, document_starts=starts.cuda(),
                                      prefix_lengths=torch.tensor([[20, 0], [5, 40]], dtype=torch.int32).cuda())
    compare(ffk, q, k, v, d_o, cap=cap, ranges=ranges, slopes=slopes_of(H) if bias else None)


RANGES = {
    # rows that see nothing beside rows that see one key, the last key, or all
    "mixed": lambda B, Sq, Skv: [[[0, 0], [i % Skv, i % Skv + 1], [Skv - 1, Skv], [0, Skv], [5, 2], [-7, 1 << 30]][i % 6] for i in range(Sq)],
    "none": lambda B, Sq, Skv: [[0, 0]] * Sq,
    "window": lambda B, Sq, Skv: [[max(0, i - 40), min(Skv, i + 3)] for i in range(Sq)],
    # whole blocks of rows without keys between blocks with some, far apart
    "blocks": lambda B, Sq, Skv: [[0, 0] if (i // 50) % 2 else [Skv - 64 - i // 50, Skv - i // 50] for i in range(Sq)],
    "descending": lambda B, Sq, Skv: [[max(0, Skv - 20 - i), max(1, Skv - i)] for i in range(Sq)],
}


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kind", sorted(RANGES))
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_given_ranges(ffk, kind, D, dtype):
    say("masked attention, ranges", kind, D, dtype)
    B, Sq, Skv, H, KH = 2, 260, 290, 2, 1
    q, k, v, d_o = make(D + 1, B, Sq, Skv, H, KH, D, D, dtype)
    rows = RANGES[kind](B, Sq, Skv)
    ranges = torch.tensor([rows, rows[::-1]], dtype=torch.int32).cuda()
    got = compare(ffk, q, k, v, d_o, ranges=ranges)
    if kind == "none":
        assert all(not got[n].any() for n in ("o", "dq", "dk", "dv"))


@pytest.mark.parametrize("kind", sorted(RANGES) + ["causal"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, False), (0.0, True), (5.0, True)])
def test_every_kind_of_score(ffk, kind, D, cap, bias):
    """The kernels of heads of 64 and 128 over every kind of range, with heads that share keys."""
    say("masked attention", kind, D, cap, bias)
    B, Sq, Skv, H, KH = 2, 210, 290, 6, 2
    q, k, v, d_o = make(D + 2, B, Sq, Skv, H, KH, D, D, BF, 3.0 if cap else 1.0)
    ranges = None
    if kind != "causal":
        rows = RANGES[kind](B, Sq, Skv)
        ranges = torch.tensor([rows, rows[::-1]], dtype=torch.int32).cuda()
    compare(ffk, q, k, v, d_o, causal=kind == "causal", cap=cap, ranges=ranges, slopes=slopes_of(H) if bias else None)


@pytest.mark.parametrize("G", [1, 3, 8])
def test_heads_that_share_keys(ffk, G):
    """Row tiles that begin inside a query row's heads (G does not divide 64), and those that do not."""
    compare(ffk, *make(50 + G, 1, 90, 150, 2 * G, 2, 64, 64, BF), causal=True)


def test_kernels_that_the_size_asks_for(ffk):
    """Workgroups for every CU, so that the kernels for many rows and keys run by themselves."""
    compare(ffk, *make(40, 4, 70, 1030, 64, 64, 64, 64, BF), causal=False, cap=20.0)


@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles_of_rows(ffk, D, cap, bias):
    """More tiles of rows than the dK/dV kernel lists at a time, most of which see none of a workgroup's keys."""
    B, Sq, Skv, H, KH = 1, 6000, 300, 6, 1
    q, k, v, d_o = make(D + 3, B, Sq, Skv, H, KH, D, D, BF)
    ranges = torch.tensor([[[0, 0] if i % 700 < 300 else [i * 37 % 250, i * 37 % 250 + 1 + i % 50] for i in range(Sq)]], dtype=torch.int32).cuda()
    compare(ffk, q, k, v, d_o, ranges=ranges, cap=cap, slopes=slopes_of(H) if bias else None)


@pytest.mark.parametrize("D,Dv", [(8, 8), (40, 40), (72, 72), (88, 96), (96, 64), (104, 104), (120, 16), (16, 128)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, True)])
def test_heads_of_other_sizes(ffk, D, Dv, cap, bias):
    """Heads that the kernels make longer with zeros: nothing of the next head, or of what lies behind a row's heads, enters."""
    H, KH, B, Sq, Skv = 4, 2, 2, 150, 170
    for rows in (Sq, 3):
        tensors = make(D + Dv, B, rows, Skv, H, KH, D, Dv, BF)
        wide = []
        for x in tensors:  # the second key head's, and behind every row, are NaN
            half = x.shape[2] * x.shape[3] // 2
            w = torch.full((B, x.shape[1], 2 * half + 8), float("nan"), dtype=BF, device="cuda")
            w[:, :, :half] = x.flatten(2)[:, :, :half]
            wide.append(w)
        q, k, v, d_o = wide
        slopes = slopes_of(H) if bias else None
        scale, offset = D ** -0.5, Skv - rows
        strides = [n for x in wide for n in x.stride()[:2]]
        desc = ffk.MaskedAttentionDesc(B, H, KH, rows, Skv, D, Dv, *strides, offset, scale, cap, 1)
        first = [x[:, :, :x.shape[2] // 2].contiguous() for x in tensors]
        want = attention(*first[:3], scale, True, cap, None, slopes[:H // 2] if bias else None, offset, first[3], UNIT[BF])
        for variant in (1, 0):
            say("heads", D, Dv, rows, variant)
            ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
            try:
                o, grads = torch.full_like(d_o, 7.0), [torch.full_like(x, 7.0) for x in (q, k, v)]
                _, lse = ffk.masked_attention_forward(q, k, v, scale, distance_slopes=slopes, desc=desc, out=o)
                ffk.masked_attention_backward(q, k, v, o, d_o, lse, scale, distance_slopes=slopes, desc=desc, grads=grads)
                torch.cuda.synchronize()
            finally:
                ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
            for name, w in zip(("o", "dq", "dk", "dv"), [o] + grads):
                assert bool((w[:, :, -8:] == 7.0).all()), name
                n = want[name].shape[2]
                check(w[:, :, :(w.shape[2] - 8) // 2].unflatten(2, (n, -1)), want, name, "variant %d, " % variant)
            check(lse[:, :H // 2].contiguous(), want, "lse")


@pytest.mark.parametrize("S,D", [(2, 64), (5, 32), (9, 256), (33, 128), (100, 80)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (50.0, True)])
def test_gradients_of_few_keys(ffk, S, D, cap, bias):
    """bf16 rows with their probability on few keys: dQ and dK have the roundings of dS and of the result, two of at most 2^-8 a
    value, spread evenly and apart: sqrt(2 / 3) 2^-8 = 0.0032 of their length, and not that of the stored O besides (which
    left 0.006)."""
    q, k, v, d_o = make(S, 8, S, S, 4, 4, D, D, BF, std=3.0)
    slopes = slopes_of(4) if bias else None
    want = attention(q, k, v, D ** -0.5, True, cap, None, slopes, 0, d_o, UNIT[BF])
    for variant in (1, 0):
        ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
        try:
            got = run(ffk, q, k, v, d_o, D ** -0.5, causal=True, score_cap=cap, distance_slopes=slopes)
        finally:
            ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
        for name in ("dq", "dk"):
            off = float((got[name].cpu().double() - want[name]).norm() / want[name].norm())
            assert off <= 0.0032, (name, variant, off)


def test_ranges_and_causal_both_apply(ffk):
    q, k, v, d_o = make(4, 1, 200, 200, 2, 2, 64, 64, BF)
    ranges = torch.tensor([[[i // 2, 200] for i in range(200)]], dtype=torch.int32).cuda()
    compare(ffk, q, k, v, d_o, causal=True, ranges=ranges)


def test_rows_further_on(ffk):
    """A chunk of rows that stand behind their first keys: the last rows of the whole sequence's."""
    q, k, v, d_o = make(5, 2, 30, 130, 4, 2, 64, 64, BF)
    compare(ffk, q, k, v, d_o, causal=True, slopes=slopes_of(4), offset=100)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sq,H,KH,D", [(1, 8, 2, 128), (3, 4, 4, 64), (1, 1, 1, 256), (17, 2, 1, 80)])
def test_few_rows_over_long_keys(ffk, Sq, H, KH, D, dtype):
    """The keys in parts, with and without scratch for them; parts that a row does not see."""
    Skv = 5000
    say("few rows", Sq, H, KH, D, dtype)
    q, k, v, d_o = make(D + Sq, 3, Sq, Skv, H, KH, D, D, dtype)
    ranges = torch.tensor([[[0, Skv]] * Sq, [[0, 0]] * Sq, [[2100, 2101 + i] for i in range(Sq)]], dtype=torch.int32).cuda()
    compare(ffk, q, k, v, d_o, ranges=ranges, cap=30.0)
    scale = D ** -0.5
    want = attention(q, k, v, scale, cap=30.0, ranges=ranges, unit=UNIT[dtype])
    desc = ffk.masked_attention_desc(q, k, v, scale, score_cap=30.0)
    need = ffk._call.ffk_masked_attention_forward_workspace_bytes(desc, ffk.dtype_of(q))
    assert need > 0
    small = torch.empty((need - 4,), dtype=torch.uint8, device="cuda")
    for workspace in (small, torch.empty((0,), dtype=torch.uint8, device="cuda")):
        o, lse = ffk.masked_attention_forward(q, k, v, scale, score_cap=30.0, key_ranges=ranges, workspace=workspace)
        torch.cuda.synchronize()
        check(o, want, "o")
        check(lse, want, "lse")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_what_no_row_sees_is_not_read(ffk, dtype):
    """Padding behind the documents holds NaN and infinities, in q, k, v and the output gradient."""
    B, S, H, KH, D = 2, 400, 2, 1, 64
    q, k, v, d_o = make(6, B, S, S, H, KH, D, D, dtype)
    for n, t in enumerate((q, k, v, d_o)):
        t[0, 250:] = float("nan")
        t[1, :60] = float("inf") if n % 2 else float("-inf")
    starts = torch.tensor([[0, 130, 250], [60, 200, 400]], dtype=torch.int32).cuda()
    ranges = ffk.attention_key_ranges(B, S, S, causal=True, document_starts=starts)
    got = compare(ffk, q, k, v, d_o, ranges=ranges)
    assert not got["o"][0, 250:].any() and not got["dk"][0, 250:].any() and not got["dq"][1, :60].any()


def test_far_scores(ffk):
    """Scores of some thousands: softmax picks, nothing overflows; a bias of thousands on far keys."""
    q, k, v, d_o = make(8, 1, 90, 90, 2, 2, 64, 64, BF, std=600.0)
    o, lse = ffk.masked_attention_forward(q, k, v, 0.125)
    grads = ffk.masked_attention_backward(q, k, v, o, d_o, lse, 0.125)
    assert all(torch.isfinite(t).all() for t in (o, lse) + grads)
    want = attention(q, k, v, 0.125, unit=2.0 ** -8)
    check(lse, want, "lse")
    # rows that see only keys more than a thousand positions away
    q, k, v, d_o = make(9, 1, 4, 1500, 2, 2, 64, 64, BF)
    ranges = torch.tensor([[[1200, 1500]] * 4], dtype=torch.int32).cuda()
    compare(ffk, q, k, v, d_o, ranges=ranges, slopes=torch.tensor([4.0, 0.5]).cuda())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_strides(ffk, dtype):
    """q, k and v in one fused buffer whose batch entries lie between each other's rows; gradients with the same strides,
    and what lies between them left as it was."""
    B, S, H, KH, D = 2, 75, 4, 2, 64
    g = torch.Generator().manual_seed(11)
    width = (H + 2 * KH) * D + 16
    fused = torch.randn((S, B, width), generator=g).to(dtype).cuda()
    q = fused[:, :, :H * D].reshape(S, B, H, D).permute(1, 0, 2, 3).contiguous()
    k = fused[:, :, H * D:(H + KH) * D].reshape(S, B, KH, D).permute(1, 0, 2, 3).contiguous()
    v = fused[:, :, (H + KH) * D:(H + 2 * KH) * D].reshape(S, B, KH, D).permute(1, 0, 2, 3).contiguous()
    d_o = torch.randn((B, S, H, D), generator=g).to(dtype).cuda()
    scale = D ** -0.5
    desc = ffk.MaskedAttentionDesc(B, H, KH, S, S, D, 0, width, B * width, width, B * width, width, B * width, S * H * D, H * D, 0, scale, 0.0, 1)
    flat = fused.view(-1)
    qf, kf, vf = flat, flat[H * D:], flat[(H + KH) * D:]
    o, lse = ffk.masked_attention_forward(qf, kf, vf, scale, desc=desc)
    grads = torch.full_like(flat, 7.0)
    ffk.masked_attention_backward(qf, kf, vf, o, d_o, lse, scale, desc=desc, grads=(grads, grads[H * D:], grads[(H + KH) * D:]))
    torch.cuda.synchronize()
    want = attention(q, k, v, scale, causal=True, d_o=d_o, unit=UNIT[dtype])
    check(o, want, "o")
    grads = grads.view(S, B, width)
    check(grads[:, :, :H * D].reshape(S, B, H, D).permute(1, 0, 2, 3), want, "dq")
    check(grads[:, :, H * D:(H + KH) * D].reshape(S, B, KH, D).permute(1, 0, 2, 3), want, "dk")
    check(grads[:, :, (H + KH) * D:-16].reshape(S, B, KH, D).permute(1, 0, 2, 3), want, "dv")
    assert bool((grads[:, :, -16:] == 7.0).all())


def test_agrees_with_the_plain_attention(ffk):
    """Without any of its additions it is ffk_attention_forward / _backward."""
    q, k, v, d_o = make(12, 2, 160, 160, 4, 4, 64, 64, BF)
    got = compare(ffk, q, k, v, d_o, causal=True)
    o, lse = ffk.attention_forward(q, k, v, 0.125, True)
    want = attention(q, k, v, 0.125, True, d_o=d_o, unit=2.0 ** -8)
    check(o, want, "o")
    assert float((lse - got["lse"]).abs().max()) < 1e-4


def test_same_bits_twice(ffk):
    q, k, v, d_o = make(13, 2, 333, 333, 4, 1, 128, 128, BF)
    first = run(ffk, q, k, v, d_o, 0.1, causal=True, score_cap=15.0)
    again = run(ffk, q, k, v, d_o, 0.1, causal=True, score_cap=15.0)
    assert all(torch.equal(first[n], again[n]) for n in first)


def test_gradients_against_differences(ffk):
    """The loss sum(o * d_o), in 64 bits, moves along a direction as the gradients say."""
    B, S, H, KH, D = 1, 40, 4, 2, 32
    q, k, v, d_o = make(14, B, S, S, H, KH, D, D, F32, 2.0)
    starts = torch.tensor([[0, 17, 36]], dtype=torch.int32)
    pre = torch.tensor([[5, 0]], dtype=torch.int32)
    ranges = ranges_of(B, S, S, True, starts, pre)
    slopes = slopes_of(H)
    got = run(ffk, q, k, v, d_o, D ** -0.5, score_cap=4.0, key_ranges=ranges.cuda(), distance_slopes=slopes)
    g, h = torch.Generator().manual_seed(15), 1e-4
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for _ in range(3):
            step = torch.randn(t.shape, generator=g, dtype=torch.float64)

            def loss(sign):
                moved = {"dq": q.cpu().double(), "dk": k.cpu().double(), "dv": v.cpu().double()}
                moved[name] = moved[name] + sign * h * step
                o = attention(moved["dq"], moved["dk"], moved["dv"], D ** -0.5, cap=4.0, ranges=ranges, slopes=slopes)["o"]
                return float((o * d_o.cpu().double()).sum())

            slope, says = (loss(1) - loss(-1)) / (2 * h), float((got[name].cpu().double() * step).sum())
            size = float((got[name].cpu().double() * step).abs().sum())
            # the difference's own error is of order h^2, the kernel's of order 2^-20 of the terms
            assert abs(slope - says) < 1e-6 * size + 1e-5, (name, slope, says)


def test_gradients_of_shared_heads_are_sums(ffk):
    """dk and dv of shared heads are those of repeated ones, added up."""
    B, S, H, KH, D = 1, 140, 6, 2, 64
    q, k, v, d_o = make(16, B, S, S, H, KH, D, D, F32)
    one = run(ffk, q, k, v, d_o, 0.125, causal=True)
    wide = run(ffk, q, k.repeat_interleave(3, dim=2).contiguous(), v.repeat_interleave(3, dim=2).contiguous(), d_o, 0.125, causal=True)
    for n in ("dk", "dv"):
        torch.testing.assert_close(one[n], wide[n].view(B, S, KH, 3, D).sum(dim=3), rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(one["o"], wide["o"], rtol=1e-5, atol=1e-5)


def test_offsets_past_32_bits(ffk):
    """Keys and values of a cache whose rows lie more than 2^32 bytes from its start."""
    S, H, KH, D = 1100, 2, 1, 64
    stride = 1 << 21  # elements of 2 bytes: 1100 rows span 4.3 GiB
    q, k, v, d_o = make(17, 1, 40, S, H, KH, D, D, BF)
    big = torch.zeros((S * stride,), dtype=BF, device="cuda")
    rows = big.view(S, stride)
    rows[:, :D], rows[:, D:2 * D] = k[0, :, 0], v[0, :, 0]
    desc = ffk.MaskedAttentionDesc(1, H, KH, 40, S, D, 0, 40 * H * D, H * D, S * stride, stride, S * stride, stride, 40 * H * D, H * D, 0,
                                   0.125, 0.0, 0)
    o, lse = ffk.masked_attention_forward(q, big, big[D:], 0.125, desc=desc)
    grads = torch.zeros_like(big)
    dq = torch.empty_like(q)
    ffk.masked_attention_backward(q, big, big[D:], o, d_o, lse, 0.125, desc=desc, grads=(dq, grads, grads[D:]))
    torch.cuda.synchronize()
    want = attention(q, k, v, 0.125, d_o=d_o, unit=2.0 ** -8)
    check(o, want, "o")
    check(dq, want, "dq")
    check(grads.view(S, stride)[:, :D].reshape(1, S, 1, D), want, "dk")
    check(grads.view(S, stride)[:, D:2 * D].reshape(1, S, 1, D), want, "dv")


@pytest.mark.parametrize("D,Sq", [(64, 70), (128, 70), (80, 3)])
def test_rows_too_far_apart_for_short_offsets(ffk, D, Sq):
    """Row strides of 2^24 elements, which the tuned kernels' offsets do not reach: the general ones, both forms."""
    S, H, KH, stride = 130, 2, 1, 1 << 24
    q, k, v, d_o = make(D, 1, Sq, S, H, KH, D, D, BF)
    keys, rows = torch.zeros((S, stride), dtype=BF, device="cuda"), torch.zeros((Sq, stride), dtype=BF, device="cuda")
    keys[:, :D], keys[:, D:2 * D], rows[:, :H * D], rows[:, H * D:2 * H * D] = k[0, :, 0], v[0, :, 0], q[0].flatten(1), d_o[0].flatten(1)
    desc = ffk.MaskedAttentionDesc(1, H, KH, Sq, S, D, 0, Sq * stride, stride, S * stride, stride, S * stride, stride, Sq * stride, stride,
                                   S - Sq, 0.125, 20.0, 1)
    want = attention(q, k, v, 0.125, causal=True, cap=20.0, offset=S - Sq, d_o=d_o, unit=2.0 ** -8)
    qf, kf = rows.view(-1), keys.view(-1)
    vf, gf = kf[D:], qf[H * D:]
    out, dkeys = torch.full_like(rows, 7.0), torch.full_like(keys, 7.0)
    for variant in (1, 0):
        say("far apart", D, Sq, variant)
        ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, variant)
        try:
            of, dk = out.view(-1), dkeys.view(-1)
            o, lse = ffk.masked_attention_forward(qf, kf, vf, 0.125, desc=desc, out=of)
            ffk.masked_attention_backward(qf, kf, vf, o, gf, lse, 0.125, desc=desc, grads=(of[H * D:], dk, dk[D:]))
            torch.cuda.synchronize()
        finally:
            ffk.set_option(ffk.OPTION_ATTENTION_VARIANT, 0)
        check(lse, want, "lse")
        for name, t, at, n in (("o", out, 0, H), ("dq", out, H * D, H), ("dk", dkeys, 0, KH), ("dv", dkeys, D, KH)):
            check(t[:, at:at + n * D].reshape(1, -1, n, D), want, name, "variant %d, " % variant)
        assert bool((out[:, 2 * H * D:2 * H * D + 64] == 7.0).all()) and bool((dkeys[:, 2 * D:2 * D + 64] == 7.0).all())


def test_another_stream_and_a_replayed_graph(ffk):
    """Ranges, forward and backward captured once and replayed on new inputs, eager calls between the replays."""
    B, S, H, KH, D = 2, 300, 4, 2, 64
    q, k, v, d_o = make(18, B, S, S, H, KH, D, D, BF)
    starts = torch.tensor([[0, 100, 280], [0, 7, 300]], dtype=torch.int32).cuda()

    def step():
        ranges = ffk.attention_key_ranges(B, S, S, causal=True, document_starts=starts)
        o, lse = ffk.masked_attention_forward(q, k, v, 0.125, score_cap=20.0, key_ranges=ranges)
        return (o, lse) + tuple(ffk.masked_attention_backward(q, k, v, o, d_o, lse, 0.125, score_cap=20.0, key_ranges=ranges))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(3):
        q.copy_(make(20 + n, B, S, S, H, KH, D, D, BF)[0])
        starts[0, 1] = 50 * n + 3
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), n
        torch.cuda.synchronize()


def test_two_calls_at_once(ffk):
    """Two streams, scratch of their own: the calls do not meet."""
    a = make(30, 1, 1, 4096, 8, 2, 128, 128, BF)
    b = make(31, 2, 500, 500, 4, 2, 64, 64, BF)
    alone = run(ffk, *a, 0.1), run(ffk, *b, 0.125)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for n, (s, t, scale) in enumerate(zip(streams, (a, b), (0.1, 0.125))):
            with torch.cuda.stream(s):
                o, lse = ffk.masked_attention_forward(*t[:3], scale)
                got[n] = (o, lse) + ffk.masked_attention_backward(*t[:3], o, t[3], lse, scale)
    torch.cuda.synchronize()
    for n in range(2):
        for x, name in zip(got[n], ("o", "lse", "dq", "dk", "dv")):
            assert torch.equal(x, alone[n][name]), name

"""Rotary positions with several axes against the definition in 64 bits."""
import math
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
UNIT = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def turned(x, positions, frequencies, sections, interleaved, sign=1):
    """(x turned, how far a result may be off) in 64 bits: the angle's cosine and sine are within 2^-21 in 32 bits, the two products and
    their sum within 2^-23 of the terms' sizes, and the result is rounded once."""
    x = x.detach().cpu().double()
    n = sum(sections)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    theta = positions.cpu().double()[axis].permute(1, 2, 0) * frequencies.cpu().double()
    c, s = theta.cos()[:, :, None], sign * theta.sin()[:, :, None]
    first = list(range(0, 2 * n, 2)) if interleaved else list(range(n))
    second = list(range(1, 2 * n, 2)) if interleaved else list(range(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out, tol = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    slack = 2.0 ** -20 * (a.abs() + b.abs())
    tol[..., first], tol[..., second] = slack, slack
    return out, tol


def check(got, want, tol, unit):
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol + unit * want.abs()).all()), float((off - tol - unit * want.abs()).max())


def make(seed, B, S, H, KH, D, dtype, axes, far):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((B, S, H, D), generator=g).to(dtype).cuda()
    k = torch.randn((B, S, KH, D), generator=g).to(dtype).cuda() if KH else None
    return q, k, torch.randint(0, far, (axes, B, S), generator=g, dtype=torch.int32).cuda()


def table(n):
    return torch.tensor([10000.0 ** (-i / n) for i in range(n)], dtype=F32).cuda()


CASES = [  # B, S, H, KH, D, sections
    (1, 1, 1, 1, 2, [1]), (2, 5, 3, 1, 64, [32]), (1, 196, 4, 4, 64, [16, 16]), (2, 37, 8, 2, 128, [16, 24, 24]),
    (1, 9, 2, 0, 80, [20, 20]), (3, 17, 4, 2, 128, [8, 8]), (1, 33, 2, 1, 96, [1, 2, 3, 4]), (2, 11, 5, 5, 40, [5, 7]),
    (1, 3, 2, 2, 256, [0, 128]), (1, 700, 12, 4, 66, [11, 11, 11]), (1, 3, 1, 1, 4096, [2048]), (2, 6, 3, 1, 10, [3]),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(ffk, case, interleaved, dtype):
    B, S, H, KH, D, sections = case
    say("rotary", case, interleaved, dtype)
    q, k, positions = make(D + S, B, S, H, KH, D, dtype, len(sections), 5000)
    freq = table(sum(sections))
    for entry, sign in ((ffk.rotary_forward, 1), (ffk.rotary_backward, -1)):
        got = entry(q, k, positions, freq, sections, interleaved=interleaved)
        torch.cuda.synchronize()
        for x, y in zip((q, k), got):
            if x is not None:
                check(y, *turned(x, positions, freq, sections, interleaved, sign), UNIT[dtype])


def test_far_positions(ffk):
    """Position 2^31 - 1 turns by its own angle, not by a rounded one."""
    q, k, _ = make(1, 1, 6, 2, 2, 64, F32, 1, 2)
    positions = torch.tensor([[[0, 1, -3, 1000003, 2147483647, -2147483648]]], dtype=torch.int32).cuda()
    freq = table(32)
    got, _ = ffk.rotary_forward(q, k, positions, freq, [32])
    check(got, *turned(q, positions, freq, [32], False), UNIT[F32])


def test_there_and_back(ffk):
    q, k, positions = make(2, 2, 50, 4, 2, 128, F32, 3, 100000)
    a, b = ffk.rotary_forward(q, k, positions, table(64), [16, 24, 24])
    a, b = ffk.rotary_backward(a, b, positions, table(64), [16, 24, 24])
    torch.testing.assert_close(a, q, rtol=0, atol=2e-6 * 5)
    torch.testing.assert_close(b, k, rtol=0, atol=2e-6 * 5)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_in_place_in_a_fused_buffer(ffk, dtype, interleaved, shift):
    """q and k turned where they lie among other columns, at any alignment; all else is left as it was."""
    B, S, H, KH, D, sections = 2, 19, 4, 2, 48, [10, 6]
    width = (H + 2 * KH) * D + (3 if shift == 1 else 8)
    g = torch.Generator().manual_seed(shift)
    flat = torch.randn((B * S * width + shift,), generator=g).to(dtype).cuda()
    positions = torch.randint(0, 900, (2, B, S), generator=g, dtype=torch.int32).cuda()
    before = flat.clone()
    desc = ffk.RotaryDesc(B, S, H, KH, D, *(S * width, width) * 4, 2, (ffk.c_i64 * 4)(*sections), int(interleaved))
    q, k = flat[shift:], flat[shift + H * D:]
    ffk.rotary_forward(q, k, positions, table(16), sections, desc=desc, q_out=q, k_out=k)
    torch.cuda.synchronize()
    rows, old = flat[shift:].view(B, S, width), before[shift:].view(B, S, width)
    for at, heads in ((0, H), (H * D, KH)):
        check(rows[..., at:at + heads * D].reshape(B, S, heads, D), *turned(old[..., at:at + heads * D].reshape(B, S, heads, D), positions,
                                                                            table(16), sections, interleaved), UNIT[dtype])
    assert torch.equal(rows[..., (H + KH) * D:], old[..., (H + KH) * D:])
    assert torch.equal(flat[:shift], before[:shift])


def test_batch_entries_between_rows_and_outputs_of_their_own_strides(ffk):
    B, S, H, KH, D, sections = 3, 7, 2, 1, 32, [16]
    q, k, positions = make(5, B, S, H, KH, D, BF, 1, 77)
    qs, ks = q.permute(1, 0, 2, 3).contiguous(), k.permute(1, 0, 2, 3).contiguous()
    desc = ffk.RotaryDesc(B, S, H, KH, D, H * D, B * H * D, KH * D, B * KH * D, S * H * D, H * D, S * KH * D, KH * D, 1,
                          (ffk.c_i64 * 4)(16, 0, 0, 0), 0)
    got = ffk.rotary_forward(qs, ks, positions, table(16), sections, desc=desc)
    for x, y in zip((q, k), got):
        check(y.view(x.shape), *turned(x, positions, table(16), sections, False), 2.0 ** -8)


def test_gradient_against_differences(ffk):
    """The loss sum(out * g) along a direction: the operator is linear, so the difference is exact but for roundings."""
    q, k, positions = make(6, 1, 20, 2, 2, 32, F32, 2, 300)
    g, step = torch.randn_like(q), torch.randn_like(q)
    dq, _ = ffk.rotary_backward(g, None, positions, table(16), [10, 6])
    up, _ = ffk.rotary_forward(q + step, None, positions, table(16), [10, 6])
    down, _ = ffk.rotary_forward(q - step, None, positions, table(16), [10, 6])
    slope = float(((up.double() - down.double()) * g.double()).sum()) / 2
    says, size = float((dq.double() * step.double()).sum()), float((dq.double() * step.double()).abs().sum())
    assert abs(slope - says) < 2.0 ** -19 * size


def test_replayed_graph(ffk):
    q, k, positions = make(7, 2, 64, 4, 4, 64, BF, 2, 99)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ffk.rotary_forward(q, k, positions, table(32), [16, 16])
    torch.cuda.synchronize()
    freq = table(32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ffk.rotary_forward(q, k, positions, freq, [16, 16])
    for n in range(3):
        q.copy_(make(8 + n, 2, 64, 4, 4, 64, BF, 2, 99)[0])
        positions.add_(n)
        graph.replay()
        torch.cuda.synchronize()
        again = ffk.rotary_forward(q, k, positions, freq, [16, 16])
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_offsets_past_32_bits(ffk):
    """A row that begins more than 2^32 bytes behind its tensor."""
    stride, D = (1 << 31) + 64, 64
    flat = torch.zeros((stride + D,), dtype=BF, device="cuda")
    x = torch.randn((1, 2, 1, D)).to(BF).cuda()
    flat[:D], flat[stride:] = x[0, 0, 0], x[0, 1, 0]
    positions = torch.tensor([[[3, 4]]], dtype=torch.int32).cuda()
    desc = ffk.RotaryDesc(1, 2, 1, 0, D, 0, stride, 0, 0, 0, stride, 0, 0, 1, (ffk.c_i64 * 4)(32, 0, 0, 0), 0)
    ffk.rotary_forward(flat, None, positions, table(32), [32], desc=desc, q_out=flat)
    got = torch.stack([flat[:D], flat[stride:]]).view(1, 2, 1, D)
    check(got, *turned(x, positions, table(32), [32], False), 2.0 ** -8)

"""The operators of a training step with packed documents one behind the other: rotary positions, key ranges, masked attention
forward and backward, the rotary gradient, the gradient norm with clipping, the update; and one step of serving a token."""
import math
import sys

import pytest
import torch

from masked_reference import attention, check, ranges_of
from test_gpu_grad_norm import NORM_TOL, check_clipped, norm_of
from test_gpu_rotary import check as check_turned
from test_gpu_rotary import table, turned

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
UNIT = {BF: 2.0 ** -8, F32: 2.0 ** -24}
SECTIONS = [8, 12, 12]


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


class Layer:
    """Queries, keys and values as the trained tensors, drawn to a target."""

    def __init__(self, ffk, seed, B, S, H, KH, D, dtype):
        g = torch.Generator().manual_seed(seed)
        self.ffk, self.B, self.S, self.scale = ffk, B, S, D ** -0.5
        self.weights = [torch.randn((B, S, n, D), generator=g).cuda() for n in (H, KH, KH)]
        self.moments = [[torch.zeros_like(w), torch.zeros_like(w)] for w in self.weights]
        self.low = [w.to(dtype) for w in self.weights]
        self.target = torch.randn((B, S, H, D), generator=g).cuda()
        self.positions = torch.randint(0, 5000, (3, B, S), generator=g, dtype=torch.int32).cuda()
        self.frequencies = table(32)
        self.starts = torch.tensor([[0, S // 3, S // 3 + 1, S - 5]] * B, dtype=torch.int32).cuda()
        self.prefixes = torch.tensor([[7, 0, 3]] * B, dtype=torch.int32).cuda()
        self.slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)]).cuda()

    def step(self):
        ffk = self.ffk
        q, k, v = self.low
        ranges = ffk.attention_key_ranges(self.B, self.S, self.S, causal=True, document_starts=self.starts, prefix_lengths=self.prefixes)
        how = dict(score_cap=15.0, key_ranges=ranges, distance_slopes=self.slopes)
        qr, kr = ffk.rotary_forward(q, k, self.positions, self.frequencies, SECTIONS)
        o, lse = ffk.masked_attention_forward(qr, kr, v, self.scale, **how)
        d_o = (o.float() - self.target).to(o.dtype)
        dqr, dkr, dv = ffk.masked_attention_backward(qr, kr, v, o, d_o, lse, self.scale, **how)
        dq, dk = ffk.rotary_backward(dqr, dkr, self.positions, self.frequencies, SECTIONS)
        grads = [dq, dk, dv]
        clipped, norm = ffk.clip_grad_norm(grads, 1.0, out=[torch.empty_like(x) for x in grads])
        for w, x, (m, s), low in zip(self.weights, clipped, self.moments, self.low):
            ffk.adam_update(w, x, m, s, 0.01, weight_lowp=low if low.dtype == BF else None)
            if low.dtype != BF:
                low.copy_(w)
        return dict(qr=qr, kr=kr, o=o, lse=lse, d_o=d_o, dqr=dqr, dkr=dkr, dq=dq, dk=dk, dv=dv, norm=norm, ranges=ranges, clipped=clipped)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,S,H,KH,D", [(1, 17, 2, 1, 64), (2, 150, 6, 2, 80), (1, 333, 8, 8, 128)])
def test_every_stage_of_a_step(ffk, dtype, B, S, H, KH, D):
    """Each operator on what the one before it left, against its definition and within its own bound."""
    say("step", dtype, B, S, H, KH, D)
    layer = Layer(ffk, S, B, S, H, KH, D, dtype)
    q, k, v = [x.clone() for x in layer.low]
    out = layer.step()
    torch.cuda.synchronize()
    assert torch.equal(out["ranges"].cpu(), ranges_of(B, S, S, True, layer.starts.cpu(), layer.prefixes.cpu(), 0))
    for x, y in ((q, "qr"), (k, "kr")):
        check_turned(out[y], *turned(x, layer.positions, layer.frequencies, SECTIONS, False), UNIT[dtype])
    want = attention(out["qr"], out["kr"], v, layer.scale, False, 15.0, out["ranges"], layer.slopes, 0, out["d_o"], UNIT[dtype])
    check(out["o"], want, "o")
    check(out["lse"], want, "lse")
    check(out["dqr"], want, "dq")
    check(out["dkr"], want, "dk")
    check(out["dv"], want, "dv")
    for x, y in (("dqr", "dq"), ("dkr", "dk")):
        check_turned(out[y], *turned(out[x], layer.positions, layer.frequencies, SECTIONS, False, sign=-1), UNIT[dtype])
    grads = [out[n] for n in ("dq", "dk", "dv")]
    norm = norm_of(grads)
    assert norm > 1.0 and abs(float(out["norm"]) - norm) <= NORM_TOL * norm
    check_clipped(out["clipped"], grads, norm, 1.0)


def test_gradient_of_the_whole(ffk):
    """fp32 against automatic differentiation of the plain form in 64 bits.  Five stages, each of a few hundred roundings of 2^-24
    that add at worst linearly: 1e-4 of a gradient's length leaves a factor of ten for what the exponentials amplify (scores
    to 15)."""
    B, S, H, KH, D = 2, 90, 4, 2, 64
    layer = Layer(ffk, 5, B, S, H, KH, D, F32)
    q, k, v = [w.detach().cpu().double().requires_grad_() for w in layer.weights]
    out = layer.step()
    torch.cuda.synchronize()
    axis = [a for a, s in enumerate(SECTIONS) for _ in range(s)]
    theta = layer.positions.cpu().double()[axis].permute(1, 2, 0) * layer.frequencies.cpu().double()
    c, s = theta.cos()[:, :, None], theta.sin()[:, :, None]

    def turn(x):
        a, b = x[..., :32], x[..., 32:]
        return torch.cat([a * c - b * s, a * s + b * c], dim=3)

    kk, vv = (x.repeat_interleave(H // KH, dim=2).permute(0, 2, 1, 3).contiguous() for x in (turn(k), v))
    x = (turn(q).permute(0, 2, 1, 3) @ kk.transpose(2, 3)) * layer.scale
    i, j = torch.arange(S)[:, None], torch.arange(S)[None, :]
    x = 15.0 * torch.tanh(x / 15.0) - layer.slopes.cpu().double()[None, :, None, None] * (i - j).abs()
    lo, hi = ranges_of(B, S, S, True, layer.starts.cpu(), layer.prefixes.cpu(), 0).unbind(dim=2)
    seen = (j >= lo[:, :, None]) & (j < hi[:, :, None])
    x = x.masked_fill(~seen[:, None], float("-inf"))
    some = seen.any(dim=2)[:, None, :, None]
    p = torch.softmax(x.masked_fill(~some, 0.0), dim=3) * some
    o = (p @ vv).permute(0, 2, 1, 3)
    (0.5 * (o - layer.target.cpu().double()).square()).sum().backward()
    for got, w in zip((out["dq"], out["dk"], out["dv"]), (q, k, v)):
        assert float((got.cpu().double() - w.grad).norm()) <= 1e-4 * float(w.grad.norm())


def test_replayed_steps(ffk):
    """Steps captured once and replayed, eager work between: the same weights as by eager steps, bit for bit."""
    a, b = (Layer(ffk, 9, 2, 150, 6, 2, 80, BF) for _ in range(2))
    a.step(), b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step()
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = b.step()
        torch.cuda.synchronize()
        assert math.isfinite(float(out["norm"])) and torch.equal(out["norm"], want["norm"]), n
        for x, y in zip(a.weights + a.low, b.weights + b.low):
            assert torch.equal(x, y), n


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_a_token_at_a_time(ffk, dtype):
    """A sequence's last tokens served one by one over the keys before them: what the whole sequence's rows give, to the roundings of
    both."""
    B, S, H, KH, D = 2, 700, 8, 2, 128
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((B, S, n, D), generator=g).to(dtype).cuda() for n in (H, KH, KH))
    positions = torch.arange(S, dtype=torch.int32).expand(1, B, S).contiguous().cuda()
    frequencies = table(64)
    qr, kr = ffk.rotary_forward(q, k, positions, frequencies, [64])
    begin = torch.tensor([0, 123], dtype=torch.int32)  # a padded batch: keys in front of the second sequence's first
    starts = torch.stack([begin, torch.full((B,), S, dtype=torch.int32)], dim=1).cuda()
    want = attention(qr, kr, v, D ** -0.5, False, 30.0, ranges_of(B, S, S, True, starts.cpu(), None, 0).cuda(), None, 0, None, UNIT[dtype])
    for at in (S - 3, S - 1):
        q1, _ = ffk.rotary_forward(q[:, at:at + 1].contiguous(), None, positions[:, :, at:at + 1].contiguous(), frequencies, [64])
        assert torch.equal(q1, qr[:, at:at + 1])
        ranges = ffk.attention_key_ranges(B, 1, S, causal=True, document_starts=starts, query_offset=at)
        o, lse = ffk.masked_attention_forward(q1, kr, v, D ** -0.5, score_cap=30.0, key_ranges=ranges, query_offset=at)
        torch.cuda.synchronize()
        row = {n: want[n][:, at:at + 1] for n in ("o", "o_tol")}
        check(o, row, "o")
        check(lse, {n: want[n][:, :, at:at + 1] for n in ("lse", "lse_tol")}, "lse")

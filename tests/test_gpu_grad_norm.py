"""The global gradient norm and clipping against 64-bit sums."""
import math
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
# the norm: squares and sums in 64 bits, one rounding to fp32.  A clipped value: the factor's rounding, the product's and, in
# bf16, the store's.
NORM_TOL, UNIT = 2.0 ** -23, {BF: 2.0 ** -8 + 2.0 ** -22, F32: 2.0 ** -22}


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def make(sizes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn((n,), generator=g) * scale).to(BF if i % 3 == 1 else F32).cuda() for i, n in enumerate(sizes)]


def norm_of(grads):
    return math.sqrt(sum(float(g.cpu().double().square().sum()) for g in grads))


def check_clipped(got, grads, norm, max_norm):
    factor = min(1.0, max_norm / (norm + 1e-6))
    for a, b in zip(got, grads):
        want = b.cpu().double() * factor
        assert bool(((a.cpu().double() - want).abs() <= UNIT[b.dtype] * want.abs() + 2.0 ** -133).all())


LISTS = [[1], [7, 8, 9], [0, 5, 0], [8191, 8192, 8193], [100] * 95, [3] * 96, [33] * 97, [5] * 500, [1000003, 64, 262144], [40000000]]


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: "%dx%d" % (len(s), s[0]))
@pytest.mark.parametrize("max_norm", [0.25, 1e9])
def test_lists(ffk, sizes, max_norm):
    say("clip", len(sizes), sizes[:3], max_norm)
    grads = make(sizes)
    want = norm_of(grads)
    norm = ffk.global_grad_norm(grads)
    assert abs(float(norm) - want) <= NORM_TOL * want
    out, norm2 = ffk.clip_grad_norm(grads, max_norm, out=[torch.full_like(g, 3.0) for g in grads])
    assert float(norm2) == float(norm)
    check_clipped(out, grads, want, max_norm)
    before = [g.clone() for g in grads]
    same, norm3 = ffk.clip_grad_norm(grads, max_norm)
    assert same is grads and float(norm3) == float(norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))
    if max_norm > want:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_no_tensors(ffk):
    for grads in ([], [torch.empty((0,), device="cuda")]):
        assert float(ffk.global_grad_norm(grads)) == 0.0
        assert float(ffk.clip_grad_norm(grads, 1.0)[1]) == 0.0


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_sizes_whose_squares_leave_fp32(ffk, scale):
    grads = make([1000, 333, 4097], 2, scale)
    want = norm_of(grads)
    assert abs(float(ffk.global_grad_norm(grads)) - want) <= NORM_TOL * want
    out, _ = ffk.clip_grad_norm(grads, 0.5, out=[torch.empty_like(g) for g in grads])
    check_clipped(out, grads, want, 0.5)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_norms_that_are_no_number(ffk, value):
    grads = make([100, 50], 3)
    grads[0][17] = value
    out, norm = ffk.clip_grad_norm(grads, 1.0, out=[torch.empty_like(g) for g in grads])
    if math.isinf(value):  # factor 0
        assert math.isinf(float(norm))
        assert not out[1].any() and bool(torch.isnan(out[0][17])) and not out[0][:17].any()
    else:
        assert math.isnan(float(norm)) and bool(torch.isnan(out[0]).all()) and bool(torch.isnan(out[1]).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shift", [1, 2, 3, 4, 7])
def test_any_alignment(ffk, dtype, shift):
    """Views that begin and end anywhere; what lies around the clipped one is left as it was."""
    base = torch.randn((20000,)).to(dtype).cuda()
    out = torch.full((20020,), 9.0, dtype=dtype, device="cuda")
    grad, to = base[shift:shift + 17001], out[shift + 3:shift + 3 + 17001]
    _, norm = ffk.clip_grad_norm([grad], 1.0, out=[to])
    want = norm_of([grad])
    assert abs(float(norm) - want) <= NORM_TOL * want
    check_clipped([to], [grad], want, 1.0)
    assert bool((out[:shift + 3] == 9.0).all()) and bool((out[shift + 3 + 17001:] == 9.0).all())


def test_same_bits_twice_and_in_any_split(ffk):
    """The sum's order is fixed: one call after the other gives the same bits."""
    grads = make([300000, 77, 123457], 5)
    first = ffk.global_grad_norm(grads)
    assert all(torch.equal(first, ffk.global_grad_norm(grads)) for _ in range(3))


def test_replayed_graph_and_another_stream(ffk):
    grads = make([5000, 40000, 1], 6)
    out = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ffk.clip_grad_norm(grads, 1.0, out=out)
    torch.cuda.synchronize()
    check_clipped(out, grads, norm_of(grads), 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = ffk.clip_grad_norm(grads, 1.0, out=out)
    for n in range(3):
        for g in grads:
            g.mul_(1.5).add_(0.01 * n)
        graph.replay()
        torch.cuda.synchronize()
        want = norm_of(grads)
        assert abs(float(norm) - want) <= NORM_TOL * want
        check_clipped(out, grads, want, 1.0)


def test_a_step_clipped_before_its_update(ffk):
    """Clipped gradients through ffk_adam_update: the update's own fp32 operations on the scaled values."""
    weight, m, v = torch.randn((5000,)).cuda(), torch.zeros((5000,)).cuda(), torch.zeros((5000,)).cuda()
    other = weight.clone(), m.clone(), v.clone()
    grads = make([5000, 300], 7)
    want = [g.clone() for g in grads]
    factor = torch.tensor(min(1.0, 0.5 / (norm_of(grads) + 1e-6)), dtype=torch.float64).float().cuda()
    ffk.clip_grad_norm(grads, 0.5)
    ffk.adam_update(weight, grads[0], m, v, 1e-2)
    ffk.adam_update(other[0], want[0] * factor, other[1], other[2], 1e-2)
    torch.testing.assert_close(weight, other[0], rtol=1e-6, atol=1e-7)

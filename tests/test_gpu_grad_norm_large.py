"""Gradient lists of more than 128 MB, which the norm reads by loads that keep nothing in the caches: both types, views of any
alignment, odd remainders, and lists longer than a launch's table."""
import math
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
# as in test_gpu_grad_norm.py: the norm's one rounding; a clipped value's factor, product and, in bf16, store
NORM_TOL, UNIT = 2.0 ** -23, {BF: 2.0 ** -8 + 2.0 ** -22, F32: 2.0 ** -22}


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def norm_of(grads):
    return math.sqrt(sum(float(torch.dot(d, d)) for d in (g.double() for g in grads)))


def bases(n_bf, n_f32, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((n_bf,), generator=g, device="cuda").to(BF), torch.randn((n_f32,), generator=g, device="cuda") * 0.5)


LISTS = {
    # whole pieces (of 16384 bf16 or 8192 fp32 elements) at every shift of an element, and what is left over
    "bf16": lambda b, f: [b[1:40000000], b[40000003:40000003 + 16384 * 100], b[50000005:]],
    "fp32": lambda b, f: [f[1:20000000], f[20000003:20000003 + 8192 * 100], f[30000002:]],
    "mixed": lambda b, f: [b[7:30000000], f[3:17], f[101:20000102], b[40000001:40016386], f[30000001:]],
    "long": lambda b, f: [b[300001 * i + i % 8:300001 * (i + 1)] for i in range(200)] + [f[100003 * i + i % 4:100003 * (i + 1)] for i in range(300)],
}


@pytest.mark.parametrize("kind", sorted(LISTS))
@pytest.mark.parametrize("max_norm", [1.0, 1e9])
def test_large_lists(ffk, kind, max_norm):
    b, f = bases(90000001, 45000001, 3)
    grads = LISTS[kind](b, f)
    assert sum(g.numel() * g.element_size() for g in grads) > 128 << 20
    say("large list", kind, len(grads), max_norm)
    want = norm_of(grads)
    norm = ffk.global_grad_norm(grads)
    assert abs(float(norm) - want) <= NORM_TOL * want, (float(norm), want)
    guard = {BF: torch.full_like(b, 9.0), F32: torch.full_like(f, 9.0)}
    base = {BF: b, F32: f}
    outs = [guard[g.dtype][g.storage_offset():g.storage_offset() + g.numel()] for g in grads]
    _, norm2 = ffk.clip_grad_norm(grads, max_norm, out=outs)
    assert float(norm2) == float(norm)
    factor = min(1.0, max_norm / (want + 1e-6))
    for a, g in zip(outs, grads):
        exact = g.double() * factor
        assert bool(((a.double() - exact).abs() <= UNIT[g.dtype] * exact.abs() + 2.0 ** -133).all())
    for dtype in (BF, F32):  # what lies between the tensors is left as it was
        between = torch.ones(base[dtype].shape, dtype=torch.bool, device="cuda")
        for g in grads:
            if g.dtype == dtype:
                between[g.storage_offset():g.storage_offset() + g.numel()] = False
        assert bool((guard[dtype][between] == 9.0).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_one_norm_however_it_is_cut(ffk, dtype):
    """A tensor whole, and in parts of any size: the same norm, by either kind of load."""
    whole = bases(80000000, 40000000, 4)[dtype == F32]
    want = norm_of([whole])
    for n in (1, 3, 97, 250):
        ends = [whole.numel() * i // n for i in range(n + 1)]
        say("cut", dtype, n)
        got = float(ffk.global_grad_norm([whole[a:z] for a, z in zip(ends, ends[1:])]))
        assert abs(got - want) <= NORM_TOL * want, n
    part = whole[:20000001]
    assert abs(float(ffk.global_grad_norm([part])) - norm_of([part])) <= NORM_TOL * norm_of([part])

"""Sizes past what one launch takes (2^32 threads) are refused by masked attention, rotary positions and the gradient norm before
any launch, and the largest that fit are not (no device is touched: the addresses are made up)."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")
AT = [ctypes.c_void_p((i + 1) << 24) for i in range(16)]


def lists(dtypes, elems):
    n = len(dtypes)
    return (ctypes.c_int * n)(*dtypes), (ctypes.c_void_p * n)(*[(i + 1) << 44 for i in range(n)]), (ctypes.c_int64 * n)(*elems), n


def test_gradients(ffk):
    """A workgroup of 256 threads scales 16 KB: tensors below 2^24 of those, 256 GB."""
    lib = ffk.lib()
    for dtype, size in ((ffk.BF16, 2), (ffk.FLOAT, 4)):
        most = ((1 << 38) - (1 << 14)) // size
        for elems, rc in ((most, ffk.ERR_WORKSPACE), (most + 1, ffk.ERR_INVALID), (1 << 37, ffk.ERR_INVALID), (1 << 39, ffk.ERR_INVALID)):
            d, g, e, n = lists([dtype, dtype], [5, elems])
            # (what is not refused for its size stops at the scratch that is missing)
            assert lib.ffk_global_grad_norm(None, d, g, e, n, AT[0], None, 0) == rc, elems
            assert lib.ffk_clip_grad_norm(None, d, g, g, e, n, 1.0, AT[0], None, 0) == rc, elems


def test_scratch_of_the_norm_holds_every_launch(ffk):
    """1024 sums of 64 bits for each table of 96 tensors; a table is never cut short by the tensors' sizes: 96 of the largest
    are below 2^31 pieces of 32 KB."""
    size = ffk.lib().ffk_grad_norm_workspace_bytes
    for n in (1, 96, 97, 500, 9600, 9601):
        assert size(n) >= -(-n // 96) * 1024 * 8
    assert 96 * ((1 << 38) >> 15) < 1 << 31


def desc(ffk, B, H, KH, Sq, Skv, D, **more):
    d = ffk.MaskedAttentionDesc(B, H, KH, Sq, Skv, D, 0, Sq * H * D, H * D, Skv * KH * D, KH * D, Skv * KH * D, KH * D, Sq * H * D, H * D, 0, 0.125, 0.0, 0)
    for name, value in more.items():
        setattr(d, name, value)
    return d


ATTENTION = [  # dtype, (B, H, KH, Sq, Skv, D), whether forward and backward fit
    # 64 threads for 32 rows of one sequence and key head in the forward, 256 in the backward
    ("BF16", ((1 << 21) - 1, 8, 8, 1, 1, 64), True, True), ("BF16", (1 << 21, 8, 8, 1, 1, 64), True, False),
    ("BF16", ((1 << 23) - 1, 8, 8, 1, 1, 64), True, False), ("BF16", (1 << 23, 8, 8, 1, 1, 64), False, False),
    # 256 for them in the kernels of any head size
    ("BF16", ((1 << 21) - 1, 8, 8, 1, 1, 256), True, True), ("BF16", (1 << 21, 8, 8, 1, 1, 256), False, False),
    ("FLOAT", (1 << 21, 8, 8, 1, 1, 64), False, False),
    # 256 for 128 rows, and for 128 keys
    ("BF16", ((1 << 14) - 1, 8, 8, 16384, 64, 8), True, True), ("BF16", (1 << 14, 8, 8, 16384, 64, 8), False, False),
    ("BF16", ((1 << 14) - 1, 8, 8, 64, 16384, 8), True, True), ("BF16", (1 << 14, 8, 8, 64, 16384, 8), True, False),
]


@pytest.mark.parametrize("dtype,shape,forward,backward", ATTENTION)
def test_attention(ffk, dtype, shape, forward, backward):
    lib, d, dtype = ffk.lib(), desc(ffk, *shape), getattr(ffk, dtype)
    # (what is not refused for its size stops at a tensor that is missing)
    rc = lib.ffk_masked_attention_forward(None, dtype, ctypes.byref(d), None, AT[1], AT[2], None, None, AT[3], AT[4], None, 0)
    assert rc == ffk.ERR_INVALID and (b"NULL tensor" if forward else b"too many workgroups") in lib.ffk_last_error()
    rc = lib.ffk_masked_attention_backward(None, dtype, ctypes.byref(d), None, *AT[1:3], None, None, *AT[3:9], AT[9], 1 << 62)
    assert rc == ffk.ERR_INVALID and (b"NULL tensor" if backward else b"too many workgroups") in lib.ffk_last_error()
    assert (lib.ffk_masked_attention_backward_workspace_bytes(ctypes.byref(d), dtype) > 0) == backward


@pytest.mark.parametrize("batch,seq,heads,dim", [(1 << 14, 1 << 10, 16, 1024), (1 << 12, 1 << 15, 1, 4096), (1 << 25, 8, 40, 128)])
def test_rotary(ffk, batch, seq, heads, dim):
    """A workgroup of 256 threads takes one token of many heads, or of many pairs, or a few of others."""
    n = heads * dim
    d = ffk.RotaryDesc(batch, seq, heads, 0, dim, seq * n, n, 0, 0, seq * n, n, 0, 0, 1, (ffk.c_i64 * 4)(dim // 2), 0)
    for entry in (ffk.lib().ffk_rotary_forward, ffk.lib().ffk_rotary_backward):
        rc = entry(None, ffk.BF16, ctypes.byref(d), AT[0], None, AT[4], AT[5], AT[2], None)
        assert rc == ffk.ERR_INVALID and b"too many workgroups" in ffk.lib().ffk_last_error()


@pytest.mark.parametrize("scale,cap", [(1e-39, 0.0), (1e-38, 0.0), (1e-36, 0.0), (1e-38, 1e-36)])
def test_scales_that_leave_no_room_for_slopes(ffk, scale, cap):
    """Biases are added in units of the raw product (or of the cap's tanh): 0.5 * 7 over a scale of 1e-38 is no number there."""
    lib, d = ffk.lib(), desc(ffk, 2, 4, 2, 16, 16, 64, scale=scale, score_cap=cap)
    for dtype in (ffk.BF16, ffk.FLOAT):
        rc = lib.ffk_masked_attention_forward(None, dtype, ctypes.byref(d), *AT[:3], None, AT[10], AT[3], AT[4], None, 0)
        assert rc == ffk.ERR_INVALID and b"slopes" in lib.ffk_last_error()
        need = lib.ffk_masked_attention_backward_workspace_bytes(ctypes.byref(d), dtype)
        rc = lib.ffk_masked_attention_backward(None, dtype, ctypes.byref(d), *AT[:3], None, AT[10], *AT[3:9], AT[9], need)
        assert rc == ffk.ERR_INVALID and b"slopes" in lib.ffk_last_error()

"""What masked attention, rotary positions and the gradient norm refuse, before any launch (no device is touched: the
addresses are made up)."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")
AT = [ctypes.c_void_p((i + 1) << 24) for i in range(16)]


def desc(ffk, **more):
    B, H, KH, S, D = 2, 4, 2, 16, 64
    d = ffk.MaskedAttentionDesc(B, H, KH, S, S, D, 0, S * H * D, H * D, S * KH * D, KH * D, S * KH * D, KH * D, S * H * D, H * D, 0, 0.125, 0.0, 0)
    for name, value in more.items():
        setattr(d, name, value)
    return d


def forward(ffk, d, dtype=None, q=AT[0], ranges=None):
    rc = ffk.lib().ffk_masked_attention_forward(None, ffk.BF16 if dtype is None else dtype, None if d is None else ctypes.byref(d), q, AT[1], AT[2],
                                                ranges, None, AT[3], AT[4], None, 0)
    return rc, ffk.lib().ffk_last_error().decode()


BAD = [dict(batch=0), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(seq_q=0), dict(seq_kv=0), dict(seq_kv=-1), dict(head_dim=60),
       dict(head_dim=264), dict(head_dim=0), dict(v_head_dim=12), dict(v_head_dim=512), dict(v_head_dim=-8), dict(q_seq_stride=255),
       dict(k_seq_stride=129), dict(q_seq_stride=128), dict(o_seq_stride=248), dict(v_batch_stride=8), dict(q_batch_stride=-1024),
       dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(score_cap=-1.0), dict(score_cap=float("nan")),
       dict(score_cap=float("inf")), dict(score_cap=1e-40), dict(query_offset=-1), dict(query_offset=1 << 30), dict(seq_kv=1 << 30),
       dict(batch=1 << 29)]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: "%s=%s" % next(iter(b.items())))
def test_descriptors(ffk, bad):
    d = desc(ffk, **bad)
    rc, text = forward(ffk, d)
    assert rc == ffk.ERR_INVALID and text.startswith("masked_attention_forward: "), (rc, text)
    lib = ffk.lib()
    assert lib.ffk_masked_attention_forward_workspace_bytes(ctypes.byref(d), ffk.BF16) == 0
    assert lib.ffk_masked_attention_backward_workspace_bytes(ctypes.byref(d), ffk.BF16) == 0
    rc = lib.ffk_masked_attention_backward(None, ffk.BF16, ctypes.byref(d), *AT[:3], None, None, *AT[3:9], AT[9], 1 << 30)
    assert rc == ffk.ERR_INVALID


def test_types_and_tensors(ffk):
    for dtype in (ffk.HALF, ffk.DOUBLE, ffk.INT32, 99, -1):
        assert forward(ffk, desc(ffk), dtype)[0] == ffk.ERR_INVALID
    assert forward(ffk, None)[0] == ffk.ERR_INVALID
    assert "NULL tensor" in forward(ffk, desc(ffk), q=None)[1]
    assert "16-byte aligned" in forward(ffk, desc(ffk), q=ctypes.c_void_p((1 << 24) + 8))[1]
    assert "8-byte aligned" in forward(ffk, desc(ffk), ranges=ctypes.c_void_p((1 << 24) + 4))[1]
    # bf16 rows are whole 16 bytes at multiples of 8; fp32 takes multiples of 4
    assert forward(ffk, desc(ffk, head_dim=60, q_seq_stride=260), ffk.BF16)[0] == ffk.ERR_INVALID


def test_backward_needs_its_workspace(ffk):
    lib, d = ffk.lib(), desc(ffk)
    need = lib.ffk_masked_attention_backward_workspace_bytes(ctypes.byref(d), ffk.BF16)
    assert need >= 2 * 4 * 16 * 4
    for workspace, room in ((AT[9], need - 1), (None, need), (AT[9], 0), (ctypes.c_void_p((1 << 24) + 4), need)):
        rc = lib.ffk_masked_attention_backward(None, ffk.BF16, ctypes.byref(d), *AT[:3], None, None, *AT[3:9], workspace, room)
        assert rc == ffk.ERR_WORKSPACE and b"workspace" in lib.ffk_last_error()
    for n in range(9):  # any tensor missing
        t = AT[:3] + AT[3:9]
        t[n] = None
        rc = lib.ffk_masked_attention_backward(None, ffk.BF16, ctypes.byref(d), *t[:3], None, None, *t[3:], AT[9], need)
        assert rc == ffk.ERR_INVALID, n


def test_forward_workspace_is_for_few_rows_over_long_keys(ffk):
    lib = ffk.lib()
    assert lib.ffk_masked_attention_forward_workspace_bytes(ctypes.byref(desc(ffk)), ffk.BF16) == 0
    long = desc(ffk, seq_q=1, seq_kv=8192, k_batch_stride=8192 * 128, v_batch_stride=8192 * 128)
    assert lib.ffk_masked_attention_forward_workspace_bytes(ctypes.byref(long), ffk.BF16) > 0


def test_key_ranges(ffk):
    call = ffk.lib().ffk_attention_key_ranges
    for bad in ((0, 4, 4, 0, 0, None, 0, None, AT[0]), (1, 0, 4, 0, 0, None, 0, None, AT[0]), (1, 4, 0, 0, 0, None, 0, None, AT[0]),
                (1, 4, 4, -1, 0, None, 0, None, AT[0]), (1, 4, 4, 0, 0, None, 0, None, None), (1, 4, 4, 0, 0, None, 2, None, AT[0]),
                (1, 4, 4, 0, 0, AT[1], 0, None, AT[0]), (1, 4, 4, 0, 0, AT[1], 1, AT[2], AT[0]), (1 << 16, 1 << 15, 4, 0, 0, None, 1, None, AT[0]),
                (1, 4, 4, 0, 1, None, 1, None, ctypes.c_void_p((1 << 24) + 4))):
        assert call(None, *bad) == ffk.ERR_INVALID, bad
        assert ffk.lib().ffk_last_error().startswith(b"attention_key_ranges: ")


def rotary(ffk, q=AT[0], k=AT[1], q_out=AT[2], k_out=AT[3], positions=AT[4], frequencies=AT[5], dtype=None, sections=(16, 16), **more):
    B, S, H, KH, D = 2, 8, 4, 2, 64
    d = ffk.RotaryDesc(B, S, H, KH, D, S * H * D, H * D, S * KH * D, KH * D, S * H * D, H * D, S * KH * D, KH * D, len(sections),
                       (ffk.c_i64 * 4)(*sections[:4]), 0)
    for name, value in more.items():
        setattr(d, name, value)
    lib = ffk.lib()
    got = {entry(None, ffk.BF16 if dtype is None else dtype, ctypes.byref(d), q, k, positions, frequencies, q_out, k_out)
           for entry in (lib.ffk_rotary_forward, lib.ffk_rotary_backward)}
    assert len(got) == 1
    return got.pop()


def test_rotary(ffk):
    for bad in (dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(positions=None), dict(frequencies=None), dict(dtype=ffk.HALF),
                dict(sections=(16, 17)), dict(sections=(0, 0)), dict(sections=(-1, 8)), dict(num_axes=0), dict(num_axes=5), dict(batch=0), dict(seq=0),
                dict(q_heads=0), dict(k_heads=-1), dict(head_dim=0), dict(q_seq_stride=255), dict(k_out_seq_stride=127), dict(q_batch_stride=8),
                dict(q_out=AT[0], q_out_seq_stride=512), dict(k_out=AT[1], k_out_batch_stride=1 << 20), dict(q=ctypes.c_void_p((1 << 24) + 1)),
                dict(batch=1 << 20, seq=1 << 20), dict(sections=(2049,), head_dim=5000, q_seq_stride=1 << 20, k_seq_stride=1 << 20,
                                                       q_out_seq_stride=1 << 20, k_out_seq_stride=1 << 20, q_batch_stride=1 << 25)):
        assert rotary(ffk, **bad) == ffk.ERR_INVALID, bad
        assert b"rotary_backward: " in ffk.lib().ffk_last_error()
    lib = ffk.lib()
    assert lib.ffk_rotary_forward(None, ffk.BF16, None, *AT[:6]) == ffk.ERR_INVALID


def lists(dtypes, elems, at=None):
    n = len(dtypes)
    at = at or [(i + 1) << 24 for i in range(n)]
    return (ctypes.c_int * n)(*dtypes), (ctypes.c_void_p * n)(*at), (ctypes.c_int64 * n)(*elems), n


def test_grad_norm(ffk):
    lib = ffk.lib()
    room = lib.ffk_grad_norm_workspace_bytes(2)
    good = lists([ffk.FLOAT, ffk.BF16], [5, 6])
    for d, g, e, n in (lists([ffk.FLOAT, ffk.HALF], [5, 6]), lists([ffk.FLOAT, ffk.BF16], [5, -1]), lists([ffk.FLOAT, ffk.BF16], [5, 6], [1 << 24, None]),
                       lists([ffk.FLOAT, ffk.BF16], [5, 6], [(1 << 24) + 2, 1 << 25]), (good[0], good[1], good[2], -1), (None, good[1], good[2], 2),
                       (good[0], None, good[2], 2), (good[0], good[1], None, 2)):
        assert lib.ffk_global_grad_norm(None, d, g, e, n, AT[0], AT[1], room) == ffk.ERR_INVALID
        assert lib.ffk_clip_grad_norm(None, d, g, g, e, n, 1.0, AT[0], AT[1], room) == ffk.ERR_INVALID
    d, g, e, n = good
    assert lib.ffk_global_grad_norm(None, d, g, e, n, None, AT[1], room) == ffk.ERR_INVALID
    assert lib.ffk_clip_grad_norm(None, d, g, None, e, n, 1.0, AT[0], AT[1], room) == ffk.ERR_INVALID
    for bad in (-1.0, float("nan")):
        assert lib.ffk_clip_grad_norm(None, d, g, g, e, n, bad, AT[0], AT[1], room) == ffk.ERR_INVALID
    for workspace, size in ((AT[1], room - 1), (None, room), (ctypes.c_void_p((1 << 24) + 4), room)):
        assert lib.ffk_global_grad_norm(None, d, g, e, n, AT[0], workspace, size) == ffk.ERR_WORKSPACE
        assert lib.ffk_clip_grad_norm(None, d, g, g, e, n, 1.0, AT[0], workspace, size) == ffk.ERR_WORKSPACE


def test_tables_of_many_tensors_ask_for_more_room(ffk):
    size = ffk.lib().ffk_grad_norm_workspace_bytes
    assert size(0) == size(96) < size(97) <= size(192) < size(193)


def test_outputs_that_are_inputs_or_each_other(ffk):
    lib, d = ffk.lib(), desc(ffk)
    for n in range(3):  # q, k, v
        rc = lib.ffk_masked_attention_forward(None, ffk.BF16, ctypes.byref(d), *AT[:3], None, None, AT[n], AT[4], None, 0)
        assert rc == ffk.ERR_INVALID and b"is an input" in lib.ffk_last_error()
    need = lib.ffk_masked_attention_backward_workspace_bytes(ctypes.byref(d), ffk.BF16)
    inputs = AT[:5]  # q, k, v, o, d_o
    for grad in range(3):
        for other in inputs:
            grads = AT[6:9]
            grads[grad] = other
            rc = lib.ffk_masked_attention_backward(None, ffk.BF16, ctypes.byref(d), *inputs[:3], None, None, *inputs[3:], AT[5], *grads, AT[9], need)
            assert rc == ffk.ERR_INVALID and b"is an input" in lib.ffk_last_error()
        grads = AT[6:9]
        grads[grad] = grads[grad - 1]
        rc = lib.ffk_masked_attention_backward(None, ffk.BF16, ctypes.byref(d), *inputs[:3], None, None, *inputs[3:], AT[5], *grads, AT[9], need)
        assert rc == ffk.ERR_INVALID and b"are one" in lib.ffk_last_error()
    for more in (dict(q_out=AT[3]), dict(q_out=AT[1]), dict(k_out=AT[0])):
        assert rotary(ffk, **more) == ffk.ERR_INVALID and b"the other tensor" in lib.ffk_last_error()


def test_clipping_of_tensors_that_overlap(ffk):
    lib, room = ffk.lib(), ffk.lib().ffk_grad_norm_workspace_bytes(3)
    a, b, c = 1 << 24, 1 << 25, 1 << 26
    F, elems = [ffk.FLOAT] * 3, [100, 200, 50]
    for ins, outs in (([a, b, a], [a, b, a]),              # the same tensor twice, in place
                      ([a, b, c], [a, b, b + 796]),        # an output in another's last element
                      ([a, b, c], [b, a, c]),              # two tensors exchanged
                      ([a, a + 4, c], [a, 1 << 27, 1 << 28]),  # in place, over the input of another
                      ([a, b, c], [a + 4, b, c])):         # moved along by one element
        d, g, e, n = lists(F, elems, ins)
        out = lists(F, elems, outs)[1]
        assert lib.ffk_clip_grad_norm(None, d, g, out, e, n, 1.0, AT[0], AT[1], room) == ffk.ERR_INVALID, (ins, outs)
        assert b"overlap" in lib.ffk_last_error()

"""Refusals of the serving operators (8-bit product, residual norm, cross
attention): every bad argument is an error with its reason before any CUDA
call, so these run without a GPU.  The pointers are numbers that nothing may
read."""
import ctypes as C

import numpy as np
import pytest

from conftest import load_pkg

nb = load_pkg()
P = 1 << 20  # stands for an aligned device pointer


def refused(match, call, *a, **k):
    with pytest.raises(nb.NeedleError, match=match):
        call(*a, **k)


def test_row_bytes():
    assert [nb.int8_row_bytes(k) for k in (1, 15, 16, 17, 512, 1000)] == [16, 16, 16, 32, 512, 1008]


@pytest.mark.parametrize("bad", [dict(x=None), dict(M=0), dict(K=0), dict(dtype=nb.I8), dict(dtype=7), dict(ldx=63), dict(q=P + 8),
                                 dict(x=P + 2), dict(s=None), dict(s=P + 2)])
def test_quantize_tokens_refuses(bad):
    a = dict(x=P, M=4, K=64, dtype=nb.F32, ldx=64, q=P, s=P, **{})
    a.update(bad)
    refused("invalid quantize", nb.int8_quantize_tokens, a["x"], a["M"], a["K"], a["q"], a["s"], a["dtype"], a["ldx"])


@pytest.mark.parametrize("bad", [dict(w=None), dict(K=0), dict(N=0), dict(dtype=nb.I8), dict(d=P + 4), dict(s=None)])
def test_quantize_weight_refuses(bad):
    a = dict(w=P, K=64, N=8, dtype=nb.F16, d=P, s=P)
    a.update(bad)
    refused("invalid quantize", nb.int8_quantize_weight, a["w"], a["K"], a["N"], a["d"], a["s"], a["dtype"])


@pytest.mark.parametrize("bad,match", [(dict(w=None), "invalid plan"), (dict(w=P + 1), "invalid plan"), (dict(N=0), "invalid plan"),
                                       (dict(m=0), "invalid plan"), (dict(K=131072), "overflow")])
def test_int8_plan_refuses(bad, match):
    a = dict(w=P, s=P, K=64, N=8, m=4)
    a.update(bad)
    refused(match, nb.Int8Plan, a["w"], a["s"], a["K"], a["N"], a["m"])


def test_null_plans():
    L = nb.lib()
    assert L.needle_int8_plan_matmul(None, P, 0, 1, 64, None, P, 0, 64, None) == -1
    assert L.needle_int8_plan_matmul_quantized(None, P, P, 1, None, P, 0, 64, None) == -1
    assert L.needle_int8_plan_status(None) == -1 and nb.last_error() == "null plan"
    assert L.needle_cross_attn_plan_run(None, P, 64, 64, P, 64, 64, P, 64, 64, None, 1.0, P, 64, 64, None, None) == -1
    assert L.needle_cross_attn_plan_status(None) == -1 and nb.last_error() == "null plan"
    L.needle_int8_plan_free(None)
    L.needle_cross_attn_plan_free(None)


NORM = dict(x_ptr=P, x_dtype=nb.F32, y_ptr=P, y_dtype=nb.BF16, M=4, d=64, pre_scale_ptr=P, r_ptr=P, h_ptr=P, h_dtype=nb.BF16)


@pytest.mark.parametrize("bad,match", [
    (dict(x_ptr=None), "invalid residual"), (dict(M=0), "invalid residual"), (dict(d=0), "invalid residual"),
    (dict(x_dtype=9), "invalid residual"), (dict(ldx=63), "invalid residual"), (dict(x_ptr=P + 2), "invalid residual"),
    (dict(d=32769), "above 32768"),
    (dict(x_dtype=nb.F16), "f32 or of y's type"),
    (dict(r_ptr=None), "exactly when"), (dict(y_ptr=None), "exactly when"),
    (dict(y_ptr=None, r_ptr=None, post_scale_ptr=P), "without y"), (dict(y_ptr=None, r_ptr=None, gate_ptr=P, gate_flags=1), "without y"),
    (dict(ldy=63), "invalid strides"), (dict(ldr=8), "invalid strides"),
    (dict(gate_ptr=P), "disagree"), (dict(gate_flags=1), "disagree"), (dict(gate_flags=8), "disagree"),
    (dict(gate_ptr=P, gate_flags=4), "invalid residual"), (dict(gate_ptr=P, gate_flags=3, ldg=9), "gate stride"),
    (dict(pre_scale_ptr=None), "go together"), (dict(h_ptr=None), "go together"),
    (dict(h_dtype=nb.F16), "of y's type"), (dict(ldh=63), "of y's type"), (dict(h_ptr=P + 1), "of y's type"),
    (dict(h_dtype=nb.I8, h_ptr=P + 8, h_scales_ptr=P), "16-byte"), (dict(h_dtype=nb.I8, ldh=72, h_scales_ptr=P), "16-byte"),
    (dict(h_dtype=nb.I8), "h_scales"), (dict(h_scales_ptr=P), "h_scales"),
    (dict(r_ptr=None, h_ptr=None, pre_scale_ptr=None, y_ptr=None), "invalid residual"),
])
def test_residual_norm_refuses(bad, match):
    a = dict(NORM)
    a.update(bad)
    refused(match, nb.residual_norm, **a)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=nb.F32), "f16 or bf16"), (dict(dtype=nb.I8), "f16 or bf16"), (dict(D=0), "head_dim"), (dict(D=60), "head_dim"),
    (dict(D=136), "head_dim"), (dict(H=6, KVH=4), "num_heads"), (dict(H=0), "num_heads"), (dict(KVH=0), "num_heads"),
    (dict(qs=[0, 3]), "share a query row"), (dict(ks=[0, 1 << 31]), "past 2"), (dict(ql=[4, 1 << 40]), "past 2"),
    (dict(qs=[], ql=[], ks=[], kl=[]), "invalid cross"),
])
def test_cross_attn_plan_refuses(bad, match):
    a = dict(qs=[0, 4], ql=[4, 4], ks=[0, 0], kl=[9, 9], H=8, KVH=4, D=64, dtype=nb.BF16)
    a.update(bad)
    refused(match, nb.CrossAttnPlan, a["qs"], a["ql"], a["ks"], a["kl"], a["H"], a["KVH"], a["D"], a["dtype"])


def test_cross_attn_plan_lists_of_one_length():
    with pytest.raises(ValueError):
        nb.CrossAttnPlan([0, 4], [4], [0, 0], [9, 9], 8, 4, 64)
    L = nb.lib()
    a = np.zeros(1, np.uint64)
    p = a.ctypes.data_as(C.c_void_p)
    assert not L.needle_cross_attn_plan_create(None, p, p, p, 1, 8, 4, 64, nb.BF16, None)


@pytest.mark.parametrize("ql,n,H,KVH", [([(1 << 31) - 4096], 1, 64, 64), ([64] * 20000, 20000, 4096, 4096)])
def test_cross_attn_plan_refuses_more_rows_than_it_can_list(ql, n, H, KVH):
    """Before the list is made: it would not fit the host's memory."""
    at = list(np.cumsum([0] + ql[:-1]))
    refused("too many rows", nb.CrossAttnPlan, at, ql, [0] * n, [9] * n, H, KVH, 64, nb.BF16)


def test_rows_stop_at_whole_tiles_below_31_bits():
    """Counts of rows are rounded up to tiles of 256 in 32 bits."""
    refused("invalid plan", nb.Int8Plan, P, P, 64, 8, (1 << 31) - 255)
    refused("invalid plan", nb.Int8Plan, P, P, 64, (1 << 31) - 255, 8)
    refused("invalid quantize", nb.int8_quantize_tokens, P, (1 << 31) - 255, 64, P, P, nb.F32)
    refused("past 2", nb.CrossAttnPlan, [0], [4], [0], [(1 << 31) - 255], 8, 4, 64, nb.BF16)

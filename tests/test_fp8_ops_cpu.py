"""The 8-bit operators' checks of arguments, their C entry points' refusals and
their fake implementations, without a GPU."""

import ctypes

import pytest
import torch

import fused_decode_b200 as fd
from fused_decode_b200 import _capi

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


X, W, W32 = z(2, 16), z(4, 16), z(16, dtype=F32)
X8, W8, XS, WS = z(2, 16, dtype=E4M3), z(4, 16, dtype=E4M3), z(2, dtype=F32), z(4, dtype=F32)
MLP = (z(2, 16), W32, z(48, 16, dtype=E4M3), z(48, dtype=F32), z(16, 24, dtype=E4M3), z(16, dtype=F32))


def _mlp(**changes):
    names = ("hidden", "norm_weight", "w_gate_up", "gate_up_scale", "w_down", "down_scale")
    return lambda: fd.post_attn_mlp_fp8(**{**dict(zip(names, MLP)), **changes})


REFUSALS = [
    (lambda: fd.quantize_fp8(X), ValueError, "x must be a CUDA tensor"),
    (lambda: fd.quantize_fp8([1.0]), TypeError, "x must be a tensor"),
    (lambda: fd.quantize_fp8(X.float()), TypeError, "float16 or bfloat16"),
    (lambda: fd.quantize_fp8(z(())), ValueError, "last dimension"),
    (lambda: fd.quantize_fp8(X, out=X), TypeError, "out must be float8_e4m3fn"),
    (lambda: fd.quantize_fp8(X, out=X8[:1]), ValueError, "out shape"),
    (lambda: fd.quantize_fp8(X, scale_out=z(2)), TypeError, "scale_out must be float32"),
    (lambda: fd.quantize_fp8(X, scale_out=z(2, 1, dtype=F32)), ValueError, "scale_out shape"),
    (lambda: fd.quantize_fp8(X, scale_out=z(4, dtype=F32)[::2]), ValueError, "scale_out must be contiguous"),
    (lambda: fd.rms_norm_fp8(X, W32), ValueError, "x must be a CUDA tensor"),
    (lambda: fd.rms_norm_fp8(X, W32[:8]), ValueError, "weight must have shape"),
    (lambda: fd.rms_norm_fp8(X, W32.double()), TypeError, "weight must be"),
    (lambda: fd.rms_norm_fp8(X, W32, -1.0), ValueError, "eps"),
    (lambda: fd.rms_norm_fp8(X, W32, float("nan")), ValueError, "eps"),
    (lambda: fd.add_rms_norm_fp8(X, X[:1], W32), ValueError, "residual shape"),
    (lambda: fd.add_rms_norm_fp8(X, X.half(), W32), TypeError, "residual dtype"),
    (lambda: fd.add_rms_norm_fp8(X, X, W32, residual_out=X.half()), TypeError, "residual_out dtype"),
    (lambda: fd.add_rms_norm_fp8(X, X, W32), ValueError, "x must be a CUDA tensor"),
    (lambda: fd.swiglu_fp8(X, X[:1]), ValueError, "up shape"),
    (lambda: fd.swiglu_fp8(X, X.half()), TypeError, "up dtype"),
    (lambda: fd.swiglu_fp8(X, X), ValueError, "gate must be a CUDA tensor"),
    (lambda: fd.linear_act(X, W), ValueError, "x must be a CUDA tensor"),
    (lambda: fd.linear_act(X8, W8), TypeError, "x must be float16 or bfloat16"),
    (lambda: fd.linear_act(X, W.half()), TypeError, "weight must be"),
    (lambda: fd.linear_act(X, W[0]), ValueError, r"weight must have shape \[N, K\]"),
    (lambda: fd.linear_act(X, W[:, :8]), ValueError, "x last dim 16 != weight K 8"),
    (lambda: fd.linear_act(X, W, activation="tanh"), ValueError, "activation must be"),
    (lambda: fd.linear_act(X, W, z(4, dtype=F16)), TypeError, "bias must be"),
    (lambda: fd.linear_act(X, W, z(3)), ValueError, "bias must have shape"),
    (lambda: fd.linear_act(X, W, row_add=z(3, 4)), ValueError, "not broadcastable"),
    (lambda: fd.linear_act(X, W, row_add=z(1, 2, 4)), ValueError, "not broadcastable"),
    (lambda: fd.linear_act(X, W, row_add=z(2, 4, dtype=torch.int32)), TypeError, "row_add must be"),
    (lambda: fd.linear_act(X, W, out=z(2, 5)), ValueError, "out shape"),
    (lambda: fd.linear_act(X, W, out=z(2, 4, dtype=F32)), TypeError, "out must be"),
    (lambda: fd.linear_act(X, W, out=z(4, 2).t()), ValueError, "out must be contiguous"),
    (lambda: fd.linear_fp8(X8, XS, W8, WS), ValueError, "x must be a CUDA tensor"),
    (lambda: fd.linear_fp8(X, XS, W8, WS), TypeError, "x must be float8_e4m3fn"),
    (lambda: fd.linear_fp8(X8, XS, W, WS), TypeError, "weight must be float8_e4m3fn"),
    (lambda: fd.linear_fp8(X8, XS[:1], W8, WS), ValueError, "x_scale shape"),
    (lambda: fd.linear_fp8(X8, XS, W8, WS[:3]), ValueError, "weight_scale shape"),
    (lambda: fd.linear_fp8(X8, XS.half(), W8, WS), TypeError, "x_scale must be float32"),
    (lambda: fd.linear_fp8(X8, XS, W8, WS, out_dtype=F32), TypeError, "out_dtype"),
    (lambda: fd.linear_fp8(X8, XS, W8, WS, z(4), out_dtype=F16), TypeError, "bias must be"),
    (_mlp(), ValueError, "hidden must be a CUDA tensor"),
    (_mlp(w_down=z(16, 23, dtype=E4M3)), ValueError, r"expected w_gate_up \[2I, H\]"),
    (_mlp(w_gate_up=z(48, 16)), TypeError, "w_gate_up must be float8_e4m3fn"),
    (_mlp(gate_up_scale=z(24, dtype=F32)), ValueError, "gate_up_scale must have shape"),
    (_mlp(down_scale=z(16)), TypeError, "down_scale must be float32"),
    (_mlp(norm_weight=z(8)), ValueError, "norm_weight must have shape"),
    (_mlp(eps=-1.0), ValueError, "eps"),
]


@pytest.mark.parametrize("index", range(len(REFUSALS)))
def test_refusals(index):
    call, error, message = REFUSALS[index]
    with pytest.raises(error, match=message):
        call()


def _grid(t, dtype, n=16, rows=2):
    return _capi.FdRows(t.data_ptr(), dtype, 0, 1, 1, rows, 0, 0, n, 1, n)


def test_c_entries_refuse_before_any_launch():
    """Host buffers stand in for device ones: every call is refused, or is empty, before a launch."""
    lib = _capi.load()
    x, q, s = _grid(X, _capi.FD_BF16), _grid(X8, _capi.FD_E4M3), XS.data_ptr()
    bad = 1  # FD_ERR_ARG
    assert lib.fd_quantize_fp8_out(None, q, s, None) == bad
    assert lib.fd_quantize_fp8_out(x, q, None, None) == bad
    assert lib.fd_quantize_fp8_out(x, x, s, None) == bad            # output not e4m3
    assert lib.fd_quantize_fp8_out(q, q, s, None) == bad            # input not 16-bit
    assert lib.fd_quantize_fp8_out(x, _grid(X8, _capi.FD_E4M3, n=8), s, None) == bad
    assert lib.fd_quantize_fp8_out(_grid(X, 1, rows=0), _grid(X8, 3, rows=0), s, None) == 0
    assert lib.fd_swiglu_fp8_out(x, _grid(X, _capi.FD_F16), q, s, None) == bad
    assert lib.fd_rms_fp8_out(x, x, W32.data_ptr(), 2, 1, q, s, None, 1e-6, None) == bad  # residual without residual_out
    assert lib.fd_rms_fp8_out(x, None, None, 2, 1, q, s, None, 1e-6, None) == bad
    assert lib.fd_rms_fp8_out(x, None, W32.data_ptr(), 3, 1, q, s, None, 1e-6, None) == bad
    # the first output dtype refused here was new: 3 is no weight type, nor an activation one
    assert lib.fd_rms_out(q, None, W32.data_ptr(), 2, 1, q, None, 1e-6, None) == bad

    def linear(x=X.data_ptr(), y=W.data_ptr(), dtype=1, act=0, m=2, n=4, k=16, bias_dtype=1):
        return lib.fd_linear_act_out(x, 16, 1, W.data_ptr(), 16, 1, None, bias_dtype, 0, None, 0, 0, 0, y, 4, 1, dtype,
                                     act, m, n, k, None)

    assert linear(x=None) == bad and linear(y=None) == bad
    assert linear(dtype=2) == bad and linear(dtype=3) == bad
    assert linear(act=5) == bad and linear(act=-1) == bad
    assert linear(m=-1) == bad and linear(k=-1) == bad and linear(bias_dtype=3) == bad
    assert linear(m=0) == 0 and linear(n=0) == 0

    def linear8(xs=XS.data_ptr(), ws=WS.data_ptr(), dtype=1):
        return lib.fd_linear_fp8_out(X8.data_ptr(), 16, 1, xs, W8.data_ptr(), 16, 1, ws, None, 0, 0, None, 0, 0, 0,
                                     W.data_ptr(), 4, 1, dtype, 0, 2, 4, 16, None)

    assert linear8(xs=None) == bad and linear8(ws=None) == bad and linear8(dtype=3) == bad

    need = lib.fd_post_attn_mlp_fp8_workspace_bytes(2, 16, 24)
    assert need >= 2 * 16 + 8 + 2 * 48 * 2 + 2 * 24 + 8
    assert lib.fd_post_attn_mlp_fp8_workspace_bytes(-1, 16, 24) == 0
    ws = (ctypes.c_uint8 * (need + 32))()
    base = (ctypes.addressof(ws) + 15) & ~15

    def mlp(p=base, nbytes=need, hidden=MLP[0].data_ptr(), dtype=1, i=24):
        return lib.fd_post_attn_mlp_fp8_out(hidden, 16, W32.data_ptr(), 2, 1, MLP[2].data_ptr(), 16, MLP[3].data_ptr(),
                                            MLP[4].data_ptr(), 24, MLP[5].data_ptr(), X.data_ptr(), dtype, 2, 16, i,
                                            1e-6, p, nbytes, None)

    assert mlp(p=None) == 3 and mlp(nbytes=need - 1) == 3 and mlp(p=base + 1) == 3
    assert mlp(hidden=None) == bad and mlp(dtype=2) == bad and mlp(i=0) == bad


def test_custom_ops_fake_outputs():
    """Every operator resolves under torch.ops and its fake implementation gives the real one's shapes and types."""
    ops = torch.ops.fused_decode_b200

    def m(*shape, dtype=BF):
        return torch.empty(*shape, device="meta", dtype=dtype)

    x = m(2, 3, 64, dtype=F16)
    for out in (ops.quantize_fp8(x), ops.rms_norm_fp8(x, m(64)), ops.swiglu_fp8(x, x),
                ops.add_rms_norm_fp8(x, x, m(64))[:2]):
        assert (out[0].shape, out[0].dtype) == (x.shape, E4M3)
        assert (out[1].shape, out[1].dtype) == ((2, 3), F32)
    res = ops.add_rms_norm_fp8(x, x, m(64))[2]
    assert (res.shape, res.dtype) == (x.shape, F16)
    y = ops.linear_act(x, m(48, 64, dtype=F16), None, "silu", x)
    assert (y.shape, y.dtype) == ((2, 3, 48), F16)
    y = ops.linear_fp8(m(5, 64, dtype=E4M3), m(5, dtype=F32), m(48, 64, dtype=E4M3), m(48, dtype=F32), out_dtype=F16)
    assert (y.shape, y.dtype) == ((5, 48), F16)
    h = ops.post_attn_mlp_fp8(m(4, 64), m(64), m(96, 64, dtype=E4M3), m(96, dtype=F32), m(64, 48, dtype=E4M3),
                              m(64, dtype=F32))
    assert (h.shape, h.dtype) == ((4, 64), BF)


def test_compiled_dispatch_declines_cpu_tensors():
    fp = _capi.fast()
    assert fp.quantize_fp8(X, None, None) is None
    assert fp.rms_norm_fp8(X, W32, 1e-6, None, None) is None
    assert fp.add_rms_norm_fp8(X, X, W32, 1e-6, None, None, None) is None
    assert fp.swiglu_fp8(X, X, None, None) is None
    assert fp.linear_act(X, W, None, None, None, None) is None
    assert fp.linear_fp8(X8, XS, W8, WS, None, None, None, None, True) is None
    assert fp.post_attn_mlp_fp8(*MLP, 1e-6) is None
    assert fp.linear_act("x", None, None, "tanh", None, None) is None

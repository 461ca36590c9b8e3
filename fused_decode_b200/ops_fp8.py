"""Public operators of the 8-bit path, and the 16-bit product with an epilogue.

They stand beside the operators of ``ops`` (the reference has no 8-bit ones):
rows quantised to e4m3 with one fp32 scale each -- on their own
(``quantize_fp8``), behind the RMS norm (``rms_norm_fp8``,
``add_rms_norm_fp8``) or behind SwiGLU (``swiglu_fp8``) -- and the products
that read them (``linear_fp8``), with ``linear_act`` as the same product of
16-bit operands.  ``post_attn_mlp_fp8`` is ``post_attn_mlp`` built from them.

The 8-bit form of an fp32 row ``y``::

    a = max(max|y|, 2**-64);  scale = a / 448;  values = e4m3(y * (448 / a))

to nearest even, saturating; a NaN in the row makes its scale NaN.  Inference
only, any number of rows, no host synchronisation; like the rest of the
package the operators launch on the current stream of their tensors' device
and may be captured in a CUDA graph, and each first offers its arguments to
the compiled dispatch (``_fastpath``), which takes the common case.

The products' in-kernel waits are bounded (about 2 s).  An expired one leaves
that call's output invalid without an error: ``kernels.product_status()`` tells
of it, ``kernels.product_reset()`` clears it.
"""

from __future__ import annotations

import math

import torch

from fused_decode_b200._capi import ACTIVATIONS
from fused_decode_b200._capi import fast_or_none as _fast
from fused_decode_b200.kernels import (
    linear_act_out,
    linear_fp8_out,
    post_attn_mlp_fp8_out,
    quantize_fp8_out,
    rms_fp8_out,
    swiglu_fp8_out,
)

E4M3 = torch.float8_e4m3fn
_HALF = (torch.float16, torch.bfloat16)
_REAL = (torch.float16, torch.bfloat16, torch.float32)

__all__ = [
    "add_rms_norm_fp8",
    "linear_act",
    "linear_fp8",
    "post_attn_mlp_fp8",
    "quantize_fp8",
    "rms_norm_fp8",
    "swiglu_fp8",
]


# ---------------------------------------------------------------- checks
# Types and shapes first, the device last, so that a wrong call is told what
# is wrong with it wherever its tensors are.
def _check_tensor(t: torch.Tensor, name: str, dtypes: tuple[torch.dtype, ...], what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {what}, got {t.dtype}")


def _check_rows(t: torch.Tensor, name: str) -> None:
    _check_tensor(t, name, _HALF, "float16 or bfloat16")
    if t.ndim == 0:
        raise ValueError(f"{name} must have a last dimension")


def _check_like(t: torch.Tensor, like: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.shape != like.shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} != {tuple(like.shape)}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} dtype {t.dtype} != {like.dtype}")


def _check_norm(weight: torch.Tensor, x: torch.Tensor, eps: float, name: str = "weight") -> float:
    _check_tensor(weight, name, _REAL, "float16, bfloat16, or float32")
    if weight.ndim != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(weight.shape)}")
    eps = float(eps)
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be a finite value >= 0")
    return eps


def _check_device(x: torch.Tensor, name: str, **others: torch.Tensor | None) -> None:
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    for other, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{other} is on {t.device}, expected {x.device}")


def _check_rows8(out: torch.Tensor | None, scale_out: torch.Tensor | None, x: torch.Tensor) -> None:
    if out is not None:
        _check_tensor(out, "out", (E4M3,), "float8_e4m3fn")
        if out.shape != x.shape:
            raise ValueError(f"out shape {tuple(out.shape)} != {tuple(x.shape)}")
    if scale_out is not None:
        _check_tensor(scale_out, "scale_out", (torch.float32,), "float32")
        if scale_out.shape != x.shape[:-1]:
            raise ValueError(f"scale_out shape {tuple(scale_out.shape)} != {tuple(x.shape[:-1])}")
        if not scale_out.is_contiguous():
            raise ValueError("scale_out must be contiguous")


def _rows8(out: torch.Tensor | None, scale_out: torch.Tensor | None,
           x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``out`` and ``scale_out``, fresh where they are not given."""
    if out is None:
        out = torch.empty(x.shape, device=x.device, dtype=E4M3)
    if scale_out is None:
        scale_out = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    return out, scale_out


# ---------------------------------------------------------------- rows to 8 bits
def quantize_fp8(
    x: torch.Tensor,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``x`` (its last dimension) to ``(values, scale)``: e4m3 of
    ``x``'s shape and fp32 of ``x.shape[:-1]``, ``x ~ values * scale[..., None]``.

    Weights ``[N, K]`` are laid out with it once; activations that no operator
    here produces (the attention's output, say) on every step.
    """
    fp = _fast()
    done = fp.quantize_fp8(x, out, scale_out) if fp is not None else None
    if done is not None:
        return done
    _check_rows(x, "x")
    _check_rows8(out, scale_out, x)
    _check_device(x, "x", out=out, scale_out=scale_out)
    out, scale_out = _rows8(out, scale_out, x)
    quantize_fp8_out(x, out, scale_out)
    return out, scale_out


def rms_norm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``rms_norm`` with the normalised rows in 8 bits: ``(values, scale)``.

    The fp32 rows are quantised directly, without the rounding to ``x``'s type
    that ``rms_norm`` makes.
    """
    fp = _fast()
    done = fp.rms_norm_fp8(x, weight, eps, out, scale_out) if fp is not None else None
    if done is not None:
        return done
    _check_rows(x, "x")
    eps = _check_norm(weight, x, eps)
    _check_rows8(out, scale_out, x)
    _check_device(x, "x", weight=weight, out=out, scale_out=scale_out)
    out, scale_out = _rows8(out, scale_out, x)
    rms_fp8_out(x, weight, eps, out, scale_out)
    return out, scale_out


def add_rms_norm_fp8(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``add_rms_norm`` with the normalised rows in 8 bits: ``(values, scale, residual_out)``.

    ``residual_out = x + residual`` in ``x``'s type; the norm sees the fp32
    sum.  Pass ``residual_out=residual`` to update the residual stream in place.
    """
    fp = _fast()
    done = fp.add_rms_norm_fp8(x, residual, weight, eps, out, scale_out, residual_out) if fp is not None else None
    if done is not None:
        return done
    _check_rows(x, "x")
    _check_like(residual, x, "residual")
    eps = _check_norm(weight, x, eps)
    _check_rows8(out, scale_out, x)
    if residual_out is not None:
        _check_like(residual_out, x, "residual_out")
    _check_device(x, "x", residual=residual, weight=weight, out=out, scale_out=scale_out, residual_out=residual_out)
    out, scale_out = _rows8(out, scale_out, x)
    if residual_out is None:
        residual_out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    rms_fp8_out(x, weight, eps, out, scale_out, residual=residual, residual_out=residual_out)
    return out, scale_out, residual_out


def swiglu_fp8(
    gate: torch.Tensor,
    up: torch.Tensor,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``silu(gate) * up`` in 8 bits: ``(values, scale)``.  ``gate`` and ``up``
    may be views, such as the halves of one gate/up product."""
    fp = _fast()
    done = fp.swiglu_fp8(gate, up, out, scale_out) if fp is not None else None
    if done is not None:
        return done
    _check_rows(gate, "gate")
    _check_like(up, gate, "up")
    _check_rows8(out, scale_out, gate)
    _check_device(gate, "gate", up=up, out=out, scale_out=scale_out)
    out, scale_out = _rows8(out, scale_out, gate)
    swiglu_fp8_out(gate, up, out, scale_out)
    return out, scale_out


# ---------------------------------------------------------------- products
def _check_product(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, activation: str | None,
                   row_add: torch.Tensor | None, out: torch.Tensor | None, out_dtype: torch.dtype) -> tuple[int, ...]:
    """Shapes and types of a product's arguments; returns the output's shape."""
    if x.ndim == 0:
        raise ValueError("x must have a last dimension")
    if weight.ndim != 2:
        raise ValueError(f"weight must have shape [N, K], got {tuple(weight.shape)}")
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"x last dim {x.shape[-1]} != weight K {k}")
    if activation not in ACTIVATIONS:
        names = ", ".join(repr(a) for a in ACTIVATIONS if a)
        raise ValueError(f"activation must be None or one of {names}, got {activation!r}")
    expected = (*x.shape[:-1], n)
    if bias is not None:
        _check_tensor(bias, "bias", (out_dtype, torch.float32), f"{out_dtype} or float32")
        if bias.ndim != 1 or bias.shape[0] != n:
            raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
    if row_add is not None:
        _check_tensor(row_add, "row_add", _REAL, "float16, bfloat16, or float32")
        try:
            row_add.expand(expected)
        except RuntimeError as exc:
            raise ValueError(f"row_add shape {tuple(row_add.shape)} is not broadcastable to {expected}") from exc
    if out is not None:
        _check_tensor(out, "out", (out_dtype,), str(out_dtype))
        if tuple(out.shape) != expected:
            raise ValueError(f"out shape {tuple(out.shape)} != {expected}")
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    return expected


def _as_2d(x: torch.Tensor) -> torch.Tensor:
    """``x`` as [M, K], a view where its strides allow one."""
    return x if x.ndim == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def _row_add_2d(row_add: torch.Tensor | None, m: int, n: int, expected: tuple[int, ...]) -> torch.Tensor | None:
    """``row_add`` as a 2-D [1|M, 1|N] operand (it broadcasts to ``expected``)."""
    if row_add is None:
        return None
    if row_add.numel() == 0:
        return row_add.new_zeros(1, 1)  # the output is empty too
    last = row_add.shape[-1] if row_add.ndim else 1
    if row_add.numel() == last:  # one row for every row
        return row_add.reshape(1, last)
    if len(expected) == 2:
        return row_add
    return row_add.expand(*expected[:-1], last).reshape(m, last)


def linear_act(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    row_add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``y = act(x @ weight.T + bias) + row_add``, any number of rows.

    ``weight`` is ``[N, K]`` as in ``F.linear``; ``activation`` is None,
    ``"relu"``, ``"silu"``, ``"gelu"`` (erf) or ``"gelu_tanh"``.  ``bias`` is
    of ``x``'s type or float32; ``row_add`` (a residual) is any 16- or 32-bit
    float tensor that broadcasts to the output.  The sum, the activation and
    both additions are fp32 and the result is rounded once.  ``out`` may be
    ``row_add`` itself and may not overlap ``x`` or ``weight``.
    """
    fp = _fast()
    done = fp.linear_act(x, weight, bias, activation, row_add, out) if fp is not None else None
    if done is not None:
        return done
    _check_tensor(x, "x", _HALF, "float16 or bfloat16")
    _check_tensor(weight, "weight", (x.dtype,), str(x.dtype))
    expected = _check_product(x, weight, bias, activation, row_add, out, x.dtype)
    _check_device(x, "x", weight=weight, bias=bias, row_add=row_add, out=out)
    x2, n = _as_2d(x), weight.shape[0]
    m = x2.shape[0]
    if out is None:
        out = torch.empty(expected, device=x.device, dtype=x.dtype)
    linear_act_out(x2, weight, out.view(m, n), bias=bias, activation=activation,
                   row_add=_row_add_2d(row_add, m, n, expected))
    return out


def linear_fp8(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    row_add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``linear_act`` of 8-bit operands: ``act((x @ weight.T) * x_scale * weight_scale + bias) + row_add``.

    ``x`` is e4m3 ``[..., K]`` with fp32 ``x_scale`` of ``x.shape[:-1]`` and
    ``weight`` e4m3 ``[N, K]`` with fp32 ``weight_scale`` ``[N]``, as
    ``quantize_fp8`` and its companions return them.  The output is of
    ``out_dtype`` (float16 or bfloat16), ``bias`` of that type or float32.
    """
    fp = _fast() if out_dtype in _HALF else None
    done = fp.linear_fp8(x, x_scale, weight, weight_scale, bias, activation, row_add, out,
                         out_dtype == torch.bfloat16) if fp is not None else None
    if done is not None:
        return done
    _check_tensor(x, "x", (E4M3,), "float8_e4m3fn")
    _check_tensor(weight, "weight", (E4M3,), "float8_e4m3fn")
    if out_dtype not in _HALF:
        raise TypeError(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    expected = _check_product(x, weight, bias, activation, row_add, out, out_dtype)
    for name, scale, shape in (("x_scale", x_scale, x.shape[:-1]), ("weight_scale", weight_scale, weight.shape[:1])):
        _check_tensor(scale, name, (torch.float32,), "float32")
        if scale.shape != shape:
            raise ValueError(f"{name} shape {tuple(scale.shape)} != {tuple(shape)}")
    _check_device(x, "x", x_scale=x_scale, weight=weight, weight_scale=weight_scale, bias=bias, row_add=row_add,
                  out=out)
    x2, n = _as_2d(x), weight.shape[0]
    m = x2.shape[0]
    if out is None:
        out = torch.empty(expected, device=x.device, dtype=out_dtype)
    linear_fp8_out(x2, x_scale.contiguous().view(m), weight, weight_scale.contiguous(), out.view(m, n), bias=bias,
                   activation=activation, row_add=_row_add_2d(row_add, m, n, expected))
    return out


# ---------------------------------------------------------------- MLP block
def post_attn_mlp_fp8(
    hidden: torch.Tensor,
    norm_weight: torch.Tensor,
    w_gate_up: torch.Tensor,
    gate_up_scale: torch.Tensor,
    w_down: torch.Tensor,
    down_scale: torch.Tensor,
    eps: float = 1e-6,
) -> torch.Tensor:
    """``post_attn_mlp`` with 8-bit weights and activations, any number of rows.

    ``w_gate_up`` is e4m3 ``[2I, H]`` (gate stacked above up) with
    ``gate_up_scale`` ``[2I]``, ``w_down`` e4m3 ``[H, I]`` with ``down_scale``
    ``[H]``, both from ``quantize_fp8``.  The same values as ``rms_norm_fp8``
    -> ``linear_fp8`` -> ``swiglu_fp8`` -> ``linear_fp8`` with ``hidden`` as
    ``row_add``, enqueued by one call.
    """
    fp = _fast()
    done = fp.post_attn_mlp_fp8(hidden, norm_weight, w_gate_up, gate_up_scale, w_down, down_scale, eps) if fp is not None else None
    if done is not None:
        return done
    _check_rows(hidden, "hidden")
    for name, w in (("w_gate_up", w_gate_up), ("w_down", w_down)):
        _check_tensor(w, name, (E4M3,), "float8_e4m3fn")
        if w.ndim != 2:
            raise ValueError("w_gate_up and w_down must be rank-2")
    two_i, h = w_gate_up.shape
    h_down, i = w_down.shape
    if two_i != 2 * i or h != h_down or hidden.shape[-1] != h:
        raise ValueError(
            f"expected w_gate_up [2I, H] and w_down [H, I] with hidden [..., H], "
            f"got {tuple(w_gate_up.shape)}, {tuple(w_down.shape)}, {tuple(hidden.shape)}"
        )
    if h == 0 or i == 0:
        raise ValueError("H and I must be positive")
    for name, scale, rows in (("gate_up_scale", gate_up_scale, two_i), ("down_scale", down_scale, h)):
        _check_tensor(scale, name, (torch.float32,), "float32")
        if scale.shape != (rows,):
            raise ValueError(f"{name} must have shape ({rows},), got {tuple(scale.shape)}")
    eps = _check_norm(norm_weight, hidden, eps, "norm_weight")
    _check_device(hidden, "hidden", norm_weight=norm_weight, w_gate_up=w_gate_up, gate_up_scale=gate_up_scale,
                  w_down=w_down, down_scale=down_scale)
    out = torch.empty(hidden.shape, device=hidden.device, dtype=hidden.dtype)
    hidden2 = _as_2d(hidden)
    if hidden2.stride(1) != 1:
        hidden2 = hidden2.contiguous()
    if hidden2.shape[0] == 0:
        return out
    w_gate_up, w_down = (w if w.stride(1) == 1 else w.contiguous() for w in (w_gate_up, w_down))
    post_attn_mlp_fp8_out(hidden2, norm_weight, w_gate_up, gate_up_scale.contiguous(), w_down,
                          down_scale.contiguous(), out.view(hidden2.shape), eps)
    return out

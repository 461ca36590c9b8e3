"""The 8-bit operators and the products with an epilogue in 64 bits, from their
definitions, with bounds on what fp32 arithmetic may be off.

U32 = 2^-24 is half a step of fp32.  Bounds count the roundings of the longest
chain an element goes through:

* a row's value y: the norm's sum of n squares (a chain of at most n / 256 + 16
  additions per thread and reduction tree, halved by the square root), the
  hardware exp's 2^-22-ish error scaled by |gate| <= 16, and a few products --
  all together within (n / 256 + 64) U32 relative.
* a product's sum: chains of k / 16 + 32 additions, each off by at most a whole
  step (the tensor cores may truncate): (k / 16 + 32) 2 U32 of sum |x||w|.
  The activations' slopes are below 1.2.
"""

import math

import torch

U32 = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
FLOOR = 2.0 ** -64


def silu(v):
    return v * torch.special.expit(v)


ACTIVATIONS = {
    None: lambda v: v,
    "relu": lambda v: torch.where(v < 0, torch.zeros_like(v), v),
    "silu": silu,
    "gelu": lambda v: 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0)),
    "gelu_tanh": lambda v: 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))),
}


def rms(x, w, eps, residual=None):
    v = x.double() if residual is None else x.double() + residual.double()
    return v / (v.square().mean(dim=-1, keepdim=True) + eps).sqrt() * w.double()


def swiglu(gate, up):
    return silu(gate.double()) * up.double()


def check_rows8(values, scale, y):
    """Values and scales of fp64 rows ``y``: the scale within the rows' fp32
    bound, every value within half an 8-bit step of y / scale, the largest of a
    row at 448."""
    assert values.dtype == E4M3 and scale.dtype == torch.float32
    assert values.shape == y.shape and scale.shape == y.shape[:-1]
    if y.numel() == 0:
        return
    rel = (y.shape[-1] / 256 + 64) * U32
    a = y.abs().amax(dim=-1).clamp_min(FLOOR)
    torch.testing.assert_close(scale.double(), a / 448.0, rtol=rel, atol=0.0)
    got, s = values.double(), scale.double()[..., None]
    half = torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10)  # normal numbers, and the subnormal ones' 2^-9 steps
    off = (got * s - y).abs()
    assert (off <= half * (1 + 1e-6) + 4 * rel * y.abs()).all(), float((off / half).max())
    assert (got.abs().amax(dim=-1)[a > FLOOR * 2] == 448.0).all()


def product(x, w, bias, activation, row_add, xs=None, ws=None):
    """(y, bound): the product in 64 bits and how far its fp32 form may be from it before the last rounding."""
    xd, wd = x.double(), w.double()
    if xs is not None:
        xd, wd = xd * xs.double()[..., None], wd * ws.double()[:, None]
    v = xd @ wd.T
    bound = (x.shape[-1] / 16 + 32) * 2 * U32 * (xd.abs() @ wd.abs().T)
    if bias is not None:
        v = v + bias.double()
        bound = bound + 4 * U32 * bias.double().abs()
    bound = 1.2 * bound + 64 * U32 * v.abs()
    v = ACTIVATIONS[activation](v)
    if row_add is not None:
        v = v + row_add.double()
        bound = bound + 4 * U32 * row_add.double().abs()
    return v, bound


def check_product(y, ref, bound):
    assert y.shape == ref.shape
    half = torch.finfo(y.dtype).eps / 2
    smallest = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps  # a subnormal step
    allowed = half * ref.abs() + (1 + 2 * half) * bound + smallest
    off = (y.double() - ref).abs()
    assert (off <= allowed).all(), (float((off / allowed).max()), float(off.max()))

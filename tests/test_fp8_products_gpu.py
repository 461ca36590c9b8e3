"""How the products' kernels split their work on the GPU, against 64-bit forms
(tests/_fp8_ref.py, which derives the bounds)."""

import pytest
import torch

from tests import _fp8_ref as R

pytestmark = pytest.mark.gpu

import fused_decode_b200 as fd  # noqa: E402

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def rows8(g, n, k, scale=1.0):
    """e4m3 rows with every exponent in use, and scales of their own."""
    q = (torch.randn(n, k, device="cuda", generator=g) * 40).clamp(-448, 448).to(R.E4M3)
    return q, (torch.rand(n, device="cuda", generator=g) * 1e-2 + 1e-3) * scale


def both_types(seed, m, n, k, act, times=1):
    """The product in 16 and in 8 bits with bias and row_add: every element, the same bits every time."""
    g = gen(seed)
    bias, res = rn(g, n, dtype=F32), rn(g, m, n)
    x, w = rn(g, m, k), rn(g, n, k, scale=k ** -0.5)
    y = fd.linear_act(x, w, bias, activation=act, row_add=res)
    R.check_product(y, *R.product(x, w, bias, act, res))
    for _ in range(times - 1):
        assert torch.equal(fd.linear_act(x, w, bias, activation=act, row_add=res), y)
    (x, xs), (w, ws) = rows8(g, m, k), rows8(g, n, k, k ** -0.5)
    y = fd.linear_fp8(x, xs, w, ws, bias, activation=act, row_add=res)
    R.check_product(y, *R.product(x, w, bias, act, res, xs, ws))
    for _ in range(times - 1):
        assert torch.equal(fd.linear_fp8(x, xs, w, ws, bias, activation=act, row_add=res), y)


# N that leaves most of the last tile without rows of w, K long enough that a
# cluster shares each tile
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (2, 8, 8192), (3, 136, 4096), (40, 1000, 4096), (80, 520, 4096),
                                   (81, 264, 4096), (200, 300, 4096), (640, 520, 4096)])
def test_shared_tiles_past_the_last_row(m, n, k):
    both_types(m + n, m, n, k, "silu", times=4)


@pytest.mark.parametrize("m,n,k", [(8, 4096, 16384), (64, 9472, 8192), (512, 1024, 16384), (1024, 4096, 8192)])
def test_long_inner_widths(m, n, k):
    """Many steps to a tile, so that the MMAs follow the copies through every
    stage of the ring many times over: whatever landed between two looks, the
    same bits."""
    both_types(m, m, n, k, None, times=8)


# One block that lets the next kernel on the stream start at once and then takes
# 5e9 cycles (2.5 s at 1.97 GHz, 5 s at 1 GHz: more than a bounded wait's 4e9).
LONG_KERNEL = r"""
extern "C" __global__ void long_kernel() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long t0 = clock64();
  while (clock64() - t0 < 5000000000ll) __nanosleep(1000);
}
"""


@pytest.mark.parametrize("m,n,k", [(3, 4096, 1024), (300, 512, 1024)])
def test_a_long_kernel_ahead_expires_no_wait(m, n, k):
    """A product that starts early behind a kernel of seconds waits for it
    without counting that time against its own bound."""
    from fused_decode_b200 import kernels as K

    g = gen(m)
    (x, xs), (w, ws) = rows8(g, m, k), rows8(g, n, k, k ** -0.5)
    ref = fd.linear_fp8(x, xs, w, ws)
    y = torch.zeros_like(ref)
    long_kernel = torch.cuda._compile_kernel(LONG_KERNEL, "long_kernel", compute_capability="100")
    torch.cuda.synchronize()
    long_kernel(grid=(1, 1, 1), block=(1, 1, 1))
    fd.linear_fp8(x, xs, w, ws, out=y)
    assert torch.equal(y, ref)
    assert K.product_status() == 0


# Up to 80 rows: N above 256 rows of w for each of the 148 SMs, so that a CTA goes
# over several tiles -- with two accumulators (up to 64 rows) and with one.
@pytest.mark.parametrize("m,n,k", [(1, 128256, 1024), (64, 128256, 1024), (65, 128256, 1024), (80, 100003, 640),
                                   (17, 40000, 2000)])
def test_several_tiles_to_a_block(m, n, k):
    both_types(n + m, m, n, k, "relu", times=2)


# More rows: at least 149 tiles of 256 by 256 for the 74 pairs of CTAs, both sides
# ragged, so that each pair goes over three tiles or more with the ring, the
# accumulators and the scales of x carried from one to the next.
@pytest.mark.parametrize("m,n,k", [(1990, 5130, 720), (1030, 10313, 528), (300, 40000, 1040), (5000, 2049, 272)])
def test_several_tiles_to_a_pair(m, n, k):
    both_types(n + m, m, n, k, "gelu", times=2)

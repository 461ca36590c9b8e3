"""The 8-bit row operators between other kernels on the stream."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import fused_decode_b200 as fd  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32


# rows of vectors, rows too long for them, and an input at an odd offset
@pytest.mark.parametrize("rows,n,offset", [(2048, 4096, 0), (8192, 2048, 0), (600, 33000, 0), (4096, 1024, 1)])
def test_residual_out_becomes_the_next_products_weight(rows, n, offset):
    """linear_decode streams its weight before it waits for the kernel before
    it; the norm's residual_out is finished by then, to its last rows."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, res, y = (torch.randn(r, n + offset, device="cuda", generator=g).to(BF)[:, offset:] for r in (rows, rows, 2))
    nw = torch.ones(n, device="cuda")
    w = torch.zeros(rows, n, device="cuda", dtype=BF)
    ref_w = (x.float() + res.float()).to(BF)
    ref = fd.linear_decode(y, ref_w)
    for _ in range(20):
        w.zero_()
        fd.add_rms_norm_fp8(x, res, nw, 1e-5, residual_out=w)
        assert torch.equal(fd.linear_decode(y, w), ref)
        assert torch.equal(w, ref_w)


@pytest.mark.parametrize("dtype", [torch.float16, BF])
@pytest.mark.parametrize("rows,n", [(1, 1), (40, 4096), (2000, 1024), (9, 77), (300, 5001), (3, 40000)])
def test_values_and_scales_to_the_bit(rows, n, dtype):
    """scale = a / 448 and values e4m3(x * (448 / a)), each operation rounded
    once in fp32: no other value, even where x lies midway between two."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, n, device="cuda", generator=g).to(dtype)
    q, s = fd.quantize_fp8(x)
    a = x.float().abs().amax(dim=-1).clamp_min(2.0 ** -64)
    most = torch.full_like(a, 448.0)  # a tensor: torch divides by a number, or a number, through a reciprocal
    assert torch.equal(s, a / most)
    want = (x.float() * (most / a)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("rows,n", [(1, 4096), (16, 4096), (148, 8192), (100, 512), (7, 256), (9, 14336), (2, 32768)])
def test_residual_out_of_few_rows_becomes_the_next_products_weight(rows, n):
    """As above for few rows, back to back in a graph, without the host's pace between the calls."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, res, y = (torch.randn(r, n, device="cuda", generator=g).to(BF) for r in (rows, rows, 2))
    nw = torch.ones(n, device="cuda")
    w = torch.zeros(rows, n, device="cuda", dtype=BF)
    ref_w = (x.float() + res.float()).to(BF)
    ref = fd.linear_decode(y, ref_w)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = []
        for _ in range(20):
            w.zero_()
            fd.add_rms_norm_fp8(x, res, nw, 1e-5, residual_out=w)
            outs.append(fd.linear_decode(y, w))
    for _ in range(10):
        graph.replay()
        for out in outs:
            assert torch.equal(out, ref)

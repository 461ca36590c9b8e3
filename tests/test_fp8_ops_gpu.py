"""The 8-bit operators and ``linear_act`` on the GPU against 64-bit forms
(tests/_fp8_ref.py, which derives the bounds)."""

import pytest
import torch

from tests import _fp8_ref as R

pytestmark = pytest.mark.gpu

import fused_decode_b200 as fd  # noqa: E402

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = [BF, F16]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def weight8(g, n, k):
    """e4m3 rows with every exponent in use, and scales of their own."""
    q = (torch.randn(n, k, device="cuda", generator=g) * 40).clamp(-448, 448).to(R.E4M3)
    return q, torch.rand(n, device="cuda", generator=g) * 1e-2 + 1e-3


# ------------------------------------------------------------------ rows to 8 bits
# widths: one element, odd, below and at a vector, the decode widths, above the
# widest row that is kept in registers
ROWS = [(1, 1), (3, 7), (1, 8), (5, 72), (2, 128), (9, 250), (4, 256), (3, 520), (1, 4096), (33, 1000), (150, 4096),
        (7, 5123), (300, 640), (2, 14336), (2, 16392), (1, 28672), (3, 32768), (2, 32776), (1, 50001)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n", ROWS)
def test_rows8(m, n, dtype):
    g = gen(m * 100003 + n)
    x, r = rn(g, m, n, dtype=dtype, scale=3.0), rn(g, m, n, dtype=dtype)
    w = (1 + 0.1 * torch.randn(n, device="cuda", generator=g)).to(dtype)
    R.check_rows8(*fd.quantize_fp8(x), x.double())
    R.check_rows8(*fd.rms_norm_fp8(x, w, 1e-5), R.rms(x, w, 1e-5))
    q, s, ro = fd.add_rms_norm_fp8(x, r, w.float(), 1e-5)
    R.check_rows8(q, s, R.rms(x, w, 1e-5, r))
    assert torch.equal(ro, (x.float() + r.float()).to(dtype))
    R.check_rows8(*fd.swiglu_fp8(x, r), R.swiglu(x, r))


def test_rows8_views_and_leading_dims():
    """Halves of a product, transposed rows, four and five dimensions, odd
    offsets, a broadcast input, given outputs inside larger buffers."""
    g = gen(1)
    for n in (64, 77, 1024):
        gu = rn(g, 5, 2 * n)
        gate, up = gu.split(n, dim=-1)
        R.check_rows8(*fd.swiglu_fp8(gate, up), R.swiglu(gate, up))
    x = rn(g, 96, 40).t()
    R.check_rows8(*fd.quantize_fp8(x), x.double())
    x = rn(g, 2, 3, 4, 136)
    R.check_rows8(*fd.quantize_fp8(x.transpose(0, 2)), x.transpose(0, 2).double())
    R.check_rows8(*fd.quantize_fp8(x[..., 1:]), x[..., 1:].double())
    w = rn(g, 136, dtype=F32)
    R.check_rows8(*fd.rms_norm_fp8(x[:, 1:], w, 1e-6), R.rms(x[:, 1:], w, 1e-6))
    x5 = rn(g, 2, 2, 2, 3, 64)
    R.check_rows8(*fd.quantize_fp8(x5), x5.double())
    out5 = torch.zeros(2, 2, 2, 3, 128, device="cuda", dtype=R.E4M3)[..., ::2]
    q, s = fd.quantize_fp8(x5, out=out5)
    assert q is out5
    R.check_rows8(q, s, x5.double())
    xe = rn(g, 1, 256).expand(6, 256)
    R.check_rows8(*fd.quantize_fp8(xe), xe.double())
    v = rn(g, 512)  # one row, no leading dimension
    q, s = fd.quantize_fp8(v)
    assert s.shape == ()
    R.check_rows8(q, s, v.double())
    for off in (0, 1, 8):
        big = torch.zeros(4, 640, device="cuda", dtype=R.E4M3)
        scales = torch.zeros(6, device="cuda")
        x = rn(g, 2, 512)
        fd.quantize_fp8(x, out=big[1:3, off:off + 512], scale_out=scales[2:4])
        R.check_rows8(big[1:3, off:off + 512], scales[2:4], x.double())
        rest = big.float()
        rest[1:3, off:off + 512] = 0
        assert torch.count_nonzero(rest) == 0 and torch.count_nonzero(scales[[0, 1, 4, 5]]) == 0


def test_rows8_strided_norm_weight():
    g = gen(2)
    x, w = rn(g, 3, 256), rn(g, 512, dtype=F32)[::2]
    R.check_rows8(*fd.rms_norm_fp8(x, w, 1e-6), R.rms(x, w, 1e-6))


@pytest.mark.parametrize("n", [96, 100, 4096, 33000])
def test_rows8_residual_in_place(n):
    g = gen(3)
    x, r = rn(g, 9, n), rn(g, 9, n)
    w = rn(g, n)
    q0, s0, ro0 = fd.add_rms_norm_fp8(x, r, w)
    keep = r.clone()
    q, s, ro = fd.add_rms_norm_fp8(x, r, w, residual_out=r)
    assert ro is r and torch.equal(r, ro0) and not torch.equal(r, keep)
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)


@pytest.mark.parametrize("n", [64, 77, 4096, 32776])
def test_rows8_zero_tiny_and_not_finite(n):
    """Rows of zeros, of the smallest values, with infinities and NaN: each row
    goes its own way and leaves its neighbours alone."""
    g = gen(4)
    x = rn(g, 6, n)
    x[1] = 0
    x[2] = 1e-30  # below the floor 2^-64: values 0 under the floor's scale
    x[3, n // 2] = float("inf")
    x[4, n - 1] = float("nan")
    q, s = fd.quantize_fp8(x)
    for i in (0, 5):
        R.check_rows8(q[i], s[i], x[i].double())
    for i in (1, 2):
        assert s[i].item() == pytest.approx(R.FLOOR / 448, rel=1e-6) and torch.count_nonzero(q[i].float()) == 0
    assert s[3].item() == float("inf") and q[3].float()[n // 2].isnan() and torch.count_nonzero(q[3].float()[:n // 2]) == 0
    assert s[4].isnan() and q[4].float().isnan().all()
    w = torch.ones(n, device="cuda")
    w_inf = w.clone()
    w_inf[0] = float("inf")
    q, s = fd.rms_norm_fp8(x, w, 1e-6)
    for i in (0, 1, 2, 5):
        R.check_rows8(q[i], s[i], R.rms(x[i], w, 1e-6))
    assert s[3].isnan() and s[4].isnan()  # inf * rsqrt(inf) is NaN
    q, s = fd.rms_norm_fp8(x[:1], w_inf, 1e-6)
    assert s[0].item() == float("inf") and torch.count_nonzero(q[0].float()[1:]) == 0
    w_inf[0] = float("nan")
    assert fd.rms_norm_fp8(x[:1], w_inf, 1e-6)[1].isnan().all()
    # squares beyond fp32: rsqrt(inf) = 0 and every finite element becomes 0,
    # though value times weight alone would not be finite
    big = torch.full((2, n), 1e30, device="cuda", dtype=BF)
    q, s = fd.rms_norm_fp8(big, w * 1e20, 1e-6)
    assert torch.count_nonzero(q.float()) == 0 and (s == s[0]).all() and s[0].item() == pytest.approx(R.FLOOR / 448, rel=1e-6)
    gate, up = rn(g, 4, n), rn(g, 4, n)
    gate[1, 0] = float("-inf")
    up[2, n - 1] = float("nan")
    q, s = fd.swiglu_fp8(gate, up)
    for i in (0, 3):
        R.check_rows8(q[i], s[i], R.swiglu(gate[i], up[i]))
    assert s[1].isnan() and s[2].isnan()


def test_rows8_empty():
    w = torch.ones(64, device="cuda")
    x = torch.empty(0, 64, device="cuda", dtype=BF)
    for q, s in (fd.quantize_fp8(x), fd.rms_norm_fp8(x, w), fd.swiglu_fp8(x, x), fd.add_rms_norm_fp8(x, x, w)[:2]):
        assert q.shape == (0, 64) and s.shape == (0,)
    q, s = fd.quantize_fp8(torch.empty(3, 0, device="cuda", dtype=BF))  # no element: the floor's scale
    assert q.shape == (3, 0) and (s > 0).all()


# ------------------------------------------------------------------ products
# (m, n, k): single tokens, tile edges of either side, odd everything, inner
# widths below a vector and across steps, several tiles
PRODUCTS = [(1, 1, 1), (1, 128, 64), (1, 129, 4096), (2, 7, 5), (3, 1000, 136), (5, 384, 16), (8, 2048, 1024),
            (16, 255, 2048), (17, 520, 144), (33, 1, 512), (40, 130, 100), (64, 1024, 512), (100, 333, 2064),
            (129, 257, 640), (255, 640, 1040), (257, 512, 272), (300, 1000, 528), (520, 200, 4096), (1025, 768, 256),
            (2000, 1336, 112), (777, 2309, 801)]
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("index,shape", list(enumerate(PRODUCTS)))
def test_linear_act(index, shape, dtype):
    m, n, k = shape
    g = gen(index)
    x, w = rn(g, m, k, dtype=dtype), rn(g, n, k, dtype=dtype, scale=k ** -0.5)
    bias, res = rn(g, n, dtype=dtype), rn(g, m, n, dtype=dtype)
    R.check_product(fd.linear_act(x, w), *R.product(x, w, None, None, None))
    act = ACTS[index % 5]
    y = fd.linear_act(x, w, bias, activation=act, row_add=res)
    R.check_product(y, *R.product(x, w, bias, act, res))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("index,shape", list(enumerate(PRODUCTS)))
def test_linear_fp8(index, shape, dtype):
    m, n, k = shape
    g = gen(index)
    x, xs = weight8(g, m, k)
    w, ws = weight8(g, n, k)
    ws = ws * k ** -0.5
    bias, res = rn(g, n, dtype=F32), rn(g, m, n, dtype=dtype)
    y = fd.linear_fp8(x, xs, w, ws, out_dtype=dtype)
    assert y.dtype == dtype
    R.check_product(y, *R.product(x, w, None, None, None, xs, ws))
    act = ACTS[(index + 2) % 5]
    y = fd.linear_fp8(x, xs, w, ws, bias, activation=act, row_add=res, out_dtype=dtype)
    R.check_product(y, *R.product(x, w, bias, act, res, xs, ws))


@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(act):
    """Sums from -30 to 30, where exp and tanh saturate, as a product with the identity."""
    v = torch.linspace(-30, 30, 4096, device="cuda").to(F16).view(64, 64)
    eye = torch.eye(64, device="cuda", dtype=F16)
    R.check_product(fd.linear_act(v, eye, activation=act), *R.product(v, eye, None, act, None))


@pytest.mark.parametrize("m", [1, 12, 40, 270])
def test_row_add_forms_and_in_place(m):
    """Residuals that broadcast, of every type, strided; out= the residual itself; bias strided or fp32."""
    g = gen(m)
    n, k = 328, 192
    x, w = rn(g, m, k), rn(g, n, k, scale=k ** -0.5)
    wide = rn(g, m, 2 * n, dtype=F32)
    forms = [rn(g, n), rn(g, 1, n, dtype=F16), rn(g, m, 1, dtype=F32), rn(g, 1, 1), rn(g, 1)[0], rn(g, m, n, dtype=F32),
             rn(g, m, n, dtype=F16), wide[:, ::2], wide[:, 1:n + 1], rn(g, n, m).t(), rn(g, m, n)]
    for ra in forms:
        y = fd.linear_act(x, w, activation="relu", row_add=ra)
        R.check_product(y, *R.product(x, w, None, "relu", ra.expand(m, n)))
    for bias in (rn(g, n, dtype=F32), rn(g, 2 * n)[::2]):
        R.check_product(fd.linear_act(x, w, bias), *R.product(x, w, bias, None, None))
    buffer = rn(g, m + 2, n)
    keep = buffer.clone()
    res = buffer[1:m + 1]
    ref = R.product(x, w, None, None, keep[1:m + 1])
    assert fd.linear_act(x, w, row_add=res, out=res) is res
    R.check_product(res, *ref)
    assert torch.equal(buffer[0], keep[0]) and torch.equal(buffer[-1], keep[-1])  # rows around the output


@pytest.mark.parametrize("m", [1, 6, 50, 300])
def test_product_layouts(m):
    """Operands as views: rows apart by more than their length, by a length that
    is no multiple of 16 bytes, transposed, at odd offsets, with more
    dimensions, every row the same."""
    g = gen(m)
    n, k = 264, 320

    def check(x, w):
        y = fd.linear_act(x, w)
        R.check_product(y, *R.product(x, w, None, None, None))

    x, w = rn(g, m, k), rn(g, n, k, scale=k ** -0.5)
    check(rn(g, m, 2 * k)[:, k:], rn(g, n, 2 * k)[:, :k])
    check(rn(g, m, k + 3)[:, 3:], w)
    check(x, rn(g, n, k + 5)[:, 1:k + 1])
    check(rn(g, k, m).t(), w)
    check(x, rn(g, k, n).t())
    check(rn(g, m, 2 * k)[:, ::2], w)
    check(rn(g, 1, k).expand(m, k), w)
    check(x, rn(g, 1, k).expand(n, k))
    check(rn(g, m + 1, 328)[1:, :k], w[3:])
    x3 = rn(g, 2, m, k)
    check(x3, w)
    check(x3.transpose(0, 1), w)
    y = fd.linear_act(x[0], w)
    assert y.shape == (n,)
    R.check_product(y, *R.product(x[0], w, None, None, None))
    q, s = weight8(g, n, k)
    wide, ws = weight8(g, m, k + 24)
    for x8 in (wide[:, 16:16 + k], wide[:, 1:1 + k]):
        R.check_product(fd.linear_fp8(x8, ws, q, s), *R.product(x8, q, None, None, None, ws, s))
    xs1 = torch.full((), 0.5, device="cuda").expand(m)
    R.check_product(fd.linear_fp8(wide[:, :k], xs1, q, s), *R.product(wide[:, :k], q, None, None, None, xs1, s))


def test_product_empty():
    g = gen(9)
    w, bias = rn(g, 24, 16), rn(g, 24)
    assert fd.linear_act(torch.empty(0, 16, device="cuda", dtype=BF), w).shape == (0, 24)
    assert fd.linear_act(torch.empty(2, 0, 16, device="cuda", dtype=BF), w, row_add=bias).shape == (2, 0, 24)
    assert fd.linear_act(rn(g, 5, 16), w[:0]).shape == (5, 0)
    # no inner width: the epilogue of a zero sum
    y = fd.linear_act(torch.empty(5, 0, device="cuda", dtype=BF), w[:, :0], bias)
    assert torch.equal(y, bias.expand(5, 24))


@pytest.mark.parametrize("m", [1, 20, 200, 600])
def test_product_not_finite_rows(m):
    """A NaN or an infinity stays in its own row of the output, padding reads as zero."""
    g = gen(m)
    n, k = 200, 328
    x, w = rn(g, m + 2, k), rn(g, n + 2, k, scale=k ** -0.5)
    x[0], x[-1], w[0], w[-1] = float("nan"), float("inf"), float("nan"), float("inf")
    x, w = x[1:-1], w[1:-1]  # neighbours in memory are not finite
    R.check_product(fd.linear_act(x, w), *R.product(x, w, None, None, None))
    x = x.clone()
    x[m // 2, 5] = float("nan")
    y = fd.linear_act(x, w, activation="relu")
    assert y[m // 2].isnan().all() and y.isnan().sum() == n


def test_large_magnitudes_saturate_as_the_type_does():
    x = torch.full((2, 64), 200.0, device="cuda", dtype=F16)
    w = torch.full((8, 64), 200.0, device="cuda", dtype=F16)
    assert fd.linear_act(x, w).isinf().all()  # 2.56e6 is beyond f16
    want = torch.tensor(2.56e6).to(BF).item()
    assert (fd.linear_act(x.to(BF), w.to(BF)) == want).all()
    q = torch.full((2, 4096), 448.0, device="cuda").to(R.E4M3)
    one = torch.ones(2, device="cuda")
    y = fd.linear_fp8(q, one, q, one)
    assert torch.equal(y.float(), torch.full((2, 2), 448.0 * 448 * 4096, device="cuda").to(BF).float())


# ------------------------------------------------------------------ the MLP and the operators together
def mlp_weights(g, h, i):
    wgu, sgu = fd.quantize_fp8(rn(g, 2 * i, h, scale=h ** -0.5))
    wd, sd = fd.quantize_fp8(rn(g, h, i, scale=i ** -0.5))
    return wgu, sgu, wd, sd


def mlp_steps(x, nw, wgu, sgu, wd, sd, eps):
    q, s = fd.rms_norm_fp8(x, nw, eps)
    gate, up = fd.linear_fp8(q, s, wgu, sgu, out_dtype=x.dtype).chunk(2, dim=-1)
    q, s = fd.swiglu_fp8(gate, up)
    return fd.linear_fp8(q, s, wd, sd, row_add=x, out_dtype=x.dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,h,i", [(1, 512, 1024), (3, 136, 200), (7, 100, 37), (16, 1024, 2048), (45, 256, 336),
                                   (300, 512, 640), (1100, 384, 512)])
def test_mlp(m, h, i, dtype):
    """One call gives the bits of the four operators, whose values are within
    the stages' bounds of the 64-bit form."""
    g = gen(m)
    x, nw = rn(g, m, h, dtype=dtype), rn(g, h, dtype=F32)
    weights = mlp_weights(g, h, i)
    y = fd.post_attn_mlp_fp8(x, nw, *weights, 1e-5)
    assert torch.equal(y, mlp_steps(x, nw, *weights, 1e-5))
    assert torch.equal(fd.post_attn_mlp_fp8(x.view(1, m, h), nw, *weights, 1e-5).view(m, h), y)
    # the MLP's own part against the block on the dequantised weights: the two
    # quantisations of activations move it by at most 2^-4 relative each
    # per element, in random directions
    wgu, sgu, wd, sd = (t.double() for t in weights)
    gu = R.rms(x, nw, 1e-5) @ (wgu * sgu[:, None]).T
    ref = R.swiglu(gu[:, :i], gu[:, i:]) @ (wd * sd[:, None]).T
    off = (y.double() - x.double() - ref).norm() / ref.norm()
    assert off < 2 ** -4 + 2 ** -4, float(off)


def test_layer_chain():
    """A decode layer's tail as it is used: attention output to 8 bits, output
    projection onto the residual stream, norm, MLP products, in place."""
    g = gen(5)
    m, h, i = 4, 512, 768
    attn, stream = rn(g, m, h), rn(g, m, h, scale=2.0)
    wo, so = fd.quantize_fp8(rn(g, h, h, scale=h ** -0.5))
    nw = rn(g, h, dtype=F32)
    wgu, sgu, wd, sd = mlp_weights(g, h, i)
    q, s = fd.quantize_fp8(attn)
    o = fd.linear_fp8(q, s, wo, so)
    R.check_product(o, *R.product(q, wo, None, None, None, s, so))
    before = stream.clone()
    q, s, _ = fd.add_rms_norm_fp8(o, stream, nw, 1e-5, residual_out=stream)
    assert torch.equal(stream, (o.float() + before.float()).to(BF))
    R.check_rows8(q, s, R.rms(o, nw, 1e-5, before))
    gu = fd.linear_fp8(q, s, wgu, sgu)
    R.check_product(gu, *R.product(q, wgu, None, None, None, s, sgu))
    q, s = fd.swiglu_fp8(*gu.chunk(2, dim=-1))
    R.check_rows8(q, s, R.swiglu(*gu.chunk(2, dim=-1)))
    ref = R.product(q, wd, None, None, stream.clone(), s, sd)
    fd.linear_fp8(q, s, wd, sd, row_add=stream, out=stream)
    R.check_product(stream, *ref)


def test_offsets_beyond_31_bits():
    """Rows whose elements lie past 2^31: the last ones are right."""
    g = gen(13)
    m, n = 66000, 32768
    x = torch.zeros(m, n, device="cuda", dtype=BF)
    x[-3:] = rn(g, 3, n)
    q, s = fd.quantize_fp8(x)
    R.check_rows8(q[-3:], s[-3:], x[-3:].double())
    del q, x
    x, w = rn(g, m, 64), rn(g, n, 64, scale=0.125)
    y = fd.linear_act(x, w)
    R.check_product(y[-300:], *R.product(x[-300:], w, None, None, None))


def test_product_becomes_the_next_products_weight():
    """linear_decode streams its weight before it waits for the kernel before
    it; a product's output is finished by then."""
    g = gen(14)
    for rows in (48, 512):
        a, b, x = rn(g, rows, 2048), rn(g, 2048, 2048, scale=0.02), rn(g, 2, 2048)
        w = torch.zeros(rows, 2048, device="cuda", dtype=BF)
        ref_w = fd.linear_act(a, b)
        torch.cuda.synchronize()
        ref = fd.linear_decode(x, ref_w)
        for _ in range(5):
            w.zero_()
            fd.linear_act(a, b, out=w)
            assert torch.equal(fd.linear_decode(x, w), ref)


def test_weights_quantised_just_before_use():
    """A product launched behind the kernel that writes its weights waits for it."""
    g = gen(6)
    w = rn(g, 4096, 4096, scale=1 / 64)
    x, xs = weight8(g, 3, 4096)
    wq = torch.zeros(4096, 4096, device="cuda", dtype=R.E4M3)
    ws = torch.zeros(4096, device="cuda")
    q0, s0 = fd.quantize_fp8(w)
    ref = fd.linear_fp8(x, xs, q0, s0)
    torch.cuda.synchronize()
    for _ in range(5):
        wq.view(torch.uint8).zero_()
        fd.quantize_fp8(w, out=wq, scale_out=ws)
        assert torch.equal(fd.linear_fp8(x, xs, wq, ws), ref)


def test_repeat_gives_the_same_bits():
    g = gen(7)
    for m, n, k in ((1, 4096, 4096), (24, 1000, 4096), (700, 1024, 2048)):
        x, xs = weight8(g, m, k)
        w, ws = weight8(g, n, k)
        first = fd.linear_fp8(x, xs, w, ws)
        for _ in range(5):
            assert torch.equal(fd.linear_fp8(x, xs, w, ws), first)


def test_streams_and_graphs():
    """Two captured graphs of the block replayed at once on two streams, while
    a third stream calls it, each with its own input."""
    g = gen(8)
    h, i = 512, 1024
    nw = rn(g, h, dtype=F32)
    weights = mlp_weights(g, h, i)
    xs = [rn(g, m, h) for m in (1, 9, 320)]
    want = [fd.post_attn_mlp_fp8(x, nw, *weights, 1e-5) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fd.post_attn_mlp_fp8(x, nw, *weights, 1e-5))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = fd.post_attn_mlp_fp8(xs[2], nw, *weights, 1e-5)
        torch.cuda.synchronize()
        for out, ref in zip([*outs, third], want):
            assert torch.equal(out, ref)


def test_no_wait_expired():
    from fused_decode_b200 import kernels as K

    assert K.product_status() == 0


def test_compiled_and_python_paths_agree(monkeypatch):
    """The compiled dispatch and the Python path behind it give the same bits."""
    from fused_decode_b200 import ops_fp8

    g = gen(11)
    x, r, w = rn(g, 3, 4, 256), rn(g, 3, 4, 256), rn(g, 256, dtype=F32)
    wl, bias = rn(g, 320, 256, scale=0.06), rn(g, 320)
    res = rn(g, 3, 4, 320)
    weights = mlp_weights(g, 256, 512)

    def bits(t):
        return t.view(torch.uint8) if t.dtype == R.E4M3 else t

    def all_calls():
        q, s = fd.quantize_fp8(x)
        wq, ws = fd.quantize_fp8(wl)
        outs = [q, s, *fd.rms_norm_fp8(x, w), *fd.add_rms_norm_fp8(x, r, w), *fd.swiglu_fp8(x, r)]
        outs += [fd.linear_act(x, wl, bias, activation="gelu", row_add=res), fd.linear_act(x, wl, row_add=bias)]
        outs += [fd.linear_fp8(q, s, wq, ws, bias, activation="silu", row_add=res)]
        outs += [fd.linear_fp8(q, s, wq, ws, out_dtype=F16), fd.post_attn_mlp_fp8(x, w, *weights, 1e-5)]
        return [bits(t) for t in outs]

    assert ops_fp8._fast().linear_act(x, wl, bias, "gelu", res, None) is not None
    compiled = all_calls()
    monkeypatch.setattr(ops_fp8, "_fast", lambda: None)
    python = all_calls()
    assert all(torch.equal(a, b) for a, b in zip(compiled, python, strict=True))


def test_custom_ops():
    ops = torch.ops.fused_decode_b200
    g = gen(12)
    x, w = rn(g, 5, 128), rn(g, 96, 128, scale=0.09)
    wq, ws = ops.quantize_fp8(w)
    q, s = ops.rms_norm_fp8(x, torch.ones(128, device="cuda"), 1e-5)
    assert torch.equal(ops.linear_fp8(q, s, wq, ws, None, "silu", None, F16),
                       fd.linear_fp8(q, s, wq, ws, activation="silu", out_dtype=F16))
    assert torch.equal(ops.linear_act(x, w, None, None, None), fd.linear_act(x, w))
    compiled = torch.compile(lambda t: ops.linear_act(t, w, None, "relu", None), fullgraph=True, backend="eager")
    assert torch.equal(compiled(x), fd.linear_act(x, w, activation="relu"))


def test_cuda_refusals():
    """What the checks let through on any device and refuse on a GPU."""
    x = torch.zeros(2, 16, device="cuda", dtype=BF)
    with pytest.raises(ValueError, match="weight is on cpu"):
        fd.linear_act(x, torch.zeros(4, 16, dtype=BF))
    with pytest.raises(ValueError, match="residual is on cpu"):
        fd.add_rms_norm_fp8(x, x.cpu(), torch.ones(16, device="cuda"))
    with pytest.raises(ValueError, match="out must be contiguous"):
        fd.linear_act(x, x, out=torch.zeros(2, 4, device="cuda", dtype=BF)[:, ::2])

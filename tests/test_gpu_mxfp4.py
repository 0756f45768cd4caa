"""Microscaled 4-bit quantization, products and gradients against the formulas
in 64 bits.  Codes, scales and values are compared bit for bit; sums within
the bound of float32 additions of exact products (_mxfp4.limit)."""
import pytest
import torch

from tests import _mxfp4 as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _data(shape, dtype, seed=0):
    g = _gen(seed)
    x = torch.randn(shape, generator=g)
    x[torch.rand(shape, generator=g) < 0.02] *= 30
    return x.to(dtype)


def _same_bits(a, b):
    view = {4: torch.int32, 2: torch.int16}[a.element_size()]
    nan = torch.isnan(a) & torch.isnan(b)
    return torch.equal(a.view(view).masked_fill(nan, 0), b.view(view).masked_fill(nan, 0))


# ---------------------------------------------------------------- quantize, dequantize
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 100), (2, 3, 64), (16, 4096), (33, 2080), (40,),
                                   (4100, 1056), (0, 64), (4, 0)])
def test_codes_scales_and_values(shape, dtype):
    import qtpytorch_amd as qa
    x = _data(shape, dtype)
    q = qa.mxfp4_quantize(x.cuda())
    codes, scales = R.pack(x) if x.numel() else (q.codes.cpu(), q.scales.cpu())
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    ref = R.unpack(codes, scales, shape[-1])
    for out in FLOATS:
        y = q.dequantize(out)
        assert y.dtype == out and _same_bits(y.cpu(), ref.to(out))


@pytest.mark.parametrize("dtype", FLOATS)
def test_ties_saturation_and_zeros(dtype):
    """Each midpoint, a value either side of it, the largest value and signed zeros."""
    import qtpytorch_amd as qa
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    row = [4.0, 7.5, -7.5, 0.0, -0.0, 6.0, -6.0]
    for m in mids:
        row += [m, -m, m * (1 - 2 ** -7), m * (1 + 2 ** -7)]
    row += [5.5] * (64 - len(row))
    x = torch.tensor([row, [0.0] * 32 + [-0.0] * 32]).to(dtype)
    q = qa.mxfp4_quantize(x.cuda())
    codes, scales = R.pack(x)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)


@pytest.mark.parametrize("exponent", [-149, -140, -130, -127, -126, -125, -124, -100, 0, 100, 124, 127])
def test_range_of_float32(exponent):
    import qtpytorch_amd as qa
    x = torch.ldexp(1 + torch.rand(3, 64, generator=_gen(1)).double() * 0.99, torch.tensor(exponent)).float()
    x[:, 1::2] *= -0.5
    q = qa.mxfp4_quantize(x.cuda())
    codes, scales = R.pack(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    assert _same_bits(q.dequantize().cpu(), R.unpack(codes, scales, 64).float())


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_non_number_is_nan(dtype, bad):
    import qtpytorch_amd as qa
    x = _data((4, 96), dtype)
    x[2, 40] = bad
    q = qa.mxfp4_quantize(x.cuda())
    assert q.scales[2].tolist()[1] == 255 and int(q.codes[2, 16:32].max()) == 0
    y = q.dequantize().cpu()
    assert bool(torch.isnan(y[2, 32:64]).all()) and int(torch.isnan(y).sum()) == 32
    good, gs = R.pack(x[[0, 1, 3]])
    assert torch.equal(q.codes[[0, 1, 3]].cpu(), good) and torch.equal(q.scales[[0, 1, 3]].cpu(), gs)


def test_every_code_and_scale_dequantizes():
    import qtpytorch_amd as qa
    codes = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(256, 16)
    codes = codes.roll(1, 1)
    codes[:, :8] = torch.arange(8, dtype=torch.uint8) * 0x22 + 0x10
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1)
    q = qa.mxfp4_tensor(codes.cuda(), scales.cuda(), (256, 32))
    ref = R.unpack(codes, scales, 32)
    for out in FLOATS:
        assert _same_bits(q.dequantize(out).cpu(), ref.to(out))


def test_rows_apart_offsets_and_transposes():
    import qtpytorch_amd as qa
    big = _data((9, 200), torch.bfloat16).cuda()
    for x in (big[:, :96], big[1::2, 3:99], big[:, 7:], big.t(), big[2:3, :50], big.float()[:, 1:34]):
        codes, scales = R.pack(x.cpu())
        q = qa.mxfp4_quantize(x)
        assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)


# ---------------------------------------------------------------- products
def _operands(M, N, K, seed=0):
    import qtpytorch_amd as qa
    a, b = _data((M, K), torch.float32, seed), _data((N, K), torch.float32, seed + 1) * 0.05
    return a, b, qa.mxfp4_quantize(a.cuda()), qa.mxfp4_quantize(b.cuda())


SHAPES = [(1, 1, 1), (1, 17, 33), (3, 64, 32), (16, 48, 128), (16, 512, 4096), (17, 100, 96), (31, 257, 500), (33, 33, 64),
          (64, 64, 128), (65, 70, 160), (100, 300, 1000), (128, 128, 256), (129, 255, 2080), (256, 256, 512),
          (257, 513, 544), (300, 16, 1024), (512, 768, 1056), (5, 2000, 8224), (40, 640, 2048), (48, 96, 12000)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("out", FLOATS)
def test_product(shape, out):
    import qtpytorch_amd as qa
    M, N, K = shape
    a, b, qa_, qb = _operands(M, N, K)
    y = qa.mxfp4_matmul(qa_, qb, out_dtype=out)
    ra, rb = R.rounded(a), R.rounded(b)
    assert y.shape == (M, N) and y.dtype == out
    R.assert_close(y, ra @ rb.t(), ra.abs() @ rb.abs().t(), K / 32 + 2)


@pytest.mark.parametrize("shape", [(33, 1, 1024), (34, 8208, 512), (49, 300, 4128), (64, 33, 8224), (64, 8193, 96), (65, 5, 3000),
                                   (400, 1, 2080), (1000, 63, 96), (65, 8193, 64)])
def test_product_of_33_to_64_rows_and_of_narrow_weights(shape):
    test_product(shape, torch.float32)
    test_product(shape, torch.bfloat16)


@pytest.mark.parametrize("shape", [(65, 3, 64), (100, 4, 64), (65, 1, 256), (70, 1, 200), (3000, 3900, 96), (129, 130, 250), (300, 257, 288),
                                   (129, 400, 3328), (300, 300, 12000), (66, 129, 2049)])
def test_product_of_few_stages(shape):
    test_product(shape, torch.float32)
    test_product(shape, torch.float16)


@pytest.mark.parametrize("shape", [(70, 40, 64), (130, 129, 288), (200, 70, 480), (1100, 1030, 5000)])
def test_nan_of_a_row_reaches_no_other(shape):
    """First and last blocks of rows next to each other, whose scale bytes are read together."""
    import qtpytorch_amd as qa
    M, N, K = shape
    a, b, _, _ = _operands(M, N, K)
    for m in (1, M // 2, M - 1):
        a[m, 0] = float("nan")
    for n in (2, N // 2, N - 1):
        b[n, 0] = float("inf")
        b[n, K - 1] = float("nan")
    y = qa.mxfp4_matmul(qa.mxfp4_quantize(a.cuda()), qa.mxfp4_quantize(b.cuda()), out_dtype=torch.float32)
    want = torch.zeros(M, N, dtype=torch.bool)
    want[[1, M // 2, M - 1]] = True
    want[:, [2, N // 2, N - 1]] = True
    assert torch.equal(torch.isnan(y.cpu()), want)


def test_product_of_more_columns_than_a_tile_can_store_by_32_bits():
    import qtpytorch_amd as qa
    M, N, K = 65, (1 << 21) + 3, 64
    a, b = _data((M, K), torch.float32, 3), _data((N, K), torch.float32, 4)
    y = qa.mxfp4_matmul(qa.mxfp4_quantize(a.cuda()), qa.mxfp4_quantize(b.cuda()), out_dtype=torch.float32)
    ra = R.rounded(a)
    for lo in (0, N // 2, N - 301):
        rb = R.rounded(b[lo:lo + 301])
        R.assert_close(y[:, lo:lo + 301], ra @ rb.t(), ra.abs() @ rb.abs().t(), K / 32 + 2)


@pytest.mark.parametrize("shape", [(16, 64, 128), (1, 48, 160), (70, 130, 320), (300, 300, 512)])
def test_product_with_bias_and_leading_dimensions(shape):
    import qtpytorch_amd as qa
    M, N, K = shape
    a, b, _, qb = _operands(M, N, K)
    bias = torch.randn(N, generator=_gen(5)).to(torch.bfloat16)
    y = qa.mxfp4_matmul(qa.mxfp4_quantize(a.view(1, M, K).cuda()), qb, bias.cuda(), torch.float32)
    ra, rb = R.rounded(a), R.rounded(b)
    assert y.shape == (1, M, N)
    R.assert_close(y[0], ra @ rb.t() + bias.double(), ra.abs() @ rb.abs().t() + bias.double().abs(), K / 32 + 3)


@pytest.mark.parametrize("shape", [(16, 64, 256), (130, 70, 320), (300, 520, 1024)])
def test_product_with_nan_blocks(shape):
    import qtpytorch_amd as qa
    M, N, K = shape
    a, b, _, _ = _operands(M, N, K)
    a[M // 2, K - 1] = float("nan")
    b[N - 1, 0] = float("inf")
    y = qa.mxfp4_matmul(qa.mxfp4_quantize(a.cuda()), qa.mxfp4_quantize(b.cuda()), out_dtype=torch.float32)
    nan = torch.isnan(y.cpu())
    want = torch.zeros(M, N, dtype=torch.bool)
    want[M // 2] = True
    want[:, N - 1] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("shape", [(4, 40, 96), (200, 300, 640)])
def test_product_of_a_wide_range_of_scales(shape):
    """Scales from 2^-40 to 2^40: exact products, sums within the bound of their own mass."""
    import qtpytorch_amd as qa
    M, N, K = shape
    a, b, _, _ = _operands(M, N, K)
    a *= torch.exp2(torch.randint(-20, 21, (M, 1), generator=_gen(7)).float())
    b *= torch.exp2(torch.randint(-20, 21, (N, K // 32), generator=_gen(8)).float()).repeat_interleave(32, 1)
    y = qa.mxfp4_matmul(qa.mxfp4_quantize(a.cuda()), qa.mxfp4_quantize(b.cuda()), out_dtype=torch.float32)
    ra, rb = R.rounded(a), R.rounded(b)
    R.assert_close(y, ra @ rb.t(), ra.abs() @ rb.abs().t(), K / 32 + 2)


@pytest.mark.parametrize("m", [0, 1, 5])
@pytest.mark.parametrize("k", [0, 64])
def test_product_of_empty_operands(m, k):
    import qtpytorch_amd as qa
    a, b = torch.randn(m, k), torch.randn(7, k)
    y = qa.mxfp4_matmul(qa.mxfp4_quantize(a.cuda()), qa.mxfp4_quantize(b.cuda()), torch.ones(7).cuda(), torch.float32)
    assert y.shape == (m, 7)
    R.assert_close(y, R.rounded(a) @ R.rounded(b).t() + 1 if k else torch.ones(m, 7, dtype=torch.float64),
                   torch.full((m, 7), 100.0, dtype=torch.float64), 8)


def test_product_repeats_bit_for_bit_on_another_stream():
    import qtpytorch_amd as qa
    for shape in ((8, 512, 8192), (200, 300, 4096), (1024, 1024, 1024)):
        _, _, a, b = _operands(*shape)
        want = qa.mxfp4_matmul(a, b, out_dtype=torch.float32)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [qa.mxfp4_matmul(a, b, out_dtype=torch.float32) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(g, want) for g in got)


# ---------------------------------------------------------------- linear
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 64, 128), (1, 200, 4096), (7, 48, 1000), (16, 256, 8192), (16, 100, 33), (20, 96, 512),
                                   (40, 130, 2080), (150, 257, 544), (260, 512, 1024)])
def test_linear(shape, dtype):
    import qtpytorch_amd as qa
    M, N, K = shape
    x, w = _data((M, K), dtype), (_data((N, K), torch.float32, 1) * 0.05)
    bias = torch.randn(N, generator=_gen(2))
    rx, rw = R.rounded(x), R.rounded(w)
    ref, mass = rx @ rw.t() + bias.double(), rx.abs() @ rw.abs().t() + bias.double().abs()
    held = qa.mxfp4_quantize(w.cuda())
    y = qa.mxfp4_linear(x.cuda(), held, bias.cuda())
    assert y.dtype == dtype
    R.assert_close(y, ref, mass, K / 32 + 3)
    R.assert_close(qa.mxfp4_linear(x.cuda(), w.cuda(), bias.cuda()), ref, mass, K / 32 + 3)
    R.assert_close(qa.mxfp4_linear(x.cuda().view(M, 1, K), held)[:, 0], rx @ rw.t(), mass, K / 32 + 2)


@pytest.mark.parametrize("m", [1, 9])
def test_linear_of_strided_rows(m):
    import qtpytorch_amd as qa
    big, w = _data((2 * m, 300), torch.bfloat16), _data((40, 256), torch.float32, 1)
    x = big.cuda()[::2, 5:261]
    rx, rw = R.rounded(x), R.rounded(w)
    R.assert_close(qa.mxfp4_linear(x, qa.mxfp4_quantize(w.cuda())), rx @ rw.t(), rx.abs() @ rw.abs().t(), 256 / 32 + 2)


@pytest.mark.parametrize("m", [3, 70])
def test_linear_of_nan_activations(m):
    import qtpytorch_amd as qa
    x, w = _data((m, 96), torch.bfloat16), _data((40, 96), torch.float32, 1)
    x[1, 50] = float("nan")
    y = qa.mxfp4_linear(x.cuda(), qa.mxfp4_quantize(w.cuda())).cpu()
    assert bool(torch.isnan(y[1]).all()) and int(torch.isnan(y).sum()) == 40


# ---------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 17, 40), (16, 64, 128), (33, 70, 96), (64, 200, 333), (130, 129, 257),
                                   (300, 260, 512), (513, 130, 320)])
def test_gradients(shape, dtype):
    import qtpytorch_amd as qa
    M, N, K = shape
    x, w, dy = _data((M, K), dtype), (_data((N, K), torch.float32, 1) * 0.05).to(dtype), _data((M, N), dtype, 2)
    xg, wg, bg = x.cuda().requires_grad_(), w.cuda().requires_grad_(), torch.zeros(N, device="cuda", requires_grad=True)
    y = qa.mxfp4_linear(xg, wg, bg)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy.cuda())
    rx, rw, d = R.rounded(x), R.rounded(w), dy.double()
    R.assert_close(y, rx @ rw.t(), rx.abs() @ rw.abs().t(), K / 32 + 3)
    # f16 and f32 gradients enter as two and three exact terms
    R.assert_close(dx, d @ rw, d.abs() @ rw.abs(), 3 * (N / 8 + 2))
    R.assert_close(dw, d.t() @ rx, d.abs().t() @ rx.abs(), 3 * (M / 8 + 2))
    R.assert_close(db, d.sum(0), d.abs().sum(0), 3 * (M / 8 + 2))
    assert dx.dtype == dtype and dw.dtype == dtype and db.dtype == torch.float32
    # a weight held packed has the same output and input gradient
    yh = qa.mxfp4_linear(xg, qa.mxfp4_quantize(w.cuda()))
    (dxh,) = torch.autograd.grad(yh, xg, dy.cuda())
    assert torch.equal(dxh, dx)


def test_gradient_is_the_slope_between_representable_points():
    """Where x moves from one grid value to the next the product moves by exactly the gradient's entry."""
    import qtpytorch_amd as qa
    M, N, K = 3, 20, 64
    x = torch.full((M, K), 2.0)
    x[:, ::32] = 4.0  # the scale of every block stays 2^0
    w = R.rounded(_data((N, K), torch.float32, 1)).float().cuda()
    dy = torch.randint(-3, 4, (M, N), generator=_gen(3)).float().cuda()
    xg = x.cuda().requires_grad_()
    y = qa.mxfp4_linear(xg, w)
    (dx,) = torch.autograd.grad(y, xg, dy)
    for m, k in ((0, 1), (1, 40), (2, 63)):
        moved = x.clone()
        moved[m, k] = 3.0
        step = (qa.mxfp4_linear(moved.cuda(), w).double() - y.detach().double()).mul(dy.double()).sum()
        assert abs(float(step) - float(dx[m, k])) <= 2e-5 * (1 + abs(float(step)))


def test_gradient_of_infinite_and_nan_entries():
    import qtpytorch_amd as qa
    w = _data((20, 64), torch.float32, 1)
    w[:, 3] = 0.5
    dy = _data((4, 20), torch.float32, 2)
    dy[1, 4], dy[2, 5] = float("inf"), float("nan")
    x = _data((4, 64), torch.float32).cuda().requires_grad_()
    (dx,) = torch.autograd.grad(qa.mxfp4_linear(x, qa.mxfp4_quantize(w.cuda())), x, dy.cuda())
    ref = dy.double() @ R.rounded(w)
    dx = dx.cpu()
    assert torch.equal(torch.isnan(dx), torch.isnan(ref)) and torch.equal(torch.isinf(dx), torch.isinf(ref))
    assert torch.isfinite(dx[[0, 3]]).all()


def test_gradient_of_a_strided_output_gradient():
    import qtpytorch_amd as qa
    x, w = _data((10, 96), torch.bfloat16).cuda().requires_grad_(), _data((24, 96), torch.float32, 1)
    held = qa.mxfp4_quantize(w.cuda())
    dy = _data((24, 10), torch.bfloat16, 2).cuda().t()
    (dx,) = torch.autograd.grad(qa.mxfp4_linear(x, held), x, dy)
    d, rw = dy.double().cpu(), R.rounded(w)
    R.assert_close(dx, d @ rw, d.abs() @ rw.abs(), 8)
    (dx,) = torch.autograd.grad(qa.mxfp4_linear(x, held).sum(), x)  # a broadcast gradient of ones
    R.assert_close(dx, rw.sum(0).expand(10, 96), rw.abs().sum(0).expand(10, 96), 8)


def test_product_of_views_that_start_anywhere():
    """Codes and scales at odd addresses of larger buffers, as a loaded checkpoint has them."""
    import qtpytorch_amd as qa
    for M, N, K in ((9, 100, 544), (40, 70, 96), (300, 200, 1056)):
        a, b, qa_, qb = _operands(M, N, K)
        held = []
        for q in (qa_, qb):
            codes, scales = torch.zeros(q.codes.numel() + 3, dtype=torch.uint8).cuda(), \
                torch.zeros(q.scales.numel() + 1, dtype=torch.uint8).cuda()
            codes[3:].copy_(q.codes.view(-1))
            scales[1:].copy_(q.scales.view(-1))
            held.append(qa.mxfp4_tensor(codes[3:].view(q.codes.shape), scales[1:].view(q.scales.shape), q.shape))
        want = qa.mxfp4_matmul(qa_, qb, out_dtype=torch.float32)
        assert torch.equal(qa.mxfp4_matmul(*held, out_dtype=torch.float32), want)
        y = torch.randn(M, N, generator=_gen(3)).cuda()
        x = a.cuda().requires_grad_()
        d0, = torch.autograd.grad(qa.mxfp4_linear(x, qb), x, y)
        d1, = torch.autograd.grad(qa.mxfp4_linear(x, held[1]), x, y)
        assert torch.equal(d0, d1)


def test_tensor_moves_and_sizes():
    import qtpytorch_amd as qa
    q = qa.mxfp4_quantize(torch.randn(6, 70).cuda())
    assert q.shape == (6, 70) and q.dim() == 2 and q.nbytes == 6 * 3 * 17 and "6, 70" in repr(q)
    back = q.to("cpu").to("cuda")
    assert torch.equal(back.dequantize(), q.dequantize())
    with pytest.raises(qa._lib.MXKError):
        q.to("cpu").dequantize()


# ---------------------------------------------------------------- offsets past 32 bits
def _random_packed(shape, seed):
    """A packed tensor of random codes and scales from 2^-7 to 2^7, made on the GPU."""
    import qtpytorch_amd as qa
    g = torch.Generator(device="cuda").manual_seed(seed)
    kb = -(-shape[-1] // 32)
    codes = torch.randint(0, 256, (*shape[:-1], 16 * kb), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(120, 135, (*shape[:-1], kb), dtype=torch.uint8, device="cuda", generator=g)
    return qa.mxfp4_tensor(codes, scales, shape)


def test_quantize_of_more_than_2_31_elements():
    import qtpytorch_amd as qa
    rows, cols = 70001, 32768 + 64
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    q = qa.mxfp4_quantize(x)
    y = q.dequantize(torch.bfloat16)
    for lo in (0, 65530, rows - 3):
        part = qa.mxfp4_quantize(x[lo:lo + 3])
        assert torch.equal(q.codes[lo:lo + 3], part.codes) and torch.equal(q.scales[lo:lo + 3], part.scales)
        assert torch.equal(y[lo:lo + 3], part.dequantize(torch.bfloat16))


@pytest.mark.parametrize("rows", [3, 40, 400])
def test_experts_of_more_than_2_31_bytes(rows):
    """The last of many large experts: its product and its input's gradient are those of its weight alone."""
    import qtpytorch_amd as qa
    E, N, K = 40, 16384, 8192
    w = _random_packed((E, N, K), 1)
    assert w.codes.numel() > 1 << 31
    ids = torch.full((rows, 1), E - 1, device="cuda")
    plan = qa.expert_sort(ids, E)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, K, device="cuda", generator=g).bfloat16().requires_grad_()
    alone = qa.mxfp4_tensor(w.codes[-1], w.scales[-1], (N, K))
    y, z = qa.expert_linear(x, w, plan, gather=True), qa.mxfp4_linear(x, alone)
    dy = torch.randn(rows, N, device="cuda", generator=g).bfloat16()
    # the kernels may differ in the order of their sums
    assert float((y.detach().double() - z.detach().double()).norm() / z.detach().double().norm()) < 1e-3
    dx, dz = torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(z, x, dy)[0]
    assert float((dx.double() - dz.double()).norm() / dz.double().norm()) < 1e-3


# ---------------------------------------------------------------- refusals
def test_refusals():
    import qtpytorch_amd as qa
    x = torch.randn(4, 64, device="cuda")
    q = qa.mxfp4_quantize(x)
    with pytest.raises(ValueError):
        qa.mxfp4_quantize(torch.tensor(1.0, device="cuda"))
    with pytest.raises(ValueError):
        qa.mxfp4_matmul(q, qa.mxfp4_quantize(torch.randn(4, 96, device="cuda")))
    with pytest.raises(TypeError):
        qa.mxfp4_matmul(q, x)
    with pytest.raises(ValueError):
        qa.mxfp4_matmul(q, q, torch.zeros(5, device="cuda"))
    with pytest.raises(qa._lib.MXKError):
        qa.mxfp4_matmul(q, q, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        qa.mxfp4_linear(x[:, :32], q)
    with pytest.raises(TypeError):
        qa.mxfp4_linear(x.double(), q)
    with pytest.raises(ValueError):
        qa.mxfp4_tensor(q.codes, q.scales, (4, 128))
    with pytest.raises(TypeError):
        qa.mxfp4_tensor(q.codes.int(), q.scales, (4, 64))
    with pytest.raises(qa._lib.MXKError):
        qa.mxfp4_quantize(x.cpu())
    with pytest.raises(qa._lib.MXKError):
        q.dequantize(torch.float64)
    lib = qa._lib.lib()
    assert lib.mxk_mxfp4_quantize(0, 0, 4, 64, 64, 0, 0, 0) == qa._lib.MXK_EINVAL
    assert lib.mxk_mxfp4_quantize(x.data_ptr(), 9, 4, 64, 64, q.codes.data_ptr(), q.scales.data_ptr(), 0) == \
        qa._lib.MXK_EINVAL
    assert lib.mxk_mxfp4_dequantize(q.codes.data_ptr() + 1, q.scales.data_ptr(), 4, 64, 0, x.data_ptr(), 0) == \
        qa._lib.MXK_EINVAL

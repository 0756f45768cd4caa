"""The tile kernels where large products and training steps run them: workgroups
that take a second and a third tile, several stages of K, ragged sides, large tiles
of every form.  References are products of the dequantized operands (which are
tested bit for bit elsewhere) in 64 bits on the GPU."""
import pytest
import torch

from tests import _mxfp4 as R
from tests.test_gpu_experts import _gen, _ids

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _up(a, b):
    return -(-a // b)


def _rand(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, device="cuda", generator=g) * scale
    x[torch.rand(shape, device="cuda", generator=g) < 0.01] *= 20
    return x


def _values(x):
    """x after packing, in 64 bits on the GPU."""
    import qtpytorch_amd as qa
    return qa.mxfp4_quantize(x).dequantize().double()


def _close(got, ref, mass, terms):
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), "NaNs are not where the formula has them"
    over = ((got.double() - ref).abs() - R.limit(got.dtype, ref, mass, terms)).masked_fill(nan, -1.0)
    assert got.numel() == 0 or float(over.max()) <= 0, f"error {float(over.max()):.3g} above the bound"


def _same(run, want, times=3):
    """A race between a tile's stages would not give the same bits every time."""
    for _ in range(times):
        assert torch.equal(run().nan_to_num(77.0), want.nan_to_num(77.0))


# ---------------------------------------------------------------- dense products
def _dense(M, N, K, out, biased, nans=False):
    import qtpytorch_amd as qa
    a, b = _rand(M, K), _rand(N, K, seed=1, scale=0.05)
    if nans:  # first and last blocks, whose scales neighbours' lie beside
        a[[0, M // 2, M - 1], [0, K - 1, K // 2]] = float("nan")
        b[[1, N // 2, N - 1], [K - 1, 0, 0]] = float("inf")
    bias = torch.randn(N, generator=_gen(2)).cuda() if biased else None
    pa, pb = qa.mxfp4_quantize(a), qa.mxfp4_quantize(b)
    y = qa.mxfp4_matmul(pa, pb, bias, out)
    ra, rb = _values(a), _values(b).t().contiguous()
    ref, mass = ra @ rb, ra.abs() @ rb.abs()
    if biased:
        ref, mass = ref + bias.double(), mass + bias.double().abs()
    _close(y, ref, mass, K / 32 + 3)
    _same(lambda: qa.mxfp4_matmul(pa, pb, bias, out), y)


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("M,N,K", [(5701, 5704, 1000), (5633, 5701, 520), (4353, 6000, 256), (4400, 4402, 2400)])
def test_large_tiles_in_turn(M, N, K, biased, out):
    """More tiles of 256 x 256 than workgroups, two and three to one; results that leave in whole pieces and not."""
    assert _up(M, 256) * _up(N, 256) > _cus()
    _dense(M, N, K, out, biased)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_large_tiles_in_turn_with_nans(out):
    _dense(4801, 4792, 800, out, False, nans=True)


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("M,N,K", [(2900, 2944, 1600), (2817, 2939, 1800), (2900, 2944, 1200), (2945, 2821, 64)])
def test_small_tiles_in_turn(M, N, K, biased, out):
    """Too few tiles of 256, more of 128 than the two a compute unit holds; scales in stage order (the first two) and from
    their rows."""
    assert _up(M, 256) * _up(N, 256) < 192 and _up(M, 128) * _up(N, 128) > 2 * _cus()
    _dense(M, N, K, out, biased)


@pytest.mark.parametrize("K", [1000, 1700])
def test_small_tiles_in_turn_with_nans(K):
    _dense(2900, 2939, K, torch.float32, False, nans=True)


@pytest.mark.parametrize("M,N,K", [(128, 8192, 8192), (129, 3001, 9000), (300, 1100, 12000)])
def test_stages_in_parts(M, N, K):
    _dense(M, N, K, torch.float32, True)
    _dense(M, N, K, torch.bfloat16, False, nans=True)


# ---------------------------------------------------------------- products by expert
def _experts(tokens, top, E, N, K, dtype, gather, biased, dropped, first=0):
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, E + first, skew=0.5, dropped=dropped)
    plan = qa.expert_sort(ids.cuda(), E + first)
    plan = plan._replace(offsets=plan.offsets[first:])
    rows = tokens * top
    x = _rand(tokens if gather else rows, K).to(dtype)
    w = qa.mxfp4_quantize(_rand(E, N, K, seed=1, scale=0.05))
    bias = torch.randn(E, N, generator=_gen(2)).cuda() if biased else None
    y = qa.expert_linear(x, w, plan, bias, gather=gather)
    rx, rw = _values(x), w.dequantize().double()
    offsets = plan.offsets.tolist()
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        a = rx[(plan.order[lo:hi] // top).long()] if gather else rx[lo:hi]
        b = rw[e].t().contiguous()
        ref, mass = a @ b, a.abs() @ b.abs()
        if biased:
            ref, mass = ref + bias[e].double(), mass + bias[e].double().abs()
        _close(y[lo:hi], ref, mass, K / 32 + 3)
    assert not y[:offsets[0]].any() and not y[offsets[-1]:].any()
    _same(lambda: qa.expert_linear(x, w, plan, bias, gather=gather), y)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,E,N,K,biased,dropped,first", [
    (3000, 2, 3, 5704, 600, False, 0.0, 0), (3001, 2, 4, 5701, 520, True, 0.1, 0), (3500, 2, 3, 5632, 256, True, 0.0, 2)])
def test_large_tiles_by_expert(tokens, top, E, N, K, biased, dropped, first, gather, dtype):
    """Uneven experts of more than 128 rows on average over more large tiles than workgroups."""
    assert tokens * top > 128 * E and tokens * top // 256 * _up(N, 256) > _cus()
    _experts(tokens, top, E, N, K, dtype, gather, biased, dropped, first)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,E,N,K,biased,dropped,first", [
    (2000, 2, 40, 2000, 600, False, 0.0, 0), (2001, 2, 40, 2001, 1000, True, 0.1, 0), (1100, 4, 64, 1800, 256, True, 0.0, 3)])
def test_small_tiles_by_expert(tokens, top, E, N, K, biased, dropped, first, gather, dtype):
    """25 to 128 rows an expert: 128-row tiles, more than the two a compute unit holds."""
    assert 24 * E < tokens * top <= 128 * E and E * _up(N, 128) > 2 * _cus()
    _experts(tokens, top, E, N, K, dtype, gather, biased, dropped, first)


@pytest.mark.parametrize("rows", [1000, 5200])
def test_tiles_of_experts_past_2_31_bytes(rows):
    """The last of many large experts on either tile size (more than 24 and more than 128 rows an expert on average)."""
    import qtpytorch_amd as qa
    E, N, K = 40, 16384, 8192
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(120, 135, (E, N, K // 32), dtype=torch.uint8, device="cuda", generator=g)
    w = qa.mxfp4_tensor(codes, scales, (E, N, K))
    assert codes.numel() > 1 << 31 and rows > 24 * E
    plan = qa.expert_sort(torch.full((rows, 1), E - 1, device="cuda"), E)
    x = _rand(rows, K).bfloat16()
    y = qa.expert_linear(x, w, plan, gather=True)
    cols = torch.cat([torch.arange(300), torch.arange(N // 2, N // 2 + 300), torch.arange(N - 300, N)]).cuda()
    rw = qa.mxfp4_tensor(codes[-1][cols], scales[-1][cols], (cols.numel(), K)).dequantize().double().t().contiguous()
    rx = _values(x)
    _close(y[:, cols], rx @ rw, rx.abs() @ rw.abs(), K / 32 + 3)


# ---------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,N,K", [(3300, 3304, 3400), (3301, 3303, 3401), (3329, 3352, 3336)])
def test_gradients_on_large_tiles(M, N, K, dtype):
    """At least 160 tiles of 256 for either gradient, sides that end inside one."""
    import qtpytorch_amd as qa
    assert _up(M, 256) * _up(K, 256) >= 160 and _up(N, 256) * _up(K, 256) >= 160
    x, w = _rand(M, K).to(dtype), _rand(N, K, seed=1, scale=0.05).to(dtype)
    dy = _rand(M, N, seed=2).to(dtype)
    xg, wg, bg = x.clone().requires_grad_(), w.clone().requires_grad_(), torch.zeros(N, device="cuda", requires_grad=True)
    y = qa.mxfp4_linear(xg, wg, bg)
    grads = torch.autograd.grad(y, (xg, wg, bg), dy, retain_graph=True)
    rx, rw, d = _values(x), _values(w), dy.double()
    _close(grads[0], d @ rw, d.abs() @ rw.abs(), 3 * (N / 8 + 2))
    dt = d.t().contiguous()
    _close(grads[1], dt @ rx, dt.abs() @ rx.abs(), 3 * (M / 8 + 2))
    _close(grads[2], d.sum(0), d.abs().sum(0), 3 * (M / 8 + 2))
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (xg, wg, bg), dy, retain_graph=True), grads))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,E,N,K,dropped,first", [(1500, 2, 3, 1500, 2800, 0.0, 0), (1501, 2, 4, 1301, 2801, 0.2, 1)])
def test_gradients_on_large_tiles_by_expert(tokens, top, E, N, K, dropped, first, gather, dtype):
    import qtpytorch_amd as qa
    rows = tokens * top
    assert rows // 256 * _up(K, 256) >= 110 and _up(N, 256) * E * _up(K, 256) >= 160
    ids = _ids(tokens, top, E + first, skew=0.3, dropped=dropped)
    plan = qa.expert_sort(ids.cuda(), E + first)
    plan = plan._replace(offsets=plan.offsets[first:])
    x, w = _rand(tokens if gather else rows, K).to(dtype), _rand(E, N, K, seed=1, scale=0.05).to(dtype)
    dy = _rand(rows, N, seed=2).to(dtype)
    dy[plan.order < 0] = float("nan")  # rows in no one's use
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = qa.expert_linear(xg, wg, plan, gather=gather)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    rx, d = _values(x), dy.double()
    offsets = plan.offsets.tolist()
    rows_dx, mass_dx = (torch.zeros(rows, K, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        rw = _values(w[e])
        a = rx[(plan.order[lo:hi] // top).long()] if gather else rx[lo:hi]
        rows_dx[lo:hi], mass_dx[lo:hi] = d[lo:hi] @ rw, d[lo:hi].abs() @ rw.abs()
        dt = d[lo:hi].t().contiguous()
        _close(dw[e], dt @ a, dt.abs() @ a.abs(), 3 * ((hi - lo) / 8 + 2))
    if gather:
        live, at = (plan.place >= 0)[..., None], plan.place.clamp(min=0).long()
        _close(dx, torch.where(live, rows_dx[at], 0.0).sum(1), torch.where(live, mass_dx[at], 0.0).sum(1),
               3 * (N / 8 + 2) + top)
    else:
        _close(dx, rows_dx, mass_dx, 3 * (N / 8 + 2))

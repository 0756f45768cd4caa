"""What the differentiable calls on microscaled 4-bit operands take, refuse and round."""
import pytest
import torch
from torch.autograd import forward_ad

from tests import _mxfp4 as R
from tests.test_gpu_experts import _gen, _ids

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _rand(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=_gen(seed)) * scale).cuda()


# ---------------------------------------------------------------- tangents
def _calls():
    """name, arguments that may have a tangent, the call."""
    import qtpytorch_amd as qa
    plan = qa.expert_sort(_ids(6, 2, 4).cuda(), 4)
    held, experts = qa.mxfp4_quantize(_rand(20, 64, seed=1)), qa.mxfp4_quantize(_rand(4, 20, 64, seed=2))
    return [
        ("linear", (_rand(6, 64), _rand(20, 64), _rand(20)), lambda x, w, b: qa.mxfp4_linear(x, w, b)),
        ("linear, held weight", (_rand(2, 3, 64), _rand(20)), lambda x, b: qa.mxfp4_linear(x, held, b)),
        ("matmul", (_rand(20),), lambda b: qa.mxfp4_matmul(held, held, b)),
        ("gather", (_rand(6, 64),), lambda x: qa.expert_gather(x, plan)),
        ("expert linear", (_rand(12, 64), _rand(4, 20, 64), _rand(4, 20)),
         lambda x, w, b: qa.expert_linear(x, w, plan, b)),
        ("expert linear, gathered", (_rand(6, 64),), lambda x: qa.expert_linear(x, experts, plan, gather=True)),
        ("combine", (_rand(12, 64), _rand(6, 2)), lambda h, g: qa.expert_combine(h, plan, g)),
        ("combine without gates", (_rand(12, 64),), lambda h: qa.expert_combine(h, plan)),
    ]


@pytest.mark.parametrize("call", range(8))
def test_a_tangent_is_refused(call):
    """No forward-mode derivative: an error in place of a result without its tangent."""
    import qtpytorch_amd as qa
    name, args, run = _calls()[call]
    want = run(*args)
    with forward_ad.dual_level():
        assert torch.equal(run(*args), want)  # no tangents: as ever
        for i in range(len(args)):
            duals = list(args)
            duals[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(qa._lib.MXKError, match="forward-mode"):
                run(*duals)
    assert torch.equal(run(*args), want)


# ---------------------------------------------------------------- biases
@pytest.mark.parametrize("m", [3, 70])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
def test_gradient_of_a_bias_of_any_float_type(dtype, m):
    """Sums in float32, then the bias's own type."""
    import qtpytorch_amd as qa
    x, w, bias = _rand(m, 64), _rand(20, 64, seed=1), _rand(20, seed=2).to(dtype).requires_grad_()
    dy = _rand(m, 20, seed=3)
    d = dy.double().cpu()
    as32 = torch.float32 if dtype == torch.float64 else dtype
    held = qa.mxfp4_quantize(w)
    for y in (qa.mxfp4_linear(x, held, bias), qa.mxfp4_linear(x, w, bias),
              qa.mxfp4_matmul(qa.mxfp4_quantize(x), held, bias, torch.float32),
              qa.mxfp4_matmul(qa.mxfp4_quantize(x.view(1, m, 64)), held, bias, torch.float32)[0]):
        (db,) = torch.autograd.grad(y, bias, dy)
        assert db.dtype == dtype
        R.assert_close(db.to(as32), d.sum(0), d.abs().sum(0), 3 * (m / 8 + 2))
    E, top = 4, 2
    ids = _ids(m, top, E)
    order, _, offsets = R.plan(ids, E)
    bias = _rand(E, 20, seed=4).to(dtype).requires_grad_()
    dy = _rand(m * top, 20, seed=5)
    d = dy.double().cpu()
    y = qa.expert_linear(x, qa.mxfp4_quantize(_rand(E, 20, 64, seed=6)), qa.expert_sort(ids.cuda(), E), bias, gather=True)
    (db,) = torch.autograd.grad(y, bias, dy)
    assert db.dtype == dtype
    for e in range(E):
        part = d[int(offsets[e]):int(offsets[e + 1])]
        R.assert_close(db[e].to(as32), part.sum(0), part.abs().sum(0), 3 * (len(part) / 8 + 2))


def test_packed_operands_alone_have_no_gradient():
    import qtpytorch_amd as qa
    q = qa.mxfp4_quantize(_rand(8, 64))
    bias = _rand(8).requires_grad_()
    assert not qa.mxfp4_matmul(q, q).requires_grad
    with torch.no_grad():
        assert not qa.mxfp4_matmul(q, q, bias).requires_grad
    assert torch.equal(qa.mxfp4_matmul(q, q, bias), qa.mxfp4_matmul(q, q, bias.detach()))


# ---------------------------------------------------------------- types
@pytest.mark.parametrize("dtype", [torch.float64, torch.int8, torch.uint8, torch.int32, torch.int64, torch.bool,
                                   torch.complex64])
def test_quantize_of_other_types_is_refused(dtype):
    """They would pass float32 on the way: rounded twice, out of its range, or without their imaginary part."""
    import qtpytorch_amd as qa
    for shape in ((4, 64), (2, 3, 32), (0, 32)):
        with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
            qa.mxfp4_quantize(torch.zeros(shape, dtype=dtype, device="cuda"))


def test_complex_biases_and_gates_are_refused():
    import qtpytorch_amd as qa
    x, plan = _rand(6, 64), qa.expert_sort(_ids(6, 2, 4).cuda(), 4)
    q, experts = qa.mxfp4_quantize(x), qa.mxfp4_quantize(_rand(4, 20, 64, seed=2))
    with pytest.raises(TypeError, match="real"):
        qa.mxfp4_matmul(q, q, torch.ones(6, dtype=torch.complex64, device="cuda"))
    with pytest.raises(TypeError, match="real"):
        qa.mxfp4_linear(x, q, torch.ones(6, dtype=torch.complex64, device="cuda"))
    with pytest.raises(TypeError, match="real"):
        qa.expert_linear(x, experts, plan, torch.ones(4, 20, dtype=torch.complex64, device="cuda"), gather=True)
    with pytest.raises(TypeError, match="real"):
        qa.expert_combine(_rand(12, 64), plan, torch.ones(6, 2, dtype=torch.complex64, device="cuda"))


# ---------------------------------------------------------------- rows without columns
def test_linear_over_rows_without_columns():
    """K = 0: the bias, for leading dimensions of any number."""
    import qtpytorch_amd as qa
    bias, w = _rand(7), torch.empty(7, 0).cuda()
    for lead in ((4,), (2, 3), (2, 1, 3), (0, 3), ()):
        x = torch.empty(*lead, 0).cuda()
        want = bias.expand(*lead, 7)
        assert torch.equal(qa.mxfp4_linear(x, qa.mxfp4_quantize(w), bias), want)
        xg, wg, bg = x.requires_grad_(), w.clone().requires_grad_(), bias.clone().requires_grad_()
        y = qa.mxfp4_linear(xg, wg, bg)
        assert torch.equal(y, want)
        dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape
        assert torch.equal(db, torch.full_like(db, want.numel() // 7))


# ---------------------------------------------------------------- gathered rows
def test_gathered_gradient_beyond_float16_in_its_parts():
    """A token's rows are added in float32: parts above float16's range that cancel leave what is left."""
    import qtpytorch_amd as qa
    plan = qa.expert_sort(torch.tensor([[0, 1]] * 5).cuda(), 2)
    x = torch.ones(5, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    w = torch.full((2, 8, 64), 4.0, device="cuda")
    w[1] = -3.0
    held = qa.mxfp4_quantize(w)
    dy = torch.full((10, 8), 5000.0, dtype=torch.float16, device="cuda")
    (dx,) = torch.autograd.grad(qa.expert_linear(x, held, plan, gather=True), x, dy)
    # 8 columns of 5000 * 4 and of 5000 * -3, 160000 and -120000
    assert torch.equal(dx, torch.full_like(dx, 40000.0))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("tokens,top,experts,n,k,dropped", [(1, 4, 8, 16, 32, 0.0), (64, 8, 16, 130, 320, 0.2),
                                                            (200, 4, 3, 257, 543, 0.3), (300, 2, 8, 64, 96, 0.0)])
def test_gathered_gradient_is_rounded_once(tokens, top, experts, n, k, dropped, dtype):
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, experts, dropped=dropped)
    order, place, offsets = R.plan(ids, experts)
    x = _rand(tokens, k).to(dtype).requires_grad_()
    w = _rand(experts, n, k, seed=1, scale=0.1)
    dy = _rand(tokens * top, n, seed=2).to(dtype)
    y = qa.expert_linear(x, qa.mxfp4_quantize(w), qa.expert_sort(ids.cuda(), experts), gather=True)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx.dtype == dtype
    rw, d = R.rounded(w), dy.double().cpu()
    rows, mass = (torch.zeros(tokens * top, k, dtype=torch.float64) for _ in range(2))
    for e in range(experts):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        rows[lo:hi], mass[lo:hi] = d[lo:hi] @ rw[e], d[lo:hi].abs() @ rw[e].abs()
    live = (place >= 0)[..., None]
    parts = torch.where(live, rows[place.clamp(min=0)], 0.0)
    masses = torch.where(live, mass[place.clamp(min=0)], 0.0)
    R.assert_close(dx, parts.sum(1), masses.sum(1), 3 * (n / 8 + 2) + top)

"""Plans that a routing makes by hand: places dropped after the sort (an expert's
capacity), and some experts' part of a larger plan."""
import pytest
import torch

from tests import _mxfp4 as R
from tests.test_gpu_experts import _gen, _ids

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _poison(*shape, dtype):
    """Leave NaNs in the memory that the next allocations of this size take."""
    held = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(3)]
    del held


def _dropped(ids, experts, keep_order):
    """The plan of ids with some of its places taken out, on the CPU; the picks that are out."""
    order, place, offsets = R.plan(ids, experts)
    out = (torch.rand(place.shape, generator=_gen(7)) < 0.3) & (place >= 0)
    out.view(-1)[::9] |= place.view(-1)[::9] >= 0
    if not keep_order:
        order[place[out].long()] = -1
    place = place.masked_fill(out, -1)
    place.view(-1)[out.view(-1).nonzero()[::2, 0]] = place.numel() + 3  # any place outside is none
    return order, place, offsets, out


def _cuda(plan):
    import qtpytorch_amd as qa
    return qa.expert_plan(*(t.cuda() for t in plan))


# ---------------------------------------------------------------- dropped places
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("keep_order", [True, False])
@pytest.mark.parametrize("tokens,top,experts,cols", [(1, 4, 8, 8), (40, 3, 5, 257), (130, 2, 16, 4096), (33, 6, 4, 1), (9, 8, 8, 520)])
def test_gradients_of_a_sum_without_the_dropped(tokens, top, experts, cols, keep_order, gated, dtype):
    """Rows that no place names pass nothing on and have a gradient of zero."""
    import qtpytorch_amd as qa
    order, place, offsets, out = _dropped(_ids(tokens, top, experts, dropped=0.1), experts, keep_order)
    rows = tokens * top
    named = torch.full((rows,), -1, dtype=torch.long)
    here = (place >= 0) & (place < rows)
    named[place[here].long()] = torch.arange(rows).view(place.shape)[here]
    h = torch.randn(rows, cols, generator=_gen(1)).to(dtype)
    h[named < 0] = float("nan")
    gates = torch.rand(tokens, top, generator=_gen(2)) if gated else torch.ones(tokens, top)
    dy = torch.randn(tokens, cols, generator=_gen(3)).to(dtype)
    hg, gg = h.cuda().requires_grad_(), gates.cuda().requires_grad_(gated)
    y = qa.expert_combine(hg, _cuda((order, place, offsets)), gg if gated else None)
    _poison(rows, cols, dtype=dtype)
    grads = torch.autograd.grad(y, (hg, gg) if gated else (hg,), dy.cuda())
    read = torch.where(here[..., None], h.double()[place.long().clamp(0, rows - 1)], 0.0)
    w = gates.double()[..., None]
    R.assert_close(y, (w * read).sum(1), (w * read.abs()).sum(1), top + 1)
    pick = named.clamp(min=0)
    dh = torch.where(named[:, None] >= 0, gates.double().reshape(-1)[pick][:, None] * dy.double()[pick // top], 0.0)
    R.assert_close(grads[0], dh, dh.abs(), 1)
    assert not grads[0].cpu()[named < 0].any()
    if gated:
        prod = read * dy.double()[:, None]
        R.assert_close(grads[1], prod.sum(-1), prod.abs().sum(-1), cols / 64 + 12)
        assert not grads[1].cpu()[out].any()


def test_gradients_of_a_sum_follow_its_places():
    """The sum reads places alone: so do its gradients, whatever the order says."""
    import qtpytorch_amd as qa
    place = torch.tensor([[3, 0], [-1, 5], [2, 9]], dtype=torch.int32).cuda()
    h = torch.randn(6, 40, generator=_gen(1)).cuda().requires_grad_()
    dy = torch.randn(3, 40, generator=_gen(2)).cuda()
    for order in ([0] * 6, [-1] * 6, [5, 4, 3, 2, 1, 0], [77] * 6):
        plan = qa.expert_plan(torch.tensor(order, dtype=torch.int32).cuda(), place,
                              torch.tensor([0, 6], dtype=torch.int32).cuda())
        for gates in (None, torch.full((3, 2), 2.0).cuda().requires_grad_()):
            y = qa.expert_combine(h, plan, gates)
            _poison(6, 40, dtype=torch.float32)
            dh = torch.autograd.grad(y, h, dy)[0]
            want = torch.stack([dy[0], dy[0] * 0, dy[2], dy[0], dy[0] * 0, dy[1]])
            assert torch.equal(dh, want if gates is None else 2 * want)


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens", [6, 200])
def test_a_layer_without_the_dropped(tokens, gather):
    """The layer of a plan with dropped places is the one whose dropped picks have no expert."""
    import qtpytorch_amd as qa
    E, top, D, N = 5, 3, 96, 70
    ids = _ids(tokens, top, E)
    order, place, offsets, out = _dropped(ids, E, True)
    x = torch.randn(tokens, D, generator=_gen(1)).cuda().requires_grad_()
    w = (torch.randn(E, N, D, generator=_gen(2)) * 0.1).cuda().requires_grad_()
    gates = torch.rand(tokens, top, generator=_gen(3)).cuda().requires_grad_()
    dy = torch.randn(tokens, N, generator=_gen(4)).cuda()

    def step(plan):
        _poison(tokens * top, N, dtype=torch.float32)
        rows = x if gather else qa.expert_gather(x, plan)
        y = qa.expert_combine(qa.expert_linear(rows, w, plan, gather=gather), plan, gates)
        return (y.detach(), *torch.autograd.grad(y, (x, w, gates), dy))

    got = step(_cuda((order, place, offsets)))
    want = step(qa.expert_sort(ids.masked_fill(out, -1).cuda(), E))
    for a, b in zip(got, want):  # the same sums, of rows in other places
        assert torch.isfinite(a).all() and float((a - b).norm()) <= 1e-6 * float(b.norm())


# ---------------------------------------------------------------- some experts of a larger plan
SLICES = [  # tokens, top, experts, the first of them and their number, n, k
    (6, 2, 5, 1, 3, 40, 96), (64, 4, 9, 2, 4, 130, 320), (300, 2, 8, 3, 4, 257, 544), (500, 2, 4, 2, 2, 64, 160),
    (40, 1, 70, 3, 64, 20, 64), (300, 1, 66, 1, 63, 20, 64), (30, 2, 4, 3, 1, 8, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,experts,first,held,n,k", SLICES)
def test_experts_of_a_part_of_a_plan(tokens, top, experts, first, held, n, k, gather, dtype):
    """offsets[first : first + held + 1]: those experts' rows are computed, all others are zeros."""
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, experts, dropped=0.1)
    order, place, offsets = R.plan(ids, experts)
    part = offsets[first:first + held + 1]
    plan = _cuda((order, place, part))
    x = torch.randn(tokens if gather else tokens * top, k, generator=_gen(1)).to(dtype)
    w = (torch.randn(held, n, k, generator=_gen(2)) * 0.1).to(dtype)
    bias = torch.randn(held, n, generator=_gen(3))
    dy = torch.randn(tokens * top, n, generator=_gen(4)).to(dtype)
    xg, wg, bg = x.cuda().requires_grad_(), w.cuda().requires_grad_(), bias.cuda().requires_grad_()
    rx, rw, d = R.rounded(x), R.rounded(w), dy.double()
    ref, mass = (torch.zeros(tokens * top, n, dtype=torch.float64) for _ in range(2))
    rows_dx, mass_dx = (torch.zeros(tokens * top, k, dtype=torch.float64) for _ in range(2))
    y = qa.expert_linear(xg, wg, plan, bg, gather=gather)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy.cuda())
    for e in range(held):
        lo, hi = int(part[e]), int(part[e + 1])
        rows = rx[order[lo:hi] // top] if gather else rx[lo:hi]
        ref[lo:hi] = rows @ rw[e].t() + bias[e].double()
        mass[lo:hi] = rows.abs() @ rw[e].abs().t() + bias[e].double().abs()
        rows_dx[lo:hi], mass_dx[lo:hi] = d[lo:hi] @ rw[e], d[lo:hi].abs() @ rw[e].abs()
        terms = 3 * ((hi - lo) / 8 + 2)
        R.assert_close(dw[e], d[lo:hi].t() @ rows, d[lo:hi].abs().t() @ rows.abs(), terms)
        R.assert_close(db[e], d[lo:hi].sum(0), d[lo:hi].abs().sum(0), terms)
    R.assert_close(y, ref, mass, k / 32 + 3)
    assert not y[:int(part[0])].any() and not y[int(part[-1]):].any()
    if not gather:
        R.assert_close(dx, rows_dx, mass_dx, 3 * (n / 8 + 2))
        assert not dx[:int(part[0])].any() and not dx[int(part[-1]):].any()
    held_w = qa.mxfp4_quantize(w.cuda())
    assert torch.equal(qa.expert_linear(x.cuda(), held_w, plan, bias.cuda(), gather=gather), y)


@pytest.mark.parametrize("gated", [True, False])
def test_gradients_of_a_sum_over_a_part_of_a_plan(gated):
    """The sum takes every row that a place names, in or out of the part."""
    import qtpytorch_amd as qa
    ids = _ids(50, 4, 8, dropped=0.2)
    plan = qa.expert_sort(ids.cuda(), 8)
    h = torch.randn(200, 64, generator=_gen(1)).cuda().requires_grad_()
    gates = torch.rand(50, 4, generator=_gen(2)).cuda().requires_grad_() if gated else None
    dy = torch.randn(50, 64, generator=_gen(3)).cuda()
    want = torch.autograd.grad(qa.expert_combine(h, plan, gates), (h, gates) if gated else (h,), dy)
    part = plan._replace(offsets=plan.offsets[2:5])
    for _ in range(4):
        y = qa.expert_combine(h, part, gates)
        _poison(200, 64, dtype=torch.float32)
        got = torch.autograd.grad(y, (h, gates) if gated else (h,), dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))

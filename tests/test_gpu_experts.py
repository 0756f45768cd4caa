"""Expert routing and products on the GPU against loops in 64 bits on the CPU."""
import pytest
import torch

from tests import _mxfp4 as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ids(tokens, top, experts, seed=0, skew=0.0, dropped=0.0, dtype=torch.int64):
    g = _gen(seed)
    logits = torch.randn(tokens, experts, generator=g) + skew * torch.randn(experts, generator=g)
    if top > experts:  # a token may pick an expert twice
        ids = torch.randint(0, experts, (tokens, top), generator=g)
    else:
        ids = logits.topk(top, dim=1).indices
    ids = ids.masked_fill(torch.rand(ids.shape, generator=g) < dropped, -1)
    return ids.to(dtype)


def _plan(ids, experts):
    import qtpytorch_amd as qa
    return qa.expert_sort(ids.cuda(), experts)


# ---------------------------------------------------------------- sort
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,top,experts", [(0, 2, 4), (1, 1, 1), (1, 4, 8), (3, 2, 300), (16, 4, 32), (64, 8, 128), (500, 3, 7),
                                                (1024, 2, 1000), (1025, 2, 16), (4100, 8, 256), (40000, 1, 3)])
def test_sort(tokens, top, experts, dtype):
    ids = _ids(tokens, top, experts, skew=1.0, dropped=0.2, dtype=dtype)
    for got, want in zip(_plan(ids, experts), R.plan(ids, experts)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("ids", [[[0, 0, 0]] * 70, [[5, -1, 2]] * 3000, [[-1]] * 10, [[9, 8, 1 << 40, -(1 << 40)]] * 5,
                                 [[7]] * 5000])
def test_sort_of_repeated_and_outside_ids(ids):
    ids = torch.tensor(ids)
    for got, want in zip(_plan(ids, 8), R.plan(ids, 8)):
        assert torch.equal(got.cpu(), want)


def test_sort_of_a_strided_view():
    ids = _ids(50, 4, 16)
    for got, want in zip(_plan(ids.t().contiguous().t(), 16), R.plan(ids, 16)):
        assert torch.equal(got.cpu(), want)


# ---------------------------------------------------------------- gather, combine
CASES = [(1, 1, 1, 8, 0.0), (5, 2, 4, 33, 0.3), (16, 4, 64, 4096, 0.0), (7, 3, 5, 100, 1.0), (300, 8, 16, 257, 0.25),
         (129, 1, 2, 64, 0.0), (2100, 2, 8, 1030, 0.1), (40, 6, 9, 1, 0.2), (33, 12, 20, 72, 0.4)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("tokens,top,experts,cols,dropped", CASES)
def test_gather_and_its_gradient(tokens, top, experts, cols, dropped, dtype):
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, experts, dropped=dropped)
    order, place, _ = R.plan(ids, experts)
    x = torch.randn(tokens, cols, generator=_gen(1)).to(dtype)
    xg = x.cuda().requires_grad_()
    y = qa.expert_gather(xg, _plan(ids, experts))
    want = torch.where(order[:, None] >= 0, x[order.clamp(min=0) // top], torch.zeros((), dtype=dtype))
    assert torch.equal(y.cpu(), want)
    dy = torch.randn(tokens * top, cols, generator=_gen(2)).to(dtype)
    dy[order < 0] = float("nan")  # rows that no pick holds add nothing
    (dx,) = torch.autograd.grad(y, xg, dy.cuda())
    rows = torch.where(place[..., None] >= 0, dy.double()[place.clamp(min=0)], 0.0)
    R.assert_close(dx, rows.sum(1), rows.abs().sum(1), top)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("tokens,top,experts,cols,dropped", CASES)
def test_combine_and_its_gradients(tokens, top, experts, cols, dropped, gated, dtype):
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, experts, dropped=dropped)
    order, place, offsets = R.plan(ids, experts)
    h = torch.randn(tokens * top, cols, generator=_gen(1)).to(dtype)
    h[order < 0] = float("nan")
    gates = torch.rand(tokens, top, generator=_gen(2)) if gated else torch.ones(tokens, top)
    hg, gg = h.cuda().requires_grad_(), gates.cuda().requires_grad_(gated)
    y = qa.expert_combine(hg, _plan(ids, experts), gg if gated else None)
    rows = torch.where(place[..., None] >= 0, h.double()[place.clamp(min=0)], 0.0)
    w = gates.double()[..., None]
    R.assert_close(y, (w * rows).sum(1), (w * rows.abs()).sum(1), top + 1)
    dy = torch.randn(tokens, cols, generator=_gen(3)).to(dtype)
    grads = torch.autograd.grad(y, (hg, gg) if gated else (hg,), dy.cuda())
    live, pick = order[:, None] >= 0, order.clamp(min=0)
    dh = torch.where(live, gates.double().reshape(-1)[pick][:, None] * dy.double()[pick // top], 0.0)
    R.assert_close(grads[0], dh, dh.abs(), 1)
    if gated:
        prod = rows * dy.double()[:, None]
        R.assert_close(grads[1], prod.sum(-1), prod.abs().sum(-1), cols / 64 + 12)


def test_combine_gradient_is_the_difference_quotient():
    import qtpytorch_amd as qa
    ids = _ids(6, 3, 4, dropped=0.2)
    plan = _plan(ids, 4)
    h, gates = torch.randn(18, 40, generator=_gen(1)), torch.rand(6, 3, generator=_gen(2))
    dy = torch.randn(6, 40, generator=_gen(3)).cuda()
    hg, gg = h.cuda().requires_grad_(), gates.cuda().requires_grad_()
    dh, dg = torch.autograd.grad(qa.expert_combine(hg, plan, gg), (hg, gg), dy)

    def loss(hh, g):
        return float((qa.expert_combine(hh.cuda(), plan, g.cuda()).double() * dy.double()).sum())

    # linear in either argument: the central difference has no error but the sums' rounding
    for i, j in ((0, 0), (7, 13), (17, 39)):
        up, down = h.clone(), h.clone()
        up[i, j] += 0.5
        down[i, j] -= 0.5
        assert abs(loss(up, gates) - loss(down, gates) - float(dh[i, j])) < 2e-4
    for t, j in ((0, 0), (3, 1), (5, 2)):
        up, down = gates.clone(), gates.clone()
        up[t, j] += 0.5
        down[t, j] -= 0.5
        assert abs(loss(h, up) - loss(h, down) - float(dg[t, j])) < 2e-4


def test_gather_of_rows_apart():
    import qtpytorch_amd as qa
    ids = _ids(20, 2, 4)
    big = torch.randn(20, 200, generator=_gen(1)).bfloat16()
    order, _, _ = R.plan(ids, 4)
    y = qa.expert_gather(big.cuda()[:, 3:150], _plan(ids, 4))
    assert torch.equal(y.cpu(), big[:, 3:150][order // 2])
    y = qa.expert_gather(big.cuda().t()[:20, :20], _plan(ids, 4))
    assert torch.equal(y.cpu(), big.t()[:20, :20][order // 2])


# ---------------------------------------------------------------- products by expert
EXPERT_CASES = [  # tokens, top, experts, n, k, dropped, skew
    (1, 1, 1, 16, 32, 0.0, 0.0), (8, 4, 32, 96, 128, 0.0, 0.0), (5, 2, 3, 70, 100, 0.4, 0.0), (64, 2, 4, 130, 320, 0.2, 1.0),
    (300, 2, 8, 64, 96, 0.0, 2.0), (200, 4, 3, 257, 544, 0.3, 0.5), (700, 1, 2, 512, 256, 0.1, 0.0), (16, 2, 1000, 20, 64, 0.5, 0.0),
    (30, 3, 8, 48, 2080, 0.0, 0.5), (10, 2, 4, 33, 64, 1.0, 0.0), (900, 2, 5, 300, 160, 0.2, 1.0)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,experts,n,k,dropped,skew", EXPERT_CASES)
def test_expert_linear(tokens, top, experts, n, k, dropped, skew, gather, dtype):
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, experts, skew=skew, dropped=dropped)
    order, _, offsets = R.plan(ids, experts)
    x = torch.randn(tokens if gather else tokens * top, k, generator=_gen(1)).to(dtype)
    if not gather:
        x[order < 0] = float("nan")  # rows that no expert reads
    w = torch.randn(experts, n, k, generator=_gen(2)) * 0.1
    bias = torch.randn(experts, n, generator=_gen(3))
    y = qa.expert_linear(x.cuda(), qa.mxfp4_quantize(w.cuda()), _plan(ids, experts), bias.cuda(), gather=gather)
    rx, rw = R.rounded(x), R.rounded(w)
    ref, mass = torch.zeros(tokens * top, n, dtype=torch.float64), torch.zeros(tokens * top, n, dtype=torch.float64)
    for e in range(experts):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        rows = rx[order[lo:hi] // top] if gather else rx[lo:hi]
        ref[lo:hi] = rows @ rw[e].t() + bias[e].double()
        mass[lo:hi] = rows.abs() @ rw[e].abs().t() + bias[e].double().abs()
    R.assert_close(y, ref, mass, k / 32 + 3)
    assert not y[int(offsets[-1]):].any()


@pytest.mark.parametrize("tokens", [33, 34, 48, 50, 64])
@pytest.mark.parametrize("n,k", [(17, 100), (130, 1056)])
def test_expert_linear_of_16_to_32_rows_an_expert(tokens, n, k):
    test_expert_linear(tokens, 2, 4, n, k, 0.1, 0.5, True, torch.float32)
    test_expert_linear(tokens, 2, 4, n, k, 0.0, 0.0, False, torch.bfloat16)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,experts,n,k,dropped,skew", [c for c in EXPERT_CASES if c[2] < 100])
def test_expert_gradients(tokens, top, experts, n, k, dropped, skew, gather, dtype):
    import qtpytorch_amd as qa
    ids = _ids(tokens, top, experts, skew=skew, dropped=dropped)
    order, place, offsets = R.plan(ids, experts)
    x = torch.randn(tokens if gather else tokens * top, k, generator=_gen(1)).to(dtype)
    w = (torch.randn(experts, n, k, generator=_gen(2)) * 0.1).to(dtype)
    dy = torch.randn(tokens * top, n, generator=_gen(3)).to(dtype)
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    bg = torch.zeros(experts, n, device="cuda", requires_grad=True)
    y = qa.expert_linear(xg, wg, _plan(ids, experts), bg, gather=gather)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy.cuda())
    rx, rw, d = R.rounded(x), R.rounded(w), dy.double()
    rows_dx = torch.zeros(tokens * top, k, dtype=torch.float64)
    mass_dx = torch.zeros_like(rows_dx)
    for e in range(experts):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        rows = rx[order[lo:hi] // top] if gather else rx[lo:hi]
        rows_dx[lo:hi], mass_dx[lo:hi] = d[lo:hi] @ rw[e], d[lo:hi].abs() @ rw[e].abs()
        terms = 3 * ((hi - lo) / 8 + 2)
        R.assert_close(dw[e], d[lo:hi].t() @ rows, d[lo:hi].abs().t() @ rows.abs(), terms)
        R.assert_close(db[e], d[lo:hi].sum(0), d[lo:hi].abs().sum(0), terms)
    if gather:  # each row rounded to dtype once, then added per token
        live = (place >= 0)[..., None]
        parts = torch.where(live, rows_dx[place.clamp(min=0)], 0.0)
        masses = torch.where(live, mass_dx[place.clamp(min=0)], 0.0)
        room = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype] * 2.0 ** 23
        R.assert_close(dx, parts.sum(1), masses.sum(1), 3 * (n / 8 + 2) + top + room)
    else:
        R.assert_close(dx, rows_dx, mass_dx, 3 * (n / 8 + 2))
    assert not dw[[e for e in range(experts) if offsets[e] == offsets[e + 1]]].any()


def test_a_plan_that_names_no_such_row_reads_zeros():
    """Places, offsets and picks outside the arrays are kept out by the kernels."""
    import qtpytorch_amd as qa
    order = torch.tensor([0, 90, 5, -7], dtype=torch.int32).cuda()
    place = torch.tensor([[0, 400], [2, -3]], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 3, 77], dtype=torch.int32).cuda()
    plan = qa.expert_plan(order, place, offsets)
    x = torch.randn(2, 64, generator=_gen(1)).cuda()
    y = qa.expert_gather(x, plan)
    assert torch.equal(y, torch.stack([x[0], x[0] * 0, x[0] * 0, x[0] * 0]))
    h = torch.randn(4, 64, generator=_gen(2)).cuda()
    assert torch.equal(qa.expert_combine(h, plan), torch.stack([h[0], h[2]]))
    w = qa.mxfp4_quantize(torch.randn(2, 8, 64, generator=_gen(3)).cuda())
    y = qa.expert_linear(x, w, plan, gather=True)
    assert torch.isfinite(y).all() and not y[1:].any()


# ---------------------------------------------------------------- the layer
@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_expert_mlp(tokens):
    import qtpytorch_amd as qa
    E, D, F, top = 8, 128, 96, 2
    g = _gen(0)
    router, up, down = torch.randn(E, D, generator=g), torch.randn(E, 2 * F, D, generator=g) * 0.1, \
        torch.randn(E, D, F, generator=g) * 0.1
    x = torch.randn(1, tokens, D, generator=g)
    layer = qa.mxfp4_expert_mlp(router.cuda(), up.cuda(), down.cuda(), top)
    xg = x.cuda().requires_grad_()
    y = layer(xg)
    y.sum().backward()
    assert y.shape == x.shape and xg.grad.isfinite().all() and layer.router.grad.isfinite().all()
    # in 64 bits; activations are packed twice, so a value at a tie may round the other way: compared by norm
    r = x[0].double()
    top_l, top_i = (x[0] @ router.t()).topk(top, dim=1)
    gates = top_l.double().softmax(1)
    rx, ru, rd = R.rounded(x[0]), R.rounded(up), R.rounded(down)
    want = torch.zeros_like(r)
    for t in range(tokens):
        for j in range(top):
            e = int(top_i[t, j])
            h = ru[e] @ rx[t]
            h = torch.nn.functional.silu(h[:F]) * h[F:]
            want[t] += gates[t, j] * (rd[e] @ R.rounded(h.float()[None])[0])
    assert float((y[0].detach().cpu().double() - want).norm() / want.norm()) < 5e-3


def test_rows_past_2_31_elements():
    """Gather, combine and the gradients of rows whose offsets pass 32 bits."""
    import qtpytorch_amd as qa
    tokens, top, cols = 70000, 4, 8192
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, 16, (tokens, top), device="cuda", generator=g)
    plan = qa.expert_sort(ids, 16)
    x = torch.empty(tokens, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=g).requires_grad_()
    y = qa.expert_gather(x, plan)
    assert y.numel() > 1 << 31
    pick = torch.tensor([0, 1, 262143, 262144, 279998, 279999], device="cuda")
    assert torch.equal(y[pick], x[(plan.order[pick] // top).long()])
    gates = torch.rand(tokens, top, device="cuda", generator=g).requires_grad_()
    z = qa.expert_combine(y, plan, gates)
    tok = torch.tensor([0, 3, 65535, 65536, 69999], device="cuda")
    rows = y.detach()[plan.place[tok].long()].float()
    assert torch.equal(z[tok], (gates[tok, :, None] * rows).sum(1).bfloat16()) or \
        float((z[tok].float() - (gates[tok, :, None] * rows).sum(1)).norm() / z[tok].float().norm()) < 4e-3
    dy = torch.empty_like(z).normal_(generator=g)
    dx, dg = torch.autograd.grad(z, (x, gates), dy)
    dots = (rows * dy[tok, None].float()).sum(-1)
    assert float((dg[tok] - dots).norm() / dots.norm()) < 1e-4
    # every row of a token is the token itself: its gradient is dy times the sum of its gates, each part rounded once
    ref = dy[tok].float() * gates.detach()[tok].sum(1, keepdim=True)
    assert float((dx[tok].float() - ref).norm() / ref.norm()) < 6e-3


def test_no_tokens():
    """A batch without tokens, and one whose picks are all other devices': empty or zero results and gradients."""
    import qtpytorch_amd as qa
    w = torch.randn(4, 48, 64, generator=_gen(1)).cuda().requires_grad_()
    for ids in (torch.zeros(0, 2, dtype=torch.int64), torch.full((5, 2), -1)):
        plan = _plan(ids, 4)
        x = torch.randn(ids.shape[0], 64, generator=_gen(2)).cuda().requires_grad_()
        gates = torch.ones(ids.shape, device="cuda", requires_grad=True)
        y = qa.expert_combine(qa.expert_linear(x, w, plan, gather=True), plan, gates)
        z = qa.expert_linear(qa.expert_gather(x, plan), w, plan)
        assert y.shape == (ids.shape[0], 48) and z.shape == (ids.numel(), 48)
        assert not y.any() and not z.any()
        grads = torch.autograd.grad(y.sum() + z.sum(), (x, w, gates))
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (x, w, gates)))


def test_gradients_of_gradients_are_refused():
    import qtpytorch_amd as qa
    plan = _plan(_ids(6, 2, 4), 4)
    x = torch.randn(6, 64, generator=_gen(1)).cuda().requires_grad_()
    w = torch.randn(4, 32, 64, generator=_gen(2)).cuda().requires_grad_()
    y = qa.expert_combine(qa.expert_linear(qa.expert_gather(x, plan), w, plan), plan)
    (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# ---------------------------------------------------------------- graphs
@pytest.mark.parametrize("tokens", [1, 12, 200])
def test_expert_layer_in_a_graph(tokens):
    """Replays of a captured layer and its gradient, with eager work in between, against eager calls bit for bit."""
    import qtpytorch_amd as qa
    E, D, F, top = 8, 256, 128, 2
    g = _gen(0)
    layer = qa.mxfp4_expert_mlp(torch.randn(E, D, generator=g).cuda(), (torch.randn(E, 2 * F, D, generator=g) * 0.1).cuda(),
                                (torch.randn(E, D, F, generator=g) * 0.1).cuda(), top)
    w = (torch.randn(D, D, generator=g) * 0.05).bfloat16().cuda().requires_grad_()
    x = torch.zeros(tokens, D, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.zeros(tokens, D, device="cuda", dtype=torch.bfloat16)

    def step():
        with torch.no_grad():
            routed = layer(x)
        y = qa.mxfp4_linear(x, w)
        return (routed, y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(tokens, D, generator=_gen(10 + i)))
            dy.copy_(torch.randn(tokens, D, generator=_gen(20 + i)))
        graph.replay()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- refusals
def test_refusals():
    import qtpytorch_amd as qa
    ids = _ids(6, 2, 4).cuda()
    plan = qa.expert_sort(ids, 4)
    x = torch.randn(6, 64, device="cuda")
    w = qa.mxfp4_quantize(torch.randn(4, 8, 64, device="cuda"))
    with pytest.raises(ValueError):
        qa.expert_sort(ids.view(-1), 4)
    with pytest.raises(TypeError):
        qa.expert_sort(ids.float(), 4)
    for n in (0, -1, 1001):
        with pytest.raises(qa._lib.MXKError):
            qa.expert_sort(ids, n)
    with pytest.raises(ValueError):
        qa.expert_gather(x[:5], plan)
    with pytest.raises(TypeError):
        qa.expert_gather(x.long(), plan)
    with pytest.raises(ValueError):
        qa.expert_combine(x, plan)
    with pytest.raises(ValueError):
        qa.expert_combine(torch.randn(12, 8, device="cuda"), plan, torch.rand(6, 3, device="cuda"))
    with pytest.raises(ValueError):
        qa.expert_linear(x, w, plan)
    with pytest.raises(ValueError):
        qa.expert_linear(x, qa.mxfp4_quantize(torch.randn(5, 8, 64, device="cuda")), plan, gather=True)
    with pytest.raises(ValueError):
        qa.expert_linear(x, w, plan, torch.zeros(8, device="cuda"), gather=True)
    with pytest.raises(TypeError):
        qa.expert_gather(x, plan._replace(order=plan.order.long()))
    with pytest.raises(ValueError):
        qa.expert_gather(x, plan._replace(place=plan.place[:5]))
    with pytest.raises(qa._lib.MXKError):
        qa.expert_sort(ids.cpu(), 4)
    with pytest.raises(ValueError):
        qa.mxfp4_expert_mlp(torch.zeros(4, 32), torch.zeros(4, 6, 16), torch.zeros(4, 32, 3), 2)

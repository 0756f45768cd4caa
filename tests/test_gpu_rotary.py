"""Rotary positions on the GPU against complex turns in 64 bits on the CPU."""
import pytest
import torch

from tests import _pages as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _table(pairs, axes, interleaved, base=1e4):
    import qtpytorch_amd as qa
    freqs = base ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))
    axis = (torch.arange(pairs) * axes // max(1, pairs)).int()
    return freqs, axis, qa.rotary_table(freqs.cuda(), axis.cuda() if axes > 1 else None, interleaved=interleaved)


def _positions(tokens, axes, far, wide, seed):
    p = torch.randint(-3, 50, (tokens, axes), generator=R.gen(seed)) + far
    return p if wide else p.int()


# tokens, heads, D, rotated, axes, far
CASES = [(1, 1, 64, 64, 1, 0), (1, 32, 128, 128, 1, 100000), (3, 5, 80, 80, 1, 0), (7, 2, 72, 36, 2, 1000),
         (16, 32, 128, 64, 3, 0), (130, 3, 96, 96, 3, 1 << 20), (33, 1, 256, 256, 2, 1 << 30), (5, 7, 10, 6, 1, 0),
         (4, 3, 7, 2, 1, 9), (1100, 4, 64, 64, 1, 0), (2, 2, 66, 0, 1, 0), (600, 9, 128, 128, 3, 77), (3, 2, 1024, 1024, 2, 5)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotated,axes,far", CASES)
def test_rotary_and_its_gradient(tokens, heads, dim, rotated, axes, far, interleaved, dtype):
    import qtpytorch_amd as qa
    freqs, axis, table = _table(rotated // 2, axes, interleaved)
    pos = _positions(tokens, axes, far, far > 1000, 1)
    x = (3 * torch.randn(tokens, heads, dim, generator=R.gen(2))).to(dtype)
    dy = torch.randn(tokens, heads, dim, generator=R.gen(3)).to(dtype)
    xg = x.cuda().requires_grad_()
    y = qa.rotary(xg, (pos if axes > 1 else pos[:, 0]).cuda(), table)
    (dx,) = torch.autograd.grad(y, xg, dy.cuda())
    for got, src, sign in ((y, x, 1.0), (dx, dy, -1.0)):
        want, size = R.rotate(src, pos, freqs, axis, interleaved, sign)
        assert got.dtype == dtype
        R.near(got, want, R.rotation_error(want, size, dtype))
        assert torch.equal(got.detach().cpu()[..., rotated:], src[..., rotated:])


def test_gradient_is_the_difference_quotient():
    import qtpytorch_amd as qa
    _, _, table = _table(8, 2, False)
    pos = _positions(5, 2, 3, True, 1).cuda()
    x, dy = torch.randn(5, 2, 20, generator=R.gen(1)), torch.randn(5, 2, 20, generator=R.gen(2)).cuda()
    xg = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(qa.rotary(xg, pos, table), xg, dy)
    for i in ((0, 0, 0), (2, 1, 7), (4, 0, 15), (4, 1, 19)):
        up, down = x.clone(), x.clone()
        up[i] += 0.5
        down[i] -= 0.5
        loss = [float((qa.rotary(v.cuda(), pos, table).double() * dy.double()).sum()) for v in (up, down)]
        # linear in x: the difference has the roundings of the two results alone, 2^-20 of at most 4 * 4 each
        assert abs(loss[0] - loss[1] - float(dx[i])) < 2.0 ** -12


@pytest.mark.parametrize("layout", ["heads first", "apart", "odd address", "last strided", "four dims", "broadcast"])
@pytest.mark.parametrize("dtype", FLOATS)
def test_layouts(layout, dtype):
    import qtpytorch_amd as qa
    freqs, axis, table = _table(32, 1, False)
    x = torch.randn(6, 4, 64, generator=R.gen(4)).to(dtype)
    pos = _positions(6, 1, 5, True, 2)
    if layout == "heads first":
        v = x.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    elif layout == "apart":
        v = torch.zeros(6, 9, 70, dtype=dtype, device="cuda")[:, 2:6, 3:67]
        v.copy_(x)
    elif layout == "odd address":
        v = torch.zeros(6 * 4 * 64 + 1, dtype=dtype, device="cuda")[1:].view(6, 4, 64)
        v.copy_(x)
    elif layout == "last strided":
        v = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    elif layout == "four dims":
        v = x.view(2, 3, 4, 64).cuda()
        pos = pos.view(2, 3, 1)
    else:
        x = x[:, :1].expand(6, 4, 64)
        v = x[:, :1].cuda().expand(6, 4, 64)
    want, size = R.rotate(x.reshape(6, 4, 64), pos.view(6, 1), freqs, axis, False)
    R.near(qa.rotary(v, pos.cuda(), table).reshape(6, 4, 64), want, R.rotation_error(want, size, dtype))


def test_gradient_of_a_broadcast_input_and_of_a_shared_one():
    import qtpytorch_amd as qa
    freqs, axis, table = _table(32, 1, True)
    pos = _positions(6, 1, 0, True, 2)
    x = torch.randn(6, 1, 64, generator=R.gen(4)).cuda().requires_grad_()
    dy = torch.randn(6, 3, 64, generator=R.gen(5))
    y = qa.rotary(x.expand(6, 3, 64), pos.cuda(), table)
    (dx,) = torch.autograd.grad(y, x, dy.cuda())
    want, size = R.rotate(dy, pos, freqs, axis, True, -1.0)
    R.near(dx, want.sum(1, keepdim=True), (R.rotation_error(want, size, torch.float32)
                                           + 2.0 ** -23 * want.abs()).sum(1, keepdim=True))


def test_gradient_of_the_gradient():
    """dx is linear in dy: its gradient towards dy is the rotation of the vector that it is weighted with."""
    import qtpytorch_amd as qa
    _, _, table = _table(32, 1, False)
    pos = _positions(6, 1, 0, True, 2).cuda()
    x, dy, v = (torch.randn(6, 3, 64, generator=R.gen(i)).cuda().requires_grad_() for i in range(3))
    (dx,) = torch.autograd.grad(qa.rotary(x, pos, table), x, dy, create_graph=True)
    assert dx.requires_grad
    (back,) = torch.autograd.grad(dx, dy, v.detach())
    assert torch.equal(back, qa.rotary(v.detach(), pos, table))
    # and it adds up along two uses of one leaf
    y = qa.rotary(x, pos, table) * qa.rotary(x, pos + 1, table).detach()
    (one,) = torch.autograd.grad(y.sum(), x)
    want = qa.rotary(qa.rotary(x, pos + 1, table).detach(), -pos, table)
    assert (one - want).abs().max() < 2.0 ** -19 * 2 * want.abs().max()  # the opposite angles, rounded apart


@pytest.mark.parametrize("shape", [(0, 4, 64), (5, 0, 64), (2, 0, 3, 64)])
def test_nothing_to_rotate(shape):
    import qtpytorch_amd as qa
    _, _, table = _table(32, 1, False)
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    y = qa.rotary(x, torch.zeros(shape[:-2], dtype=torch.int64, device="cuda"), table)
    assert y.shape == x.shape
    assert torch.autograd.grad(y, x, torch.zeros_like(y))[0].shape == x.shape


def test_far_positions_keep_their_angles():
    """2^40 positions on: float64 has the angle to 2^-12 of a radian; the reference multiplies as the kernel does."""
    import qtpytorch_amd as qa
    freqs, axis, table = _table(32, 1, False)
    pos = torch.tensor([[1 << 40], [-(1 << 40)], [(1 << 31) + 5], [0]])
    x = torch.randn(4, 2, 64, generator=R.gen(4))
    want, size = R.rotate(x, pos, freqs, axis, False)
    angle = (pos.double() * freqs).abs()[:, None].repeat(1, 1, 2) * 2.0 ** -51
    R.near(qa.rotary(x.cuda(), pos.cuda(), table), want, R.rotation_error(want, size, torch.float32) + angle * size)


def test_an_axis_without_positions_turns_nothing():
    import qtpytorch_amd as qa
    freqs = torch.ones(4, dtype=torch.float64).cuda()
    table = qa.rotary_table(freqs, torch.tensor([0, 5, -1, 1], dtype=torch.int32).cuda())
    x = torch.randn(3, 2, 8, generator=R.gen(1)).cuda()
    y = qa.rotary(x, torch.full((3, 2), 7).cuda(), table)
    assert torch.equal(y[..., [1, 2, 5, 6]], x[..., [1, 2, 5, 6]])
    assert not torch.equal(y[..., [0, 3]], x[..., [0, 3]])


def test_one_axis_of_positions_turns_all_pairs():
    import qtpytorch_amd as qa
    freqs, axis, table = _table(32, 3, False)
    x, pos = torch.randn(5, 2, 64, generator=R.gen(1)).cuda(), torch.arange(5).cuda() + 3
    want = qa.rotary(x, pos[:, None].repeat(1, 3), table)
    for p in (pos, pos[:, None], pos.int()):
        assert torch.equal(qa.rotary(x, p, table), want)
    one = qa.rotary_table(freqs.cuda())
    assert torch.equal(qa.rotary(x, pos, one), want)


def test_more_blocks_than_one_dimension_has():
    """2^22 workgroups and more: the last tokens get what they get alone."""
    import qtpytorch_amd as qa
    _, _, table = _table(129, 1, False)
    n = (1 << 22) + 5
    x = torch.zeros(n, 1, 258, dtype=torch.float16, device="cuda")
    at = torch.tensor([0, 1, (1 << 22) - 1, 1 << 22, n - 1], device="cuda")
    x[at] = torch.randn(5, 1, 258, generator=R.gen(1)).half().cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    got = qa.rotary(x, pos, table)
    assert torch.equal(got[at], qa.rotary(x[at], pos[at], table))


def test_packed_heads_are_their_values():
    import qtpytorch_amd as qa
    _, _, table = _table(32, 1, False)
    x = qa.mx_tensor.quantize(torch.randn(3, 4, 64, generator=R.gen(1)).cuda(), "int8d")
    pos = torch.arange(3).cuda()
    assert torch.equal(qa.rotary(x, pos, table), qa.rotary(x.dequantize(), pos, table))


def test_nan_and_infinity_stay_in_their_pair():
    import qtpytorch_amd as qa
    _, _, table = _table(32, 1, False)
    x = torch.randn(2, 2, 64, generator=R.gen(1)).cuda()
    x[0, 1, 3], x[1, 0, 40] = float("nan"), float("inf")
    y = qa.rotary(x, torch.tensor([5, 9]).cuda(), table)
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, 1, [3, 35]] = bad[1, 0, [8, 40]] = True
    assert torch.equal(~torch.isfinite(y), bad)


def test_make():
    import qtpytorch_amd as qa
    t = qa.rotary_table.make(128, 1e6, sections=(16, 24, 24))
    i = torch.arange(64, dtype=torch.float64)
    assert torch.allclose(t.freqs.cpu(), 1e6 ** (-i / 64), rtol=1e-14, atol=0)
    assert t.axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    t = qa.rotary_table.make(64, 100.0, sections=(16, 16), restart=True)
    assert torch.equal(t.freqs[:16], t.freqs[16:])
    assert qa.rotary_table.make(64).axis is None


def test_refusals():
    import qtpytorch_amd as qa
    _, _, table = _table(32, 1, False)
    x, pos = torch.zeros(3, 2, 64).cuda(), torch.zeros(3, dtype=torch.int64).cuda()
    with pytest.raises(ValueError, match="rotates 64"):
        qa.rotary(x[..., :40], pos, table)
    with pytest.raises(ValueError, match="positions"):
        qa.rotary(x, pos[:2], table)
    with pytest.raises(ValueError, match="positions"):
        qa.rotary(x, pos.view(3, 1)[:, :0], table)
    with pytest.raises(TypeError, match="int32 or int64"):
        qa.rotary(x, pos.float(), table)
    with pytest.raises(TypeError, match="bfloat16"):
        qa.rotary(x.double(), pos, table)
    with pytest.raises(ValueError, match="heads, D"):
        qa.rotary(x[0, 0], pos, table)
    with pytest.raises(qa._lib.MXKError, match="GPU only"):
        qa.rotary(x.cpu(), pos.cpu(), table)
    with pytest.raises(TypeError, match="float64"):
        qa.rotary_table(table.freqs.float())
    with pytest.raises(TypeError, match="int32"):
        qa.rotary_table(table.freqs, torch.zeros(32, dtype=torch.int64).cuda())
    with pytest.raises(ValueError, match="add up"):
        qa.rotary_table.make(64, sections=(16, 15))
    with pytest.raises(ValueError, match="even"):
        qa.rotary_table.make(63)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(qa._lib.MXKError, match="forward-mode"):
            qa.rotary(torch.autograd.forward_ad.make_dual(x, x), pos, table)


def test_graph_of_forward_and_gradient():
    import qtpytorch_amd as qa
    freqs, axis, table = _table(64, 3, False)
    x = torch.randn(40, 6, 128, generator=R.gen(1)).cuda().requires_grad_()
    dy = torch.randn(40, 6, 128, generator=R.gen(2)).cuda()
    pos = torch.zeros(40, 3, dtype=torch.int64).cuda()

    def step():
        y = qa.rotary(x, pos, table)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        pos.copy_(_positions(40, 3, 1000 * seed, True, seed))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))

"""Bits that the paged cache's attention keeps, where others than the tested rows or keys could take them away."""
import math

import pytest
import torch

from tests import _pages as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _pages(codes, scales):
    import qtpytorch_amd as qa
    return qa.kv_pages(codes.cuda(), scales.cuda())


# ---------------------------------------------------------------- probabilities of 22 bits in tiles of 16 rows
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("group", [1, 4])
def test_probabilities_of_few_rows_keep_22_bits(group, dtype):
    """Three keys whose weighted values nearly cancel: the result is far below the values, and with it the rounding
    of the result, so that what is left is the error of the probabilities.  The queries are integers with a
    largest of 127, which 16 and 24 bits of that largest hold exactly."""
    D, held = 64, 2
    batch = R.Batch([held], [1], 16)
    codes, scales = R.pool(batch, 1, D, 3)
    g = R.gen(5)
    q = torch.randint(-20, 21, (1, 1, D), generator=g).float()
    q[..., 0] = 127.0
    q = q.expand(1, group, D).contiguous().to(dtype)
    at = [batch.place(0, i) for i in range(3)]
    for i, (page, off) in enumerate(at):
        codes[page, 0, 0, off] = torch.randint(-127, 128, (D,), generator=g).to(torch.int8)
        scales[page, 0, 0, off] = 2.0 ** -10
        scales[page, 1, 0, off] = 1.0
    (k, _), _ = R.rows(batch, codes, scales, 0, 3)
    p = torch.softmax(D ** -0.5 * (k[0] @ q[0, 0].double()), 0)
    assert (p > 0.02).all()
    # of many triples of codes those with the least sum
    x, y = torch.randint(-127, 128, (2, 1 << 16), generator=g).double()
    z = -((p[0] * x + p[1] * y) / p[2]).round()
    rest = (p[0] * x + p[1] * y + p[2] * z).abs()
    rest = torch.where((z.abs() > 127) | (x.abs() < 40) | (y.abs() < 40), math.inf, rest)
    best = rest.argsort()[:D]
    for (page, off), c in zip(at, (x, y, z)):
        codes[page, 1, 0, off] = c[best].to(torch.int8)
    want = torch.stack([x, y, z])[:, best].mul(p[:, None]).sum(0)
    mean = torch.stack([x, y, z])[:, best].abs().mul(p[:, None]).sum(0)
    assert (want.abs() < 2.0 ** -9 * mean).all()
    # the probabilities' 2^-21; scores of below 2^3 in float32, so 2^-20 of a weight and of their sum, which is divided by
    error = mean * (2.0 ** -21 + 2 * 2.0 ** -20 + 2.0 ** -20) + want.abs() * R.HALF[dtype] + R.LEAST[dtype]
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu())
    R.near(got, want.expand(1, group, D), error.expand(1, group, D))


# ---------------------------------------------------------------- large scales of keys that a row does not see
def _coarse(batch, scales, mask, head=0):
    """What bfloat16 rows of large tiles may be off beside R.attend's error: a value's scale is a float16 there, relative
    to 2^e, e up to 4 above the exponent of the largest that the row sees: half a step of the smallest ones is 2^-25 * 2^e,
    at most 2^-21 of that largest scale, times a code of 127; the weights sum to 1."""
    out = torch.zeros(batch.tokens, 1, 1, dtype=torch.float64)
    for b, (h, n) in enumerate(zip(batch.held, batch.new)):
        where = [batch.place(b, at) for at in range(h + n)]
        vs = torch.tensor([float(scales[page, 1, head, off]) for page, off in where], dtype=torch.float64)
        out[batch.first[b]:batch.first[b] + n, 0, 0] = torch.where(R.seen(batch, b, mask), vs, 0.0).amax(1)
    return 127 * 2.0 ** -21 * out


def _check_unseen(group, masked, factor, dim, dtype, large=False):
    """A new token's values are larger than all others by a factor: the rows that do not see it, before it or on
    other branches of a tree, keep what they have without it, and the other rows are within their own bounds."""
    import qtpytorch_amd as qa
    batch = R.Batch([70, 0], [5, 4], 16)
    codes, scales = R.pool(batch, 1, dim, 1)
    mask = None
    if masked:
        mask = torch.cat([qa.kv_tree_mask([-1, 0, 0, 2, 1], device="cpu")[0], qa.kv_tree_mask([-1, -1, 0, 1], device="cpu")[0]])
    for b, i in ((0, 2), (1, 1)):
        page, off = batch.place(b, batch.held[b] + i)
        scales[page, 1, :, off] *= factor
    q = torch.randn(batch.tokens, group, dim, generator=R.gen(7)).to(dtype)
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu(), mask=None if mask is None else mask.cuda())
    want, error = R.attend(batch, codes, scales, q, mask)
    if large and dtype == torch.bfloat16:
        error = error + _coarse(batch, scales, mask)
    sees = torch.zeros(batch.tokens, dtype=torch.bool)
    for b, i in ((0, 2), (1, 1)):
        sees[batch.first[b]:batch.first[b] + batch.new[b]] = R.seen(batch, b, mask)[:, batch.held[b] + i]
    assert sees.any() and not sees.all()
    R.near(got[~sees.cuda()], want[~sees], error[~sees])
    # rows that see it: float16 has steps of 2^-24 of the largest value; a result past its type's largest is infinite
    fits = sees[:, None, None] & (want.abs() < torch.finfo(dtype).max * 0.99)
    big = torch.where(fits, want, 0.0)
    R.near(torch.where(fits.cuda(), got, 0.0), big, torch.where(fits, error, 1.0))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("factor", [32.0, 1e6, 1e12, 1e36])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("group", [2, 7])
def test_values_that_a_row_does_not_see_take_no_bits_from_it(group, masked, factor, dim, dtype):
    """Tiles of 16 rows."""
    _check_unseen(group, masked, factor, dim, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("factor", [6.0, 32.0, 1e6, 1e12, 1e36])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("group", [16, 26, 60])
def test_values_that_a_row_of_a_large_tile_does_not_see_take_no_bits_from_it(group, masked, factor, dim, dtype):
    """Tiles of 128 and of 256 rows."""
    _check_unseen(group, masked, factor, dim, dtype, large=True)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 4), (256, 2)])
@pytest.mark.parametrize("masked", [False, True])
def test_values_of_growing_sizes(masked, dim, group, dtype):
    """A prompt whose tokens' values grow by steps from 2^-60 to 2^60, the sequence's own or a tree's: every row is
    within the bounds of what it sees itself, over several steps and tiles."""
    batch = R.Batch([0, 30], [150, 90], 16)
    codes, scales = R.pool(batch, 1, dim, 1)
    for b, n in enumerate(batch.new):
        for i in range(n):
            page, off = batch.place(b, batch.held[b] + i)
            scales[page, 1, :, off] *= 2.0 ** (12 * (i // 15) - 60)
    mask = None
    if masked:
        mask = torch.zeros(batch.tokens, 3, dtype=torch.int64)
        for b, n in enumerate(batch.new):
            for i in range(n):
                for j in {i, i // 2, i // 3, max(0, i - 40), (7 * i) % n}:  # also tokens behind it
                    mask[batch.first[b] + i, j // 64] |= (1 << (j % 64)) if j % 64 < 63 else -(1 << 63)
    q = torch.randn(batch.tokens, group, dim, generator=R.gen(7)).to(dtype)
    if dtype == torch.float16:
        scales[:, 1] *= 2.0 ** -50  # below its largest
    want, error = R.attend(batch, codes, scales, q, mask)
    if dtype == torch.bfloat16:
        error = error + _coarse(batch, scales, mask)
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu(), mask=None if mask is None else mask.cuda())
    R.near(got, want, error)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("group", [3, 12])
def test_values_far_apart_in_tiles_that_are_cut(group, masked, dtype):
    """Several tiles a workgroup and several workgroups a tile, some of whose tiles have such a token."""
    batch = R.Batch([1100, 300, 0], [90, 40, 70], 16, front=2, back=3)
    codes, scales = R.pool(batch, 2, 64, 1)
    for b, i, size in ((0, 50, 1e7), (0, 77, 1e15), (1, 20, 1e5), (2, 3, 1e20)):
        page, off = batch.place(b, batch.held[b] + i)
        scales[page, 1, 1, off] *= size if dtype != torch.float16 else size ** 0.1
    mask = None
    if masked:
        mask = torch.randint(-(1 << 62), 1 << 62, (batch.tokens, 2), generator=R.gen(3))
    q = torch.randn(batch.tokens, 2 * group, 64, generator=R.gen(7)).to(dtype)
    want, error = R.attend(batch, codes, scales, q, mask)
    if dtype == torch.bfloat16:
        for head in range(2):
            error[:, head * group:(head + 1) * group] += _coarse(batch, scales, mask, head)
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu(), mask=None if mask is None else mask.cuda())
    R.near(got, want, error)


def test_values_far_apart_in_many_tiles_of_a_workgroup():
    """More tiles a workgroup than it has bits for: the first of two new tokens sees itself alone, and so gives its value."""
    import qtpytorch_amd as qa
    n, G, D = 9000, 50, 64
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = qa.kv_pages.empty(n, 16, 1, D)
    g = torch.Generator(device="cuda").manual_seed(1)
    pages.codes.copy_(torch.randint(-127, 128, pages.codes.shape, generator=g, device="cuda", dtype=torch.int8))
    pages.scales.copy_(torch.rand(pages.scales.shape, generator=g, device="cuda") + 0.5)
    pages.scales[::3, 1, :, 1] *= 1e12
    batch = qa.kv_batch(torch.arange(n, **i32)[:, None].contiguous(), torch.zeros(n, **i32), torch.arange(0, 2 * n + 1, 2, **i32))
    q = torch.randn(2 * n, G, D, generator=g, device="cuda")
    got = pages.attend(q, batch)[::2]
    want = (pages.codes[:, 1, 0, 0].float() * pages.scales[:, 1, 0, :1])[:, None]
    # one probability of 1 in two terms of 11 bits, and the division
    assert ((got - want).abs() <= 2.0 ** -20 * want.abs()).all()


def test_values_far_apart_come_and_go_in_a_graph():
    """A recorded call replayed where its tokens' values are far apart and where they are not."""
    import qtpytorch_amd as qa
    batch = R.Batch([70, 20], [30, 25], 16)
    codes, scales = R.pool(batch, 1, 64, 1)
    pages, gb = _pages(codes, scales), batch.gpu()
    q = torch.randn(batch.tokens, 8, 64, generator=R.gen(7)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages.attend(q, gb)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = pages.attend(q, gb)
    page, off = batch.place(0, 70 + 11)
    for factor in (1.0, 1e9, 1.0, 1e-9, 1e18, 1.0):
        now = scales.clone()
        now[page, 1, 0, off] *= factor
        pages.scales.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(got, pages.attend(q, gb))
        want, error = R.attend(batch, codes, now, q.cpu())
        R.near(got, want, error)


# ---------------------------------------------------------------- large queries in other rows
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [3, 40, 80])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [1e5, 1e12, 1e30])
def test_queries_of_other_rows_take_no_bits_from_a_row(size, dim, group, dtype):
    """One row's query is larger than the others' by far: theirs keep their own precision."""
    batch = R.Batch([300, 40], [2, 3], 16)
    codes, scales = R.pool(batch, 1, dim)
    q = torch.randn(5, group, dim, generator=R.gen(1))
    q[0, 1] *= size
    q[4, 0] *= size
    q = q.to(dtype)
    want, error = R.attend(batch, codes, scales, q)
    rows = torch.ones(5, group, dtype=torch.bool)
    rows[0, 1] = rows[4, 0] = False
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu())
    R.near(got[rows.cuda()], want[rows], error[rows])
    assert torch.isfinite(got).all()


def test_values_far_apart_among_many_sequences_in_tiles_of_256_rows():
    """The same in bfloat16: more sequences than a wave holds, tiles of 256 rows."""
    import qtpytorch_amd as qa
    n, G, D = 3000, 80, 64
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = qa.kv_pages.empty(n, 16, 1, D)
    g = torch.Generator(device="cuda").manual_seed(1)
    pages.codes.copy_(torch.randint(-127, 128, pages.codes.shape, generator=g, device="cuda", dtype=torch.int8))
    pages.scales.copy_(torch.rand(pages.scales.shape, generator=g, device="cuda") + 0.5)
    pages.scales[1::3, 1, :, 1] *= 1e12
    batch = qa.kv_batch(torch.arange(n, **i32)[:, None].contiguous(), torch.zeros(n, **i32), torch.arange(0, 2 * n + 1, 2, **i32))
    got = pages.attend(torch.randn(2 * n, G, D, generator=g, device="cuda").bfloat16(), batch)[::2].float()
    want = (pages.codes[:, 1, 0, 0].float() * pages.scales[:, 1, 0, :1])[:, None]
    # the scale, the probability and their product in float16, half a step of bfloat16
    assert ((got - want).abs() <= (2.0 ** -8 + 3 * 2.0 ** -11) * want.abs()).all()

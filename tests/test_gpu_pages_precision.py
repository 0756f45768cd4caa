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
def _check_unseen(group, masked, factor, dim, dtype):
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

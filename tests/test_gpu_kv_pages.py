"""The paged 8-bit cache on the GPU against loops in 64 bits on the CPU."""
import math

import pytest
import torch

from tests import _pages as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _pages(codes, scales):
    import qtpytorch_amd as qa
    return qa.kv_pages(codes.cuda(), scales.cuda())


def _rand(shape, seed, dtype=torch.float32, scale=1.0):
    return (scale * torch.randn(shape, generator=R.gen(seed))).to(dtype)


# ---------------------------------------------------------------- append, read
def _stored(pages, batch, b, i):
    p = batch.place(b, batch.held[b] + i)
    return None if p is None else (pages.codes[p[0], :, :, p[1]].cpu(), pages.scales[p[0], :, :, p[1]].cpu())


def _check_append(batch, heads, dim, dtype, group=2, rotated=None, axes=1, interleaved=False, positions=True, seed=0):
    import qtpytorch_amd as qa
    T = batch.tokens
    codes, scales = R.pool(batch, heads, dim, seed, poison=False)
    pages = _pages(codes, scales)
    k, v = _rand((T, heads, dim), seed + 1, dtype), _rand((T, heads, dim), seed + 2, dtype)
    q = _rand((T, heads * group, dim), seed + 3, dtype) if group else None
    rotated = dim if rotated is None else rotated
    freqs = 1e4 ** (-torch.arange(rotated // 2, dtype=torch.float64) / max(1, rotated // 2))
    axis = (torch.arange(rotated // 2) * axes // max(1, rotated // 2)).int()
    table = qa.rotary_table(freqs.cuda(), axis.cuda(), interleaved=interleaved)
    own = torch.zeros(T, dtype=torch.int64)
    for b in range(len(batch.held)):
        for i in range(batch.new[b]):
            own[batch.first[b] + i] = batch.held[b] + i
    pos = torch.randint(0, 9000, (T, axes), generator=R.gen(seed + 4)) if positions else own[:, None].repeat(1, axes)
    qr = pages.append(k.cuda(), v.cuda(), batch.gpu(), rotary=table, positions=pos.cuda() if positions else None,
                      q=None if q is None else q.cuda())
    kr, size = R.rotate(k, pos, freqs, axis, interleaved)
    inside = torch.zeros(T, dtype=torch.bool)
    wrote = torch.zeros(codes.shape[0], codes.shape[3], dtype=torch.bool)
    for b in range(len(batch.held)):
        for i in range(batch.new[b]):
            t = batch.first[b] + i
            inside[t] = True
            got = _stored(pages, batch, b, i)
            if got is None:
                continue
            wrote[batch.place(b, batch.held[b] + i)] = True
            for which, x, err in ((0, kr[t], 2.0 ** -21 * size[t]), (1, v[t].double(), torch.zeros(heads, dim))):
                scale = x.abs().amax(-1, keepdim=True).clamp(min=1e-12) / 127
                error = err.amax(-1, keepdim=True) / 127 + scale * 2.0 ** -22
                assert ((got[1][which].double()[:, None] - scale).abs() <= error).all()
                # half a step, and what the value, the scale (127 of them at most) and the quotient are off
                R.near(got[0][which].double() * got[1][which].double()[:, None], x,
                       (0.5 + 2.0 ** -15) * scale + err + 128 * error)
                assert (got[0][which].abs().amax(-1) == 127).all() or (scale <= 1e-12 / 127).any()
    # nothing else is written
    same = (pages.codes.cpu() == codes).all(-1) & (pages.scales.cpu() == scales)
    assert same[~wrote[:, None, None].expand_as(same)].all()
    if q is not None:
        want, size = R.rotate(q, pos, freqs, axis, interleaved)
        error = R.rotation_error(want, size, dtype)
        R.near(qr[inside.cuda()], want[inside], error[inside])
        assert (qr.cpu()[~inside] == 0).all()
    else:
        assert qr is None
    return pages, batch


SHAPES = [  # held, new, page, heads, dim
    ([0], [1], 16, 1, 64), ([37], [1], 16, 8, 128), ([5, 0, 100], [1, 1, 1], 32, 2, 256),
    ([3, 40, 0, 17], [20, 0, 33, 1], 16, 3, 128), ([15, 31], [2, 50], 16, 4, 64), ([1000], [70], 128, 1, 128)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("held,new,page,heads,dim", SHAPES)
def test_append(held, new, page, heads, dim, dtype):
    _check_append(R.Batch(held, new, page), heads, dim, dtype)


@pytest.mark.parametrize("rotated,axes,interleaved", [(128, 1, True), (128, 3, False), (64, 2, False), (72, 1, False), (20, 1, True),
                                                      (2, 1, False), (126, 3, True), (0, 1, False)])
def test_append_rotations(rotated, axes, interleaved):
    _check_append(R.Batch([5, 9], [3, 18], 16), 2, 128, torch.bfloat16, rotated=rotated, axes=axes, interleaved=interleaved)


@pytest.mark.parametrize("front,back", [(0, 5), (3, 0), (2, 4)])
def test_append_padding_and_own_positions(front, back):
    batch = R.Batch([5, 0, 9], [3, 0, 2], 16, front=front, back=back)
    _check_append(batch, 2, 64, torch.float32, positions=False)
    _check_append(batch, 2, 64, torch.float16, positions=False, group=0)


def test_append_many_tokens():
    """Four tokens a workgroup."""
    _check_append(R.Batch([0, 7], [1500, 901], 64, back=3), 1, 64, torch.bfloat16, group=1)


def test_append_beyond_the_table_and_bad_pages():
    batch = R.Batch([10, 30], [20, 5], 16, width=1)  # positions from 16 on have no entry
    _check_append(batch, 2, 64, torch.float32)
    batch = R.Batch([10, 30], [30, 5], 16)
    batch.table[0, 1], batch.table[1, 2] = batch.pages, -(1 << 31)
    _check_append(batch, 2, 64, torch.float32)


def test_append_many_sequences():
    held = [i % 19 for i in range(150)]
    _check_append(R.Batch(held, [(i * 7) % 3 for i in range(150)], 16), 1, 64, torch.float32, group=1)


def test_append_takes_the_codes_of_kv_cache_quantizer():
    """Without rotation a row's codes are those of the ring's "int8dv" rule, bit for bit."""
    import qtpytorch_amd as qa
    batch = R.Batch([20], [1], 16)
    pages = _pages(*R.pool(batch, 6, 128, poison=False))
    k, v = _rand((1, 6, 128), 1).cuda(), _rand((1, 6, 128), 2).cuda()
    assert pages.append(k, v, batch.gpu()) is None
    ring = qa.kv_cache_quantizer(6, 128, "int8dv", asymmetric_v=False)
    ring.append_kv(k, v)
    kd, vd = ring.get()
    codes, scales = _stored(pages, batch, 0, 0)
    both = codes.float() * scales[..., None]
    assert torch.equal(both[0], kd.cpu()[0, :, 0]) and torch.equal(both[1], vd.cpu()[0, :, 0])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_of_rows_that_are_not_finite(bad):
    batch = R.Batch([0], [3], 16)
    pages = _pages(*R.pool(batch, 2, 64, poison=False))
    k, v = _rand((3, 2, 64), 1), _rand((3, 2, 64), 2)
    k[1, 0, 5], v[2, 1, 63] = bad, bad
    pages.append(k.cuda(), v.cuda(), batch.gpu())
    kr, vr = pages.read(batch.gpu(), 3, torch.float32)
    want = torch.zeros(3, 2, 64, dtype=torch.bool)
    want[1, 0] = True
    assert torch.equal(torch.isnan(kr.cpu()), want)
    want[:] = False
    want[2, 1] = True
    assert torch.equal(torch.isnan(vr.cpu()), want)


@pytest.mark.parametrize("fill", [0.0, 1e-30, 3e38, 1e-45])
def test_append_of_constant_and_extreme_rows(fill):
    batch = R.Batch([0], [1], 16)
    pages = _pages(*R.pool(batch, 1, 64, poison=False))
    k = torch.full((1, 1, 64), fill)
    pages.append(k.cuda(), -k.cuda(), batch.gpu())
    kr, vr = pages.read(batch.gpu(), 1, torch.float32)
    error = torch.full((1, 1, 64), max(fill * 2.0 ** -22, 0.5 * 1e-12 / 127), dtype=torch.float64)
    R.near(kr, k.double(), error)
    R.near(vr, -k.double(), error)


@pytest.mark.parametrize("layout", ["apart", "heads first", "odd address", "fused"])
@pytest.mark.parametrize("dtype", FLOATS)
def test_append_layouts(layout, dtype):
    import qtpytorch_amd as qa
    batch = R.Batch([3, 20], [4, 3], 16)
    x = _rand((7, 8, 64), 1, dtype)  # 4 query, 2 key, 2 value heads
    table = qa.rotary_table.make(64)
    one, two = (_pages(*R.pool(batch, 2, 64, poison=False)) for _ in range(2))
    if layout == "apart":
        y = torch.zeros(7, 9, 70, dtype=dtype, device="cuda")[:, :8, 3:67]
    elif layout == "heads first":
        y = torch.zeros(8, 7, 64, dtype=dtype, device="cuda").transpose(0, 1)
    elif layout == "odd address":
        y = torch.zeros(7 * 8 * 64 + 1, dtype=dtype, device="cuda")[1:].view(7, 8, 64)
    else:
        y = torch.zeros(7, 8 * 64, dtype=dtype, device="cuda").view(7, 8, 64)
    y.copy_(x)
    x = x.cuda()
    a = one.append(x[:, 4:6].contiguous(), x[:, 6:].contiguous(), batch.gpu(), rotary=table, q=x[:, :4].contiguous())
    b = two.append(y[:, 4:6], y[:, 6:], batch.gpu(), rotary=table, q=y[:, :4])
    assert torch.equal(a, b) and torch.equal(one.codes, two.codes) and torch.equal(one.scales, two.scales)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("held,new,page,heads,dim", SHAPES)
def test_read(held, new, page, heads, dim, dtype):
    batch = R.Batch(held, new, page, front=1, back=2)
    codes, scales = R.pool(batch, heads, dim)
    batch.table[0, 0] = -1
    k, v = _pages(codes, scales).read(batch.gpu(), batch.tokens, dtype)
    want = torch.zeros(2, batch.tokens, heads, dim)
    for b in range(len(held)):
        both, _ = R.rows(batch, codes, scales, b, held[b] + new[b])
        want[:, batch.first[b]:batch.first[b] + new[b]] = both[:, :, held[b]:].transpose(1, 2).float()
    assert torch.equal(k.cpu(), want[0].to(dtype)) and torch.equal(v.cpu(), want[1].to(dtype))


# ---------------------------------------------------------------- keep
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("path", [[[0]], [[0, 2, 5], [-1, 0, 1]], [[5, 4, 3, 2, 1, 0]], [[1, 1, 0, 7, -1, 2], [9, 8, 2, 100, 0, 0]]])
def test_keep(path, dim):
    n = len(path)
    batch = R.Batch([13, 30][:n], [8, 10][:n], 16)
    codes, scales = R.pool(batch, 3, dim)
    pages = _pages(codes, scales)
    pages.keep(batch.gpu(), torch.tensor(path, dtype=torch.int32).cuda())
    want_c, want_s = codes.clone(), scales.clone()
    for b in range(n):
        for j, pick in enumerate(path[b]):
            if 0 <= pick < batch.new[b]:
                to, at = batch.place(b, batch.held[b] + j), batch.place(b, batch.held[b] + pick)
                want_c[to[0], :, :, to[1]] = codes[at[0], :, :, at[1]]
                want_s[to[0], :, :, to[1]] = scales[at[0], :, :, at[1]]
    assert torch.equal(pages.codes.cpu(), want_c)
    assert torch.equal(pages.scales.cpu().view(torch.int32), want_s.view(torch.int32))


def test_keep_of_the_longest_path_and_of_absent_pages():
    batch = R.Batch([40], [100], 32)
    codes, scales = R.pool(batch, 2, 256)
    batch.table[0, 2] = 1 << 30  # positions 64 to 95: 24 of the sources
    pages = _pages(codes, scales)
    path = torch.randint(0, 100, (1, 64), generator=R.gen(1), dtype=torch.int32)
    pages.keep(batch.gpu(), path.cuda())
    want = codes.clone()
    for j, pick in enumerate(path[0].tolist()):
        to, at = batch.place(0, 40 + j), batch.place(0, 40 + pick)
        if to and at:
            want[to[0], :, :, to[1]] = codes[at[0], :, :, at[1]]
    assert torch.equal(pages.codes.cpu(), want)


def test_keep_moves_scales_along():
    batch = R.Batch([30, 5], [40, 20], 16)
    codes, scales = R.pool(batch, 2, 64)
    pages = _pages(codes, scales)
    path = torch.tensor([[3, 3, 39, 0, 1], [-1, 19, 20, 2, 2]], dtype=torch.int32)  # twice the same, none, past the last
    pages.keep(batch.gpu(), path.cuda())
    want_c, want_s = codes.clone(), scales.clone()
    for b in range(2):
        for j, pick in enumerate(path[b].tolist()):
            if 0 <= pick < batch.new[b]:
                to, at = batch.place(b, batch.held[b] + j), batch.place(b, batch.held[b] + pick)
                want_c[to[0], :, :, to[1]] = codes[at[0], :, :, at[1]]
                want_s[to[0], :, :, to[1]] = scales[at[0], :, :, at[1]]
    assert torch.equal(pages.codes.cpu(), want_c)
    assert torch.equal(pages.scales.cpu().nan_to_num(-1.0), want_s.nan_to_num(-1.0))


# ---------------------------------------------------------------- attend
def _check_attend(batch, heads, group, dim, dtype, mask=None, scale=None, seed=0, qscale=1.5):
    codes, scales = R.pool(batch, heads, dim, seed)
    q = _rand((batch.tokens, heads * group, dim), seed + 5, dtype, qscale)
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu(), mask=None if mask is None else mask.cuda(), scale=scale)
    assert got.dtype == dtype
    want, error = R.attend(batch, codes, scales, q, mask, scale)
    R.near(got, want, error)
    return got


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("held,page", [([0], 16), ([1], 16), ([31, 32, 33], 16), ([127, 128, 129], 32), ([700, 0, 3], 64),
                                       ([1500], 16), ([0, 0, 260], 256)])
def test_attend_one_token(held, page, dim, dtype):
    _check_attend(R.Batch(held, [1] * len(held), page), 2, 4, dim, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (1, 3), (2, 5), (1, 16), (1, 17), (2, 40), (5, 6)])
def test_attend_groups(heads, group, dtype):
    _check_attend(R.Batch([50, 0, 200], [1, 2, 0], 16), heads, group, 64, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("held,new,page,group", [([0], [200], 16, 2), ([100, 0], [70, 33], 32, 1), ([10, 300, 0, 7], [0, 129, 1, 64], 16, 3),
                                                 ([129], [127], 128, 4), ([64], [300], 64, 8), ([2100], [40], 16, 4)])
def test_attend_chunks(held, new, page, group, dtype):
    _check_attend(R.Batch(held, new, page), 1, group, 128, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("held,new,page,group", [([0], [1], 16, 40), ([3, 600], [20, 20], 16, 4), ([70, 0], [63, 64], 32, 2),
                                                 ([0, 255, 9], [65, 33, 0], 64, 5), ([190], [300], 16, 1)])
def test_attend_tiles(held, new, page, group, dim, dtype):
    """Tiles of 128 and of 256 rows, for every size of head."""
    _check_attend(R.Batch(held, new, page, front=1), 2 if group < 3 else 1, group, dim, dtype)


def _tree(batch, seed=0, words=None):
    import qtpytorch_amd as qa
    words = max([1] + [-(-n // 64) for n in batch.new]) if words is None else words
    out = torch.randint(-(1 << 62), 1 << 62, (batch.tokens, words), generator=R.gen(seed))  # padding rows: anything
    for b, n in enumerate(batch.new):
        up = [-1 if i == 0 else int(torch.randint(max(0, i - 5), i, (), generator=R.gen(seed + 31 * i + b))) for i in range(n)]
        m, _ = qa.kv_tree_mask(up, device="cpu")
        out[batch.first[b]:batch.first[b] + n] = 0
        out[batch.first[b]:batch.first[b] + n, :m.shape[1]] = m[:, :words] if n else m.new_zeros(0, m.shape[1])
    return out


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("held,new,group,dim", [([0], [5], 1, 64), ([40, 7], [16, 17], 4, 64), ([100, 0, 33], [64, 0, 65], 2, 128),
                                                ([300], [130], 3, 64), ([126, 127, 128], [3, 3, 3], 8, 64), ([63, 64, 65], [30, 66, 2], 3, 256),
                                                ([1000, 70], [60, 90], 6, 128), ([1, 513], [200, 10], 2, 64)])
def test_attend_trees(held, new, group, dim, dtype):
    batch = R.Batch(held, new, 16, front=1, back=2)
    got = _check_attend(batch, 2, group, dim, dtype, mask=_tree(batch))
    inside = torch.zeros(batch.tokens, dtype=torch.bool)
    for b, n in enumerate(new):
        inside[batch.first[b]:batch.first[b] + n] = True
    assert (got.cpu()[~inside] == 0).all()


def test_attend_any_mask():
    """Bits ahead of a token count too, bits past its sequence's tokens do not, and rows may see nothing."""
    batch = R.Batch([0, 20], [70, 9], 16)
    mask = torch.randint(-(1 << 62), 1 << 62, (batch.tokens, 2), generator=R.gen(3))
    mask[3] = 0
    mask[:, 1] = -1
    mask[5] = mask[7] = 0
    got = _check_attend(batch, 1, 2, 64, torch.float32, mask=mask)
    assert (got[[3 + 0, 5, 7]].cpu()[1:] == 0).all()
    # fewer words than tokens: later tokens are not seen
    _check_attend(batch, 1, 2, 64, torch.float32, mask=mask[:, :1].contiguous())
    for group in (1, 8):
        _check_attend(batch, 1, group, 128, torch.bfloat16, mask=mask)


@pytest.mark.parametrize("group", [2, 16, 50])
@pytest.mark.parametrize("masked", [False, True])
def test_attend_non_finite_where_it_is_not_seen(masked, group):
    """Scales of NaN and infinity in places that a row does not see leave it alone; where it sees them it is NaN."""
    batch = R.Batch([40, 7], [6, 5], 16)
    codes, scales = R.pool(batch, 1, 64)
    mask = _tree(batch, 2) if masked else None
    for b, i, bad in ((0, 3, math.nan), (1, 2, math.inf)):
        p = batch.place(b, batch.held[b] + i)
        scales[p[0], b, :, p[1]] = bad  # a key of the first, a value of the second
    q = _rand((batch.tokens, group, 64), 1)
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu(), mask=None if mask is None else mask.cuda()).cpu()
    for b, i in ((0, 3), (1, 2)):
        see = R.seen(batch, b, mask)[:, batch.held[b] + i]
        rows = got[batch.first[b]:batch.first[b] + batch.new[b]]
        assert see.any() and not see.all()
        assert (~torch.isfinite(rows[see])).any(-1).all() and torch.isfinite(rows[~see]).all()
    want, error = R.attend(batch, codes, torch.where(torch.isfinite(scales), scales, 0.0), q, mask)
    fine = torch.isfinite(got).all(-1)
    R.near(got[fine], want[fine], error[fine])


@pytest.mark.parametrize("group", [2, 32, 100])
def test_attend_rows_of_q_that_are_not_finite(group):
    batch = R.Batch([40, 0], [1, 2], 16)
    codes, scales = R.pool(batch, 1, 64)
    q = _rand((3, group, 64), 1)
    q[0, 1, 5], q[2, 0, 0] = math.nan, -math.inf
    mask = torch.tensor([[1], [1], [0]])  # the last row sees nothing
    got = _pages(codes, scales).attend(q.cuda(), batch.gpu(), mask=mask.cuda()).cpu()
    assert torch.isnan(got[0, 1]).all() and torch.isfinite(got[0, 0]).all() and (got[2] == 0).all()


@pytest.mark.parametrize("dtype", FLOATS)
def test_attend_sharp_and_flat(dtype):
    batch = R.Batch([900, 500], [1, 20], 16)
    for group in (2, 4, 20):
        _check_attend(batch, 1, group, 64, dtype, scale=3.0)
        _check_attend(batch, 1, group, 64, dtype, scale=1e-6)
        _check_attend(batch, 1, group, 64, dtype, qscale=0.0)


@pytest.mark.parametrize("group", [3, 20, 80])
@pytest.mark.parametrize("dtype", FLOATS)
def test_attend_values_of_far_apart_scales(dtype, group):
    """A key that takes nearly all of the weight has small values; the others' still count."""
    batch = R.Batch([600], [2], 16)
    codes, scales = R.pool(batch, 1, 128)
    p = batch.place(0, 0)
    scales[p[0], 0, 0, p[1]] *= 6.0
    scales[p[0], 1, 0, p[1]] *= 1e-5
    q = _rand((2, group, 128), 1, dtype, 0.2)
    q[:, 0] = (codes[p[0], 0, 0, p[1]].float() / 40).to(dtype)
    want, error = R.attend(batch, codes, scales, q)
    R.near(_pages(codes, scales).attend(q.cuda(), batch.gpu()), want, error)


@pytest.mark.parametrize("group", [3, 20, 80])
@pytest.mark.parametrize("dtype", FLOATS)
def test_attend_rows_of_far_apart_sizes(dtype, group):
    """Rows of one tile whose queries differ by 2^15: each keeps its own precision."""
    batch = R.Batch([300, 40], [2, 3], 16)
    codes, scales = R.pool(batch, 1, 64)
    size = torch.tensor([1e-3, 1.0, 30.0])[torch.randint(0, 3, (5, group, 1), generator=R.gen(2))]
    q = (size * _rand((5, group, 64), 1)).to(dtype)
    want, error = R.attend(batch, codes, scales, q)
    R.near(_pages(codes, scales).attend(q.cuda(), batch.gpu()), want, error)


@pytest.mark.parametrize("group", [2, 64])
@pytest.mark.parametrize("factor", [1e-30, 1e20])
def test_attend_scales_at_both_ends(factor, group):
    batch = R.Batch([300], [2], 16)
    codes, scales = R.pool(batch, 1, 64)
    scales[:, 1] *= factor
    q = _rand((2, group, 64), 1)
    want, error = R.attend(batch, codes, scales, q)
    R.near(_pages(codes, scales).attend(q.cuda(), batch.gpu()), want, error)


@pytest.mark.parametrize("group", [2, 32])
def test_attend_absent_pages(group):
    batch = R.Batch([100, 70], [4, 1], 16)
    codes, scales = R.pool(batch, 2, 64)
    batch.table[0, 1], batch.table[0, 6], batch.table[1, 4] = batch.pages + 5, -1, -(1 << 31)
    q = _rand((5, 2 * group, 64), 1)
    want, error = R.attend(batch, codes, scales, q)
    R.near(_pages(codes, scales).attend(q.cuda(), batch.gpu()), want, error)
    batch.table[:] = -1
    assert (_pages(codes, scales).attend(q.cuda(), batch.gpu()).cpu() == 0).all()


@pytest.mark.parametrize("group", [2, 10])
def test_attend_more_positions_than_the_table(group):
    batch = R.Batch([100, 70], [40, 1], 16)
    codes, scales = R.pool(batch, 1, 64)
    batch.table, batch.width = batch.table[:, :7].contiguous(), 7  # 112 positions
    q = _rand((41, group, 64), 1)
    want, error = R.attend(batch, codes, scales, q)
    R.near(_pages(codes, scales).attend(q.cuda(), batch.gpu()), want, error)
    batch.table, batch.width = batch.table[:, :0].contiguous(), 0
    assert (_pages(codes, scales).attend(q.cuda(), batch.gpu()).cpu() == 0).all()


@pytest.mark.parametrize("group", [2, 80])
def test_attend_sequences_whose_offsets_do_not_ascend(group):
    """A sequence that would end before it begins has no tokens, whatever the distance."""
    batch = R.Batch([100], [5], 16)
    codes, scales = R.pool(batch, 1, 64)
    q = _rand((5, group, 64), 1)
    want, error = R.attend(batch, codes, scales, q)
    one = batch.gpu()
    i32 = dict(dtype=torch.int32, device="cuda")
    least = -(1 << 31)
    three = one._replace(table=one.table.repeat(3, 1), lengths=one.lengths.repeat(3), offsets=torch.tensor([0, 5, least, 5], **i32))
    pages = _pages(codes, scales)
    R.near(pages.attend(q.cuda(), three), want, error)
    before = pages.codes.clone()
    second = one._replace(offsets=torch.tensor([5, least], **i32))
    pages.keep(second, torch.tensor([[3, 1, 4]], **i32))
    assert torch.equal(before, pages.codes)


def test_more_blocks_than_one_dimension_has():
    """More than 2^24 tokens: the last ones are rotated, stored and read as they are alone."""
    import qtpytorch_amd as qa
    n, D = (1 << 24) + 3, 64
    i32 = dict(dtype=torch.int32, device="cuda")
    table = qa.rotary_table.make(D)
    x = torch.zeros(n, 1, D, dtype=torch.bfloat16, device="cuda")
    x[-20:] = _rand((20, 1, D), 1, torch.bfloat16).cuda()
    # the last 20 tokens are a sequence's, those in front of them padding
    batch = qa.kv_batch(torch.tensor([[1, 0]], **i32), torch.tensor([7], **i32), torch.tensor([n - 20, n], **i32))
    alone = batch._replace(offsets=torch.tensor([0, 20], **i32))
    big, small = qa.kv_pages.empty(2, 16, 1, D), qa.kv_pages.empty(2, 16, 1, D)
    for p in (big, small):
        p.codes.zero_()
        p.scales.zero_()
    got = big.append(x, x, batch, rotary=table, q=x)
    want = small.append(x[-20:], x[-20:], alone, rotary=table, q=x[-20:])
    assert torch.equal(got[-20:], want) and not got[:-20].any()
    assert torch.equal(big.codes, small.codes) and torch.equal(big.scales, small.scales) and big.codes.any()
    k, v = big.read(batch, n)
    k1, v1 = small.read(alone, 20)
    assert torch.equal(k[-20:], k1) and torch.equal(v[-20:], v1) and not k[:-20].any()


def test_attend_many_sequences():
    held = [(i * 37) % 150 for i in range(200)]
    _check_attend(R.Batch(held, [(i * 7) % 3 for i in range(200)], 16), 1, 2, 64, torch.bfloat16)


@pytest.mark.parametrize("count,group", [(65, 2), (70, 90), (1500, 2), (600, 90), (1100, 70)])
def test_attend_more_sequences_than_threads(count, group):
    held = [(i * 37) % 45 for i in range(count)]
    _check_attend(R.Batch(held, [(i * 7) % 5 // 2 for i in range(count)], 16, front=2, back=3), 1, group, 64, torch.float16)


@pytest.mark.parametrize("count", [63, 64, 65, 4095, 4097, 9000])
def test_every_token_finds_its_sequence(count):
    """Each sequence stores a value of its own in its page; idle ones store nothing."""
    import qtpytorch_amd as qa
    i32 = dict(dtype=torch.int32)
    new = torch.randint(0, 3, (count,), generator=R.gen(count), **i32)
    offsets = torch.cat([torch.zeros(1, **i32), new.cumsum(0).int()]) + 2
    T = int(offsets[-1]) + 3
    owner = torch.full((T,), -1)
    owner[2:T - 3] = torch.repeat_interleave(torch.arange(count), new.long())
    batch = qa.kv_batch(torch.arange(count, **i32)[:, None].cuda(), (torch.arange(count, **i32) % 13).cuda(), offsets.cuda())
    pages = qa.kv_pages.empty(count, 16, 1, 64)
    pages.scales.zero_()
    x = (owner + 1).clamp(min=0).float()[:, None, None].expand(T, 1, 64).contiguous().cuda()
    pages.append(x, -x, batch)
    k, v = pages.read(batch, T, torch.float32)
    assert torch.allclose(k, x, rtol=2.0 ** -22, atol=0) and torch.allclose(v, -x, rtol=2.0 ** -22, atol=0)
    rows = (pages.scales[:, 0, 0] != 0).sum(1).cpu()
    assert torch.equal(rows, new.long())


def test_attend_long_context_in_parts():
    _check_attend(R.Batch([20011, 3], [1, 1], 64), 1, 4, 64, torch.float32)


@pytest.mark.parametrize("layout", ["apart", "heads first", "odd address"])
@pytest.mark.parametrize("dtype", FLOATS)
def test_attend_layouts(layout, dtype):
    batch = R.Batch([30, 5], [2, 3], 16)
    pages = _pages(*R.pool(batch, 2, 64))
    x = _rand((5, 4, 64), 1, dtype).cuda()
    if layout == "apart":
        y = torch.zeros(5, 9, 70, dtype=dtype, device="cuda")[:, 2:6, 3:67]
    elif layout == "heads first":
        y = torch.zeros(4, 5, 64, dtype=dtype, device="cuda").transpose(0, 1)
    else:
        y = torch.zeros(5 * 4 * 64 + 1, dtype=dtype, device="cuda")[1:].view(5, 4, 64)
    y.copy_(x)
    assert torch.equal(pages.attend(x, batch.gpu()), pages.attend(y, batch.gpu()))


@pytest.mark.parametrize("layout", ["apart", "heads first", "odd address", "broadcast"])
@pytest.mark.parametrize("dtype", FLOATS)
def test_attend_layouts_of_large_tiles(layout, dtype):
    batch = R.Batch([30, 5], [2, 3], 16)
    pages = _pages(*R.pool(batch, 1, 128))
    x = _rand((5, 90, 128), 1, dtype).cuda()
    if layout == "apart":
        y = torch.zeros(5, 97, 150, dtype=dtype, device="cuda")[:, 2:92, 3:131]
    elif layout == "heads first":
        y = torch.zeros(90, 5, 128, dtype=dtype, device="cuda").transpose(0, 1)
    elif layout == "odd address":
        y = torch.zeros(5 * 90 * 128 + 1, dtype=dtype, device="cuda")[1:].view(5, 90, 128)
    else:
        x = x[:, :1].repeat(1, 90, 1)
        y = x[:, :1].clone().expand(5, 90, 128)
    if layout != "broadcast":
        y.copy_(x)
    assert torch.equal(pages.attend(x, batch.gpu()), pages.attend(y, batch.gpu()))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("group", [300, 513])
def test_attend_groups_larger_than_a_tile(group, dtype):
    _check_attend(R.Batch([70, 0, 9], [1, 2, 0], 16), 2, group, 64, dtype)


@pytest.mark.parametrize("group", [2, 40])
def test_attend_large_pages(group):
    batch = R.Batch([1500, 10], [3, 3], 1024)
    _check_attend(batch, 2, group, 64, torch.bfloat16)
    _check_attend(batch, 2, group, 64, torch.bfloat16, mask=_tree(batch))


@pytest.mark.parametrize("new", [1, 60])
def test_pool_of_more_than_4_gib(new):
    """The same step in pages in front and behind 4 GiB of codes: bit for bit the same."""
    import qtpytorch_amd as qa
    H, G, D, n = 2, 4, 128, 1 << 20
    pages = qa.kv_pages.empty(n, 16, H, D)
    assert pages.codes.numel() > 1 << 32
    i32 = dict(dtype=torch.int32, device="cuda")
    table = qa.rotary_table.make(D)
    got = []
    for base in (0, n - 8):
        batch = qa.kv_batch(torch.arange(base, base + 8, **i32)[None].flip(1).contiguous(), torch.tensor([0], **i32),
                            torch.tensor([0, 60], **i32))
        q, k, v = (_rand((60, h, D), 7 + h, torch.bfloat16).cuda() for h in (H * G, H, H))
        q = pages.append(k, v, batch, rotary=table, q=q)
        step = batch._replace(lengths=torch.tensor([60 - new], **i32), offsets=torch.tensor([0, new], **i32))
        o = pages.attend(q[60 - new:], step)
        pages.keep(batch, torch.tensor([[5, 50, 20]], **i32))
        got.append((q, o, *pages.read(batch, 60)))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and torch.isfinite(got[0][1]).all()


def test_repeats_bit_for_bit():
    batch = R.Batch([5000, 300, 2], [1, 1, 1], 16)
    pages = _pages(*R.pool(batch, 2, 128))
    for group in (4, 50, 200):
        q = _rand((3, 2 * group, 128), 1, torch.bfloat16).cuda()
        first = pages.attend(q, batch.gpu())
        assert all(torch.equal(first, pages.attend(q, batch.gpu())) for _ in range(5))


def test_empty_calls():
    import qtpytorch_amd as qa
    batch = R.Batch([3, 4], [0, 0], 16)
    pages = _pages(*R.pool(batch, 2, 64))
    none = torch.zeros(0, 2, 64, device="cuda")
    assert pages.append(none, none, batch.gpu()) is None
    assert pages.attend(none, batch.gpu()).shape == (0, 2, 64)
    assert pages.read(batch.gpu(), 0)[0].shape == (0, 2, 64)
    pages.keep(batch.gpu(), torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    # rows, but no sequence has them
    x = torch.ones(4, 2, 64, device="cuda")
    before = pages.codes.clone()
    pages.append(x, x, batch.gpu())
    assert torch.equal(before, pages.codes)
    assert (pages.attend(x, batch.gpu()) == 0).all() and (pages.read(batch.gpu(), 4)[0] == 0).all()
    i32 = dict(dtype=torch.int32, device="cuda")
    nobody = qa.kv_batch(torch.zeros(0, 3, **i32), torch.zeros(0, **i32), torch.zeros(1, **i32))
    assert (pages.attend(x, nobody) == 0).all()
    pages.append(x, x, nobody)
    assert torch.equal(before, pages.codes)


# ---------------------------------------------------------------- a step as a whole
def _step(qa, pages, table, batch, q, k, v, positions=None, mask=None):
    q = pages.append(k, v, batch, rotary=table, positions=positions, q=q)
    return pages.attend(q, batch, mask=mask)


def test_prompt_tokens_and_a_tree_one_after_the_other():
    """A prompt in chunks, single tokens and a drafted tree whose path is kept give what one attention over all gives."""
    import qtpytorch_amd as qa
    H, G, D, page, n = 2, 3, 64, 16, 60
    table = qa.rotary_table.make(D, sections=(8, 12, 12))
    pages = qa.kv_pages.empty(12, page, H, D)
    i32 = dict(dtype=torch.int32, device="cuda")
    pt = torch.randperm(12, generator=R.gen(0)).int()[None].cuda()
    q, k, v = _rand((n, H * G, D), 1).cuda(), _rand((n, H, D), 2).cuda(), _rand((n, H, D), 3).cuda()
    pos = torch.randint(0, 500, (n, 3), generator=R.gen(4)).cuda()

    def batch(held, new):
        return qa.kv_batch(pt, torch.tensor([held], **i32), torch.tensor([0, new], **i32))

    out, at = [], 0
    for size in (30, 21, 1, 1, 1):
        s = slice(at, at + size)
        out.append(_step(qa, pages, table, batch(at, size), q[s], k[s], v[s], pos[s]))
        at += size
    # the last six tokens are a path in a tree of eleven
    path = torch.tensor([[0, 2, 3, 6, 9, 10]], **i32)
    mask, _ = qa.kv_tree_mask([-1, 0, 0, 2, 2, 3, 3, 4, 6, 6, 9])
    tree = torch.tensor([0, -1, 1, 2, -1, -1, 3, -1, -1, 4, 5]).cuda()  # which of the six a drafted token is

    def drafted(x):
        other = torch.randn(x[at:at + 1].shape, generator=R.gen(9)).cuda()
        return torch.where((tree >= 0).view(-1, 1, 1), x[at + tree.clamp(min=0)], other)

    tp = pos[at + tree.clamp(min=0)]
    o = _step(qa, pages, table, batch(at, 11), drafted(q), drafted(k), drafted(v), tp, mask)
    out.append(o[path[0].long()])
    pages.keep(batch(at, 11), path)
    at += 6
    assert at == n
    got = torch.cat(out)
    # all at once, from a second pool
    whole = qa.kv_pages.empty(12, page, H, D)
    want = _step(qa, whole, table, batch(0, n), q, k, v, pos)
    one, two = pages.read(batch(0, n), n, torch.float32), whole.read(batch(0, n), n, torch.float32)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    # both are within the documented error of the same values: 2^-12 of the largest is far above it in float32
    assert (got - want).abs().max() < 2.0 ** -12 * want.abs().max()


def test_step_in_a_graph():
    """Recorded once, replayed with other lengths, pages and values, with eager work between."""
    import qtpytorch_amd as qa
    H, G, D, page, B = 2, 2, 128, 16, 3
    table = qa.rotary_table.make(D)
    pages, other = qa.kv_pages.empty(40, page, H, D), qa.kv_pages.empty(40, page, H, D)
    other.codes.copy_(pages.codes)
    other.scales.copy_(pages.scales)
    batch = qa.kv_batch(torch.zeros(B, 9, dtype=torch.int32).cuda(), torch.zeros(B, dtype=torch.int32).cuda(),
                        torch.arange(B + 1, dtype=torch.int32).cuda())
    q, k, v = (torch.zeros(B, h, D, dtype=torch.bfloat16).cuda() for h in (H * G, H, H))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(qa, pages, table, batch, q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    other.codes.copy_(pages.codes)
    other.scales.copy_(pages.scales)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(qa, pages, table, batch, q, k, v)
    with torch.cuda.graph(second, pool=graph.pool()):
        again = pages.attend(q, batch)
    pt = torch.randperm(40, generator=R.gen(0))[:27].int().view(B, 9).cuda()
    batch.table.copy_(pt)
    for step in range(6):
        for t, h, s in ((q, H * G, 1), (k, H, 2), (v, H, 3)):
            t.copy_(_rand((B, h, D), 10 * step + s, torch.bfloat16))
        batch.offsets.copy_(torch.tensor([[0, 1, 2, 3], [0, 0, 1, 2], [0, 1, 1, 3]][step % 3], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        second.replay()
        want = _step(qa, other, table, batch, q, k, v)
        plain = other.attend(q, batch)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, plain)
        assert torch.equal(pages.codes, other.codes)
        batch.lengths.add_(torch.tensor([20, 1, 33], dtype=torch.int32).cuda())


def test_on_another_stream():
    import qtpytorch_amd as qa
    batch = R.Batch([300, 40], [1, 1], 16)
    pages = _pages(*R.pool(batch, 2, 64))
    q = _rand((2, 4, 64), 1).cuda()
    want = pages.attend(q, batch.gpu())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pages.attend(q, batch.gpu())
        k, v = pages.read(batch.gpu(), 2)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(k, pages.read(batch.gpu(), 2)[0])


def test_refusals():
    import qtpytorch_amd as qa
    batch = R.Batch([5], [2], 16)
    codes, scales = R.pool(batch, 2, 64)
    pages, gb = _pages(codes, scales), batch.gpu()
    x = torch.zeros(2, 2, 64).cuda()
    table = qa.rotary_table.make(64)
    for c, s, kind in ((codes.float(), scales, TypeError), (codes, scales.double(), TypeError), (codes[:, :1], scales[:, :1], ValueError),
                       (codes[..., :8, :], scales[..., :8], ValueError), (codes[..., :32], scales, ValueError),
                       (codes, scales[:1], ValueError), (codes[:, :, :0], scales[:, :, :0], ValueError)):
        with pytest.raises(kind, match="kv_pages"):
            qa.kv_pages(c.cuda(), s.cuda())
    with pytest.raises(ValueError, match="contiguous"):
        qa.kv_pages(codes.cuda().transpose(3, 4).contiguous().transpose(3, 4), scales.cuda())
    with pytest.raises(qa._lib.MXKError, match="GPU only"):
        qa.kv_pages(codes, scales)
    with pytest.raises(ValueError, match="16 bytes"):
        qa.kv_pages(torch.zeros(2048 * 2 + 1, dtype=torch.int8).cuda()[1:].view(1, 2, 1, 16, 128), torch.zeros(1, 2, 1, 16).cuda())
    with pytest.raises(TypeError, match="one type"):
        pages.append(x, x.half(), gb)
    with pytest.raises(TypeError, match="one type"):
        pages.append(x.double(), x.double(), gb)
    with pytest.raises(ValueError, match="k \\[tokens, 2, 64\\]"):
        pages.append(x[:, :1], x, gb)
    with pytest.raises(ValueError, match="one row for each"):
        pages.append(x, x[:1], gb)
    with pytest.raises(ValueError, match="rotary table"):
        pages.append(x, x, gb, q=x)
    with pytest.raises(ValueError, match="rotates 128"):
        pages.append(x, x, gb, rotary=qa.rotary_table.make(128))
    with pytest.raises(ValueError, match="positions"):
        pages.append(x, x, gb, rotary=table, positions=torch.zeros(3, dtype=torch.int64).cuda())
    with pytest.raises(TypeError, match="int32"):
        pages.append(x, x, gb._replace(lengths=gb.lengths.long()))
    with pytest.raises(ValueError, match="offsets"):
        pages.append(x, x, gb._replace(offsets=gb.offsets[:1]))
    with pytest.raises(qa._lib.MXKError, match="GPU only"):
        pages.append(x, x, gb._replace(table=gb.table.cpu()))
    with pytest.raises(ValueError, match="groups"):
        pages.attend(torch.zeros(2, 3, 64).cuda(), gb)
    with pytest.raises(ValueError, match="q \\[tokens"):
        pages.attend(torch.zeros(2, 2, 128).cuda(), gb)
    with pytest.raises(TypeError, match="int64"):
        pages.attend(x, gb, mask=torch.ones(2, 1, dtype=torch.bool).cuda())
    with pytest.raises(ValueError, match="words"):
        pages.attend(x, gb, mask=torch.ones(3, 1, dtype=torch.int64).cuda())
    with pytest.raises(ValueError, match="positive"):
        pages.attend(x, gb, scale=0.0)
    with pytest.raises(TypeError, match="int32"):
        pages.keep(gb, torch.zeros(1, 2, dtype=torch.int64).cuda())
    with pytest.raises(ValueError, match="path"):
        pages.keep(gb, torch.zeros(2, 2, dtype=torch.int32).cuda())
    with pytest.raises(qa._lib.MXKError, match="64"):
        pages.keep(gb, torch.zeros(1, 65, dtype=torch.int32).cuda())
    with pytest.raises(qa._lib.MXKError, match="dtype"):
        pages.read(gb, 2, torch.float64)
    with pytest.raises(ValueError, match="number"):
        pages.read(gb, -1)
    leaf = x.clone().requires_grad_()
    for call in (lambda t: pages.append(t, x, gb), lambda t: pages.append(x, t, gb), lambda t: pages.attend(t, gb),
                 lambda t: pages.append(x, x, gb, rotary=table, q=t)):
        with pytest.raises(qa._lib.MXKError, match="no gradient"):
            call(leaf)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(qa._lib.MXKError, match="forward-mode"):
                call(torch.autograd.forward_ad.make_dual(x, x))
        with torch.no_grad():
            call(leaf)
    with pytest.raises(qa._lib.MXKError, match="without pages"):
        qa.kv_pages.empty(0, 16, 2, 64).attend(x, gb)

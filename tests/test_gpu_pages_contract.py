"""What rotary and the paged cache do where gradients are recorded, and pools made by `empty`."""
import math

import pytest
import torch

from tests import _pages as R

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32)


def _calls(qa, pages, batch):
    """Each of a pool's calls by name."""
    T = batch.tokens
    _, _, H, _, D = pages.codes.shape
    x = torch.ones(T, H, D, device="cuda")
    gb = batch.gpu()
    return {"append": lambda: pages.append(x, x, gb), "attend": lambda: pages.attend(x, gb), "read": lambda: pages.read(gb, T),
            "keep": lambda: pages.keep(gb, torch.zeros(len(batch.held), 1, **I32).cuda())}


@pytest.mark.parametrize("call", ["append", "attend", "read", "keep"])
def test_scales_that_need_a_gradient_are_refused(call):
    import qtpytorch_amd as qa
    batch = R.Batch([5, 20], [2, 1], 16)
    codes, scales = (t.cuda() for t in R.pool(batch, 2, 64, poison=False))
    leaf = scales.clone().requires_grad_()
    run = _calls(qa, qa.kv_pages(codes, leaf), batch)[call]
    with pytest.raises(qa._lib.MXKError, match=f"kv_pages.{call} has no gradient"):
        run()
    assert torch.equal(leaf.detach(), scales)
    with torch.no_grad():
        run()
    leaf.requires_grad_(False)
    run()
    # asked for after the pool was made
    leaf.requires_grad_()
    with pytest.raises(qa._lib.MXKError, match="no gradient"):
        run()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(scales, scales.clone())
        with pytest.raises(qa._lib.MXKError, match=f"kv_pages.{call} has no forward-mode"):
            _calls(qa, qa.kv_pages(codes, dual), batch)[call]()


@pytest.mark.parametrize("call", ["append", "keep"])
def test_a_pool_that_autograd_has_saved_counts_as_changed(call):
    import qtpytorch_amd as qa
    batch = R.Batch([5, 20], [2, 1], 16)
    pages = qa.kv_pages(*(t.cuda() for t in R.pool(batch, 2, 64, poison=False)))
    w = torch.ones((), device="cuda", requires_grad=True)
    loss = (w * pages.scales).sum()
    _calls(qa, pages, batch)[call]()
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    for other in ("attend", "read"):
        loss = (w * pages.scales).sum()
        _calls(qa, pages, batch)[other]()
        loss.backward()
    with torch.inference_mode():  # tensors without versions
        pages = qa.kv_pages.empty(4, 16, 2, 64)
        _calls(qa, pages, batch)[call]()


# ---------------------------------------------------------------- a rotary table's tensors
def _turned(qa, freqs, axis, seed=1):
    x = torch.randn(5, 3, 64, generator=R.gen(seed)).cuda().requires_grad_()
    pos = torch.arange(10).view(5, 2).cuda()
    return x, qa.rotary(x, pos, qa.rotary_table(freqs, axis))


@pytest.mark.parametrize("which", ["freqs", "axis"])
def test_a_table_changed_before_the_gradient_is_an_error(which):
    import qtpytorch_amd as qa
    table = {"freqs": torch.rand(32, dtype=torch.float64).cuda(), "axis": (torch.arange(32) % 2).int().cuda()}
    x, y = _turned(qa, **table)
    table[which].mul_(0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()
    # the change counts for what is called after it
    x, y = _turned(qa, **table)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    if which == "freqs":
        assert torch.equal(y, x) and torch.equal(dx, torch.ones_like(x))


def test_a_table_whose_pairing_changes_before_the_gradient():
    import qtpytorch_amd as qa
    table = qa.rotary_table.make(64)
    x = torch.randn(5, 3, 64, generator=R.gen(1)).cuda().requires_grad_()
    pos = torch.arange(5).cuda()
    y = qa.rotary(x, pos, table)
    want = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)[0]
    table.interleaved = True
    assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], want)


def test_frequencies_that_need_a_gradient_are_refused():
    import qtpytorch_amd as qa
    freqs = torch.rand(32, dtype=torch.float64).cuda()
    leaf = freqs.clone().requires_grad_()
    table = qa.rotary_table(leaf)
    batch = R.Batch([5], [2], 16)
    pages = qa.kv_pages(*(t.cuda() for t in R.pool(batch, 2, 64, poison=False)))
    x, pos = torch.ones(2, 2, 64).cuda(), torch.arange(2).cuda()
    for name, call in (("rotary", lambda t: qa.rotary(x, pos, t)),
                       ("rotary", lambda t: qa.rotary(x.clone().requires_grad_(), pos, t)),
                       ("kv_pages.append", lambda t: pages.append(x, x, batch.gpu(), rotary=t, q=x))):
        with pytest.raises(qa._lib.MXKError, match=f"{name} towards a table's frequencies has no gradient"):
            call(table)
        with torch.no_grad():
            call(table)
        with torch.autograd.forward_ad.dual_level():
            dual = qa.rotary_table(torch.autograd.forward_ad.make_dual(freqs, freqs.clone()))
            with pytest.raises(qa._lib.MXKError, match=f"{name} towards a table's frequencies has no forward-mode"):
                call(dual)


# ---------------------------------------------------------------- pools made by empty
def test_an_empty_pool_reads_as_zeros_whatever_its_memory_held():
    import qtpytorch_amd as qa
    n, D = 20000, 64
    torch.cuda.empty_cache()
    # blocks of the sizes of the pool's tensors, as the allocator gives them out again
    before = [torch.full((m,), math.nan, device="cuda") for m in (n * 2 * 16 * D // 4, n * 2 * 16)]
    del before
    pages = qa.kv_pages.empty(n, 16, 1, D)
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = qa.kv_batch(torch.arange(n, **i32)[None], torch.tensor([0], **i32), torch.tensor([0, 16 * n], **i32))
    k, v = pages.read(batch, 16 * n, torch.float32)
    assert not k.any() and not v.any()
    one = batch._replace(lengths=torch.tensor([16 * n - 1], **i32), offsets=torch.tensor([0, 1], **i32))
    assert not pages.attend(torch.ones(1, 4, D, device="cuda"), one).any()


def test_a_step_in_a_graph_on_pools_with_values():
    """Recorded once and replayed with other lengths, pages and values over contexts that hold values, eager work between."""
    import qtpytorch_amd as qa
    H, G, D, page, B = 2, 2, 128, 16, 3
    table = qa.rotary_table.make(D)
    g = R.gen(11)
    codes = (40 * torch.randn(40, 2, H, page, D, generator=g)).round().clamp(-127, 127).to(torch.int8)
    scales = (torch.rand(40, 2, H, page, generator=g) + 0.5) / 40
    pages, other = qa.kv_pages(codes.cuda(), scales.cuda()), qa.kv_pages(codes.cuda(), scales.cuda())
    batch = qa.kv_batch(torch.zeros(B, 9, **I32).cuda(), torch.zeros(B, **I32).cuda(), torch.arange(B + 1, **I32).cuda())
    q, k, v = (torch.zeros(B, h, D, dtype=torch.bfloat16).cuda() for h in (H * G, H, H))

    def step(pages):
        return pages.attend(pages.append(k, v, batch, rotary=table, q=q), batch)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pages)
    torch.cuda.current_stream().wait_stream(side)
    step(other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(pages)
    batch.table.copy_(torch.randperm(40, generator=g)[:27].int().view(B, 9))
    last = None
    for n in range(6):
        for t, h in ((q, H * G), (k, H), (v, H)):
            t.copy_(torch.randn(B, h, D, generator=g).bfloat16())
        batch.offsets.copy_(torch.tensor([[0, 1, 2, 3], [0, 0, 1, 2], [0, 1, 1, 3]][n % 3], **I32))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        want = step(other)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(pages.codes, other.codes) and torch.equal(pages.scales, other.scales)
        rows = int(batch.offsets[-1])
        assert torch.isfinite(got).all() and (got[:rows] != 0).any(-1).all() and not got[rows:].any()
        assert last is None or not torch.equal(got, last)
        last = got
        batch.lengths.add_(torch.tensor([20, 1, 25], **I32).cuda())


# ---------------------------------------------------------------- calls that the documentation allows
@pytest.mark.parametrize("new", [1, 40])
def test_a_page_in_several_tables(new):
    """Two sequences that share a prefix's pages read and attend as two with pages of their own."""
    import qtpytorch_amd as qa
    own = R.Batch([96, 96], [new, new], 16)
    codes, scales = R.pool(own, 2, 64, poison=False)
    for i in range(6):  # the prefix's six pages have the same contents in both
        codes[own.table[1, i]], scales[own.table[1, i]] = codes[own.table[0, i]], scales[own.table[0, i]]
    pages = qa.kv_pages(codes.cuda(), scales.cuda())
    q = torch.randn(2 * new, 6, 64, generator=R.gen(1)).cuda()
    batch = own.gpu()
    shared = batch.table.clone()
    shared[1, :6] = shared[0, :6]
    both = batch._replace(table=shared)
    assert torch.equal(pages.attend(q, batch), pages.attend(q, both))
    whole = dict(lengths=torch.zeros(2, **I32).cuda(), offsets=torch.tensor([0, 96 + new, 2 * (96 + new)], **I32).cuda())
    one, two = (pages.read(b._replace(**whole), 2 * (96 + new)) for b in (batch, both))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_packed_keys_values_and_queries_are_their_values():
    import qtpytorch_amd as qa
    batch = R.Batch([5, 20], [2, 3], 16)
    k, v, q = (qa.mx_tensor.quantize(torch.randn(5, h, 64, generator=R.gen(h)).cuda(), "int8d") for h in (2, 2, 6))
    table = qa.rotary_table.make(64)
    one, two = (qa.kv_pages(*(t.cuda() for t in R.pool(batch, 2, 64, poison=False))) for _ in range(2))
    a = one.append(k, v, batch.gpu(), rotary=table, q=q)
    b = two.append(k.dequantize(), v.dequantize(), batch.gpu(), rotary=table, q=q.dequantize())
    assert torch.equal(a, b) and torch.equal(one.codes, two.codes) and torch.equal(one.scales, two.scales)
    assert torch.equal(one.attend(q, batch.gpu()), one.attend(q.dequantize(), batch.gpu()))


@pytest.mark.parametrize("group", [2, 40])
def test_masks_of_any_strides(group):
    import qtpytorch_amd as qa
    batch = R.Batch([30, 7], [9, 9], 16)
    pages = qa.kv_pages(*(t.cuda() for t in R.pool(batch, 1, 64)))
    q = torch.randn(18, group, 64, generator=R.gen(1)).cuda()
    mask = torch.randint(-(1 << 62), 1 << 62, (18, 2), generator=R.gen(2)).cuda()
    wide = torch.zeros(18, 5, dtype=torch.int64).cuda()
    wide[:, 1::2] = mask
    want = pages.attend(q, batch.gpu(), mask=mask)
    assert torch.equal(pages.attend(q, batch.gpu(), mask=wide[:, 1::2]), want)
    assert torch.equal(pages.attend(q, batch.gpu(), mask=mask.t().contiguous().t()), want)
    row = mask[:1]
    assert torch.equal(pages.attend(q, batch.gpu(), mask=row.expand(18, 2)), pages.attend(q, batch.gpu(), mask=row.repeat(18, 1)))


@pytest.mark.parametrize("group", [2, 40])
def test_two_streams_at_once_over_one_pool(group):
    import qtpytorch_amd as qa
    batch = R.Batch([3000, 40, 700], [5, 1, 3], 16)
    pages = qa.kv_pages(*(t.cuda() for t in R.pool(batch, 2, 64)))
    gb = batch.gpu()
    q = [torch.randn(9, 2 * group, 64, generator=R.gen(i)).cuda() for i in range(2)]
    want = [pages.attend(x, gb) for x in q]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in q]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(side):
            with torch.cuda.stream(s):
                got[i].append(pages.attend(q[i], gb))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for many, w in zip(got, want) for g in many)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name,held,new", [("tokens beside a chunk", [(7 * i) % 90 for i in range(30)] + [50], [1] * 30 + [140]),
                                           ("a chunk beside many tokens", [(11 * i) % 60 for i in range(90)] + [0], [1] * 90 + [70]),
                                           ("a chunk among idle slots", [0] * 40 + [90] + [17] * 60, [0] * 40 + [130] + [0] * 60),
                                           ("a tree-sized step among idle slots", [3] * 70 + [200], [0] * 70 + [9])])
def test_steps_of_several_kinds_at_once(name, held, new, dtype):
    """Single tokens, chunks and idle slots of one call: every row is within its own bounds, whichever tiles it takes."""
    import qtpytorch_amd as qa
    batch = R.Batch(held, new, 16, front=1, back=2)
    codes, scales = R.pool(batch, 1, 64)
    q = torch.randn(batch.tokens, 4, 64, generator=R.gen(5)).to(dtype)
    want, error = R.attend(batch, codes, scales, q)
    R.near(qa.kv_pages(codes.cuda(), scales.cuda()).attend(q.cuda(), batch.gpu()), want, error)

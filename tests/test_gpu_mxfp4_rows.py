"""Rows of x that lie anywhere for the kernel that packs them itself, and the products
that fit no tile kernel's 32-bit offsets."""
import pytest
import torch

from tests import _mxfp4 as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,apart,at", [(1, 40, 98, 0, 3), (2, 17, 98, 1, 1), (5, 64, 250, 3, 5), (16, 33, 514, 7, 1),
                                            (16, 520, 2050, 1, 1), (7, 48, 8190, 3, 2)])
def test_few_rows_at_odd_addresses_with_ragged_ends(m, n, k, apart, at, dtype):
    """Rows that start on one element's alignment and end inside a 16-byte load; what lies around them is NaN."""
    import qtpytorch_amd as qa
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(m, k, generator=g).to(dtype), torch.randn(n, k, generator=g) * 0.1
    big = torch.full((m, at + k + apart), float("nan"), dtype=dtype)
    big[:, at:at + k] = x
    rows = big.cuda()[:, at:at + k]
    assert rows.data_ptr() % 16
    y = qa.mxfp4_linear(rows, qa.mxfp4_quantize(w.cuda()))
    rx, rw = R.rounded(x), R.rounded(w)
    R.assert_close(y, rx @ rw.t(), rx.abs() @ rw.abs().t(), k / 32 + 2)


def test_gathered_rows_past_the_tile_kernels_offsets():
    """By expert from more than 2^30 bytes of packed rows: the plain kernel."""
    import qtpytorch_amd as qa
    tokens, k, n, E = (1 << 19) + 300, 4096, 40, 3
    assert tokens * k // 2 > 1 << 30
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(tokens, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = qa.mxfp4_quantize(torch.randn(E, n, k, device="cuda", generator=g) * 0.05)
    bias = torch.randn(E, n, device="cuda", generator=g)
    ids = torch.randint(-1, E, (tokens, 1), device="cuda", generator=g)
    plan = qa.expert_sort(ids, E)
    y = qa.expert_linear(x, w, plan, bias, gather=True)
    rw = w.dequantize().double()
    used = int(plan.offsets[-1])
    assert not y[used:].any()
    for at in ([0, 1, 63, 64], list(range(used - 70, used)), [used // 2, used // 3]):
        at = torch.tensor(at, device="cuda")
        token = plan.order[at].long()
        rx = qa.mxfp4_quantize(x[token]).dequantize().double()
        e = ids[token, 0]
        ref = (rx[:, None] * rw[e]).sum(-1) + bias[e].double()
        mass = (rx[:, None] * rw[e]).abs().sum(-1) + bias[e].double().abs()
        R.assert_close(y[at], ref.cpu(), mass.cpu(), k / 32 + 3)


def test_experts_without_columns():
    """K = 0: each expert's bias, zeros in rows without one."""
    import qtpytorch_amd as qa
    ids = torch.tensor([[0, 2], [-1, 1], [2, 2], [1, 0]]).cuda()
    plan = qa.expert_sort(ids, 3)
    bias = torch.arange(1.0, 22.0).view(3, 7).cuda()
    y = qa.expert_linear(torch.empty(4, 0).cuda(), qa.mxfp4_quantize(torch.empty(3, 7, 0).cuda()), plan, bias, gather=True)
    want = torch.zeros(8, 7).cuda()
    for e in range(3):
        want[int(plan.offsets[e]):int(plan.offsets[e + 1])] = bias[e]
    assert torch.equal(y, want)

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

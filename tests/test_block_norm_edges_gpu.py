"""The norms between two blocks on rows and shapes at the end of what they take."""
import pytest
import torch

from oracle import blocks
from tests.blocks_util import DEV, close
from tests.test_block_norm_gpu import make, run, sizes

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize('types', [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize('D', [40, 96, 300, 1000, 1030, 4096, 8192])
def test_constant_rows_with_a_norm_behind_the_block(fwp, D, types):
    """Rows of one value each, exact in every sum: both normalised rows are zero, forward and backward, and so are the gradients of the
    weights, whatever 1 / sqrt(eps) makes of a rounding.  (The oracle's own means are off by 2^-53, so it is not asked for those two.)"""
    a, gy, gr = make(1, 2, 3, D, *types, parts=('residual', 'post'))
    a['x'], a['residual'] = torch.full_like(a['x'], 3.75), torch.full_like(a['residual'], 1.25)
    a['post_bias'] = torch.full_like(a['post_bias'], 0.5)
    y, r, grads = run(fwp, a, gy, gr)
    assert torch.equal(r, torch.full_like(r, 1.75)) and torch.equal(y, a['bias'].to(y.dtype).expand_as(y))
    assert not grads.pop('weight').any() and not grads.pop('post_weight').any()
    sums = blocks.block_norm(**a, gy=gy, gr=gr)[2]
    for k, g in grads.items():
        close('gradient of ' + k, g, sums[k][0], sizes(*sums[k], D))


@pytest.mark.parametrize('shape', [(2, 0), (2, 3, 0), (2, 3, 4, 0), (2, 0, 4, 8)])
def test_rows_without_elements(fwp, shape):
    x, res, gate = (torch.zeros(shape, device=DEV).requires_grad_() for _ in range(3))
    w = torch.ones(shape[-1], device=DEV).requires_grad_()
    y, r = fwp.block_norm(x, w, residual=res, gate=gate)
    assert y.shape == r.shape == shape
    grads = torch.autograd.grad([y, r], [x, w, res, gate], [torch.ones_like(y), torch.ones_like(r)])
    assert [g.shape for g in grads] == [t.shape for t in (x, w, res, gate)] and not any(g.any() for g in grads)

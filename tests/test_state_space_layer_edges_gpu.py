"""The state-space layer's operators where a test of their outputs alone would not see it: memories by value, tensors whose rows are far
apart, forward and backward."""
import pytest
import torch

from tests import util
from tests.blocks_util import DEV
from tests.test_state_space_layer_gpu import arguments, memories, models, together

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def test_memories_token_by_token_are_the_segments(fwp):
    gpu, _ = models(True)
    gpu.pos_emb.inv_freq.zero_()        # positions count backwards from the end of a segment
    tokens = torch.randint(0, 50, (20, 5), generator=util.gen(4)).to(DEV)
    with torch.no_grad():
        _, end = gpu(tokens[:-1], tokens[1:], None, carry_over_fast_weight=True)
        mems = None
        for t in range(19):
            _, mems = gpu(tokens[t:t + 1], tokens[t + 1:t + 2], mems, carry_over_fast_weight=True)
    for p, q in zip(mems, end):
        assert all(s.shape == t.shape and util.max_abs(s, t) <= 1e-4 * (1 + t.abs().max().item()) for s, t in zip(p, q))
        assert all(t.abs().max() > 0 for t in q)


def training(fwp, a, gy):
    mem = memories(a['x'].shape[0], a['x'].shape[2])
    leaves = {k: t.detach().requires_grad_() for k, t in a.items()}
    y, r = together(fwp, leaves, *mem)
    return [y.detach(), r.detach(), *mem] + list(torch.autograd.grad([y, r], list(leaves.values()), [gy, gy]))


@pytest.mark.parametrize('apart', ['sequences', 'steps'])
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_a_training_step_beyond_31_bits(fwp, dtype, apart):
    """Sequences more than 2^31 elements apart, or steps that reach beyond 2^31 from the sequence's first."""
    N, L, D = (2, 9, 64) if apart == 'sequences' else (1, 9, 64)
    sN, sL = (2 ** 31 + 64, D) if apart == 'sequences' else (0, 2 ** 28 + 64)
    a = arguments(9, N, L, D, 16, dtype)
    gy = torch.randn(N, L, D, generator=util.gen(10)).to(dtype).to(DEV)
    ref = training(fwp, a, gy)
    room = torch.empty((N - 1) * sN + (L - 1) * sL + D, dtype=dtype, device=DEV)
    far = room.as_strided((N, L, D), (sN, sL, 1))
    for k in ('x', 'dt', 'z', 'res', 'gy'):
        far.copy_(gy if k == 'gy' else a[k])
        got = training(fwp, a, far) if k == 'gy' else training(fwp, dict(a, **{k: far}), gy)
        assert all(torch.equal(p, q) for p, q in zip(got, ref)), k

"""The selective scan where a form of it could leave the definition: growing and infinite states, rates without bound, long sequences."""
import pytest
import torch

from oracle import blocks
from recurrent_fwp_b200 import _lib
from tests import util
from tests.blocks_util import DEV, close
from tests.test_selective_scan_gpu import check, make, run

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(params=[0, 128, 1 << 20], ids=['automatic', 'spans of 128', 'one span'])
def chunk(request):
    _lib.tune('scan.chunk', request.param)
    yield request.param
    _lib.tune('scan.chunk', 0)


def growing(seed, N, L, D=40, S=16, **kw):
    """Steps of factors e^0.9 to e: 128 of them pass the range of a float, forty do not."""
    a, gy = make(seed, N, L, D, S, bias=False, **kw)
    a['dt'] = torch.ones_like(a['dt'])
    a['A'] = 0.9 + 0.1 * torch.rand(D, S, generator=util.gen(seed)).to(DEV)
    return a, gy


def test_states_that_grow_from_zero(fwp, chunk):
    """Inputs that start late and gradients that end early: zero states and gradients pass spans whose factor is infinite.  Forty steps of
    growth have at most 6 U each (argument 2, exponential 3, product 1): within the 4 U for each of 300 steps that the bound has."""
    a, gy = growing(1, 2, 300, state=False)
    a['x'][:, :260] = 0
    gy[:, 40:] = 0
    check(fwp, a, gy, softplus=False)


def test_small_states_that_grow(fwp, chunk):
    """1e-30 grows by e^140 to 1e31: finite, though the factor alone is not."""
    a, gy = growing(2, 2, 150)
    a['x'] = torch.zeros_like(a['x'])
    a['state'] = a['state'].sign() * 1e-30
    gy[:, 40:] = 0
    with torch.no_grad():
        ref = a['state'].double() * torch.exp(150 * a['A'].double())
        state = a['state'].clone()
        out = fwp.selective_scan(**dict(a, state=state), softplus=False)
    assert torch.isfinite(out).all()
    # 150 steps (or a span's factor at an argument of 128 log2(e), off by 2^-24 of it) of 6 U each
    assert ((state.double() / ref) - 1).abs().max() <= 150 * 6 * 2.0 ** -24


def test_infinite_states_stay_infinite(fwp, chunk):
    """A decaying state that is infinite once stays so step after step; a span's factor of zero makes no NaN of it."""
    a, _ = make(3, 2, 300, 40, 16)
    a['dt'], a['dt_bias'], a['A'] = torch.ones_like(a['dt']), None, -1 + 0 * a['A']
    a['state'][1, 7, 3] = float('inf')
    state = a['state'].clone()
    with torch.no_grad():
        fwp.selective_scan(**dict(a, state=state), softplus=False)
    assert torch.isinf(state[1, 7, 3])
    state[1, 7, 3] = 0
    assert torch.isfinite(state).all()


@pytest.mark.parametrize('lengths', [None, 'inside'])
@pytest.mark.parametrize('L', [1, 12, 300])
def test_states_that_keep_nothing(fwp, chunk, L, lengths):
    """A of minus infinity: the state is the last step's input alone, and steps behind the end leave it.  In the definition -1e30 stands for it:
    its gradient of the step size would be zero times infinity."""
    a, gy = make(4, 3, L, 24, 16, lengths=lengths)
    a['A'][::3, 5] = -1e30
    b = dict(a, A=torch.where(a['A'] < -1e29, -float('inf'), a['A']))
    ref, end, sums = blocks.selective_scan(**a, gy=gy)
    out, state, grads = run(fwp, b, gy)
    close('out', out, ref, steps=L)
    close('state', state, end, steps=L)
    for k, g in grads.items():
        close('gradient of ' + k, g, *sums[k], steps=L)
    state = a['state'].clone()
    with torch.no_grad():
        close('out', fwp.selective_scan(**dict(b, state=state)), ref, steps=L)
    close('state', state, end, steps=L)

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


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize('band', [(0.002, 0.1), (0.0001, 0.002)])
def test_the_mean_error_of_a_decay(fwp, band):
    """A slow channel multiplies a thousand decays, so their mean error is what its state shows: -9e-9 for arguments of the base-2 exponential
    between -0.1 and -0.002, +5e-9 towards zero (the instruction by itself: -19e-9 and -5e-9).  65536 states of 64 steps: the mean's own
    deviation is below 1e-10 (a step rounds to within 6e-8), so 12e-9 tells them apart and holds both."""
    L, M, S = 64, 4096, 16
    g = util.gen(5)
    lo, hi = (torch.tensor(b).log() for b in band)
    A = -torch.exp(lo + torch.rand(M, S, generator=g) * (hi - lo)).to(DEV) * 0.6931471805599453
    dt = (1 + 0.1 * torch.randn(1, L, M, generator=g)).to(DEV)
    state, zero = torch.ones(1, M, S, device=DEV), torch.zeros(1, L, M, device=DEV)
    _lib.tune('scan.chunk', 1 << 20)
    try:
        with torch.no_grad():
            fwp.selective_scan(zero, dt, A, zero[..., :S], zero[..., :S], state=state, softplus=False)
    finally:
        _lib.tune('scan.chunk', 0)
    ref = torch.exp(dt.double().sum(1)[..., None] * A.double())
    assert abs((state.double() / ref - 1).mean().item() / L) <= 12e-9


def test_long_sequences_to_the_accuracy_of_their_decays(fwp, chunk):
    """2048 steps of channels that keep 10 to 500 of them.  A state that keeps T steps is off by T times the decays' mean error; its square
    grows like T, so over T spread evenly on a logarithmic scale the 2-norm is off by 500 / sqrt(3) mean errors of 9e-9: 2.6e-6.  The
    gradient of A is made of two such recurrences: twice that."""
    g = util.gen(6)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)         # noqa: E731
    N, L, M, S = 1, 2048, 32, 16
    rate = torch.exp(torch.rand(M, S, generator=g) * torch.tensor(50.).log()).to(DEV) * 0.002
    a = dict(x=r(N, L, M), dt=0.1 * r(N, L, M), A=-rate / 0.05, B=r(N, L, S), C=r(N, L, S), D=r(M), z=r(N, L, M),
             dt_bias=torch.full((M,), -2.97, device=DEV), state=r(N, M, S))      # softplus(-2.97) = 0.05
    gy = r(N, L, M)
    ref, end, sums = blocks.selective_scan(**a, gy=gy)
    out, state, grads = run(fwp, a, gy)
    most = 500 / 3 ** 0.5 * 9e-9
    assert rel(out, ref) <= most and rel(state, end) <= most
    for k, t in grads.items():
        assert rel(t, sums[k][0]) <= (2 * most if k == 'A' else most), k


def test_a_training_step_of_a_wide_layer(fwp):
    """8 x 2048 steps of 2048 channels in bf16, step sizes over 0.001 ... 0.1 and rates 1 ... 16: a few channels, which are recurrences of
    their own, against the definition.  bf16 results are off by half a step of 2^-8 each; the slowest channel keeps 1000 steps (see above)."""
    g = util.gen(7)
    N, L, M, S = 8, 2048, 2048, 16
    cuda = torch.Generator(device=DEV)
    cuda.manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=cuda, device=DEV).to(BF16)         # noqa: E731
    step = torch.exp(torch.rand(M, generator=g) * torch.tensor(100.).log()).to(DEV) * 0.001
    a = dict(x=r(N, L, M), dt=r(N, L, M), A=-torch.arange(1., S + 1, device=DEV).repeat(M, 1), B=r(N, L, S), C=r(N, L, S),
             D=torch.ones(M, device=DEV), z=r(N, L, M), dt_bias=torch.log(torch.expm1(step)), state=r(N, M, S).float() * 0.1, lengths=None)
    gy = r(N, L, M)
    out, state, grads = run(fwp, a, gy)
    some = torch.randperm(M, generator=g)[:12].to(DEV)
    b = {k: a[k][..., some] if k in ('x', 'dt', 'z', 'dt_bias', 'D') else a[k] for k in a}
    b.update(A=a['A'][some], state=a['state'][:, some])
    ref, end, sums = blocks.selective_scan(**b, gy=gy[..., some])
    slow = 1000 / 3 ** 0.5 * 9e-9
    assert rel(out[..., some], ref) <= 2 ** -8 and rel(state[:, some], end) <= slow
    for k in ('x', 'dt', 'z'):
        assert rel(grads[k][..., some], sums[k][0]) <= 2 ** -8, k
    for k in ('A', 'D', 'dt_bias'):
        assert rel(grads[k][some], sums[k][0]) <= 2 * slow, k


def test_the_relative_error_of_small_step_sizes(fwp):
    """softplus: 3e-7 + 7e-8 |x| relative, which comes from the product in the exponential's argument, down to -87; zero below -87.4."""
    x = torch.cat([torch.linspace(-100, 30, 1 << 20), torch.linspace(-1, 1, 1 << 18)]).to(DEV)
    M = 4096
    state, one = torch.zeros(x.numel() // M, M, 1, device=DEV), torch.ones(x.numel() // M, 1, M, device=DEV)
    with torch.no_grad():       # one step from zero with unit inputs leaves the step size itself
        fwp.selective_scan(one, x.view(-1, 1, M), -torch.ones(M, 1, device=DEV), one[..., :1], one[..., :1], state=state)
    got, x = state.flatten().double(), x.double()
    ref = x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))
    kept = x >= -87
    assert (((got - ref) / ref).abs() <= 3e-7 + 7e-8 * x.abs())[kept].all()
    assert not got[x < -87.4].any()

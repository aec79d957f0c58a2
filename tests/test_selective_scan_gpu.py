"""The selective scan against its definition in 64 bits: outputs, carried states and every gradient."""
import pytest
import torch

from oracle import blocks
from tests import util
from tests.blocks_util import DEV, close, lengths_of, streams

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, N, L, D, S, G=1, dtype=F32, layout='packed', lengths=None, z=True, skip=True, bias=True, state=True, flat=False):
    g = util.gen(seed)
    x, zz, gy = streams(g, N, L, [D, D, D], dtype, layout)
    dt, B, C = streams(g, N, L, [D, G * S, G * S], dtype, layout)
    if not (flat and G == 1):
        B, C = B.unflatten(-1, (G, S)), C.unflatten(-1, (G, S))
    dev = lambda t: t.to(DEV)           # noqa: E731
    a = dict(x=x, dt=dt, A=dev(-torch.rand(D, S, generator=g) * 4 - 0.05), B=B, C=C,
             D=dev(torch.randn(D, generator=g)) if skip else None, z=zz if z else None,
             dt_bias=dev(torch.randn(D, generator=g) - 2) if bias else None,
             state=dev(torch.randn(N, D, S, generator=g)) if state else None, lengths=lengths_of(lengths, N, L, g))
    return a, gy


def leaves_of(a):
    return {k: t for k, t in a.items() if isinstance(t, torch.Tensor) and k not in ('state', 'lengths')}


def run(fwp, a, gy, **kw):
    b = dict(a)
    for k, t in leaves_of(a).items():
        b[k] = t.detach().requires_grad_()
    if a['state'] is not None:
        b['state'] = a['state'].clone()
    out = fwp.selective_scan(**b, **kw)
    grads = dict(zip(leaves_of(a), torch.autograd.grad(out, [b[k] for k in leaves_of(a)], gy)))
    return out.detach(), b['state'], grads


def check(fwp, a, gy, **kw):
    ref, end, sums = blocks.selective_scan(**a, gy=gy, **kw)
    L = a['x'].shape[1]
    with torch.no_grad():
        state = None if a['state'] is None else a['state'].clone()
        out = fwp.selective_scan(**dict(a, state=state), **kw)
    close('out', out, ref, steps=L)
    if state is not None:
        close('state', state, end, steps=L)
    out, state, grads = run(fwp, a, gy, **kw)
    close('out', out, ref, steps=L)
    if state is not None:
        close('state', state, end, steps=L)
    for k, g in grads.items():
        assert g.dtype == a[k].dtype and g.shape == a[k].shape
        close('gradient of ' + k, g, sums[k][0], sums[k][1], steps=L)


SHAPES = [  # N, L, D, S, G
    (1, 1, 1, 1, 1), (2, 2, 3, 2, 1), (3, 7, 8, 4, 1), (2, 8, 33, 16, 1), (2, 9, 64, 16, 2), (1, 31, 100, 12, 4), (3, 33, 20, 8, 1),
    (2, 40, 36, 3, 3), (1, 65, 18, 32, 1), (2, 64, 70, 24, 1), (2, 37, 10, 64, 2), (1, 130, 130, 16, 1), (4, 17, 9, 5, 9), (2, 50, 12, 61, 1)]


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', SHAPES)
def test_against_the_definition(fwp, shape, dtype):
    N, L, D, S, G = shape
    check(fwp, *make(1, N, L, D, S, G, dtype))
    check(fwp, *make(2, N, L, D, S, G, dtype, layout='sliced', lengths='inside'))
    check(fwp, *make(22, N, L, D, S, G, dtype, layout='expanded'))


@pytest.mark.parametrize('leave_out', ['z', 'skip', 'bias', 'state', 'all'])
def test_optional_arguments(fwp, leave_out):
    kw = {k: False for k in ('z', 'skip', 'bias', 'state') if leave_out in (k, 'all')}
    check(fwp, *make(3, 2, 21, 40, 16, flat=True, **kw))
    check(fwp, *make(4, 2, 1, 40, 16, flat=True, **kw))


def test_without_softplus(fwp):
    a, gy = make(5, 2, 19, 24, 16)
    a['dt'] = a['dt'].abs() * 0.1
    a['dt_bias'] = a['dt_bias'].abs() * 0.1
    check(fwp, a, gy, softplus=False)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('S', [4, 8, 16, 32, 64, 11])
def test_many_channels(fwp, S, dtype):
    """Enough sequences for the form that takes several channels per lane."""
    check(fwp, *make(6, 620, 11, 64, S, 1, dtype, layout='sliced', lengths='inside'))


@pytest.mark.parametrize('chunk', [32, 64])
@pytest.mark.parametrize('shape', [(2, 161, 20, 16, 1), (1, 97, 70, 7, 2), (2, 200, 6, 64, 1), (3, 129, 40, 4, 1)])
def test_spans_side_by_side(fwp, shape, chunk):
    """Time cut into spans, forward and backward, with sequences that end inside them or before them."""
    from recurrent_fwp_b200 import _lib
    try:
        _lib.tune('scan.chunk', chunk)
        N, L, D, S, G = shape
        check(fwp, *make(7, N, L, D, S, G, lengths='inside'))
        check(fwp, *make(8, N, L, D, S, G, dtype=BF16, state=False))
    finally:
        _lib.tune('scan.chunk', 0)


def test_few_channels_take_spans_by_themselves(fwp):
    check(fwp, *make(9, 1, 700, 48, 16, layout='sliced'))


def test_extreme_step_sizes(fwp):
    """Step sizes from 1e-9 to 100 (softplus far from zero on both sides): relative accuracy where they are tiny."""
    a, gy = make(10, 2, 6, 64, 16, bias=False)
    a['dt'] = torch.linspace(-20, 100, a['dt'].numel(), device=DEV).view(a['dt'].shape)
    a['A'] = a['A'] * 0.01
    check(fwp, a, gy)
    a['x'] = a['x'] * 0 + 1
    a['state'], a['z'], a['D'] = torch.zeros_like(a['state']), None, None
    a['dt'] = torch.full_like(a['dt'], -18.)
    a['B'] = torch.ones_like(a['B'])
    state = a['state'].clone()
    fwp.selective_scan(**dict(a, x=a['x'][:, :1], dt=a['dt'][:, :1], B=a['B'][:, :1], C=a['C'][:, :1], state=state))
    # h = log(1 + e^-18), to 64 U of itself
    assert ((state.double() / torch.log1p(torch.exp(torch.tensor(-18., dtype=torch.float64))).item()) - 1).abs().max() < 64 * 2.0 ** -24


def test_step_sizes_of_minus_infinity_leave_the_state(fwp):
    a, gy = make(21, 2, 12, 40, 16, bias=False)
    for L in (12, 1):
        b = {k: t[:, :L].clone() if k in ('x', 'dt', 'z', 'B', 'C') else t for k, t in a.items()}
        b['dt'][0] = -float('inf')
        b['dt'][1, :, :20] = torch.finfo(F32).min
        out, state, grads = run(fwp, b, gy[:, :L])
        assert torch.equal(state[0], a['state'][0]) and torch.equal(state[1, :20], a['state'][1, :20])
        assert torch.isfinite(out).all() and not grads['dt'][0].any() and all(torch.isfinite(g).all() for g in grads.values())


def test_lengths_outside_the_range_and_as_int64(fwp):
    a, gy = make(11, 4, 23, 33, 16, lengths='outside')
    check(fwp, a, gy)
    check(fwp, dict(a, lengths=a['lengths'].long() + (a['lengths'] > 23).long() * 2 ** 40), gy)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('L', [1, 21])
@pytest.mark.parametrize('S', [16, 6])
def test_steps_behind_the_end_are_not_read(fwp, S, L, dtype):
    a, gy = make(12, 5, L, 40, S, dtype=dtype, lengths='inside')
    ref = run(fwp, a, gy)
    behind = (torch.arange(L, device=DEV) >= a['lengths'][:, None])
    for fill in (float('nan'), float('inf'), torch.finfo(dtype).min):
        b = dict(a)
        for k in ('x', 'dt', 'z', 'B', 'C'):
            b[k] = a[k].clone()
            b[k][behind] = fill
        bad = gy.clone()
        bad[behind] = fill
        got = run(fwp, b, bad)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        for k in ref[2]:
            assert torch.equal(got[2][k], ref[2][k]), k
    assert not ref[0][behind].any()
    ended = a['lengths'] == 0
    assert torch.equal(ref[1][ended], a['state'][ended])


@pytest.mark.parametrize('S', [16, 6])
def test_a_bad_channel_stays_by_itself(fwp, S):
    """NaN and Inf in one channel's stream reach that channel's outputs and states, and of the others only gradients that sum over channels."""
    for fill in (float('nan'), float('inf')):
        a, gy = make(13, 2, 20, 40, S)
        ref = run(fwp, a, gy)
        b = dict(a, x=a['x'].clone())
        b['x'][1, 5, 17] = fill
        out, state, _ = run(fwp, b, gy)
        keep = torch.ones(2, 20, 40, dtype=torch.bool, device=DEV)
        keep[1, 5:, 17] = False
        assert torch.equal(out[keep], ref[0][keep]) and not torch.isfinite(out[1, 5, 17])
        good = torch.ones(2, 40, dtype=torch.bool, device=DEV)
        good[1, 17] = False
        assert torch.equal(state[good], ref[1][good])


def test_segments_and_single_steps_follow_on(fwp):
    """A sequence in one call, in segments, and token by token: the same outputs and end state to rounding."""
    a, _ = make(14, 3, 70, 48, 16, layout='sliced')
    cut = lambda lo, hi, state: {k: t[:, lo:hi] if k in ('x', 'dt', 'z', 'B', 'C') else t for k, t in dict(a, state=state).items()}  # noqa: E731
    with torch.no_grad():
        ref, end, _ = blocks.selective_scan(**a)
        for borders in ([0, 70], [0, 13, 14, 56, 70], list(range(71))):
            state = a['state'].clone()
            out = torch.cat([fwp.selective_scan(**cut(lo, hi, state)) for lo, hi in zip(borders, borders[1:])], 1)
            close('out', out, ref, steps=70)
            close('state', state, end, steps=70)


def test_empty_calls(fwp):
    for N, L, D in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        a, gy = make(15, max(N, 1), max(L, 1), max(D, 1), 16)
        for k in ('x', 'dt', 'z'):
            a[k] = a[k][:N, :L, :D]
        for k in ('B', 'C'):
            a[k] = a[k][:N, :L]
        a.update(A=a['A'][:D], D=a['D'][:D], dt_bias=a['dt_bias'][:D], state=a['state'][:N, :D])
        out, state, grads = run(fwp, a, gy[:N, :L, :D])
        assert out.shape == (N, L, D) and torch.equal(state, a['state'])
        for k, g in grads.items():
            assert g.shape == a[k].shape and not g.any()


def test_results_do_not_change_from_run_to_run(fwp):
    a, gy = make(16, 6, 120, 200, 16, dtype=BF16)
    first = run(fwp, a, gy)
    for _ in range(3):
        again = run(fwp, a, gy)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])


def test_states_through_strides(fwp):
    """A batch prefix of a larger state, and a state whose channels are a slice: the rest stays as it is."""
    a, _ = make(17, 3, 9, 20, 16)
    whole = torch.randn(5, 24, 16, generator=util.gen(18)).to(DEV)
    for L in (9, 1):
        b = {k: t[:, :L] if k in ('x', 'dt', 'z', 'B', 'C') else t for k, t in a.items()}
        room = whole.clone()
        state = whole[:3, 2:22].clone()
        with torch.no_grad():
            ref = fwp.selective_scan(**dict(b, state=state))
            out = fwp.selective_scan(**dict(b, state=room[:3, 2:22]))
        assert torch.equal(out, ref) and torch.equal(room[:3, 2:22], state)
        room[:3, 2:22] = whole[:3, 2:22]
        assert torch.equal(room, whole)


def test_gradients_against_differences(fwp):
    """The gradient along a random direction against a central difference of the 64-bit loss."""
    a, gy = make(19, 2, 30, 24, 16)
    _, _, grads = run(fwp, a, gy)
    for k, t in leaves_of(a).items():
        v = torch.randn(t.shape, generator=util.gen(20)).to(DEV).double()
        h = 1e-5
        loss = [(blocks.selective_scan(**{q: (s.double() + e * v if q == k else s) for q, s in a.items()})[0] * gy.double()).sum() for e in (h, -h)]
        diff = ((loss[0] - loss[1]) / (2 * h)).item()
        along = (grads[k].double() * v).sum().item()
        size = (grads[k].double() * v).abs().sum().item()
        assert abs(along - diff) <= (64 + 4 * 30) * 2.0 ** -24 * size + 1e-6 * abs(diff) + 1e-5, k

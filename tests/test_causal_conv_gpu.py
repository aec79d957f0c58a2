"""The short causal convolution against its definition in 64 bits: outputs, carried windows and gradients."""
import pytest
import torch

from oracle import blocks
from tests import util
from tests.blocks_util import DEV, close, lengths_of, streams

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, N, L, D, K, dtype=F32, layout='packed', lengths=None, bias=True, state=True):
    g = util.gen(seed)
    x, gy = streams(g, N, L, [D, D], dtype, layout)
    a = dict(x=x, weight=torch.randn(D, K, generator=g).to(DEV), bias=torch.randn(D, generator=g).to(DEV) if bias else None,
             state=torch.randn(N, K - 1, D, generator=g).to(DEV) if state else None, lengths=lengths_of(lengths, N, L, g))
    return a, gy


def run(fwp, a, gy, **kw):
    names = [k for k in ('x', 'weight', 'bias') if a[k] is not None]
    b = dict(a, **{k: a[k].detach().requires_grad_() for k in names})
    if a['state'] is not None:
        b['state'] = a['state'].clone()
    out = fwp.causal_conv(**b, **kw)
    return out.detach(), b['state'], dict(zip(names, torch.autograd.grad(out, [b[k] for k in names], gy)))


def check(fwp, a, gy, **kw):
    ref, end, sums = blocks.causal_conv(**a, gy=gy, **kw)
    with torch.no_grad():
        state = None if a['state'] is None else a['state'].clone()
        close('out', fwp.causal_conv(**dict(a, state=state), **kw), ref)
    out, after, grads = run(fwp, a, gy, **kw)
    close('out', out, ref)
    for s in (state, after):
        assert s is None or torch.equal(s.double(), end)
    for k, g in grads.items():
        assert g.dtype == a[k].dtype and g.shape == a[k].shape
        close('gradient of ' + k, g, *sums[k], steps=16)       # sums of up to a thousand terms, 64 to a lane before they are joined


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('K', [1, 2, 3, 4, 5, 6, 7, 8])
def test_against_the_definition(fwp, K, dtype):
    for N, L, D in ((1, 1, 1), (2, 2, 5), (3, 7, 128), (2, 9, 132), (1, 65, 33), (2, 130, 12)):
        check(fwp, *make(1, N, L, D, K, dtype))
        check(fwp, *make(2, N, L, D, K, dtype, layout='sliced', lengths='inside'))


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_long_and_wide(fwp, dtype):
    check(fwp, *make(3, 1, 1000, 1028, 4, dtype))
    check(fwp, *make(4, 40, 24, 1024, 4, dtype, lengths='outside'))


@pytest.mark.parametrize('layout', ['packed', 'expanded'])
def test_optional_arguments(fwp, layout):
    check(fwp, *make(5, 2, 21, 40, 4, layout=layout, bias=False, state=False))
    check(fwp, *make(6, 2, 21, 40, 4, layout=layout, state=False), silu=False)
    check(fwp, *make(7, 2, 3, 40, 8, layout=layout, bias=False), silu=False)


def test_segments_and_single_steps_follow_on(fwp):
    a, _ = make(8, 3, 60, 48, 4, layout='sliced')
    with torch.no_grad():
        ref, end, _ = blocks.causal_conv(**a)
        for borders in ([0, 60], [0, 1, 3, 4, 40, 60], list(range(61))):
            state = a['state'].clone()
            out = torch.cat([fwp.causal_conv(**dict(a, x=a['x'][:, lo:hi], state=state)) for lo, hi in zip(borders, borders[1:])], 1)
            close('out', out, ref)
            assert torch.equal(state.double(), end)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_steps_behind_the_end_are_not_read(fwp, dtype):
    for L in (1, 2, 21):
        a, gy = make(9, 5, L, 40, 4, dtype=dtype, lengths='inside')
        ref = run(fwp, a, gy)
        behind = torch.arange(L, device=DEV) >= a['lengths'][:, None]
        for fill in (float('nan'), float('inf'), torch.finfo(dtype).min):
            x, bad = a['x'].clone(), gy.clone()
            x[behind], bad[behind] = fill, fill
            got = run(fwp, dict(a, x=x), bad)
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
            assert all(torch.equal(got[2][k], ref[2][k]) for k in ref[2])
        assert not ref[0][behind].any()


def test_a_bad_input_reaches_its_window_only(fwp):
    for fill in (float('nan'), float('inf')):
        for K in (2, 4, 5):
            a, gy = make(10, 2, 30, 40, K)
            ref = run(fwp, a, gy)
            x = a['x'].clone()
            x[1, 9, 7] = fill
            out, state, _ = run(fwp, dict(a, x=x), gy)
            keep = torch.ones(2, 30, 40, dtype=torch.bool, device=DEV)
            keep[1, 9:9 + K, 7] = False
            assert torch.equal(out[keep], ref[0][keep]) and torch.equal(state, ref[1])


def test_empty_calls(fwp):
    for N, L, D in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        a, gy = make(11, max(N, 1), max(L, 1), max(D, 1), 4)
        a.update(x=a['x'][:N, :L, :D], weight=a['weight'][:D], bias=a['bias'][:D], state=a['state'][:N, :, :D])
        out, state, grads = run(fwp, a, gy[:N, :L, :D])
        assert out.shape == (N, L, D) and torch.equal(state, a['state'])
        assert all(g.shape == a[k].shape and not g.any() for k, g in grads.items())


def test_results_do_not_change_from_run_to_run(fwp):
    a, gy = make(12, 6, 300, 260, 4, dtype=BF16)
    first = run(fwp, a, gy)
    again = run(fwp, a, gy)
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[2][k], again[2][k]) for k in first[2])


def test_gradients_against_differences(fwp):
    a, gy = make(13, 2, 30, 24, 4)
    _, _, grads = run(fwp, a, gy)
    for k in grads:
        v = torch.randn(a[k].shape, generator=util.gen(20)).to(DEV).double()
        h = 1e-5
        loss = [(blocks.causal_conv(**{q: (s.double() + e * v if q == k else s) for q, s in a.items()})[0] * gy.double()).sum() for e in (h, -h)]
        diff = ((loss[0] - loss[1]) / (2 * h)).item()
        along = (grads[k].double() * v).sum().item()
        size = (grads[k].double() * v).abs().sum().item()
        assert abs(along - diff) <= 128 * 2.0 ** -24 * size + 1e-6 * abs(diff) + 1e-5, k

"""The norms between two blocks against their definition in 64 bits."""
import itertools

import pytest
import torch

from oracle import blocks
from tests import util
from tests.blocks_util import DEV, close, half_step, streams

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, N, L, D, dtype=F32, rdtype=None, layout='packed', rms=False, parts='all'):
    g = util.gen(seed)
    x, gate, gy = streams(g, N, L, [D, D, D], dtype, layout)
    residual, gr = streams(g, N, L, [D, D], rdtype or dtype, layout)
    vec = lambda at: (torch.randn(D, generator=g) * 0.3 + at).to(DEV)         # noqa: E731
    on = lambda k: parts == 'all' or k in parts           # noqa: E731
    a = dict(x=x, weight=vec(1.), bias=None if rms else vec(0.), residual=residual if on('residual') else None,
             scale=vec(0.5) if on('scale') else 0.75 if on('number') else None, gate=gate if on('gate') else None,
             post_weight=vec(1.) if on('post') else None, post_bias=vec(0.) if on('post') and not rms else None)
    return a, gy, gr if on('residual') else gr.to(dtype)


def run(fwp, a, gy, gr, **kw):
    names = [k for k, t in a.items() if isinstance(t, torch.Tensor)]
    b = dict(a, **{k: a[k].detach().requires_grad_() for k in names})
    y, r = fwp.block_norm(**b, **kw)
    outs = [(o, g) for o, g in ((y, gy), (r, gr)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [b[k] for k in names], [g for _, g in outs], allow_unused=True)
    return y.detach(), r.detach(), dict(zip(names, grads))


def sizes(ref, sums, D):
    """What a row's gradient is made of: its largest term, times the four sums over the row it is corrected by."""
    return torch.maximum(sums.abs(), ref.abs()).max() * 4 * torch.ones_like(ref)


def check(fwp, a, gy, gr, **kw):
    ref_y, ref_r, sums = blocks.block_norm(**a, gy=gy, gr=gr, **kw)
    with torch.no_grad():
        y, r = fwp.block_norm(**a, **kw)
    assert y.dtype == a['x'].dtype and r.dtype == (a['x'] if a['residual'] is None else a['residual']).dtype
    close('y', y, ref_y)
    close('r', r, ref_r)
    y, r, grads = run(fwp, a, gy, gr, **kw)
    close('y', y, ref_y)
    close('r', r, ref_r)
    for k, g in grads.items():
        assert g.dtype == a[k].dtype and g.shape == a[k].shape
        close('gradient of ' + k, g, sums[k][0], sizes(*sums[k], g.shape[-1]))


@pytest.mark.parametrize('types', [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize('D', [4, 33, 64, 128, 129, 256, 260, 512, 513, 1000, 1024, 1030, 2048, 2050, 4096, 4099, 8192, 8190])
def test_against_the_definition(fwp, D, types):
    dtype, rdtype = types
    for rms in (False, True):
        check(fwp, *make(1, 2, 5, D, dtype, rdtype, rms=rms), rms=rms)
        check(fwp, *make(2, 3, 2, D, dtype, rdtype, layout='sliced', rms=rms, parts=('residual',)), rms=rms)


@pytest.mark.parametrize('act', ['silu', 'sigmoid', 'identity'])
@pytest.mark.parametrize('parts', [p for n in range(5) for p in itertools.combinations(('residual', 'scale', 'gate', 'post'), n)] +
                         [('number',), ('number', 'residual'), ('number', 'gate', 'post')])
def test_every_set_of_parts(fwp, parts, act):
    for D in (72, 300):
        check(fwp, *make(3, 2, 7, D, parts=parts), gate_act=act)
    check(fwp, *make(4, 1, 9, 77, BF16, rms=True, parts=parts), gate_act=act, rms=True)


def test_one_gradient_or_the_other(fwp):
    a, gy, gr = make(5, 2, 6, 96)
    check(fwp, a, gy, None)
    check(fwp, a, None, gr)


def test_many_rows(fwp):
    """More rows than a pass of the machine, so that a CTA sums over many of them."""
    check(fwp, *make(6, 40, 251, 64, F32, parts=('residual', 'scale')))
    check(fwp, *make(7, 5, 1000, 520, BF16, F32, rms=True), rms=True)


@pytest.mark.parametrize('layout', ['sliced', 'expanded'])
def test_layouts(fwp, layout):
    check(fwp, *make(8, 3, 9, 100, BF16, F32, layout=layout))


def test_other_shapes(fwp):
    a, gy, gr = make(9, 6, 4, 48)
    y, r, grads = run(fwp, a, gy, gr)
    for shape in ((24, 48), (2, 3, 4, 48), (2, 3, 2, 2, 48)):
        b = {k: t.reshape(shape) if k in ('x', 'residual', 'gate') else t for k, t in a.items()}
        y2, r2, grads2 = run(fwp, b, gy.reshape(shape), gr.reshape(shape))
        assert y2.shape == shape and torch.equal(y2.reshape(y.shape), y) and torch.equal(r2.reshape(r.shape), r)
        for k in grads:
            close(k, grads2[k].reshape(grads[k].shape), grads[k].double())


def test_an_expanded_gate_takes_the_sum_of_its_gradients(fwp):
    """A gate per sequence, shared by its steps."""
    a, gy, gr = make(10, 3, 8, 64)
    small = torch.randn(3, 1, 64, generator=util.gen(11)).to(DEV).requires_grad_()
    y, r = fwp.block_norm(**dict(a, gate=small.expand(3, 8, 64)))
    got, = torch.autograd.grad([y, r], [small], [gy, gr])
    _, _, sums = blocks.block_norm(**dict(a, gate=small.detach().expand(3, 8, 64)), gy=gy, gr=gr)
    close('gate', got, sums['gate'][0].sum(1, keepdim=True), 4 * sums['gate'][1].sum(1, keepdim=True))


def test_the_residual_gradient_without_anything_in_between(fwp):
    a, gy, gr = make(12, 2, 9, 80, parts=('residual',))
    _, _, grads = run(fwp, a, gy, gr)
    assert torch.equal(grads['x'], grads['residual'])


def test_constant_and_huge_rows(fwp):
    """A row of equal values has the variance zero; rows of 1e18 would overflow a sum of squares without the mean being taken off first."""
    a, gy, gr = make(13, 1, 4, 96, parts=('residual',))
    a['x'] = torch.zeros_like(a['x'])
    a['residual'] = torch.full_like(a['residual'], 3.)
    y, r, _ = run(fwp, a, gy, gr)
    assert torch.equal(r, a['residual']) and (y - a['bias']).abs().max() <= 1e-4
    a['residual'] = torch.full_like(a['residual'], 1e20)
    assert torch.isfinite(run(fwp, a, gy, gr)[0]).all()


def test_a_bad_row_stays_by_itself(fwp):
    for D in (96, 700):
        a, gy, gr = make(14, 2, 7, D)
        ref = run(fwp, a, gy, gr)
        b = dict(a, x=a['x'].clone())
        b['x'][1, 3, 5] = float('nan')
        got = run(fwp, b, gy, gr)
        keep = torch.ones(2, 7, dtype=torch.bool, device=DEV)
        keep[1, 3] = False
        for i in (0, 1):
            assert torch.equal(got[i][keep], ref[i][keep]) and got[i][1, 3].isnan().all()
        for k in ('x', 'residual', 'gate'):
            assert torch.equal(got[2][k][keep], ref[2][k][keep])


def test_empty_calls(fwp):
    for N, L in ((0, 5), (2, 0)):
        a, gy, gr = make(15, max(N, 1), max(L, 1), 40)
        a = {k: t[:N, :L] if k in ('x', 'residual', 'gate') else t for k, t in a.items()}
        y, r, grads = run(fwp, a, gy[:N, :L], gr[:N, :L])
        assert y.shape == r.shape == (N, L, 40)
        assert all(g.shape == a[k].shape and not g.any() for k, g in grads.items())


def test_results_do_not_change_from_run_to_run(fwp):
    a, gy, gr = make(16, 7, 130, 200, BF16, F32)
    first, again = run(fwp, a, gy, gr), run(fwp, a, gy, gr)
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[2][k], again[2][k]) for k in first[2])


def test_gradients_against_differences(fwp):
    a, gy, gr = make(17, 2, 5, 64)
    _, _, grads = run(fwp, a, gy, gr)
    for k, t in a.items():
        v = torch.randn(t.shape, generator=util.gen(20)).to(DEV).double()
        h, loss = 1e-5, []
        for e in (h, -h):
            y, r, _ = blocks.block_norm(**{q: (s.double() + e * v if q == k else s) for q, s in a.items()})
            loss.append(((y * gy.double()).sum() + (r * gr.double()).sum()).item())
        diff, along = (loss[0] - loss[1]) / (2 * h), (grads[k].double() * v).sum().item()
        size = (grads[k].double() * v).abs().sum().item()
        assert abs(along - diff) <= 256 * 2.0 ** -24 * size + 1e-6 * abs(diff) + 1e-5, k

"""What the tests of the state-space layer's operators share: inputs and the bounds that outputs are held to."""
import torch

from tests import util

DEV = 'cuda:0'
U = 2.0 ** -24          # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(name, got, ref, sums=None, steps=0):
    """|got - ref| <= half a step of got's type at the value + (64 + 4 steps) U at the size of the terms it is made of.

    An output is a sum of products of a few factors; each factor is a rounded operation or an exponential, reciprocal or sigmoid with a
    documented error of at most 2^-22.5 (3 U), the step size's logarithm and the norms' statistics among them: at most 64 U in all.  A
    state that is `steps` steps old was multiplied by that many decays, each with 3 U of the exponential and 1 U of the product.
    The sizes: of the largest term sum where the sums of absolute terms are known, else of the largest value."""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    g, r = got.double().cpu(), ref.double().cpu()
    size = (r if sums is None else sums.double().cpu()).abs().max().item() if r.numel() else 0.
    err = (g - r).abs()
    bound = half_step(got.dtype) * r.abs() + (64 + 4 * steps) * U * size
    assert torch.isfinite(g).all(), '%s is not finite' % name
    if r.numel():
        util.record(name, worst=(err / bound.clamp_min(1e-300)).max().item())
    assert (err <= bound).all(), '%s: %.3g of the bound' % (name, (err / bound.clamp_min(1e-300)).max().item())


def streams(g, N, L, widths, dtype, layout):
    """(N, L, width) tensors of their own, slices of a projection in (L, N) order at odd offsets, or batch-expanded ones."""
    if layout == 'packed':
        return [torch.randn(N, L, w, generator=g).to(dtype).to(DEV) for w in widths]
    if layout == 'expanded':
        return [torch.randn(1, L, w, generator=g).to(dtype).to(DEV).expand(N, L, w) for w in widths]
    x = torch.randn(L, N, sum(widths) + len(widths), generator=g).to(dtype).to(DEV)
    return [t[..., 1:].transpose(0, 1) for t in torch.split(x, [w + 1 for w in widths], -1)]


def lengths_of(kind, N, L, g):
    """None, lengths from 0 to L with both ends among them where there is room, or values outside that range."""
    if kind is None:
        return None
    n = torch.randint(0, L + 1, (N,), generator=g, dtype=torch.int32)
    n[0] = L
    if N > 1:
        n[1] = 0
    if kind == 'outside':
        n[0] = L + 7
        if N > 1:
            n[1] = -3
    return n.to(DEV)

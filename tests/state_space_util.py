"""The plain 64-bit forms with the ops' calling conventions, for the language-model harness."""
import torch

from oracle import blocks


def conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    """Differentiable, in the inputs' type; the window is left in ``state``."""
    N, L, D = x.shape
    K = weight.shape[1]
    ext = torch.cat([torch.zeros(N, K - 1, D, dtype=x.dtype) if state is None else state.to(x.dtype), x], 1)
    p = bias + sum(weight[:, j] * ext[:, j:j + L] for j in range(K))
    if state is not None:
        state.copy_(ext[:, L:].detach())
    return torch.nn.functional.silu(p)


def scan(x, dt, A, B, C, D, z=None, dt_bias=None, state=None):
    delta = torch.nn.functional.softplus(dt + dt_bias)
    h, ys = state.to(x.dtype), []
    for t in range(x.shape[1]):
        h = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * x[:, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1))
    state.copy_(h.detach())
    return (torch.stack(ys, 1) + D * x) * torch.nn.functional.silu(z)


def norm(x, weight, bias=None, residual=None, eps=1e-5):
    r = x if residual is None else residual + x
    return torch.nn.functional.layer_norm(r, r.shape[-1:], weight, bias, eps), r


OPS = dict(conv=conv, scan=scan)


def check_against_the_definitions():
    """These forms are what oracle.blocks computes."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)      # noqa: E731
    x, w, b, st = r(2, 9, 6), r(6, 4), r(6), r(2, 3, 6)
    ref, end, _ = blocks.causal_conv(x, w, b, st)
    assert torch.allclose(conv(x, w, b, st), ref, atol=1e-12) and torch.allclose(st, end, atol=1e-12)
    a = dict(x=x, dt=r(2, 9, 6), A=-r(6, 4).abs(), B=r(2, 9, 4), C=r(2, 9, 4), D=r(6), z=r(2, 9, 6), dt_bias=r(6), state=r(2, 6, 4))
    ref, end, _ = blocks.selective_scan(**a)
    assert torch.allclose(scan(**a), ref, atol=1e-12) and torch.allclose(a['state'], end, atol=1e-12)
    y, s, _ = blocks.block_norm(x, b, b, residual=r(2, 9, 6) * 0 + 1)
    y2, s2 = norm(x, b, b, residual=torch.ones_like(x))
    assert torch.allclose(y, y2, atol=1e-12) and torch.allclose(s, s2, atol=1e-12)

"""Plain 64-bit forms of the state-space layer's operators, step by step (TEST INFRASTRUCTURE ONLY).

Each takes the op's arguments (any type; computed in float64 on their device) and returns the output, the state after the last step
where there is one, and, given the gradient of the output, the gradients.  Every gradient comes with the sum of the absolute values
of its terms: weights, B and C are differentiated as if each (step, channel) had a copy of its own, and the copies' gradients are
added up afterwards.  That sum is what an error bound of a sum in finite precision is a multiple of.
"""
import torch
import torch.nn.functional as F


def _double(t):
    return None if t is None else t.detach().double()


def _leaf(t, *shape):
    return None if t is None else t.detach().double().expand(*shape).clone().requires_grad_()


def _inside(x, lengths):
    N, L = x.shape[:2]
    if lengths is None:
        return torch.ones(N, L, 1, dtype=torch.bool, device=x.device)
    return (torch.arange(L, device=x.device) < lengths[:, None])[..., None]


def _summed(grad, dims):
    """(sum of the terms, sum of their absolute values)"""
    return (grad.sum(dims), grad.abs().sum(dims)) if dims else (grad, grad.abs())


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True, gy=None):
    N, L, D = x.shape
    K = weight.shape[1]
    inside = _inside(x, lengths)
    xs = _leaf(torch.where(inside, x.detach(), 0), N, L, D)
    w, b = _leaf(weight, N, L, D, K), _leaf(bias, N, L, D)
    before = torch.zeros(N, K - 1, D, dtype=torch.float64, device=x.device) if state is None else _double(state)
    ext = torch.cat([before, xs], 1)
    p = sum(w[..., j] * ext[:, j:j + L] for j in range(K))
    p = p if b is None else p + b
    out = torch.where(inside, F.silu(p) if silu else p, 0)
    ends = [L] * N if lengths is None else [min(max(int(n), 0), L) for n in lengths]
    end = torch.stack([ext[n, e:e + K - 1] for n, e in enumerate(ends)]).detach()
    grads = None
    if gy is not None:
        # rows behind a sequence's end take no gradient, whatever stands in gy there
        leaves = [t for t in (xs, w, b) if t is not None]
        got = iter(torch.autograd.grad(out, leaves, torch.where(inside, gy.double(), 0)))
        grads = {'x': _summed(next(got), ()), 'weight': _summed(next(got), (0, 1))}
        if b is not None:
            grads['bias'] = _summed(next(got), (0, 1))
    return out.detach(), end, grads


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None, softplus=True, gy=None):
    N, L, M = x.shape
    S = A.shape[1]
    grouped = B if B.dim() == 4 else B.unsqueeze(2)
    G = grouped.shape[2]
    per = M // G
    inside = _inside(x, lengths)
    clean = lambda t: t if lengths is None else torch.where(inside if t.dim() == 3 else inside[..., None], t.detach(), 0)    # noqa: E731
    xs, dts, zs = _leaf(clean(x), N, L, M), _leaf(clean(dt), N, L, M), None if z is None else _leaf(clean(z), N, L, M)
    grouped, C = clean(grouped), clean(C if C.dim() == 4 else C.unsqueeze(2))
    each = lambda t: _leaf(t.unsqueeze(3), N, L, G, per, S)           # noqa: E731
    Bs, Cs = each(grouped), each(C)
    As, skip, bias = _leaf(A, N, L, M, S), _leaf(D, N, L, M), _leaf(dt_bias, N, L, M)
    raw = dts if bias is None else dts + bias
    delta = F.softplus(raw, threshold=700.) if softplus else raw
    delta = torch.where(inside, delta, 0)
    h = torch.zeros(N, M, S, dtype=torch.float64, device=x.device) if state is None else _double(state)
    Bc, Cc = Bs.flatten(2, 3), Cs.flatten(2, 3)
    ys = []
    for t in range(L):
        new = torch.exp(delta[:, t, :, None] * As[:, t]) * h + (delta[:, t] * xs[:, t])[..., None] * Bc[:, t]
        h = torch.where(inside[:, t, :, None], new, h)
        ys.append((h * Cc[:, t]).sum(-1))
    y = torch.stack(ys, 1)
    if skip is not None:
        y = y + skip * xs
    out = torch.where(inside, y if zs is None else y * F.silu(zs), 0)
    grads = None
    if gy is not None:
        names = [('x', xs, ()), ('dt', dts, ()), ('A', As, (0, 1)), ('B', Bs, (3,)), ('C', Cs, (3,)), ('D', skip, (0, 1)), ('z', zs, ()),
                 ('dt_bias', bias, (0, 1))]
        names = [q for q in names if q[1] is not None]
        got = torch.autograd.grad(out, [q[1] for q in names], torch.where(inside, gy.double(), 0))
        grads = {n: _summed(g, dims) for (n, _, dims), g in zip(names, got)}
        for n in ('B', 'C'):
            grads[n] = tuple(g if B.dim() == 4 else g.squeeze(2) for g in grads[n])
    return out.detach(), h.detach(), grads


ACTS = {'silu': F.silu, 'sigmoid': torch.sigmoid, 'identity': lambda g: g}


def block_norm(x, weight, bias=None, residual=None, scale=None, gate=None, post_weight=None, post_bias=None, gate_act='silu', eps=1e-5,
               rms=False, gy=None, gr=None):
    shape = x.shape
    leaf = lambda t: _leaf(t, *shape) if isinstance(t, torch.Tensor) else t      # noqa: E731
    v = {'x': x, 'weight': weight, 'bias': bias, 'residual': residual, 'scale': scale, 'gate': gate, 'post_weight': post_weight,
         'post_bias': post_bias}
    v = {n: leaf(t) for n, t in v.items() if t is not None}

    def norm(t, w, b):
        mean = 0. if rms else t.mean(-1, keepdim=True)
        c = t - mean
        n = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * w
        return n if b is None else n + b

    t = norm(v['x'], v['post_weight'], v.get('post_bias')) if 'post_weight' in v else v['x']
    if 'gate' in v:
        t = t * ACTS[gate_act](v['gate'])
    r = t * v['scale'] if 'scale' in v else t
    if 'residual' in v:
        r = r + v['residual']
    y = norm(r, v['weight'], v.get('bias'))
    grads = None
    if gy is not None or gr is not None:
        outs = [(o, g) for o, g in ((y, gy), (r, gr)) if g is not None]
        leaves = {n: t for n, t in v.items() if isinstance(t, torch.Tensor)}
        got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g.double() for _, g in outs], allow_unused=True)
        rows = tuple(range(len(shape) - 1))
        grads = {n: _summed(torch.zeros(shape, dtype=torch.float64, device=x.device) if g is None else g,
                            () if n in ('x', 'residual', 'gate') else rows) for n, g in zip(leaves, got)}
    return y.detach(), r.detach(), grads

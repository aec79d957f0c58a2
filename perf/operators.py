"""Workloads of the state-space layer's operators: the short causal convolution, the selective scan and the fused norms
between two blocks, each in its plain form (elementary torch operations) and through the framework's entry points.

A case's keys:

  op        conv (``causal_conv``), scan (``selective_scan``), norm (``block_norm``)
  mode      train: forward and backward through autograd; eval: forward under no_grad; for one step (L = 1) that is decoding
  N L D     sequences, steps, channels
  dtype     fp32 or bf16 streams; weights and carried states are fp32 either way
  layout    packed: contiguous (N, L, D) tensors; sliced: what a layer hands over, slices of wider projections whose
            outer order is (L, N)
  ragged    sequences of different lengths in one padded batch
  conv      K taps
  scan      S states per channel, G groups of channels that share B and C, gated: with a gate z
  norm      rms or layer norm; post: a norm of the block's output as well; gate: silu, sigmoid, identity or none; scale: the
            residual scale, vector, number or none; wide: an fp32 residual stream beside bf16 block outputs
"""
import math

import torch

own = False

DTYPE = {'fp32': torch.float32, 'bf16': torch.bfloat16}
EPS = 1e-5
NUMBER = 0.5        # the residual scale where it is a number


def _conv(mode, N, L, D, K=4, dtype='bf16', layout='sliced', ragged=False, **name):
    return dict(name, op='conv', mode=mode, N=N, L=L, D=D, K=K, dtype=dtype, layout=layout, ragged=ragged)


def _scan(mode, N, L, D, S=16, G=1, dtype='bf16', layout='sliced', ragged=False, gated=True, **name):
    return dict(name, op='scan', mode=mode, N=N, L=L, D=D, S=S, G=G, dtype=dtype, layout=layout, ragged=ragged, gated=gated)


def _norm(mode, N, L, D, dtype='bf16', layout='packed', rms=False, post=False, gate='none', scale='none', wide=False, **name):
    return dict(name, op='norm', mode=mode, N=N, L=L, D=D, dtype=dtype, layout=layout, rms=rms, post=post, gate=gate,
                scale=scale, wide=wide)


def listed():
    return [
        # decoding: the next token of 32 sequences through a layer of the 256-wide language model (inner width 512)
        _conv('eval', 32, 1, 512, layout='packed', name='conv_step'),
        # prompts of different lengths in one padded batch, a width that fits no vector
        _conv('eval', 6, 997, 519, dtype='fp32', ragged=True, name='conv_ragged'),
        # a training step of a 2048-channel layer on eight sequences
        _conv('train', 8, 2048, 2048, name='conv_train'),
        # decoding: the next token of 64 sequences at 2048 channels; reading and writing the carried state is the work
        _scan('eval', 64, 1, 2048, layout='packed', name='scan_step'),
        # padded prompts, odd sizes, two groups
        _scan('eval', 6, 777, 518, G=2, dtype='fp32', ragged=True, name='scan_ragged'),
        # one long prompt: few channels, many steps
        _scan('eval', 1, 16384, 2048, name='scan_prompt'),
        # a training segment of the language-model recipe: 64 sequences of 256 steps, inner width 512, fp32
        _scan('train', 64, 256, 512, dtype='fp32', name='scan_lm'),
        # a training step of a 2048-channel layer on eight sequences
        _scan('train', 8, 2048, 2048, name='scan_train'),
        # decoding: 32 rows of the 256-wide language model
        _norm('eval', 32, 1, 256, dtype='fp32', name='norm_step'),
        # between two blocks of the 16-layer language model: 32 sequences of 512 steps, d_model 256, LayerNorm, fp32
        _norm('train', 32, 512, 256, dtype='fp32', layout='sliced', name='norm_lm'),
        # prompts at an odd width, root-mean-square norm, gated, the residual scale a number
        _norm('eval', 3, 1999, 1001, rms=True, gate='sigmoid', scale='number', name='norm_odd'),
        # a wide model: norms on both sides of the block, gate, learned residual scale, fp32 residual stream
        _norm('train', 4, 4096, 4096, rms=True, post=True, gate='silu', scale='vector', wide=True, name='norm_train'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: an operator and a way to call it, sizes spread over their logarithm, cut to the largest listed work."""
    op = rng.choice(['conv', 'scan', 'scan', 'norm'])
    use = rng.choice(['step', 'prompt', 'long', 'train', 'train'])
    D = _log(rng, 64, 4096)
    if rng.random() < 0.7:
        D = max(64, D // 64 * 64)
    N = {'step': _log(rng, 1, 256), 'prompt': _log(rng, 1, 32), 'long': rng.choice([1, 2]), 'train': _log(rng, 1, 64)}[use]
    L = {'step': 1, 'prompt': _log(rng, 2, 4096), 'long': _log(rng, 2048, 32768), 'train': _log(rng, 32, 4096)}[use]
    dtype, layout = rng.choice(['fp32', 'bf16', 'bf16']), rng.choice(['packed', 'sliced'])
    most = {'conv': 8 * 2048 * 2048, 'scan': 16384 * 2048, 'norm': 4 * 4096 * 4096}[op]
    if dtype == 'fp32':
        most //= 2
    mode = 'train' if use == 'train' else 'eval'
    ragged = use != 'step' and rng.random() < 0.3
    if op == 'conv':
        L = max(1, min(L, most // (N * D)))
        return _conv(mode, N, L, D, rng.choice([2, 3, 4, 4, 4]), dtype, layout, ragged)
    if op == 'norm':
        L = max(1, min(L, most // (N * D)))
        return _norm(mode, N, L, D, dtype, layout, rng.random() < 0.5, rng.random() < 0.5,
                     rng.choice(['none', 'silu', 'sigmoid', 'identity']), rng.choice(['none', 'number', 'vector']),
                     dtype == 'bf16' and rng.random() < 0.5)
    S = rng.choice([4, 8, 16, 16, 16, 16, 32, 64])
    D = min(D, 2048) * 16 // max(16, S)
    G = rng.choice([1, 1, 2, 4])
    D = max(G, D // G * G)
    L = max(1, min(L, most * 16 // (N * D * max(16, S))))
    return _scan(mode, N, L, D, S, G, dtype, layout, ragged, rng.random() < 0.8)


# ------------------------------------------------------------------------------------------------------------ inputs
def _random(g, *shape):
    return torch.randn(*shape, generator=g, device='cuda')


def _streams(g, case, widths):
    """N(0,1) streams (N, L, width): tensors of their own, or slices of one projection in (L, N) order."""
    N, L, dt = case['N'], case['L'], DTYPE[case['dtype']]
    if case['layout'] == 'packed':
        return [_random(g, N, L, w).to(dt) for w in widths]
    x = _random(g, L, N, sum(widths)).to(dt)
    return [t.transpose(0, 1) for t in torch.split(x, widths, -1)]


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    op, N, L, D, train = case['op'], case['N'], case['L'], case['D'], case['mode'] == 'train'
    s = dict(case=case, train=train, lengths=None)
    if case.get('ragged'):
        n = torch.randint(1, L + 1, (N,), generator=g, device='cuda', dtype=torch.int32)
        n[0] = L
        s['lengths'] = n
    if op == 'conv':
        x, gy = _streams(g, case, [D, D])
        s.update(x=x, weight=_random(g, D, case['K']) / math.sqrt(case['K']), bias=_random(g, D) * 0.1,
                 state=_random(g, N, case['K'] - 1, D))
        names = ['x', 'weight', 'bias']
    elif op == 'scan':
        S, G = case['S'], case['G']
        x, z, gy = _streams(g, case, [D, D, D])
        dt, B, C = _streams(g, case, [D, G * S, G * S])
        # step sizes spread over 0.001 ... 0.1 through the bias, decay rates 1 ... S, as such layers start out
        step = torch.exp(torch.rand(D, generator=g, device='cuda') * math.log(100.) + math.log(0.001))
        s.update(x=x, dt=dt, z=z if case['gated'] else None, B=B.unflatten(-1, (G, S)), C=C.unflatten(-1, (G, S)),
                 A=-torch.arange(1, S + 1, device='cuda', dtype=torch.float32) * torch.exp(0.2 * _random(g, D, S)),
                 D=1 + 0.1 * _random(g, D), dt_bias=torch.log(torch.expm1(step)), state=_random(g, N, D, S) * 0.1)
        names = ['x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias'] + (['z'] if case['gated'] else [])
    else:
        x, gate, gy = _streams(g, case, [D, D, D])
        wide = dict(case, dtype='fp32') if case['wide'] else case
        residual, gr = _streams(g, wide, [D, D])
        s.update(x=x, residual=residual, gate=None if case['gate'] == 'none' else gate, gr=gr,
                 weight=1 + 0.1 * _random(g, D), bias=None if case['rms'] else 0.1 * _random(g, D),
                 post_weight=1 + 0.1 * _random(g, D) if case['post'] else None,
                 post_bias=0.1 * _random(g, D) if case['post'] and not case['rms'] else None,
                 scale={'none': None, 'number': NUMBER, 'vector': 0.2 + 0.1 * _random(g, D)}[case['scale']])
        names = [k for k in ('x', 'residual', 'gate', 'weight', 'bias', 'post_weight', 'post_bias', 'scale')
                 if isinstance(s[k], torch.Tensor)]
    s.update(gy=gy, names=names)
    if train:
        for k in names:
            s[k] = s[k].detach().requires_grad_()
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _silu_grad(x):
    """silu'(x)"""
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def _valid(s, shape):
    """(N, L, 1): the steps below their sequence's length; None where all are."""
    if s['lengths'] is None:
        return None
    return (torch.arange(shape[1], device='cuda') < s['lengths'][:, None])[..., None]


def _cut(valid, t):
    return t if valid is None else torch.where(valid, t, 0)


def _plain_conv(s):
    x, w, K, dt = s['x'].detach().float(), s['weight'].detach(), s['case']['K'], s['x'].dtype
    N, L, D = x.shape
    valid = _valid(s, x.shape)
    ext = torch.cat([s['state'], _cut(valid, x)], 1)
    taps = [ext[:, j:j + L] for j in range(K)]
    p = s['bias'].detach() + sum(w[:, j] * taps[j] for j in range(K))
    out = _cut(valid, p * torch.sigmoid(p)).to(dt)
    ends = torch.full((N,), L, device='cuda') if s['lengths'] is None else s['lengths']
    rows = (ends[:, None] + torch.arange(K - 1, device='cuda')).long()
    state = ext.gather(1, rows[..., None].expand(N, K - 1, D))
    if not s['train']:
        s['state'].copy_(state)
        return out, s['state']
    gp = _cut(valid, s['gy'].float() * _silu_grad(p))
    pad = torch.cat([gp, gp.new_zeros(N, K - 1, D)], 1)
    gx = sum(w[:, j] * pad[:, K - 1 - j:K - 1 - j + L] for j in range(K))
    gw = torch.stack([(gp * taps[j]).sum((0, 1), dtype=torch.float64) for j in range(K)], -1)
    return out, state, [_cut(valid, gx).to(dt), gw.float(), gp.sum((0, 1), dtype=torch.float64).float()]


def _forward_scan(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1, in place of u: spans of steps joined in pairs, log2(L) times."""
    k, L = 1, u.shape[1]
    while k < L:
        u[:, k:] += a[:, k:] * u[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return u


def _backward_scan(a, u):
    """g_t = u_t + a_t g_{t+1}, likewise."""
    k, L = 1, u.shape[1]
    while k < L:
        u[:, :-k] += a[:, :-k] * u[:, k:]
        a[:, :-k] = a[:, :-k] * a[:, k:]
        k *= 2
    return u


def _plain_scan(s):
    case, dt = s['case'], s['x'].dtype
    x, raw, B, C = (s[k].detach().float() for k in ('x', 'dt', 'B', 'C'))
    A, skip, bias = (s[k].detach() for k in ('A', 'D', 'dt_bias'))
    N, L, D = x.shape
    per = D // case['G']
    valid = _valid(s, x.shape)
    raw = raw + bias
    delta = _cut(valid, torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())))    # softplus
    channels = lambda t: t.repeat_interleave(per, 2) if case['G'] > 1 else t            # noqa: E731
    groups = lambda t: t.unflatten(2, (case['G'], per)).sum(3)                          # noqa: E731
    h = (delta * x)[..., None] * channels(B)
    if valid is not None:
        h = torch.where(valid[..., None], h, 0)
    a = torch.exp(delta[..., None] * A)
    h[:, 0] += a[:, 0] * s['state']
    start = s['state'].clone()
    h = _forward_scan(a.clone() if s['train'] else a, h)
    y = (h * channels(C)).sum(-1) + skip * x
    z = s['z'].detach().float() if case['gated'] else None
    out = _cut(valid, y * z * torch.sigmoid(z) if case['gated'] else y).to(dt)
    if not s['train']:
        s['state'].copy_(h[:, -1])
        return out, s['state']
    state = h[:, -1].clone()
    go = _cut(valid, s['gy'].float())
    gy = go * z * torch.sigmoid(z) if case['gated'] else go
    gz = [(go * y * _silu_grad(z)).to(dt)] if case['gated'] else []
    gC = groups(gy[..., None] * h)
    h[:, 1:] = h[:, :-1].clone()            # from here on the state before each step
    h[:, 0] = start
    h *= a
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    del a
    g = _backward_scan(later, gy[..., None] * channels(C))
    del later
    gB = groups(g * (delta * x)[..., None])
    p = (g * channels(B)).sum(-1)
    h *= g
    gx = _cut(valid, delta * p + skip * gy)
    graw = _cut(valid, (x * p + (h * A).sum(-1)) * torch.sigmoid(raw))
    h *= delta[..., None]
    sums = [t.sum((0, 1), dtype=torch.float64).float() for t in (gy * x, graw)]
    return out, state, [gx.to(dt), graw.to(dt), h.sum((0, 1), dtype=torch.float64).float(), gB.to(dt), gC.to(dt)] + sums + gz


def _plain_statistics(x, rms):
    mean = torch.zeros_like(x[..., :1]) if rms else x.mean(-1, keepdim=True)
    return mean, torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)


def _plain_norm_grad(gy, x, mean, rstd, w, rms):
    """The gradients of a norm's input, weight and bias."""
    n = (x - mean) * rstd
    gn = gy * w
    gx = rstd * (gn - n * (gn * n).mean(-1, keepdim=True) - (0 if rms else gn.mean(-1, keepdim=True)))
    return gx, (gy * n).sum((0, 1), dtype=torch.float64).float(), gy.sum((0, 1), dtype=torch.float64).float()


def _plain_act(case, gate):
    """The gate's factor and its derivative."""
    if case['gate'] == 'silu':
        return gate * torch.sigmoid(gate), _silu_grad(gate)
    if case['gate'] == 'sigmoid':
        v = torch.sigmoid(gate)
        return v, v * (1 - v)
    return gate, torch.ones_like(gate)


def _plain_norm(s):
    case, rms = s['case'], s['case']['rms']
    x, dt, rdt = s['x'].detach().float(), s['x'].dtype, s['residual'].dtype
    val = {k: s[k].detach() if isinstance(s[k], torch.Tensor) else s[k] for k in ('weight', 'bias', 'post_weight', 'post_bias', 'scale')}
    t = x
    if case['post']:
        pm, pr = _plain_statistics(x, rms)
        t = (x - pm) * pr * val['post_weight'] + (0 if rms else val['post_bias'])
    u = t
    if s['gate'] is not None:
        act, dact = _plain_act(case, s['gate'].detach().float())
        u = t * act
    scale = 1. if val['scale'] is None else val['scale']
    r = s['residual'].detach().float() + scale * u
    m, rs = _plain_statistics(r, rms)
    y = (r - m) * rs * val['weight'] + (0 if rms else val['bias'])
    out = y.to(dt), r.to(rdt)
    if not s['train']:
        return out
    g, gw, gb = _plain_norm_grad(s['gy'].float(), r, m, rs, val['weight'], rms)
    g = g + s['gr'].float()
    got = {'residual': g.to(rdt), 'weight': gw, 'bias': gb}
    if case['scale'] == 'vector':
        got['scale'] = (g * u).sum((0, 1), dtype=torch.float64).float()
    gu = g * scale
    gt = gu
    if s['gate'] is not None:
        got['gate'] = (gu * t * dact).to(dt)
        gt = gu * act
    if case['post']:
        gt, got['post_weight'], got['post_bias'] = _plain_norm_grad(gt, x, pm, pr, val['post_weight'], rms)
    got['x'] = gt.to(dt)
    return out, [got[k] for k in s['names']]


# --------------------------------------------------------------------------------------------------- the entry points
def _own_call(s, state):
    op = s['case']['op']
    if op == 'conv':
        from recurrent_fwp_b200.causal_conv import causal_conv
        return causal_conv(s['x'], s['weight'], s['bias'], state=state, lengths=s['lengths'])
    if op == 'scan':
        from recurrent_fwp_b200.selective_scan import selective_scan
        return selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], s['D'], z=s['z'], dt_bias=s['dt_bias'], state=state,
                              lengths=s['lengths'])
    from recurrent_fwp_b200.block_norm import block_norm
    return block_norm(s['x'], s['weight'], s['bias'], residual=s['residual'], scale=s['scale'], gate=s['gate'],
                      gate_act='silu' if s['gate'] is None else s['case']['gate'], post_weight=s['post_weight'],
                      post_bias=s['post_bias'], eps=EPS, rms=s['case']['rms'])


def run(state):
    """One pass.  eval: the output and the carried state, updated in place (decoding and prompts).  train: the output, the state after
    the segment (the start's is a clone, as a trainer that carries it keeps it) and the gradients."""
    s = state
    if not own:
        return {'conv': _plain_conv, 'scan': _plain_scan, 'norm': _plain_norm}[s['case']['op']](s)
    if not s['train']:
        with torch.no_grad():
            out = _own_call(s, s.get('state'))
        return out if s['case']['op'] == 'norm' else (out, s['state'])
    leaves = [s[k] for k in s['names']]
    if s['case']['op'] == 'norm':
        y, r = _own_call(s, None)
        return (y.detach(), r.detach()), list(torch.autograd.grad([y, r], leaves, [s['gy'], s['gr']]))
    carried = s['state'].clone()
    out = _own_call(s, carried)
    grads = list(torch.autograd.grad(out, leaves, s['gy']))
    return out.detach(), carried, grads


def work(case):
    """Streams read once and written once over the pass (weights, states and B, C with them), and the operations of the formulas
    with an exponential counted as one."""
    op, N, L, D, train = case['op'], case['N'], case['L'], case['D'], case['mode'] == 'train'
    esz, units = 2 if case['dtype'] == 'bf16' else 4, N * L * D
    if op == 'conv':
        K = case['K']       # x, out; gy, gx
        return {'bytes': units * esz * (4 if train else 2) + 2 * 4 * N * (K - 1) * D + 4 * D * (K + 1) * (2 if train else 1),
                'flops': units * (2 * K + 5 + (4 * K + 10 if train else 0))}
    if op == 'scan':
        S, G, z = case['S'], case['G'], 1 if case['gated'] else 0
        streams = (3 + z) + (3 + z if train else 0)         # x, dt, z, out; gy, gx, gdt, gz
        shared = 2 * N * L * G * S * (2 if train else 1)
        return {'bytes': esz * (units * streams + shared) + 2 * 4 * N * D * S + 4 * D * (S + 2) * (2 if train else 1),
                'flops': units * (S * (6 + (16 if train else 0)) + 10 + (20 if train else 0))}
    gate, wide = 0 if case['gate'] == 'none' else 1, 4 if case['wide'] else esz
    vectors = 1 + (not case['rms']) + case['post'] * (1 + (not case['rms'])) + (case['scale'] == 'vector')
    plain = 2 + gate + (2 + gate if train else 0)           # x, gate, y; gy, gx, ggate
    return {'bytes': units * (plain * esz + (4 if train else 2) * wide) + 4 * D * vectors * (2 if train else 1),
            'flops': units * (10 + 5 * gate + 6 * case['post']) * (3 if train else 1)}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits
def _definition_conv(s, v):
    K, (N, L, D) = s['case']['K'], v['x'].shape
    rows, ends = [], []
    for n in range(N):      # a sequence at a time, the inputs behind those that the state holds
        length = L if s['lengths'] is None else int(s['lengths'][n])
        ext = torch.cat([s['state'][n].double(), v['x'][n, :length]])
        p = torch.nn.functional.conv1d(ext.t().unsqueeze(0), v['weight'].unsqueeze(1), v['bias'], groups=D)[0].t()
        rows.append(torch.cat([torch.nn.functional.silu(p), p.new_zeros(L - length, D)]))
        ends.append(ext[length:].detach())
    return torch.stack(rows), torch.stack(ends)


def _definition_scan(s, v):
    case, (N, L, D) = s['case'], v['x'].shape
    per = D // case['G']
    delta = torch.nn.functional.softplus(v['dt'] + v['dt_bias'])
    h, ys = s['state'].double(), []
    Bs, Cs = (v[k].unsqueeze(3).expand(-1, -1, -1, per, -1).flatten(2, 3) for k in ('B', 'C'))
    for t in range(L):
        d = delta[:, t, :, None]
        new = torch.exp(d * v['A']) * h + d * v['x'][:, t, :, None] * Bs[:, t]
        h = new if s['lengths'] is None else torch.where((t < s['lengths'])[:, None, None], new, h)
        ys.append((h * Cs[:, t]).sum(-1))
    y = torch.stack(ys, 1) + v['D'] * v['x']
    if case['gated']:
        y = y * torch.nn.functional.silu(v['z'])
    if s['lengths'] is not None:
        y = y * (torch.arange(L, device='cuda') < s['lengths'][:, None])[..., None]
    return y, h.detach()


def _definition_norm(s, v):
    case = s['case']

    def norm(x, w, b):
        if case['rms']:
            return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, EPS)

    t = norm(v['x'], v['post_weight'], v['post_bias']) if case['post'] else v['x']
    if s['gate'] is not None:
        t = t * {'silu': torch.nn.functional.silu, 'sigmoid': torch.sigmoid, 'identity': lambda g: g}[case['gate']](v['gate'])
    if v['scale'] is not None:
        t = t * v['scale']
    r = v['residual'] + t
    return norm(r, v['weight'], v['bias']), r


def exact(case, seed):
    """What ``run`` returns, in 64 bits: the definitions step by step, their gradients by autograd."""
    steps = case['L'] if case['op'] == 'scan' else 1
    # autograd keeps about five values of every (step, state); beyond this it would not fit, or take too long
    if steps > 40000 or (case['op'] == 'scan' and case['mode'] == 'train' and case['N'] * case['L'] * case['D'] * case['S'] > 6e8):
        return None
    s = prepare(case, seed)
    v = {k: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for k, t in s.items()}
    if s['train']:
        for k in s['names']:
            v[k].requires_grad_()
    with torch.set_grad_enabled(s['train']):
        out = {'conv': _definition_conv, 'scan': _definition_scan, 'norm': _definition_norm}[case['op']](s, v)
    if not s['train']:
        return out
    leaves = [v[k] for k in s['names']]
    if case['op'] == 'norm':
        return tuple(t.detach() for t in out), list(torch.autograd.grad(out, leaves, [v['gy'], v['gr']]))
    return out[0].detach(), out[1], list(torch.autograd.grad(out[0], leaves, v['gy']))

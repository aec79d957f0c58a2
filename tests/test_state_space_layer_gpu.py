"""causal_conv, selective_scan and block_norm together, as the language model's state-space layer and a serving loop use them: against
64 bits, token by token, captured into graphs, on streams of their own, from several threads, under autograd's other users."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from oracle import blocks
from recurrent_fwp_b200.lm_harness import DeltaNetLM
from tests import state_space_util as plain
from tests import util
from tests.blocks_util import DEV, close

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def models(fused_norm, n_layer=3):
    """The same model with the CUDA ops on the GPU and with the plain forms, in 64 bits, on the CPU."""
    torch.manual_seed(2)
    gpu = DeltaNetLM(50, n_layer, 2, 32, 16, 48, attn_type='scan', fused_norm=fused_norm)
    cpu = DeltaNetLM(50, n_layer, 2, 32, 16, 48, attn_type='scan', ops=plain.OPS).double()
    cpu.load_state_dict(gpu.state_dict())
    return gpu.to(DEV), cpu


@pytest.mark.parametrize('fused_norm', [False, True])
def test_losses_and_gradients_of_the_language_model(fwp, fused_norm):
    gpu, cpu = models(fused_norm)
    tokens = torch.randint(0, 50, (41, 3), generator=util.gen(3))
    got, mems = gpu(tokens[:-1].to(DEV), tokens[1:].to(DEV), None, carry_over_fast_weight=True)
    ref, ref_mems = cpu(tokens[:-1], tokens[1:], None, carry_over_fast_weight=True)
    assert util.max_abs(got, ref) <= 1e-4
    for p, q in zip(mems, ref_mems):
        assert all(util.max_abs(s, t) <= 1e-4 for s, t in zip(p, q))
    got.mean().backward()
    ref.mean().backward()
    for (n, p), (_, q) in zip(gpu.named_parameters(), cpu.named_parameters()):
        assert util.scaled_rel(p.grad, q.grad) <= 1e-3, n


def test_token_by_token_is_the_segment(fwp):
    gpu, _ = models(True)
    gpu.pos_emb.inv_freq.zero_()        # positions count backwards from the end of a segment
    tokens = torch.randint(0, 50, (20, 5), generator=util.gen(4)).to(DEV)
    with torch.no_grad():
        whole, end = gpu(tokens[:-1], tokens[1:], None, carry_over_fast_weight=True)
        mems, parts = None, []
        for t in range(19):
            loss, mems = gpu(tokens[t:t + 1], tokens[t + 1:t + 2], mems, carry_over_fast_weight=True)
            parts.append(loss)
        # and a short last batch on a prefix of the memories
        prefix, _ = gpu(tokens[:3, :2], tokens[1:4, :2], end, carry_over_fast_weight=True)
    assert util.max_abs(torch.cat(parts), whole) <= 1e-4 and torch.isfinite(prefix).all()
    for p, q in zip(mems, end):
        assert all(s.shape == t.shape for s, t in zip(p, q))


def arguments(seed, N, L, D, S=16, dtype=F32, grad=False):
    g = util.gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)         # noqa: E731
    a = dict(x=r(N, L, D).to(dtype), dt=r(N, L, D).to(dtype), z=r(N, L, D).to(dtype), B=r(N, L, S).to(dtype), C=r(N, L, S).to(dtype),
             A=-r(D, S).abs(), D=r(D), dt_bias=r(D) - 2, w=r(D, 4), b=r(D), nw=r(D), res=r(N, L, D).to(dtype))
    return {k: t.to(DEV).requires_grad_(grad) for k, t in a.items()}


def together(fwp, a, window, state):
    """Convolution, scan, norm: what a layer runs."""
    u = fwp.causal_conv(a['x'], a['w'], a['b'], state=window)
    y = fwp.selective_scan(u, a['dt'], a['A'], a['B'], a['C'], a['D'], z=a['z'], dt_bias=a['dt_bias'], state=state)
    return fwp.block_norm(y, a['nw'], residual=a['res'], gate=a['z'], rms=True)


def memories(N, D, S=16):
    return torch.zeros(N, 3, D, device=DEV), torch.zeros(N, D, S, device=DEV)


def test_a_decoding_step_replayed_from_a_graph(fwp):
    N, D, steps = 6, 64, 7
    seq = arguments(5, N, steps, D)
    at = lambda t: {k: v[:, t:t + 1].clone() if v.dim() == 3 else v for k, v in seq.items()}       # noqa: E731
    eager_mem, graph_mem = memories(N, D), memories(N, D)
    with torch.no_grad():
        ref = [together(fwp, at(t), *eager_mem) for t in range(steps)]
        static = at(0)
        together(fwp, static, *memories(N, D))           # warm-up outside the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = together(fwp, static, *graph_mem)
        for m in graph_mem:
            m.zero_()
        for t in range(steps):
            for k, v in at(t).items():
                static[k].copy_(v)
            graph.replay()
            assert torch.equal(out[0], ref[t][0]) and torch.equal(out[1], ref[t][1])
    assert all(torch.equal(p, q) for p, q in zip(eager_mem, graph_mem))


@pytest.mark.parametrize('chunk', [0, 32])
def test_training_steps_replayed_from_two_graphs_in_turn(fwp, chunk):
    """Each graph has workspaces of its own (partial sums, checkpoints, span states): replayed alternately they disturb nothing."""
    from recurrent_fwp_b200 import _lib
    N, L, D = 2, 100, 48
    try:
        _lib.tune('scan.chunk', chunk)
        sets = [arguments(s, N, L, D, grad=True) for s in (6, 7)]
        gy = torch.randn(N, L, D, generator=util.gen(8)).to(DEV)

        def step(a, mem):
            for m in mem:
                m.zero_()
            y, r = together(fwp, a, *mem)
            return [y, r] + list(torch.autograd.grad([y, r], list(a.values()), [gy, gy]))
        refs = [[t.detach().clone() for t in step(a, memories(N, D))] for a in sets]
        graphs = []
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for a in sets:
                step(a, memories(N, D))
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a in sets:
            mem, graph = memories(N, D), torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(a, mem)
            graphs.append((graph, out, mem))
        for _ in range(3):
            for graph, _, _ in graphs:
                graph.replay()
        for (_, out, _), ref in zip(graphs, refs):
            assert all(torch.equal(p, q) for p, q in zip(out, ref))
    finally:
        _lib.tune('scan.chunk', 0)


def test_threads_and_streams_of_their_own(fwp):
    """Several host threads, each on its own stream, forward and backward at once: bit for bit what one after the other gives."""
    def work(seed):
        a = arguments(seed, 2 + seed % 3, 90 + seed, 40, grad=True)
        y, r = together(fwp, a, *memories(a['x'].shape[0], 40))
        return [t.detach() for t in (y, r)] + list(torch.autograd.grad([y, r], list(a.values()), [torch.ones_like(y), torch.ones_like(r)]))
    serial = [work(s) for s in range(8)]
    got, errors = [None] * 8, []

    def run(s):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[s] = work(s)
            stream.synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(s,)) for s in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for p, q in zip(serial, got):
        assert all(torch.equal(s, t) for s, t in zip(p, q))


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_offsets_beyond_31_bits(fwp, dtype):
    """Sequences more than 2^31 elements apart."""
    N, L, D, S = 2, 9, 64, 16
    far = 2 ** 31 + 64
    a = arguments(9, N, L, D, S, dtype)
    room = torch.empty(far + L * D, dtype=dtype, device=DEV)
    for k in ('x', 'dt', 'z', 'res'):
        apart = room.as_strided((N, L, D), (far, D, 1))
        apart.copy_(a[k])
        b = dict(a, **{k: apart})
        mem, mem2 = memories(N, D), memories(N, D)
        with torch.no_grad():
            got, ref = together(fwp, b, *mem), together(fwp, a, *mem2)
        assert all(torch.equal(p, q) for p, q in zip(got, ref)) and all(torch.equal(p, q) for p, q in zip(mem, mem2)), k


def test_sizes_beyond_the_kernels_are_refused(fwp):
    x = torch.randn(2, 3, 8, device=DEV)
    with pytest.raises(RuntimeError, match='beyond what the kernels cover'):
        fwp.causal_conv(x, torch.randn(8, 9, device=DEV))
    with pytest.raises(RuntimeError, match='beyond what the kernels cover'):
        fwp.selective_scan(x, x, -torch.ones(8, 65, device=DEV), torch.randn(2, 3, 65, device=DEV), torch.randn(2, 3, 65, device=DEV))
    with pytest.raises(RuntimeError, match='beyond what the kernels cover'):
        fwp.block_norm(torch.randn(2, 3, 8200, device=DEV), torch.ones(8200, device=DEV))
    with pytest.raises(RuntimeError, match='expanded'):
        fwp.causal_conv(x, torch.randn(8, 4, device=DEV), state=torch.zeros(1, 3, 8, device=DEV).expand(2, 3, 8))
    with pytest.raises(RuntimeError, match='lengths is'):
        fwp.causal_conv(x, torch.randn(8, 4, device=DEV), lengths=torch.tensor([3, 3]))


def ops(fwp):
    """name -> (leaves, call); every call starts from zero memories of its own."""
    a = arguments(10, 2, 120, 32)
    conv = [a['x'], a['w'], a['b']]
    scan = [a[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias')]
    norm = [a[k] for k in ('x', 'nw', 'b', 'res', 'dt_bias', 'z', 'D')]
    return {'conv': (conv, lambda *t: fwp.causal_conv(*t, state=t[0].new_zeros(2, 3, 32))),
            'scan': (scan, lambda *t: fwp.selective_scan(*t, state=t[0].new_zeros(2, 32, 16))),
            'norm': (norm, lambda *t: sum(fwp.block_norm(t[0], t[1], t[2], residual=t[3], scale=t[4], gate=t[5], post_weight=t[6])))}


@pytest.mark.parametrize('name', ['conv', 'scan', 'norm'])
def test_checkpointing_and_offloading(fwp, name):
    leaves, call = ops(fwp)[name]
    gy = torch.randn(2, 120, 32, generator=util.gen(11)).to(DEV)

    def grads(f):
        x = [t.clone().requires_grad_() for t in leaves]
        return torch.autograd.grad(f(*x), x, gy)

    def offloaded(*x):
        with torch.autograd.graph.save_on_cpu():
            return call(*x)
    ref = grads(call)
    for f in (offloaded, lambda *x: checkpoint(call, *x, use_reentrant=False)):
        assert all(torch.equal(p, q) for p, q in zip(ref, grads(f)))


@pytest.mark.parametrize('name', ['conv', 'scan', 'norm'])
def test_tracing_and_transforms(fwp, name):
    leaves, call = ops(fwp)[name]
    traced = torch.jit.trace(lambda *t: call(*t) * 2, tuple(t.flip(0) for t in leaves))
    x, r = ([t.clone().requires_grad_() for t in leaves] for _ in range(2))
    y, ref = traced(*x), call(*r) * 2
    assert torch.equal(y, ref)
    gy = torch.randn(y.shape, generator=util.gen(12)).to(DEV)
    for a, b in zip(torch.autograd.grad(y, x, gy), torch.autograd.grad(ref, r, gy)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: call(t, *leaves[1:]))(torch.stack([leaves[0]] * 2))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call(t, *leaves[1:]).sum())(leaves[0])


@pytest.mark.parametrize('name', ['conv', 'scan'])
def test_a_state_overwritten_before_the_backward(fwp, name):
    """No backward reads the state: a caller may reset it, or go on with the next segment, first."""
    a = arguments(14, 2, 40, 32, grad=True)
    window, state = (torch.randn_like(m) for m in memories(2, 32))

    def call():
        if name == 'conv':
            m = window.clone()
            return m, fwp.causal_conv(a['x'], a['w'], a['b'], state=m), [a['x'], a['w'], a['b']]
        m = state.clone()
        leaves = [a[k] for k in ('x', 'dt', 'A', 'B', 'C')]
        return m, fwp.selective_scan(*leaves, state=m), leaves
    m, y, leaves = call()
    ref = torch.autograd.grad(y.sum(), leaves)
    m, y, leaves = call()
    m.fill_(float('nan'))
    assert all(torch.equal(p, q) for p, q in zip(ref, torch.autograd.grad(y.sum(), leaves)))


def test_undefined_and_partial_gradients(fwp):
    """Leaves that need no gradient, outputs that nobody uses, gradients of another type."""
    a = arguments(13, 2, 30, 32, dtype=BF16)
    x = a['x'].clone().requires_grad_()
    y = fwp.selective_scan(x, a['dt'], a['A'], a['B'], a['C'])
    g, = torch.autograd.grad(y, [x], torch.ones(2, 30, 32, device=DEV).to(BF16))
    ref = blocks.selective_scan(a['x'], a['dt'], a['A'], a['B'], a['C'], gy=torch.ones(2, 30, 32, device=DEV))[2]['x']
    close('x', g, *ref, steps=30)
    w = a['nw'].clone().requires_grad_()
    y, r = fwp.block_norm(a['x'], w)
    assert not r.requires_grad or torch.autograd.grad(r.sum(), [w], retain_graph=True, allow_unused=True)[0].abs().sum() == 0
    assert torch.autograd.grad(y.float().sum(), [w])[0].shape == (32,)

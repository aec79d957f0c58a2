"""The state-space layer's operators refuse what their kernels would misread, on the host: the Python entry points by dtype, shape and
device, the C interface before any launch.  CPU tensors reach every check of the former (the CUDA-only one comes last)."""
import ctypes

import pytest
import torch

import recurrent_fwp_b200 as fwp
from recurrent_fwp_b200 import _lib

N, L, D, S, K = 2, 5, 8, 4, 4


def conv_args(dtype=torch.float32):
    return dict(x=torch.rand(N, L, D, dtype=dtype), weight=torch.rand(D, K), bias=torch.rand(D), state=torch.zeros(N, K - 1, D),
                lengths=torch.tensor([5, 3]))


def scan_args(dtype=torch.float32):
    r = lambda *s: torch.rand(*s, dtype=dtype)          # noqa: E731
    return dict(x=r(N, L, D), dt=r(N, L, D), A=-torch.rand(D, S), B=r(N, L, S), C=r(N, L, S), D=torch.rand(D), z=r(N, L, D),
                dt_bias=torch.rand(D), state=torch.zeros(N, D, S), lengths=torch.tensor([5, 3], dtype=torch.int32))


def norm_args(dtype=torch.float32):
    r = lambda: torch.rand(N, L, D, dtype=dtype)        # noqa: E731
    return dict(x=r(), weight=torch.rand(D), bias=torch.rand(D), residual=r(), scale=torch.rand(D), gate=r(), post_weight=torch.rand(D),
                post_bias=torch.rand(D))


def refuse(op, args, error, match, **change):
    with pytest.raises(error, match=match):
        op(**dict(args, **change))


def test_causal_conv_refusals():
    op, a = fwp.causal_conv, conv_args()
    refuse(op, a, RuntimeError, 'x must be', x=a['x'][0])
    refuse(op, a, TypeError, 'float32 or bfloat16', x=a['x'].half())
    refuse(op, a, RuntimeError, 'weight has shape', weight=torch.rand(D + 1, K))
    refuse(op, a, TypeError, 'weight must be float32', weight=a['weight'].bfloat16())
    refuse(op, a, RuntimeError, 'bias has shape', bias=torch.rand(D, 1))
    refuse(op, a, RuntimeError, 'state has shape', state=torch.zeros(N, K, D))
    refuse(op, a, TypeError, 'state must be float32', state=a['state'].bfloat16())
    refuse(op, a, TypeError, 'lengths must be', lengths=torch.tensor([5., 3.]))
    refuse(op, a, RuntimeError, 'lengths is', lengths=torch.tensor([5]))
    refuse(op, a, RuntimeError, 'no CPU path')
    refuse(op, conv_args(torch.bfloat16), RuntimeError, 'no CPU path')


def test_selective_scan_refusals():
    op, a = fwp.selective_scan, scan_args()
    refuse(op, a, RuntimeError, 'x must be', x=a['x'][0])
    refuse(op, a, TypeError, 'float32 or bfloat16', x=a['x'].double())
    refuse(op, a, TypeError, 'dt is torch.bfloat16', dt=a['dt'].bfloat16())
    refuse(op, a, TypeError, 'z is', z=a['z'].bfloat16())
    refuse(op, a, RuntimeError, 'dt has shape', dt=a['dt'][:, 1:])
    refuse(op, a, RuntimeError, 'C has shape', C=torch.rand(N, L, S + 1))
    refuse(op, a, RuntimeError, 'C has shape', B=a['B'].unsqueeze(2))
    refuse(op, a, RuntimeError, 'B has shape', B=torch.rand(N, L + 1, S))
    refuse(op, a, RuntimeError, 'do not fall into', B=torch.rand(N, L, 3, S), C=torch.rand(N, L, 3, S))
    refuse(op, a, RuntimeError, 'A has shape', A=torch.rand(D + 1, S))
    refuse(op, a, TypeError, 'A must be float32', A=a['A'].bfloat16())
    refuse(op, a, RuntimeError, 'at least one state', A=torch.rand(D, 0))
    refuse(op, a, RuntimeError, 'D has shape', D=torch.rand(1))
    refuse(op, a, RuntimeError, 'dt_bias has shape', dt_bias=torch.rand(D + 1))
    refuse(op, a, RuntimeError, 'state has shape', state=torch.zeros(N, S, D))
    refuse(op, a, TypeError, 'state must be float32', state=a['state'].double())
    refuse(op, a, RuntimeError, 'lengths is', lengths=torch.tensor([[5, 3]]))
    refuse(op, a, RuntimeError, 'no CPU path')


def test_block_norm_refusals():
    op, a = fwp.block_norm, norm_args()
    refuse(op, a, RuntimeError, 'x must be', x=a['x'][0, 0])
    refuse(op, a, TypeError, 'float32 or bfloat16', x=a['x'].half())
    refuse(op, a, TypeError, 'residual is', residual=a['residual'].bfloat16())
    refuse(op, a, RuntimeError, 'residual is', residual=a['residual'][:1])
    refuse(op, a, TypeError, 'gate is', gate=a['gate'].bfloat16())
    refuse(op, a, RuntimeError, 'gate has shape', gate=a['gate'][:, :1])
    for k in ('weight', 'bias', 'scale', 'post_weight', 'post_bias'):
        refuse(op, a, RuntimeError, k + ' has shape', **{k: torch.rand(D + 1)})
        refuse(op, a, TypeError, k + ' must be float32', **{k: torch.rand(D).bfloat16()})
    refuse(op, a, TypeError, 'scale must be', scale='half')
    refuse(op, a, RuntimeError, 'give post_weight', post_weight=None)
    refuse(op, a, ValueError, 'gate_act', gate_act='tanh')
    refuse(op, a, RuntimeError, 'no CPU path')
    refuse(op, dict(norm_args(torch.bfloat16), residual=torch.rand(N, L, D)), RuntimeError, 'no CPU path')


def test_states_that_cannot_be_written_in_place():
    with pytest.raises(RuntimeError, match='expanded'):
        _lib.require_state(torch.zeros(1, 3, 8).expand(4, 3, 8))
    with pytest.raises(RuntimeError, match='unit innermost'):
        _lib.require_state(torch.zeros(4, 8, 3).transpose(1, 2))
    _lib.require_state(torch.zeros(4, 3, 8)[:, 1:])
    _lib.require_state(None)


def fake(ptr=0x1000, stride3=1):
    t = _lib.FwpTensor()
    t.data = ptr
    t.stride[0], t.stride[1], t.stride[2], t.stride[3] = 4096, 0, 64, stride3
    return t


def test_the_c_interface_refuses_before_any_launch():
    ok, null, before = fake(), _lib.FwpTensor(), _lib.launch_count()
    vp = ctypes.c_void_p

    def conv(n=2, k=4, x=ok, w=0x1000, out=ok, dtype=0):
        return _lib.lib.fwp_causal_conv_forward(n, 5, 8, k, x, vp(w), None, null, None, out, 1, dtype, None, -1)
    assert conv(n=-1) == 2 and conv(k=0) == 2 and conv(n=70000) == 2
    assert conv(dtype=7) == 5 and conv(k=9) == 6 and conv(w=None) == 1 and conv(w=0x1002) == 4
    assert conv(x=null) == 1 and conv(out=null) == 1 and conv(x=fake(stride3=2)) == 3 and conv(x=fake(0x1002)) == 4
    assert conv(n=0) == 0
    assert _lib.lib.fwp_causal_conv_backward(2, 5, 8, 4, ok, vp(0x1000), None, null, None, ok, ok, None, None, None, 0, 1, 0, None, -1) == 1
    assert _lib.lib.fwp_causal_conv_backward_scratch_floats(2, 5, 8, 4) > 0

    def scan(d=8, s=4, g=1, a=0x1000, b=ok, z=null, keep=None, dtype=0):
        return _lib.lib.fwp_selective_scan_forward(2, 5, d, s, g, ok, ok, vp(a), b, ok, None, z, None, null, None, ok, vp(keep), None, 0, 1,
                                                   dtype, None, -1)
    assert scan(d=-8) == 2 and scan(s=0) == 2 and scan(g=0) == 2 and scan(g=3) == 2
    assert scan(s=65) == 6 and scan(dtype=2) == 5 and scan(a=None) == 1 and scan(a=0x1001) == 4
    assert scan(b=null) == 1 and scan(b=fake(stride3=3)) == 3 and scan(z=fake(0x1002)) == 4 and scan(keep=0x1004) == 4
    assert scan(d=0) == 0
    assert _lib.lib.fwp_selective_scan_checkpoint_floats(2, 9, 8, 3) == 2 * 2 * 8 * 4
    assert _lib.lib.fwp_selective_scan_checkpoint_floats(2, 9, 8, 65) == 0

    def norm(d=8, w=0x1000, x=ok, res=null, act=0, dtype=0, rdtype=0):
        return _lib.lib.fwp_block_norm_forward(2, 5, d, x, res, null, None, 1., None, None, vp(w), None, ok, ok, None, 1e-5, 0, act, dtype,
                                               rdtype, None, -1)
    assert norm(d=-1) == 2 and norm(d=8193) == 6 and norm(act=3) == 6 and norm(dtype=3) == 5 and norm(dtype=0, rdtype=1) == 5
    assert norm(w=None) == 1 and norm(w=0x1003) == 4 and norm(x=null) == 1 and norm(res=fake(0x1002)) == 4
    assert norm(d=0) == 0
    assert _lib.launch_count() == before


def test_the_definitions_agree_with_differences():
    """The oracle's gradients against central differences of its own outputs."""
    from oracle import blocks
    torch.manual_seed(1)
    d = lambda a: {k: t.double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for k, t in a.items()}      # noqa: E731
    for f, a, skip in ((blocks.causal_conv, d(conv_args()), ('state', 'lengths')), (blocks.selective_scan, d(scan_args()), ('state', 'lengths')),
                       (blocks.block_norm, d(norm_args()), ())):
        gy = torch.randn(N, L, D, dtype=torch.float64)
        grads = f(**a, gy=gy)[2]
        for k in set(a) - set(skip):
            v = torch.randn_like(a[k])
            plus, minus = (f(**dict(a, **{k: a[k] + e * v}))[0] for e in (1e-6, -1e-6))
            diff = ((plus - minus) * gy).sum() / 2e-6
            assert abs(diff - (grads[k][0] * v).sum()) < 1e-6 * (1 + abs(diff)), (f.__name__, k)

"""What stands between two blocks of a layer, in one launch: the norm behind a block, its gate and residual scale, the residual sum
and the norm before the next block.

    y, r = block_norm(x, weight, bias, residual=residual, scale=scale, gate=gate, post_weight=pw, post_bias=pb)

    t = norm(x) pw + pb   (x without post_weight)       u = t act(gate)   (t without gate)
    r = residual + scale u                              y = norm(r) weight + bias

  * ``x``, the output of a block, and ``gate`` (..., D) share one type, float32 or bfloat16; ``y`` has it too.  ``residual`` has that
    type or float32, and ``r``, the new residual, has the residual's.  Rows may have any outer strides, D <= 8192; with more than
    three dimensions, streams whose outer dimensions do not merge into one are copied first.
  * ``weight``, ``bias``, ``post_weight``, ``post_bias`` (D,) are float32; ``scale`` is a float32 (D,) tensor or a number.
  * ``gate_act``: 'silu', 'sigmoid' or 'identity'.  ``rms=True``: root-mean-square norms (no mean is taken off) instead of LayerNorms.
  * everything but x and weight may be left out; without a residual r is scale u.

Statistics are float32 over the values before r is rounded to its type.
"""
from recurrent_fwp_b200 import _lib

_ACTS = {'silu': 0, 'sigmoid': 1, 'identity': 2}


def _normalise(x, weight, bias, residual, scale, gate, post_weight, post_bias, gate_act, eps, rms):
    import torch
    if x.dim() < 2:
        raise RuntimeError('x must be of shape (..., D) with at least two dimensions, got %s' % (tuple(x.shape),))
    M = x.shape[-1]
    _lib.io_dtype(x)
    _lib.require_streams(x, {'gate': (gate, x.shape)})
    if residual is not None:
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError('residual is %s: it has the type of x (%s) or float32' % (residual.dtype, x.dtype))
        if residual.device != x.device or residual.shape != x.shape:
            raise RuntimeError('residual is %s on %s, expected %s on %s'
                               % (tuple(residual.shape), residual.device, tuple(x.shape), x.device))
    if scale is not None and not isinstance(scale, (int, float, torch.Tensor)):
        raise TypeError('scale must be a tensor or a number, got %s' % type(scale).__name__)
    vectors = {'weight': weight, 'bias': bias, 'scale': scale, 'post_weight': post_weight, 'post_bias': post_bias}
    _lib.require_f32(x, {n: (t, (M,)) for n, t in vectors.items() if isinstance(t, torch.Tensor)})
    if post_bias is not None and post_weight is None:
        raise RuntimeError('post_bias belongs to a norm behind the block: give post_weight too')
    _lib.require_cuda(x)
    x, residual, gate = (None if t is None else _lib.unit_inner(t) for t in (x, residual, gate))
    vec = {n: t.contiguous() if isinstance(t, torch.Tensor) else t for n, t in vectors.items()}
    return [x, vec['weight'], vec['bias'], residual, vec['scale'], gate, vec['post_weight'], vec['post_bias'], gate_act, eps, rms]


_block_norm = _lib.entry_point('block_norm', _normalise)


def block_norm(x, weight, bias=None, residual=None, scale=None, gate=None, post_weight=None, post_bias=None, gate_act='silu',
               eps=1e-5, rms=False):
    """The next block's normalised input y and the new residual r; see the module's text."""
    if gate_act not in _ACTS:
        raise ValueError("gate_act is 'silu', 'sigmoid' or 'identity', got %r" % (gate_act,))
    if x.dim() > 3:
        shape = x.shape
        x, residual, gate = (None if t is None else t.flatten(0, -2) if t.shape == shape else t for t in (x, residual, gate))
        y, r = _block_norm(x, weight, bias, residual, scale, gate, post_weight, post_bias, _ACTS[gate_act], eps, rms)
        return y.view(shape), r.view(shape)
    return _block_norm(x, weight, bias, residual, scale, gate, post_weight, post_bias, _ACTS[gate_act], eps, rms)

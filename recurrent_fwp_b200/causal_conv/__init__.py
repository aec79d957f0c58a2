"""Short causal convolution per channel with a carried window: what stands before the selective scan in a state-space layer.

    out = causal_conv(x, weight, bias, state=state)

    p_t = bias + sum_j weight[:, j] * x_{t-K+1+j},   out_t = silu(p_t)

  * ``x`` (N, L, D) in float32 or bfloat16, any outer strides; ``weight`` (D, K) with 1 <= K <= 8 and ``bias`` (D,) float32.
  * ``state`` (N, K-1, D) float32 holds the inputs before the first step, oldest first, and is overwritten with the last K - 1
    inputs, so that segments of a sequence, and single tokens (L = 1), follow on from one another.  Without it the steps before the
    first are zero.  No gradient flows to it, and ``backward`` leaves it alone.
  * ``lengths`` (N,) int32 or int64: a padded batch.  Steps at or beyond a sequence's length are not read, give zeros and take no
    gradient; the state is the one after the sequence's own last step.  Values outside 0 ... L count as the nearest of the two.
  * ``silu=False`` leaves the activation out.

The output's rows lie in the order of x's: (L, N, D) where x is a transposed (L, N, D) tensor.
"""
from recurrent_fwp_b200 import _lib


def _normalise(x, weight, bias, state, lengths, silu):
    if x.dim() != 3 or weight.dim() != 2:
        raise RuntimeError('x must be of shape (N, L, D) and weight (D, K), got %s and %s' % (tuple(x.shape), tuple(weight.shape)))
    N, L, D = x.shape
    K = weight.shape[1]
    _lib.io_dtype(x)
    _lib.require_f32(x, {'weight': (weight, (D, K))})
    _lib.require_f32(x, {n: (t, s) for n, t, s in (('bias', bias, (D,)), ('state', state, (N, K - 1, D))) if t is not None})
    lengths = _lib.sequence_lengths(x, lengths, N)
    _lib.require_cuda(x)
    _lib.require_state(state)
    return [_lib.unit_inner(x), weight.contiguous(), None if bias is None else bias.contiguous(), state, lengths, silu]


_causal_conv = _lib.entry_point('causal_conv', _normalise)


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    """Causal convolution of each channel over K steps; ``state`` carries the window in place.  Returns (N, L, D)."""
    return _causal_conv(x, weight, bias, state, lengths, silu)

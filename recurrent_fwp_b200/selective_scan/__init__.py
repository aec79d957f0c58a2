"""Selective scan: a state space per channel whose step size, input and output maps depend on the input, with a carried state.

    out = selective_scan(x, dt, A, B, C, D, z=z, dt_bias=dt_bias, state=state)

    delta_t = softplus(dt_t + dt_bias)
    h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,   y_t = <C_t, h_t> + D x_t,   out_t = y_t silu(z_t)

  * ``x``, ``dt``, ``z`` (N, L, D) and ``B``, ``C`` (N, L, S), or (N, L, G, S) for G groups of D / G channels, share one type,
    float32 or bfloat16, and take any outer strides (slices of a projection as they are).  ``A`` (D, S) with S <= 64, ``D`` (D,)
    and ``dt_bias`` (D,) are float32.  ``D``, ``z`` and ``dt_bias`` may be left out; ``softplus=False`` takes dt + dt_bias as it is.
    A may have either sign: states that grow (A > 0, or negative step sizes) are as far from the definition as float32 steps leave them.
    Minus infinity is a state that keeps nothing.
  * ``state`` (N, D, S) float32 enters as the state before the first step and is overwritten with the state after the last, so that
    segments, and single tokens (L = 1), follow on from one another.  Without it the scan starts from zeros.  As with the fast weight
    ops no gradient flows to it; unlike theirs, ``backward`` does not rewind it (a state that decays cannot be run backwards).
  * ``lengths`` (N,) int32 or int64: a padded batch.  Steps at or beyond a sequence's length are not read, give zeros and take no
    gradient; the state is the one after the sequence's own last step.  Values outside 0 ... L count as the nearest of the two.

A call that needs gradients keeps the state before every eighth step for its backward, 4 S / 8 bytes per (step, channel).  The backward
itself takes, while it runs, partial sums for the gradients of B and C: about S * S / 128 bytes per (step, channel), so 2 at 16 states and
32 at 64, and no less than 8 S bytes per step and group.
The output's rows lie in the order of x's.  States are float32 and all sums are taken in float32.
"""
from recurrent_fwp_b200 import _lib


def _normalise(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus):
    if x.dim() != 3 or A.dim() != 2 or B.dim() not in (3, 4):
        raise RuntimeError('x must be of shape (N, L, D), A (D, S) and B (N, L, S) or (N, L, G, S), got %s, %s and %s'
                           % (tuple(x.shape), tuple(A.shape), tuple(B.shape)))
    N, L, M = x.shape
    S = A.shape[1]
    _lib.io_dtype(x)
    shared = (N, L, S) if B.dim() == 3 else (N, L, B.shape[2], S)
    if B.dim() == 4 and (B.shape[2] == 0 or M % B.shape[2]):
        raise RuntimeError('%d channels do not fall into %d groups' % (M, B.shape[2]))
    if S < 1:
        raise RuntimeError('A must have at least one state per channel')
    _lib.require_streams(x, {'dt': (dt, (N, L, M)), 'B': (B, shared), 'C': (C, shared), 'z': (z, (N, L, M))})
    _lib.require_f32(x, {'A': (A, (M, S))})
    _lib.require_f32(x, {n: (t, s) for n, t, s in (('D', D, (M,)), ('dt_bias', dt_bias, (M,)), ('state', state, (N, M, S)))
                         if t is not None})
    lengths = _lib.sequence_lengths(x, lengths, N)
    _lib.require_cuda(x)
    _lib.require_state(state)
    x, dt, B, C, z = (None if t is None else _lib.unit_inner(t) for t in (x, dt, B, C, z))
    A, D, dt_bias = (None if t is None else t.contiguous() for t in (A, D, dt_bias))
    return [x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus]


_selective_scan = _lib.entry_point('selective_scan', _normalise)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None, softplus=True):
    """Selective scan over (N, L, D) streams; ``state`` is carried in place.  Returns (N, L, D)."""
    return _selective_scan(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus)

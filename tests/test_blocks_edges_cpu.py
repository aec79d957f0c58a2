"""Host side of the state-space layer's operators at the end of what they take: sizes of zero, plans, workspaces."""
import pytest
import torch

import recurrent_fwp_b200 as fwp
from recurrent_fwp_b200 import _lib


@pytest.mark.parametrize('shape', [(2, 0), (2, 3, 0), (2, 3, 4, 0), (2, 0, 4, 0), (2, 0, 4, 8)])
def test_rows_without_elements_get_as_far_as_others(shape):
    """Every check but the last, which is that the tensors are on a GPU."""
    with pytest.raises(RuntimeError, match='no CPU path'):
        fwp.block_norm(torch.zeros(shape), torch.zeros(shape[-1]), residual=torch.zeros(shape), gate=torch.zeros(shape))


def spans_of(N, L, D, S, G=1):
    """How many spans the forward of the selective scan takes, from the size of its workspace."""
    floats = _lib.lib.fwp_selective_scan_scratch_floats(N, L, D, S, G, -1)
    assert floats % (N * D * (S + 1)) == 0
    return max(1, floats // (N * D * (S + 1)))


@pytest.mark.parametrize('shape', [(1, 2048, 16), (2, 2048, 16), (1, 512, 16), (6, 518, 16), (1, 64, 4), (1, 1024, 64), (4, 2048, 16), (8, 2048, 16)])
def test_spans_are_taken_where_they_shorten_the_chain(shape):
    """A span is walked twice, with two launches between: less than the sequence in one go, or one go it is."""
    N, D, S = shape
    taken = []
    for L in list(range(2, 400)) + [777, 2048, 16384]:
        n = spans_of(N, L, D, S)
        span = next(s for s in range(32, L + 32, 32) if -(-L // s) <= n)
        assert n == 1 or 2 * span < L, (L, n)
        taken.append(n)
    many = N * -(-D // (256 // max(1, -(-S // 4)))) * 3 > 148 * 2       # CTAs, of 64 channels at 16 states
    assert (max(taken) == 1) == many


def test_the_last_step_of_the_last_span_is_an_int():
    """Spans asked for by ``scan.chunk`` are rounded up to 32 steps each; behind the longest sequence all of them end below 2^31."""
    longest = 0x7fff0000
    try:
        _lib.tune('scan.chunk', 32)
        n = spans_of(1, longest, 1, 1)
    finally:
        _lib.tune('scan.chunk', 0)
    span = -(-(-(-longest // n)) // 32) * 32
    assert n * span < 2 ** 31

"""The language model's state-space layer and its fused norms, with plain forms in place of the CUDA ops."""
import pytest
import torch

from recurrent_fwp_b200.lm_harness import DeltaNetLM
from tests import state_space_util as plain
from tests import util
from tests.test_lm_harness_cpu import CHECKER_OPS, RECURRENT, build, checker_delta


def model(fused_norm=False, **kw):
    torch.manual_seed(2)
    return DeltaNetLM(50, 3, 2, 32, 16, 48, attn_type='scan', ops=plain.OPS, fused_norm=fused_norm, norm_fn=plain.norm, **kw).double().eval()


def test_the_plain_forms_are_the_definitions():
    plain.check_against_the_definitions()


def test_carried_segments_are_one_sequence():
    m = model()
    tokens = torch.randint(0, 50, (25, 2), generator=util.gen(3))
    # positions count backwards from a segment's end, so the layers' inputs are the same only without them
    m.pos_emb.inv_freq.zero_()
    with torch.no_grad():
        whole, mems = m(tokens[:-1], tokens[1:], None, carry_over_fast_weight=True)
        carried, parts = None, []
        for lo, hi in ((0, 7), (7, 8), (8, 24)):
            loss, carried = m(tokens[lo:hi], tokens[lo + 1:hi + 1], carried, carry_over_fast_weight=True)
            parts.append(loss)
    assert torch.allclose(torch.cat(parts), whole, atol=1e-5)       # the memories are float32
    for a, b in zip(mems, carried):
        assert all(torch.allclose(p, q, atol=1e-5) for p, q in zip(a, b))
    assert [t.shape for t in mems[0]] == [(2, 3, 64), (2, 64, 16)]


@pytest.mark.parametrize('kind', ['scan', 24] + sorted(RECURRENT))
def test_fused_norms_change_nothing_but_rounding(kind):
    if kind == 'scan':
        a, b = model(), model(True)
        tokens = torch.randint(0, 50, (14, 2), generator=util.gen(4))
        L = 13
    else:
        gd = util.golden('lm_delta' if kind == 24 else kind)
        kw = dict(delta_fn=checker_delta) if kind == 24 else dict(delta_fn=None, attn_type=RECURRENT[kind], ops=CHECKER_OPS)
        a, b = build(gd, **kw), build(gd, **kw)
        b.norm_fn = plain.norm
        tokens, L = gd['tokens'], gd['loss_plain'].shape[0]
    la, ma = a(tokens[:L], tokens[1:L + 1], None, carry_over_fast_weight=True)
    lb, mb = b(tokens[:L], tokens[1:L + 1], None, carry_over_fast_weight=True)
    assert util.max_abs(la, lb) <= 1e-5
    for p, q in zip(ma, mb):
        assert all(s is None or util.max_abs(s, t) <= 1e-5 for s, t in zip(p, q))


def test_unknown_layer_types_are_refused():
    with pytest.raises(ValueError, match='scan'):
        DeltaNetLM(50, 1, 2, 32, 16, 48, attn_type='other')

"""Host side of the state-space layer's operators at the end of what they take: sizes of zero, plans, workspaces."""
import pytest
import torch

import recurrent_fwp_b200 as fwp


@pytest.mark.parametrize('shape', [(2, 0), (2, 3, 0), (2, 3, 4, 0), (2, 0, 4, 0), (2, 0, 4, 8)])
def test_rows_without_elements_get_as_far_as_others(shape):
    """Every check but the last, which is that the tensors are on a GPU."""
    with pytest.raises(RuntimeError, match='no CPU path'):
        fwp.block_norm(torch.zeros(shape), torch.zeros(shape[-1]), residual=torch.zeros(shape), gate=torch.zeros(shape))

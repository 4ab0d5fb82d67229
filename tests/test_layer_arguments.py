"""What the modules around the operators do with arguments and with being moved (no GPU: nothing is launched)."""
import pytest
import torch

import simplical_attn_b200 as sab


@pytest.mark.parametrize("module", [sab.CausalSelfAttention, sab.TwoSimplicialSelfAttention])
def test_positions_without_rotary_are_refused(module):
    """A module made without `rotary` has no use for positions: given some, a rotation was meant."""
    m = module(32, 2, 16, dtype=torch.float32)
    with pytest.raises(ValueError, match="rotary"):
        m(torch.zeros(1, 4, 32), positions=torch.arange(4))

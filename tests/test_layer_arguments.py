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


def same(a, b):
    return a.dtype == b.dtype == torch.float64 and a.device == b.device and torch.equal(a, b)


def test_frequencies_survive_being_moved():
    """The frequencies are not in a state_dict: a module that is made without memory, or emptied, has them all the same."""
    args = dict(rotary_dim=16, base=500000.0, scaling="parts", factor=4.0, original_length=4096)
    want = sab.rotary_frequencies(**args)
    assert same(sab.RotaryPositions(**args).to_empty(device="cpu").frequencies, want)
    for made in (lambda: sab.RotaryPositions(**args, device="meta"), lambda: in_context(torch.device("meta"), lambda: sab.RotaryPositions(**args))):
        m = made()
        assert m.frequencies.is_meta and m.frequencies.dtype == torch.float64
        assert m.half().frequencies.is_meta and m.frequencies.dtype == torch.float64
        assert same(m.to_empty(device="cpu").frequencies, want) and same(m.bfloat16().frequencies, want)
    layer = in_context(torch.device("meta"), lambda: sab.CausalSelfAttention(32, 2, 16, rotary=sab.RotaryPositions(**args)))
    assert same(layer.to_empty(device="cpu").rotary.frequencies, want)
    m = sab.RotaryPositions(**args)
    m.frequencies.mul_(2)                       # (one's own values stay)
    assert same(m.half().to("cpu").frequencies, 2 * want)


def in_context(context, make):
    with context:
        return make()

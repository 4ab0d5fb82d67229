"""Causal attention with the same starts for queries and keys, in tensors of different rows."""
import pytest
import torch

import simplical_attn_b200 as sab
from simplical_attn_b200 import _abi
from tests.test_causal import make, step

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_starts_given_for_both(native, monkeypatch):
    """K and V in a longer buffer than Q: `cu_k` may be the tensor that `cu_q` is.  Left out, other rows are taken for a mistake."""
    (q, k, v, d_o), (cu, _), _ = make([(70, 70), (33, 33)], 4, 2, 64, "bf16", seed=61)
    want = step(q, k, v, d_o, cu_q=cu)
    longer = [torch.cat((t, t[:20])) for t in (k, v)]
    if not native:
        monkeypatch.setattr(_abi, "_binding", False)
    got = step(q, *longer, d_o, cu_q=cu, cu_k=cu)
    for n in want:
        assert torch.equal(got[n][:103] if n in ("dk", "dv") else got[n], want[n]), n
    assert not got["dk"][103:].any() and not got["dv"][103:].any()
    o, lse = sab.causal_attention_fwd(q, *longer, 0.125, cu, cu)
    assert torch.equal(sab.causal_attention_bwd(q, *longer, o, lse, d_o, 0.125, cu, cu)[2][:103], want["dv"])
    for call in (lambda: sab.causal_attention(q, *longer, cu_q=cu), lambda: sab.causal_attention_fwd(q, *longer, 0.125, cu),
                 lambda: sab.causal_attention_bwd(q, *longer, o, lse, d_o, 0.125, cu)):
        with pytest.raises(ValueError, match="without cu_k"):
            call()

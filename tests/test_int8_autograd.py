"""What the int8 operators do under autograd beyond the plain backward pass."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from int_model_approximation_b200 import int8
from test_int8 import make, status_clean


# ---------------------------------------------------------------------------
# forward-mode tangents
# ---------------------------------------------------------------------------
def test_tangents_are_seen():
    t = torch.ones(3)
    int8._refuse_tangents(t, None)
    with forward_ad.dual_level():
        int8._refuse_tangents(t, None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            int8._refuse_tangents(None, forward_ad.make_dual(t, t))


@pytest.mark.gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(cuda_device, requires_grad):
    x, w, b = make(4, 8, 32, torch.float32, 61, cuda_device, bias=True)
    wt = int8.Int8Weight.from_float(w)
    x.requires_grad_(requires_grad)
    with forward_ad.dual_level():
        dual, dual_bias = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(b, torch.ones_like(b))
        calls = [lambda: int8.int8_linear(dual, wt), lambda: int8.int8_linear(x, wt, dual_bias),
                 lambda: int8.int8_linear(x, forward_ad.make_dual(w, w)), lambda: int8.int8_gated(dual, wt, wt),
                 lambda: int8.int8_gated(x, wt, wt, None, dual_bias)]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        y = int8.int8_linear(x, wt)
    assert torch.equal(y, int8.int8_linear(x, wt))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: int8.int8_linear(t, wt), (x.detach(),), (torch.ones_like(x),))
    status_clean(cuda_device)

"""Sizes near the limits that the header states for ``tsc_unembed_*``."""
import pytest
import torch

from test_unembed import DEV


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
def test_no_rows_of_more_than_2_to_the_32_weights(tied):
    """The gradients of no rows are zero everywhere, also where dW has more elements than a launch has threads."""
    import tsc_hip

    D, V = 32768, 131201  # 4.3e9: 8.6 GB
    W = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV).t() if tied else torch.zeros(D, V, dtype=torch.bfloat16, device=DEV)
    b = torch.zeros(V, dtype=torch.bfloat16, device=DEV)
    head = tsc_hip.UnembedHead(W, b)
    x, none = torch.empty(0, D, dtype=torch.bfloat16, device=DEV), torch.empty(0, device=DEV)
    dirty = torch.full((D * V,), 1.0, dtype=torch.bfloat16, device=DEV)  # what dW's memory holds before
    del dirty
    dx, dW, db = head.loss_backward(none, x, torch.empty(0, dtype=torch.long, device=DEV), none)
    assert dx.shape == x.shape and dW.shape == W.shape and not db.any()
    flat = (dW.t() if tied else dW).view(-1)
    assert not any(bool(part.any()) for part in flat.split(1 << 30))

"""Changes of a model's weights that its head has to see (``lm_head.model_head``)."""
import pytest
import torch

from test_lm_head import model_of, tokens_of
from test_unembed import DEV


def fresh(m, tok):
    """The loss through a head that was made of the weights as they are."""
    import lm_head
    import tsc_hip

    final = m.run_with_cache(tok)[1]["ln_final.hook_normalized"]
    return lm_head.next_token_loss(final, tok, tsc_hip.UnembedHead(m.W_U.clone(), m.b_U.clone()), per_token=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inference", [False, True])
def test_changes_in_place(inference, dtype):
    with torch.inference_mode(inference):
        m = model_of(DEV, dtype=dtype)
        assert m.W_U.is_inference() == inference
        tok = tokens_of(m)
        last = m(tok, return_type="loss", loss_per_token=True)
        for change in (lambda: m.W_U.mul_(1.5), lambda: m.b_U.add_(torch.arange(301, device=DEV, dtype=dtype) / 64),
                       lambda: m.W_U.copy_(m.W_U.flip(1)), lambda: m.b_U.zero_()):
            change()
            got = m(tok, return_type="loss", loss_per_token=True)
            assert torch.equal(got, fresh(m, tok)) and not torch.equal(got, last)
            last = got

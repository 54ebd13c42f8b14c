"""``TaskEvaluation.answer_loss`` / ``loss_directions`` go through a final layer norm without weights and an unembedding: a model
whose head is another one is refused, where its loss would be wrong without a word."""
from types import SimpleNamespace

import pytest
import torch


@pytest.mark.parametrize("cfg,more", [
    ({"normalization_type": "LN"}, {}), ({"normalization_type": "RMSPre"}, {}), ({"normalization_type": None}, {}),
    ({"normalization_type": "LNPre"}, {"ln_final": SimpleNamespace(w=torch.ones(4), b=torch.zeros(4))}),
    ({"normalization_type": "LNPre", "output_logits_soft_cap": 30.0}, {}),
])
def test_other_heads_are_refused(cfg, more):
    from task_evaluation import TaskEvaluation

    te = object.__new__(TaskEvaluation)
    te.model, te.prompts = SimpleNamespace(cfg=SimpleNamespace(n_layers=2, eps=1e-5, **cfg), **more), []
    for call in (te.answer_loss, te.loss_directions, lambda: te.loss_directions(at="resid")):
        with pytest.raises(NotImplementedError):
            call()

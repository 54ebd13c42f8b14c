"""Task-level entry to the batched CircuitLens pass ("CircuitLens feature-contribution
decomposition for batched IOI prompts, all layers, logit-diff direction").

Drop-in for the hot-path part of ``TaskEvaluation`` (reference ``src/task_evaluation.py``): the constructor
(:111-139: prompts -> token matrix, optional mean cache), ``str_prompts`` (:153-155) and ``logit_difference``
(:141-151), which defines the direction the decomposition is scored against.  The circuit-discovery driver, the
mean-ablation faithfulness loop and the plots of that class are the graph-search layer (out
of scope) and raise.  New here: ``logit_difference_directions`` and ``contribution_decomposition`` -- all prompts
in one ``BatchedCircuitLens`` pass instead of one ``CircuitLens`` per prompt.
"""
from __future__ import annotations

from typing import Callable, List, Optional

import torch

import lm_head
import tsc_hip
from circuit_lens import BatchedCircuitLens
from load_model_and_encoders import get_model_encoders


def all_allowed(_component: str) -> bool:  # circuit_discovery.all_allowed, the reference's default filter
    return True


class TaskEvaluation:
    def __init__(self, prompts: List[dict], circuit_discovery_strategy: Optional[Callable] = None,
                 allowed_components_filter: Callable[[str], bool] = all_allowed, eval_index: int = -1,
                 no_mean_cache=False):
        self.device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
        self.model = get_model_encoders(self.device)[0]
        self.circuit_discovery_strategy = circuit_discovery_strategy
        self.prompts = prompts
        self.tokens = self.model.to_tokens(self.str_prompts)
        self.eval_index = eval_index
        self.allowed_components_filter = allowed_components_filter
        self._batched: Optional[BatchedCircuitLens] = None
        if no_mean_cache:
            return
        with torch.no_grad():
            logits, cache = self.model.run_with_cache(self.tokens, return_type="logits")
        self.mean_cache = {key: value.mean(dim=0) for key, value in cache.items()}  # :133-138
        self.mean_logits = logits.mean(dim=0)

    @property
    def str_prompts(self):
        return [p["text"] for p in self.prompts]

    def logit_difference(self, prompt_idx: int):
        """Unembedding direction ``correct - counter`` (:141-151), exactly as the reference computes it:
        ``to_tokens`` prepends BOS (and may split a name into several tokens), so the result has one row per
        token of the tokenised answers, all but the last being ``W_U[:, bos] - W_U[:, bos] = 0``."""
        correct_token = self.prompts[prompt_idx]["correct"]
        counter_token = self.prompts[prompt_idx]["counter"]
        if correct_token is None or counter_token is None:
            raise ValueError("Prompt does not have correct or counter token")
        toks = self.model.to_tokens([correct_token, counter_token]).squeeze()
        unembed = self.model.tokens_to_residual_directions(toks)
        return unembed[0] - unembed[1]

    # ------------------------------------------------------------------ batched form (new)
    def logit_difference_directions(self) -> torch.Tensor:
        """``[n_prompts, d_model]``: for every prompt the last row of ``logit_difference`` -- the answer tokens'
        ``W_U[:, correct] - W_U[:, counter]`` -- gathered in one indexing operation."""
        correct = self.model.to_tokens([p["correct"] for p in self.prompts])[:, -1]
        counter = self.model.to_tokens([p["counter"] for p in self.prompts])[:, -1]
        w_u = self.model.W_U
        return (w_u[:, correct] - w_u[:, counter]).t().contiguous()

    def batched_lens(self, positions="eval") -> BatchedCircuitLens:
        """All prompts through ONE dictionary pass; ``positions="eval"`` covers ``eval_index`` of every prompt,
        ``"all"`` every position (what per-prompt circuit discovery walks back through)."""
        pos = self.eval_index if positions == "eval" else positions
        if self._batched is None or self._batched.positions != pos:
            self._batched = BatchedCircuitLens(self.str_prompts, positions=pos)
        return self._batched

    def contribution_decomposition(self, k: int = 10, positions="eval", directions: Optional[torch.Tensor] = None):
        """Per prompt, at ``eval_index``: every component's normalised contribution to the prompt's direction (its
        logit difference, or ``directions [n_prompts, d_model]``, e.g. ``loss_directions()``) and the top-``k`` of them
        (``BatchedCircuitLens.direction_lens``)."""
        if directions is None:
            directions = self.logit_difference_directions()
        return self.batched_lens(positions).direction_lens(directions, k=k)

    # ------------------------------------------------------------------ the answer's loss (new)
    @torch.no_grad()
    def _answer_rows(self):
        """Every prompt's final residual at ``eval_index`` of its own length (as ``BatchedCircuitLens``: padding sits behind
        it), normalised, and its answer's last token."""
        model = self.model
        if getattr(model.cfg, "normalization_type", "LNPre") != "LNPre" or not lm_head._plain_head(model):
            raise NotImplementedError("the answer's loss is that of a model with a folded final layer norm and uncapped logits")
        if any(p["correct"] is None for p in self.prompts):
            raise ValueError("Prompt does not have correct token")
        name = f"blocks.{model.cfg.n_layers - 1}.hook_resid_post"
        cache = model.run_with_cache(self.tokens, return_type=None, names_filter=[name])[1]
        pos = [self.eval_index % int(model.to_tokens(t).shape[1]) for t in self.str_prompts]
        resid = cache[name][torch.arange(len(pos), device=self.tokens.device), torch.tensor(pos, device=self.tokens.device)]
        answers = torch.cat([model.to_tokens(p["correct"])[0, -1:] for p in self.prompts]).to(resid.device)
        return resid, tsc_hip.layer_norm(resid, eps=model.cfg.eps), answers, lm_head.model_head(model)

    @torch.no_grad()
    def answer_loss(self) -> torch.Tensor:
        """``[n_prompts]``: the cross entropy of every prompt's correct answer (its last token) at ``eval_index``."""
        _, (normalized, _, _), answers, head = self._answer_rows()
        return head.loss(normalized, answers)[0]

    @torch.no_grad()
    def loss_directions(self, at: str = "normalized") -> torch.Tensor:
        """``[n_prompts, d_model]``: the direction that lowers each prompt's ``answer_loss`` fastest.  ``at="normalized"``:
        the negative gradient at the final normalised residual, ``W_U[:, correct] - sum_v p_v W_U[:, v]`` -- what
        ``logit_difference_directions`` is with the model's own distribution in the counter token's place;
        ``at="resid"``: the negative gradient at the residual before the layer norm."""
        if at not in ("normalized", "resid"):
            raise ValueError(f"at must be 'normalized' or 'resid' (got {at!r})")
        resid, (normalized, mean, scale), answers, head = self._answer_rows()
        lse = head.loss(normalized, answers)[1]
        down = head.loss_backward(torch.full_like(lse, -1.0), normalized, answers, lse, want_weight=False, want_bias=False)[0]
        return down if at == "normalized" else tsc_hip.layer_norm_backward(down, resid, mean, scale)[0]

    # ------------------------------------------------------------------ out of scope
    def _out_of_scope(self, *a, **k):
        raise NotImplementedError("circuit discovery and mean-ablation evaluation are the reference's graph-search "
                                  "layer (SURVEY.md section 2.1); use BatchedCircuitLens.lens(i) to feed it")

    get_circuit_discovery_for_prompt = _out_of_scope
    get_faithfulness_curve_over_data = _out_of_scope
    get_attn_head_freqs_over_dataset = _out_of_scope
    get_features_at_heads_over_dataset = _out_of_scope

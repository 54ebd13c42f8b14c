"""``get_test_loss`` with the model that a user has: one that is hooked like TransformerLens' and computes its own ``"loss"`` from
its logits.  On a GPU it is asked for its final normalised residual only (``lm_head.hooked_loss``)."""
from types import SimpleNamespace

import pytest
import torch
from torch import nn

from test_lm_head import _dictionary_configs, model_of, tokens_of
from test_unembed import DEV


class Hooked(nn.Module):
    """A model around the stand-in's layers, with parameters as weights of its unembedding, that notes what it is asked for."""

    def __init__(self, inner, **more):
        super().__init__()
        self.inner, self.asked = inner, []
        self.unembed_W, self.unembed_b = nn.Parameter(inner.W_U.clone()), nn.Parameter(inner.b_U.clone())
        self.cfg = SimpleNamespace(output_logits_soft_cap=-1.0)
        for k, v in more.items():
            setattr(self, k, v)

    W_U = property(lambda self: self.unembed_W)
    b_U = property(lambda self: self.unembed_b)

    def run_with_hooks(self, tokens, return_type="logits", fwd_hooks=()):
        self.asked.append(return_type)
        if return_type is None:
            return self.inner.run_with_hooks(tokens, return_type=None, fwd_hooks=fwd_hooks)
        logits = self.inner.run_with_hooks(tokens, return_type="logits", fwd_hooks=fwd_hooks)
        tokens = torch.atleast_2d(tokens).to(logits.device)
        return torch.nn.functional.cross_entropy(logits[:, :-1].double().flatten(0, 1), tokens[:, 1:].flatten())


def dictionaries(m, monkeypatch):
    """A transcoder, an SAE and a z-SAE that reconstruct with a factor."""
    from mlp_transcoder import SparseTranscoder
    from z_sae import ZSAE

    cfg = _dictionary_configs(m, 1)
    tc, sae = SparseTranscoder(cfg(True, "blocks.1.ln2.hook_normalized")), SparseTranscoder(cfg(False, "blocks.0.hook_resid_post"))
    z = ZSAE({"dict_size": 64, "l1_coeff": 1.0, "enc_dtype": "fp32", "seed": 0, "act_size": 48, "device": "cpu", "layer": 0})
    monkeypatch.setattr(tc, "forward", lambda x: (0.5 * x,))
    monkeypatch.setattr(sae, "forward", lambda x: (0.75 * x,))
    monkeypatch.setattr(z, "forward", lambda x: (None, 0.25 * x))
    return tc, sae, z


def test_on_the_cpu_the_model_computes_its_loss(monkeypatch):
    inner = model_of()
    m, tok = Hooked(inner), tokens_of(inner)
    for d in dictionaries(inner, monkeypatch):
        assert abs(float(d.get_test_loss(tok, m)) - float(d.get_test_loss(tok, inner))) < 1e-5  # (fp32 there, fp64 here)
    assert m.asked == ["loss"] * 3


@pytest.mark.gpu
def test_no_logits_on_the_gpu(monkeypatch):
    inner = model_of(DEV)
    m, tok = Hooked(inner), tokens_of(inner)
    got, want = [], []
    for d in dictionaries(inner, monkeypatch):
        got.append(d.get_test_loss(tok, m))
        assert torch.equal(d.get_test_loss(tok[1], m), d.get_test_loss(tok[1:2].cpu(), m))
        want.append(d.get_test_loss(tok, inner))
    assert set(m.asked) == {None}
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and len({float(g) for g in got}) == 3
    for g, d in zip(got, dictionaries(inner, monkeypatch)):
        own = Hooked(inner, tokenizer=SimpleNamespace(padding_side="left"))
        assert abs(float(g) - float(d.get_test_loss(tok, own))) < 1e-5 and own.asked == ["loss"]
    with torch.no_grad():  # an optimiser's step on the parameters
        for p, q in ((m.unembed_W, inner.W_U), (m.unembed_b, inner.b_U)):
            p.mul_(1.5)
            q.mul_(1.5)
    for g, d in zip(got, dictionaries(inner, monkeypatch)):
        again = d.get_test_loss(tok, m)
        assert torch.equal(again, d.get_test_loss(tok, inner)) and not torch.equal(again, g)


@pytest.mark.gpu
@pytest.mark.parametrize("more", [
    {"ln_final": SimpleNamespace(w=torch.ones(48), b=torch.zeros(48))},       # a norm that kept its weights
    {"cfg": SimpleNamespace(output_logits_soft_cap=30.0)},
    {"tokenizer": SimpleNamespace(padding_side="left")},
    {"hook_dict": {"blocks.0.hook_resid_post": None}},                        # no final norm
])
def test_a_head_that_is_more_computes_its_own_loss(more, monkeypatch):
    inner = model_of(DEV)
    m, tok = Hooked(inner, **more), tokens_of(inner)
    for d in dictionaries(inner, monkeypatch):
        d.get_test_loss(tok, m)
    assert m.asked == ["loss"] * 3


@pytest.mark.gpu
def test_types_that_the_operator_does_not_take(monkeypatch):
    inner = model_of(DEV, dtype=torch.float64)
    m, tok = Hooked(inner), tokens_of(inner)
    for d in dictionaries(inner, monkeypatch):
        d.get_test_loss(tok, m)
    assert m.asked == ["loss"] * 3
    m = Hooked(model_of(DEV))
    m.unembed_W = nn.Parameter(m.unembed_W.detach().bfloat16())
    m.unembed_b = nn.Parameter(m.unembed_b.detach().bfloat16())
    d = dictionaries(m.inner, monkeypatch)[0]
    d.get_test_loss(tok, m)
    assert m.asked == [None, "loss"]  # (its residual is of another type than its unembedding)


@pytest.mark.gpu
def test_the_loss_of_a_model_in_64_bits():
    m = model_of(DEV, dtype=torch.float64)
    tok = tokens_of(m)
    logits, loss = m(tok, return_type="both")
    want = torch.nn.functional.cross_entropy(logits[:, :-1].flatten(0, 1), tok[:, 1:].flatten())
    assert loss.dtype == torch.float64 and abs(float(loss) - float(want)) < 1e-12
    each = m(tok, return_type="loss", loss_per_token=True)
    assert each.shape == (3, 8) and abs(float(each.mean()) - float(want)) < 1e-12

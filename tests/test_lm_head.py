"""Layer norm and the loss behind the unembedding as one runs them: as autograd operators in a row, as a model's loss, as the
loss with a dictionary in the model, and as the direction of a prompt's answer (``lm_head``, ``standins``,
``SparseTranscoder`` / ``ZSAE.get_test_loss``, ``TaskEvaluation``).

The kernels have their own bounds against float64 (``test_layer_norm``, ``test_unembed``); a chain of them is compared bit for
bit with the same calls made one by one, and with differences of the formulas in float64."""
import copy
import math

import pytest
import torch

from test_unembed import reference as loss_reference

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def model_of(device="cpu", **kw):
    from standins.synthetic_model import SyntheticHookedTransformer

    args = dict(n_layers=2, d_model=48, n_heads=4, d_vocab=301, n_ctx=16, seed=3, device=device)
    return SyntheticHookedTransformer(**{**args, **kw})


def tokens_of(model, b=3, n=9, seed=0):
    return torch.randint(0, model.cfg.d_vocab, (b, n), generator=torch.Generator().manual_seed(seed)).to(model.device)


# ---------------------------------------------------------------------------------------------- CPU
def test_loss_of_a_model_on_the_cpu():
    m = model_of()
    tok = tokens_of(m)
    logits, cache = m.run_with_cache(tok)
    lp = torch.log_softmax((cache["ln_final.hook_normalized"].double() @ m.W_U.double() + m.b_U.double())[:, :-1], -1)
    want = -lp.gather(-1, tok[:, 1:, None])[..., 0]
    got = m(tok, return_type="loss", loss_per_token=True)
    # 48 products and a sum of 301 exponentials, each off by at most its count of additions u; |logit| < 8
    assert got.shape == (3, 8) and (got - want).abs().max() < (2 * 48 * 8 + 301 + 8) * U
    assert torch.equal(m(tok, return_type="loss"), got.mean())
    both, loss = m(tok, return_type="both")
    assert torch.equal(both, logits) and torch.equal(loss, got.mean())
    assert torch.equal(m(tok), logits) and m(tok, return_type=None) is None
    assert torch.equal(m.run_with_hooks(tok, return_type="loss"), got.mean())
    assert m(tok[:, :1], return_type="loss", loss_per_token=True).shape == (3, 0)


def _dictionary_configs(model, layer):
    from types import SimpleNamespace

    d = model.cfg.d_model
    return lambda is_transcoder, hook: SimpleNamespace(
        d_in=d, d_sae=64, l1_coefficient=0.0, dtype=torch.float32, device="cpu", is_transcoder=is_transcoder, d_out=d,
        is_sparse_connection=False, use_ghost_grads=False, hook_point=hook, hook_point_layer=layer)


def test_a_perfect_dictionary_leaves_the_loss(monkeypatch):
    """The reconstruction goes where it belongs: one that is exact changes nothing, zeros are what an ablation gives."""
    from mlp_transcoder import SparseTranscoder
    from z_sae import ZSAE

    m = model_of()
    tok = tokens_of(m)
    clean = m(tok, return_type="loss")
    cfg = _dictionary_configs(m, 1)
    tc = SparseTranscoder(cfg(True, "blocks.1.ln2.hook_normalized"))
    monkeypatch.setattr(tc, "forward", lambda x: (m.blocks[1].mlp(x),))
    got = tc.get_test_loss(tok, m)
    assert abs(float(got - clean)) < 1e-5  # the rows are multiplied as [27, d] here, as [3, 9, d] there
    monkeypatch.setattr(tc, "forward", lambda x: (torch.zeros_like(x),))
    ablated = m.run_with_hooks(tok, return_type="loss", fwd_hooks=[("blocks.1.hook_mlp_out", lambda a, hook: torch.zeros_like(a))])
    assert torch.equal(tc.get_test_loss(tok, m), ablated) and abs(float(ablated - clean)) > 1e-3
    sae = SparseTranscoder(cfg(False, "blocks.0.hook_resid_post"))
    monkeypatch.setattr(sae, "forward", lambda x: (x,))
    assert torch.equal(sae.get_test_loss(tok, m), clean)
    z = ZSAE({"dict_size": 64, "l1_coeff": 1.0, "enc_dtype": "fp32", "seed": 0, "act_size": 48, "device": "cpu"})
    monkeypatch.setattr(z, "forward", lambda x: (None, x))
    assert torch.equal(z.get_test_loss(tok, m, layer=1), clean)
    with pytest.raises(ValueError):
        z.get_test_loss(tok, m)
    monkeypatch.setattr(z, "forward", lambda x: (None, torch.zeros_like(x)))
    z.cfg["layer"] = 0
    ablated = m.run_with_hooks(tok, return_type="loss", fwd_hooks=[("blocks.0.attn.hook_z", lambda a, hook: torch.zeros_like(a))])
    assert torch.equal(z.get_test_loss(tok, m), ablated)
    sae.cfg.hook_point_head_index = 3
    with pytest.raises(NotImplementedError):
        sae.get_test_loss(tok, m)


def test_refusals_on_the_cpu():
    import lm_head
    import tsc_hip

    with pytest.raises(tsc_hip.TscError):
        lm_head.unembed_loss(torch.zeros(2, 4), torch.zeros(2, dtype=torch.long), None, reduction="median")
    with pytest.raises(tsc_hip.TscError):
        lm_head.layer_norm(torch.zeros(2, 4))
    with pytest.raises(tsc_hip.TscError):
        lm_head.layer_norm(torch.zeros(2, 4, requires_grad=True))
    with pytest.raises(tsc_hip.TscError):
        lm_head.model_head(model_of())


@pytest.mark.parametrize("n", [0, 1, 1023, 1024, 1025, 40000, 1024 * 1024 + 1])
def test_total(n):
    import lm_head

    v = torch.arange(n, dtype=torch.float64) % 7
    assert float(lm_head._total(v)) == float(v.sum())


# ---------------------------------------------------------------------------------------------- GPU
def leaves(M, D, V, dtype, tied=False, seed=0, B=2):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (B, M // B), generator=g)
    t[:, 1] = -100
    rnd = lambda *s, scale=1.0, at=0.0: (at + scale * torch.randn(*s, generator=g)).to(dtype).to(DEV).requires_grad_()  # noqa: E731
    x, w, b = rnd(B, M // B, D), rnd(D, scale=0.2, at=1.0), rnd(D, scale=0.1)
    W = rnd(*((V, D) if tied else (D, V)), scale=1 / math.sqrt(D))
    return x, w, b, W, rnd(V, scale=0.3), t.to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_chain_equals_its_calls(dtype, tied):
    """Norm, loss and the backward pass through both, next to the same calls one by one: the same bits, for each reduction
    (whose gradients arrive broadcast) and with gradients of strides that are no rows."""
    import lm_head
    import tsc_hip

    x, w, b, W, bu, t = leaves(34, 72, 501, dtype, tied)
    WU = W.t() if tied else W
    head = tsc_hip.UnembedHead(WU, bu)
    y, mean, scale = tsc_hip.layer_norm(x.detach(), w.detach(), b.detach())
    rows, lse = head.loss(y, t)
    n = int((t != -100).sum())
    coef = torch.randn(t.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    for reduction, dloss in (("none", coef), ("sum", torch.ones_like(rows)), ("mean", torch.ones_like(rows) / torch.tensor(float(n), device=DEV))):
        loss = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head, reduction=reduction)
        got = torch.autograd.grad((loss * coef).sum() if reduction == "none" else loss, (x, w, b, W, bu))
        dy, dW, db = head.loss_backward(dloss, y, t, lse)
        dx, dw, dbias = tsc_hip.layer_norm_backward(dy, x.detach(), mean, scale, w.detach(), b.detach())
        for name, g, ref in zip("x w b W_U b_U".split(), got, (dx, dw, dbias, dW.t() if tied else dW, db)):
            assert g.dtype == dtype and torch.equal(g, ref), (reduction, name)
        if reduction == "none":
            assert torch.equal(loss, rows)
    # only one leaf learns; a transposed and a broadcast gradient of the norm
    y1 = lm_head.layer_norm(x.detach(), w, b.detach())
    dy = torch.randn(x.shape[2], x.shape[1], x.shape[0], generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV).permute(2, 1, 0)
    got = torch.autograd.grad(y1, w, dy)[0]
    assert torch.equal(got, tsc_hip.layer_norm_backward(dy.contiguous(), x.detach(), mean, scale, w.detach())[1])
    one = torch.ones((), dtype=dtype, device=DEV)
    got = torch.autograd.grad(lm_head.layer_norm(x, w), x, one.expand(x.shape))[0]
    assert torch.equal(got, tsc_hip.layer_norm_backward(torch.ones_like(x), x.detach(), mean, scale, w.detach())[0])


@pytest.mark.gpu
def test_chain_against_differences():
    """fp32: the slope of the float64 formula along random directions.  A logit here is a sum of 48 products below 4 in
    size: off by 4 sqrt(3 * 48) u * 48 * 0.2 + 3 * 2^-22 * 10 < 4e-5; so is an exponential, relative; the norm's factors are
    good to (64 + 12) u < 5e-6.  Every term of a gradient passes at most three such factors: 2^-12 of the absolute terms
    covers them."""
    import lm_head
    import tsc_hip

    x, w, b, W, bu, t = leaves(40, 48, 230, torch.float32, seed=5)
    head = tsc_hip.UnembedHead(W, bu)
    got = torch.autograd.grad(lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head), (x, w, b, W, bu))
    args = [q.detach().double().cpu() for q in (x, w, b, W, bu)]
    tc = t.cpu().reshape(-1)

    def f(x, w, b, W, bu):
        y = torch.nn.functional.layer_norm(x, (48,), w, b, 1e-5)
        return torch.nn.functional.cross_entropy(y.reshape(-1, 48) @ W + bu, tc)

    ref = [q.requires_grad_() for q in args]
    exact = torch.autograd.grad(f(*ref), ref)
    for i, (g, e) in enumerate(zip(got, exact)):
        v = torch.randn(g.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        h = 2.0 ** -12
        plus, minus = [[q.detach() + s * h * v if j == i else q.detach() for j, q in enumerate(args)] for s in (1, -1)]
        slope = float(f(*plus) - f(*minus)) / (2 * h)
        size = float((e * v).abs().sum())
        assert abs(float((g.cpu().double() * v).sum()) - slope) <= 2.0 ** -12 * size, i
        assert abs(float((e * v).sum()) - slope) <= 2.0 ** -16 * size, i  # (what the difference itself leaves)


@pytest.mark.gpu
def test_learning_weights_and_changes_between_the_passes():
    import lm_head
    import tsc_hip

    x, w, b, E, bu, t = leaves(24, 40, 333, torch.bfloat16, tied=True, seed=7)
    head = tsc_hip.UnembedHead(E.t(), bu)
    for _ in range(3):
        loss = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head)
        fresh = tsc_hip.UnembedHead(E.detach().clone().t(), bu.detach().clone())
        assert torch.equal(loss, lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, fresh))
        loss.backward()
        with torch.no_grad():
            for p in (x, w, b, E, bu):
                p -= 0.1 * p.grad
                p.grad = None
    loss = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head)
    with torch.no_grad():
        E.mul_(2)
    with pytest.raises(RuntimeError):
        loss.backward()
    loss = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(loss, x, create_graph=True)[0].float().sum(), x)


@pytest.mark.gpu
def test_empty_and_ignored():
    import lm_head
    import tsc_hip

    x, w, b, W, bu, t = leaves(12, 16, 50, torch.float32, seed=9)
    head = tsc_hip.UnembedHead(W, bu)
    none = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), torch.full_like(t, -100), head)
    assert none.isnan()
    total = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), torch.full_like(t, -100), head, reduction="sum")
    assert float(total) == 0 and all(not g.any() for g in torch.autograd.grad(total, (x, w, b, W, bu)))
    xe = x.detach()[:, :0].requires_grad_()
    total = lm_head.unembed_loss(lm_head.layer_norm(xe, w, b), t[:, :0].contiguous(), head, reduction="sum")
    g = torch.autograd.grad(total, (xe, w, b, W, bu))
    assert float(total) == 0 and g[0].shape == xe.shape and all(not q.any() for q in g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_captured_training_step(dtype):
    """Forward, backward and the weights' own step in one graph; replays with eager work between give what eager steps give."""
    import lm_head
    import tsc_hip

    def step(x, ps, t, head):
        loss = lm_head.unembed_loss(lm_head.layer_norm(x, ps[0], ps[1]), t, head)
        grads = torch.autograd.grad(loss, ps)
        with torch.no_grad():
            for p, g in zip(ps, grads):
                p.sub_(g)
        return loss.detach()

    x, *ps, t = leaves(34, 64, 700, dtype, seed=11)
    x = x.detach()
    other = [p.detach().clone().requires_grad_() for p in ps]
    keep = [p.detach().clone() for p in ps]
    head, head2 = tsc_hip.UnembedHead(ps[2], ps[3]), tsc_hip.UnembedHead(other[2], other[3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, ps, t, head)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x, ps, t, head)
    with torch.no_grad():
        for p, k in zip(ps, keep):
            p.copy_(k)
    for _ in range(4):
        g.replay()
        want = step(x, other, t, head2)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(p, q) for p, q in zip(ps, other))


@pytest.mark.gpu
def test_capture_while_an_eager_pass_lives_is_refused():
    import lm_head
    import tsc_hip

    x, w, b, W, bu, t = leaves(12, 16, 50, torch.float32, seed=13)
    head = tsc_hip.UnembedHead(W, bu)
    eager = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head)
    y = lm_head.layer_norm(x, w, b)
    torch.cuda.synchronize()
    static = torch.zeros(2, 6, 16, device=DEV)
    for call in (lambda: lm_head.layer_norm(static, w, b), lambda: lm_head.unembed_loss(static, t, head)):
        g = torch.cuda.CUDAGraph()
        with pytest.raises(tsc_hip.TscError, match="alive"):
            with torch.cuda.graph(g):
                static.add_(0.0)
                call()
    want = float(eager)
    del eager, y
    E = W.detach().t().contiguous().requires_grad_()
    tied = tsc_hip.UnembedHead(E.t(), bu.detach())
    with pytest.raises(tsc_hip.TscError, match="view"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            static.add_(0.0)
            lm_head.unembed_loss(static, t, tied)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head)
        grads = torch.autograd.grad(loss, (x, w, b, W, bu))
    for _ in range(3):
        g.replay()
        eager = torch.autograd.grad(lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head), (x, w, b, W, bu))
        torch.cuda.synchronize()
        assert float(loss) == want and all(torch.equal(p, q) for p, q in zip(grads, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_of_a_model(dtype):
    m = model_of(DEV, dtype=dtype)
    for b, n in ((3, 9), (1, 2), (2, 16)):
        tok = tokens_of(m, b, n)
        logits, cache = m.run_with_cache(tok)
        got = m(tok, return_type="loss", loss_per_token=True)
        x = cache["ln_final.hook_normalized"][:, :-1].reshape(-1, 48)
        want, err = loss_reference(x, m.W_U, m.b_U, tok[:, 1:].reshape(-1), torch.ones(b * (n - 1), device=DEV))["loss"]
        assert got.dtype == torch.float32 and ((got.reshape(-1).double() - want).abs() <= err + U * want.abs()).all()
        both, loss = m(tok, return_type="both")
        assert torch.equal(both, logits) and torch.equal(loss, m(tok, return_type="loss"))
        assert abs(float(loss) - float(want.mean())) <= float(err.mean()) + 16 * U * float(want.mean())
    m2 = copy.deepcopy(m)  # (the head is no part of the model)
    m2.W_U = m2.W_U * 2
    assert not torch.equal(m2(tok, return_type="loss"), loss) and torch.equal(m(tok, return_type="loss"), loss)
    m.b_U.add_(torch.arange(301, device=DEV, dtype=dtype) / 64)  # a change in place is seen
    assert not torch.equal(m(tok, return_type="loss"), loss)


def _world():
    import load_model_and_encoders as lme
    from standins.synthetic_model import SyntheticHookedTransformer

    model = SyntheticHookedTransformer(n_layers=2, d_vocab=1000, n_ctx=32, seed=7, device=DEV)
    lme.install_synthetic(DEV, n_layers=2, d_sae=512, d_vocab=1000, n_ctx=32, model=model)
    return lme.get_model_encoders(DEV)


@pytest.mark.gpu
def test_loss_with_a_dictionary_in_the_model():
    model, z_saes, transcoders = _world()
    tok = tokens_of(model, 4, 20)
    clean = model(tok, return_type="loss")

    def spliced(hooks):
        seen = {}

        def tap(a, hook):
            seen["x"] = a

        model.run_with_hooks(tok, fwd_hooks=hooks + [("ln_final.hook_normalized", tap)])
        want, err = loss_reference(seen["x"][:, :-1].reshape(-1, 768), model.W_U, model.b_U, tok[:, 1:].reshape(-1),
                                   torch.ones(4 * 19, device=DEV))["loss"]
        return float(want.mean()), float(err.mean()) + 16 * U * float(want.mean())

    for layer in (0, 1):
        tc, z, box = transcoders[layer], z_saes[layer], {}

        def read(a, hook):
            box["in"] = a.reshape(-1, 768)

        want, err = spliced([(f"blocks.{layer}.ln2.hook_normalized", read),
                             (f"blocks.{layer}.hook_mlp_out", lambda a, hook: tc(box["in"])[0].reshape(a.shape))])
        got = tc.get_test_loss(tok, model)
        assert got.shape == () and abs(float(got) - want) <= err and not torch.equal(got, clean)
        want, err = spliced([(f"blocks.{layer}.attn.hook_z", lambda a, hook: z(a.reshape(-1, 768))[1].reshape(a.shape))])
        got = z.get_test_loss(tok, model)
        assert abs(float(got) - want) <= err and not torch.equal(got, clean)
    assert torch.equal(model(tok, return_type="loss"), clean)


@pytest.mark.gpu
def test_directions_of_the_answers_loss():
    """Prompts of different lengths: every row at the prompt's own last position, whatever it is padded with."""
    from task_evaluation import TaskEvaluation

    model = _world()[0]
    prompts = [{"text": "when anna and bert went to the shop anna gave milk to", "correct": " bert", "counter": " anna"},
               {"text": "she said", "correct": " no", "counter": " yes"}, {"text": "one two three", "correct": " four", "counter": " six"}]
    te = TaskEvaluation(prompts, None, no_mean_cache=True)
    loss, down, down_resid = te.answer_loss(), te.loss_directions(), te.loss_directions(at="resid")
    assert loss.shape == (3,) and down.shape == down_resid.shape == (3, 768)
    W, b = model.W_U.double(), model.b_U.double()
    for i, p in enumerate(prompts):
        cache = model.run_with_cache(model.to_tokens(p["text"]), names_filter=["blocks.1.hook_resid_post"])[1]
        resid = cache["blocks.1.hook_resid_post"][0, -1].double().requires_grad_()
        tok = model.to_tokens(p["correct"])[0, -1:]
        xh = torch.nn.functional.layer_norm(resid, (768,), eps=1e-5)
        xh.retain_grad()
        want = torch.nn.functional.cross_entropy((xh @ W + b)[None], tok)
        want.backward()
        # the model's own fp32 forward over the padded batch (other products, other order) is good to 1e-4 of a residual's
        # size; the loss and its direction have slopes of order one in it
        assert abs(float(loss[i]) - float(want)) < 1e-3
        assert float((down[i].double() + xh.grad).norm()) < 1e-3 * float(xh.grad.norm())
        assert float((down_resid[i].double() + resid.grad).norm()) < 1e-3 * float(resid.grad.norm())
        pr = torch.softmax(xh.detach() @ W + b, -1)
        assert float((down[i].double() - (W[:, tok[0]] - W @ pr)).norm()) < 1e-3 * float(xh.grad.norm())
    out = te.contribution_decomposition(k=5, directions=down)
    ref = te.batched_lens().direction_lens(down, k=5)
    assert torch.equal(out["top_values"], ref["top_values"]) and out["top_values"].shape == (3, 5)
    same = te.contribution_decomposition(k=5)
    assert torch.equal(same["top_values"], te.batched_lens().direction_lens(te.logit_difference_directions(), k=5)["top_values"])
    with pytest.raises(ValueError):
        te.loss_directions(at="logits")
    with pytest.raises(ValueError):
        TaskEvaluation([{"text": "a b", "correct": None, "counter": " x"}], None, no_mean_cache=True).answer_loss()

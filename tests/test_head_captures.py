"""``UnembedHead`` and ``model_head`` around a capture: what cannot be captured is refused and leaves the capture whole; what is
captured stays valid for as long as the model lives, and a pass captures one layout at most."""
import pytest
import torch

from test_lm_head import leaves, model_of, tokens_of
from test_unembed import DEV, make

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_making_a_head_inside_a_capture_is_refused(dtype):
    import tsc_hip

    x, W, b, t, _ = make(20, 64, 300, dtype, seed=71)
    some = torch.zeros(4, device=DEV)
    for mode in ("global", "relaxed"):
        some.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode=mode):
            some.add_(1)
            with pytest.raises(tsc_hip.TscError, match="capture"):
                tsc_hip.UnembedHead(W, b)
            some.add_(1)
        for k in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert some.eq(2 * (k + 1)).all()
    head = tsc_hip.UnembedHead(W, b)
    assert torch.equal(head.loss(x, t)[0], tsc_hip.UnembedHead(W, b).loss(x, t)[0])


@pytest.mark.gpu
def test_a_head_dropped_inside_a_capture_leaves_it_whole():
    import tsc_hip

    x, W, b, t, _ = make(20, 64, 300, torch.float32, seed=72)
    keep, drop = tsc_hip.UnembedHead(W, b), tsc_hip.UnembedHead(W, b)
    want = keep.loss(x, t)[0]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        first = keep.loss(x, t)[0]
        drop.close()
        second = keep.loss(x, t)[0]
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.gpu
def test_a_model_without_a_head_is_not_captured():
    import tsc_hip

    m = model_of(DEV)
    tok = tokens_of(m)
    final = m.run_with_cache(tok)[1]["ln_final.hook_normalized"].clone()
    import lm_head

    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        final.add_(0.0)
        with pytest.raises(tsc_hip.TscError, match="capture"):
            lm_head.next_token_loss(final, tok, lm_head.model_head(m))
    want = lm_head.next_token_loss(final, tok, lm_head.model_head(m))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = lm_head.next_token_loss(final, tok, lm_head.model_head(m))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_captured_loss_outlives_the_models_tensors():
    """A graph of a model's loss is replayed after the model got other weights (and a head of them): the captured weights, which
    the caller still has, are what it reads, through the layout that was made of them."""
    import lm_head

    m = model_of(DEV)
    tok = tokens_of(m)
    final = m.run_with_cache(tok)[1]["ln_final.hook_normalized"].clone()
    want = lm_head.next_token_loss(final, tok, lm_head.model_head(m)).clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = lm_head.next_token_loss(final, tok, lm_head.model_head(m))
    first = m.W_U
    for k in range(3):
        m.W_U = first * (k + 2.0)
        other = lm_head.next_token_loss(final, tok, lm_head.model_head(m))
        assert len(lm_head._captured[m]) == 1 and lm_head._heads[m][1] not in lm_head._captured[m]
        assert all(h._handle for h in lm_head._captured[m])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and not torch.equal(got, other)
    models = len(lm_head._captured)
    del g
    del m, first
    assert len(lm_head._captured) == models - 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("learning", [True, False])
def test_a_captured_pass_lays_out_once(learning, dtype, monkeypatch):
    """After a change of the weights: of weights that learn the capture takes one layout, of frozen ones the one that their change
    asks for; replays with changes between them give what eager passes give."""
    import lm_head
    import tsc_hip

    x, w, b, W, bu, t = leaves(34, 64, 700, dtype, seed=73)
    if not learning:
        W, bu = W.detach(), bu.detach()
    ps = [w, b] + ([W, bu] if learning else [])
    head = tsc_hip.UnembedHead(W, bu)

    def grads():
        loss = lm_head.unembed_loss(lm_head.layer_norm(x, w, b), t, head)
        return (loss.detach(),) + torch.autograd.grad(loss, [x] + ps)

    def change(k):
        with torch.no_grad():
            W.mul_(k)
            bu.add_(k - 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
        change(1.25)
    torch.cuda.current_stream().wait_stream(side)
    layouts = []
    refresh = tsc_hip.UnembedHead.refresh
    monkeypatch.setattr(tsc_hip.UnembedHead, "refresh", lambda self: (layouts.append(self), refresh(self))[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = grads()
    assert layouts == [head]
    monkeypatch.undo()
    for k in (1.0, 0.75, 1.5):
        change(k)
        g.replay()
        torch.cuda.synchronize()
        kept = [q.clone() for q in got]
        want = grads()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, want)) and all(torch.equal(p, q) for p, q in zip(got, want))

"""``UnembedHead`` and ``model_head`` around a capture: what cannot be captured is refused and leaves the capture whole; what is
captured stays valid for as long as the model lives."""
import pytest
import torch

from test_lm_head import model_of, tokens_of
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

"""What the rounding of the targets' entries of G takes is added to dW as well as to dx (``tsc_unembed_loss_backward``, 16-bit
elements, more than 64 rows).

One entry of a row of G, its target's, is of order one and all others are probabilities: dW's error is the result's own
rounding plus what is lost of the other entries.  The bound is ``test_unembed.reference``'s with the targets' half step taken
out (rows x |G_t| x half a step on column t) and the fp32 evaluation of that part, 4 u of it, put in its place."""
import math

import pytest
import torch

from test_unembed import DEV, U, close, make, reference, run

HALF = [torch.bfloat16, torch.float16]


def want_dW(x, W, b, t, dloss, ignore=-100):
    ref = reference(x, W, b, t, dloss, ignore)
    want, err = ref["dW"]
    live = t != ignore
    half = torch.finfo(x.dtype).eps / 2
    g_t = torch.where(live, dloss.double() * (1.0 - torch.exp(-ref["loss"][0])), 0.0)  # |G_t|
    at = torch.where(live, t, 0)
    taken = torch.zeros(err.shape[1], err.shape[0], dtype=torch.float64, device=err.device)
    taken.index_add_(0, at, torch.where(live[:, None], x.double().abs(), 0.0) * g_t[:, None])
    return want, err - (half - 4 * U) * taken.t()


def check(x, W, b, t, dloss, ignore=-100, **want):
    import tsc_hip

    head = tsc_hip.UnembedHead(W, b)
    _, lse = head.loss(x, t, ignore)
    dW = head.loss_backward(dloss, x, t, lse, ignore, **want)[1]
    close(dW, want_dW(x, W, b, t, dloss, ignore), "dW")
    return dW


# one part and several of the rows' axis, whole tiles of 128 and of 256, a last tile of few entries, widths that end in a vector
SIZES = [(65, 63, 300), (130, 100, 513), (300, 72, 5003), (257, 768, 2049), (200, 1000, 16500), (1500, 513, 700), (2100, 40, 7500)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_weights_gradient(size, tied, dtype):
    check(*make(*size, dtype, tied=tied, bias=not tied, ignored=0.1, seed=sum(size)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tied", [False, True])
def test_tokens_that_many_rows_have(tied, dtype):
    """A token of every row, of every other row, of a run of them, and rows whose target is taken out or unknown."""
    M, D, V = 9001, 72, 333
    for share in (1, 2):
        x, W, b, t, dloss = make(M, D, V, dtype, tied=tied, seed=31 + share)
        t[::share] = 70
        t[4000:4500] = 69
        check(x, W, b, t, dloss)
    t[::3] = -100
    check(x, W, b, t, dloss)
    first = check(x, W, b, t, dloss, want_x=False, want_bias=False)
    assert all(torch.equal(first, check(x, W, b, t, dloss)) for _ in range(2)), "the same call gives the same bits"
    assert not run(x, W, b, torch.full_like(t, -100), dloss)["dW"].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_error_of_the_whole_is_the_results_rounding(dtype):
    """In the 2-norm: a stored value is off by at most half a step, and what is lost of the entries that are no target's, at most
    half a step of each, adds up over the rows without the targets' share."""
    M, D, V = 4096, 128, 8001
    x, W, b, t, dloss = make(M, D, V, dtype, seed=35)
    dW = check(x, W, b, t, dloss).double()
    want = reference(x, W, b, t, dloss)["dW"][0]
    rounded = want.to(dtype).double()
    own = float((rounded - want).norm() / want.norm())
    l = x.double() @ W.double().contiguous() + b.double()
    p = torch.softmax(l, -1)
    p[torch.arange(M, device=DEV), t] = 0.0
    half = torch.finfo(dtype).eps / 2
    others = half * float(torch.sqrt((x.double().square().t().contiguous() @ (p * dloss.double()[:, None]).square()).sum()) / want.norm())
    got = float((dW - want).norm() / want.norm())
    # (the two are independent; 1.05: the second one's terms are taken as uncorrelated, 128 x 8001 of them)
    assert got <= 1.05 * math.hypot(own, others) + 2.0 ** -20, (got, own, others)


@pytest.mark.gpu
def test_workspace_of_more_rows_than_tokens():
    """The sums are kept by token then: a further row costs its 16-bit copy, its row of G and some numbers, not 4 D bytes more."""
    import tsc_hip

    D, V = 512, 300
    head = tsc_hip.UnembedHead(torch.zeros(D, V, dtype=torch.bfloat16, device=DEV))
    size = [tsc_hip.lib().tsc_unembed_workspace_bytes(head._handle, m, 1, 0, 1, 0) for m in (100_000, 200_000)]
    parts = 128 * 4 * D * V  # of a split dW, at most
    assert size[1] - size[0] <= 100_000 * (2 * D + 2 * 512 + 16) + parts < 100_000 * (2 * D + 2 * 512 + 4 * D)

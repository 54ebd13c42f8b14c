"""Rows of fp32 elements without a single element, in a call with others: they hold nothing, so they must not decide how the
gradients of the other rows are held (``tsc_unembed_loss_backward``; a constant row through a layer norm without parameters
is such a row).  The bounds are ``test_unembed.reference``'s: its floor of G, 2^-50 of the largest |dloss| max|x|, knows no
row without elements."""
import pytest
import torch

from test_unembed import DEV, close, make, reference, run


def check(x, W, b, t, dloss, zero):
    got, ref = run(x, W, b, t, dloss), reference(x, W, b, t, dloss)
    full = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    full[zero] = False
    for k in ("loss", "lse"):
        close(got[k], ref[k], k)
    close(got["dW"], ref["dW"], "dW")
    close(got["db"], ref["db"], "db")
    close(got["dx"][full], tuple(q[full] for q in ref["dx"]), "dx")
    if not len(zero):
        return
    # their own gradient: G is held at half the largest |dloss| max|x| at least, so a fixed 2^-48 of |dloss| covers its floor
    want, err = reference(x[zero], W, b, t[zero], dloss[zero])["dx"]
    close(got["dx"][zero], (want, err + 2.0 ** -48 * dloss[zero].double()[:, None] * W.double().abs().sum(1)), "dx of rows without elements")


@pytest.mark.gpu
@pytest.mark.parametrize("M", [40, 96, 300])
def test_rows_without_elements_among_others(M):
    x, W, b, t, dloss = make(M, 64, 1003, torch.float32, seed=41)
    b[500:] -= 12.0  # entries whose probability is small in every row: what a coarser G loses first
    t = t % 500
    check(x, W, b, t, dloss, [])
    for zero in ([3], [0, M - 1], list(range(1, M))):
        x0 = x.clone()
        x0[zero] = 0.0
        check(x0, W, b, t, dloss, zero)
        d = dloss.clone()
        d[zero[0]] *= 1e3
        d[zero[-1]] = 0.0
        check(x0, W, b, t, d, zero)
    small = x * 1e-3
    small[7] = 0.0
    check(small, W, b, t, dloss, [7])


@pytest.mark.gpu
def test_only_rows_without_elements():
    x, W, b, t, dloss = make(70, 64, 1003, torch.float32, seed=42)
    for scale in (1.0, 1e-20, 1e20):
        check(torch.zeros_like(x), W, b, t, dloss * scale, list(range(70)))

"""The gradient of more rows than one piece of the vocabulary holds of G (2 GiB of workspace), in every type and order of W.

Rows are compared a chunk at a time with ``test_unembed.reference``: the losses' gradients are all the same and so is every row's
largest element, so that a chunk's largest |dloss| max|x|, from which the bounds' floors come, is the whole call's."""
import math

import pytest
import torch

from test_unembed import DEV, TYPES, U, close, make, reference

M, CHUNK = 40000, 5000
SIZES = [(24, 60001), (64, 60032)]  # laid out; 16-bit weights that are read where they are


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("D,V", SIZES)
def test_three_pieces_and_more(D, V, tied, dtype):
    import tsc_hip

    x, W, b, t, dloss = make(M, D, V, dtype, tied=tied, ignored=0.05, seed=81 + tied)
    x[:, 0] = 8.0
    dloss.fill_(1.0 / M)
    t[:3] = torch.tensor([0, V - 1, V // 2], device=DEV)
    head = tsc_hip.UnembedHead(W, b)
    planes = 2 if dtype == torch.float32 else 1
    whole = 2 * planes * M * V  # bytes of G
    assert whole > 2 * 2 ** 31 and tsc_hip.lib().tsc_unembed_workspace_bytes(head._handle, M, 1, 1, 1, 1) < whole
    loss, lse = head.loss(x, t)
    dx, dW, db = head.loss_backward(dloss, x, t, lse)
    wd = W.double().contiguous()
    want_W, want_b = [[torch.zeros(s, dtype=torch.float64, device=DEV) for _ in range(2)] for s in ((D, V), (V,))]
    for at in range(0, M, CHUNK):
        c = slice(at, at + CHUNK)
        ref = reference(x[c], W, b, t[c], dloss[c])
        live = t[c] != -100
        close(loss[c], ref["loss"], "loss")
        close(lse[c][live], tuple(q[live] for q in ref["lse"]), "lse")
        close(dx[c], ref["dx"], "dx")
        for total, key in ((want_W, "dW"), (want_b, "db")):
            total[0] += ref[key][0]
            total[1] += ref[key][1]
        # the sums go over all rows and not over a chunk's: 4 sqrt(M) u of the absolute terms
        G = torch.softmax(x[c].double() @ wd + b.double(), -1)
        G[torch.arange(len(live), device=DEV), torch.where(live, t[c], 0)] -= 1.0
        G *= torch.where(live, dloss[c].double(), 0.0)[:, None]
        G.abs_()
        passes = 3 if dtype == torch.float32 else 1
        want_W[1] += 4 * math.sqrt(passes * M) * U * (x[c].double().abs().t().contiguous() @ G)
        want_b[1] += 4 * math.sqrt(M) * U * G.sum(0)
        del G, ref
    close(dW, tuple(want_W), "dW")
    close(db, tuple(want_b), "db")
    # each gradient alone goes through the same pieces
    assert torch.equal(head.loss_backward(dloss, x, t, lse, want_weight=False, want_bias=False)[0], dx)
    assert torch.equal(head.loss_backward(dloss, x, t, lse, want_x=False, want_bias=False)[1], dW)

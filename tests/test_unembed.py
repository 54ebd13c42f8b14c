"""Cross entropy behind the unembedding (``tsc_unembed_*``, ``tsc_hip.UnembedHead``) against its definition in float64.

Tolerances.  u = 2^-24.  A product of split fp32 operands is off by at most 3 * 2^-22 of its size (two residuals, the dropped
product of the second planes), plus 2^-39 of either operand's largest times the other operand; 16-bit operands multiply exactly.  Sums: Higham and Mary's
probabilistic bound 4 sqrt(n) u of the sum of the absolute terms for n additions (a fixed order, so a run repeats itself).
An error e of a logit is a relative error e of its exponential; G is rounded to 16 bits as an operand (bf16 2^-8, fp16 2^-11,
fp32 2^-22 and the floors that the header names; squared where a row's remainder is kept); results are rounded once to their type."""
import ctypes
import math

import pytest
import torch

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(M, D, V, dtype, tied=False, bias=True, ignored=0.0, seed=0, sure=1.0, pitch=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D + (pitch if tied else 0), generator=g)[:, :D] / math.sqrt(D)
    t = torch.randint(0, V, (M,), generator=g)
    x = torch.randn(M, D, generator=g) + sure * w[t]
    if ignored:
        t = torch.where(torch.rand(M, generator=g) < ignored, -100, t)
    b = (0.3 * torch.randn(V, generator=g)).to(dtype).to(DEV) if bias else None
    dloss = ((0.5 + torch.rand(M, generator=g)) / M).to(DEV)
    if tied:
        full = torch.zeros(V, D + pitch, dtype=dtype, device=DEV)
        full[:, :D] = w.to(dtype).to(DEV)
        W = full[:, :D].t()
    else:
        full = torch.zeros(D, V + pitch, dtype=dtype, device=DEV)
        full[:, :V] = w.to(dtype).to(DEV).t()
        W = full[:, :V]
    return x.to(dtype).to(DEV), W, b, t.to(DEV), dloss


def reference(x, W, b, t, dloss, ignore=-100):
    """Values and error bounds, all in float64 on the device."""
    dt = x.dtype
    live = t != ignore
    xd = torch.where(live[:, None], x.double(), 0.0)
    wd = W.double().contiguous()
    M, D = xd.shape
    V = wd.shape[1]
    l = xd @ wd
    mag = xd.abs() @ wd.abs()
    passes = 3 if dt == torch.float32 else 1
    e_l = 4 * math.sqrt(passes * D) * U * mag
    if dt == torch.float32:
        e_l += 3 * 2.0 ** -22 * mag + 2.0 ** -39 * (xd.abs().amax(-1, keepdim=True) * wd.abs().sum(0)
                                                    + xd.abs().sum(-1, keepdim=True) * wd.abs().max())
    if b is not None:
        bd = b.double()
        bd = torch.where(bd < -1e38, -math.inf, bd)
        l = l + bd
    finite = l.isfinite()
    e_l += torch.where(finite, U * l.abs(), 0.0)
    lse = torch.logsumexp(l, -1)
    p = torch.exp(l - lse[:, None])
    e_x = torch.where(finite, e_l + 4 * U * (l - lse[:, None]).abs().clamp_max(150) + 4 * U, 0.0)  # of an exponential
    e_lse = (p * e_x).sum(-1) + 4 * math.sqrt(V) * U + 4 * U * lse.abs()
    at = torch.where(live, t, 0)[:, None]
    hit = l.gather(1, at)[:, 0]
    loss = torch.where(live, lse - hit, 0.0)
    e_loss = torch.where(live, e_lse + e_l.gather(1, at)[:, 0] + 2 * U * (lse.abs() + hit.abs().nan_to_num(0, 0, 0)), 0.0)
    out = {"lse": (lse, e_lse), "loss": (loss, e_loss)}
    g = torch.where(live, dloss.double(), 0.0)[:, None]
    G = p.clone()
    G[torch.arange(M, device=x.device), at[:, 0]] -= 1.0
    e_G = p * (e_x + e_lse[:, None] + 2 * U) + U * G.abs()
    out_G, e_raw = G * g, e_G * g.abs()
    if dt == torch.float32:
        top = (xd.abs().amax(-1, keepdim=True) * g.abs()).max()
        floor = 2.0 ** -50 * 2 * top / xd.abs().amax(-1, keepdim=True).clamp_min(1e-30)  # 2: the row's scale is a power of two
        rnd = 2.0 ** -22 * out_G.abs() + torch.where(g == 0, 0.0, floor)
    else:  # up to 64 rows what the rounding took is kept, rounded itself
        half = 2.0 ** -11 if dt == torch.float16 else 2.0 ** -8
        rnd = half * (half if M <= 64 else 1.0) * out_G.abs() + (2.0 ** -39 * g.abs().max() if dt == torch.float16 else 0.0)
    e_op = e_raw + rnd
    e_dx = e_op  # what the rounding took of the target's entry is added in fp32
    if dt != torch.float32 and M > 64:
        e_dx = e_op.clone()
        e_dx[torch.arange(M, device=x.device), at[:, 0]] = (e_raw + 4 * U * out_G.abs()).gather(1, at)[:, 0]
    passes_rel = 3 * 2.0 ** -22 if dt == torch.float32 else 0.0
    aG, aw = out_G.abs(), wd.abs()
    wt = wd.t().contiguous()
    out["dx"] = (out_G @ wt, e_dx @ aw.t().contiguous() + (4 * math.sqrt(passes * V) * U + passes_rel) * (aG @ aw.t().contiguous())
                 + (2 * 2.0 ** -39 * wd.abs().max() * aG.sum(-1, keepdim=True) if dt == torch.float32 else 0.0))
    xt = xd.t().contiguous()
    # (an element of x is held against its row's largest: 2^-39 of that, twice for its h1 / 2048)
    e_x_ = 2 * 2.0 ** -39 * (xd.abs().amax(-1) @ aG) if dt == torch.float32 else 0.0
    out["dW"] = (xt @ out_G, xt.abs() @ e_op + (4 * math.sqrt(passes * M) * U + passes_rel) * (xt.abs() @ aG) + e_x_)
    out["db"] = (out_G.sum(0), e_raw.sum(0) + 4 * math.sqrt(M) * U * aG.sum(0))
    return out


def close(got, want, what):
    want, err = want
    dt = got.dtype
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bound = err + torch.finfo(dt).eps / 2 * (want.abs() + err) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    d = (got.double() - want).abs()
    bad = ~(d <= bound) & ~((got.double() == want) & want.isinf())
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d / bound).nan_to_num(1e9).max()):.2f} x the bound"


def run(x, W, b, t, dloss, ignore=-100, head=None):
    import tsc_hip

    head = head or tsc_hip.UnembedHead(W, b)
    loss, lse = head.loss(x, t, ignore)
    dx, dW, db = head.loss_backward(dloss, x, t, lse, ignore)
    return {"loss": loss, "lse": lse, "dx": dx, "dW": dW, "db": db}


def check(x, W, b, t, dloss, ignore=-100):
    got = run(x, W, b, t, dloss, ignore)
    want = reference(x, W, b, t, dloss, ignore)
    live = t != ignore
    for k, v in got.items():
        if k == "db" and b is None:
            assert v is None
            continue
        if k in ("lse", "loss"):
            close(v[live], tuple(q[live] for q in want[k]), k)
        else:
            close(v, want[k], k)
    assert got["dW"].stride() == (W.stride() if W.is_contiguous() or W.t().is_contiguous() else got["dW"].stride())
    if not live.all():
        assert not got["loss"][~live].any() and not got["dx"][~live].any()
    return got


SIZES = [(1, 1, 1), (1, 768, 1003), (3, 16, 2), (2, 5, 129), (33, 64, 257), (64, 65, 128), (65, 63, 300), (130, 100, 513), (300, 72, 5003),
         (257, 768, 2049)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    check(*make(*size, dtype, seed=sum(size)))
    check(*make(*size, dtype, tied=True, bias=False, ignored=0.3, seed=sum(size) + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes_of_the_large_tiles(dtype):
    check(*make(2100, 40, 7500, dtype, seed=1))            # logits
    check(*make(16400, 1000, 300, dtype, seed=2))          # dx
    check(*make(200, 1000, 16500, dtype, tied=True, seed=3))  # dW, both orders
    check(*make(200, 1000, 16500, dtype, seed=4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces_of_the_vocabulary(dtype):
    check(*make(16400, 24, 40001, dtype, ignored=0.1, seed=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tied", [False, True])
def test_padded_weights_and_strided_rows(dtype, tied):
    import tsc_hip

    x, W, b, t, dloss = make(6 * 7, 50, 333, dtype, tied=tied, pitch=3, seed=6)
    whole = check(x, W, b, t, dloss)
    head = tsc_hip.UnembedHead(W, b)
    x3, t3, d3 = x.view(6, 7, 50), t.view(6, 7), dloss.view(6, 7)
    for cut in ((slice(None), slice(0, 6)), (slice(None), -1), (slice(1, 6, 2), slice(2, 5))):
        tc, dc = t3[cut].contiguous(), d3[cut].contiguous()
        loss, lse = head.loss(x3[cut], tc)
        assert torch.equal(loss, whole["loss"].view(6, 7)[cut]) and torch.equal(lse, whole["lse"].view(6, 7)[cut])
        dx, _, _ = head.loss_backward(dc, x3[cut], tc, lse, want_weight=False, want_bias=False)
        xc = x3[cut].reshape(-1, 50)
        close(dx.reshape(-1, 50), reference(xc, W, b, tc.reshape(-1), dc.reshape(-1))["dx"], "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_each_gradient_alone(dtype):
    import tsc_hip

    x, W, b, t, dloss = make(90, 48, 700, dtype, seed=7)
    head = tsc_hip.UnembedHead(W, b)
    _, lse = head.loss(x, t)
    every = head.loss_backward(dloss, x, t, lse)
    for i in range(3):
        want = [k == i for k in range(3)]
        got = head.loss_backward(dloss, x, t, lse, want_x=want[0], want_weight=want[1], want_bias=want[2])
        assert all((g is None) if k != i else torch.equal(g, every[k]) for k, g in enumerate(got))
    assert head.loss_backward(dloss, x, t, lse, want_x=False, want_weight=False, want_bias=False) == (None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_taken_out_and_rows_without_a_loss(dtype):
    x, W, b, t, dloss = make(70, 32, 600, dtype, ignored=0.5, seed=8)
    b[100:300] = -math.inf
    if dtype != torch.float16:
        b[400:410] = torch.finfo(dtype).min
    t = torch.where((t >= 100) & (t < 410), 50, t)
    x[t == -100] = math.nan  # padding holds anything
    check(x, W, b, t, dloss)
    got = run(x, W, b, t, dloss)
    assert not got["dW"][:, 100:300].any() and not got["db"][100:300].any()
    # an ignore_index that is a token; every row without a loss
    x, W, b, t, dloss = make(70, 32, 600, dtype, seed=9)
    t[::3] = 7
    check(x, W, b, t, dloss, ignore=7)
    got = run(x, W, b, torch.full_like(t, 7), dloss, 7)
    assert not got["loss"].any() and not got["dx"].any() and not got["dW"].any() and not got["db"].any()
    # no token left
    assert run(x, W, torch.full_like(b, -math.inf), t, dloss)["loss"].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_targets_outside_and_rows_that_are_not_finite(dtype):
    import tsc_hip

    x, W, b, t, dloss = make(40, 32, 300, dtype, seed=10)
    good = run(x, W, b, t, dloss)
    bad_t = t.clone()
    bad_t[3], bad_t[4], bad_t[5] = 300, -1, 2 ** 40
    got = run(x, W, b, bad_t, dloss)
    rest = [i for i in range(40) if i not in (3, 4, 5)]
    assert got["loss"][3:6].isnan().all() and torch.equal(got["loss"][rest], good["loss"][rest])
    assert got["dx"][3:6].isnan().all() and torch.equal(got["dx"][rest], good["dx"][rest])
    x2 = x.clone()
    x2[0, 1], x2[1, 2], x2[2, 3] = math.nan, math.inf, -math.inf
    head = tsc_hip.UnembedHead(W, b)
    loss, lse = head.loss(x2, t)
    assert loss[:3].isnan().all() and torch.equal(loss[3:], good["loss"][3:]) and torch.equal(lse[3:], good["lse"][3:])
    dx = head.loss_backward(dloss, x2, t, lse, want_weight=False)[0]
    assert dx[:3].isnan().all() and dx[3:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sure_rows_large_logits_and_rows_of_many_sizes(dtype):
    x, W, b, t, dloss = make(64, 96, 900, dtype, sure=40.0, seed=11)
    check(x, W, b, t, dloss)
    x, W, b, t, dloss = make(64, 96, 900, dtype, seed=12)
    x = (x.float() * torch.logspace(-4, 2, 64, device=DEV)[:, None]).to(dtype)
    dloss = dloss * torch.logspace(-3, 3, 64, device=DEV).flip(0)
    if dtype == torch.float32:
        W = W * 1e4
        x = x * 1e-5
    check(x, W, b, t, dloss)
    zero = torch.zeros_like(x)
    check(zero, W, b, t, dloss)
    check(x, torch.zeros_like(W), b, t, dloss)
    check(x, W, b, t, torch.zeros_like(dloss))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    import tsc_hip

    x, W, b, t, dloss = make(4, 24, 50, dtype, seed=13)
    head = tsc_hip.UnembedHead(W, b)
    loss, lse = head.loss(x[:0], t[:0])
    dx, dW, db = head.loss_backward(dloss[:0], x[:0], t[:0], lse)
    assert loss.shape == lse.shape == (0,) and dx.shape == (0, 24) and not dW.any() and not db.any()


@pytest.mark.gpu
def test_changed_weights_are_laid_out_again():
    import tsc_hip

    x, W, b, t, dloss = make(50, 64, 400, torch.float32, seed=14)
    head = tsc_hip.UnembedHead(W, b)
    first = run(x, W, b, t, dloss, head=head)
    W.mul_(1.5)
    b.add_(torch.linspace(-1, 1, 400, device=DEV))
    again = run(x, W, b, t, dloss, head=head)
    assert not torch.equal(first["loss"], again["loss"])
    new = run(x, W, b, t, dloss)
    assert all(torch.equal(again[k], new[k]) for k in new)
    with torch.inference_mode():
        Wi, bi = W.clone(), b.clone()
        head = tsc_hip.UnembedHead(Wi, bi)
        Wi.mul_(0.5)
        head.refresh()
        assert torch.equal(head.loss(x, t)[0], tsc_hip.UnembedHead(W * 0.5, b).loss(x, t)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_against_differences(dtype):
    """Central differences of the kernel's own loss along directions in the rows, the weights and the bias; what separates
    them from the slope is the curvature (taken from float64) and the rounding of the two losses."""
    x, W, b, t, dloss = make(30, 40, 200, torch.float32, seed=15)
    x, W, b = (q.to(dtype) for q in (x, W, b))
    got = run(x, W, b, t, dloss)
    h = 2.0 ** -4

    def f(x_, W_, b_):
        import tsc_hip

        loss = tsc_hip.UnembedHead(W_, b_).loss(x_, t)[0]
        return float((loss.double() * dloss.double()).sum())

    def exact(x_, W_, b_):
        return reference(x_, W_, b_, t, dloss)

    for i, k in enumerate(("dx", "dW", "db")):
        v = torch.randn(got[k].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        arg = [x, W, b]
        plus, minus = list(arg), list(arg)
        plus[i], minus[i] = (arg[i].float() + h * v).to(dtype), (arg[i].float() - h * v).to(dtype)
        step = (plus[i].double() - minus[i].double()) / 2
        rp, rm, r0 = exact(*plus), exact(*minus), exact(*arg)
        true = float(((rp["loss"][0] - rm["loss"][0]) * dloss.double()).sum()) / 2
        slope0 = float((r0[k][0] * step).sum())
        slope = float((got[k].double() * step).sum())
        eps = torch.finfo(dtype).eps / 2
        noise = float(((rp["loss"][1] + rm["loss"][1] + 4 * U * rp["loss"][0]) * dloss.double()).sum()) / 2
        slack = float(((r0[k][1] + eps * r0[k][0].abs() + torch.finfo(dtype).smallest_normal * eps) * step.abs()).sum())
        assert abs((f(*plus) - f(*minus)) / 2 - slope) <= abs(true - slope0) + noise + slack, k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_replayed(dtype):
    """Loss and gradients in one graph, replayed over changed inputs with eager work between; a second graph of the same head."""
    import tsc_hip

    sets = [make(130, 64, 900, dtype, ignored=0.2, seed=s) for s in (16, 17)]
    W, b = sets[0][1], sets[0][2]
    head = tsc_hip.UnembedHead(W, b)
    want = [{k: v.clone() for k, v in run(s[0], W, b, s[3], s[4], head=head).items()} for s in sets]
    x, t, d = sets[0][0].clone(), sets[0][3].clone(), sets[0][4].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, W, b, t, d, head=head)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x, W, b, t, d, head=head))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1):
        x.copy_(sets[i][0]), t.copy_(sets[i][3]), d.copy_(sets[i][4])
        graphs[0].replay()
        graphs[1].replay()
        eager = run(*[sets[1 - i][k] for k in (0, 1, 2, 3, 4)], head=head)
        torch.cuda.synchronize()
        for k in want[i]:
            assert torch.equal(outs[0][k], want[i][k]) and torch.equal(outs[1][k], want[i][k]), k
            assert torch.equal(eager[k], want[1 - i][k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_changed_before_a_capture(dtype):
    """The capture lays out nothing by itself: an eager call before the first replay sees the change all the same, and so does
    every replay, also of a change that comes after it."""
    import tsc_hip

    x, W, b, t, _ = make(20, 64, 300, dtype, seed=23)
    head = tsc_hip.UnembedHead(W, b)
    head.loss(x, t)
    W.mul_(1.5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = head.loss(x, t)
    fresh = lambda: tsc_hip.UnembedHead(W.clone(), b).loss(x, t)  # noqa: E731
    assert all(torch.equal(p, q) for p, q in zip(head.loss(x, t), fresh()))
    for k in (1.0, 0.5, 1.25):
        W.mul_(k)
        want = fresh()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        assert all(torch.equal(p, q) for p, q in zip(head.loss(x, t), want))


@pytest.mark.gpu
def test_two_streams_share_a_head():
    import tsc_hip

    sets = [make(100, 64, 2000, torch.bfloat16, seed=s) for s in (18, 19)]
    W, b = sets[0][1], sets[0][2]
    head = tsc_hip.UnembedHead(W, b)
    want = [run(s[0], W, b, s[3], s[4], head=head) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(run(s[0], W, b, s[3], s[4], head=head))
    torch.cuda.synchronize()
    assert all(torch.equal(g[k], w[k]) for g, w in zip(got, want) for k in w)


@pytest.mark.gpu
def test_refusals_on_device():
    import tsc_hip

    x, W, b, t, dloss = make(8, 16, 60, torch.float32, seed=20)
    head = tsc_hip.UnembedHead(W, b)
    _, lse = head.loss(x, t)
    E = tsc_hip.TscError
    for bad in (lambda: tsc_hip.UnembedHead(W.double()), lambda: tsc_hip.UnembedHead(W[0]), lambda: tsc_hip.UnembedHead(W[:, ::2]),
                lambda: tsc_hip.UnembedHead(W[:0]), lambda: tsc_hip.UnembedHead(W, b[:5]), lambda: tsc_hip.UnembedHead(W, b.half()),
                lambda: tsc_hip.UnembedHead(W, b.cpu()), lambda: tsc_hip.UnembedHead(W[:1].expand(16, 60)),
                lambda: head.loss(x.half(), t), lambda: head.loss(x[:, :15], t), lambda: head.loss(x, t.int()),
                lambda: head.loss(x, t[:7]), lambda: head.loss(x.cpu(), t), lambda: head.loss(x, t.cpu()),
                lambda: head.loss(x.t().contiguous().t(), t),
                lambda: head.loss_backward(dloss.double(), x, t, lse), lambda: head.loss_backward(dloss[:3], x, t, lse),
                lambda: head.loss_backward(dloss[:1].expand(8), x, t, lse), lambda: head.loss_backward(dloss, x, t, lse[:2])):
        with pytest.raises(E):
            bad()
    lib = tsc_hip.lib()
    R = tsc_hip._RowsStruct(x.data_ptr(), 1, 16, 16)
    n = lib.tsc_unembed_workspace_bytes(head._handle, 8, 0, 0, 0, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    loss = torch.empty(8, device=DEV)
    call = lambda rows=8, w=ws.data_ptr(), size=n: lib.tsc_unembed_loss(  # noqa: E731
        head._handle, ctypes.byref(R), rows, t.data_ptr(), -100, loss.data_ptr(), lse.data_ptr(), w, size, None)
    assert call(rows=-1) == -1 and call(rows=1 << 24) == -3 and call(w=None) == -1 and call(w=ws.data_ptr() + 8) == -1
    assert call(size=n - 1) == -1 and b"workspace" in lib.tsc_last_error()
    head.close()
    with pytest.raises(E):
        head.loss(x, t)


def test_c_entry_points_refuse_bad_arguments():
    import os

    import tsc_hip

    if not os.path.exists(tsc_hip.library_path()):
        pytest.skip("libtsc_hip.so not built")
    lib = tsc_hip.lib()
    h = ctypes.c_void_p()
    make_ = lambda d=8, v=9, e=0, W=4096, sd=9, sv=1, be=0, b=None: lib.tsc_unembed_create(  # noqa: E731
        ctypes.byref(h), d, v, e, W, sd, sv, b, be, None)
    assert make_(d=0) == -1 and make_(v=-1) == -1 and make_(e=3) == -1 and make_(be=9) == -1 and make_(W=None) == -1
    assert make_(sd=8) == -1 and make_(sd=9, sv=2) == -1 and make_(sd=1, sv=7) == -1 and make_(W=4098) == -1 and make_(b=4097) == -1
    assert make_(d=40000, sd=1 << 40) == -3 and make_(v=(1 << 20) + 1, sd=1 << 40) == -3
    assert lib.tsc_unembed_create(None, 8, 9, 0, 4096, 9, 1, None, 0, None) == -1
    assert lib.tsc_unembed_refresh(None, None) == -1 and lib.tsc_unembed_destroy(None) == 0
    assert lib.tsc_unembed_workspace_bytes(None, 4, 0, 0, 0, 0) == 0
    assert lib.tsc_unembed_loss(None, None, 4, None, 0, None, None, None, 0, None) == -1
    assert lib.tsc_unembed_loss_backward(None, None, None, 4, None, 0, None, None, None, None, None, 0, None) == -1


def test_cpu_tensors_are_refused():
    import tsc_hip

    with pytest.raises(tsc_hip.TscError):
        tsc_hip.UnembedHead(torch.zeros(4, 8))

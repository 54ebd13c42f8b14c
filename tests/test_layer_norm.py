"""Layer norm (``tsc_layer_norm``, ``tsc_layer_norm_backward``) against its definition in float64.

Tolerances count roundings: u = 2^-24 for every fp32 operation, half a step of the type for the stored result.  A sum of n
terms in which every term meets at most K additions is off by at most K u times the sum of the absolute terms; a thread adds
at most 40 elements of a row here and at most 16 further partial sums follow, so K = 64 covers every row sum."""
import ctypes

import pytest
import torch

DEV = "cuda:0"
U = 2.0 ** -24
K = 64
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def reference(x, w, b, eps):
    """Definition in float64, with the bounds of an fp32 evaluation's error."""
    x = x.double()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    scale = (var + eps).sqrt()
    xh = (x - mean) / scale
    y = xh * w + b
    # mean: K u mean|x|; a deviation carries that and its own rounding; the variance is a sum of squares (relative error of
    # K u, and the square of the mean's error); then a root, a reciprocal and two products
    d_mean = K * U * x.abs().mean(-1, keepdim=True)
    r_scale = (K + 8) * U + d_mean.square() / scale.square().clamp_min(1e-300)
    y_err = w.abs() * (d_mean / scale + xh.abs() * (r_scale + 4 * U)) + 2 * U * (y.abs() + b.abs())
    return y, mean[..., 0], scale[..., 0], y_err, d_mean[..., 0], (r_scale * scale)[..., 0]


def reference_backward(dy, x, mean, scale, w, eps_u=U):
    x, dy, mean, scale = x.double(), dy.double(), mean.double()[..., None], scale.double()[..., None]
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    xh = (x - mean) / scale
    dn = dy * w
    dx = (dn - dn.mean(-1, keepdim=True) - xh * (dn * xh).mean(-1, keepdim=True)) / scale
    err = (6 * U * dn.abs() + (K + 6) * U * dn.abs().mean(-1, keepdim=True)
           + xh.abs() * (K + 12) * U * (dn * xh).abs().mean(-1, keepdim=True)) / scale
    rows = x.numel() // D
    # a thread's own rows one after the other (256 workgroups; at the sizes with more than 37 rows here each has two or more
    # groups of threads), at most 128 groups of a workgroup by halves, 256 / 32 and 32 partial sums
    n = (rows + 511) // 512 + 100
    flat = dy.reshape(-1, D), (dy * xh).reshape(-1, D)
    dw, db = flat[1].sum(0), flat[0].sum(0)
    return dx, err, dw, (n + 4) * U * flat[1].abs().sum(0), db, n * U * flat[0].abs().sum(0)


def close(got, want, err, what):
    t = got.dtype
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps  # the smallest subnormal: results below the normal range
    bound = err + half_step(t) * (want.abs() + err) + tiny
    d = (got.cpu().double() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d / bound).nan_to_num(1e9).max()):.2f} x the bound"


def inputs(rows, D, dtype, param, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + offset).to(dtype)
    dy = torch.randn(rows, D, generator=g).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(param) if param else None
    b = (0.2 * torch.randn(D, generator=g)).to(param) if param else None
    return x, dy, w, b


def cu(t):
    return t.to(DEV) if t is not None else None


def check(x, dy, w, b, eps=1e-5, xg=None, dyg=None):
    import tsc_hip

    xg, dyg = cu(x) if xg is None else xg, cu(dy) if dyg is None else dyg
    y, mean, scale = tsc_hip.layer_norm(xg, cu(w), cu(b), eps)
    ry, rm, rs, ey, em, es = reference(x, w, b, eps)
    close(y, ry, ey, "y")
    close(mean, rm, em, "mean")
    close(scale, rs, es, "scale")
    dx, dw, db = tsc_hip.layer_norm_backward(dyg, xg, mean, scale, cu(w), cu(b))
    rdx, edx, rdw, edw, rdb, edb = reference_backward(dy, x, mean.cpu(), scale.cpu(), w)
    close(dx, rdx, edx, "dx")
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    if dw is not None:
        close(dw, rdw, edw, "dweight")
    if db is not None:
        close(db, rdb, edb, "dbias")
    return y, dx, dw, db


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 2, 5, 8, 31, 64, 65, 127, 257, 768, 769, 1000, 2047, 4099, 8200, 40001])
def test_widths(D, dtype):
    for rows, param in ((1, dtype), (37, torch.float32), (3, None)):
        check(*inputs(rows, D, dtype, param, seed=D + rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dtype):
    check(*inputs(4999, 768, dtype, dtype, seed=3))
    check(*inputs(20011, 24, dtype, torch.float32, seed=4))
    check(*inputs(1301, 1001, dtype, dtype, seed=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_one_parameter_only(dtype):
    x, dy, w, b = inputs(70, 96, dtype, dtype, seed=6)
    check(x, dy, w, None)
    check(x, dy, None, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_strides(dtype):
    D = 77
    x, dy, w, b = inputs(6 * 9, D, dtype, dtype, seed=7)
    x3, dy3 = x.view(6, 9, D), dy.view(6, 9, D)
    xg, dyg = x3.to(DEV), dy3.to(DEV)
    whole = check(x3, dy3, w, b)
    for cut in ((slice(None), slice(0, 8)), (slice(None), slice(-1, None)), (slice(1, 5, 2), slice(2, 7)), (slice(None), 3),
                (slice(None), slice(None, None, 3))):
        y, dx, _, _ = check(x3[cut], dy3[cut], w, b, xg=xg[cut], dyg=dyg[cut])
        assert torch.equal(y, whole[0][cut]) and torch.equal(dx, whole[1][cut])
    # an expanded gradient (what sum().backward() passes on) and a base that is aligned to one element only
    ones = torch.ones(1, 1, D, dtype=dtype).expand(6, 9, D)
    check(x3, ones, w, b, dyg=torch.ones(1, 1, D, dtype=dtype, device=DEV).expand(6, 9, D))
    buf = torch.zeros(6 * 9 * D + 3, dtype=dtype, device=DEV)
    odd = buf[3:].view(6, 9, D)
    odd.copy_(xg)
    y, dx, _, _ = check(x3, dy3, w, b, xg=odd)
    assert torch.equal(y, whole[0]) and torch.equal(dx, whole[1])


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0.0, 100.0, 3e4])
def test_rows_far_from_zero(offset):
    """The variance comes from deviations, not from the difference of two large sums."""
    check(*inputs(65, 768, torch.float32, torch.float32, seed=8, offset=offset))


@pytest.mark.gpu
def test_constant_and_extreme_rows():
    import tsc_hip

    x = torch.zeros(5, 64)
    x[1] = 7.0
    x[2] = torch.linspace(-1e18, 1e18, 64)
    x[3, 5] = float("inf")
    x[4, 6] = float("nan")
    y, mean, scale = tsc_hip.layer_norm(x.to(DEV), eps=1e-5)
    assert torch.equal(y[:2].cpu(), torch.zeros(2, 64)) and torch.equal(mean[:2].cpu(), torch.tensor([0.0, 7.0]))
    ry, _, rs, ey, _, es = reference(x[2:3], None, None, 1e-5)
    close(y[2:3], ry, ey, "y")
    close(scale[2:3], rs, es, "scale")
    assert y[3:].isnan().all(), "a row that is not finite has no layer norm"
    dy = torch.ones(5, 64, device=DEV)
    dx, _, _ = tsc_hip.layer_norm_backward(dy, x.to(DEV), mean, scale)
    assert dx[:3].isfinite().all() and dx[3:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    import tsc_hip

    x = torch.empty(0, 3, 10, dtype=dtype, device=DEV)
    w = torch.ones(10, dtype=dtype, device=DEV)
    y, mean, scale = tsc_hip.layer_norm(x, w, w)
    assert y.shape == x.shape and mean.shape == scale.shape == (0, 3)
    dx, dw, db = tsc_hip.layer_norm_backward(x, x, mean, scale, w, w)
    assert dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.gpu
def test_backward_against_differences():
    import tsc_hip

    x, dy, w, b = inputs(33, 130, torch.float32, torch.float32, seed=9)
    v = torch.randn(33, 130, generator=torch.Generator().manual_seed(10))
    h = 2.0 ** -7

    def f(p):
        y = tsc_hip.layer_norm(p.to(DEV), cu(w), cu(b))[0].cpu()
        return float((y.double() * dy.double()).sum())

    def f64(p):
        return float((reference(p, w, b, 1e-5)[0] * dy.double()).sum())

    _, mean, scale = tsc_hip.layer_norm(x.to(DEV), cu(w), cu(b))
    dx, dw, db = tsc_hip.layer_norm_backward(dy.to(DEV), x.to(DEV), mean, scale, cu(w), cu(b))
    plus, minus = x + h * v, x - h * v  # the points that are evaluated are the rounded ones
    step = (plus.double() - minus.double()) / 2
    got = (f(plus) - f(minus)) / 2
    slope = float((dx.cpu().double() * step).sum())
    curve = abs((f64(plus) - f64(minus)) / 2 - float((reference_backward(dy, x, mean.cpu(), scale.cpu(), w)[0] * step).sum()))
    _, _, _, ey, _, _ = reference(x, w, b, 1e-5)
    noise = float((ey * 1.1 * dy.double().abs()).sum() + U * ((reference(x, w, b, 1e-5)[0].abs()) * dy.double().abs()).sum())
    assert abs(got - slope) <= 1.1 * curve + 2 * noise
    # y is linear in the parameters: their gradients are exact differences
    y0 = tsc_hip.layer_norm(x.to(DEV))[0].cpu().double()
    e0 = reference(x, None, None, 1e-5)[3]
    assert ((dw.cpu().double() - (y0 * dy.double()).sum(0)).abs() <= (e0 * dy.double().abs()).sum(0) + 200 * U * (y0 * dy.double()).abs().sum(0)).all()
    assert ((db.cpu().double() - dy.double().sum(0)).abs() <= 200 * U * dy.double().abs().sum(0)).all()


@pytest.mark.gpu
def test_captured_and_replayed_on_another_stream():
    import tsc_hip

    x, dy, w, b = (cu(t) for t in inputs(300, 768, torch.bfloat16, torch.float32, seed=11))
    x2, dy2, _, _ = (cu(t) for t in inputs(300, 768, torch.bfloat16, torch.float32, seed=12))

    def both(xx, dd):
        y, mean, scale = tsc_hip.layer_norm(xx, w, b)
        return (y, mean, scale) + tsc_hip.layer_norm_backward(dd, xx, mean, scale, w, b)

    want = [[t.clone() for t in both(x, dy)], [t.clone() for t in both(x2, dy2)]]
    xs, ds = x.clone(), dy.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(xs, ds)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(xs, ds)
    for i in (0, 1, 0, 1):
        xs.copy_((x, x2)[i])
        ds.copy_((dy, dy2)[i])
        graph.replay()
        eager = both((x, x2)[1 - i], (dy, dy2)[1 - i])  # the program's own work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want[i]))
        assert all(torch.equal(a, c) for a, c in zip(eager, want[1 - i]))


@pytest.mark.gpu
def test_refusals_on_device():
    import tsc_hip

    x = torch.zeros(4, 6, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    y, mean, scale = tsc_hip.layer_norm(x, w)
    E = tsc_hip.TscError
    for bad in (lambda: tsc_hip.layer_norm(x.double()), lambda: tsc_hip.layer_norm(x.transpose(1, 2)),
                lambda: tsc_hip.layer_norm(torch.zeros(4, 4, 4, 4, 8, device=DEV)[::2, ::2, ::2]),
                lambda: tsc_hip.layer_norm(x, w[:7]), lambda: tsc_hip.layer_norm(x, w.half()),
                lambda: tsc_hip.layer_norm(x, w, w.bfloat16()), lambda: tsc_hip.layer_norm(x, w.cpu()),
                lambda: tsc_hip.layer_norm(x, eps=-1.0), lambda: tsc_hip.layer_norm(x[..., :0]),
                lambda: tsc_hip.layer_norm(x, eps=float("nan")), lambda: tsc_hip.layer_norm(torch.zeros((), device=DEV)),
                lambda: tsc_hip.layer_norm_backward(x.half(), x, mean, scale, w),
                lambda: tsc_hip.layer_norm_backward(x[:3], x, mean, scale, w),
                lambda: tsc_hip.layer_norm_backward(x, x, mean[:3], scale, w),
                lambda: tsc_hip.layer_norm_backward(x, x, mean, scale.double(), w)):
        with pytest.raises(E):
            bad()


def test_c_entry_points_refuse_bad_arguments():
    import os

    import tsc_hip

    if not os.path.exists(tsc_hip.library_path()):
        pytest.skip("libtsc_hip.so not built")
    lib = tsc_hip.lib()
    R = tsc_hip._RowsStruct
    ok = R(4096, 1, 8, 8)
    ref = ctypes.byref
    fwd = lambda elem=0, rows=ref(ok), n=4, d=8, pe=0, eps=1e-5, y=4096: lib.tsc_layer_norm(  # noqa: E731
        elem, rows, n, d, None, None, pe, eps, y, 4096, 4096, None)
    assert fwd(elem=3) == -1 and fwd(pe=-1) == -1 and fwd(rows=None) == -1 and fwd(n=-1) == -1 and fwd(d=0) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1 and fwd(y=None) == -1 and fwd(d=1 << 25) == -3
    assert fwd(rows=ref(R(None, 1, 8, 8))) == -1 and fwd(rows=ref(R(4098, 1, 8, 8))) == -1
    assert fwd(rows=ref(R(4096, 0, 8, 8))) == -1 and fwd(rows=ref(R(4096, 1, -8, -8))) == -1
    assert fwd(n=0) == 0, "no rows: nothing is launched"
    need = lib.tsc_layer_norm_workspace_bytes(4, 8)
    assert need == 2 * 4 * 4 * 8 and lib.tsc_layer_norm_workspace_bytes(0, 8) == 0
    bwd = lambda ws=4096, n=need, dx=4096, dy=ref(ok): lib.tsc_layer_norm_backward(  # noqa: E731
        0, dy, ref(ok), 4096, 4096, 4, 8, None, 0, dx, 4096, None, ws, n, None)
    assert bwd(ws=None) == -1 and b"workspace" in lib.tsc_last_error() and bwd(n=need - 1) == -1 and bwd(dx=None) == -1
    assert bwd(dy=None) == -1


def test_cpu_tensors_are_refused():
    import tsc_hip

    with pytest.raises(tsc_hip.TscError):
        tsc_hip.layer_norm(torch.zeros(2, 4))

"""The operators of a language model's head as measurable cases: layer norm (forward, and the backward pass with the
weight's and the bias' gradient) and the cross entropy behind the unembedding without the ``[rows, d_vocab]`` logits
(per-row loss; gradient of the rows alone; the whole training step with the gradients of ``W_U`` and ``b_U``).

``own = False``: elementary torch operations in 32 bits, rounded once at the end.  ``own = True``: the library's calls."""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transcoder-sae-circuits_amd")
_DEV = "cuda:0"
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_IGNORE = -100
_EPS = 1e-5


def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import tsc_hip

    return tsc_hip


# ------------------------------------------------------------------------------------------------ cases
def _norm(name, rows, width, dtype, affine, backward):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "affine": affine, "backward": backward}


def _loss(name, what, rows, width, vocab, dtype, tied, ignored):
    return {"name": name, "op": what, "rows": rows, "width": width, "vocab": vocab, "dtype": dtype, "tied": tied, "ignored": ignored}


def listed():
    return [
        # ln_final at one position of each of 512 prompts, folded weights (no affine part): the smallest call
        _norm("norm 512x768 fp32", 512, 768, "fp32", False, False),
        # one sweep batch (512 sequences x 128 positions) through a layer norm that kept its weights
        _norm("norm 65536x768 bf16", 65536, 768, "bf16", True, False),
        # backward pass of a training batch (128 x 128), with the weight's and the bias' gradient
        _norm("norm grad 16384x768 fp32", 16384, 768, "fp32", True, True),
        # an odd number of rows of an odd width
        _norm("norm grad 1021x4099 bf16", 1021, 4099, "bf16", True, True),
        # the loss of one token: what a loop over single positions pays
        _loss("loss 1x768x50257 fp32", "loss", 1, 768, 50257, "fp32", False, 0.0),
        # the answer's loss of 512 prompts, one position each
        _loss("loss 512x768x50257 fp32", "loss", 512, 768, 50257, "fp32", False, 0.0),
        # the loss of a whole sweep batch, for a model whose dictionary was spliced in: the largest call
        _loss("loss 65536x768x50257 bf16", "loss", 65536, 768, 50257, "bf16", False, 0.0),
        # attribution: the gradient of the residual rows only, 512 prompts
        _loss("grad of rows 512x768x50257 fp32", "rowgrad", 512, 768, 50257, "fp32", False, 0.0),
        # the same for a handful of padded rows and an embedding that is also the unembedding
        _loss("grad of rows 24x768x50257 bf16 tied", "rowgrad", 24, 768, 50257, "bf16", True, 0.25),
        # a training step's head: loss, then the gradients of the rows, of W_U and of b_U
        _loss("step 16384x768x50257 fp32", "step", 16384, 768, 50257, "fp32", False, 0.0),
        _loss("step 16384x768x50257 bf16 tied", "step", 16384, 768, 50257, "bf16", True, 0.01),
        # ragged in every size, a third of the rows padding
        _loss("step 1999x1001x32003 fp16", "step", 1999, 1001, 32003, "fp16", False, 0.33),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if rng.random() < 0.35:
        width = _spread(rng, 8, 8192)
        rows = _spread(rng, 1, min(65536, (65536 * 768) // width))
        c = _norm("", rows, width, dtype, rng.random() < 0.7, rng.random() < 0.5)
    else:
        what = rng.choice(["loss", "rowgrad", "step"])
        width = _spread(rng, 16, 1600)
        vocab = _spread(rng, 2, 131072)
        top = 65536 if what == "loss" else 16384  # rows, work and rows x vocab within the largest listed case's
        most = min(top, top * 50257 // vocab, top * 768 * 50257 // (width * vocab))
        rows = _spread(rng, 1, max(1, most))
        c = _loss("", what, rows, width, vocab, dtype, rng.random() < 0.4, rng.choice([0.0, 0.05, 0.5]))
    del c["name"]
    return c


def work(case):
    b = 4 if case["dtype"] == "fp32" else 2
    m, d = case["rows"], case["width"]
    if case["op"] == "norm":
        stats = 8 * m
        par = d * b if case["affine"] else 0
        if case["backward"]:  # reads dy, x, the statistics, the weight; writes dx, dweight, dbias
            return {"bytes": 3 * m * d * b + stats + 3 * par, "flops": 12 * m * d}
        return {"bytes": 2 * m * d * b + stats + 2 * par, "flops": 7 * m * d}
    v = case["vocab"]
    read = (m * d + d * v + v) * b + 8 * m
    if case["op"] == "loss":
        return {"bytes": read + 8 * m, "flops": 2 * m * d * v}
    if case["op"] == "rowgrad":
        return {"bytes": read + 12 * m + m * d * b, "flops": 4 * m * d * v}
    return {"bytes": read + 12 * m + (m * d + d * v + v) * b, "flops": 6 * m * d * v}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(int(seed))
    dt = _TYPES[case["dtype"]]
    m, d = case["rows"], case["width"]

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=_DEV)

    s = {"case": case}
    if case["op"] == "norm":
        # a residual stream: rows of different lengths around an offset, a few features far above the others
        x = rnd(m, d) * (0.5 + 3.0 * torch.rand(m, 1, generator=g, device=_DEV)) + 0.3 * rnd(m, 1)
        x[:, :: 97] *= 8.0
        s["x"] = x.to(dt)
        s["w"] = (1.0 + 0.2 * rnd(d)).to(dt) if case["affine"] else None
        s["b"] = (0.1 * rnd(d)).to(dt) if case["affine"] else None
        if case["backward"]:
            s["dy"] = (rnd(m, d) / math.sqrt(d)).to(dt)
            xf = s["x"].float()
            mean = xf.mean(-1)
            s["mean"] = mean
            s["scale"] = ((xf - mean[:, None]).square().mean(-1) + _EPS).sqrt()  # what the forward pass kept
        return s
    v = case["vocab"]
    w = rnd(v, d) / math.sqrt(d)
    targets = torch.randint(0, v, (m,), generator=g, device=_DEV)
    # normalised rows; the model is between clueless and fairly sure of the target
    sure = (1.0 + math.log(v)) * torch.rand(m, 1, generator=g, device=_DEV)
    x = rnd(m, d) + sure * w[targets]
    s["x"] = x.to(dt)
    if case["ignored"] > 0:  # padding: no loss, no gradient
        targets = torch.where(torch.rand(m, generator=g, device=_DEV) < case["ignored"], _IGNORE, targets)
    s["targets"] = targets
    w = w.to(dt)
    s["W"] = w.t() if case["tied"] else w.t().contiguous()  # [width, vocab]; tied: the embedding [vocab, width], transposed
    s["b"] = (0.1 * rnd(v)).to(dt)
    if case["op"] != "loss":
        n = max(1, m - int(case["ignored"] * m))
        # a weighted mean over the rows, with the usual scaling of the loss where gradients are fp16
        s["dloss"] = (0.5 + torch.rand(m, generator=g, device=_DEV)) * ((256.0 if dt == torch.float16 else 1.0) / n)
    if own:
        s["head"] = _lib().UnembedHead(s["W"], s["b"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    hip, case = _lib(), s["case"]
    if case["op"] == "norm":
        if case["backward"]:
            dx, dw, db = hip.layer_norm_backward(s["dy"], s["x"], s["mean"], s["scale"], s["w"], bias=s["b"])
            return {"dx": dx, "dw": dw, "db": db} if case["affine"] else {"dx": dx}
        y, mean, scale = hip.layer_norm(s["x"], s["w"], s["b"], eps=_EPS)
        return {"y": y, "mean": mean, "scale": scale}
    head = s["head"]
    if case["op"] == "step":
        head.refresh()  # the last step changed the weights: what the head lays out of them is laid out again
    loss, lse = head.loss(s["x"], s["targets"], ignore_index=_IGNORE)
    if case["op"] == "loss":
        return {"loss": loss, "lse": lse}
    step = case["op"] == "step"
    dx, dw, db = head.loss_backward(s["dloss"], s["x"], s["targets"], lse, ignore_index=_IGNORE, want_weight=step, want_bias=step)
    return {"loss": loss, "dx": dx, "dW": dw, "db": db} if step else {"loss": loss, "dx": dx}


def _run_plain(s):
    case = s["case"]
    dt = _TYPES[case["dtype"]]
    x = s["x"].float()
    if case["op"] == "norm":
        if case["backward"]:
            xhat = (x - s["mean"][:, None]) / s["scale"][:, None]
            dy = s["dy"].float()
            dn = dy * s["w"].float() if case["affine"] else dy
            dx = (dn - dn.mean(-1, keepdim=True) - xhat * (dn * xhat).mean(-1, keepdim=True)) / s["scale"][:, None]
            out = {"dx": dx.to(dt)}
            if case["affine"]:
                out["dw"], out["db"] = (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)
            return out
        mean = x.mean(-1)
        c = x - mean[:, None]
        scale = (c.square().mean(-1) + _EPS).sqrt()
        y = c / scale[:, None]
        if case["affine"]:
            y = y * s["w"].float() + s["b"].float()
        return {"y": y.to(dt), "mean": mean, "scale": scale}
    w = s["W"].float()
    logits = x @ w
    logits += s["b"].float()
    top = logits.amax(-1, keepdim=True)
    targets, live = s["targets"], s["targets"] != _IGNORE
    at = torch.where(live, targets, 0)[:, None]
    hit = logits.gather(1, at)[:, 0]
    logits -= top
    logits.exp_()
    total = logits.sum(-1, keepdim=True)
    lse = (top + total.log())[:, 0]
    loss = torch.where(live, lse - hit, 0.0)
    if case["op"] == "loss":
        return {"loss": loss, "lse": lse}
    logits /= total
    logits.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    logits *= torch.where(live, s["dloss"], 0.0)[:, None]
    out = {"loss": loss, "dx": (logits @ w.t()).to(dt)}
    if case["op"] == "step":
        dw = logits.t() @ x
        out["dW"] = (dw.to(dt).t() if case["tied"] else dw.t().to(dt))
        out["db"] = logits.sum(0).to(dt)
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """From the definitions, in float64: torch's own layer norm and log-softmax with their derivatives by autograd."""
    s = prepare({**case}, seed)
    x = s["x"].double()
    if case["op"] == "norm":
        w = s["w"].double() if case["affine"] else None
        b = s["b"].double() if case["affine"] else None
        norm = torch.nn.functional.layer_norm
        if not case["backward"]:
            var, mean = torch.var_mean(x, dim=-1, unbiased=False)
            return {"y": norm(x, (case["width"],), w, b, _EPS), "mean": mean, "scale": (var + _EPS).sqrt()}
        leaves = [x.requires_grad_()] + ([w.requires_grad_(), b.requires_grad_()] if case["affine"] else [])
        grads = torch.autograd.grad(norm(x, (case["width"],), w, b, _EPS), leaves, s["dy"].double())
        return dict(zip(("dx", "dw", "db"), grads))
    w, b = s["W"].double(), s["b"].double()
    live = s["targets"] != _IGNORE
    targets = torch.where(live, s["targets"], 0)
    rows = max(1, min(x.shape[0], (1 << 28) // case["vocab"]))
    parts, dw, db = [], torch.zeros_like(w), torch.zeros_like(b)
    for at in range(0, x.shape[0], rows):
        xs, ts, lv = x[at: at + rows], targets[at: at + rows], live[at: at + rows]
        logits = torch.addmm(b, xs, w)
        lse = torch.logsumexp(logits, -1)
        loss = torch.where(lv, torch.nn.functional.nll_loss(torch.log_softmax(logits, -1), ts, reduction="none"), 0.0)
        part = {"loss": loss, "lse": lse}
        if case["op"] != "loss":
            p = torch.softmax(logits, -1)
            p[torch.arange(len(ts), device=_DEV), ts] -= 1.0
            p = p * torch.where(lv, s["dloss"][at: at + rows].double(), 0.0)[:, None]
            part["dx"] = torch.mm(p, w.t().contiguous())
            if case["op"] == "step":
                dw += torch.mm(xs.t().contiguous(), p)
                db += p.sum(0)
        parts.append(part)
    out = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
    if case["op"] != "loss":
        del out["lse"]
    if case["op"] == "step":
        out["dW"], out["db"] = dw, db
    return out

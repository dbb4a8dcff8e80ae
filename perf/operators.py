"""The calls that train what stands in front of the experts -- the norm of the
MoE input and the router -- and what their speed is measured on.

Five operators:

  norm         residual add + layer norm (or RMS norm), forward
  norm_grad    its gradients: the input's, with the residual stream's own
               gradient added, and the sums over tokens for weight and bias
  balance      per-expert counts, summed probabilities and the balance loss
  topk_grad    the router logits' gradient, from the routing weights' and
               from the balance loss's
  router_grad  the router product's gradients: of its rows and of its input

`run` computes them in plain torch in 32 bits, or, with `own` set, through
q36_amd.moe.
"""
import math

import torch

own = False

D, E, K = 2048, 256, 8      # the q36 layer: width, experts, picks
EPS = 1e-6
COEF = 1e-3                 # weight of the balance loss
GRAD = 1e-3                 # size of the gradients that come from above


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decoded token, residual in fp32, the norm's output in half the bits
        {"name": "norm1", "kind": "norm", "T": 1, "D": D, "x": "f32", "y": "bf16", "rms": True, "add": True, "pad": 0},
        # a packed batch of prompts and decoding sequences of a model kept in bf16
        {"name": "norm4006_bf16", "kind": "norm", "T": 4006, "D": D, "x": "bf16", "y": "bf16", "rms": False, "add": True, "pad": 0},
        # a short sequence of the framework's own norm
        {"name": "norm_grad61", "kind": "norm_grad", "T": 61, "D": D, "x": "f32", "y": "f32", "rms": True, "add": True, "pad": 0},
        # an odd width in the left part of wider rows
        {"name": "norm_grad1000_odd", "kind": "norm_grad", "T": 1000, "D": 1531, "x": "f32", "y": "bf16", "rms": False, "add": False, "pad": 5},
        # the micro-batch of a wider model, residual in fp32
        {"name": "norm_grad16384", "kind": "norm_grad", "T": 16384, "D": 4096, "x": "f32", "y": "bf16", "rms": False, "add": True, "pad": 0},
        # the load of one small batch
        {"name": "balance203", "kind": "balance", "T": 203, "E": E, "k": K, "mask": False},
        # a micro-batch of padded sequences
        {"name": "balance32768", "kind": "balance", "T": 32768, "E": E, "k": K, "mask": True},
        # a layer that learns from the routing weights alone
        {"name": "topk_grad64", "kind": "topk_grad", "T": 64, "E": E, "k": K, "mask": False, "balance": False, "renorm": True},
        # both gradients of a padded micro-batch
        {"name": "topk_grad16384", "kind": "topk_grad", "T": 16384, "E": E, "k": K, "mask": True, "balance": True, "renorm": True},
        # a ragged batch of the router with its shared-expert row
        {"name": "router_grad203", "kind": "router_grad", "T": 203, "E": E, "shared": True, "x": "f32"},
        # a prompt's worth of tokens, fp32 activations
        {"name": "router_grad4096", "kind": "router_grad", "T": 4096, "E": E, "shared": True, "x": "f32"},
        # a micro-batch of bf16 activations, no shared expert
        {"name": "router_grad16384_bf16", "kind": "router_grad", "T": 16384, "E": E, "shared": False, "x": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "balance", "topk_grad", "router_grad"])
    c = {"kind": kind}
    if kind in ("norm", "norm_grad"):
        c["D"] = rng.choice([D, _spread(rng, 16, 8192)])
        c["T"] = _spread(rng, 1, min(32768, 16384 * 4096 // c["D"]))
        c |= {"x": rng.choice(["f32", "bf16"]), "y": rng.choice(["f32", "bf16"]), "rms": rng.choice([True, False]),
              "add": rng.choice([True, False]), "pad": rng.choice([0, 0, rng.randint(1, 64)])}
    elif kind == "balance":
        e = rng.choice([E, _spread(rng, 8, E)])
        c |= {"T": _spread(rng, 1, 32768), "E": e, "k": rng.randint(1, 8), "mask": rng.choice([True, False])}
    elif kind == "topk_grad":
        e = rng.choice([E, _spread(rng, 8, E)])
        c |= {"T": _spread(rng, 1, 32768), "E": e, "k": rng.randint(1, 8), "mask": rng.choice([True, False]),
              "balance": rng.choice([True, False]), "renorm": rng.choice([True, True, False])}
    else:
        c |= {"T": _spread(rng, 1, 16384), "E": rng.choice([E, _spread(rng, 8, E)]), "shared": rng.choice([True, False]),
              "x": rng.choice(["f32", "bf16"])}
    return c


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(g, T, n, pad, dtype, size=1.0, offset=None):
    """[T, n] normal values, the left part of rows of n + pad."""
    v = _normal(g, T, n + pad)
    v *= size
    if offset is not None:
        v += offset
    return v.to(dtype)[:, :n]


def _logits(g, T, e):
    """Router logits of a trained layer: per-token noise on a popularity of each expert's own."""
    return _normal(g, T, e) + 0.7 * _normal(g, e)


def _mask(g, T, on):
    """The last eighth or so of the tokens is padding."""
    if not on:
        return None
    n = T - int(T * 0.25 * float(torch.rand(1, generator=g, device="cuda")))
    return (torch.arange(T, device="cuda") < n).to(torch.uint8)


def _counts(idx, mask, e):
    """int32 [e + 1]: picks of each expert over the live tokens, and the number of those."""
    live = torch.ones(idx.shape[0], device="cuda", dtype=torch.int64) if mask is None else (mask != 0).long()
    c = torch.zeros(e + 1, device="cuda", dtype=torch.int64)
    c.scatter_add_(0, idx.long().reshape(-1), live[:, None].expand(idx.shape).reshape(-1))
    c[e] = live.sum()
    return c.int()


def prepare(case, seed):
    g = _gen(seed, 1)
    T, kind = case["T"], case["kind"]
    s = {"case": case}
    if kind in ("norm", "norm_grad"):
        n, pad, xt, yt = case["D"], case["pad"], _TYPE[case["x"]], _TYPE[case["y"]]
        # a residual stream: one size per channel, an offset that a layer norm takes out
        size = torch.exp(0.5 * _normal(g, n + pad))
        x = _rows(g, T, n, pad, xt, size, 0.3)
        s["w"] = 1 + 0.1 * _normal(g, n)
        if kind == "norm":
            s |= {"x": x, "a": _rows(g, T, n, pad, xt, 0.5) if case["add"] else None}
            s["b"] = None if case["rms"] else 0.1 * _normal(g, n)
        else:
            s |= {"h": x, "dy": _rows(g, T, n, pad, yt, GRAD), "dres": _rows(g, T, n, pad, xt, GRAD) if case["add"] else None}
    elif kind == "router_grad":
        rows = case["E"] + int(case["shared"])
        s["w"] = _normal(g, rows, D) / math.sqrt(D)
        s["x"] = _normal(g, T, D).to(_TYPE[case["x"]])
        s["dlogits"] = GRAD * _normal(g, T, case["E"])
        s["dshg"] = GRAD * _normal(g, T) if case["shared"] else None
    else:
        s["logits"] = _logits(g, T, case["E"])
        s["idx"] = torch.topk(s["logits"], case["k"], dim=1).indices.int()
        s["mask"] = _mask(g, T, case["mask"])
        if kind == "topk_grad":
            s["dwt"] = GRAD * _normal(g, T, case["k"])
            s["counts"] = _counts(s["idx"], s["mask"], case["E"]) if case["balance"] else None
            s["dloss"] = torch.rand((), generator=g, device="cuda") + 0.5 if case["balance"] else None
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"norm": _norm, "norm_grad": _norm_grad, "balance": _balance, "topk_grad": _topk_grad,
            "router_grad": _router_grad}[case["kind"]](s, case)


def _own(s, case):
    from q36_amd import moe
    kind = case["kind"]
    if kind == "norm":
        y, h = moe.layernorm(s["x"], s["w"], s["b"], a=s["a"], eps=EPS, rms=case["rms"], out_dtype=_TYPE[case["y"]])
        return {"y": y, "h": h}
    if kind == "norm_grad":
        dx, dw, db = moe.layernorm_backward(s["dy"], s["h"], s["w"], dres=s["dres"], eps=EPS, rms=case["rms"])
        return {"dx": dx, "dw": dw, "db": db}
    if kind == "balance":
        loss, counts, psum = moe.balance_loss(s["logits"], s["idx"], coef=COEF, mask=s["mask"])
        return {"loss": loss, "counts": counts, "psum": psum}
    if kind == "topk_grad":
        return moe.router_topk_backward(s["logits"], s["idx"], s["dwt"], renorm=case["renorm"], counts=s["counts"], coef=COEF,
                                        mask=s["mask"], dloss=s["dloss"])
    dw, dx = moe.router_logits_backward(s["w"], s["x"], case["E"], s["dlogits"], s["dshg"])
    return {"dw": dw, "dx": dx}


def _stats(v, rms):
    """Rows less their mean (a layer norm's), and one over their deviation."""
    if not rms:
        v = v - v.mean(1, keepdim=True)
    return v, (v.square().mean(1, keepdim=True) + EPS).rsqrt()


def _norm(s, case):
    v = s["x"].float()
    if s["a"] is not None:
        v = v + s["a"].float()
    h = v.to(s["x"].dtype) if s["a"] is not None else None
    v, r = _stats(v, case["rms"])
    y = v * r * s["w"]
    if s["b"] is not None:
        y = y + s["b"]
    return {"y": y.to(_TYPE[case["y"]]), "h": h}


def _norm_grad(s, case):
    v, r = _stats(s["h"].float(), case["rms"])
    n, dy = v * r, s["dy"].float()
    dw = (dy * n).sum(0)
    g = dy * s["w"]
    dx = g - n * (g * n).mean(1, keepdim=True)
    if not case["rms"]:
        dx = dx - g.mean(1, keepdim=True)
    dx = dx * r
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(s["h"].dtype), "dw": dw, "db": None if case["rms"] else dy.sum(0)}


def _probs(logits):
    e = (logits - logits.amax(1, keepdim=True)).exp()
    return e / e.sum(1, keepdim=True)


def _balance(s, case):
    e, k = case["E"], case["k"]
    counts = _counts(s["idx"], s["mask"], e)
    p = _probs(s["logits"])
    if s["mask"] is not None:
        p = p * s["mask"][:, None]
    psum = p.sum(0)
    n = counts[e].float()
    loss = COEF * e / k * (counts[:e] / n * (psum / n)).sum()
    return {"loss": loss, "counts": counts, "psum": psum}


def _topk_grad(s, case):
    e, k, logits, idx = case["E"], case["k"], s["logits"], s["idx"].long()
    if case["renorm"]:
        wt = _probs(logits.gather(1, idx))
        picks = wt * (s["dwt"] - (wt * s["dwt"]).sum(1, keepdim=True))
        d = torch.zeros_like(logits).scatter_add_(1, idx, picks)
    else:
        p = _probs(logits)
        up = torch.zeros_like(logits).scatter_add_(1, idx, s["dwt"])
        d = p * (up - (p * up).sum(1, keepdim=True))
    if s["counts"] is not None:
        p, n = _probs(logits), s["counts"][e].float()
        f = s["counts"][:e] / (n * k)
        d = d + (s["dloss"] * COEF * e / n) * p * (f - (p * f).sum(1, keepdim=True))
    if s["mask"] is not None:
        d = d * s["mask"][:, None]
    return d


def _router_grad(s, case):
    d = s["dlogits"] if s["dshg"] is None else torch.cat([s["dlogits"], s["dshg"][:, None]], 1)
    return {"dw": d.T @ s["x"].float(), "dx": (d @ s["w"]).to(s["x"].dtype)}


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    T, kind = case["T"], case["kind"]
    if kind in ("norm", "norm_grad"):
        n = case["D"]
        xb, yb = (2 if case[c] == "bf16" else 4 for c in "xy")
        if kind == "norm":      # x in and y out; the addend in and the sum out; weight and bias
            return {"bytes": T * n * (xb * (3 if case["add"] else 1) + yb) + n * (4 if case["rms"] else 8), "flops": 8 * T * n}
        # h and dy in and dx out; the residual's gradient; weight in, its and the bias's gradient out
        return {"bytes": T * n * (xb * (3 if case["add"] else 2) + yb) + n * (8 if case["rms"] else 12), "flops": 16 * T * n}
    e = case["E"]
    if kind == "router_grad":
        rows = e + int(case["shared"])
        xb = 2 if case["x"] == "bf16" else 4
        # rows, x and the logits' gradient in, both gradients out
        return {"bytes": 2 * (rows * D * 4 + T * D * xb) + T * rows * 4, "flops": 4 * T * rows * D}
    k, m = case["k"], int(case["mask"])
    if kind == "balance":
        return {"bytes": T * (4 * e + 4 * k + m) + 8 * e + 8, "flops": 5 * T * e}
    return {"bytes": T * (8 * e + 8 * k + m) + (4 * e + 8 if case["balance"] else 0), "flops": (10 if case["balance"] else 2) * T * e}


# --------------------------------------------------------------------------
# the same in 64 bits, from the operators' definitions: what a gradient is of
# stands as a formula, and is differentiated
# --------------------------------------------------------------------------
def _normalise(h, w, b, rms):
    d = h if rms else h - h.sum(1, keepdim=True) / h.shape[1]
    y = d / torch.sqrt((d * d).sum(1, keepdim=True) / h.shape[1] + EPS) * w
    return y if b is None else y + b


def _balance_of(logits, idx, mask, e, k):
    """Loss, and the sum of the live tokens' probabilities."""
    live = torch.ones(logits.shape[0], 1, device="cuda", dtype=torch.float64) if mask is None else mask[:, None].double()
    psum = (torch.softmax(logits, 1) * live).sum(0)
    picked = (torch.nn.functional.one_hot(idx.long(), e).sum(1) * live).sum(0)
    return COEF * e * ((picked / (live.sum() * k)) * (psum / live.sum())).sum(), psum


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h = s["x"].double() + (s["a"].double() if s["a"] is not None else 0)
        b = None if s["b"] is None else s["b"].double()
        return {"y": _normalise(h, s["w"].double(), b, case["rms"]), "h": h if s["a"] is not None else None}
    if kind == "norm_grad":
        h, w = s["h"].double().requires_grad_(), s["w"].double().requires_grad_()
        b = None if case["rms"] else torch.zeros_like(w).requires_grad_()
        got = torch.autograd.grad(_normalise(h, w, b, case["rms"]), [h, w] + ([] if b is None else [b]), s["dy"].double())
        dx = got[0] + (s["dres"].double() if s["dres"] is not None else 0)
        return {"dx": dx, "dw": got[1], "db": None if b is None else got[2]}
    if kind == "balance":
        loss, psum = _balance_of(s["logits"].double(), s["idx"], s["mask"], case["E"], case["k"])
        return {"loss": loss, "counts": None, "psum": psum}
    if kind == "topk_grad":
        logits, live = s["logits"].double().requires_grad_(), 1 if s["mask"] is None else s["mask"][:, None].double()
        wt = torch.softmax(logits, 1).gather(1, s["idx"].long())
        if case["renorm"]:
            wt = wt / wt.sum(1, keepdim=True)
        of = (wt * s["dwt"].double() * live).sum()
        if s["counts"] is not None:
            of = of + s["dloss"].double() * _balance_of(logits, s["idx"], s["mask"], case["E"], case["k"])[0]
        return torch.autograd.grad(of, logits)[0]
    w, x = s["w"].double().requires_grad_(), s["x"].double().requires_grad_()
    up = s["dlogits"].double() if s["dshg"] is None else torch.cat([s["dlogits"], s["dshg"][:, None]], 1).double()
    dw, dx = torch.autograd.grad(x @ w.T, [w, x], up)
    return {"dw": dw, "dx": dx}

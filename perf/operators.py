"""Cases of the training-step operators next to the FP8 linears: the
root-mean-square norm with the residual's addition and an FP8 output, the
softmax cross entropy of an output projection, and the global gradient norm
with clipping.

``run`` computes a case in its plain form (elementary torch operations in
fp32) or, with ``own`` set, through this package's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
_NORM_EPS = 1e-5
_QUANT_EPS = 1e-12
_CLIP_EPS = 1e-6
_IGNORE = -100


# ------------------------------------------------------------------- cases ---
def _norm_fwd(rows, dim, dtype, quant="block", fp8="e4m3", residual=True, keep=True):
    # keep: the normalised rows are wanted in the input's type too (a training
    # step quantizes them again along the tokens for the weight gradient).
    return {"op": "norm_fwd", "rows": rows, "dim": dim, "dtype": dtype, "quant": quant, "fp8": fp8,
            "residual": residual, "keep": keep}


def _norm_bwd(rows, dim, dtype, wdtype, residual=True):
    return {"op": "norm_bwd", "rows": rows, "dim": dim, "dtype": dtype, "wdtype": wdtype, "residual": residual}


def _loss(tokens, vocab, dim, dtype, reduction="mean", train=True, ignored=0.0):
    return {"op": "loss", "tokens": tokens, "vocab": vocab, "dim": dim, "dtype": dtype, "reduction": reduction,
            "train": train, "ignored": ignored}


def _clip(layers, dim, ffn, vocab, dtype, odd=0):
    # The gradients of a decoder of these sizes; odd: elements added to every
    # tensor, so that none starts on a 16-byte boundary but the first.
    return {"op": "clip", "layers": layers, "dim": dim, "ffn": ffn, "vocab": vocab, "dtype": dtype, "odd": odd}


def listed():
    named = {
        # One token through a decoder layer's norm while serving: latency.
        "norm_fwd one token": _norm_fwd(1, 4096, "bf16", keep=False),
        # The norm before the projections of a training step, 16384 tokens.
        "norm_fwd train 16384x4096": _norm_fwd(16384, 4096, "bf16"),
        # A per-row FP8 scale and a ragged number of tokens, no residual.
        "norm_fwd rows 2049x7168": _norm_fwd(2049, 7168, "fp16", quant="row", residual=False, keep=False),
        # Its backward pass in the training step.
        "norm_bwd train 16384x4096": _norm_bwd(16384, 4096, "bf16", "bf16"),
        # The backward pass of a small fp32 model with a width that is not a power of two.
        "norm_bwd fp32 513x1000": _norm_bwd(513, 1000, "fp32", "fp32", residual=False),
        # Scoring a few tokens: the projection's weights are read once.
        "loss score 8 tokens": _loss(8, 32000, 4096, "bf16", reduction="none", train=False),
        # Evaluating a sequence: the loss alone.
        "loss eval 4096 tokens": _loss(4096, 32000, 4096, "bf16", train=False),
        # The training step's loss with both gradients.
        "loss train 4096 tokens": _loss(4096, 32000, 4096, "bf16"),
        # A ragged batch with prompt tokens left out, weighted token by token.
        "loss train ragged": _loss(1021, 50001, 2056, "fp16", reduction="none", ignored=0.3),
        # A small model's gradients: many small tensors, latency.
        "clip small model": _clip(2, 128, 352, 1000, "fp32"),
        # Tensors whose sizes are odd.
        "clip odd sizes": _clip(6, 1024, 2816, 8000, "bf16", odd=3),
        # The 8-layer decoder's gradients, about two billion values.
        "clip 8-layer decoder": _clip(8, 4096, 14336, 32000, "bf16"),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "loss", "loss", "clip"])
    if op in ("norm_fwd", "norm_bwd"):
        dim = _log_int(rng, 64, 16384)
        if rng.random() < 0.7:
            dim = max(64, dim // 8 * 8)
        rows = _log_int(rng, 1, min(16384, 16384 * 4096 // dim))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if op == "norm_bwd":
            return _norm_bwd(rows, dim, dtype, rng.choice([dtype, "fp32"]), residual=rng.random() < 0.7)
        return _norm_fwd(rows, dim, dtype, quant=rng.choice(["block", "block", "row"]),
                         fp8=rng.choice(["e4m3", "e4m3", "e5m2"]), residual=rng.random() < 0.7,
                         keep=rng.random() < 0.5)
    if op == "loss":
        dim = _log_int(rng, 128, 4096)
        if rng.random() < 0.75:
            dim = max(128, dim // 8 * 8)
        return _loss(_log_int(rng, 1, 4096), _log_int(rng, 500, 32000), dim, rng.choice(["bf16", "bf16", "fp16"]),
                     reduction=rng.choice(["mean", "sum", "none"]), train=rng.random() < 0.6,
                     ignored=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.6), 2)]))
    dim = _log_int(rng, 64, 4096)
    return _clip(rng.randint(1, 6), dim, int(dim * rng.uniform(2.0, 3.5)), _log_int(rng, 256, 32000),
                 rng.choice(["bf16", "fp16", "fp32"]), odd=rng.choice([0, 0, rng.randint(1, 7)]))


def _clip_sizes(case):
    d, f, odd = case["dim"], case["ffn"], case["odd"]
    # Query and key, value and output projections are held fused here: seven
    # tensors a layer.
    layer = [d, 2 * d * d, 2 * d * d, d, d * f, d * f, f * d]
    sizes = [case["vocab"] * d] + layer * case["layers"] + [d, case["vocab"] * d]
    return [n + odd for n in sizes]


# ------------------------------------------------------------------ inputs ---
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, dim):
    # N(0, 1) with one value in a thousand a hundred times larger, as hidden states have.
    x = _normal(g, rows, dim)
    outlier = torch.rand((rows, dim), generator=g, device="cuda") < 1e-3
    return torch.where(outlier, 100.0 * x, x)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "clip":
        sizes = _clip_sizes(case)
        dtype = _DTYPES[case["dtype"]]
        total = sum(sizes)
        flat = torch.empty(total, device="cuda", dtype=dtype)
        flat.normal_(0.0, 1e-3, generator=g)
        out = torch.empty_like(flat)
        max_norm = 0.3 * 1e-3 * math.sqrt(total)  # about 0.3 of the norm: the gradients are clipped
        return {"case": case, "flat": flat, "grads": list(flat.split(sizes)), "out_flat": out,
                "out": list(out.split(sizes)), "max_norm": max_norm}
    dtype = _DTYPES[case["dtype"]]
    if op == "norm_fwd":
        rows, dim = case["rows"], case["dim"]
        return {"case": case, "x": _activations(g, rows, dim).to(dtype),
                "residual": _activations(g, rows, dim).to(dtype) if case["residual"] else None,
                "weight": (1.0 + 0.1 * _normal(g, dim)).to(dtype)}
    if op == "norm_bwd":
        rows, dim = case["rows"], case["dim"]
        h = _activations(g, rows, dim).to(dtype)
        return {"case": case, "h": h, "dy": (1e-2 * _normal(g, rows, dim)).to(dtype),
                "dh": (1e-2 * _normal(g, rows, dim)).to(dtype) if case["residual"] else None,
                "weight": (1.0 + 0.1 * _normal(g, dim)).to(_DTYPES[case["wdtype"]]),
                "rstd": (h.float().square().mean(1) + _NORM_EPS).rsqrt()}
    tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
    weight = 0.02 * _normal(g, vocab, dim)
    target = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    # Hidden states that have learnt something: each leans towards its own
    # target's row, some by nothing and some so far that the token is sure.
    lean = torch.rand((tokens, 1), generator=g, device="cuda") * 16.0 / (0.02 ** 2 * dim)
    x = _normal(g, tokens, dim) + lean * weight[target]
    left_out = torch.rand((tokens,), generator=g, device="cuda") < case["ignored"]
    target = torch.where(left_out, torch.full_like(target, _IGNORE), target)
    # The loss's own gradient: 1, or the loss scale that training in fp16 keeps;
    # a weight for each token where the loss is not reduced.
    upstream = torch.ones((), device="cuda")
    if case["reduction"] == "none":
        upstream = torch.rand((tokens,), generator=g, device="cuda") + 0.5
    if dtype is torch.float16:
        upstream = upstream * (256.0 * tokens if case["reduction"] == "mean" else 256.0)
    return {"case": case, "x": x.to(dtype).requires_grad_(case["train"]),
            "weight": weight.to(dtype).requires_grad_(case["train"]), "target": target, "upstream": upstream}


# --------------------------------------------------------------------- run ---
def run(state):
    op = state["case"]["op"]
    if op == "norm_fwd":
        return _own_norm_fwd(state) if own else _plain_norm_fwd(state)
    if op == "norm_bwd":
        return _own_norm_bwd(state) if own else _plain_norm_bwd(state)
    if op == "loss":
        return _own_loss(state) if own else _plain_loss(state)
    return _own_clip(state) if own else _plain_clip(state)


def _own_norm_fwd(state):
    from practice_cuda_b200.rms_norm import rms_norm_quant

    case = state["case"]
    r = rms_norm_quant(state["x"], state["weight"], state["residual"], eps=_NORM_EPS, quant=case["quant"],
                       fp8_dtype=_FP8[case["fp8"]], return_y=case["keep"])
    out = {"q": r.quant.tensor, "scale": r.quant.dequant_scale, "rstd": r.rstd}
    if case["keep"]:
        out["y"] = r.y
    if case["residual"]:
        out["h"] = r.residual
    return out


def _own_norm_bwd(state):
    from practice_cuda_b200.rms_norm import rms_norm_backward

    dx, dw = rms_norm_backward(state["dy"], state["h"], state["weight"], state["rstd"], dresidual=state["dh"])
    return {"dx": dx, "dw": dw}


def _own_loss(state):
    from practice_cuda_b200.cross_entropy import linear_cross_entropy

    case, x, weight = state["case"], state["x"], state["weight"]
    loss = linear_cross_entropy(x, weight, state["target"], reduction=case["reduction"], ignore_index=_IGNORE)
    if not case["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (x, weight), state["upstream"])
    return {"loss": loss, "dx": dx, "dw": dw}


def _own_clip(state):
    from practice_cuda_b200.grad_clip import clip_grad_norm

    norm = clip_grad_norm(state["grads"], state["max_norm"], eps=_CLIP_EPS, out=state["out"])
    return {"norm": norm, "clipped": state["out_flat"]}


def _plain_norm_fwd(state):
    case = state["case"]
    x, weight, dtype = state["x"].float(), state["weight"].float(), state["x"].dtype
    # The sum is held in the input's type, as the next layer's residual reads
    # it, and the norm is that of the held values.
    h = (x + state["residual"].float()).to(dtype) if case["residual"] else state["x"]
    hf = h.float()
    rstd = 1.0 / (hf.square().mean(1) + _NORM_EPS).sqrt()
    y = hf * rstd[:, None] * weight
    q, scale = _plain_quant(y, case)
    out = {"q": q, "scale": scale, "rstd": rstd}
    if case["keep"]:
        out["y"] = y.to(dtype)
    if case["residual"]:
        out["h"] = h
    return out


def _plain_quant(y, case):
    rows, dim = y.shape
    top = _FP8_MAX[case["fp8"]]
    block = 128 if case["quant"] == "block" else dim
    blocks = -(-dim // block)
    padded = torch.nn.functional.pad(y, (0, blocks * block - dim)).view(rows, blocks, block)
    factor = top * (1.0 / padded.abs().amax(2).clamp_min(_QUANT_EPS))
    scale = 1.0 / factor if case["quant"] == "block" else padded.abs().amax(2).clamp_min(_QUANT_EPS) / top
    q = (padded * factor[:, :, None]).clamp(-top, top).view(rows, blocks * block)[:, :dim].to(_FP8[case["fp8"]])
    return q, scale if case["quant"] == "block" else scale[:, 0]


def _plain_norm_bwd(state):
    h, dy, weight, rstd = state["h"].float(), state["dy"].float(), state["weight"].float(), state["rstd"][:, None]
    n = h * rstd
    wdy = dy * weight
    dx = rstd * (wdy - n * (n * wdy).mean(1, keepdim=True))
    if state["dh"] is not None:
        dx = dx + state["dh"].float()
    return {"dx": dx.to(state["h"].dtype), "dw": (dy * n).sum(0).to(state["weight"].dtype)}


@torch.no_grad()
def _plain_loss(state):
    case, x, weight, target = state["case"], state["x"].float(), state["weight"].float(), state["target"]
    logits = x @ weight.t()
    valid = target != _IGNORE
    at = torch.where(valid, target, 0)[:, None]
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    total = e.sum(1, keepdim=True)
    nll = (total.log() + logits.amax(1, keepdim=True) - logits.gather(1, at))[:, 0]
    loss = torch.where(valid, nll, 0.0)
    if case["reduction"] != "none":
        loss = loss.sum()
    if case["reduction"] == "mean":
        loss = loss / valid.sum()
    if not case["train"]:
        return {"loss": loss}
    share = state["upstream"] / valid.sum() if case["reduction"] == "mean" else state["upstream"]
    share = torch.where(valid, share, 0.0)[:, None]
    g = e / total
    g.scatter_add_(1, at, torch.full_like(total, -1.0))
    g = g * share
    return {"loss": loss, "dx": (g @ weight).to(state["x"].dtype), "dw": (g.t() @ x).to(state["weight"].dtype)}


def _plain_clip(state):
    g = torch.cat([t.float() for t in state["grads"]])
    norm = g.square().sum().sqrt()
    factor = (state["max_norm"] / (norm + _CLIP_EPS)).clamp_max(1.0)
    return {"norm": norm, "clipped": (g * factor).to(state["flat"].dtype)}


# -------------------------------------------------------------------- work ---
def work(case):
    op = case["op"]
    if op == "clip":
        n = sum(_clip_sizes(case))
        return {"bytes": 2 * n * _DTYPES[case["dtype"]].itemsize, "flops": 3 * n}
    size = _DTYPES[case["dtype"]].itemsize
    if op == "norm_fwd":
        n = case["rows"] * case["dim"]
        scales = case["rows"] * (-(-case["dim"] // 128) if case["quant"] == "block" else 1)
        tensors = 1 + (2 if case["residual"] else 0) + (1 if case["keep"] else 0)
        return {"bytes": n * (size * tensors + 1) + 4 * (scales + case["rows"]) + case["dim"] * size, "flops": 7 * n}
    if op == "norm_bwd":
        n = case["rows"] * case["dim"]
        wsize = _DTYPES[case["wdtype"]].itemsize
        return {"bytes": n * size * (4 if case["residual"] else 3) + 4 * case["rows"] + 2 * case["dim"] * wsize,
                "flops": 10 * n}
    tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
    operands = (tokens + vocab) * dim * size + 8 * tokens + 4 * tokens
    product = 2 * tokens * vocab * dim
    if not case["train"]:
        return {"bytes": operands, "flops": product}
    return {"bytes": operands + (tokens + vocab) * dim * size, "flops": 3 * product}


# ------------------------------------------------------------------- exact ---
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        norm = torch.linalg.vector_norm(state["flat"], dtype=torch.float64)
        factor = min(1.0, state["max_norm"] / (norm.item() + _CLIP_EPS))
        return {"norm": norm, "clipped": state["flat"].double().mul_(factor)}
    if op == "norm_bwd":
        h, dy, w = (state[k].double() for k in ("h", "dy", "weight"))
        # y_j = w_j h_j / r with r = sqrt(mean(h^2) + eps): the gradient of the
        # product of a vector and 1 / r, term by term.
        inv = state["rstd"].double()
        inner = torch.einsum("td,td,d->t", dy, h, w) * inv ** 3 / case["dim"]
        dx = torch.einsum("td,d,t->td", dy, w, inv) - torch.einsum("td,t->td", h, inner)
        dx = dx if state["dh"] is None else dx + state["dh"].double()
        return {"dx": dx, "dw": torch.einsum("td,td,t->d", dy, h, inv)}
    if op == "norm_fwd":
        h64 = state["x"].double()
        if case["residual"]:
            h64 = h64 + state["residual"].double()
        h = h64.to(state["x"].dtype).double()  # the norm is that of the sum as it is held
        rstd = (h.pow(2).sum(1) / case["dim"] + _NORM_EPS).pow(-0.5)
        y = torch.einsum("td,t,d->td", h, rstd, state["weight"].double())
        top = _FP8_MAX[case["fp8"]]
        edges = list(range(0, case["dim"], 128 if case["quant"] == "block" else case["dim"])) + [case["dim"]]
        parts = [y[:, a:b] for a, b in zip(edges, edges[1:])]
        peaks = [torch.linalg.vector_norm(p, math.inf, 1).clamp_min(_QUANT_EPS) for p in parts]
        q = torch.cat([p * (top / peak)[:, None] for p, peak in zip(parts, peaks)], 1)
        scale = torch.stack(peaks, 1) / top
        out = {"q": q.to(_FP8[case["fp8"]]).double(), "rstd": rstd,
               "scale": scale if case["quant"] == "block" else scale[:, 0]}
        if case["keep"]:
            out["y"] = y
        if case["residual"]:
            out["h"] = h64
        return out
    x, w, target = state["x"].double(), state["weight"].double(), state["target"]
    rows = torch.arange(case["tokens"], device="cuda")[target != _IGNORE]
    logp = torch.log_softmax(x[rows] @ w.t(), 1)
    picked = logp[torch.arange(len(rows), device="cuda"), target[rows]]
    loss = torch.zeros(case["tokens"], device="cuda", dtype=torch.float64)
    loss[rows] = -picked
    share = state["upstream"].double()
    if case["reduction"] == "none":
        share = share[rows]
    else:
        loss, share = loss.sum(), share.expand(len(rows))
        if case["reduction"] == "mean":
            loss, share = loss / loss.new_tensor(len(rows)), share / max(1, len(rows))
    if not case["train"]:
        return {"loss": loss}
    g = logp.exp()
    g[torch.arange(len(rows), device="cuda"), target[rows]] -= 1.0
    g *= share[:, None]
    dx = torch.zeros_like(x)
    dx[rows] = g @ w
    return {"loss": loss, "dx": dx, "dw": g.t() @ x[rows]}

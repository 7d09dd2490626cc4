"""Cases for measuring the training operators beside the dense layers: layer norm (forward; backward with the gradients
of its weight and bias), embedding lookup with scaling and its gradient, and the orthogonalisation of an update by
Newton-Schulz products.

`run` computes an operator from elementary torch operations in 32 bits, or, with `own` true, through
tensorfrost_amd.runtime. Both leave their results in tensors; the second in ones the state holds, since the framework's
calls write into buffers that the caller owns.
"""
import math
import random

import numpy as np
import torch

own = False

MUON = (3.4445, -4.7750, 2.0315)  # coefficients of the quintic that optimisers commonly take, five steps of it
NORM_EPS = 1e-7
LAYER_EPS = 1e-5


def listed():
    return [
        # a handful of tokens at a time: the call itself is what it costs
        {"name": "ln_forward_few_rows", "op": "ln_forward", "rows": 8, "cols": 1024, "shift": 0.5},
        # odd row and column counts: no vector loads line up with the rows
        {"name": "ln_forward_odd", "op": "ln_forward", "rows": 4099, "cols": 1001, "shift": 2.0},
        # the matrix of this repository's reduction and softmax benchmark
        {"name": "ln_forward_large", "op": "ln_forward", "rows": 16384, "cols": 4096, "shift": 0.5},
        # ragged: neither rows nor columns divide evenly
        {"name": "ln_backward_ragged", "op": "ln_backward", "rows": 1037, "cols": 772, "shift": 1.0},
        # the activations of this repository's coordinate MLP: many rows of a hidden layer's width
        {"name": "ln_backward_mlp", "op": "ln_backward", "rows": 262144, "cols": 256, "shift": 0.5},
        # a short prompt with a little padding, an odd vocabulary and width
        {"name": "embed_few", "op": "embed", "n": 77, "vocab": 1009, "cols": 250, "pad": 0.1},
        # a training batch: most tokens are a few frequent ones
        {"name": "embed_batch", "op": "embed", "n": 65536, "vocab": 32768, "cols": 1024, "pad": 0.0},
        # the gradient of a small batch over an odd vocabulary
        {"name": "embed_grad_few", "op": "embed_grad", "n": 500, "vocab": 1009, "cols": 250, "pad": 0.1},
        # the gradient of the training batch
        {"name": "embed_grad_batch", "op": "embed_grad", "n": 65536, "vocab": 32768, "cols": 1024, "pad": 0.05},
        # the two hidden layers of the coordinate MLP in one call
        {"name": "orthogonal_mlp", "op": "orthogonal", "batch": 2, "rows": 256, "cols": 256},
        # an odd tall matrix
        {"name": "orthogonal_odd", "op": "orthogonal", "batch": 1, "rows": 1501, "cols": 1003},
        # a large dense layer
        {"name": "orthogonal_large", "op": "orthogonal", "batch": 1, "rows": 4096, "cols": 4096},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    op = rng.choice(["ln_forward", "ln_backward", "embed", "embed_grad", "orthogonal"])
    if op.startswith("ln"):
        cols = _log_uniform(rng, 1, 20000)
        rows = _log_uniform(rng, 1, max(1, min(300000, (16384 * 4096 if op == "ln_forward" else 262144 * 256) // cols)))
        if rng.random() < 0.5:
            cols = max(4, cols // 4 * 4)  # widths of layers are mostly whole vectors
        return {"op": op, "rows": rows, "cols": cols, "shift": round(rng.uniform(0.0, 4.0), 3)}
    if op.startswith("embed"):
        cols = _log_uniform(rng, 16, 2048)
        if rng.random() < 0.5:
            cols = cols // 4 * 4
        n = _log_uniform(rng, 1, min(131072, 65536 * 1024 // cols))
        vocab = _log_uniform(rng, 100, min(100000, 32768 * 1024 // cols))
        return {"op": op, "n": n, "vocab": vocab, "cols": cols, "pad": round(rng.choice([0.0, rng.uniform(0.0, 0.5)]), 3)}
    rows, cols = _log_uniform(rng, 16, 3000), _log_uniform(rng, 16, 3000)
    batch = rng.choice([1, 1, 2, 3, 6]) if rows * cols < 1000000 else 1
    return {"op": op, "batch": batch, "rows": rows, "cols": cols}


def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _normal(shape, seed, salt):
    return torch.randn(shape, generator=_generator(seed, salt), device="cuda", dtype=torch.float32)


def _empty(*shape):
    return torch.empty(shape, device="cuda", dtype=torch.float32)


def _tokens(case, seed):
    """Token t with probability proportional to 1 / (its rank + 1), ranks spread over the table; -1 behind the end of a padded row."""
    n, vocab = case["n"], case["vocab"]
    u = torch.rand(n, generator=_generator(seed, 1), device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).floor().clamp(0, vocab - 1).long()
    tokens = torch.randperm(vocab, generator=_generator(seed, 2), device="cuda")[rank]
    pad = int(n * case["pad"])
    if pad:
        tokens[n - pad:] = -1
    return tokens.to(torch.int32)


def _layer_inputs(case, seed):
    rows, cols = case["rows"], case["cols"]
    spread = torch.rand((rows, 1), generator=_generator(seed, 3), device="cuda") * 2 + 0.25
    x = _normal((rows, cols), seed, 4) * spread + case["shift"] * _normal((rows, 1), seed, 5)
    weight = 1.0 + 0.2 * _normal((cols,), seed, 6)
    return x.contiguous(), weight.contiguous()


def prepare(case, seed):
    op = case["op"]
    s = {"case": dict(case)}
    if op.startswith("ln"):
        rows, cols = case["rows"], case["cols"]
        s["x"], s["weight"] = _layer_inputs(case, seed)
        if op == "ln_forward":
            s["bias"] = 0.1 * _normal((cols,), seed, 7)
            s["y"], s["mean"], s["rstd"] = _empty(rows, cols), _empty(rows), _empty(rows)
        else:
            # the upstream gradient, and the row statistics that the forward pass left behind
            s["dy"] = _normal((rows, cols), seed, 8)
            mean = s["x"].mean(1)
            s["mean"] = mean
            s["rstd"] = torch.rsqrt((s["x"] - mean[:, None]).square().mean(1) + LAYER_EPS)
            s["dx"], s["dweight"], s["dbias"] = _empty(rows, cols), _empty(cols), _empty(cols)
        return s
    if op.startswith("embed"):
        n, vocab, cols = case["n"], case["vocab"], case["cols"]
        s["tokens"], s["scale"] = _tokens(case, seed), math.sqrt(cols)
        if op == "embed":
            s["table"], s["out"] = 0.02 * _normal((vocab, cols), seed, 9), _empty(n, cols)
        else:
            s["dy"], s["dtable"] = _normal((n, cols), seed, 10), _empty(vocab, cols)
        return s
    # a momentum buffer: a few strong directions over a floor of noise
    batch, rows, cols = case["batch"], case["rows"], case["cols"]
    rank = min(16, rows, cols)
    strong = torch.matmul(_normal((batch, rows, rank), seed, 11), _normal((batch, rank, cols), seed, 12).contiguous())
    s["g"] = (0.01 * (_normal((batch, rows, cols), seed, 13) + strong)).contiguous()
    s["out"] = _empty(batch, rows, cols)
    return s


# ---- the framework's calls ------------------------------------------------------------------------

def _own(s):
    """The library works on a stream of its own, which torch's does not wait for and which does not wait for torch's. The first
    call on a state waits until torch has filled it. The results are there, and the state may be dropped, once the whole
    device (torch.cuda.synchronize) or the library's stream (rt.synchronize) has been waited for."""
    from tensorfrost_amd import runtime as rt

    rt.initialize(0)
    if "filled" not in s:
        torch.cuda.synchronize()
        s["filled"] = True
    c = s["case"]
    b = {k: rt.DeviceBuffer.view(v.data_ptr(), v.numel()) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["op"] == "ln_forward":
        rt.layer_norm_rows(b["x"], b["weight"], b["bias"], b["y"], c["rows"], c["cols"], eps=LAYER_EPS, mean=b["mean"], rstd=b["rstd"])
        return s["y"], s["mean"], s["rstd"]
    if c["op"] == "ln_backward":
        rt.layer_norm_rows_backward(b["x"], b["dy"], b["weight"], b["mean"], b["rstd"], c["rows"], c["cols"], dx=b["dx"], dweight=b["dweight"], dbias=b["dbias"])
        return s["dx"], s["dweight"], s["dbias"]
    if c["op"] == "embed":
        rt.embedding_rows(b["tokens"], b["table"], b["out"], c["n"], c["vocab"], c["cols"], scale=s["scale"])
        return s["out"]
    if c["op"] == "embed_grad":
        rt.embedding_rows_backward(b["tokens"], b["dy"], b["dtable"], c["n"], c["vocab"], c["cols"], scale=s["scale"])
        return s["dtable"]
    rt.newton_schulz(b["g"], b["out"], c["rows"], c["cols"], steps=5, batch=c["batch"], coefficients=MUON, eps=NORM_EPS)
    return s["out"]


# ---- the plain forms ------------------------------------------------------------------------------

def _plain_ln_forward(s):
    x = s["x"]
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + LAYER_EPS)
    return centred * rstd * s["weight"] + s["bias"], mean[:, 0], rstd[:, 0]


def _plain_ln_backward(s):
    rstd = s["rstd"][:, None]
    xhat = (s["x"] - s["mean"][:, None]) * rstd
    g = s["dy"] * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx, (s["dy"] * xhat).sum(0), s["dy"].sum(0)


def _plain_embed(s):
    tokens, vocab = s["tokens"].long(), s["case"]["vocab"]
    known = (tokens >= 0) & (tokens < vocab)
    return torch.where(known[:, None], s["table"][tokens.clamp(0, vocab - 1)] * s["scale"], 0.0)


def _plain_embed_grad(s):
    tokens, vocab = s["tokens"].long(), s["case"]["vocab"]
    known = (tokens >= 0) & (tokens < vocab)
    # one more row takes what belongs to no token
    sums = torch.zeros((vocab + 1, s["case"]["cols"]), device=tokens.device, dtype=torch.float32)
    sums.index_add_(0, torch.where(known, tokens, vocab), s["dy"])
    return sums[:vocab] * s["scale"]


def _plain_orthogonal(s):
    a, b, c = MUON
    g = s["g"]
    tall = g.shape[1] > g.shape[2]
    x = g.transpose(1, 2).contiguous() if tall else g
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + NORM_EPS)
    for _ in range(5):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


def run(state):
    if own:
        return _own(state)
    return {"ln_forward": _plain_ln_forward, "ln_backward": _plain_ln_backward, "embed": _plain_embed,
            "embed_grad": _plain_embed_grad, "orthogonal": _plain_orthogonal}[state["case"]["op"]](state)


# ---- 64 bits, from the definitions ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.dtype == torch.float32}
    if op == "ln_forward":
        variance, mean = torch.var_mean(d["x"], 1, correction=0)
        rstd = 1.0 / torch.sqrt(variance + LAYER_EPS)
        return torch.addcmul(d["bias"], (d["x"] - mean[:, None]) * rstd[:, None], d["weight"]), mean, rstd
    if op == "ln_backward":
        # dx_j = rstd sum_k (delta_jk - 1/C - xhat_j xhat_k / C) w_k dy_k
        cols = case["cols"]
        xhat = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None]
        along = torch.matmul(d["dy"], d["weight"]) / cols
        across = torch.einsum("rc,rc,c->r", d["dy"], xhat, d["weight"]) / cols
        dx = (d["dy"] * d["weight"] - along[:, None] - xhat * across[:, None]) * d["rstd"][:, None]
        return dx, torch.einsum("rc,rc->c", d["dy"], xhat), torch.einsum("rc->c", d["dy"])
    if op.startswith("embed"):
        tokens = s["tokens"].cpu().numpy().astype(np.int64)
        known = (tokens >= 0) & (tokens < case["vocab"])
        if op == "embed":
            out = torch.zeros((case["n"], case["cols"]), dtype=torch.float64, device="cuda")
            where = torch.from_numpy(np.flatnonzero(known)).cuda()
            out[where] = d["table"].index_select(0, torch.from_numpy(tokens[known]).cuda()) * s["scale"]
            return out
        # by differences of running sums over the rows in token order
        order = np.argsort(np.where(known, tokens, case["vocab"]), kind="stable")[: int(known.sum())]
        dtable = torch.zeros((case["vocab"], case["cols"]), dtype=torch.float64, device="cuda")
        if len(order):
            values, counts = np.unique(tokens[order], return_counts=True)
            last = torch.from_numpy(np.cumsum(counts) - 1).cuda()
            ends = d["dy"].index_select(0, torch.from_numpy(order).cuda()).cumsum(0).index_select(0, last)
            dtable[torch.from_numpy(values).cuda()] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1])) * s["scale"]
        return dtable
    # X_k = X_0 Q_k with Q_k a polynomial of X_0^T X_0 on the short side
    a, b, c = MUON
    outs = []
    for g in d["g"]:
        wide = g.shape[0] <= g.shape[1]
        x0 = g.T.contiguous() if wide else g
        x0 = x0 / (torch.linalg.vector_norm(x0) + NORM_EPS)
        gram0 = x0.T.contiguous() @ x0
        q = torch.eye(gram0.shape[0], dtype=torch.float64, device=g.device)
        for _ in range(5):
            gram = q @ gram0 @ q
            q = q @ (a * torch.eye(q.shape[0], dtype=torch.float64, device=g.device) + b * gram + c * gram @ gram)
        out = x0 @ q
        outs.append(out.T.contiguous() if wide else out)
    return torch.stack(outs)


def _distinct(case):
    """Expected number of different tokens in a batch."""
    p = np.log1p(1.0 / np.arange(1, case["vocab"] + 1)) / math.log(case["vocab"] + 1.0)
    return float(-np.expm1((case["n"] - int(case["n"] * case["pad"])) * np.log1p(-p)).sum())


def work(case):
    op = case["op"]
    if op.startswith("ln"):
        rows, cols = case["rows"], case["cols"]
        if op == "ln_forward":
            return {"bytes": 8 * rows * cols + 8 * rows + 8 * cols, "flops": 8 * rows * cols}
        return {"bytes": 12 * rows * cols + 8 * rows + 12 * cols, "flops": 16 * rows * cols}
    if op == "embed":
        return {"bytes": 4 * case["n"] * (case["cols"] + 1) + 4 * _distinct(case) * case["cols"], "flops": case["n"] * case["cols"]}
    if op == "embed_grad":
        known = case["n"] - int(case["n"] * case["pad"])
        return {"bytes": 4 * known * case["cols"] + 4 * case["n"] + 4 * case["vocab"] * case["cols"], "flops": known * case["cols"]}
    m, n = sorted((case["rows"], case["cols"]))
    # two of the three products of a step are symmetric
    return {"bytes": 8 * case["batch"] * m * n, "flops": 5 * case["batch"] * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)}

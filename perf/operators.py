"""Operators of a language model's training step and of scoring, next to op::softmax, op::L2_norm and op::gather_from_rows:

* layer normalisation along the last axis and its gradient (the weights' gradient, a reduction over the rows, included),
* the log probability of a given token per row of logits with the entropy and the most probable alternatives, and the
  gradient of both with respect to the logits,
* the global norm of a list of gradients and the gradients clipped to a maximal norm.

A case names its operator, its sizes and its types; `run` makes one pass."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 3}     # element type codes of the C ABI
SIZE = {"f32": 4, "bf16": 2}

EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decoding step through a layer norm of the recurrent cell's width
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 1024, "type": "bf16", "weights": "bf16"},
        # a batch of sequences, mixed precision: 16-bit activations, 32-bit weights
        {"name": "norm batch bf16", "op": "norm", "rows": 16384, "cols": 4096, "type": "bf16", "weights": "f32"},
        # an odd width whose rows start off the 16-byte grid
        {"name": "norm odd f32", "op": "norm", "rows": 2999, "cols": 1537, "type": "f32", "weights": "f32"},
        # the gradient for a small batch: few rows, so latency and the reduction over the rows count
        {"name": "norm gradient small", "op": "norm_grad", "rows": 256, "cols": 1024, "type": "f32", "weights": "f32"},
        # the gradient of the batch above
        {"name": "norm gradient batch", "op": "norm_grad", "rows": 16384, "cols": 4096, "type": "bf16", "weights": "f32"},
        # one token of a decoding step: the chosen token's log probability, the entropy and 20 alternatives
        {"name": "score one token", "op": "score", "rows": 1, "vocab": 131072, "type": "bf16", "top": 20, "masked": 0.0},
        # scoring a prompt over an odd vocabulary, some entries masked out, five alternatives
        {"name": "score prompt", "op": "score", "rows": 1000, "vocab": 50001, "type": "f32", "top": 5, "masked": 0.1},
        # the loss of a training batch: no alternatives
        {"name": "score batch", "op": "score", "rows": 8192, "vocab": 65536, "type": "bf16", "top": 0, "masked": 0.0},
        # the gradient of a policy's log probabilities and entropies over an odd vocabulary
        {"name": "score gradient odd", "op": "score_grad", "rows": 500, "vocab": 10007, "type": "f32", "masked": 0.05, "entropy": True},
        # the loss's gradient for the training batch
        {"name": "score gradient batch", "op": "score_grad", "rows": 8192, "vocab": 65536, "type": "bf16", "masked": 0.0, "entropy": False},
        # the weights of one recurrent cell, 32-bit
        {"name": "clip cell", "op": "clip", "tensors": 6, "elements": 1000000, "type": "f32", "limit": 1.0},
        # the 16-bit gradients of a whole model; the last of the sizes are vectors among matrices
        {"name": "clip model", "op": "clip", "tensors": 60, "elements": 400000000, "type": "bf16", "limit": 1.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "score", "score_grad", "clip"])
    t = rng.choice(["f32", "bf16"])
    if op in ("norm", "norm_grad"):
        cols = _log_int(rng, 33, 20000)
        if rng.random() < 0.5:
            cols = (cols + 7) // 8 * 8
        rows = _log_int(rng, 1, max(1, min(65536, 50000000 // cols)))
        return {"op": op, "rows": rows, "cols": cols, "type": t, "weights": rng.choice([t, "f32"])}
    if op in ("score", "score_grad"):
        vocab = _log_int(rng, 100, 260000)
        if rng.random() < 0.5:
            vocab = (vocab + 63) // 64 * 64
        rows = _log_int(rng, 1, max(1, min(16384, 100000000 // vocab)))
        c = {"op": op, "rows": rows, "vocab": vocab, "type": t, "masked": rng.choice([0.0, 0.1, 0.9])}
        if op == "score":
            c["top"] = rng.choice([0, 1, 5, 20, 32])
        else:
            c["entropy"] = rng.random() < 0.5
        return c
    n = _log_int(rng, 1, 60)
    return {"op": "clip", "tensors": n, "elements": _log_int(rng, 1000 * n, 200000000), "type": t, "limit": rng.choice([0.5, 1.0, 1e9])}


def _clip_sizes(case):
    """Sizes of the tensors of a clip case: matrices and vectors in turn, some of them odd, `elements` in all."""
    n, left = case["tensors"], case["elements"]
    weight = [(1 + 7 * (i % 5)) if i % 2 == 0 else 0.01 for i in range(n)]
    total, sizes = sum(weight), []
    for i in range(n):
        sizes.append(max(1, int(case["elements"] * weight[i] / total)))
    sizes[0] += max(0, left - sum(sizes))
    return sizes


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dev, t = "cuda", DTYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    s = {"case": dict(case)}
    op = case["op"]
    if op in ("norm", "norm_grad"):
        r, c, w = case["rows"], case["cols"], DTYPES[case["weights"]]
        # activations whose rows differ in offset and scale
        s["x"] = (normal(r, c) * (0.5 + normal(r, 1).abs()) + normal(r, 1)).to(t)
        s["gamma"] = (1 + 0.1 * normal(c)).to(w)
        s["out"] = torch.empty(r, c, device=dev, dtype=t)
        if op == "norm":
            s["beta"] = (0.1 * normal(c)).to(w)
        else:
            s["dy"] = normal(r, c).to(t)
            s["dgamma"] = torch.empty(c, device=dev, dtype=w)
            s["dbeta"] = torch.empty(c, device=dev, dtype=w)
    elif op in ("score", "score_grad"):
        r, v = case["rows"], case["vocab"]
        z = 3 * normal(r, v)
        tokens = torch.randint(0, v, (r,), generator=g, device=dev, dtype=torch.int64)
        if case["masked"] > 0:
            drop = torch.rand(r, v, generator=g, device=dev) < case["masked"]
            drop.scatter_(1, tokens[:, None], False)        # the given token is one that may be chosen
            z.masked_fill_(drop, -math.inf)
            del drop
        s["logits"] = z.to(t)
        del z
        if r >= 8:
            tokens[torch.rand(r, generator=g, device=dev) < 0.05] = -1      # rows of padding
        s["tokens"] = tokens.to(torch.int32)
        f = dict(device=dev, dtype=torch.float32)
        if op == "score":
            k = case["top"]
            s["logprob"], s["entropy"], s["lse"] = (torch.empty(r, **f) for _ in range(3))
            s["top_logprobs"] = torch.empty(r, k, **f)
            s["top_tokens"] = torch.empty(r, k, device=dev, dtype=torch.int32)
        else:
            # what the forward pass left, and the gradients that arrive for it
            lse, ent = torch.empty(r, **f), torch.empty(r, **f)
            step = max(1, 50000000 // v)
            for i in range(0, r, step):
                x = s["logits"][i:i + step].double()
                l = torch.logsumexp(x, 1)
                p = torch.exp(x - l[:, None])
                ent[i:i + step] = (l - (p * torch.where(p > 0, x, 0.0)).sum(1)).float()
                lse[i:i + step] = l.float()
            s["lse"], s["entropy"] = lse, ent
            s["dlogprob"] = normal(r) / r
            s["dentropy"] = 0.01 * normal(r) / r if case["entropy"] else None
            s["dlogits"] = torch.empty(r, v, device=dev, dtype=t)
    else:
        s["grads"] = [(0.02 * normal(n)).to(t) for n in _clip_sizes(case)]
        s["outs"] = [torch.empty_like(x) for x in s["grads"]]
        s["norm"] = torch.empty((), device=dev, dtype=torch.float32)
        s["limit"] = case["limit"]
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x = s["x"].float()
    d = x - x.mean(1, keepdim=True)
    y = d * torch.rsqrt(d.square().mean(1, keepdim=True) + EPS)
    return (y * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype)


def _plain_norm_grad(s):
    x, dy = s["x"].float(), s["dy"].float()
    d = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(d.square().mean(1, keepdim=True) + EPS)
    xhat = d * rstd
    a = dy * s["gamma"].float()
    dx = rstd * (a - a.mean(1, keepdim=True) - xhat * (a * xhat).mean(1, keepdim=True))
    w = s["gamma"].dtype
    return dx.to(s["x"].dtype), (dy * xhat).sum(0).to(w), dy.sum(0).to(w)


def _plain_score(s):
    z = s["logits"].float()
    tokens = s["tokens"].long()
    m = z.max(1, keepdim=True).values
    d = z - m
    e = torch.exp(d)
    total = e.sum(1)
    lse = m[:, 0] + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * d, 0.0).sum(1) / total
    given = z.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - lse
    logprob = torch.where(tokens < 0, 0.0, given)
    k = s["case"]["top"]
    if k == 0:
        return logprob, entropy, lse
    # a stable order: among equal values the lowest index first
    values, index = torch.sort(z, dim=1, descending=True, stable=True)
    return logprob, entropy, lse, values[:, :k] - lse[:, None], index[:, :k].to(torch.int32)


def _plain_score_grad(s):
    z = s["logits"].float()
    tokens = s["tokens"].long()
    logp = z - s["lse"][:, None]
    p = torch.exp(logp)
    dlp = torch.where(tokens < 0, 0.0, s["dlogprob"])
    dz = -dlp[:, None] * p
    if s["dentropy"] is not None:
        dz -= s["dentropy"][:, None] * torch.where(p > 0, p * (logp + s["entropy"][:, None]), 0.0)
    dz.scatter_add_(1, tokens.clamp(min=0)[:, None], dlp[:, None])
    return dz.to(s["logits"].dtype)


def _plain_clip(s):
    total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum()
    norm = torch.sqrt(total)
    scale = torch.where(norm > s["limit"], s["limit"] / norm, 1.0).float()
    return norm.float(), [(g.float() * scale).to(g.dtype) for g in s["grads"]]


# ----------------------------------------------------------------------------------------------------- the own operators
_library = None


def _lib():
    global _library
    if _library is None:
        from dali_b200 import load_library
        _library = load_library()
        _library.init(1)
    return _library


def _own(s):
    lib = _lib()
    c, op = s["case"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "norm":
        lib.layer_norm(CODES[s["x"].dtype], CODES[s["gamma"].dtype], c["rows"], c["cols"], s["x"], s["gamma"], s["beta"], s["out"],
                       eps=EPS, stream=stream)
        return s["out"]
    if op == "norm_grad":
        lib.layer_norm_backward(CODES[s["x"].dtype], CODES[s["gamma"].dtype], c["rows"], c["cols"], s["dy"], s["x"], s["gamma"],
                                s["out"], s["dgamma"], s["dbeta"], eps=EPS, stream=stream)
        return s["out"], s["dgamma"], s["dbeta"]
    if op == "score":
        k = c["top"]
        lib.token_logprobs(CODES[s["logits"].dtype], c["rows"], c["vocab"], s["logits"], s["tokens"], s["logprob"], s["entropy"],
                           s["lse"], top=k, top_logprobs=s["top_logprobs"] if k else None, top_tokens=s["top_tokens"] if k else None,
                           stream=stream)
        out = s["logprob"], s["entropy"], s["lse"]
        return out + (s["top_logprobs"], s["top_tokens"]) if k else out
    if op == "score_grad":
        lib.token_logprobs_backward(CODES[s["logits"].dtype], c["rows"], c["vocab"], s["logits"], s["tokens"], s["lse"], s["entropy"],
                                    s["dlogprob"], s["dentropy"], s["dlogits"], stream=stream)
        return s["dlogits"]
    lib.clip_by_global_norm([CODES[g.dtype] for g in s["grads"]], [g.numel() for g in s["grads"]], s["grads"], s["outs"], s["limit"],
                            s["norm"], stream=stream)
    return s["norm"], s["outs"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_grad":
        return _plain_norm_grad(state)
    if op == "score":
        return _plain_score(state)
    if op == "score_grad":
        return _plain_score_grad(state)
    return _plain_clip(state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    b = SIZE[case["type"]]
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * b + 2 * case["cols"] * SIZE[case["weights"]], "flops": 8 * n}
    if case["op"] == "norm_grad":
        n = case["rows"] * case["cols"]
        return {"bytes": 3 * n * b + 3 * case["cols"] * SIZE[case["weights"]], "flops": 16 * n}
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * b + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    if case["op"] == "score_grad":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * b + case["rows"] * 20, "flops": (8 if case["entropy"] else 4) * n}
    n = sum(_clip_sizes(case))
    return {"bytes": 2 * n * b + 4, "flops": 3 * n}


# ----------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        gamma = s["gamma"].double()
        out = torch.empty(r, c, device="cuda", dtype=torch.float64)
        dg, db = torch.zeros_like(gamma), torch.zeros_like(gamma)
        step = max(1, 30000000 // c)
        for i in range(0, r, step):
            x = s["x"][i:i + step].double()
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            std = torch.sqrt(var + EPS)
            h = (x - mean) / std
            if op == "norm":
                out[i:i + step] = h * gamma + s["beta"].double()
                continue
            dy = s["dy"][i:i + step].double()
            dh = dy * gamma
            out[i:i + step] = (c * dh - dh.sum(1, keepdim=True) - h * (dh * h).sum(1, keepdim=True)) / (c * std)
            dg += (dy * h).sum(0)
            db += dy.sum(0)
        return out if op == "norm" else (out, dg, db)
    if op == "score":
        r, k, step = case["rows"], case["top"], max(1, 40000000 // case["vocab"])
        parts = []
        for i in range(0, r, step):
            logp = torch.log_softmax(s["logits"][i:i + step].double(), dim=1)
            t = s["tokens"][i:i + step].long()
            lp = torch.where(t < 0, 0.0, logp[torch.arange(len(t), device="cuda"), t.clamp(min=0)])
            ent = -torch.special.xlogy(torch.exp(logp), torch.exp(logp)).sum(1)
            row = [lp, ent, torch.logsumexp(s["logits"][i:i + step].double(), dim=1)]
            if k:
                row.append(torch.topk(logp, k, dim=1).values)
            parts.append(row)
        out = [torch.cat(p) for p in zip(*parts)]
        return tuple(out) + ((None,) if k else ())
    if op == "score_grad":
        out = torch.empty(case["rows"], case["vocab"], device="cuda", dtype=torch.float64)
        step = max(1, 40000000 // case["vocab"])
        for i in range(0, case["rows"], step):
            q = torch.softmax(s["logits"][i:i + step].double(), dim=1)
            t = s["tokens"][i:i + step].long()
            w = torch.where(t < 0, 0.0, s["dlogprob"][i:i + step].double())[:, None]
            one = torch.zeros_like(q).scatter_(1, t.clamp(min=0)[:, None], 1.0)
            dz = w * (one - q)
            if s["dentropy"] is not None:
                qlogq = torch.special.xlogy(q, q)
                dz -= s["dentropy"][i:i + step].double()[:, None] * (qlogq - q * qlogq.sum(1, keepdim=True))
            out[i:i + step] = dz
        return out
    norm = torch.sqrt(sum((torch.linalg.vector_norm(g.double()) ** 2 for g in s["grads"]), torch.zeros((), device="cuda", dtype=torch.float64)))
    scale = torch.clamp(s["limit"] / norm, max=1.0)
    return norm, [g.double() * scale for g in s["grads"]]

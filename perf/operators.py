"""What is measured of the language-model head: layer norm and its gradient, the distillation loss from a
teacher's top logits and its gradient, the linear layer in 8-bit integers, and the choice of a token.

The plain forms below are elementary torch operations in 32 bits; `own` switches to the framework's kernels.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_ONE = 1 << 40  # the integer weight of a row's likeliest token


def listed():
    return [
        # The final norm of four sequences that each decode one token: a call of a few microseconds.
        {"name": "norm decode bf16", "op": "norm", "rows": 4, "cols": 4096, "type": "bf16", "stats": False},
        # The norm of a training step's forward pass, which keeps each row's mean and deviation for the backward pass.
        {"name": "norm train f16", "op": "norm", "rows": 16384, "cols": 1024, "type": "f16", "stats": True},
        # The norm's backward pass in a training step, with the sums over rows that the weight and bias need.
        {"name": "norm grad bf16", "op": "norm_grad", "rows": 8192, "cols": 4096, "type": "bf16"},
        # The same in 32 bits, on a width and a count that no tile divides.
        {"name": "norm grad odd f32", "op": "norm_grad", "rows": 1021, "cols": 5003, "type": "f32"},
        # A step of distillation over a large vocabulary: the loss and its gradient from one call.
        {"name": "distill step bf16", "op": "distill", "rows": 2048, "vocab": 131072, "top": 64, "type": "bf16", "part": "both"},
        # Validation: the loss alone, of a few positions.
        {"name": "distill loss f32", "op": "distill", "rows": 37, "vocab": 32003, "top": 17, "type": "f32", "part": "loss"},
        # The backward pass on its own, for a caller that weighs the rows' losses first.
        {"name": "distill grad f16", "op": "distill", "rows": 512, "vocab": 50001, "top": 100, "type": "f16", "part": "grad"},
        # One token through an expanding layer: the weights' bytes are what it costs.
        {"name": "int8 decode bf16", "op": "int8", "rows": 1, "inner": 4096, "cols": 16384, "type": "bf16", "bias": False},
        # A batch of prompts: a matrix product that the tensor cores bound.
        {"name": "int8 prompts bf16", "op": "int8", "rows": 4096, "inner": 8192, "cols": 8192, "type": "bf16", "bias": False},
        # A ragged batch against a layer whose sizes no tile divides.
        {"name": "int8 odd f16", "op": "int8", "rows": 333, "inner": 1001, "cols": 4099, "type": "f16", "bias": True},
        # The next token of one sequence: latency counts.
        {"name": "sample one f32", "op": "sample", "rows": 1, "vocab": 32768, "type": "f32"},
        # The next tokens of a serving batch, each row with its own settings.
        {"name": "sample batch bf16", "op": "sample", "rows": 256, "vocab": 131071, "type": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number, evenly spread over the logarithm of the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "distill", "int8", "sample"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("norm", "norm_grad"):
        cols = _spread(rng, 64, 16384)
        most = (16 << 20 if op == "norm" else 32 << 20) // cols
        if kind == "f32":
            most //= 2
        case = {"op": op, "rows": _spread(rng, 1, min(16384, most)), "cols": cols, "type": kind}
        return dict(case, stats=rng.random() < 0.5) if op == "norm" else case
    if op == "distill":
        vocab = _spread(rng, 1000, 131072)
        most = (256 << 20) // vocab // (2 if kind == "f32" else 1)
        return {"op": op, "rows": _spread(rng, 1, min(4096, most)), "vocab": vocab, "top": _spread(rng, 1, 256),
                "type": kind, "part": rng.choice(["loss", "grad", "both"])}
    if op == "int8":
        inner, cols = _spread(rng, 64, 8192), _spread(rng, 64, 16384)
        return {"op": op, "rows": _spread(rng, 1, min(4096, (4096 << 26) // (inner * cols))), "inner": inner, "cols": cols,
                "type": kind, "bias": rng.random() < 0.5}
    vocab = _spread(rng, 1000, 131071)
    most = (256 * 131071) // vocab // (2 if kind == "f32" else 1)
    return {"op": op, "rows": _spread(rng, 1, min(256, most)), "vocab": vocab, "type": kind}


def prepare(case, seed):
    made = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=made, device="cuda")

    def even(*shape):
        return torch.rand(*shape, generator=made, device="cuda")

    kind, op, rows = _TYPES[case["type"]], case["op"], case["rows"]
    if op in ("norm", "norm_grad"):
        cols = case["cols"]
        # a residual stream: rows of different size, a few columns far larger than the rest
        x = normal(rows, cols) * torch.exp(0.5 * normal(rows, 1)) * torch.exp(0.7 * normal(cols)) + 0.3 * normal(rows, 1)
        s = {"case": case, "x": x.to(kind), "gamma": 1 + 0.2 * normal(cols), "beta": 0.1 * normal(cols), "eps": 1e-5}
        if op == "norm_grad":
            s["dy"] = (0.01 * normal(rows, cols)).to(kind)
            x = s["x"].double()
            s["mean"] = x.mean(1).float()
            s["rstd"] = (1 / torch.sqrt(x.var(1, correction=0) + s["eps"])).float()
        return s
    if op == "distill":
        vocab, top = case["vocab"], min(case["top"], case["vocab"])
        teacher = 2.5 * normal(rows, vocab)
        values, indices = teacher.topk(top, 1)
        student = (0.7 * teacher + 1.5 * normal(rows, vocab)).to(kind)
        del teacher
        # some teachers list fewer tokens than there is room for; some positions are padding
        indices = torch.where((torch.arange(top, device="cuda") > 0) & (even(rows, 1) < 0.1) & (even(rows, top) < 0.3),
                              torch.full_like(indices, -1), indices)
        weight = (even(rows) > 0.05).float()
        weight[0] = 1.0
        s = {"case": case, "logits": student, "teacher": values.to(kind), "indices": indices, "weight": weight,
             "temperature": 2.0, "dloss": even(rows) * ((4096 if case["type"] == "f16" else 1) / rows)}  # f16: a scaled loss
        if case["part"] == "grad":
            s["lse"] = torch.where(weight == 0, torch.zeros_like(weight),
                                   torch.cat([torch.logsumexp(r.double() / 2.0, 1) for r in student.split(256)]).float())
        return s
    if op == "int8":
        inner, cols = case["inner"], case["cols"]
        x = (normal(rows, inner) * torch.exp(0.8 * normal(inner))).to(kind)
        w = normal(cols, inner) / math.sqrt(inner)
        scale = w.abs().amax(1) / 127
        q = torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8)
        bias = 0.1 * normal(cols) if case["bias"] else None
        s = {"case": case, "x": x, "q": q, "scale": scale, "bias": bias}
        if own:
            import zpu_b200
            s["layer"] = zpu_b200.Int8Linear(q, scale, bias)  # the weights as the framework keeps them
        return s
    vocab = case["vocab"]
    x = 2.5 * normal(rows, vocab)
    # the tokens that the context makes likely, and those that the caller forbids
    at = torch.randint(0, vocab, (rows, 24), generator=made, device="cuda")
    x.scatter_add_(1, at, 9 * even(rows, 24))
    x.masked_fill_(even(rows, vocab) < 0.005, -math.inf)
    some = even(rows, 4)
    n = torch.randint(1, 200, (rows,), generator=made, device="cuda")
    zero = torch.zeros_like(n)
    return {"case": case, "logits": x.to(kind), "uniform": even(rows),
            "temperature": torch.where(even(rows) < 0.1, 0.0, 0.5 + even(rows)),
            "top_k": torch.where(some[:, 1] < 0.6, n, zero).to(torch.int32),
            "top_p": torch.where(some[:, 2] < 0.7, 0.7 + 0.3 * even(rows), 1.0),
            "min_p": torch.where(some[:, 3] < 0.3, 0.1 * even(rows), 0.0)}


def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    import zpu_b200 as zc

    case = s["case"]
    if case["op"] == "norm":
        if case["stats"]:
            y, mean, rstd = zc.layer_norm(s["x"], s["gamma"], s["beta"], eps=s["eps"], stats=True)
            return {"y": y, "mean": mean, "rstd": rstd}
        return {"y": zc.layer_norm(s["x"], s["gamma"], s["beta"], eps=s["eps"])}
    if case["op"] == "norm_grad":
        dx, dgamma, dbeta = zc.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if case["op"] == "distill":
        more = {"temperature": s["temperature"], "weight": s["weight"]}
        if case["part"] == "loss":
            loss, lse = zc.distill_loss(s["logits"], s["teacher"], s["indices"], **more)
            return {"loss": loss, "lse": lse}
        if case["part"] == "grad":
            return {"dlogits": zc.distill_grad(s["logits"], s["teacher"], s["indices"], s["lse"], s["dloss"], **more)}
        loss, dlogits = zc.distill_value_and_grad(s["logits"], s["teacher"], s["indices"], s["dloss"], **more)
        return {"loss": loss, "dlogits": dlogits}
    if case["op"] == "int8":
        return {"y": s["layer"](s["x"])}
    token, logprob = zc.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                               top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        x = x - mean[:, None]
        rstd = 1 / torch.sqrt((x * x).mean(1) + s["eps"])
        y = (x * rstd[:, None] * s["gamma"] + s["beta"]).to(s["x"].dtype)
        return {"y": y, "mean": mean, "rstd": rstd} if case["stats"] else {"y": y}
    if case["op"] == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
        g = dy * s["gamma"]
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if case["op"] == "distill":
        return _plain_distill(s, case["part"])
    if case["op"] == "int8":
        x = s["x"].float()
        scale = x.abs().amax(1, keepdim=True) / 127
        q = torch.where(scale > 0, torch.round(x / scale).clamp(-127, 127), 0.0)
        y = (q @ s["q"].float().t()) * scale * s["scale"]
        return {"y": (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)}
    return _plain_sample(s)


def _plain_distill(s, part):
    t, weight = s["temperature"], s["weight"]
    z = s["logits"].float() / t
    there = s["indices"] >= 0
    at = s["indices"].clamp(min=0)
    u = torch.where(there, s["teacher"].float() / t, -math.inf)
    e = torch.exp(u - u.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    if part == "grad":
        lse = s["lse"]
    else:
        m = z.amax(1)
        lse = m + torch.log(torch.exp(z - m[:, None]).sum(1))
        logq = z.gather(1, at) - lse[:, None]
        loss = weight * (t * t) * torch.where(p > 0, p * (torch.log(p) - logq), 0.0).sum(1)
        if part == "loss":
            return {"loss": loss, "lse": torch.where(weight == 0, 0.0, lse)}
    c = (weight * s["dloss"])[:, None] * t
    d = torch.exp(z - lse[:, None]).scatter_add(1, at, -p)
    d = torch.where(c == 0, 0.0, c * d).to(s["logits"].dtype)
    return {"dlogits": d} if part == "grad" else {"loss": loss, "dlogits": d}


def _plain_sample(s):
    x = s["logits"].float()
    t = s["temperature"]
    m = x.amax(1, keepdim=True)
    step = torch.where(t > 0, 1 / t, 0.0)[:, None]
    d = (x - m) * step
    e = torch.where(x == m, 1.0, torch.where(x == -math.inf, 0.0, torch.exp(d)))
    w = (e * float(_ONE)).long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(x.shape[1], device=x.device)[None]
    count = torch.where(t > 0, s["top_k"], 1)[:, None]  # temperature 0: the likeliest token
    w = torch.where((count <= 0) | (rank < count), w, 0)
    total = w.sum(1, keepdim=True)
    edge = torch.ceil(s["top_p"].double()[:, None] * total.double()).long()
    w = torch.where((s["top_p"][:, None] >= 1) | (w.cumsum(1) - w < edge), w, 0)
    w = torch.where(w >= torch.ceil(s["min_p"].double() * _ONE).long()[:, None], w, 0)
    total = w.sum(1)
    w = torch.zeros_like(w).scatter_(1, order, w)
    at = torch.floor(s["uniform"].double() * total.double()).long().clamp(max=total - 1)
    token = (w.cumsum(1) <= at[:, None]).sum(1)
    logprob = d.gather(1, token[:, None])[:, 0] - torch.log(total.float() / _ONE)
    return {"token": token, "logprob": logprob}


def work(case):
    e, op, rows = _BYTES[case["type"]], case["op"], case["rows"]
    if op == "norm":
        n = rows * case["cols"]
        return {"bytes": 2 * n * e + 8 * case["cols"] + (8 * rows if case["stats"] else 0), "flops": 8 * n}
    if op == "norm_grad":
        n = rows * case["cols"]
        return {"bytes": 3 * n * e + 12 * case["cols"] + 8 * rows, "flops": 14 * n}
    if op == "distill":
        n, k = rows * case["vocab"], rows * min(case["top"], case["vocab"])
        return {"bytes": (1 if case["part"] == "loss" else 2) * n * e + (8 + e) * k + 12 * rows,
                "flops": (8 if case["part"] == "both" else 5) * n}
    if op == "int8":
        k, n = case["inner"], case["cols"]
        return {"bytes": rows * k * e + n * k + rows * n * e + (8 if case["bias"] else 4) * n, "flops": 2 * rows * k * n}
    n = rows * case["vocab"]
    return {"bytes": n * e + 32 * rows, "flops": 6 * n}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        x, gamma = s["x"].double(), s["gamma"].double()
        if op == "norm":
            var, mean = torch.var_mean(x, 1, correction=0)
            y = (x - mean[:, None]) / torch.sqrt(var + s["eps"])[:, None] * gamma + s["beta"].double()
            return {"y": y, "mean": mean, "rstd": (var + s["eps"]).rsqrt()} if case["stats"] else {"y": y}
        dy, rstd, n = s["dy"].double(), s["rstd"].double()[:, None], x.shape[1]
        xhat = (x - s["mean"].double()[:, None]) * rstd
        a = (dy @ gamma)[:, None]
        b = ((dy * xhat) @ gamma)[:, None]
        return {"dx": rstd / n * (n * dy * gamma - a - xhat * b), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if op == "distill":
        return _exact_distill(s, case["part"])
    if op == "int8":
        x = s["x"].double()
        scale = (x.abs().amax(1) / 127).float().double()[:, None]  # the scale that a token keeps is a 32-bit number
        q = torch.where(scale > 0, torch.round(x / scale), 0.0)
        y = (q * scale) @ (s["q"].double() * s["scale"].double()[:, None]).t()
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    return _exact_sample(s)


def _exact_distill(s, part):
    t, loss, lses, grads = s["temperature"], [], [], []
    for r in range(0, s["logits"].shape[0], 128):  # some rows at a time
        z = s["logits"][r:r + 128].double() / t
        index, w = s["indices"][r:r + 128], s["weight"][r:r + 128].double()
        logp = torch.log_softmax((s["teacher"][r:r + 128].double() / t).masked_fill(index < 0, -math.inf), 1)
        p, at = logp.exp(), index.clamp(min=0)
        lse = torch.logsumexp(z, 1) if part != "grad" else s["lse"][r:r + 128].double()
        logq = z - lse[:, None]
        each = torch.where(p > 0, p * (logp - logq.gather(1, at)), torch.zeros_like(p))
        loss.append(w * t ** 2 * each.sum(1))
        lses.append(torch.where(w == 0, torch.zeros_like(lse), lse))
        if part != "loss":
            c = (w * s["dloss"][r:r + 128].double() * t)[:, None]
            grads.append(torch.where(c == 0, torch.zeros_like(c), c * logq.exp().scatter_add(1, at, -p)))
    if part == "loss":
        return {"loss": torch.cat(loss), "lse": torch.cat(lses)}
    return {"dlogits": torch.cat(grads)} if part == "grad" else {"loss": torch.cat(loss), "dlogits": torch.cat(grads)}


def _exact_sample(s):
    tokens, logprobs = [], []
    for r in range(s["logits"].shape[0]):  # one row at a time, over the tokens that may be chosen
        x, t = s["logits"][r].double(), float(s["temperature"][r])
        k, p, least = int(s["top_k"][r]), float(s["top_p"][r]), float(s["min_p"][r])
        if not t > 0:
            tokens.append(x.argmax())
            logprobs.append(torch.zeros((), dtype=torch.float64, device="cuda"))
            continue
        x, order = torch.sort(x, descending=True, stable=True)
        prob = torch.softmax(x[:k if k > 0 else None] / t, 0)
        kept = prob >= least * prob[0]
        if p < 1:
            kept &= prob.cumsum(0) - prob < p
        prob, order = prob[kept], order[:len(prob)][kept]
        order, back = torch.sort(order)
        prob = prob[back] / prob.sum()
        at = torch.searchsorted(prob.cumsum(0), s["uniform"][r].double(), right=True).clamp(max=len(prob) - 1)
        tokens.append(order[at])
        logprobs.append(prob[at].log())
    return {"token": torch.stack(tokens), "logprob": torch.stack(logprobs)}

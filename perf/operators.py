"""Workloads of the language-model training operators, in their plain form and as the library's calls.

Three operators that stand around the optimizer step in a language model's training step and write the
gradients that it reads: the embedding lookup, layer norm, and the softmax cross entropy over the
vocabulary together with the classifier's product.  The cases go from calls where launch latency is all
there is to a whole training batch; sizes are generic.
"""
import math

import torch

own = False

IGNORED = -100
TYPES = {"half": torch.float16, "float": torch.float32}


def listed():
    return [
        # one short sequence looked up: latency
        {"name": "embedding_fwd_small", "op": "embedding", "pass": "fwd", "type": "half",
         "tokens": 64, "vocab": 32000, "dim": 512},
        # a whole training batch looked up
        {"name": "embedding_fwd_batch", "op": "embedding", "pass": "fwd", "type": "half",
         "tokens": 16384, "vocab": 50021, "dim": 2048},
        # fp32 table of odd width, as in a small model kept in fp32
        {"name": "embedding_bwd_float_odd", "op": "embedding", "pass": "bwd", "type": "float",
         "tokens": 1999, "vocab": 10007, "dim": 333},
        # a training batch's gradient: every row of the dense gradient is written, frequent tokens repeat
        {"name": "embedding_bwd_batch", "op": "embedding", "pass": "bwd", "type": "half",
         "tokens": 16384, "vocab": 50021, "dim": 2048},
        # one short sequence normalised: latency
        {"name": "layernorm_fwd_small", "op": "layernorm", "pass": "fwd", "type": "half", "params": "half",
         "rows": 64, "dim": 512},
        # a training batch, fp16 activations with fp32 parameters (the optimizer's fp32 group)
        {"name": "layernorm_fwd_batch", "op": "layernorm", "pass": "fwd", "type": "half", "params": "float",
         "rows": 16384, "dim": 4096},
        # fp32 activations of odd width
        {"name": "layernorm_bwd_float_odd", "op": "layernorm", "pass": "bwd", "type": "float", "params": "float",
         "rows": 4099, "dim": 1001},
        # the gradient of the training batch, with the sums over all rows
        {"name": "layernorm_bwd_batch", "op": "layernorm", "pass": "bwd", "type": "half", "params": "float",
         "rows": 16384, "dim": 4096},
        # a small classifier's loss and gradients: latency
        {"name": "vocab_loss_step_small", "op": "vocab_loss", "pass": "step", "type": "half",
         "tokens": 64, "vocab": 1000, "dim": 256, "ignored": 0.0},
        # evaluation: losses alone
        {"name": "vocab_loss_fwd_eval", "op": "vocab_loss", "pass": "fwd", "type": "half",
         "tokens": 4096, "vocab": 50021, "dim": 2048, "ignored": 0.0},
        # fine-tuning: prompts are ignored, odd counts
        {"name": "vocab_loss_step_odd", "op": "vocab_loss", "pass": "step", "type": "half",
         "tokens": 1001, "vocab": 50021, "dim": 1032, "ignored": 0.5},
        # a training batch under a large vocabulary
        {"name": "vocab_loss_step_batch", "op": "vocab_loss", "pass": "step", "type": "half",
         "tokens": 8192, "vocab": 128000, "dim": 4096, "ignored": 0.1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embedding", "layernorm", "vocab_loss"])
    if op == "embedding":
        return {"op": op, "pass": rng.choice(["fwd", "bwd"]), "type": rng.choice(["half", "float"]),
                "tokens": _log(rng, 1, 16384), "vocab": _log(rng, 100, 50021), "dim": _log(rng, 16, 1024)}
    if op == "layernorm":
        kind = rng.choice(["half", "float"])
        return {"op": op, "pass": rng.choice(["fwd", "bwd"]), "type": kind,
                "params": "float" if kind == "float" else rng.choice(["half", "float"]),
                "rows": _log(rng, 1, 16384), "dim": _log(rng, 16, 2048)}
    return {"op": op, "pass": rng.choice(["fwd", "step"]), "type": "half", "tokens": _log(rng, 1, 8192),
            "vocab": _log(rng, 100, 128000), "dim": 8 * _log(rng, 8, 512), "ignored": rng.choice([0.0, 0.1, 0.5])}


def work(case):
    size = 2 if case["type"] == "half" else 4
    if case["op"] == "embedding":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        rows = min(t, v) if case["pass"] == "fwd" else v
        return {"bytes": 8 * t + (t + rows) * d * size, "flops": t * d}
    if case["op"] == "layernorm":
        r, d, p = case["rows"], case["dim"], 2 if case["params"] == "half" else 4
        if case["pass"] == "fwd":
            return {"bytes": 2 * r * d * size + 2 * d * p + 8 * r, "flops": 8 * r * d}
        return {"bytes": 3 * r * d * size + 3 * d * p + 8 * r, "flops": 16 * r * d}
    t, v, d = case["tokens"], case["vocab"], case["dim"]
    inputs = (t + v) * d * size + 8 * t
    if case["pass"] == "fwd":
        return {"bytes": inputs + 8 * t, "flops": 2.0 * t * v * d}
    return {"bytes": inputs + 8 * t + (t + v) * d * size, "flops": 6.0 * t * v * d}


def _tokens(n, vocab, g):
    # a few tokens are frequent, most are rare: the logarithm of the rank is uniform
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab)).long() - 1).clamp_(0, vocab - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, mean=0.0, std=1.0, to=kind):
        return torch.empty(*shape, device="cuda").normal_(mean, std, generator=g).to(to)

    s = {"op": case["op"], "pass": case["pass"]}
    if case["op"] == "embedding":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        s |= {"ids": _tokens(t, v, g), "vocab": v, "scale": math.sqrt(d)}
        if case["pass"] == "fwd":
            s["weight"] = normal(v, d, std=0.02)
        else:
            s["grad_out"] = normal(t, d, std=1e-2)
    elif case["op"] == "layernorm":
        r, d = case["rows"], case["dim"]
        p = TYPES[case["params"]]
        s |= {"x": normal(r, d, mean=0.3, std=1.5), "gamma": normal(d, mean=1.0, std=0.1, to=p),
              "beta": normal(d, std=0.1, to=p), "eps": 1e-5}
        if case["pass"] == "bwd":
            s["grad_out"] = normal(r, d, std=0.1)
            x = s["x"].double()
            mean = x.mean(1)
            var = (x - mean[:, None]).square().mean(1)
            s |= {"mean": mean.float(), "rstd": (1.0 / torch.sqrt(var + s["eps"])).float()}
    else:
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        targets = _tokens(t, v, g)
        if case["ignored"]:
            targets[torch.rand(t, generator=g, device="cuda") < case["ignored"]] = IGNORED
        # the loss scale of mixed-precision training, where the optimizer step keeps it: on the device
        s |= {"hidden": normal(t, d), "weight": normal(v, d, std=0.02), "targets": targets,
              "loss_scale": torch.full((1,), 4096.0, device="cuda")}
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from saga_b200 import layers
    if s["op"] == "embedding":
        if s["pass"] == "fwd":
            return {"out": layers.embedding_forward(s["ids"], s["weight"], scale=s["scale"])}
        return {"grad_weight": layers.embedding_backward(s["ids"], s["grad_out"], s["vocab"], scale=s["scale"])}
    if s["op"] == "layernorm":
        if s["pass"] == "fwd":
            y, mean, rstd = layers.layernorm_forward(s["x"], s["gamma"], s["beta"], eps=s["eps"])
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dgamma, dbeta = layers.layernorm_backward(s["grad_out"], s["x"], s["gamma"], s["mean"], s["rstd"])
        return {"grad_x": dx, "grad_gamma": dgamma, "grad_beta": dbeta}
    loss, lse, stats = layers.vocab_loss_forward(s["hidden"], s["weight"], s["targets"])
    out = {"loss": loss, "lse": lse, "stats": stats}
    if s["pass"] == "step":
        out["grad_hidden"], out["grad_weight"] = layers.vocab_loss_backward(
            s["hidden"], s["weight"], s["targets"], lse, stats=stats, loss_scale=s["loss_scale"])
    return out


def _plain(s):
    if s["op"] == "embedding":
        if s["pass"] == "fwd":
            w = s["weight"]
            return {"out": (w[s["ids"]].float() * s["scale"]).to(w.dtype)}
        dy = s["grad_out"]
        total = torch.zeros(s["vocab"], dy.shape[1], device=dy.device).index_add_(0, s["ids"], dy.float())
        return {"grad_weight": (total * s["scale"]).to(dy.dtype)}
    if s["op"] == "layernorm":
        x, gamma = s["x"].float(), s["gamma"].float()
        if s["pass"] == "fwd":
            mean = x.mean(1)
            centred = x - mean[:, None]
            rstd = 1.0 / torch.sqrt(centred.square().mean(1) + s["eps"])
            y = centred * rstd[:, None] * gamma + s["beta"].float()
            return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
        dy = s["grad_out"].float()
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        dxhat = dy * gamma
        dx = s["rstd"][:, None] * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
        return {"grad_x": dx.to(s["x"].dtype), "grad_gamma": (dy * xhat).sum(0).to(s["gamma"].dtype),
                "grad_beta": dy.sum(0).to(s["gamma"].dtype)}
    x, w, y = s["hidden"].float(), s["weight"].float(), s["targets"]
    valid = (y >= 0) & (y < w.shape[0])
    at = torch.where(valid, y, 0)
    z = x @ w.t()
    top = z.amax(1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    loss = torch.where(valid, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    count = valid.sum().float()
    out = {"loss": loss, "lse": lse, "stats": torch.stack([loss.sum(), count])}
    if s["pass"] == "step":
        dz = torch.exp(z - lse[:, None])
        dz.scatter_add_(1, at[:, None], torch.full_like(lse, -1.0)[:, None])
        dz = dz * torch.where(valid, s["loss_scale"] / count.clamp(min=1.0), 0.0)[:, None]
        out["grad_hidden"] = (dz @ w).to(s["hidden"].dtype)
        out["grad_weight"] = (dz.t() @ x).to(s["weight"].dtype)
    return out


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    if s["op"] == "embedding":
        if s["pass"] == "fwd":
            return {"out": torch.index_select(s["weight"], 0, s["ids"]).double().mul_(s["scale"])}
        dy = s["grad_out"].double() * s["scale"]
        order = torch.argsort(s["ids"], stable=True)
        got = torch.zeros(s["vocab"], dy.shape[1], device="cuda", dtype=torch.float64)
        return {"grad_weight": got.index_put_((s["ids"][order],), dy[order], accumulate=True)}
    if s["op"] == "layernorm":
        x, gamma = s["x"].double(), s["gamma"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = torch.rsqrt(var + s["eps"])
        xhat = (x - mean.unsqueeze(1)).mul_(rstd.unsqueeze(1))
        if s["pass"] == "fwd":
            return {"y": torch.addcmul(s["beta"].double(), xhat, gamma), "mean": mean, "rstd": rstd}
        dy = s["grad_out"].double()
        d = x.shape[1]
        a = (dy @ gamma) / d
        b = torch.einsum("rd,rd,d->r", dy, xhat, gamma) / d
        dx = (dy * gamma - a.unsqueeze(1) - xhat * b.unsqueeze(1)) * rstd.unsqueeze(1)
        return {"grad_x": dx, "grad_gamma": torch.einsum("rd,rd->d", dy, xhat),
                "grad_beta": torch.ones(x.shape[0], device="cuda", dtype=torch.float64) @ dy}
    x, w, y = s["hidden"].double(), s["weight"].double(), s["targets"]
    rows = torch.nonzero(y != IGNORED)[:, 0]
    z = torch.mm(x, w.t())
    lse = torch.logsumexp(z, 1)
    loss = torch.zeros_like(lse)
    loss[rows] = lse[rows] - (x[rows] * w[y[rows]]).sum(1)
    count = float(rows.numel())
    out = {"loss": loss, "lse": lse,
           "stats": torch.stack([loss.sum(), torch.tensor(count, device="cuda", dtype=torch.float64)])}
    if s["pass"] == "step":
        p = z.sub_(lse.unsqueeze(1)).exp_()
        keep = torch.zeros_like(lse)
        keep[rows] = float(s["loss_scale"]) / max(count, 1.0)
        p.mul_(keep.unsqueeze(1))
        p[rows, y[rows]] -= keep[rows]
        out["grad_hidden"] = torch.mm(p, w)
        out["grad_weight"] = torch.mm(p.t(), x)
    return out

"""What is measured of the training-side operators: the vocabulary loss with its gradient, and the fused mixing rule + LayerNorm.

``linear_cross_entropy`` is the softmax cross entropy of a vocabulary projection (hidden states times a ``[V, D]`` weight) whose
logits are never kept; ``fuse_layer_norm`` is the residual or gate rule of a block followed by its LayerNorm, optionally with the
sum itself as a second output.  Every case runs one of them, forward alone or forward and backward."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token scored against the whole vocabulary: the call of a decoding loop that wants a log-likelihood
        loss_case("loss one token", 1, 512, 32768, "bf16", "none", False, 0.0, True),
        # evaluation of one 8192-token row: per-token negative log-likelihood, nothing differentiated
        loss_case("loss eval row", 8192, 512, 32768, "bf16", "none", False, 0.0, True),
        # a training step over two rows of 8192 tokens
        loss_case("loss step", 16384, 512, 32768, "bf16", "mean", True, 0.0, True),
        # the whole 8 x 8192 batch of the language-model configuration
        loss_case("loss step full batch", 65536, 512, 32768, "bf16", "mean", True, 0.0, True),
        # a padded batch with a small odd vocabulary and a width that is no multiple of anything
        loss_case("loss step ragged", 3001, 300, 10007, "bf16", "sum", True, 0.3, True),
        # full-precision training, per-token weights on the loss
        loss_case("loss step fp32", 2048, 512, 32768, "fp32", "none", True, 0.1, False),
        # the residual block of a decoding step: eight sequences, one token each
        norm_case("norm eight tokens", 8, 512, "bf16", False, False, False, False),
        # the gate rule between a layer and its retrieved state, whole batch, inference
        norm_case("norm gate forward", 65536, 512, "bf16", True, False, False, False),
        # the same in training
        norm_case("norm gate step", 65536, 512, "bf16", True, False, False, True),
        # a residual block with a residual scale that hands its sum on (a norm before the next block), full precision
        norm_case("norm residual step fp32", 16384, 1024, "fp32", False, True, True, True),
        # odd number of tokens, odd width
        norm_case("norm ragged step", 4099, 771, "bf16", True, True, False, True),
    ]


def loss_case(name, tokens, width, vocab, dtype, reduction, train, ignored, bias):
    return {"name": name, "op": "loss", "tokens": tokens, "width": width, "vocab": vocab, "dtype": dtype, "reduction": reduction,
            "train": train, "ignored": ignored, "bias": bias}


def norm_case(name, tokens, width, dtype, gate, scale, with_sum, train):
    return {"name": name, "op": "norm", "tokens": tokens, "width": width, "dtype": dtype, "gate": gate, "scale": scale,
            "with_sum": with_sum, "train": train}


def spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if rng.random() < 0.6:
        width = spread(rng, 33, 1100)
        if rng.random() < 0.5:
            width = max(64, width // 64 * 64)
        vocab = spread(rng, 500, 66000)
        # no dearer than the full batch of the language-model configuration; full precision costs several times as much
        most = 65536 * 512 * 32768 // (width * vocab) // (8 if dtype == "fp32" else 1)
        tokens = spread(rng, 1, max(1, min(65536, most)))
        case = loss_case("", tokens, width, vocab, dtype, rng.choice(["mean", "sum", "none"]), rng.random() < 0.7,
                         rng.choice([0.0, 0.0, 0.25]), rng.random() < 0.6)
    else:
        width = spread(rng, 17, 4100)
        if rng.random() < 0.5:
            width = max(8, width // 8 * 8)
        tokens = spread(rng, 1, max(1, min(70000, 65536 * 1024 // width)))
        case = norm_case("", tokens, width, dtype, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.7)
    del case["name"]
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    n, d = case["tokens"], case["width"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std

    state = {"case": case}
    if case["op"] == "loss":
        v = case["vocab"]
        # hidden states as a LayerNorm leaves them, weights that give logits of a standard deviation of about two
        state["hidden"] = normal(n, d).to(dt)
        state["weight"] = normal(v, d, std=2.0 / math.sqrt(d)).to(dt)
        state["bias"] = normal(v, std=0.5).to(dt) if case["bias"] else None
        # Zipf-distributed words (exponent 1.1)
        cdf = torch.cumsum(torch.arange(1, v + 1, device="cuda", dtype=torch.float64) ** -1.1, 0)
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64) * cdf[-1]
        targets = torch.searchsorted(cdf, u).clamp_(max=v - 1)
        skip = torch.rand(n, device="cuda", generator=g) < case["ignored"]
        if n > 1:
            skip[0] = False                       # a mean needs a token to count
        else:
            skip[:] = False
        state["targets"] = torch.where(skip, torch.full_like(targets, -100), targets)
        # per-token weights of the loss (what a user multiplies the unreduced losses by)
        state["grad"] = torch.rand(n, device="cuda", generator=g) * 2.0 / n
        leaves = ["hidden", "weight", "bias"]
    else:
        state["online"] = normal(n, d).to(dt)
        state["update"] = normal(n, d, std=0.7).to(dt)
        state["gate"] = normal(n, d, std=1.5).to(dt) if case["gate"] else None
        state["scale"] = (1.0 + normal(d, std=0.2)).to(dt) if case["scale"] else None
        state["weight"] = (1.0 + normal(d, std=0.1)).to(dt)
        state["bias"] = normal(d, std=0.1).to(dt)
        state["grad"] = normal(n, d).to(dt)
        state["grad_sum"] = normal(n, d).to(dt) if case["with_sum"] else None
        leaves = ["online", "update", "gate", "scale", "weight", "bias"]
    state["leaves"] = [k for k in leaves if state[k] is not None]
    if case["train"]:
        for k in state["leaves"]:
            state[k].requires_grad_(True)
    return state


def run(state):
    if state["case"]["op"] == "loss":
        return own_loss(state) if own else plain_loss(state)
    return own_norm(state) if own else plain_norm(state)


# ---- the framework's operators, as a program calls them ----

def own_loss(s):
    from rnn_with_grm_b200.loss import linear_cross_entropy

    c = s["case"]
    loss = linear_cross_entropy(s["hidden"], s["weight"], s["targets"], s["bias"], reduction=c["reduction"])
    out = {"loss": loss.detach()}
    if c["train"]:
        upstream = s["grad"] if c["reduction"] == "none" else None
        for k, grad in zip(s["leaves"], torch.autograd.grad(loss, [s[k] for k in s["leaves"]], upstream)):
            out["d_" + k] = grad
    return out


def own_norm(s):
    from rnn_with_grm_b200.fusion import fuse_layer_norm

    c = s["case"]
    got = fuse_layer_norm(s["online"], s["update"], s["weight"], s["bias"], gate=s["gate"], scale=s["scale"], eps=1e-5,
                          return_sum=c["with_sum"])
    got = got if c["with_sum"] else (got,)
    out = {"y": got[0].detach()}
    if c["with_sum"]:
        out["sum"] = got[1].detach()
    if c["train"]:
        upstream = [s["grad"], s["grad_sum"]][: len(got)]
        for k, grad in zip(s["leaves"], torch.autograd.grad(got, [s[k] for k in s["leaves"]], upstream)):
            out["d_" + k] = grad
    return out


# ---- the plain forms ----

@torch.no_grad()
def plain_loss(s):
    c = s["case"]
    dt, n = s["hidden"].dtype, c["tokens"]
    x, w, t = s["hidden"].float(), s["weight"].float(), s["targets"]
    valid = t >= 0
    at = t.clamp(min=0).unsqueeze(1)
    logits = x @ w.T
    if s["bias"] is not None:
        logits = logits + s["bias"].float()
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    nll = torch.where(valid, (total.log() + top - picked).squeeze(1), torch.zeros_like(total).squeeze(1))
    count = valid.sum()
    if c["reduction"] == "none":
        loss, g = nll, s["grad"]
    elif c["reduction"] == "sum":
        loss, g = nll.sum(), torch.ones(n, device=x.device)
    else:
        loss, g = nll.sum() / count, torch.ones(n, device=x.device) / count
    out = {"loss": loss}
    if c["train"]:
        p = p.div_(total)
        p.scatter_add_(1, at, torch.full_like(total, -1.0))
        p.mul_((g * valid).unsqueeze(1))
        out["d_hidden"] = (p @ w).to(dt)
        out["d_weight"] = (p.T @ x).to(dt)
        if s["bias"] is not None:
            out["d_bias"] = p.sum(0).to(dt)
    return out


@torch.no_grad()
def plain_norm(s):
    c = s["case"]
    dt = s["online"].dtype
    a, b, w, beta = s["online"].float(), s["update"].float(), s["weight"].float(), s["bias"].float()
    scale = s["scale"].float() if s["scale"] is not None else None
    u = b * scale if scale is not None else b
    if s["gate"] is not None:
        gate = 1.0 / (1.0 + torch.exp(-s["gate"].float()))
        total = gate * a + (1.0 - gate) * u
    else:
        total = a + u
    centred = total - total.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    xh = centred * rstd
    out = {"y": (xh * w + beta).to(dt)}
    if c["with_sum"]:
        out["sum"] = total.to(dt)
    if c["train"]:
        dy = s["grad"].float()
        dxh = dy * w
        ds = rstd * (dxh - dxh.mean(1, keepdim=True) - xh * (dxh * xh).mean(1, keepdim=True))
        if c["with_sum"]:
            ds = ds + s["grad_sum"].float()
        du = ds
        out["d_online"] = ds
        if s["gate"] is not None:
            out["d_gate"] = (ds * (a - u) * gate * (1.0 - gate)).to(dt)
            out["d_online"] = ds * gate
            du = ds * (1.0 - gate)
        out["d_online"] = out["d_online"].to(dt)
        out["d_update"] = (du * scale if scale is not None else du).to(dt)
        if scale is not None:
            out["d_scale"] = (du * b).sum(0).to(dt)
        out["d_weight"] = (dy * xh).sum(0).to(dt)
        out["d_bias"] = dy.sum(0).to(dt)
    return out


# ---- what a pass cannot do without ----

def work(case):
    n, d, e = case["tokens"], case["width"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "loss":
        v = case["vocab"]
        tensors = (n * d + v * d + (v if case["bias"] else 0)) * e
        losses = 4 * n if case["reduction"] == "none" else 4
        if case["train"]:
            return {"bytes": 2 * tensors + 8 * n + losses + (4 * n if case["reduction"] == "none" else 0), "flops": 6 * n * v * d}
        return {"bytes": tensors + 8 * n + losses, "flops": 2 * n * v * d}
    rows = 2 + case["gate"]
    vectors = 2 + case["scale"]
    outs = 1 + case["with_sum"]
    moved = (rows + outs) * n * d * e + vectors * d * e
    flops = (12 + 6 * case["gate"]) * n * d
    if case["train"]:
        moved += (rows + outs) * n * d * e + vectors * d * e
        flops += (20 + 8 * case["gate"]) * n * d
    return {"bytes": moved, "flops": flops}


# ---- the definitions, in 64 bits ----

@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return exact_loss(state, case) if case["op"] == "loss" else exact_norm(state, case)


def exact_loss(state, case):
    """Token block by token block: log-sum-exp of the scores, then the gradient of each reduced loss by the chain rule."""
    x, w, t = state["hidden"].detach().double(), state["weight"].detach().double(), state["targets"]
    b = torch.zeros(case["vocab"], device=x.device, dtype=torch.float64) if state["bias"] is None else state["bias"].detach().double()
    keep = t != -100
    if case["reduction"] == "none":
        upstream = state["grad"].double()
    else:
        upstream = torch.ones_like(t, dtype=torch.float64) / (keep.sum() if case["reduction"] == "mean" else 1)
    upstream = torch.where(keep, upstream, torch.zeros_like(upstream))
    losses, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for block in torch.arange(case["tokens"], device=x.device).split(8192):
        z = torch.addmm(b, x[block], w.T)
        lse = torch.logsumexp(z, dim=1)
        word = t[block].clamp(min=0)
        losses.append(torch.where(keep[block], lse - z[torch.arange(len(block), device=x.device), word], torch.zeros_like(lse)))
        if case["train"]:
            z = torch.exp(z - lse[:, None])
            z[torch.arange(len(block), device=x.device), word] -= 1.0
            z *= upstream[block, None]
            dx.append(z @ w)
            dw += z.T @ x[block]
            db += z.sum(dim=0)
    loss = torch.cat(losses)
    if case["reduction"] != "none":
        loss = loss.sum() / (keep.sum() if case["reduction"] == "mean" else 1)
    out = {"loss": loss}
    if case["train"]:
        out.update(d_hidden=torch.cat(dx), d_weight=dw)
        if state["bias"] is not None:
            out["d_bias"] = db
    return out


def exact_norm(state, case):
    """The mixing rule and the normalisation in 64 bits, differentiated by autograd."""
    with torch.enable_grad():
        wide = {k: state[k].detach().double().requires_grad_(case["train"]) for k in state["leaves"]}
        update = wide["update"] * wide["scale"] if case["scale"] else wide["update"]
        if case["gate"]:
            total = update + torch.sigmoid(wide["gate"]) * (wide["online"] - update)
        else:
            total = wide["online"] + update
        var, mean = torch.var_mean(total, dim=1, unbiased=False, keepdim=True)
        y = (total - mean) / (var + 1e-5).sqrt() * wide["weight"] + wide["bias"]
        out = {"y": y.detach()}
        value = (y * state["grad"].double()).sum() if case["train"] else None
        if case["with_sum"]:
            out["sum"] = total.detach()
            value = value + (total * state["grad_sum"].double()).sum() if case["train"] else None
        if case["train"]:
            for k, grad in zip(state["leaves"], torch.autograd.grad(value, [wide[k] for k in state["leaves"]])):
                out["d_" + k] = grad
    return out

"""Cases of the training operators of large models: the orthogonalised update (Newton-Schulz), the optimizer step built on
it, and the balance loss of a gate with its counts and gradient.

`run` computes them in plain torch operations, or, where `own` is true, through the framework's entry points."""
import math

import torch

own = False

# the quintic of the orthogonalisation and its number of steps: the usual choice for momentum updates
A, B, C, STEPS, EPS = 3.4445, -4.7750, 2.0315, 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one node layer of a 68-node decoder: latency of a single small matrix
        {"name": "ortho 68x68", "op": "orthogonalize", "batch": 1, "rows": 68, "cols": 68, "dtype": "fp32"},
        # the hidden layers of a multi-branch decoder, eight residual blocks of two layers, stacked
        {"name": "ortho 16x512x512", "op": "orthogonalize", "batch": 16, "rows": 512, "cols": 512, "dtype": "fp32"},
        # first encoder layer of a 68-node model, gradients kept in 16 bits
        {"name": "ortho 1024x4624 bf16", "op": "orthogonalize", "batch": 1, "rows": 1024, "cols": 4624, "dtype": "bf16"},
        # output layer of the conditional model: more rows than columns
        {"name": "ortho 4624x1024", "op": "orthogonalize", "batch": 1, "rows": 4624, "cols": 1024, "dtype": "fp32"},
        # the dense intercept of a 68-node decoder: the largest matrix there is
        {"name": "ortho 4624x4624", "op": "orthogonalize", "batch": 1, "rows": 4624, "cols": 4624, "dtype": "fp32"},
        # the matrices of the gated mixture model at 87 nodes: two large, the rest small, odd widths
        {"name": "muon mixture 87", "op": "muon_step", "model": "mixture", "nodes": 87, "hidden": 1024, "inner": 128, "latent": 68,
         "neighbours": 32, "channels": 5, "layers": 3, "dtype": "fp32", "nesterov": True},
        # the same model's decoder alone (its encoder frozen): twenty small matrices, where launches count
        {"name": "muon decoder 68", "op": "muon_step", "model": "decoder", "nodes": 68, "hidden": 0, "inner": 0, "latent": 68,
         "neighbours": 32, "channels": 5, "layers": 3, "dtype": "fp32", "nesterov": False},
        # the kernels of the conv encoder, output channels x (input channels x taps), and its two heads, weights in 16 bits
        {"name": "muon conv 48 bf16", "op": "muon_step", "model": "conv", "nodes": 0, "hidden": 48, "inner": 0, "latent": 68,
         "neighbours": 0, "channels": 5, "layers": 0, "dtype": "bf16", "nesterov": True},
        # the gate of the mixture at the scripts' batch: latency
        {"name": "gate 256x5", "op": "gate", "rows": 256, "experts": 5, "top": 1, "dtype": "fp32", "masked": False},
        # the same at the benchmark's batch
        {"name": "gate 16384x5", "op": "gate", "rows": 16384, "experts": 5, "top": 1, "dtype": "fp32", "masked": False},
        # a padded batch through a gate over many components, several taken per row
        {"name": "gate 32771x60 top 6 bf16", "op": "gate", "rows": 32771, "experts": 60, "top": 6, "dtype": "bf16", "masked": True},
        # the widest gate on a large batch
        {"name": "gate 262144x256 top 8", "op": "gate", "rows": 262144, "experts": 256, "top": 8, "dtype": "fp32", "masked": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("orthogonalize", "muon_step", "gate"))
    dtype = rng.choice(("fp32", "bf16"))
    if op == "orthogonalize":
        rows, cols = _log(rng, 16, 4624), _log(rng, 16, 4624)
        batch = _log(rng, 1, 16) if rows * cols <= 512 * 1024 else 1
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}
    if op == "muon_step":
        model = rng.choice(("mixture", "decoder", "conv"))
        case = {"op": op, "model": model, "nodes": 0, "hidden": 0, "inner": 0, "latent": rng.randint(8, 96), "neighbours": 0,
                "channels": rng.randint(1, 5), "layers": 0, "dtype": dtype, "nesterov": rng.random() < 0.5}
        if model == "conv":
            case["hidden"] = _log(rng, 8, 48)
        else:
            case["nodes"], case["layers"] = _log(rng, 16, 87), rng.randint(1, 3)
            case["neighbours"] = rng.randint(4, case["nodes"])
            if model == "mixture":
                case["hidden"], case["inner"] = _log(rng, 64, 1024), _log(rng, 16, 256)
        return case
    experts = _log(rng, 2, 256)
    return {"op": op, "rows": _log(rng, 1, 262144), "experts": experts, "top": rng.randint(1, min(8, experts)), "dtype": dtype,
            "masked": rng.random() < 0.5}


def _shapes(case):
    """The matrices an optimizer step goes over, as (rows, columns)."""
    if case["model"] == "conv":
        d, r = case["hidden"], case["channels"]
        return [(d, 49), (2 * d, 9 * d), (4 * d, 18 * d)] + [(4 * d, 36 * d)] * (2 * r) + [(case["latent"], 16 * d)] * 2
    n, h, i, z = case["nodes"], case["hidden"], case["inner"], case["latent"]
    decoder = [(n, z)] * case["channels"] + [(n, case["neighbours"])] * (case["channels"] * case["layers"])
    return decoder if case["model"] == "decoder" else [(h, n * n)] * 2 + [(i, h)] * 2 + [(z, i)] * 2 + decoder


def _gradient(batch, rows, cols, gen):
    """What a backward pass leaves: a few strong directions of falling weight, and noise in all the others."""
    dev = gen.device
    r = min(64, rows, cols)
    weight = torch.arange(1, r + 1, device=dev, dtype=torch.float32).pow(-0.5)
    u = torch.randn(batch, rows, r, device=dev, generator=gen) * weight
    v = torch.randn(batch, r, cols, device=dev, generator=gen)
    return 1e-3 * (torch.bmm(u, v) + 0.3 * torch.randn(batch, rows, cols, device=dev, generator=gen))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    state = dict(case)
    if case["op"] == "orthogonalize":
        state["x"] = _gradient(case["batch"], case["rows"], case["cols"], gen).to(DTYPES[case["dtype"]])
    elif case["op"] == "muon_step":
        dt = DTYPES[case["dtype"]]
        state["params"], state["grads"], state["momenta"] = [], [], []
        for rows, cols in _shapes(case):
            bound = 1.0 / math.sqrt(cols)
            p = torch.empty(rows, cols, device=dev).uniform_(-bound, bound, generator=gen)
            state["params"].append(p.to(dt))
            state["grads"].append(_gradient(1, rows, cols, gen)[0].to(dt))
            state["momenta"].append(4.0 * _gradient(1, rows, cols, gen)[0])
    else:
        t, e = case["rows"], case["experts"]
        bias = torch.randn(e, device=dev, generator=gen)                 # some experts are liked by most rows
        state["logits"] = (1.5 * torch.randn(t, e, device=dev, generator=gen) + bias).to(DTYPES[case["dtype"]])
        state["valid"] = None
        if case["masked"]:                                                # the batch's tail and some rows within are padding
            valid = torch.rand(t, device=dev, generator=gen) < 0.9
            valid[t - t // 8:] = False
            state["valid"] = valid
    return state


# ---- plain forms --------------------------------------------------------------------------------------------------
def _orthogonalize(g):
    """[batch, rows, cols] in 32 bits -> the same shape."""
    x = g.transpose(1, 2).contiguous() if g.shape[1] > g.shape[2] else g
    norm = x.double().square().sum(dim=(1, 2), keepdim=True).sqrt()
    x = x / norm.clamp(min=EPS).float()
    for _ in range(STEPS):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = A * x + torch.bmm(B * gram + C * torch.bmm(gram, gram), x)
    return x.transpose(1, 2).contiguous() if g.shape[1] > g.shape[2] else x


def _muon_step(state):
    params, grads, momenta = state["params"], state["grads"], state["momenta"]
    groups = {}
    for i, p in enumerate(params):
        groups.setdefault(tuple(p.shape), []).append(i)
    for (rows, cols), at in groups.items():                              # matrices of one shape go through the products together
        g = torch.stack([grads[i] for i in at]).float()
        m = torch.stack([momenta[i] for i in at]) * MOMENTUM + g
        o = _orthogonalize(g + MOMENTUM * m if state["nesterov"] else m)
        p = torch.stack([params[i] for i in at]).float()
        p = p * (1.0 - LR * DECAY) - (LR * math.sqrt(max(1.0, rows / cols))) * o
        for j, i in enumerate(at):
            params[i].copy_(p[j])
            momenta[i].copy_(m[j])


def _gate(state):
    logits, valid, top = state["logits"], state["valid"], state["top"]
    t, e = logits.shape
    z = logits.float()
    rows = torch.ones(t, dtype=torch.bool, device=z.device) if valid is None else valid
    z = torch.where(rows[:, None], z, torch.zeros_like(z))
    w = torch.exp(z - z.max(dim=1, keepdim=True).values)
    prob = w / w.sum(dim=1, keepdim=True)
    prob = torch.where(rows[:, None], prob, torch.zeros_like(prob))
    taken = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    taken = torch.where(rows[:, None], taken, torch.full_like(taken, e))   # a padded row takes none
    counts = (taken.reshape(-1, 1) == torch.arange(e, device=z.device)).sum(dim=0) if t * top * e <= 1 << 24 else \
        torch.bincount(taken.reshape(-1), minlength=e + 1)[:e]
    n = rows.sum().clamp(min=1).double()
    mean = prob.sum(dim=0, dtype=torch.float64) / n
    share = counts.double() * (e / (top * n))
    loss = (share * mean).sum()
    slope = ((share - share.mean()) / n).float()                         # less their mean, which the softmax takes out anyway
    grad = prob * (slope - (prob * slope).sum(dim=1, keepdim=True))
    return {"loss": loss.float(), "counts": counts.to(torch.int32), "mean_probs": mean.float(), "grad": grad.to(logits.dtype)}


# ---- the framework's entry points ---------------------------------------------------------------------------------
def _own(state):
    import mdnvae_amd as M
    if state["op"] == "orthogonalize":
        return M.ops.orthogonalize(state["x"])
    if state["op"] == "muon_step":
        M.ops.muon_step(state["params"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM, nesterov=state["nesterov"],
                        weight_decay=DECAY)
        return state["params"], state["momenta"]
    loss, counts, mean_probs, grad = M.ops.gate_balance_loss_and_grads(state["logits"], top_k=state["top"], valid=state["valid"])
    return {"loss": loss, "counts": counts, "mean_probs": mean_probs, "grad": grad}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "orthogonalize":
        return _orthogonalize(state["x"].float()).to(state["x"].dtype)
    if state["op"] == "muon_step":
        _muon_step(state)
        return state["params"], state["momenta"]
    return _gate(state)


# ---- what one pass cannot do without ------------------------------------------------------------------------------
def _ortho_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m ** 3 + 2 * m * m * n)                  # the two symmetric products at half their entries


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "orthogonalize":
        entries = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * size * entries, "flops": case["batch"] * _ortho_flops(case["rows"], case["cols"])}
    if case["op"] == "muon_step":
        shapes = _shapes(case)
        return {"bytes": sum(r * c for r, c in shapes) * (3 * size + 8), "flops": sum(_ortho_flops(r, c) for r, c in shapes)}
    entries = case["rows"] * case["experts"]
    return {"bytes": 2 * size * entries + (case["rows"] if case["masked"] else 0), "flops": 12 * entries}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _exact_polar(g):
    g = g.double()
    tall = g.shape[0] > g.shape[1]
    x = g.t().contiguous() if tall else g.clone()
    x /= max(float(torch.linalg.vector_norm(x)), EPS)
    for _ in range(STEPS):
        s = torch.mm(x, x.t())
        q = C * torch.mm(s, s)
        q += B * s
        q.diagonal().add_(A)
        x = torch.mm(q, x)
    return x.t().contiguous() if tall else x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalize":
        return torch.stack([_exact_polar(x) for x in state["x"]])
    if case["op"] == "muon_step":
        params, momenta = [], []
        for p, g, m in zip(state["params"], state["grads"], state["momenta"]):
            m = m.double() * MOMENTUM + g.double()
            o = _exact_polar(g.double() + MOMENTUM * m if case["nesterov"] else m)
            s = LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            params.append(p.double() * (1.0 - LR * DECAY) - s * o)
            momenta.append(m)
        return params, momenta
    z = state["logits"].double()
    t, e = z.shape
    keep = torch.arange(t, device=z.device) if state["valid"] is None else state["valid"].nonzero()[:, 0]
    z = z[keep]
    n = max(1, z.shape[0])
    prob = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    counts = torch.zeros(e, dtype=torch.float64, device=z.device)
    left = z.clone()
    for _ in range(case["top"]):
        best = left.argmax(dim=1, keepdim=True)
        counts += torch.bincount(best[:, 0], minlength=e)
        left.scatter_(1, best, -math.inf)
    mean = prob.sum(dim=0) / n
    factor = e / (case["top"] * n)
    grad = torch.zeros(t, e, dtype=torch.float64, device=z.device)
    grad[keep] = prob * (counts - (prob @ counts)[:, None]) * (factor / n)
    return {"loss": factor * (counts @ mean), "counts": None, "mean_probs": mean, "grad": grad}

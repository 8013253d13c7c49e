"""What is measured of the operators around a network's last matrix product (alphazero_amd.head): the loss of a linear layer
over many classes with its gradient, dropout from a counter-based generator, and the product in 8-bit integers.

`own` False computes them from elementary torch operations in 32 bits; `own` True calls alphazero_amd.head."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_M32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one training batch of the 9x9 network's policy head: 256 positions, 2 * 81 features, 82 actions, targets from visit
        # counts, entropy bonus; launch latency is what counts
        {"name": "loss policy 9x9 f32", "op": "loss", "type": "f32", "rows": 256, "features": 162, "classes": 82, "target": "dense",
         "bias": True, "entropy": 1e-3, "train": True},
        # a large batch of the 19x19 head in half precision (automatic mixed precision), 2 * 361 features, 362 actions
        {"name": "loss policy 19x19 f16", "op": "loss", "type": "f16", "rows": 4096, "features": 722, "classes": 362, "target": "dense",
         "bias": True, "entropy": 1e-3, "train": True},
        # evaluation (no gradient) over a mid-sized class set in float32
        {"name": "loss eval f32", "op": "loss", "type": "f32", "rows": 2000, "features": 1024, "classes": 32000, "target": "index",
         "bias": False, "entropy": 0.0, "train": False},
        # a training batch over an odd number of classes with padded rows
        {"name": "loss ragged classes bf16", "op": "loss", "type": "bf16", "rows": 4095, "features": 2048, "classes": 50021, "target": "index",
         "bias": True, "entropy": 0.0, "train": True},
        # the largest: 8192 tokens, 131072 classes
        {"name": "loss large bf16", "op": "loss", "type": "bf16", "rows": 8192, "features": 4096, "classes": 131072, "target": "index",
         "bias": False, "entropy": 0.0, "train": True},
        # dropout in front of the 9x9 policy head, forward and backward
        {"name": "dropout 9x9 head f32", "op": "dropout", "type": "f32", "rows": 256, "features": 162, "p": 0.1, "residual": False, "train": True},
        # dropout joined with the residual of a block, forward and backward
        {"name": "dropout residual bf16", "op": "dropout", "type": "bf16", "rows": 8192, "features": 4096, "p": 0.1, "residual": True, "train": True},
        # a long ragged activation, forward alone
        {"name": "dropout long f16", "op": "dropout", "type": "f16", "rows": 65521, "features": 4099, "p": 0.25, "residual": False, "train": False},
        # one token at a time: the weights' bytes are what counts
        {"name": "int8 one token bf16", "op": "int8", "type": "bf16", "rows": 1, "features": 4096, "outputs": 16384, "bias": False},
        # a ragged handful of tokens
        {"name": "int8 37 tokens f16", "op": "int8", "type": "f16", "rows": 37, "features": 2000, "outputs": 5003, "bias": True},
        # first value layer of the 19x19 network with 256 channels: 64 * 361 features to 256 hidden units
        {"name": "int8 value head f32", "op": "int8", "type": "f32", "rows": 256, "features": 23104, "outputs": 256, "bias": True},
        # a prompt of 8192 tokens
        {"name": "int8 prompt bf16", "op": "int8", "type": "bf16", "rows": 8192, "features": 8192, "outputs": 8192, "bias": False},
    ]


def _span(rng, low, high):
    """A whole number between low and high, spread over its logarithm; two in three are odd."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n | 1 if rng.random() < 0.67 else n))


def draw(rng):
    op, kind = rng.choice(["loss", "loss", "dropout", "int8"]), rng.choice(["f32", "bf16", "f16"])
    if op == "loss":
        dense = rng.random() < 0.4
        rows, train = _span(rng, 1, 8192), rng.random() < 0.75
        features, classes = _span(rng, 64, 4096), _span(rng, 26, 4001 if dense else 131072)
        if rows * features * classes > 1 << 40:   # a float32 plain form of the whole range would take too long: thin the rows
            rows = max(1, (1 << 40) // (features * classes))
        return {"op": op, "type": kind, "rows": rows, "features": features, "classes": classes, "target": "dense" if dense else "index",
                "bias": rng.random() < 0.5, "entropy": rng.choice([0.0, 1e-3, 0.01]), "train": train}
    if op == "dropout":
        return {"op": op, "type": kind, "rows": _span(rng, 1, 32768), "features": _span(rng, 64, 4101), "p": rng.choice([0.05, 0.1, 0.25, 0.5]),
                "residual": rng.random() < 0.5, "train": rng.random() < 0.6}
    return {"op": op, "type": kind, "rows": _span(rng, 1, 8192), "features": _span(rng, 82, 8192), "outputs": _span(rng, 64, 8192), "bias": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, feats = _TYPES[case["type"]], case["rows"], case["features"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std)

    state = {"case": case}
    if case["op"] == "loss":
        classes = case["classes"]
        weight = normal(classes, feats, std=2.0 / math.sqrt(feats))
        x = normal(rows, feats)
        index = torch.randint(classes, (rows,), generator=gen, device="cuda")
        # a network in training knows some answers: the features lean towards their class, at most to 0.6 of log(classes) in its logit
        x += weight[index] * (0.15 * math.log(classes) * torch.rand((rows, 1), generator=gen, device="cuda"))
        if case["target"] == "dense":   # visit counts: most moves never, some often, summing to one
            visits = torch.exp(2.0 * normal(rows, classes)) * (torch.rand((rows, classes), generator=gen, device="cuda") < 0.4)
            visits.scatter_add_(1, index[:, None], torch.full((rows, 1), 5.0, device="cuda"))
            state["target"] = visits / visits.sum(1, keepdim=True)
        else:                           # one row in ten is padding
            state["target"] = torch.where(torch.rand((rows,), generator=gen, device="cuda") < 0.1, -100, index)
            state["target"][0] = index[0]
        state["x"], state["weight"] = x.to(kind), weight.to(kind)
        state["bias"] = normal(classes, std=0.3).to(kind) if case["bias"] else None
        # half precision is trained with a scaled loss
        state["scale"] = torch.full((), 4096.0 if case["type"] == "f16" else 1.0, device="cuda")
        if case["train"]:
            for name in ("x", "weight", "bias"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    if case["op"] == "dropout":
        state["x"] = normal(rows, feats).to(kind).requires_grad_(case["train"])
        state["residual"] = normal(rows, feats).to(kind).requires_grad_(case["train"]) if case["residual"] else None
        state["grad"] = normal(rows, feats).to(kind) if case["train"] else None
        state["seed"], state["offset"] = (seed * 0x9E3779B97F4A7C15 + 1) % (1 << 64), seed % 1000
        return state
    x = normal(rows, feats)
    x = x * torch.exp(0.5 * normal(rows, 1))
    weight = normal(case["outputs"], feats, std=1.0 / math.sqrt(feats)) * torch.exp(0.3 * normal(case["outputs"], 1))
    top = weight.abs().amax(1)          # the weights a user keeps: quantised once, a scale for each output channel
    state["qweight"] = torch.round(weight.double() * 127.0 / top[:, None].double()).to(torch.int8)
    state["wscale"] = top / 127.0
    state["x"] = x.to(kind)
    state["bias"] = normal(case["outputs"], std=0.3).to(kind) if case["bias"] else None
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_loss(x, weight, bias, target, entropy, scale, train):
    """Cross entropy minus entropy * H(softmax) of each row; in training its mean over the rows that count, and the gradients of
    `scale` times that."""
    xf, wf = x.detach().float(), weight.detach().float()
    logits = xf @ wf.t()
    if bias is not None:
        logits += bias.detach().float()
    top = logits.amax(1, keepdim=True)
    logp = logits - (top + torch.log(torch.exp(logits - top).sum(1, keepdim=True)))
    prob = torch.exp(logp)
    if target.dim() == 1:
        counts = target != -100
        row = -logp.gather(1, target.clamp(min=0)[:, None])[:, 0]
        total = 1.0
    else:
        counts = torch.ones(target.shape[0], dtype=torch.bool, device=target.device)
        row = -(target * logp).sum(1)
        total = target.sum(1, keepdim=True)
    n = counts.sum()
    if entropy:
        h = -(prob * logp).sum(1)
        row = row - entropy * h
    row = torch.where(counts, row, 0.0)
    if not train:
        return row
    g = prob * total
    if entropy:
        g += entropy * prob * (logp + h[:, None])
    if target.dim() == 1:
        g[torch.arange(g.shape[0], device=g.device), target.clamp(min=0)] -= 1.0
    else:
        g -= target
    g = torch.where(counts[:, None], g, 0.0) * (scale / n)
    out = [row.sum() / n, (g @ wf).to(x.dtype), (g.t() @ xf).to(weight.dtype)]
    if bias is not None:
        out.append(g.sum(0).to(bias.dtype))
    return out


def _philox(group, seed, offset):
    """Philox4x32-10 (Salmon et al. 2011) of the counters (group, offset) under the key `seed`: four 32-bit words each."""
    def product(a, b):
        low = (a * b) & _M32
        return ((a >> 16) * b + (((a & 0xFFFF) * b) >> 16)) >> 16, low

    c0, c1 = group & _M32, group >> 32
    c2, c3 = torch.full_like(group, offset & _M32), torch.full_like(group, offset >> 32)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        h0, l0 = product(c0, 0xD2511F53)
        h1, l1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), 1)


def _kept(shape, p, seed, offset, device):
    """Element i is kept where the 16 bits i % 8 of the words of group i // 8 reach round(65536 p)."""
    n = math.prod(shape)
    words = _philox(torch.arange((n + 7) // 8, device=device), seed, offset)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
    return (bits >= round(65536 * p)).reshape(shape)


def _plain_dropout(x, residual, grad, p, seed, offset):
    kept = _kept(x.shape, p, seed, offset, x.device)
    scale = 65536 / (65536 - round(65536 * p))
    y = torch.where(kept, x.detach().float() * scale, 0.0)
    if residual is not None:
        y += residual.detach().float()
    y = y.to(x.dtype)
    if grad is None:
        return y
    gx = torch.where(kept, grad.float() * scale, 0.0).to(x.dtype)
    return [y, gx] if residual is None else [y, gx, grad]


def _plain_int8(x, qweight, wscale, bias):
    top = x.float().abs().amax(1)
    # the nearest whole number of 127 x / top: in 64 bits, where a quotient next to a half is told from one at it
    q = torch.round(x.double() * 127.0 / torch.where(top > 0, top, 1.0)[:, None].double())
    y = q.float() @ qweight.float().t()
    y = y * (top / 127.0)[:, None] * wscale[None, :]
    if bias is not None:
        y += bias.float()
    return y.to(x.dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        from alphazero_amd import head
        if case["op"] == "loss":
            loss = head.linear_cross_entropy(state["x"], state["weight"], state["target"], state["bias"], entropy_coeff=case["entropy"],
                                             reduction="mean" if case["train"] else "none")
            if not case["train"]:
                return loss
            leaves = [state[k] for k in ("x", "weight", "bias") if state[k] is not None]
            return [loss.detach(), *torch.autograd.grad(loss, leaves, state["scale"])]
        if case["op"] == "dropout":
            y = head.dropout(state["x"], case["p"], state["seed"], state["offset"], residual=state["residual"])
            if not case["train"]:
                return y
            leaves = [state[k] for k in ("x", "residual") if state[k] is not None]
            return [y.detach(), *torch.autograd.grad(y, leaves, state["grad"])]
        return head.int8_linear(state["x"], state["qweight"], state["wscale"], state["bias"])
    if case["op"] == "loss":
        return _plain_loss(state["x"], state["weight"], state["bias"], state["target"], case["entropy"], state["scale"], case["train"])
    if case["op"] == "dropout":
        return _plain_dropout(state["x"], state["residual"], state["grad"], case["p"], state["seed"], state["offset"])
    return _plain_int8(state["x"], state["qweight"], state["wscale"], state["bias"])


def work(case):
    size, rows, feats = _BYTES[case["type"]], case["rows"], case["features"]
    if case["op"] == "loss":
        classes = case["classes"]
        inputs = size * (rows * feats + classes * feats + (classes if case["bias"] else 0))
        target = 4 * rows * classes if case["target"] == "dense" else 8 * rows
        return {"bytes": inputs * (2 if case["train"] else 1) + target + 4 * (1 if case["train"] else rows), "flops": (6 if case["train"] else 2) * rows * feats * classes}
    if case["op"] == "dropout":
        arrays = 2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)
        return {"bytes": arrays * size * rows * feats, "flops": (2 if case["train"] else 1) * rows * feats}
    outputs = case["outputs"]
    return {"bytes": size * rows * (feats + outputs) + outputs * (feats + 4 + (size if case["bias"] else 0)), "flops": 2 * rows * feats * outputs}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].detach().double()
    if case["op"] == "loss":
        with torch.enable_grad():   # the loss by its definition, its gradient by differentiation; rows in pieces, so that it fits
            leaf_x, leaf_w = x.requires_grad_(True), state["weight"].detach().double().requires_grad_(True)
            leaf_b = None if state["bias"] is None else state["bias"].detach().double().requires_grad_(True)
            target, total = state["target"], []
            n = int((target != -100).sum()) if target.dim() == 1 else target.shape[0]
            piece = max(1, min(case["rows"], (1 << 29) // case["classes"]))
            for i in range(0, case["rows"], piece):
                t = target[i:i + piece]
                z = torch.matmul(leaf_x[i:i + piece], leaf_w.t())
                if leaf_b is not None:
                    z = z + leaf_b
                norm = torch.logsumexp(z, 1)
                if t.dim() == 1:
                    part = torch.where(t == -100, 0.0, norm - z[torch.arange(len(t), device=t.device), torch.where(t == -100, 0, t)])
                    weight = (t != -100).double()
                else:
                    part = norm * t.double().sum(1) - (t.double() * z).sum(1)
                    weight = torch.ones(len(t), dtype=torch.float64, device=t.device)
                if case["entropy"]:
                    mean = (torch.softmax(z, 1) * z).sum(1)
                    part = part - case["entropy"] * weight * (norm - mean)
                total.append(part.detach())
                if case["train"]:
                    (part.sum() / n).backward(state["scale"].double())
                del z, norm, part
        total = torch.cat(total)
        if not case["train"]:
            return total
        return [total.sum() / n, leaf_x.grad, leaf_w.grad] + ([] if leaf_b is None else [leaf_b.grad])
    if case["op"] == "dropout":
        import numpy as np
        n = x.numel()
        with np.errstate(over="ignore"):   # the generator in unsigned whole numbers on the host
            c = [np.arange((n + 7) // 8, dtype=np.uint64), np.uint64(0), np.uint64(state["offset"] & _M32), np.uint64(state["offset"] >> 32)]
            c[0], c[1] = c[0] & np.uint64(_M32), c[0] >> np.uint64(32)
            k = [state["seed"] & _M32, state["seed"] >> 32]
            for r in range(10):
                a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
                key = [np.uint64((k[0] + r * 0x9E3779B9) & _M32), np.uint64((k[1] + r * 0xBB67AE85) & _M32)]
                c = [(b >> np.uint64(32)) ^ c[1] ^ key[0], b & np.uint64(_M32), (a >> np.uint64(32)) ^ c[3] ^ key[1], a & np.uint64(_M32)]
            words = np.stack([np.broadcast_to(v, c[0].shape).astype(np.uint32) for v in c], 1)
        halves = torch.from_numpy(words.view(np.uint16).astype(np.int32).reshape(-1)[:n]).to(x.device)
        threshold = round(65536 * case["p"])
        factor = (halves.view(x.shape) >= threshold).double() * (65536 / (65536 - threshold))
        y = x * factor if state["residual"] is None else torch.addcmul(state["residual"].detach().double(), x, factor)
        if not case["train"]:
            return y
        grad = state["grad"].double()
        return [y, grad * factor] + ([] if state["residual"] is None else [grad])
    top = x.abs().max(dim=1, keepdim=True).values
    whole = (x / torch.where(top == 0, torch.ones_like(top), top) * 127.0).round()
    near = x * 127.0 / torch.where(top == 0, torch.ones_like(top), top)
    whole = torch.where((near - near.floor() - 0.5).abs() < 1e-9, near.round(), whole)   # one rounding where the quotient is at a half
    y = torch.matmul(whole * (top / 127.0), (state["qweight"].double() * state["wscale"].double()[:, None]).t())
    return y if state["bias"] is None else y + state["bias"].double()

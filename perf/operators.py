"""The operators of learned per-Gaussian attributes, as a user's program calls them, with their plain forms.

A scene may carry a learned feature vector per Gaussian next to its six parameter groups. A small network turns the
features into what the rasteriser or a label needs: fully connected layers (msplat.ops.linear_forward and
linear_backward), dropout between them (msplat.ops.dropout), and a classification loss over a table of label
embeddings (msplat.ops.loss_cross_entropy). Each case below is one call of one of them.

With `own` false, run() computes the same values with elementary torch operations in 32 bits, rounded once.
"""
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "msplat-ios_b200", "python"))

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = ("none", "relu", "gelu", "silu", "sigmoid")

# what the drawn cases stay within: the largest listed one of each operator
MOST_PRODUCT = 65536 * 1024 * 1024   # rows x inputs x outputs of a layer
MOST_ELEMENTS = 1_000_000 * 128      # rows x (inputs + outputs) of a layer
MOST_DROPOUT = 1_000_000 * 64
MOST_LOGITS = 8192 * 32768
MOST_LOSS = 8192 * 32768 * 512       # rows x labels x width


def listed():
    return [
        # One appearance code of one camera through one layer: a single row, where the call's latency is all there is.
        {"name": "layer, one row", "op": "linear", "m": 1, "k": 512, "n": 512, "type": "bf16", "out": "bf16", "act": "silu",
         "bias": True, "residual": False, "preact": False, "pad": 0},
        # The hidden layer of a million Gaussians' features, in the parameters' own type, keeping what training needs.
        {"name": "layer, 1M gaussians f32", "op": "linear", "m": 1_000_000, "k": 32, "n": 64, "type": "f32", "out": "f32",
         "act": "gelu", "bias": True, "residual": False, "preact": True, "pad": 0},
        # A wide residual block over a batch of rows: a product that keeps the tensor cores busy.
        {"name": "layer, wide residual bf16", "op": "linear", "m": 65536, "k": 1024, "n": 1024, "type": "bf16", "out": "bf16",
         "act": "gelu", "bias": True, "residual": True, "preact": False, "pad": 0},
        # Colours for the rasteriser from 16-bit features: three outputs in 32 bits, features read out of a wider record.
        {"name": "layer, colours f16", "op": "linear", "m": 1_000_000, "k": 61, "n": 3, "type": "f16", "out": "f32",
         "act": "sigmoid", "bias": True, "residual": False, "preact": False, "pad": 3},
        # Training: the gradients of the hidden layer of a million Gaussians.
        {"name": "layer gradient, 1M f32", "op": "linear_grad", "m": 1_000_000, "k": 32, "n": 64, "type": "f32", "act": "gelu",
         "pad": 0},
        # Training: the gradients of the wide block.
        {"name": "layer gradient, wide bf16", "op": "linear_grad", "m": 65536, "k": 1024, "n": 1024, "type": "bf16",
         "act": "gelu", "pad": 0},
        # Dropout of a small batch's features, an odd width out of a wider record.
        {"name": "dropout, small f32", "op": "dropout", "m": 1000, "n": 33, "type": "f32", "p": 0.2, "residual": False, "pad": 5},
        # Dropout with the residual added, over a million Gaussians' hidden features.
        {"name": "dropout, 1M bf16", "op": "dropout", "m": 1_000_000, "n": 64, "type": "bf16", "p": 0.1, "residual": True,
         "pad": 0},
        # Training: labels of a million Gaussians (some without one) against a small table, in the parameters' own type.
        {"name": "labels, 1M gaussians f32", "op": "loss", "m": 1_000_000, "v": 101, "d": 32, "type": "f32", "grad": True,
         "unlabelled": 0.3, "scale": 1.0, "weight": 1.0},
        # Training: a batch of rows against a large table.
        {"name": "labels, large table bf16", "op": "loss", "m": 8192, "v": 32768, "d": 512, "type": "bf16", "grad": True,
         "unlabelled": 0.0, "scale": 1.0, "weight": 1.0},
        # Training, ragged in every size, with a loss scale as 16-bit training has it.
        {"name": "labels, ragged f16", "op": "loss", "m": 3001, "v": 50021, "d": 200, "type": "f16", "grad": True,
         "unlabelled": 0.1, "scale": 2.0, "weight": 4096.0},
        # Scoring a few rows against a very large table, without gradients.
        {"name": "labels, scoring bf16", "op": "loss", "m": 16, "v": 131072, "d": 256, "type": "bf16", "grad": False,
         "unlabelled": 0.0, "scale": 1.0, "weight": 1.0},
    ]


def _size(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 16 and rng.random() < 0.5:
        v -= v % (8 if v < 256 else 64)  # half of the sizes are round ones
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_grad", "linear_grad", "dropout", "loss", "loss"))
    kind = rng.choice(("f32", "f16", "bf16"))
    if op in ("linear", "linear_grad"):
        k, n = _size(rng, 3, 1024), _size(rng, 2, 1024)
        m = _size(rng, 1, 1_000_000)
        m = max(1, min(m, MOST_PRODUCT // (k * n), MOST_ELEMENTS // (k + n)))
        c = {"op": op, "m": m, "k": k, "n": n, "type": kind, "act": rng.choice(ACTIVATIONS), "pad": rng.choice((0, 0, 8, 5))}
        if op == "linear":
            c |= {"out": rng.choice((kind, kind, "f32")), "bias": rng.random() < 0.7, "residual": rng.random() < 0.4,
                  "preact": rng.random() < 0.4}
        return c
    if op == "dropout":
        n = _size(rng, 1, 1024)
        return {"op": op, "m": max(1, min(_size(rng, 1, 1_000_000), MOST_DROPOUT // n)), "n": n, "type": kind,
                "p": rng.choice((0.1, 0.2, 0.5)), "residual": rng.random() < 0.5, "pad": rng.choice((0, 0, 8, 5))}
    d, v = _size(rng, 8, 1024), _size(rng, 2, 131072)
    m = max(1, min(_size(rng, 1, 1_000_000), MOST_LOGITS // v, MOST_LOSS // (v * d), MOST_ELEMENTS // d))
    return {"op": op, "m": m, "v": v, "d": d, "type": kind, "grad": rng.random() < 0.7, "unlabelled": rng.choice((0.0, 0.1, 0.5)),
            "scale": rng.choice((1.0, 2.0)), "weight": 4096.0 if kind == "f16" else 1.0}


def _normal(g, rows, cols, kind, std=1.0, pad=0):
    """Normal values [rows, cols]; with pad, a view of columns inside a wider matrix, as a record's fields are."""
    t = torch.randn(rows, cols + pad, generator=g, device="cuda").mul_(std).to(TYPES[kind])
    return t[:, pad // 2:pad // 2 + cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, t = case, case["type"]
    s = {"case": dict(case)}
    if c["op"] in ("linear", "linear_grad"):
        s["x"] = _normal(g, c["m"], c["k"], t, pad=c["pad"])
        s["w"] = _normal(g, c["n"], c["k"], t, std=c["k"] ** -0.5)
        if c["op"] == "linear":
            s["bias"] = _normal(g, 1, c["n"], t, std=0.1)[0] if c["bias"] else None
            s["residual"] = _normal(g, c["m"], c["n"], c["out"]) if c["residual"] else None
        else:
            s["preact"] = _normal(g, c["m"], c["n"], t) if c["act"] != "none" else None
            s["dy"] = _normal(g, c["m"], c["n"], t, pad=c["pad"])
    elif c["op"] == "dropout":
        s["x"] = _normal(g, c["m"], c["n"], t, pad=c["pad"])
        s["residual"] = _normal(g, c["m"], c["n"], t) if c["residual"] else None
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ seed, 7 * seed + 1
    else:
        s["x"] = _normal(g, c["m"], c["d"], t)
        s["w"] = _normal(g, c["v"], c["d"], t, std=c["d"] ** -0.5)
        labels = torch.randint(0, c["v"], (c["m"],), generator=g, device="cuda", dtype=torch.int32)
        off = torch.rand(c["m"], generator=g, device="cuda") < c["unlabelled"]
        s["targets"] = torch.where(off, torch.full_like(labels, -1), labels)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _activate(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    """The derivative of the activation at z."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    q = 1 / (1 + torch.exp(-z))
    return q * (1 + z * (1 - q)) if act == "silu" else q * (1 - q)


def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _activate(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(TYPES[c["out"]])}
    if c["preact"]:
        out["preact"] = z.to(TYPES[c["out"]])
    return out


def _plain_linear_grad(s):
    t, dz = TYPES[s["case"]["type"]], s["dy"].float()
    if s["preact"] is not None:
        dz = dz * _slope(s["preact"].float(), s["case"]["act"])
    return {"dx": (dz @ s["w"].float()).to(t), "dw": (dz.T @ s["x"].float()).to(t), "dbias": dz.sum(0).to(t)}


def _plain_draws(count, seed, offset):
    """The 16-bit draws of `count` elements: Philox4x32-10 with the key `seed` and the counter (element / 8, offset)."""
    low, block = 0xFFFFFFFF, torch.arange((count + 7) // 8, device="cuda", dtype=torch.int64)
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits, which is all of the product
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:count]


def _plain_dropout(s):
    c, x = s["case"], s["x"].float()
    below = int(c["p"] * 65536 + 0.5)
    keep = _plain_draws(x.numel(), s["seed"], s["offset"]).reshape(x.shape) >= below
    y = torch.where(keep, x * (65536 / (65536 - below)), torch.zeros_like(x))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(TYPES[c["type"]])}


def _plain_loss(s):
    c, t = s["case"], TYPES[s["case"]["type"]]
    target = s["targets"].long()
    known = (target >= 0) & (target < c["v"])
    at = torch.where(known, target, torch.zeros_like(target))[:, None]
    x, w = torch.where(known[:, None], s["x"].float(), torch.zeros((), device="cuda")), s["w"].float()
    logits = (x @ w.T) * c["scale"]
    top = logits.max(1, keepdim=True).values
    chosen = logits.gather(1, at)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    row = torch.where(known, (torch.log(total) + top - chosen)[:, 0], torch.zeros((), device="cuda"))
    count = known.sum().clamp(min=1)
    out = {"loss": (row.double().sum() / count * c["weight"]).float(), "row_loss": row}
    if c["grad"]:
        p = e / total
        p.scatter_add_(1, at, torch.full_like(chosen, -1.0))
        p = p * (known[:, None] * (c["weight"] * c["scale"] / count))
        out |= {"dx": (p @ w).to(t), "dw": (p.T @ x).to(t)}
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------------


def _own(s):
    from msplat import ops
    c = s["case"]
    if c["op"] == "linear":
        z = torch.empty(c["m"], c["n"], device="cuda", dtype=TYPES[c["out"]]) if c["preact"] else None
        y = ops.linear_forward(s["x"], s["w"], s["bias"], activation=c["act"], residual=s["residual"], preact=z,
                               out_dtype=TYPES[c["out"]])
        return {"y": y, "preact": z} if c["preact"] else {"y": y}
    if c["op"] == "linear_grad":
        dx, dw, dbias = ops.linear_backward(s["x"], s["w"], s["dy"], preact=s["preact"], activation=c["act"])
        return {"dx": dx, "dw": dw, "dbias": dbias}
    if c["op"] == "dropout":
        return {"y": ops.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["residual"])}
    loss, row, dx, dw = ops.loss_cross_entropy(s["x"], s["w"], s["targets"], logit_scale=c["scale"], weight=c["weight"],
                                               grad=c["grad"])
    out = {"loss": loss, "row_loss": row}
    return out | {"dx": dx, "dw": dw} if c["grad"] else out


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "linear_grad": _plain_linear_grad, "dropout": _plain_dropout,
            "loss": _plain_loss}[state["case"]["op"]](state)


def work(case):
    c = case
    size, out = TYPES[c["type"]].itemsize, TYPES[c.get("out", c["type"])].itemsize
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        outputs = m * n * (1 + c["residual"] + c["preact"])
        return {"bytes": (m * k + n * k + n * c["bias"]) * size + outputs * out, "flops": 2 * m * k * n}
    if c["op"] == "linear_grad":
        m, k, n = c["m"], c["k"], c["n"]
        return {"bytes": (2 * m * k + 2 * n * k + m * n * (1 + (c["act"] != "none")) + n) * size, "flops": 4 * m * k * n}
    if c["op"] == "dropout":
        return {"bytes": c["m"] * c["n"] * size * (2 + c["residual"]), "flops": 2 * c["m"] * c["n"]}
    m, v, d = c["m"] * (1 - c["unlabelled"]), c["v"], c["d"]
    return {"bytes": (m * d + v * d) * size + c["m"] * 8 + (c["m"] * d + v * d) * size * c["grad"],
            "flops": (6 if c["grad"] else 2) * m * v * d}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_keep(count, seed, offset, p):
    """Whether each element is kept, from numpy's unsigned 64-bit integers."""
    u = np.uint64
    half, low = u(32), u(0xFFFFFFFF)
    ctr = np.zeros((4, (count + 7) // 8), u)
    ctr[0] = np.arange(ctr.shape[1], dtype=u) & low
    ctr[1] = np.arange(ctr.shape[1], dtype=u) >> half
    ctr[2], ctr[3] = u(offset & 0xFFFFFFFF), u(offset >> 32)
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = np.stack([(b >> half) ^ ctr[1] ^ u(key[0]), b & low, (a >> half) ^ ctr[3] ^ u(key[1]), a & low])
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    draws = ctr.T.astype("<u4").copy().view("<u2").reshape(-1)[:count]
    return torch.from_numpy(draws.astype(np.int32) >= math.floor(p * 65536 + 0.5)).to("cuda")


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] in ("linear", "linear_grad"):
        x, w = s["x"].double(), s["w"].double()
        if c["op"] == "linear":
            z = torch.mm(x, w.t())
            if s["bias"] is not None:
                z += s["bias"].double()
        else:
            z = s["preact"].double() if s["preact"] is not None else None
        if c["op"] == "linear":
            y = {"none": lambda: z.clone(), "relu": lambda: z.clamp(min=0), "sigmoid": lambda: torch.sigmoid(z),
                 "silu": lambda: z * torch.sigmoid(z), "gelu": lambda: z * torch.special.ndtr(z)}[c["act"]]()
            if s["residual"] is not None:
                y += s["residual"].double()
            return {"y": y, "preact": z} if c["preact"] else {"y": y}
        dz = s["dy"].double()
        if z is not None:
            q = torch.sigmoid(z)
            dz = dz * {"relu": lambda: (z > 0).double(), "sigmoid": lambda: q - q * q, "silu": lambda: q + z * (q - q * q),
                       "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[c["act"]]()
        return {"dx": torch.mm(dz, w), "dw": torch.mm(dz.t(), x), "dbias": dz.sum(0)}
    if c["op"] == "dropout":
        keep = _exact_keep(c["m"] * c["n"], s["seed"], s["offset"], c["p"]).reshape(c["m"], c["n"])
        y = s["x"].double() * keep / (1 - math.floor(c["p"] * 65536 + 0.5) / 65536)
        return {"y": y if s["residual"] is None else y + s["residual"].double()}
    # the loss: pieces of rows, so that the logits in 64 bits stay small
    x, w, t = s["x"].double(), s["w"].double(), s["targets"].long()
    rows = torch.nonzero((t >= 0) & (t < c["v"]))[:, 0]
    loss = torch.zeros(c["m"], dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for part in torch.split(rows, max(1, (1 << 27) // c["v"])):
        logits = torch.mm(x[part], w.t()) * c["scale"]
        lse = torch.logsumexp(logits, 1)
        loss[part] = lse - logits[torch.arange(len(part), device="cuda"), t[part]]
        if c["grad"]:
            logits = (logits - lse[:, None]).exp_()
            logits[torch.arange(len(part), device="cuda"), t[part]] -= 1
            logits *= c["weight"] * c["scale"] / max(1, len(rows))
            dx[part] = torch.mm(logits, w)
            dw += torch.mm(logits.t(), x[part])
    out = {"loss": loss.sum() / max(1, len(rows)) * c["weight"], "row_loss": loss}
    return out | {"dx": dx, "dw": dw} if c["grad"] else out

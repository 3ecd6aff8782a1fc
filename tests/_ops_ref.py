"""Plain 64-bit forms of the operators in msplat.ops with bounds on how far a
correct kernel may be from them, element by element.

u is half a step of a type (torch.finfo(t).eps / 2) and h half of its smallest
subnormal: rounding v gives an error of at most u |v| + h. A sum of r products
in 32 bits, added in any order and rounded in any direction, is off by at most
SUM * (r + 8) * (sum of the products' sizes), SUM = 2^-23, as long as r 2^-23 is
far below 1 (the 8 covers the bias, the scale factors and, for 32-bit
factors, the parts of a split product below 2^-24 that are left out).
"""
import math

import numpy as np
import torch

SUM = 2.0 ** -23
FUN = 2.0 ** -20  # relative error of exp, erf and a division in 32 bits, generously (8 steps)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HALF_TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rounded(v, t):
    return HALF_STEP[t] * v.abs() + HALF_TINY[t]


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    return z


def slope(z, name):
    q = torch.sigmoid(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        return q * (1 + z * (1 - q))
    if name == "sigmoid":
        return q * (1 - q)
    return torch.ones_like(z)


def linear(x, w, bias, name, residual, out_t):
    """(y, its bound, z, its bound)."""
    x, w = x.double(), w.double()
    z, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    off = SUM * (x.shape[1] + 8) * size
    y = act(z, name)
    # every activation changes by at most 1.13 times what its argument does; evaluating it is off by FUN of
    # its size or, for gelu's 1 + erf, FUN of its argument's
    off_y = 1.13 * off + (FUN * (z.abs() + y.abs()) if name != "none" else 0)
    if residual is not None:
        y = y + residual.double()
        off_y = off_y + HALF_STEP[torch.float32] * y.abs()
    return y, off_y + rounded(y.abs() + off_y, out_t), z, off + rounded(z.abs() + off, out_t)


def linear_grads(x, w, dy, z, name, t):
    """((dx, bound), (dw, bound), (dbias, bound))."""
    x, w, dz = x.double(), w.double(), dy.double()
    off = torch.zeros_like(dz)
    if name != "none":
        dz = dz * slope(z.double(), name)
        # the slopes are at most 1.13, with intermediate values of at most 1 + |z exp(..)| < 2
        off = FUN * 2 * dy.double().abs() * (1 + (z.double().abs() if name == "silu" else 0)) + SUM * dz.abs()
    off_sum = off.sum(0) + SUM * (dz.shape[0] + 8) * dz.abs().sum(0)
    if name != "none":
        off = off + rounded(dz.abs() + off, t)  # dz is rounded between the products
    m, n = dz.shape
    top = dz.abs() + off
    dx, dw, db = dz @ w, dz.T @ x, dz.sum(0)
    off_x = off @ w.abs() + SUM * (n + 8) * (top @ w.abs())
    off_w = off.T @ x.abs() + SUM * (m + 8) * (top.T @ x.abs())
    return ((dx, off_x + rounded(dx.abs() + off_x, t)), (dw, off_w + rounded(dw.abs() + off_w, t)),
            (db, off_sum + rounded(db.abs() + off_sum, t)))


def loss(x, w, targets, scale, weight, t):
    """{name: (value, bound)} of loss, row_loss, dx, dw."""
    known = (targets >= 0) & (targets < w.shape[0])
    target = targets.long() * known
    x = torch.where(known[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    w = w.double()
    m, d = x.shape
    v = w.shape[0]
    count = int(known.sum())
    logits = scale * (x @ w.T)
    off_l = (SUM * (d + 8) * abs(scale) * (x.abs() @ w.abs().T) + FUN * logits.abs()).max(1).values if m else x.sum(1)
    lse = torch.logsumexp(logits, 1)
    pick = logits.gather(1, target[:, None])[:, 0]
    # lse moves by at most what the logits do; its own sum of v terms and logarithm in 32 bits
    off_row = 2 * off_l + SUM * (v + 16) + 2 * FUN * (lse.abs() + pick.abs())
    row, off_row = (lse - pick) * known, off_row * known
    total = row.sum() / max(1, count) * weight
    off_total = abs(weight) * off_row.sum() / max(1, count)
    p = torch.exp(logits - lse[:, None])
    off_p = p * torch.expm1(2 * off_l + 2 * SUM * (v + 16) + 4 * FUN)[:, None]
    g = p.scatter_add(1, target[:, None], torch.full((m, 1), -1.0, dtype=torch.float64, device=x.device))
    off_g = off_p + HALF_STEP[torch.float32] * 2 * (g.abs() + off_p)
    tiny = HALF_TINY[t] / (2.0 ** 14 if t == torch.float16 else 1.0)
    off_g = off_g + HALF_STEP[t] * (g.abs() + off_g) + tiny
    a = weight * scale / max(1, count)
    g, off_g = g * known[:, None], off_g * known[:, None]
    top = g.abs() + off_g
    dx, dw = a * (g @ w), a * (g.T @ x)
    off_x = abs(a) * (off_g @ w.abs() + SUM * (v + 8) * (top @ w.abs()))
    off_w = abs(a) * (off_g.T @ x.abs() + SUM * (m + 8) * (top.T @ x.abs()))
    return {"loss": (total, off_total + rounded(total.abs() + off_total, torch.float32)),
            "row_loss": (row, off_row + rounded(row.abs() + off_row, torch.float32) * known),
            "dx": (dx, off_x + rounded(dx.abs() + off_x, t) * known[:, None]),
            "dw": (dw, off_w + rounded(dw.abs() + off_w, t))}


def philox4x32_10(counter, key):
    """Rows of four 32-bit words from rows of four counter words and two key words."""
    u = np.uint64
    c = [np.asarray(x, u) for x in counter]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & u(0xFFFFFFFF), (a >> u(32)) ^ c[3] ^ u(k[1]), a & u(0xFFFFFFFF)]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(count, seed, offset, first=0):
    """The 16-bit draws of elements first .. first + count."""
    b = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    c = philox4x32_10([b & np.uint64(0xFFFFFFFF), b >> np.uint64(32), np.full_like(b, offset & 0xFFFFFFFF),
                       np.full_like(b, offset >> 32)], (seed & 0xFFFFFFFF, seed >> 32))
    words = np.stack(c, 1)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1).astype(np.int64)
    return halves[first % 8:first % 8 + count]


def dropout(x, p, seed, offset, residual, t):
    """(y, bound); x a CPU or CUDA matrix."""
    below = math.floor(p * 65536 + 0.5)
    keep = torch.from_numpy(draws(x.numel(), seed, offset) >= below).reshape(x.shape).to(x.device)
    scale = 65536 / (65536 - below) if below < 65536 else 0.0
    y = torch.where(keep, x.double() * scale, torch.zeros((), dtype=torch.float64, device=x.device))
    off = 2 * HALF_STEP[torch.float32] * y.abs()  # the scale and the product
    if residual is not None:
        y = y + residual.double()
        off = (off + HALF_STEP[torch.float32] * (y.abs() + off))
    return y, off + rounded(y.abs() + off, t) * (off > 0)


def check(got, want, bound, name):
    """Asserts |got - want| <= bound everywhere."""
    g = got.double()
    assert g.shape == want.shape, (name, g.shape, want.shape)
    if not g.numel():
        return
    assert bool(torch.isfinite(g).all()), f"{name}: not finite"
    over = (g - want).abs() - bound
    at = int(over.argmax())
    assert float(over.max()) <= 0, (f"{name}: element {at} is {g.flatten()[at].item()!r}, should be "
                                    f"{want.flatten()[at].item()!r} within {bound.expand_as(g).flatten()[at].item():.3g}")

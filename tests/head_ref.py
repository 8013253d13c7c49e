"""Plain 64-bit forms of the operators of alphazero_amd.head, with the error that each result may have.

The bounds count roundings: a rounding to a type is off by at most half a step, U[type] relative to the value; a sum of n products in
float32 by (n + 8) 2^-24 of the sum of their magnitudes; the hardware's exp2 and the multiplication in front of it by
2^-22 (1 + |argument|)."""
import numpy as np
import torch

U = {torch.float64: 0.0, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}      # half the step of the smallest values
F32 = 2.0 ** -24


def loss_reference(x, w, target, bias, ignore=-100, c=0.0, reduction="mean", grad=None):
    """dict of value and tolerance for loss, ce, ent (rows), gx, gw, gb."""
    dt = x.dtype
    xd, wd = x.detach().double(), w.detach().double()
    rows, feats = xd.shape
    classes = wd.shape[0]
    bd = torch.zeros(classes, dtype=torch.float64, device=x.device) if bias is None else bias.detach().double()
    dense = target.is_floating_point()
    counts = torch.ones(rows, dtype=torch.bool, device=x.device) if dense else target != ignore
    xd = torch.where(counts[:, None], xd, 0.0)
    z = xd @ wd.t() + bd
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    p = torch.exp(logp)
    if dense:
        pi = target.double()
    else:
        pi = torch.zeros_like(z)
        pi[torch.arange(rows, device=x.device)[counts], target[counts]] = 1.0
    total = torch.where(counts, pi.sum(1), 0.0)
    ce = torch.where(counts, total * lse - torch.where(pi == 0, 0.0, pi * z).sum(1), 0.0)
    plogp = torch.where(p == 0, 0.0, p * logp)
    ent = -plogp.sum(1)
    row = torch.where(counts, ce - c * ent, 0.0)
    n = counts.sum().double()
    # a logit's error: the sum's, float32's two planes cover 2^-22 of each product, the bias is added in float32
    mag = xd.abs() @ wd.abs().t()
    fine = torch.where(torch.isfinite(bd), bd.abs(), 0.0)
    ez = ((feats + 8) * F32 + (2.0 ** -22 if dt == torch.float32 else 0.0)) * mag + 2 * F32 * (mag + fine)
    eo = ez.amax(1) + 2.0 ** -21 * (1 + torch.where(torch.isfinite(z), z.abs(), 0.0).amax(1))          # of lse, and of z - lse
    pa = pi.abs().sum(1)
    spread = torch.where(p > 1e-300, logp.abs() * p, 0.0).sum(1)
    t_ce = (pa + 1) * 2 * eo + (classes * F32 + 4 * F32) * (pa * (lse.abs() + z.abs().where(torch.isfinite(z), torch.zeros_like(z)).amax(1)))
    t_ent = 4 * eo * (1 + spread) + 2.0 ** -20 * (1 + ent) + 64 * F32 * spread
    t_row = t_ce + abs(c) * t_ent + 4 * F32 * row.abs()
    out = {"row": (row, t_row), "ce_row": (ce, t_ce), "ent_row": (ent, t_ent)}
    d = {"none": 1.0, "sum": 1.0, "mean": n}[reduction]
    for name, v, t in (("loss", row, t_row), ("ce", ce, t_ce), ("ent", torch.where(counts, ent, 0.0), t_ent)):
        out[name] = (v.sum() / d, torch.where(counts, t, 0.0).sum() / d + 4 * F32 * (v.sum() / d).abs()) if reduction != "none" else (v, t)
    if grad is None:
        return out
    f = torch.where(counts, (grad.double() if reduction == "none" else grad.double().expand(rows)) / d, 0.0)
    inner = c * (plogp + p * ent[:, None])
    g = torch.where(counts[:, None], (total[:, None] * p - pi + inner) * f[:, None], 0.0)
    # of G: its terms in float32, then its rounding (two planes for float32)
    terms = total[:, None].abs() * p + pi.abs() + abs(c) * (plogp.abs() + p * ent[:, None].abs())
    ep = p * (2 * eo[:, None] + 2.0 ** -22 * (2 + torch.where(torch.isfinite(logp), logp.abs(), 0.0)))
    lp = torch.where(torch.isfinite(logp), logp.abs(), 0.0)
    eg = f.abs()[:, None] * ((total.abs()[:, None] + abs(c) * (1 + lp + ent[:, None])) * ep + abs(c) * p * (2 * eo + t_ent)[:, None] + 8 * F32 * terms)
    e32 = eg + 8 * F32 * g.abs()
    eg = eg + (U[dt] if dt != torch.float32 else 2.0 ** -23) * g.abs()
    if dt == torch.float16:    # G is held with its bound between 2^13 and 2^14: the smallest step there is 2^-24
        bound = (2 * pa.max() if dense else 1.0) + abs(c) * (0.4 + np.log(classes))
        eg = eg + 2.0 ** -25 * bound * f.abs().max() / 8192
    eg = torch.where(counts[:, None], eg, 0.0)
    split = 2.0 ** -22 if dt == torch.float32 else 0.0
    gx, gw, gb = g @ wd, g.t() @ xd, g.sum(0)
    out["gx"] = (gx, (eg + ((classes + 64) * F32 + split) * g.abs()) @ wd.abs() * (1 + U[dt]) + (U[dt] + 2 * F32) * gx.abs() + TINY[dt])
    out["gw"] = (gw, (eg + ((rows + 64) * F32 + split) * g.abs()).t() @ xd.abs() * (1 + U[dt]) + (U[dt] + 2 * F32) * gw.abs() + TINY[dt])
    out["gb"] = (gb, (e32 + (rows + 8) * F32 * g.abs()).sum(0) * (1 + U[dt]) + (U[dt] + 2 * F32) * gb.abs() + TINY[dt])
    return out


def close(name, got, ref):
    value, tol = ref
    got = got.double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    bad = ~((got - value).abs() <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - value).abs() / tol.clamp(min=1e-300))[bad].max()):.3g} times the bound"


def philox_block(c, k):
    """Philox4x32-10 in unsigned whole numbers: counter words c (numbers or arrays) under the key words k."""
    m32 = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in c]
    k0, k1 = k
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def philox_kept(count, p, seed, offset):
    """(mask of alphazero_amd.head.dropout, the groups' words), on the host."""
    g = np.arange((count + 7) // 8, dtype=np.uint64)
    m32 = np.uint64(0xFFFFFFFF)
    words = np.stack(philox_block((g & m32, g >> np.uint64(32), np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)),
                                  (seed & 0xFFFFFFFF, seed >> 32)), 1)
    bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[:count]
    return bits >= np.uint64(round(65536 * p)), words


def quantize_reference(x):
    """(q, scale) in whole-number arithmetic: the nearest whole number of the real quotient, ties to even."""
    from fractions import Fraction
    xs = x.detach().double().cpu()
    q = torch.zeros(xs.shape, dtype=torch.int8)
    scale = torch.empty(xs.shape[0], dtype=torch.float32)
    for r in range(xs.shape[0]):
        row = xs[r]
        top = row.abs().max()
        if not torch.isfinite(row).all():
            scale[r] = float("nan")
            continue
        scale[r] = top.float() / 127
        if top > 0:
            t = Fraction(float(top))
            q[r] = torch.tensor([round(Fraction(float(v)) * 127 / t) for v in row], dtype=torch.int8)   # round(): ties to even
    return q, scale

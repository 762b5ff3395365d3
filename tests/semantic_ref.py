"""The semantic head's operators in 64 bits on the CPU, and bounds on what fp32 sums in any order and one rounding to the
tensors' type may be off by.  U32 = 2^-24 is half a step of fp32; a sum of n fp32 terms in any order is off by at most
(n - 1) U32 times the sum of their magnitudes (to first order), an exp / erf / log of the device library by a few U32."""
import math

import torch

U32 = 2.0 ** -24
U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # least subnormal: one step there
EV = 16 * U32  # evaluation of an activation, its slope or an exponential: a few steps of fp32 each


def act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, z * 0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if kind == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, kind):
    if kind == "relu":
        return (z > 0).double()
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def linear(x, w, b, r, kind, dy=None):
    """2-D tensors of one type -> {name: (value, bound)} in float64 on the CPU."""
    dt = x.dtype
    u, tiny = U[dt], TINY[dt]
    x, w = x.detach().cpu().double(), w.detach().cpu().double()
    bb = b.detach().cpu().double() if b is not None else torch.zeros(w.shape[0], dtype=torch.float64)
    K, N, M = w.shape[1], w.shape[0], x.shape[0]
    z = x @ w.t() + bb
    size = x.abs() @ w.abs().t() + bb.abs()
    ez = (K + 2) * U32 * size
    y = act(z, kind)
    ey = 1.13 * ez + EV * (z.abs() + y.abs())  # (the activations' slopes stay below 1.13)
    if r is not None:
        rr = r.detach().cpu().double()
        y = y + rr
        ey = ey + U32 * (y.abs() + rr.abs())
    out = {"y": (y, ey + u * (y.abs() + ey) + tiny)}
    if dy is None:
        return out
    g = dy.detach().cpu().double()
    dz = g * slope(z, kind)
    if kind == "relu":  # (a pre-activation inside its own error may fall on either side)
        edz = g.abs() * (z.abs() <= ez)
    elif kind == "none":
        edz = torch.zeros_like(g)
    else:  # |slope'| <= 0.8
        edz = g.abs() * (0.8 * ez + EV * (1 + z.abs())) + U32 * dz.abs()
    if kind != "none" and dt != torch.float32:
        edz = edz + u * dz.abs() + tiny  # rounded to the type before its two products
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    edx = edz @ w.abs() + (N + 2) * U32 * (dz.abs() @ w.abs())
    edw = edz.t() @ x.abs() + (M + 2) * U32 * (dz.abs().t() @ x.abs())
    edb = edz.sum(0) + (M + 2) * U32 * dz.abs().sum(0)
    for name, v, e in (("dx", dx, edx), ("dw", dw, edw), ("db", db, edb)):
        out[name] = (v, e + u * (v.abs() + e) + tiny)
    return out


def distill(logits, idx, top, T=1.0, weight=None, reduction="mean", g=None):
    """2-D logits -> {"loss": (value, bound), "dlogits": (value, bound)} in float64 on the CPU."""
    dt = logits.dtype
    u, tiny = U[dt], TINY[dt]
    s = logits.detach().cpu().double()
    idx, tu = idx.cpu().long(), top.detach().cpu().double()
    R, V = s.shape
    K = idx.shape[1]
    there = (idx >= 0) & (idx < V)
    tu = torch.where(there, tu, torch.full_like(tu, -math.inf))
    alive = (tu != -math.inf).any(1)
    w = torch.ones(R, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    alive = alive & (w != 0)
    w = torch.where(alive, w, torch.zeros_like(w))
    s = torch.where(alive[:, None], s, torch.zeros_like(s))
    tu = torch.where(alive[:, None], tu, torch.zeros_like(tu))
    a = (s - s.max(1, keepdim=True).values) / T
    q = torch.softmax(a, 1)
    lq_all = torch.log_softmax(a, 1)
    ut = (tu - tu.max(1, keepdim=True).values) / T
    p = torch.softmax(ut, 1)
    lp = torch.log_softmax(ut, 1)
    lq = torch.gather(lq_all, 1, torch.where(there, idx, torch.zeros_like(idx)))
    term = torch.where(p > 0, p * (lp - lq), torch.zeros_like(p))
    kl = term.sum(1) * T * T
    # an exponent (s - m) / T is off by 3 U32 of itself; relative errors of q and p, absolute ones of their logarithms
    def fin(t):
        return torch.where(torch.isfinite(t), t, torch.zeros_like(t)).abs()
    ea, eu = fin(a) * 3 * U32, fin(ut) * 3 * U32
    es = (q * ea).sum(1, keepdim=True) + (V + 16) * U32
    eq = ea + es + EV
    ez = (p * eu).sum(1, keepdim=True) + (K + 16) * U32
    ep = eu + ez + EV
    elq = torch.gather(ea + es, 1, torch.where(there, idx, torch.zeros_like(idx))) + EV * (1 + fin(lq))
    elp = eu + ez + EV * (1 + fin(lp))
    pos = p > 0
    ekl = torch.where(pos, p * (elq + elp) + (ep + (K + 4) * U32) * p * (fin(lp) + fin(lq)), torch.zeros_like(p)).sum(1) * T * T
    row = torch.where(alive, kl * w, torch.zeros_like(kl))
    erow = ekl * w.abs() + 8 * U32 * row.abs() + 2.0 ** -149
    total = float(w.sum())
    scale = 1.0
    if reduction == "mean":
        scale = 1.0 / total if total != 0 else 0.0
    if reduction == "none":
        loss, eloss = row, erow
    else:
        loss, eloss = row.sum() * scale, (erow.sum() + 8 * U32 * row.abs().sum()) * abs(scale)
    out = {"loss": (loss, eloss)}
    if g is not None:
        up = g.detach().cpu().double()
        coef = T * scale * w * up
        mass = torch.zeros_like(q).scatter_add_(1, torch.where(there, idx, torch.zeros_like(idx)),
                                                torch.where(there, p, torch.zeros_like(p)))
        emass = torch.zeros_like(q).scatter_add_(1, torch.where(there, idx, torch.zeros_like(idx)),
                                                 torch.where(there, p * (ep + K * U32), torch.zeros_like(p)))
        d = coef[:, None] * (q - mass)
        ed = coef.abs()[:, None] * (q * eq + emass + 8 * U32 * (q + mass))
        out["dlogits"] = (d, ed + u * (d.abs() + ed) + tiny)
    return out


def check(got, want, what):
    v, e = want
    got = got.detach().cpu().double().reshape(v.shape)
    bad = ~((got - v).abs() <= e)
    bad &= ~((got == v) | (torch.isnan(got) & torch.isnan(v)))
    if bad.any():
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got.reshape(-1)[i].item()!r}, "
                             f"want {v.reshape(-1)[i].item()!r} +- {e.reshape(-1)[i].item():.3g}")

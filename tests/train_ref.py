"""The operators of rwkvq.train in 64 bits on the CPU, and how far a result of
their kernels may be from that, element by element.

The bounds follow from the arithmetic alone.  u(T) is half the distance of
neighbouring values of type T at 1 (2^-8 bf16, 2^-11 f16, 2^-24 fp32), which is
the largest relative error of one rounding.  A sum of n products in fp32, in any
order, is within (n + 8) u(fp32) of the sum of the products' magnitudes.  The
activation functions and their slopes are within 16 u(fp32) of their values and
change by at most 1.2 (slope) per unit of v (relu2: 2 |v|)."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
U32 = 2.0 ** -24


def act(name, v):
    """act(v) and act'(v)."""
    if name is None:
        return v, torch.ones_like(v)
    if name == "relu":
        return v.clamp(min=0), (v > 0).double()
    if name == "relu2":
        return v.clamp(min=0) ** 2, 2 * v.clamp(min=0)
    if name == "sigmoid":
        s = torch.sigmoid(v)
        return s, s * torch.sigmoid(-v)
    if name == "tanh":
        return torch.tanh(v), 1 / torch.cosh(v) ** 2
    if name == "silu":
        s = torch.sigmoid(v)
        return v * s, s + v * s * torch.sigmoid(-v)
    p = torch.special.ndtr(v)
    return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)


def slope_error(name, dtype, residual):
    """The relative error of the slope as the backward pass reads it."""
    if name is None:
        return 0.0
    if dtype == torch.bfloat16:
        return U[torch.float16]
    if not residual and name == "relu2":
        return 2 * U32                        # from y: half its relative error, and the root's
    return U32


class Linear:
    """The forward and backward of act(x w^T + b) + r with a bound for each result."""

    def __init__(self, x, w, b, r, name, dy=None):
        T = x.dtype
        ydt = T if r is None else r.dtype
        X, W = x.detach().double().cpu(), w.detach().double().cpu()
        k, n, m = W.shape[1], W.shape[0], X.shape[:-1].numel()
        X = X.reshape(m, k)
        v = X @ W.t()
        mag = X.abs() @ W.abs().t()
        if b is not None:
            B = b.detach().double().cpu()
            v, mag = v + B, mag + B.abs()
        ev = (k + 8) * U32 * mag              # of v
        a, s = act(name, v)
        lip = 2 * v.abs() + 2 * ev if name == "relu2" else 1.2
        ea = ev * lip + 16 * U32 * a.abs()
        if name == "gelu" or name == "silu":  # v * Phi(v): the factor's error against 1
            ea = ea + 16 * U32 * v.abs()
        y = a
        if r is not None:
            R = r.detach().double().cpu().reshape(m, n)
            y, ea = a + R, ea + U32 * (a.abs() + R.abs())
        self.y, self.ey = y, ea + U[ydt] * (y.abs() + ea) + TINY[ydt]
        if dy is None:
            return
        D = dy.detach().double().cpu().reshape(m, n)
        g = D * s
        es = slope_error(name, T, r is not None) * s.abs() + 16 * U32 * (1 + v.abs()) + 2 * ev
        if name is None:
            es = torch.zeros_like(s)
        if name == "relu":                    # 0 or 1, unless v is too near 0 to tell
            es = (v.abs() <= ev).double()
        elif T == torch.bfloat16 and name == "relu2":   # below 2^-14 eight bits are kept
            es = es + 2.0 ** -14 * U[torch.bfloat16]
        elif T == torch.bfloat16 and name is not None:
            es = es + TINY[torch.float16]
        eg = D.abs() * es + 2 * U32 * g.abs()
        eg_r = eg + U[T] * (g.abs() + eg) + TINY[T]     # as the products take it

        def product(p, ep, q, count):
            val = p @ q
            e = ep @ q.abs() + (count + 8) * U32 * ((p.abs() + ep) @ q.abs())
            return val, e + U[T] * (val.abs() + e) + TINY[T]

        self.dx, self.edx = product(g, eg_r, W, n)
        self.dw, self.edw = product(g.t(), eg_r.t(), X, m)
        self.db = g.sum(0)
        e = eg.sum(0) + (m + 8) * U32 * (g.abs() + eg).sum(0)
        self.edb = e + U[T] * (self.db.abs() + e) + TINY[T]


def embedding_grad(idx, dout, vocab, scale, padding_idx):
    """The table's gradient and its bound."""
    i = idx.detach().cpu().reshape(-1).long()
    d = dout.detach().double().cpu().reshape(-1, dout.shape[-1])
    keep = (i >= 0) & (i < vocab)
    if padding_idx is not None:
        keep &= i != padding_idx
    i, d = i[keep], d[keep]
    dw = torch.zeros(vocab, d.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(dw)
    dw.index_add_(0, i, d)
    mag.index_add_(0, i, d.abs())
    count = torch.bincount(i, minlength=vocab)[:vocab].double()[:, None]
    e = abs(scale) * (count + 4) * U32 * mag
    dw = dw * scale
    return dw, e + U[dout.dtype] * (dw.abs() + e) + TINY[dout.dtype] * (count > 0)


def close(got, want, bound, what):
    """Every element within its bound; equal where the value is not finite."""
    g = got.detach().double().cpu().reshape(want.shape)
    off = (g - want).abs()
    bad = ~(off <= bound)
    if bad.any():
        at = tuple(int(t) for t in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, first at "
                             f"{at}: {g[at].item()} against {want[at].item()} +- {bound[at].item()}")

"""The recurrence of RWKV-7's time mixing as it is written, one token after the other in
64 bits, and how far a kernel in 32 bits may be from it.

The bounds are on the 2-norm of the difference over the 2-norm of the result.  A value of
the state passes through at most N = 300 roundings of 2^-24 in one chunk of 16 tokens (a
product of 64 channels for a pair of tokens, one of 64 keys and 16 tokens for S a, the
inverse's 16 rows, 32 terms of the update, and the factors e^L, whose exponents of up to 14
are sums of 16 roundings).  They fall up and down alike, so that n of them add up to sqrt(n);
the chunks' errors are carried on by a transition that does not grow them for a and b as the
model makes them, and add up alike.  A factor of 8 stands for what is above the mean:

    y and state:  8 sqrt(300 (1 + chunks)) 2^-24
    gradients:    8 sqrt(1000 (1 + chunks)) 2^-24    (both passes, the pairs and the running sums)

and the rounding to the output's type is at most half a step of it.
"""
import math

import torch

D = 64
NAMES = "rwkvab"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U32 = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


def inputs(g, *lead, dtype=torch.float32, w=None):
    """r, w, k, v, a, b of shape [*lead, 64] as the time mixing makes them."""
    def n():
        return torch.randn(*lead, D, generator=g)

    kk = torch.nn.functional.normalize(n(), dim=-1)
    r, k, v = n(), n(), n()
    x = -torch.nn.functional.softplus(2 * n()) - 0.5
    w = x if w is None else torch.full_like(x, w)
    return [t.to(dtype) for t in (r, w, k, v, -kk, kk * torch.sigmoid(n()))]


def scan(six, state):
    """(y, last state) in float64 of [batch, time, heads, 64]."""
    r, w, k, v, a, b = six
    decay = torch.exp(-torch.exp(w))
    ys = []
    for t in range(r.shape[1]):
        sa = (state * a[:, t, :, None, :]).sum(-1, keepdim=True)
        state = state * decay[:, t, :, None, :] + sa * b[:, t, :, None, :] + v[:, t, :, :, None] * k[:, t, :, None, :]
        ys.append((state * r[:, t, :, None, :]).sum(-1))
    return (torch.stack(ys, 1) if ys else r * 1), state


def packed(six, state, lens):
    """The same of packed sequences: y is 0 behind the last."""
    ys, states, at = [], [], 0
    for i, n in enumerate(lens):
        y, s = scan([x[:, at:at + n] for x in six], state[i:i + 1])
        ys.append(y)
        states.append(s)
        at += n
    ys.append(six[0][:, at:] * 0)
    return torch.cat(ys, 1), torch.cat(states, 0)


def reference(six, state, dy=None, dstate=None, lens=None):
    """{"y", "state"} and, with dy, the gradients {"dr", ... "dstate"}, all in float64."""
    six = [x.detach().double().cpu().requires_grad_(dy is not None) for x in six]
    first = state.detach().double().cpu().requires_grad_(dy is not None)
    y, last = scan(six, first) if lens is None else packed(six, first, lens)
    out = {"y": y.detach(), "state": last.detach()}
    if dy is not None:
        loss = (y * dy.double().cpu()).sum()
        if dstate is not None:
            loss = loss + (last * dstate.double().cpu()).sum()
        got = torch.autograd.grad(loss, [*six, first], allow_unused=True)
        for name, x, t in zip([*NAMES, "state"], [*six, first], got):
            t = torch.zeros_like(x) if t is None else t
            # d decay / dw is 0 where the decay is 0 for an infinite w (inf * 0 above)
            out["d" + name] = t.nan_to_num(0.0) if name == "w" else t
    return out


def bound(what, dtype, time):
    chunks = -(-time // 16)
    n = 1000 if what.startswith("d") else 300
    return U[dtype] + 8 * math.sqrt(n * (1 + chunks)) * U32


def close(got, want, what, time):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.numel():
        return
    got64 = got.detach().double().cpu()
    assert got64.isfinite().all(), f"{what}: not finite"
    norm = want.norm().item()
    off = (got64 - want).norm().item()
    e = bound(what, got.dtype, time)
    assert off <= e * norm + 1e-30, f"{what}: off by {off / max(norm, 1e-30):.3g} of its norm, bound {e:.3g}"

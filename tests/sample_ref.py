"""The sampler's definition in float64, row by row, by sorting."""
import math

import torch


def sample_row(logits, u, temperature, top_k, top_p, min_p):
    """(token, log-probability, indices that stay in the order of their logits)."""
    l = logits.double().cpu()
    if l.isnan().any() or not (l > -math.inf).any():
        return -1, math.nan, []
    index = torch.nonzero(l > -math.inf)[:, 0]
    order = index[torch.sort(l[index], descending=True, stable=True).indices]
    if not temperature > 0:
        order = order[:1]
        temperature = 1.0
    z = (l[order] - l[order[0]]) / temperature
    if l[order[0]] == math.inf:   # those that are infinite share everything, at any temperature
        z = torch.where(l[order] == math.inf, 0.0, -math.inf).double()
    if top_k > 0:
        order, z = order[:top_k], z[:top_k]
    e = torch.exp(z)
    if top_p < 1:
        keep = e.cumsum(0) - e < max(top_p, 1e-30) * e.sum()
        order, z, e = order[keep], z[keep], e[keep]
    keep = e >= min(min_p, 1.0)
    order, z, e = order[keep], z[keep], e[keep]
    by_index = torch.sort(order).indices
    upto = e[by_index].cumsum(0)
    whole = upto[-1]
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    at = int((upto <= u * whole).sum())
    # u of 1 and more: the last that has any share
    at = min(at, int((e[by_index] > 2.0 ** -37).nonzero()[-1]))
    at = by_index[at]
    return int(order[at]), float(z[at] - math.log(whole)), order.tolist()


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = u.numel()

    def of(x):
        return x.flatten().tolist() if isinstance(x, torch.Tensor) else [float(torch.tensor(x, dtype=torch.float32))] * rows

    got = [sample_row(l, v, t, int(k), p, m) for l, v, t, k, p, m in
           zip(logits.reshape(rows, -1), u.flatten().tolist(), of(temperature), of(top_k), of(top_p), of(min_p))]
    return (torch.tensor([x[0] for x in got]).view(u.shape),
            torch.tensor([x[1] for x in got], dtype=torch.float64).view(u.shape))

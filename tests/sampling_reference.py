"""The pick of a token by chance in 64 bits, from its definition."""
import math

import torch


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, logarithm of its probability, distance of u from the next border of the set's sums)."""
    x = torch.where(torch.isnan(x.double()), -math.inf, x.double())
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    temperature, top_p, min_p, u = f32(temperature), f32(top_p), f32(min_p), f32(u)
    value, index = torch.sort(x, descending=True, stable=True)
    n = int((value > -math.inf).sum())
    if n == 0:
        return -1, -math.inf, math.inf
    value, index = value[:n], index[:n]
    if temperature == 0 or top_p <= 0:
        top_k = 1
    z = torch.where(value == value[0], 0.0, (value - value[0]) / (temperature or 1.0))
    keep = top_k if 0 < top_k < len(x) else n
    z, index = z[:keep], index[:keep]
    if min_p > 0:
        keep = int((z >= math.log(min(min_p, 1.0))).sum())
        z, index = z[:keep], index[:keep]
    w = z.exp()
    if top_p < 1:
        sums = w.cumsum(0)
        keep = max(1, int((sums - w < top_p * sums[-1]).sum()))
        z, w, index = z[:keep], w[:keep], index[:keep]
    order = index.argsort()
    z, w, index = z[order], w[order], index[order]
    sums = w.cumsum(0)
    total = float(sums[-1])
    goal = max(u, 0.0) * total if u == u else 0.0
    at = int((sums <= goal).sum())
    if at >= len(w) or u >= 1:
        at = int((w > 0).nonzero()[-1])
    border = float((sums / total - (u if u == u else 0.0)).abs().min())
    return int(index[at]), float(z[at]) - math.log(total), border

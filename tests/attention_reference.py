"""Attention over chosen keys in 64 bits, and how far a kernel may be from it.

A kernel that rounds P to bf16 for the product with V and its result to bf16 is off by at most
    sum_j p_j |v_j| 2^-8 / sum_j p_j  +  2^-8 |result|
(half a step of bf16 each, relative to the value). Its fp32 scores add 128 products, each sum off by at most
2^-24 of what it holds: below 128 * 2^-24 * scale * sum |q_i k_i| < 1e-4 for the inputs here (unit normals:
scale * sum |q_i k_i| < 12), which moves p_j by 1e-4 relative, 2.6 % of 2^-8; exp2 and the fp32 sums are far below
that. 5 % on top covers them."""
import torch

HALF_STEP = 2.0 ** -8


def attend(q, k, v, visible, scale):
    """q [rows, 128], k / v [keys, 128], visible [rows, keys] -> (result, bound) in 64 bits; rows that see nothing
    are zero."""
    q, k, v = q.double(), k.double(), v.double()
    v = torch.where(visible.any(0)[:, None], v, 0.0)        # what nobody sees may be NaN
    k = torch.where(visible.any(0)[:, None], k, 0.0)
    s = (q @ k.T * scale).masked_fill(~visible, -torch.inf)
    top = s.amax(1, keepdim=True) if s.shape[1] else torch.full((q.shape[0], 1), -torch.inf, dtype=torch.float64)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    return out, 1.05 * HALF_STEP * (p @ v.abs() + out.abs()) + 1e-6


def window_visible(at, keys, window, sinks):
    """[rows, keys]: what rows at the positions `at` see of `keys` keys."""
    at, j = torch.as_tensor(at)[:, None], torch.arange(keys)[None]
    return (j <= at) & ((j > at - window) | (j < sinks))


def assert_close(got, want, bound):
    got = got.double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() / bound
    assert over.max().item() <= 1, f"{over.max().item():.3f} of the bound at {over.argmax().item()}"

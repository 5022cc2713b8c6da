"""Attention inputs whose only error above the last bits of f32 would be a
rounding of the probabilities, and the bound that holds them.

Query head g of a group is the unit vector of dim g, so its score of a slot is
one element of the key, exactly, whatever the order of the sum; scores are
multiples of 1/64 in [-1, 1] (scale 1), probabilities differ by less than e^2,
and values lie in [1, 2), where half a step of the output's type is eps / 2.

Relative error of an output before its rounding:
  scores        |s| <= 1.4427 in base 2: the constant, the product and the
                difference to the maximum round by 2^-24 each, of 2.9 at most:
                3 * 2.9 * ln 2 * 2^-24 = 2^-21.4 of p, with ex2.approx's 2^-22
                2^-20.7 of p, the same of l
  l             up to 20 sums of positive numbers: 20 * 2^-24 = 2^-19.7
  the quotient  2^-23
                together less than 2^-18
  P V           n slots take 2 ceil(n / 16) tile products (high and low parts),
                each a sum of 17 numbers, not more than 2^-23 of it lost a number
  P             16 bits or more, 2^-16, as the operator promises
"""
import torch


def fill(c, group, seed=0):
    """Keys and values of a cache's (paged_ref.Cache) held slots, and queries [rows, heads * head_dim] on the CPU."""
    g = torch.Generator().manual_seed(seed)
    k, v = c.k.cpu(), c.v.cpu()
    held = ~torch.isnan(k[..., 0])
    keys = torch.zeros(int(held.sum()), c.D, dtype=torch.float64)
    keys[:, :group] = torch.randint(-64, 65, (keys.shape[0], group), generator=g).double() / 64
    k[held] = keys.to(c.dtype)
    steps = round(1 / torch.finfo(c.dtype).eps)
    v[held] = (1 + torch.randint(0, steps, (keys.shape[0], c.D), generator=g).double() / steps).to(c.dtype)
    c.k, c.v = k.to(c.k.device), v.to(c.v.device)
    return torch.eye(group, c.D).repeat(len(c.lens), c.H, 1).reshape(len(c.lens), -1).to(c.dtype)


def answers(c, group):
    """For each sequence: probabilities [kv_heads, group, n] and values [kv_heads, n, head_dim], float64."""
    for b in range(len(c.lens)):
        k = torch.stack([c.rows(c.k, b, h) for h in range(c.H)])
        v = torch.stack([c.rows(c.v, b, h) for h in range(c.H)])
        yield torch.softmax(k[..., :group].transpose(1, 2), -1), v


def bound(c, b):
    """What an output of sequence b may be off, rounded to the cache's type."""
    rel = 2.0 ** -18 + 2 * -(-c.lens[b] // 16) * 17 * 2.0 ** -23 + 2.0 ** -16
    return torch.finfo(c.dtype).eps / 2 + 2 * rel

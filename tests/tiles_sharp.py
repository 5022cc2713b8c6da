"""The bound of tests/paged_sharp.py (inputs whose only error above the last bits
of f32 would be a rounding of the probabilities) for the attention tiles' units of
few rows, which multiply what rounding P leaves as a second operand.

Relative error of an output before its rounding, where it differs from there:
  scores        the exponent is s log2 e + (u - m) with u = 8 for f16 (P is held
                2^8 higher): constant, m, difference and sum round by 2^-24 of
                at most 11 each, 4 * 11 * ln 2 * 2^-24 = 2^-19.0 of p, with
                ex2.approx's 2^-22 2^-18.9 of p, the same of l
  l             64 keys are 16 sums in each of four places and two more, a
                sequence's up to two blocks of 64 in each of up to eight places, and
                the places' sums: 50 * 2^-24 = 2^-18.3, with ex2 and a product for
                each place 2^-18.0
  the quotient  a reciprocal and two products, 2^-22
                together less than 2^-16.6
  P             rounded to nearest, and what that leaves rounded to nearest:
                2^-8 * 2^-8 in bf16, less in f16
"""
import torch

from tests import paged_sharp as sharp


def held(c, sequence):
    """Keys and values [kv_heads, n, head_dim] of a sequence's held slots, float64."""
    return [torch.stack([c.rows(pool, sequence, h) for h in range(c.H)]) for pool in (c.k, c.v)]


def answers(k, v, group, slots):
    """Probabilities [kv_heads, group, n] of those slots, and their values."""
    return torch.softmax(k[:, slots, :group].transpose(1, 2), -1), v[:, slots]


def bound(c, n):
    """What an output over n slots may be off, rounded to the cache's type."""
    rel = 2.0 ** -16.6 + 2 * -(-n // 16) * 17 * 2.0 ** -23 + 2.0 ** -16
    return torch.finfo(c.dtype).eps / 2 + 2 * rel


def queries(c, group, rows):
    """For every row the unit vectors of fill."""
    return torch.eye(group, c.D).repeat(rows, c.H, 1).reshape(rows, -1).to(c.dtype)


fill = sharp.fill

"""Softmax attention in 64 bits for rows whose small weights count, with a bound that allows little for them."""
import torch

from tests import _serving_ref as ref


def attend_rows(q, k, v, scale, dtype, weights):
    """softmax(scale q k^T) v for query rows q (n, d) that all see the keys k / v (t, d) of one head, in 64 bits: (out, bound).

    A weight is rounded once to `weights`' type: off by half a step of itself, and in fp16, where it lies below 2^-14, by at most
    2^-25; the largest of a row stands at 2^7 or above, so that is 2^-32 of the largest weight, whatever scales the values
    have (the ratios here stay within the 2^7 above and 2^15 below the first page's).  A score is off by (d + 4) 2^-24 of the
    sum of |q k|, twice (numerator and denominator); the exponentials and sums add a few 2^-22."""
    s = scale * (q @ k.t())
    p = torch.softmax(s, -1)
    out = p @ v
    mass = p @ v.abs()
    score = (q.shape[1] + 4) * 2.0 ** -24 * scale * (q.abs() @ k.abs().t()).amax(1, keepdim=True)
    lost = 2.0 ** -32 * p.amax(1, keepdim=True) * v.abs().sum(0) if weights == torch.float16 else 0.0
    return out, (ref.eps(weights) + 2 * score + 2.0 ** -20) * mass + lost + ref.eps(dtype) * out.abs() + 2.0 ** -25

"""Plain restatements, in 64 bits on the CPU, of the operators that serve a quantised decoder, with the bounds that
their roundings have."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def eps(dtype):
    """Largest relative error of one rounding: half a step."""
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, first, scale, dtype, vmax=None):
    """softmax(scale q k^T) v for q (n, hq, d), k / v (t, hkv, d) in 64 bits; query i sees keys 0..first + i (all: None).
    Returns (out, bound): |kernel - out| <= bound elementwise, for weights rounded once to a type of 11 bits (8 for
    bfloat16 weights), products exact, sums in 32 bits and one rounding to `dtype` at the end.

    The weights w <= 1 carry a relative error u (and, where they are subnormal in fp16, an absolute one of 2^-25), so the
    numerator is off by u sum p|v| + 2^-25 sum |v| in units of the largest weight; a score is a sum of d products in 32
    bits, off by (d + 4) 2^-24 sum |q k| scale, which moves a weight and the denominator by that much each, relatively;
    the exponential and the sums add a few 2^-22."""
    n, hq, d = q.shape
    t, hkv = k.shape[:2]
    u = eps(dtype) if vmax is None else 2.0 ** -11
    out, bound = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = scale * (q[:, h] @ kk.t())
        see = torch.ones(n, t, dtype=torch.bool) if first is None else torch.arange(t)[None] <= first + torch.arange(n)[:, None]
        s = s.masked_fill(~see, -math.inf)
        some = see.any(1)
        p = torch.zeros(n, t, dtype=torch.float64)
        p[some] = torch.softmax(s[some], -1)
        # a masked value takes no part, whatever it is
        for i in range(n) if not torch.isfinite(vv).all() else []:
            out[i, h] = p[i, see[i]] @ vv[see[i]]
        if torch.isfinite(vv).all():
            out[:, h] = p @ vv
        va = torch.nan_to_num(vv.abs(), 0, 0, 0)
        mass = p @ va
        score = (d + 4) * 2.0 ** -24 * scale * (q[:, h].abs() @ kk.abs().t()).masked_fill(~see, 0).amax(1, keepdim=True) if t else torch.zeros(n, 1)
        tiny = 2.0 ** -25 * (see.double() @ va if vmax is None else (see.double() @ (va / vmax[:, h // (hq // hkv), None])) * vmax.max())
        bound[:, h] = (u + 2 * score + 2.0 ** -20) * mass + tiny + eps(dtype) * out[:, h].abs() + 2.0 ** -24
    # fp16 outputs are subnormal below 2^-14: half a step there is 2^-25
    return out, bound * 1.02


def rotate(x, pos, cos, sin, interleaved):
    """x (t, heads, d) by rows of the fp32 tables, in 32 bits, each operation rounded once"""
    x, rot = x.float().clone(), 2 * cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    lo = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    hi = lo + 1 if interleaved else lo + rot // 2
    a, b = x[..., lo].clone(), x[..., hi].clone()
    x[..., lo] = a * c - b * s
    x[..., hi] = b * c + a * s
    return x


def exponent(amax):
    """smallest e >= -100 with amax 2^-e <= 448"""
    if amax == 0:
        return -100
    e = math.ceil(math.log2(amax / 448.0)) - 2
    while amax * 2.0 ** -e > 448.0:
        e += 1
    return min(120, max(-100, e))


def encode(x):
    """float -> e4m3, infinities at the ends"""
    return x.clamp(-448.0, 448.0).to(E4M3)   # clamp keeps NaN


class Cache:
    """The cache as a list of pages, appended to token run by token run."""

    def __init__(self, n_pages, heads, page, d):
        self.page = page
        self.k = torch.zeros(n_pages, heads, page, d).to(E4M3)
        self.v = torch.zeros(n_pages, heads, d, page).to(E4M3)
        self.ks, self.vs = torch.ones(n_pages, heads), torch.ones(n_pages, heads)

    def append(self, k, v, table, past, cu, max_pos=None):
        """k (rotated) / v in fp32"""
        for b in range(len(past)):
            if past[b] < 0:
                continue
            n = cu[b + 1] - cu[b]
            end = past[b] + n if max_pos is None else min(past[b] + n, max_pos)
            for first in range(past[b] // self.page * self.page, end, self.page):
                s0, s1 = max(0, past[b] - first), min(self.page, end - first)
                if s1 <= s0 or first // self.page >= table.shape[1]:
                    continue
                pid = int(table[b, first // self.page])
                if not 0 <= pid < self.k.shape[0]:
                    continue
                r0 = cu[b] + first + s0 - past[b]
                for h in range(k.shape[1]):
                    for x, codes, scale in ((k[r0:r0 + s1 - s0, h], self.k[pid, h], self.ks), (v[r0:r0 + s1 - s0, h], self.v[pid, h].t(), self.vs)):
                        fin = x[torch.isfinite(x)].abs()
                        e = exponent(float(fin.max()) if fin.numel() else 0.0)
                        if s0:
                            old = float(scale[pid, h])
                            e = max(e, round(math.log2(old)))
                            codes[:s0] = encode(codes[:s0].float() * (old * 2.0 ** -e))
                        codes[s0:s1] = encode(x * 2.0 ** -e)
                        scale[pid, h] = 2.0 ** e

    def tokens(self, table, n):
        """the first n tokens of one sequence, (n, heads, d) in 64 bits, and the value scale of each (n, heads)"""
        ids = [int(i) for i in table[:-(-n // self.page)]]
        k = torch.cat([(self.k[i].double() * self.ks[i].double()[:, None, None]).transpose(0, 1) for i in ids])[:n]
        v = torch.cat([(self.v[i].double() * self.vs[i].double()[:, None, None]).permute(2, 0, 1) for i in ids])[:n]
        return k, v, torch.cat([self.vs[i].double()[None].expand(self.page, -1) for i in ids])[:n]


def log_probs(logits, tokens, top):
    """(logprob, entropy, top logprob, top token) in 64 bits; top by a stable sort"""
    x = logits.double()
    lp = torch.log_softmax(x, -1)
    ent = -torch.where(lp > -math.inf, lp.exp() * lp, torch.zeros((), dtype=torch.float64)).sum(-1)
    ent = torch.where(torch.isnan(lp).any(-1), torch.full_like(ent, math.nan), ent)
    order = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :top]
    return lp.gather(1, tokens[:, None])[:, 0], ent, lp.gather(1, order), order

"""The operators that serve a quantised decoder, as measurable cases: attention over a whole prompt (packed sequences,
grouped heads), appending rotated keys and values to a paged 8-bit cache, attention over that cache, and the log
probabilities of tokens with entropy and top alternatives.

``own`` False computes each in its plain form (elementary torch operations in 32 bits, rounded once at the end), True
through the framework's entry points.  A case is a dict of plain values; ``op`` says which operator it is of."""
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_E4M3_MAX = 448.0
_MIN_EXP = -100   # exponent of the scale of a block of zeros


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one short text of a 12-head model with heads of 64: latency counts
        {"name": "prompt short 77", "op": "prompt", "lens": "77", "hq": 12, "hkv": 12, "d": 64, "causal": True, "dtype": "f16"},
        # a calibration batch of the block walk: 4 sequences of 2048 tokens, 32 heads of 128
        {"name": "prompt 4x2048", "op": "prompt", "lens": "2048,2048,2048,2048", "hq": 32, "hkv": 32, "d": 128, "causal": True, "dtype": "f16"},
        # requests of many lengths packed into one prefill, 64 heads on 8
        {"name": "prompt packed ragged", "op": "prompt", "lens": "1,17,3001,256,799,64,1500,333,2049,5,127,700", "hq": 64, "hkv": 8, "d": 128,
         "causal": True, "dtype": "bf16"},
        # one long document
        {"name": "prompt long 16384", "op": "prompt", "lens": "16384", "hq": 32, "hkv": 8, "d": 128, "causal": True, "dtype": "bf16"},
        # one new token for each of 64 running requests, into half-filled pages
        {"name": "append 64x1", "op": "append", "batch": 64, "past": 400, "new": 1, "mix": 1, "hq": 64, "hkv": 8, "d": 128, "page": 64, "rot": 128,
         "interleaved": False, "dtype": "bf16"},
        # a prefill of 8 prompts with different lengths, all heads of their own
        {"name": "append prefill ragged", "op": "append", "batch": 8, "past": 0, "new": 2048, "mix": 2, "hq": 32, "hkv": 32, "d": 128, "page": 64, "rot": 128,
         "interleaved": False, "dtype": "f16"},
        # a chunk behind a prefix, small pages, interleaved pairs over part of the head
        {"name": "append chunk partial", "op": "append", "batch": 3, "past": 77, "new": 511, "mix": 3, "hq": 16, "hkv": 4, "d": 64, "page": 16, "rot": 32,
         "interleaved": True, "dtype": "bf16"},
        # the first tokens of one conversation: latency counts
        {"name": "paged 1x100", "op": "paged", "batch": 1, "ctx": 100, "nq": 1, "mix": 1, "hq": 32, "hkv": 32, "d": 128, "page": 16, "dtype": "f16"},
        # 64 running requests of up to 8192 tokens, 64 heads on 8
        {"name": "paged 64x8192", "op": "paged", "batch": 64, "ctx": 8192, "nq": 1, "mix": 2, "hq": 64, "hkv": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # one very long conversation, four tokens checked at once
        {"name": "paged 1x131071", "op": "paged", "batch": 1, "ctx": 131071, "nq": 4, "mix": 3, "hq": 64, "hkv": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # a sampler's step: one row of logits, five alternatives
        {"name": "logprobs 1x32000", "op": "logprobs", "rows": 1, "vocab": 32000, "top": 5, "dtype": "f16"},
        # scoring of two sequences of 2048 tokens on a 50272-word vocabulary with the alternatives beside
        {"name": "logprobs 4096x50272", "op": "logprobs", "rows": 4096, "vocab": 50272, "top": 10, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["prompt", "append", "paged", "logprobs"])
    dtype = rng.choice(["f16", "bf16"])
    hkv, group = rng.choice([1, 2, 4, 8, 12, 32]), rng.choice([1, 2, 4, 5, 8])
    while hkv * group > 64:
        hkv, group = rng.choice([1, 2, 4, 8, 12, 32]), rng.choice([1, 2, 4, 5, 8])
    hq = hkv * group
    if op == "prompt":
        lens = [_log_int(rng, 1, 4096) for _ in range(rng.choice([1, 1, 2, 3, 5, 9, 16]))]
        if len(lens) == 1:
            lens = [_log_int(rng, 16, 16384)]
        case = {"op": op, "lens": ",".join(map(str, lens)), "hq": hq, "hkv": hkv, "d": rng.choice([64, 80, 96, 128]), "causal": rng.random() < 0.8, "dtype": dtype}
        while work(case)["flops"] > 2.1e12:   # no more than the longest listed one
            lens = [(n + 1) // 2 + 1 for n in lens]
            case["lens"] = ",".join(map(str, lens))
        return case
    if op == "append":
        d = rng.choice([64, 80, 96, 128])
        batch = _log_int(rng, 1, 128)
        new = rng.choice([1, 1, _log_int(rng, 1, max(1, 16384 // batch))])
        return {"op": op, "batch": batch, "past": rng.choice([0, rng.randint(1, 700)]), "new": new, "mix": rng.randint(1, 1 << 20), "hq": hq, "hkv": hkv, "d": d,
                "page": rng.choice([16, 32, 64, 128]), "rot": rng.choice([d, d, d // 2, 16]), "interleaved": rng.random() < 0.3, "dtype": dtype}
    if op == "paged":
        d = rng.choice([64, 80, 96, 128])
        batch = _log_int(rng, 1, 128)
        ctx = _log_int(rng, 1, min(131072, max(64, (1 << 29) // (batch * hkv * d))))
        return {"op": op, "batch": batch, "ctx": ctx, "nq": rng.choice([1, 1, 1, rng.randint(2, 16)]), "mix": rng.randint(1, 1 << 20), "hq": hq, "hkv": hkv,
                "d": d, "page": rng.choice([16, 32, 64, 128]), "dtype": dtype}
    vocab = rng.randint(1000, 160000)
    return {"op": op, "rows": _log_int(rng, 1, max(1, 200_000_000 // vocab)), "vocab": vocab, "top": rng.choice([0, 1, 5, 10, 20]),
            "dtype": rng.choice(["f16", "bf16", "f32"])}


def _lens(case):
    """(tokens already there, new tokens) of each sequence, from the case alone."""
    rng = random.Random(case["mix"])
    if case["op"] == "append":
        past = [rng.randint(max(0, case["past"] // 2), case["past"]) for _ in range(case["batch"])]
        new = [case["new"] if case["new"] == 1 else rng.randint(max(1, case["new"] // 4), case["new"]) for _ in range(case["batch"])]
        return past, new
    total = [case["ctx"]] + [rng.randint(1, case["ctx"]) for _ in range(case["batch"] - 1)]
    return [max(0, t - case["nq"]) for t in total], [min(case["nq"], t) for t in total]


# ---- inputs --------------------------------------------------------------------------------------------------------

def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _pages(case, gen, past, new):
    """A block table over a shuffled pool with as many pages as the sequences take."""
    page = case["page"]
    counts = [(p + n + page - 1) // page for p, n in zip(past, new)]
    n_pages, width = sum(counts), max(max(counts), 1)
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    have = torch.tensor(counts, device="cuda")
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None] < have[:, None]] = order
    return n_pages, table


def _pow2(e):
    """2^e in 32 bits, exactly, for -126 <= e <= 127"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The smallest e with amax * 2^-e <= 448 (= 0.875 * 2^9), of an amax >= 0"""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (m > 0.875).to(x.dtype), torch.full_like(x, _MIN_EXP)).clamp(min=_MIN_EXP)


def _cache(case, gen, n_pages):
    """Pages of keys and values with outlying channels, as projections give them: codes and power-of-two scales."""
    hkv, d, page = case["hkv"], case["d"], case["page"]
    channel = torch.exp(0.5 * _normal(gen, hkv, d))
    out = []
    for key in (True, False):
        codes = torch.empty((n_pages, hkv, page, d) if key else (n_pages, hkv, d, page), dtype=_E4M3, device="cuda")
        scale = torch.empty(n_pages, hkv, device="cuda")
        for lo in range(0, n_pages, 2048):   # in pieces: the pool may be large
            hi = min(n_pages, lo + 2048)
            x = _normal(gen, hi - lo, hkv, page, d) * channel[:, None, :]
            e = _exponent(x.abs().amax((2, 3)))
            codes[lo:hi] = ((x if key else x.transpose(2, 3)) * _pow2(-e)[:, :, None, None]).to(_E4M3)
            scale[lo:hi] = _pow2(e)
        out += [codes, scale]
    return {"k8": out[0], "ks": out[1], "v8": out[2], "vs": out[3]}


def _merged(gen, tokens, case, dtype):
    """q, k, v as the slices of one merged product, as the block walk has them."""
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = _normal(gen, tokens, hq + 2 * hkv, d)
    x[:, :hq + hkv] *= torch.exp(0.3 * _normal(gen, 1, hq + hkv, d))
    x = x.to(dtype)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = _TYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "prompt":
        lens = [int(n) for n in case["lens"].split(",")]
        st["lens"], st["cu"] = lens, _cu(lens)
        st["q"], st["k"], st["v"] = _merged(gen, sum(lens), case, dtype)
    elif case["op"] == "append":
        past, new = _lens(case)
        n_pages, st["table"] = _pages(case, gen, past, new)
        st.update(_cache(case, gen, n_pages))
        st["past"], st["cu"] = torch.tensor(past, dtype=torch.int32, device="cuda"), _cu(new)
        st["single"] = case["new"] == 1
        st["q"], st["k"], st["v"] = _merged(gen, sum(new), case, dtype)
        # tables of the positions' angles, made once as a program does
        freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        ang = torch.arange(max(p + n for p, n in zip(past, new)), dtype=torch.float64, device="cuda")[:, None] * freq
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    elif case["op"] == "paged":
        past, new = _lens(case)
        n_pages, st["table"] = _pages(case, gen, past, new)
        st.update(_cache(case, gen, n_pages))
        st["lens"], st["cu"] = torch.tensor([p + n for p, n in zip(past, new)], dtype=torch.int32, device="cuda"), _cu(new)
        st["single"] = case["nq"] == 1
        st["q"] = _normal(gen, sum(new), case["hq"], case["d"]).to(dtype)
        st["most"] = max(new)
    else:
        # a few likely words above a broad rest
        x = 2.0 * _normal(gen, case["rows"], case["vocab"])
        x += 4.0 * torch.exp(_normal(gen, case["rows"], 1)) * (torch.rand(x.shape, generator=gen, device="cuda") < 3e-4)
        st["logits"] = x.to(dtype)
        st["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda")
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _plain_prompt(st):
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda")
    at = 0
    for n in st["lens"]:
        q = st["q"][at:at + n].float().view(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, hq // hkv * n, d)
        k = st["k"][at:at + n].float().permute(1, 2, 0)
        v = st["v"][at:at + n].float().transpose(0, 1)
        s = torch.matmul(q, k).view(hkv, hq // hkv, n, n).mul_(d ** -0.5)
        if case["causal"]:
            s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu_(1), float("-inf"))
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(hkv, hq // hkv * n, n), v).view(hkv, hq // hkv, n, d) / total
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, hq, d)
        at += n
    return out


def _rotated(x, cos, sin, rot, interleaved):
    """x (tokens, heads, d) in 32 bits, cos / sin (tokens, rot / 2)"""
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(st):
    case = st["case"]
    page, hkv, d = case["page"], case["hkv"], case["d"]
    n_pages, tokens = st["k8"].shape[0], st["k"].shape[0]
    seq = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), st["cu"].diff(), output_size=tokens)
    pos = st["past"][seq] + torch.arange(tokens, device="cuda") - st["cu"][seq]
    where, slot = st["table"][seq, pos // page].long(), pos % page
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotated(st["q"].float(), cos, sin, case["rot"], case["interleaved"]).to(st["q"].dtype)
    k = _rotated(st["k"].float(), cos, sin, case["rot"], case["interleaved"])
    # the page that each sequence goes on in, and how many of its tokens it holds
    open_, held = st["table"].gather(1, (st["past"] // page).long()[:, None])[:, 0].long(), st["past"] % page
    kept = torch.arange(page, device="cuda") < held[:, None]                       # (batch, page)
    for x, codes, scale, key in ((k, st["k8"], st["ks"], True), (st["v"].float(), st["v8"], st["vs"], False)):
        e = torch.full((n_pages, hkv), _MIN_EXP, dtype=torch.int32, device="cuda")
        old = torch.frexp(scale[open_])[1] - 1                                     # (batch, hkv)
        e[open_] = torch.where((held > 0)[:, None], old, e[open_])
        amax = torch.zeros(n_pages, hkv, device="cuda").scatter_reduce_(0, where[:, None].expand(tokens, hkv), x.abs().amax(-1), "amax")
        e = torch.maximum(e, _exponent(amax))
        # tokens that are there already are re-expressed in a scale that has grown
        flat = codes.view(torch.uint8)
        before = flat[open_]
        again = (before.view(_E4M3).float() * _pow2(old - e[open_])[:, :, None, None]).to(_E4M3).view(torch.uint8)
        flat[open_] = torch.where(kept[:, None, :, None] if key else kept[:, None, None, :], again, before)
        scale[where] = _pow2(e[where])
        y = (x * _pow2(-e[where])[:, :, None]).to(_E4M3).view(torch.uint8)
        if key:
            flat[where, :, slot] = y
        else:
            flat[where, :, :, slot] = y
    return {"q": q, "k8": st["k8"], "ks": st["ks"], "v8": st["v8"], "vs": st["vs"]}


def _plain_paged(st):
    case = st["case"]
    hq, hkv, d, page, b, nq = case["hq"], case["hkv"], case["d"], case["page"], case["batch"], st["most"]
    g, ctx = hq // hkv, st["table"].shape[1] * page
    table = st["table"].clamp(min=0).long()
    k = st["k8"].view(torch.uint8)[table].view(_E4M3).float().mul_(st["ks"][table][..., None, None])      # (b, pages, hkv, page, d)
    k = k.permute(0, 2, 4, 1, 3).reshape(b, hkv, d, ctx)
    new = st["cu"].diff()
    row = torch.arange(nq, device="cuda")
    real = row[None] < new[:, None]                                                # (b, nq)
    q = torch.zeros(b, nq, hq, d, device="cuda")
    q[real] = st["q"].float()
    q = q.view(b, nq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * nq, d)
    s = torch.matmul(q, k).view(b, hkv, g, nq, ctx).mul_(d ** -0.5)
    del k
    last = (st["lens"] - new)[:, None] + row                                       # position of each query token
    s.masked_fill_((torch.arange(ctx, device="cuda") > last[..., None])[:, None, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    v = st["v8"].view(torch.uint8)[table].view(_E4M3).float().mul_(st["vs"][table][..., None, None])       # (b, pages, hkv, d, page)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, hkv, ctx, d)
    o = torch.matmul(s.view(b, hkv, g * nq, ctx), v).view(b, hkv, g, nq, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(b, nq, hq, d)[real].to(st["q"].dtype)


def _plain_logprobs(st):
    x, top = st["logits"].float(), st["case"]["top"]
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1)
    log_total = total.log()
    res = {"logprob": x.gather(1, st["tokens"][:, None])[:, 0] - log_total, "entropy": log_total - (e * x).sum(-1) / total}
    if top:
        order = torch.sort(st["logits"], dim=-1, descending=True, stable=True)[1][:, :top]
        res["top_logprob"], res["top_token"] = x.gather(1, order) - log_total[:, None], order
    return res


# ---- the calls -----------------------------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if not own:
        with torch.no_grad():
            return {"prompt": _plain_prompt, "append": _plain_append, "paged": _plain_paged, "logprobs": _plain_logprobs}[op](st)
    from gptq_v2_amd import ops
    if op == "prompt":
        return ops.attention_prompt(st["q"], st["k"], st["v"], st["cu"], causal=st["case"]["causal"])
    if op == "logprobs":
        r = ops.token_logprobs(st["logits"], st["tokens"], top=st["case"]["top"])
        res = {"logprob": r.logprob, "entropy": r.entropy}
        return dict(res, top_logprob=r.top_logprob, top_token=r.top_token) if st["case"]["top"] else res
    cache = ops.PagedCache(st["k8"], st["v8"], st["ks"], st["vs"])
    cu = None if st["single"] else st["cu"]   # None: one token for each sequence
    if op == "paged":
        return ops.attention_paged(st["q"], cache, st["table"], st["lens"], cu)
    q = ops.kv_append(cache, st["k"], st["v"], st["table"], st["past"], cu, q=st["q"], cos=st["cos"], sin=st["sin"], interleaved=st["case"]["interleaved"])
    return {"q": q, "k8": st["k8"], "ks": st["ks"], "v8": st["v8"], "vs": st["vs"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    if case["op"] == "prompt":
        lens = [int(n) for n in case["lens"].split(",")]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * (2 * case["hq"] + 2 * case["hkv"]) * case["d"] * 2, "flops": 4 * case["d"] * case["hq"] * pairs}
    if case["op"] == "append":
        past, new = _lens(case)
        t, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["d"]
        # q in and out, k and v in 16 bits, codes out; the angles once
        return {"bytes": t * (4 * hq * d + 4 * hkv * d + 2 * hkv * d) + t * case["rot"] * 4, "flops": 3 * t * (hq + hkv) * case["rot"]}
    if case["op"] == "paged":
        past, new = _lens(case)
        # each query token sees the keys up to its own position; the cache is read once
        seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
        cached = sum(p + n for p, n in zip(past, new))
        return {"bytes": cached * case["hkv"] * case["d"] * 2 + 4 * sum(new) * case["hq"] * case["d"], "flops": 4 * seen * case["hq"] * case["d"]}
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 6 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _attend(q, k, v, first):
    """q (n, hq, d), k / v (t, hkv, d) in 64 bits; query i sees the keys up to first + i (all where first is None)."""
    n, hq, d = q.shape
    t, hkv = k.shape[:2]
    out = torch.empty(n, hq, d, dtype=torch.float64, device=q.device)
    for h in range(hq):
        j = h // (hq // hkv)
        for lo in range(0, n, 4096):
            hi = min(n, lo + 4096)
            s = q[lo:hi, h] @ k[:, j].t() / math.sqrt(d)
            if first is not None:
                s = s.masked_fill(torch.arange(t, device=q.device)[None] > first + torch.arange(lo, hi, device=q.device)[:, None], -math.inf)
            out[lo:hi, h] = torch.softmax(s, -1) @ v[:, j]
    return out


def _turn(x, pos, rot, interleaved):
    """x (t, heads, d) in 64 bits, by the angles of its positions"""
    pair = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    ang = pos.double()[:, None] * torch.exp(-2 * pair / rot * math.log(10000.0))
    z = torch.polar(torch.ones_like(ang), ang)[:, None]
    lo = 2 * torch.arange(rot // 2, device=x.device) if interleaved else torch.arange(rot // 2, device=x.device)
    hi = lo + 1 if interleaved else lo + rot // 2
    w = torch.complex(x[..., lo], x[..., hi]) * z
    y = x.clone()
    y[..., lo], y[..., hi] = w.real, w.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "prompt":
        parts, at = [], 0
        for n in st["lens"]:
            sl = slice(at, at + n)
            parts.append(_attend(st["q"][sl].double(), st["k"][sl].double(), st["v"][sl].double(), 0 if case["causal"] else None))
            at += n
        return torch.cat(parts)
    if case["op"] == "logprobs":
        x = st["logits"].double()
        lp = torch.log_softmax(x, -1)
        res = {"logprob": lp[torch.arange(case["rows"], device="cuda"), st["tokens"]], "entropy": torch.special.entr(lp.exp()).sum(-1)}
        if case["top"]:
            res["top_logprob"], res["top_token"] = lp.topk(case["top"], -1)[0], None   # whole numbers: by the plain form
        return res
    past, new = _lens(case)
    if case["op"] == "append":
        pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(past, new)])
        # codes and scales are whole: they are held to the plain form's, which computes them bit for bit
        return {"q": _turn(st["q"].double(), pos, case["rot"], case["interleaved"]), "k8": None, "ks": None, "v8": None, "vs": None}
    parts, at = [], 0
    for b, (p, n) in enumerate(zip(past, new)):
        pages = st["table"][b, :-(-(p + n) // case["page"])].long()
        k = st["k8"].view(torch.uint8)[pages].view(_E4M3).double() * st["ks"][pages].double()[..., None, None]
        v = st["v8"].view(torch.uint8)[pages].view(_E4M3).double() * st["vs"][pages].double()[..., None, None]
        k = k.transpose(1, 2).reshape(-1, case["hkv"], case["d"])[:p + n]
        v = v.permute(0, 3, 1, 2).reshape(-1, case["hkv"], case["d"])[:p + n]
        parts.append(_attend(st["q"][at:at + n].double(), k, v, p))
        at += n
    return torch.cat(parts)

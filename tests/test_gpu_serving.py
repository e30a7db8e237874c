"""The operators that serve a quantised decoder -- attention over prompts, the 8-bit paged cache's append and attention, token
log probabilities -- against plain restatements in 64 bits (tests/_serving_ref.py)."""
import math

import pytest
import torch

from tests import _serving_ref as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cu(lens, dev=None):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=dev)


def _close(got, want, bound):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    ok = torch.isfinite(want)
    over = ((got - want).abs() - bound)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, f"off by {float((got - want).abs()[ok].max())}, bound exceeded by {float(over.max())}"


# ---- attention over prompts ------------------------------------------------------------------------------------------

def _qkv(gen, t, hq, hkv, d, dtype, layout, dev):
    x = torch.randn(t, hq + 2 * hkv, d, generator=gen).to(dtype)
    if layout == "merged":
        y = x.to(dev)
        return x, (y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:])
    if layout == "heads first":
        y = x.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
        return x, (y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:])
    y = x.to(dev)
    return x, tuple(p.contiguous() for p in (y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:]))


def _check_prompt(ops, x, views, lens, hq, hkv, causal, dtype, scale=None, rows_behind=0):
    d = x.shape[2]
    dev = views[0].device
    out = torch.full((x.shape[0], hq, d), 7.0, dtype=dtype, device=dev)
    got = ops.attention_prompt(*views, _cu(lens, dev), causal=causal, scale=scale, out=out)
    assert got is out
    at = 0
    for n in lens:
        s = x[at:at + n].double()
        if n:
            want, bound = ref.attend(s[:, :hq], s[:, hq:hq + hkv], s[:, hq + hkv:], 0 if causal else None, d ** -0.5 if scale is None else scale, dtype)
            _close(out[at:at + n], want, bound)
        at += n
    assert (out[at:] == 7.0).all()


@pytest.mark.parametrize("lens,hq,hkv,d,causal,dtype,layout", [
    ([1], 1, 1, 64, True, torch.float16, "plain"),
    ([77], 12, 12, 64, True, torch.float16, "merged"),
    ([64, 65, 1, 0, 127, 2], 4, 2, 64, True, torch.bfloat16, "merged"),
    ([128, 129, 31], 3, 1, 128, True, torch.float16, "heads first"),
    ([300, 33], 5, 1, 128, False, torch.bfloat16, "merged"),
    ([255, 256, 257], 8, 1, 128, True, torch.bfloat16, "merged"),
    ([513], 8, 8, 80, True, torch.float16, "merged"),
    ([100, 200], 6, 2, 96, False, torch.float16, "plain"),
    ([190], 2, 2, 96, True, torch.bfloat16, "merged"),
    ([70, 3], 2, 1, 8, True, torch.float16, "plain"),
    ([70, 3], 2, 1, 40, False, torch.float16, "merged"),
    ([130], 16, 4, 120, True, torch.bfloat16, "heads first"),
])
def test_prompt_attention_against_64_bits(amd, gpu, lens, hq, hkv, d, causal, dtype, layout):
    x, views = _qkv(_gen(sum(lens) + d), sum(lens), hq, hkv, d, dtype, layout, gpu)
    _check_prompt(amd.ops, x, views, lens, hq, hkv, causal, dtype)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16), (96, torch.float16)])
def test_prompt_attention_at_the_borders_of_blocks(amd, gpu, causal, d, dtype):
    """Lengths around the 32, 64 and 128 rows and tokens that blocks, tiles and workgroups have; more than 64 sequences, the
    empty ones among them."""
    lens = [m + e for m in (32, 64, 96, 128, 160, 192, 256) for e in (-1, 0, 1)]
    x, views = _qkv(_gen(d), sum(lens), 2, 1, d, dtype, "merged", gpu)
    _check_prompt(amd.ops, x, views, lens, 2, 1, causal, dtype)
    many = [(7 * i) % 5 * (40 if i % 29 == 3 else 1) for i in range(200)]
    x, views = _qkv(_gen(d + 1), sum(many) + 3, 2, 1, d, dtype, "merged", gpu)
    _check_prompt(amd.ops, x, views, many, 2, 1, causal, dtype)


@pytest.mark.parametrize("at", [0, 1, 31, 32, 63, 64, 95, 96, 127, 128, 138])
def test_prompt_attention_keeps_infinite_values_from_earlier_rows_everywhere(amd, gpu, at):
    """An infinite value of any token of a tile reaches the rows from its own on; of a following sequence, none at all."""
    x, _ = _qkv(_gen(50), 139 + 20, 2, 1, 64, torch.float16, "plain", gpu)
    x[at, 3, 5], x[139:, 2:] = math.inf, math.nan
    y = x.to(gpu)
    for causal in (True, False):
        out = amd.ops.attention_prompt(y[:, :2], y[:, 2:3], y[:, 3:], _cu([139], gpu), causal=causal)[:139].cpu()
        clean = x[:139].clone()
        clean[at, 3] = 0.5
        s = clean.double()
        want, bound = ref.attend(s[:, :2], s[:, 2:3], s[:, 3:], 0 if causal else None, 64 ** -0.5, torch.float16)
        first = at if causal else 0
        _close(out[:first], want[:first], bound[:first])
        rest = [c for c in range(64) if c != 5]
        s[at, 3] = x[at, 3].double()
        s[at, 3, 5] = 0.5
        want, bound = ref.attend(s[:, :2], s[:, 2:3], s[:, 3:], 0 if causal else None, 64 ** -0.5, torch.float16)
        _close(out[..., rest], want[..., rest], bound[..., rest])
        assert not torch.isfinite(out[first:, :, 5]).any()


def test_prompt_attention_of_one_token_with_any_stride(amd, gpu):
    """A dimension of one element may have any stride: one row of a transposed or odd-strided tensor is taken."""
    x = torch.randn(1, 4, 64, generator=_gen(51)).half()
    for stride in (0, 3, 1 << 30):
        q, k, v = (t.to(gpu).as_strided((1, n, 64), (stride, 64, 1)) for t, n in ((x[:, :2], 2), (x[:, 2:3], 1), (x[:, 3:], 1)))
        got = amd.ops.attention_prompt(q, k, v)
        # one key: its value
        assert torch.equal(got.cpu(), x[:, 3:].expand(1, 2, 64))


def test_prompt_attention_one_sequence_scale_and_large_scores(amd, gpu):
    """No cu_seqlens; a scale of its own; scores in the hundreds, where the softmax is a choice of one key."""
    x, views = _qkv(_gen(3), 150, 4, 4, 64, torch.float16, "merged", gpu)
    got = amd.ops.attention_prompt(*views, scale=0.3)
    s = x.double()
    _close(got, *ref.attend(s[:, :4], s[:, 4:8], s[:, 8:], 0, 0.3, torch.float16))
    x = x.clone()
    x[:, :8] *= 8
    y = x.to(gpu)
    s = x.double()
    _close(amd.ops.attention_prompt(y[:, :4], y[:, 4:8], y[:, 8:]), *ref.attend(s[:, :4], s[:, 4:8], s[:, 8:], 0, 64 ** -0.5, torch.float16))


def test_prompt_attention_rows_behind_the_last_sequence(amd, gpu):
    """A padded batch: rows behind cu_seqlens[-1] hold NaN, reach nothing and are not written."""
    x, _ = _qkv(_gen(4), 200, 4, 2, 64, torch.bfloat16, "plain", gpu)
    x[150:] = math.nan
    y = x.to(gpu)
    _check_prompt(amd.ops, x, (y[:, :4], y[:, 4:6], y[:, 6:]), [90, 60], 4, 2, True, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_attention_keeps_later_infinities_from_earlier_rows(amd, gpu, dtype, bad):
    """An infinite or NaN value (or key) of token 70 reaches the rows from 70 on and no other."""
    for part in ("k", "v"):
        x, _ = _qkv(_gen(5), 140, 2, 1, 64, dtype, "plain", gpu)
        x[70, 2 if part == "k" else 3, 5] = bad
        y = x.to(gpu)
        out = amd.ops.attention_prompt(y[:, :2], y[:, 2:3], y[:, 3:]).cpu()
        clean = x.clone()
        clean[70, 2:] = 0.5
        s = clean.double()
        want, bound = ref.attend(s[:, :2], s[:, 2:3], s[:, 3:], 0, 64 ** -0.5, dtype)
        _close(out[:70], want[:70], bound[:70])
        if part == "v":
            assert not torch.isfinite(out[70:, :, 5]).any() and torch.isfinite(out[70:, :, :5]).all() and torch.isfinite(out[70:, :, 6:]).all()


def test_prompt_attention_offsets_past_32_bits(amd, gpu):
    """70000 rows 2^15 elements apart (4.6 GB): the last sequence lies behind 2^31 elements."""
    lens = [69900, 100]
    big = torch.empty(70000, 1 << 15, dtype=torch.float16, device=gpu)
    x = torch.randn(100, 3, 64, generator=_gen(6)).half()
    big[69900:, :192] = x.view(100, 192).to(gpu)
    q, k, v = (big[:, 64 * i:64 * i + 64].unsqueeze(1) for i in range(3))
    cu = torch.tensor([69900, 70000], dtype=torch.int32, device=gpu)
    out = amd.ops.attention_prompt(q, k, v, cu)
    s = x.double()
    _close(out[69900:], *ref.attend(s[:, :1], s[:, 1:2], s[:, 2:], 0, 64 ** -0.5, torch.float16))


# ---- the paged cache -------------------------------------------------------------------------------------------------

def _tables(n, rot):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return ang.cos().float(), ang.sin().float()


class Both:
    """The cache on the device and its restatement, appended to together."""

    def __init__(self, amd, gpu, batch, pages_each, heads, page, d, seed, spare=2):
        self.ops, self.gpu, self.gen = amd.ops, gpu, _gen(seed)
        self.heads, self.d, self.batch = heads, d, batch
        n = batch * pages_each + spare
        self.cpu = ref.Cache(n, heads, page, d)
        self.dev = amd.ops.PagedCache.empty(n, heads, page, d, gpu)
        self.table = torch.randperm(n, generator=self.gen)[:batch * pages_each].view(batch, pages_each).int()
        self.past = [0] * batch

    def append(self, new, dtype, rot=0, interleaved=False, q_heads=0, scale=1.0, single=False, k=None, v=None):
        t = sum(new)
        cu = [0] + torch.tensor(new).cumsum(0).tolist()
        k = scale * torch.randn(t, self.heads, self.d, generator=self.gen) if k is None else k
        v = scale * torch.randn(t, self.heads, self.d, generator=self.gen) if v is None else v
        k, v = k.to(dtype), v.to(dtype)
        q = torch.randn(t, max(q_heads, 1), self.d, generator=self.gen).to(dtype)
        pos = torch.tensor([p + i for p, n in zip(self.past, new) for i in range(n)], dtype=torch.long)
        cos, sin = _tables(int(pos.max()) + 1, rot) if rot else (None, None)
        dev = lambda x: None if x is None else x.to(self.gpu)   # noqa: E731
        got = self.ops.kv_append(self.dev, dev(k), dev(v), dev(self.table), dev(torch.tensor(self.past, dtype=torch.int32)),
                                 None if single else dev(torch.tensor(cu, dtype=torch.int32)), q=dev(q) if q_heads else None, cos=dev(cos), sin=dev(sin),
                                 interleaved=interleaved)
        if q_heads:
            # one rounding of the same 32-bit operations
            assert torch.equal(got.cpu(), ref.rotate(q, pos, cos, sin, interleaved).to(dtype))
        self.cpu.append(ref.rotate(k, pos, cos, sin, interleaved) if rot else k.float(), v.float(), self.table, self.past, cu)
        self.past = [p + n for p, n in zip(self.past, new)]
        self.same()

    def same(self):
        for a, b in zip(self.dev, (self.cpu.k, self.cpu.v, self.cpu.ks, self.cpu.vs)):
            x, y = a.cpu(), b
            if x.dtype == E4M3:
                x, y = x.view(torch.uint8), y.view(torch.uint8)
                nan = (x & 127) == 127   # the sign of a NaN is not laid down
                assert torch.equal(nan, (y & 127) == 127)
                x, y = x.masked_fill(nan, 0), y.masked_fill(nan, 0)
            assert torch.equal(x, y)


@pytest.mark.parametrize("batch,new,heads,page,d,rot,interleaved,dtype", [
    (1, [[5], [1], [12]], 2, 16, 64, 64, False, torch.float16),
    (3, [[17, 0, 40], [1, 3, 16], [33, 1, 1]], 2, 16, 64, 32, True, torch.bfloat16),
    (2, [[64, 63], [1, 1], [70, 2]], 1, 64, 128, 128, False, torch.float16),
    (2, [[130, 1], [127, 128]], 2, 128, 128, 128, True, torch.bfloat16),
    (2, [[31, 32], [33, 95]], 3, 32, 80, 16, False, torch.float16),
    (1, [[3], [13], [16]], 1, 16, 16, 0, False, torch.bfloat16),
    (1, [[100]], 2, 64, 96, 96, False, torch.bfloat16),
])
def test_append_is_the_restatement_bit_for_bit(amd, gpu, batch, new, heads, page, d, rot, interleaved, dtype):
    most = max(sum(n[b] for n in new) for b in range(batch))
    c = Both(amd, gpu, batch, -(-most // page), heads, page, d, seed=page + d)
    for i, n in enumerate(new):
        c.append(n, dtype, rot, interleaved, q_heads=3 if rot else 0, scale=4.0 ** i)   # scales grow on the way


def test_append_single_tokens_with_growing_and_falling_sizes(amd, gpu):
    """Token by token through two pages: the scale grows where it must, never falls, codes are re-expressed."""
    c = Both(amd, gpu, 2, 2, 2, 16, 32, seed=1)
    for i in range(32):
        c.append([1, 1], torch.float16, rot=32, q_heads=2, scale=[1.0, 8.0, 0.01, 300.0, 1.0][i % 5], single=True)


def test_append_zeros_infinities_and_nan(amd, gpu):
    c = Both(amd, gpu, 1, 2, 1, 16, 16, seed=2)
    z = torch.zeros(3, 1, 16)
    c.append([3], torch.float16, k=z, v=z.clone())
    x = torch.randn(4, 1, 16, generator=_gen(1))
    x[0, 0, 3], x[1, 0, 4], x[2, 0, 5] = math.inf, -math.inf, math.nan
    c.append([4], torch.float16, k=x, v=-x)
    c.append([1], torch.bfloat16, k=torch.full((1, 1, 16), 3.0e38), v=torch.full((1, 1, 16), 1.0e-38))
    # exactly at the border between two scales, and a step above it
    for top in (448.0, 449.0, 450.0):
        d = Both(amd, gpu, 1, 1, 1, 16, 16, seed=3)
        y = torch.full((2, 1, 16), 1.0)
        y[1, 0, 7] = top
        d.append([2], torch.float16, k=y, v=y.clone())
        assert float(d.dev.k_scale.cpu().max()) >= (1.0 if top == 448 else 2.0)


def test_append_skips_what_has_no_place(amd, gpu):
    """Pages outside the pool, tokens behind the table, positions without an angle, inactive sequences, rows behind the last
    sequence: nothing is stored for them, everything else is."""
    ops, page, d = amd.ops, 16, 32
    cpu, dev = ref.Cache(6, 1, page, d), ops.PagedCache.empty(6, 1, page, d, gpu)
    table = torch.tensor([[0, 99], [-1, 1], [2, 3], [4, 5]], dtype=torch.int32)
    past, new = [10, 12, -1, 20], [10, 8, 4, 30]   # the last runs over its table
    t = sum(new) + 3
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    gen = _gen(9)
    k, v, q = (torch.randn(t, h, d, generator=gen).half() for h in (1, 1, 2))
    cos, sin = _tables(30, d)   # positions 30.. have none
    out = torch.full((t, 2, d), 5.0, dtype=torch.float16, device=gpu)
    got = ops.kv_append(dev, k.to(gpu), v.to(gpu), table.to(gpu), torch.tensor(past, dtype=torch.int32, device=gpu),
                        torch.tensor(cu, dtype=torch.int32, device=gpu), q=q.to(gpu), cos=cos.to(gpu), sin=sin.to(gpu), q_out=out)
    assert got is out
    pos = torch.tensor([p + i if p >= 0 else -1 for p, n in zip(past, new) for i in range(n)])
    has = (pos >= 0) & (pos < 30)
    rk = ref.rotate(k[:len(pos)], pos.clamp(0, 29), cos, sin, False)
    cpu.append(rk, v[:len(pos)].float(), table, past, cu, max_pos=30)
    both = Both.__new__(Both)
    both.cpu, both.dev = cpu, dev
    both.same()
    got = got.cpu()
    want = ref.rotate(q[:len(pos)], pos.clamp(0, 29), cos, sin, False).half()
    assert torch.equal(got[:len(pos)][has], want[has]) and torch.isnan(got[:len(pos)][~has]).all() and (got[len(pos):] == 5.0).all()


def test_append_of_many_sequences(amd, gpu):
    """More sequences than one look at the starts sees, empty ones and pages that are begun among them."""
    c = Both(amd, gpu, 150, 3, 1, 16, 32, seed=23)
    for i in range(3):
        c.append([(5 * b + 3 * i) % 7 if b % 13 else 13 for b in range(150)], torch.float16, 32, i == 1, q_heads=2)


def test_append_rotates_q_in_place(amd, gpu):
    gen = _gen(11)
    for inter in (False, True):
        dev = amd.ops.PagedCache.empty(2, 2, 16, 64, gpu)
        qkv = torch.randn(20, 8, 64, generator=gen).half()
        x = qkv.to(gpu)
        cos, sin = _tables(20, 32)
        q = x[:, :4]
        got = amd.ops.kv_append(dev, x[:, 4:6], x[:, 6:], torch.tensor([[1, 0]], dtype=torch.int32, device=gpu),
                                torch.zeros(1, dtype=torch.int32, device=gpu), _cu([20], gpu), q=q, cos=cos.to(gpu), sin=sin.to(gpu),
                                interleaved=inter, q_out=q)
        assert torch.equal(got.cpu(), ref.rotate(qkv[:, :4], torch.arange(20), cos, sin, inter).half())
        assert torch.equal(x[:, 4:].cpu(), qkv[:, 4:])


def _filled(amd, gpu, lens, heads, page, d, seed, width=None, spread=0.0):
    """A device cache with random codes and scales and its copy on the CPU; slots behind the lengths hold NaN."""
    gen = _gen(seed)
    width = width or max(1, -(-max(lens) // page))
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 1
    c = ref.Cache(n_pages, heads, page, d)
    c.k = torch.randn(c.k.shape, generator=gen).mul(100).clamp(-448, 448).to(E4M3)
    c.v = torch.randn(c.v.shape, generator=gen).mul(100).clamp(-448, 448).to(E4M3)
    c.ks = torch.exp2(torch.round(spread * torch.randn(n_pages, heads, generator=gen)) - 7)
    c.vs = torch.exp2(torch.round(spread * torch.randn(n_pages, heads, generator=gen)) - 7)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    order = torch.randperm(n_pages, generator=gen).int()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    for b, n in enumerate(lens):
        if n % page:
            p = int(table[b, n // page])
            c.k.view(torch.uint8)[p, :, n % page:] = 0x7f
            c.v.view(torch.uint8)[p, :, :, n % page:] = 0xff
    dev = amd.ops.PagedCache(*(x.to(gpu) for x in (c.k, c.v, c.ks, c.vs)))
    return c, dev, table


def _check_paged(got, q, c, table, lens, new, dtype, scale=None):
    at = 0
    d = q.shape[2]
    for b, (n, m) in enumerate(zip(lens, new)):
        if n:
            k, v, vs = c.tokens(table[b], n)
            want, bound = ref.attend(q[at:at + m].double(), k, v, n - m, d ** -0.5 if scale is None else scale, dtype, vmax=vs)
            _close(got[at:at + m], want, bound)
        else:
            assert (got[at:at + m] == 0).all()
        at += m


@pytest.mark.parametrize("lens,hq,hkv,page,d,dtype", [
    ([1], 1, 1, 16, 64, torch.float16),
    ([100], 32, 32, 16, 128, torch.float16),
    ([64, 0, 65, 1, 63], 8, 2, 64, 128, torch.bfloat16),
    ([300, 17, 129], 16, 1, 32, 64, torch.float16),
    ([257, 128], 40, 2, 128, 96, torch.bfloat16),
    ([500, 3], 6, 2, 16, 80, torch.float16),
    ([1000], 72, 1, 64, 128, torch.float16),
    ([40, 50], 4, 4, 16, 16, torch.bfloat16),
])
def test_paged_attention_of_single_tokens(amd, gpu, lens, hq, hkv, page, d, dtype):
    c, dev, table = _filled(amd, gpu, lens, hkv, page, d, seed=d + page, spread=1.5)
    q = torch.randn(len(lens), hq, d, generator=_gen(2)).to(dtype)
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu))
    _check_paged(got, q, c, table, lens, [1] * len(lens), dtype)


@pytest.mark.parametrize("lens,new,hq,hkv,page,d,dtype", [
    ([10, 100, 64], [3, 5, 1], 8, 2, 16, 64, torch.float16),
    ([200, 5], [9, 5], 4, 4, 64, 128, torch.bfloat16),
    ([130, 0, 70], [40, 0, 70], 8, 1, 32, 128, torch.float16),
    ([90, 33], [2, 40], 4, 2, 16, 96, torch.float16),        # more query tokens than the sequence has: the first see nothing
    ([700], [130], 5, 1, 64, 64, torch.bfloat16),
])
def test_paged_attention_of_several_tokens(amd, gpu, lens, new, hq, hkv, page, d, dtype):
    c, dev, table = _filled(amd, gpu, lens, hkv, page, d, seed=d + page, spread=1.0)
    q = torch.randn(sum(new) + 2, hq, d, generator=_gen(3)).to(dtype)
    out = torch.full(q.shape, 3.0, dtype=dtype, device=gpu)
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu), scale=0.2, out=out)
    _check_paged(got, q, c, table, lens, new, dtype, scale=0.2)
    assert (got[sum(new):] == 3.0).all()


@pytest.mark.parametrize("lens,new", [([5000], [1]), ([9001, 70, 4097], [1, 1, 1]), ([6000, 33], [4, 2])])
def test_paged_attention_in_runs_of_a_long_sequence(amd, gpu, lens, new):
    """Long enough to be cut into runs that a second kernel joins, with scales that differ by 2^20 between pages."""
    c, dev, table = _filled(amd, gpu, lens, 2, 64, 64, seed=8, spread=6.0)
    q = torch.randn(sum(new), 8, 64, generator=_gen(4)).half()
    assert amd._lib.load().gq_attention_paged_workspace(sum(new), len(lens), int(new[0] > 1), 8, 2, 64, 64, table.shape[1]) > 0
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), None if max(new) == 1 else _cu(new, gpu))
    _check_paged(got, q, c, table, lens, new, torch.float16)


def test_paged_attention_of_a_bad_table(amd, gpu):
    """A missing page, one outside the pool, a length beyond the table: NaN for that sequence, the others as ever."""
    lens = [100, 90, 80, 70]
    c, dev, table = _filled(amd, gpu, lens, 2, 16, 64, seed=5)
    q = torch.randn(4, 4, 64, generator=_gen(5)).half()
    bad = table.clone()
    bad[0, 3], bad[2, 0] = -1, 10 ** 6
    short = torch.tensor([100, 90, 80, 10 ** 9], dtype=torch.int32)
    got = amd.ops.attention_paged(q.to(gpu), dev, bad.to(gpu), short.to(gpu)).cpu()
    assert torch.isnan(got[[0, 2, 3]]).all()
    k, v, vs = c.tokens(table[1], 90)
    want, bound = ref.attend(q[1:2].double(), k, v, 89, 0.125, torch.float16, vmax=vs)
    _close(got[1:2], want, bound)


@pytest.mark.parametrize("page,width", [(16, 16), (64, 4), (32, 9), (128, 16), (16, 512)])
@pytest.mark.parametrize("more", [1, 40, 70000])
def test_paged_attention_of_sequences_longer_than_their_table(amd, gpu, page, width, more):
    """NaN, also where the table ends with a tile or with the last run of one; a full table is none."""
    full = page * width
    c, dev, table = _filled(amd, gpu, [full, full], 1, page, 64, seed=9)
    q = torch.randn(2, 4, 64, generator=_gen(6)).half()
    lens = torch.tensor([full, full + more], dtype=torch.int32)
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), lens.to(gpu)).cpu()
    assert torch.isnan(got[1]).all()
    _check_paged(got[:1], q[:1], c, table[:1], [full], [1], torch.float16)


def test_paged_attention_of_the_smallest_scales(amd, gpu):
    """Values of 2^-100 times a code: bf16 holds the result."""
    c, dev, table = _filled(amd, gpu, [50, 200], 1, 16, 64, seed=10)
    q = torch.randn(2, 4, 64, generator=_gen(7)).bfloat16()
    lens = torch.tensor([50, 200], dtype=torch.int32, device=gpu)
    one = dev._replace(v_scale=torch.ones_like(dev.v_scale))
    low = dev._replace(v_scale=torch.full_like(dev.v_scale, 2.0 ** -100))
    a, b = (amd.ops.attention_paged(q.to(gpu), x, table.to(gpu), lens).double() for x in (one, low))
    # the weights differ by the rounding of y + log2 vs alone: |y| < 128 rounds by 2^-18, the weight by ln 2 of that
    assert ((b * 2.0 ** 100 - a).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -9).all()


def test_paged_attention_of_many_ragged_sequences(amd, gpu):
    lens = [(37 * b) % 90 for b in range(150)]
    new = [min(n, (11 * b) % 4) for b, n in enumerate(lens)]
    c, dev, table = _filled(amd, gpu, lens, 1, 32, 64, seed=24)
    q = torch.randn(sum(new), 4, 64, generator=_gen(52)).half()
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu))
    _check_paged(got, q, c, table, lens, new, torch.float16)


@pytest.mark.parametrize("lens,new,hq,hkv,page", [([1500], [1490], 4, 1, 64), ([40, 900, 20], [33, 700, 20], 8, 4, 16), ([1300, 64], [1300, 1], 2, 1, 128)])
def test_paged_attention_of_chunks_in_runs(amd, gpu, lens, new, hq, hkv, page):
    """Chunks whose first rows see none of the later runs of their sequence, and workgroups that end inside a token's heads."""
    c, dev, table = _filled(amd, gpu, lens, hkv, page, 64, seed=27, spread=2.0)
    q = torch.randn(sum(new), hq, 64, generator=_gen(54)).to(torch.bfloat16)
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu))
    _check_paged(got, q, c, table, lens, new, torch.bfloat16)


def test_paged_attention_of_a_chunk_with_a_missing_page(amd, gpu):
    """Rows that see the missing page, or a token behind the table, are NaN; another sequence is as ever."""
    lens, new = [300, 100], [200, 3]
    c, dev, table = _filled(amd, gpu, lens, 1, 16, 64, seed=28)
    q = torch.randn(203, 4, 64, generator=_gen(55)).half()
    bad = table.clone()
    bad[0, 17] = -1   # tokens 272..287: rows from 172 on
    got = amd.ops.attention_paged(q.to(gpu), dev, bad.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu)).cpu()
    assert torch.isnan(got[172:200]).all()
    _check_paged(got[200:], q[200:], c, table[1:], lens[1:], new[1:], torch.float16)
    got = amd.ops.attention_paged(q.to(gpu), dev, table[:, :18].contiguous().to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu)).cpu()
    assert torch.isnan(got[188:200]).all()
    _check_paged(got[200:], q[200:], c, table[1:], lens[1:], new[1:], torch.float16)


def test_paged_attention_of_shared_pages(amd, gpu):
    """Sequences that begin with the same pages, and one that names a page twice."""
    c, dev, table = _filled(amd, gpu, [128, 128, 128], 2, 64, 64, seed=25)
    table[1, 0], table[2, 1] = table[0, 0], table[2, 0]
    q = torch.randn(3, 4, 64, generator=_gen(53)).half()
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.full((3,), 128, dtype=torch.int32, device=gpu))
    _check_paged(got, q, c, table, [128] * 3, [1] * 3, torch.float16)


def test_paged_attention_keeps_later_nan_from_earlier_rows(amd, gpu):
    """A NaN among the values (keys) of the second of three query tokens does not reach the first."""
    for part in ("k", "v"):
        lens, new = [77, 64], [3, 3]
        c, dev, table = _filled(amd, gpu, lens, 1, 16, 64, seed=6)
        p, s = int(table[0, 75 // 16]), 75 % 16
        if part == "v":
            dev.v.view(torch.uint8)[p, 0, 9, s] = 0x7f
        else:
            dev.k.view(torch.uint8)[p, 0, s, 9] = 0x7f
        q = torch.randn(6, 4, 64, generator=_gen(6)).half()
        got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu)).cpu()
        k, v, vs = c.tokens(table[0], 75)
        _close(got[:1], *ref.attend(q[:1].double(), k, v, 74, 0.125, torch.float16, vmax=vs))
        assert torch.isnan(got[1:3, :, 9]).all() and (part == "k" or torch.isfinite(got[1:3, :, 10:]).all())
        _check_paged(got[3:], q[3:], c, table[1:], lens[1:], new[1:], torch.float16)


def test_paged_cache_offsets_past_32_bits(amd, gpu):
    """A pool of more than 2^32 bytes of keys: pages at its end are written and read."""
    heads, page, d = 8, 128, 128
    n_pages = (1 << 32) // (heads * page * d) + 3
    dev = amd.ops.PagedCache.empty(n_pages, heads, page, d, gpu)
    c = ref.Cache(2, heads, page, d)
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32)
    gen = _gen(7)
    k, v = torch.randn(150, heads, d, generator=gen).half(), torch.randn(150, heads, d, generator=gen).half()
    amd.ops.kv_append(dev, k.to(gpu), v.to(gpu), table.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu), _cu([150], gpu))
    c.append(k.float(), v.float(), torch.tensor([[1, 0]]), [0], [0, 150])
    both = Both.__new__(Both)
    both.cpu, both.dev = c, amd.ops.PagedCache(*(x[-2:] for x in dev))
    both.same()
    q = torch.randn(1, 16, d, generator=gen).half()
    lens = torch.tensor([150], dtype=torch.int32, device=gpu)
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), lens)
    _check_paged(got, q, c, torch.tensor([[1, 0]]), [150], [1], torch.float16)


# ---- log probabilities -----------------------------------------------------------------------------------------------

def _check_logprobs(res, logits, tokens, top):
    """A sum of V exponentials in 32 bits, pairwise over at least 256 threads and then along a thread: off by at most
    (V / 256 + 20) 2^-24 relatively, an exponential by |x - m| 2^-23 more (its argument's rounding); the logarithm turns that
    into an absolute error, and x - m rounds by 2^-24 of itself."""
    lp, ent, tlp, tok = ref.log_probs(logits, tokens, top)
    vocab = logits.shape[1]
    fin = torch.nan_to_num(logits.double(), 0, 0, 0)
    # beyond 100 below the maximum an exponential is below 2^-144 and its error too
    span = (fin.amax(1) - fin.amin(1)).clamp(max=100)
    rel = (vocab / 256 + 20 + 4 * span + 4) * 2.0 ** -24
    for got, want, b in ((res.logprob, lp, rel + lp.abs() * 2.0 ** -23), (res.entropy, ent, rel * (2 + span)),
                         *(((res.top_logprob, tlp, rel[:, None] + tlp.abs() * 2.0 ** -23),) if top else ())):
        _close(got, want, torch.nan_to_num(b, 0, 0, 0) + 1e-7)
    if top:
        assert torch.equal(res.top_token.cpu(), tok)


@pytest.mark.parametrize("rows,vocab,top,dtype", [
    (1, 32000, 5, torch.float16), (1, 1, 1, torch.float32), (3, 7, 7, torch.bfloat16), (2, 50257, 20, torch.bfloat16), (5, 50257, 0, torch.float16),
    (700, 1003, 32, torch.bfloat16), (600, 4099, 10, torch.float32), (2, 151936, 20, torch.float32), (4, 129, 32, torch.float16), (513, 33, 3, torch.float32),
])
def test_token_logprobs_against_64_bits(amd, gpu, rows, vocab, top, dtype):
    gen = _gen(vocab + rows)
    logits = (3 * torch.randn(rows, vocab, generator=gen)).to(dtype)   # 16-bit logits tie often
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    _check_logprobs(amd.ops.token_logprobs(logits.to(gpu), tokens.to(gpu), top=top), logits, tokens, top)


@pytest.mark.parametrize("rows", [4, 520])
def test_token_logprobs_ties_order_and_crowds(amd, gpu, rows):
    """Constant rows, rising and falling rows, +-0, and a row whose largest elements crowd into one thread's part of it."""
    vocab = 40000
    for kind in range(5):
        x = torch.zeros(rows, vocab)
        if kind == 1:
            x += torch.arange(vocab) / 4096
        elif kind == 2:
            x -= torch.arange(vocab) / 4096
        elif kind == 3:
            x[:, 1::2] = -0.0
            x[:, 5] = -1
        elif kind == 4:
            for c in range(0, vocab, 8192):   # chunks a whole number of strides apart
                x[:, c:c + 512] = 5.0 + torch.arange(512) / 1024
        for dtype in (torch.float32, torch.bfloat16):
            y = x.to(dtype)
            tokens = torch.full((rows,), 11)
            _check_logprobs(amd.ops.token_logprobs(y.to(gpu), tokens.to(gpu), top=20), y, tokens, 20)


def test_token_logprobs_infinities_and_nan(amd, gpu):
    gen = _gen(1)
    x = torch.randn(9, 500, generator=gen)
    tokens = torch.randint(0, 500, (9,), generator=gen)
    x[0, ::2] = -math.inf
    x[1, :] = -math.inf
    x[2, 1:] = -math.inf
    tokens[2] = 0
    x[3, 77] = math.inf
    x[4, 70] = math.nan
    x[5, :490] = -math.inf
    x[6] = math.nan
    x[7, 3], tokens[7] = -math.inf, 3
    for dtype in (torch.float32, torch.float16):
        y = x.to(dtype)
        _check_logprobs(amd.ops.token_logprobs(y.to(gpu), tokens.to(gpu), top=12), y, tokens, 12)


@pytest.mark.parametrize("rows,vocab", [(3, 32003), (600, 1003), (2, 40)])
def test_token_logprobs_of_masked_words(amd, gpu, rows, vocab):
    """Words masked by the type's lowest value: all of a row (a uniform one), all but a few, whole stretches; the same by -inf
    but for the row without a word."""
    gen = _gen(vocab)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for low in (torch.finfo(dtype).min, -math.inf, *((-1e30, -1e38, -2e38) if dtype != torch.float16 else (-1e4,))):
            x = (3 * torch.randn(rows, vocab, generator=gen)).to(dtype)
            x[0, :] = low
            x[0, 17], x[0, vocab - 1] = 1.5, 1.0
            if low > -math.inf:
                x[1, :] = low
            else:
                x[1, : vocab // 2] = low
            if rows > 2:
                x[2, 8:vocab - 8] = low
            tokens = torch.randint(0, vocab, (rows,), generator=gen)
            tokens[0] = 17
            _check_logprobs(amd.ops.token_logprobs(x.to(gpu), tokens.to(gpu), top=6), x, tokens, 6)


def test_token_logprobs_of_large_numbers(amd, gpu):
    """Logits far from 0, where their differences are exact but their size is not small; the type's largest and lowest."""
    gen = _gen(12)
    for dtype, base in (*((torch.float32, 2.0 ** 31 + 2.0 ** 20 * i) for i in range(12)), (torch.float32, 2.0 ** 20), (torch.float32, -2.0 ** 22), (torch.float32, 2.0 ** 100), (torch.float32, -3.0e38), (torch.bfloat16, 3.0e38), (torch.float16, 6.0e4)):
        x = torch.randint(-8, 9, (4, 5003), generator=gen).to(torch.float64)
        x = (base + x * max(1.0, abs(base) * torch.finfo(dtype).eps)).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
        tokens = torch.randint(0, 5003, (4,), generator=gen)
        tokens[0] = int(x[0].argmax())
        _check_logprobs(amd.ops.token_logprobs(x.to(gpu), tokens.to(gpu), top=4), x, tokens, 4)


def test_token_logprobs_tokens_shapes_and_strides(amd, gpu):
    gen = _gen(2)
    x = torch.randn(2, 9, 1001, generator=gen).half()
    tokens = torch.randint(0, 1001, (2, 9), generator=gen)
    tokens[0, 1], tokens[1, 2], tokens[1, 3] = -100, 1001, -1
    y = x.to(gpu)
    # a slice of each sequence, rows of a wider matrix, and an odd first element
    res = amd.ops.token_logprobs(y[:, :-1], tokens[:, :-1].to(gpu), top=2)
    assert res.logprob.shape == (2, 8) and res.top_token.shape == (2, 8, 2) and res.entropy.shape == (2, 8)
    want = ref.log_probs(x[:, :-1].reshape(16, 1001), tokens[:, :-1].clamp(0, 1000).reshape(16), 2)
    got = res.logprob.cpu().reshape(16)
    assert got[1] == 0 and torch.isnan(got[[10, 11]]).all()
    keep = [i for i in range(16) if i not in (1, 10, 11)]
    assert (got[keep].double() - want[0][keep]).abs().max() < 1e-5 and torch.equal(res.top_token.cpu().reshape(16, 2), want[3])
    wide = y.view(18, 1001)[:, 3:900]
    t = torch.randint(0, 897, (18,), generator=gen)
    _check_logprobs(amd.ops.token_logprobs(wide, t.to(gpu), top=4), wide.cpu().contiguous(), t, 4)
    none = amd.ops.token_logprobs(y[:, :0], tokens[:, :0].to(gpu), top=1)
    assert none.logprob.shape == (2, 0) and none.top_token.shape == (2, 0, 1)


def test_token_logprobs_offsets_past_32_bits(amd, gpu):
    big = torch.zeros(70, 1 << 26, dtype=torch.float16, device=gpu)   # 9.4 GB
    x = torch.randn(70, 300, generator=_gen(3)).half()
    big[:, -300:] = x.to(gpu)
    t = torch.randint(0, 300, (70,), generator=_gen(4))
    _check_logprobs(amd.ops.token_logprobs(big[:, -300:], t.to(gpu), top=3), x, t, 3)


# ---- together --------------------------------------------------------------------------------------------------------

def _serve(ops, dev, qkv, dims, chunks, cos, sin, stream_ops=None):
    """Prompts in chunks, then single tokens: append and attend; returns all attention rows."""
    hq, hkv, d, page = dims
    batch, total = qkv.shape[0], qkv.shape[1]
    width = -(-total // page)
    cache = ops.PagedCache.empty(batch * width, hkv, page, d, dev)
    table = torch.arange(batch * width, dtype=torch.int32, device=dev).view(batch, width).flip(1).contiguous()
    past = torch.zeros(batch, dtype=torch.int32, device=dev)
    rows, at = [], 0
    for n in chunks:
        x = qkv[:, at:at + n].reshape(batch * n, hq + 2 * hkv, d)
        cu = None if n == 1 else torch.arange(0, batch * n + 1, n, dtype=torch.int32, device=dev)
        q = ops.kv_append(cache, x[:, hq:hq + hkv], x[:, hq + hkv:], table, past, cu, q=x[:, :hq], cos=cos, sin=sin)
        past = past + n
        rows.append(ops.attention_paged(q, cache, table, past, cu).view(batch, n, hq, d))
        at += n
    return torch.cat(rows, 1), cache


def test_prefill_chunks_and_steps_agree_with_prompt_attention(amd, gpu):
    """The serving loop against attention over the whole prompt with keys and values that were rounded through the cache:
    the two differ by their own roundings alone."""
    ops, hq, hkv, d, page = amd.ops, 8, 2, 64, 16
    gen = _gen(12)
    qkv = torch.randn(2, 90, hq + 2 * hkv, d, generator=gen).half()
    cos, sin = _tables(90, d)
    got, cache = _serve(ops, gpu, qkv.to(gpu), (hq, hkv, d, page), [37, 1, 1, 50, 1], cos.to(gpu), sin.to(gpu))
    c = ref.Cache(12, hkv, page, d)
    c.k, c.v, c.ks, c.vs = (x.cpu() for x in cache)
    table = torch.arange(12).view(2, 6).flip(1)
    pos = torch.arange(90)
    for b in range(2):
        k, v, vs = c.tokens(table[b], 90)
        q = ref.rotate(qkv[b, :, :hq], pos, cos, sin, False).half()
        # (scales grow while a page fills: codes seen by early steps were finer, so the bound of those steps adds that)
        exactk = ref.rotate(qkv[b, :, hq:hq + hkv], pos, cos, sin, False).double()
        want, bound = ref.attend(q.double(), k, v, 0, d ** -0.5, torch.float16, vmax=vs)
        _close(got[b, 40:], want[40:], bound[40:] + 1e-3)
        # what 8 bits cost: every key and value is within half a step of its own
        assert ((k - exactk).abs() <= 2.0 ** -4 * exactk.abs() + 2.0 ** -9 * 2).all()
        # and the prompt kernel on the rounded keys and values
        same = ops.attention_prompt(q.to(gpu), k.half().to(gpu), v.half().to(gpu))
        _close(same, *ref.attend(q.double(), k.half().double(), v.half().double(), 0, d ** -0.5, torch.float16))


def test_a_captured_step_replays_with_new_lengths(amd, gpu):
    """One decoder step (append, attention, log probabilities) captured once; each replay sees the lengths, tokens and pages of
    its time, and equals the eager calls bit for bit.  Two graphs with scratch memory of their own run alternately."""
    ops, hq, hkv, d, page, vocab = amd.ops, 8, 2, 64, 64, 1000
    gen = _gen(13)
    w = torch.randn(hq * d, vocab, generator=gen).half().to(gpu) / 20

    def build(total):
        qkv = torch.randn(3, total, hq + 2 * hkv, d, generator=gen).half().to(gpu)
        cos, sin = (x.to(gpu) for x in _tables(total, d))
        width = -(-total // page)
        st = {"cache": ops.PagedCache.empty(3 * width, hkv, page, d, gpu), "past": torch.zeros(3, dtype=torch.int32, device=gpu),
              "table": torch.randperm(3 * width, generator=gen).int().view(3, width).to(gpu), "x": qkv[:, 0].clone(), "tok": torch.tensor([1, 2, 3], device=gpu)}

        def step():
            x = st["x"]
            q = ops.kv_append(st["cache"], x[:, hq:hq + hkv], x[:, hq + hkv:], st["table"], st["past"], q=x[:, :hq], cos=cos, sin=sin)
            o = ops.attention_paged(q, st["cache"], st["table"], st["past"] + 1)
            r = ops.token_logprobs((o.view(3, -1) @ w), st["tok"], top=3)
            return o, r.logprob, r.entropy, r.top_logprob, r.top_token

        # a long history first
        pre = total - 8
        xx = qkv[:, :pre].reshape(3 * pre, hq + 2 * hkv, d)
        cu = torch.arange(0, 3 * pre + 1, pre, dtype=torch.int32, device=gpu)
        ops.kv_append(st["cache"], xx[:, hq:hq + hkv], xx[:, hq + hkv:], st["table"], st["past"], cu, q=xx[:, :hq], cos=cos, sin=sin)
        st["past"].fill_(pre)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        return st, step, graph, outs, qkv, pre

    made = [build(700), build(3000)]
    for i in range(4):
        for st, step, graph, outs, qkv, pre in made:
            st["x"].copy_(qkv[:, pre + i])
            st["past"].fill_(pre + i)
            graph.replay()
            got = [x.clone() for x in outs]
            kept = [x.clone() for x in st["cache"]]
            eager = step()
            for a, b in zip(got, eager):
                assert torch.equal(a, b)
            for a, b in zip(kept, st["cache"]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            torch.cuda.synchronize()


def test_serving_operators_run_on_the_current_stream(amd, gpu):
    """On a side stream behind a long-running producer the operators see its results; inputs of another stream are fine once waited for."""
    ops = amd.ops
    gen = _gen(14)
    a = torch.randn(4096, 4096, generator=gen).half().to(gpu)
    qkv = torch.randn(130, 12, 64, generator=gen).half().to(gpu)
    want = ops.attention_prompt(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.zeros_like(qkv)
        for _ in range(20):
            b = a @ a
        x.copy_(qkv)
        got = ops.attention_prompt(x[:, :8], x[:, 8:10], x[:, 10:])
        lp = ops.token_logprobs(x.view(130, -1), torch.zeros(130, dtype=torch.int64, device=gpu), top=2)
    s.synchronize()
    assert torch.equal(got, want) and b is not None
    again = ops.token_logprobs(qkv.view(130, -1), torch.zeros(130, dtype=torch.int64, device=gpu), top=2)
    assert torch.equal(lp.logprob, again.logprob) and torch.equal(lp.top_token, again.top_token)


def test_two_calls_at_once(amd, gpu):
    """The same long sequence read from two streams while other calls run: every call has its own scratch memory."""
    c, dev, table = _filled(amd, gpu, [9000], 2, 64, 128, seed=26)
    table, lens = table.to(gpu), torch.tensor([9000], dtype=torch.int32, device=gpu)
    qs = [torch.randn(1, 16, 128, generator=_gen(60 + i)).half().to(gpu) for i in range(8)]
    x = torch.randn(700, 12, 128, generator=_gen(61)).half().to(gpu)
    want = [amd.ops.attention_paged(q, dev, table, lens) for q in qs]
    prompt = amd.ops.attention_prompt(x[:, :8], x[:, 8:10], x[:, 10:])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[], [], []]
    for i in range(8):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[n].append(amd.ops.attention_prompt(x[:, :8], x[:, 8:10], x[:, 10:]) if n == 2 else amd.ops.attention_paged(qs[i], dev, table, lens))
    torch.cuda.synchronize()
    for i in range(8):
        assert torch.equal(got[0][i], want[i]) and torch.equal(got[1][i], want[i]) and torch.equal(got[2][i], prompt)


def test_results_do_not_depend_on_the_run(amd, gpu):
    """No atomics on the way of a sum: the same call twice gives the same bits."""
    c, dev, table = _filled(amd, gpu, [5000, 900], 2, 64, 128, seed=21)
    q = torch.randn(2, 16, 128, generator=_gen(15)).to(torch.bfloat16).to(gpu)
    lens = torch.tensor([5000, 900], dtype=torch.int32, device=gpu)
    x = torch.randn(300, 12, 128, generator=_gen(16)).half().to(gpu)
    lg = torch.randn(600, 5000, generator=_gen(17)).to(gpu)
    tk = torch.zeros(600, dtype=torch.int64, device=gpu)
    run = lambda: (amd.ops.attention_paged(q, dev, table.to(gpu), lens), amd.ops.attention_prompt(x[:, :8], x[:, 8:10], x[:, 10:]),   # noqa: E731
                   *amd.ops.token_logprobs(lg, tk, top=5))
    for a, b in zip(run(), run()):
        assert torch.equal(a, b)


def test_serving_operators_refuse_what_they_do_not_take(amd, gpu):
    ops = amd.ops
    h = dict(dtype=torch.float16, device=gpu)
    q, k = torch.zeros(4, 4, 64, **h), torch.zeros(4, 2, 64, **h)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=gpu)
    bad = [
        lambda: ops.attention_prompt(q, k, k[:, :1]), lambda: ops.attention_prompt(q, k[:3], k[:3]), lambda: ops.attention_prompt(q[0], k, k),
        lambda: ops.attention_prompt(q[:, :3], k, k), lambda: ops.attention_prompt(q, k, k, cu.long()), lambda: ops.attention_prompt(q, k, k, cu.cpu()),
        lambda: ops.attention_prompt(q, k, k, cu, scale=0.0), lambda: ops.attention_prompt(q, k, k, cu, scale=math.nan),
        lambda: ops.attention_prompt(q, k.bfloat16(), k), lambda: ops.attention_prompt(torch.zeros(4, 4, 65, **h)[..., :64], k, k),
        lambda: ops.attention_prompt(q.transpose(1, 2).contiguous().transpose(1, 2), k, k), lambda: ops.attention_prompt(q, k.expand(4, 2, 64)[:1].expand(4, 2, 64), k),
        lambda: ops.attention_prompt(torch.zeros(4, 4, 136, **h), torch.zeros(4, 2, 136, **h), torch.zeros(4, 2, 136, **h)),
        lambda: ops.attention_prompt(q, k, k, out=q[:3]), lambda: ops.attention_prompt(q, k, k, out=torch.zeros(1, 4, 64, **h).expand(4, 4, 64)), lambda: ops.attention_prompt(q.cpu(), k, k),
    ]
    cache = ops.PagedCache.empty(4, 2, 16, 64, gpu)
    table = torch.zeros(4, 2, dtype=torch.int32, device=gpu)
    lens = torch.ones(4, dtype=torch.int32, device=gpu)
    cos = torch.zeros(8, 32, device=gpu)
    odd = ops.PagedCache.empty(4, 2, 24, 64, gpu)
    wide = ops.PagedCache.empty(4, 2, 16, 144, gpu)
    bad += [
        lambda: ops.kv_append(cache, k, k, table, lens[:3]), lambda: ops.kv_append(cache, k[:3], k[:3], table, lens), lambda: ops.kv_append(odd, k, k, table, lens),
        lambda: ops.kv_append(cache, k, k, table, lens, q=q), lambda: ops.kv_append(cache, k, k, table, lens, q=q, cos=cos),
        lambda: ops.kv_append(cache, k, k, table, lens, cos=cos[:, :4].contiguous(), sin=cos[:, :4].contiguous()),
        lambda: ops.kv_append(cache, k, k, table, lens, cos=cos.half(), sin=cos.half()), lambda: ops.kv_append(cache, k, k, table.long(), lens),
        lambda: ops.kv_append(cache, k, k, table, lens, q_out=q), lambda: ops.kv_append(cache, q, q, table, lens),
        lambda: ops.kv_append(cache._replace(k_scale=cache.k_scale[:2]), k, k, table, lens), lambda: ops.kv_append(cache._replace(v=cache.k), k, k, table, lens),
        lambda: ops.kv_append(wide, torch.zeros(4, 2, 144, **h), torch.zeros(4, 2, 144, **h), table, lens),
        lambda: ops.attention_paged(q, cache, table, lens[:2]), lambda: ops.attention_paged(q[:3], cache, table, lens), lambda: ops.attention_paged(q[:, :3], cache, table, lens),
        lambda: ops.attention_paged(q[..., :32], cache, table, lens), lambda: ops.attention_paged(q, odd, table, lens), lambda: ops.attention_paged(q, cache, table, lens, scale=-1.0),
        lambda: ops.attention_paged(q, cache, table[0], lens), lambda: ops.attention_paged(q, cache, table, lens, cu),
    ]
    x, t = torch.zeros(4, 100, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    bad += [
        lambda: ops.token_logprobs(x, t[:3]), lambda: ops.token_logprobs(x, t.int()), lambda: ops.token_logprobs(x, t, top=33), lambda: ops.token_logprobs(x[:, :5], t, top=6),
        lambda: ops.token_logprobs(x, t, top=-1), lambda: ops.token_logprobs(x.cpu(), t), lambda: ops.token_logprobs(x, t.cpu()), lambda: ops.token_logprobs(x[:, :0], t),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    for call in (lambda: ops.token_logprobs(x.double(), t), lambda: ops.attention_prompt(q.float(), k.float(), k.float())):
        with pytest.raises(NotImplementedError):
            call()
    for call in (lambda: ops.token_logprobs(x.clone().requires_grad_(), t), lambda: ops.attention_prompt(q.clone().requires_grad_(), k, k),
                 lambda: ops.attention_paged(q.clone().requires_grad_(), cache, table, lens), lambda: ops.kv_append(cache, k.clone().requires_grad_(), k, table, lens)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with torch.no_grad():
        ops.token_logprobs(x.clone().requires_grad_(), t)
    empty = ops.attention_prompt(q[:0], k[:0], k[:0])
    assert empty.shape == (0, 4, 64)
    assert ops.attention_paged(q[:0], cache, table[:0], lens[:0]).shape == (0, 4, 64)
    assert ops.kv_append(cache, k[:0], k[:0], table[:0], lens[:0]) is None

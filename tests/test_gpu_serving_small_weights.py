"""Attention rows in which many weights far below the largest add up: they must not be lost in the weights' 16 bits."""
import math

import pytest
import torch

from tests._serving_small import attend_rows
from tests.test_gpu_serving import _close, _gen

pytestmark = pytest.mark.gpu


def _sink(n, d, powers, dtype, gen):
    """q, k, v (n, d): the first key's score is `powers` powers of two above the others' (which differ by up to one); its value is
    0 in the first half of the channels, the others' values are between 1/2 and 1 there."""
    scale = d ** -0.5
    q = torch.ones(n, d, dtype=torch.float64)
    k = torch.zeros(n, d, dtype=torch.float64)
    k[1:] = -(powers + torch.rand(n - 1, 1, generator=gen, dtype=torch.float64)) * math.log(2) / (scale * d)
    v = torch.rand(n, d, generator=gen, dtype=torch.float64) / 2 + 0.5
    v[0, :d // 2] = 0.0
    v[1:, d // 2:] -= 0.75
    return (x.to(dtype) for x in (q, k, v)), scale


@pytest.mark.parametrize("powers", [16, 20, 24, 26, 28])
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 64)])
def test_prompt_rows_under_a_dominant_token(amd, gpu, powers, dtype, d):
    n, rows = 16384, 3
    (q, k, v), scale = _sink(n, d, powers, dtype, _gen(powers))
    got = amd.ops.attention_prompt(*(x.to(gpu).unsqueeze(1) for x in (q, k, v)), causal=False)[:rows, 0]
    want, bound = attend_rows(q[:rows].double(), k.double(), v.double(), scale, dtype, dtype)
    assert float(want[0, 0]) > 4 * float(bound[0, 0])   # (what is looked for is larger than what is allowed)
    _close(got, want, bound)


def test_prompt_rows_whose_largest_token_comes_last(amd, gpu):
    """The reference lags up to 2^8 behind a maximum that creeps up: weights at the upper end of fp16."""
    n, d = 4096, 64
    scale = d ** -0.5
    gen = _gen(3)
    q = torch.ones(n, d).half()
    k = (torch.linspace(-20.0, 0.0, n)[:, None] * math.log(2) / (scale * d)).expand(n, d).half()
    v = (torch.rand(n, d, generator=gen) - 0.25).half()
    got = amd.ops.attention_prompt(*(x.to(gpu).unsqueeze(1) for x in (q, k, v)), causal=False)[:2, 0]
    _close(got, *attend_rows(q[:2].double(), k.double(), v.double(), scale, torch.float16, torch.float16))


# ---- over the paged cache ----------------------------------------------------------------------------------------------

E4M3 = torch.float8_e4m3fn


def _pages(x, page, codes_of):
    """Tokens x (n, d) of one head as codes in pages, the last filled up: (pages, page, d)"""
    n, d = x.shape
    out = torch.full((-(-n // page) * page, d), 1.0)
    out[:n] = x
    return codes_of(out.view(-1, page, d))


def _paged_sink(n, d, page, powers, ratio, at, gen):
    """A cache of one sequence and head in which token `at` stands `powers` powers of two above all others, on a page whose value
    scale is 2^ratio of the others'; its codes are 0 in the first half of the channels, the others' of one sign there.
    (cache tensors, q row, softmax scale, keys, values in 64 bits)"""
    k8 = torch.zeros(n, d)
    k8[:, 0] = -16.0 * powers
    k8[:, 1] = -16 * torch.rand(n, generator=gen)
    k8[at] = 0.0
    v8 = 224 + 224 * torch.rand(n, d, generator=gen)
    v8[at, :d // 2] = 0.0
    v8[:, d // 2:] *= torch.rand(n, d - d // 2, generator=gen).round() * 2 - 1
    k, v = (_pages(x, page, lambda y: y.clamp(-448, 448).to(E4M3)) for x in (k8, v8))
    ks = torch.full((k.shape[0], 1), 2.0 ** -7)
    vs = torch.full((k.shape[0], 1), 1.25 * 2.0 ** -9)
    vs[at // page] *= 2.0 ** ratio
    kk = (k.double() * ks.double()[..., None]).view(-1, d)[:n]
    vv = (v.double() * vs.double()[..., None]).view(-1, d)[:n]
    return (k.unsqueeze(1), v.transpose(1, 2).contiguous().unsqueeze(1), ks, vs), torch.ones(1, d, dtype=torch.float64), math.log(2) * 8, kk, vv


@pytest.mark.parametrize("n,d,page,heads,dtype", [(131071, 64, 64, 1, torch.float16), (131071, 128, 64, 20, torch.bfloat16), (40000, 128, 16, 4, torch.float16),
                                                  (70001, 64, 32, 24, torch.float16), (3000, 80, 128, 2, torch.bfloat16)])
@pytest.mark.parametrize("powers", [14, 18, 24])
@pytest.mark.parametrize("ratio", [-7, 0, 8, 14])
def test_paged_rows_under_a_dominant_token(amd, gpu, n, d, page, heads, dtype, powers, ratio):
    """The first token, a page with a value scale of its own."""
    cache, q, scale, k, v = _paged_sink(n, d, page, powers, ratio, 0, _gen(powers + d))
    dev = amd.ops.PagedCache(*(x.to(gpu) for x in cache))
    table = torch.arange(cache[0].shape[0], dtype=torch.int32, device=gpu)[None]
    got = amd.ops.attention_paged(q.to(dtype).to(gpu).expand(1, heads, d).contiguous(), dev, table, torch.tensor([n], dtype=torch.int32, device=gpu), scale=scale)
    want, bound = attend_rows(q, k, v, scale, dtype, torch.float16)
    if n > 40000 and powers < 24:
        assert float(want[0, 0]) > 4 * float(bound[0, 0])
    for h in range(heads):
        _close(got[:, h], want, bound)


@pytest.mark.parametrize("ratio", [-15, 3, 7])
def test_paged_rows_under_a_dominant_token_in_the_middle(amd, gpu, ratio):
    """Two sequences of several query tokens whose dominant token lies in the middle, on a page of a smaller or a larger scale."""
    n, d, page = 20000, 64, 16
    cache, q, scale, k, v = _paged_sink(n, d, page, 17, ratio, 9007, _gen(40 + ratio))
    dev = amd.ops.PagedCache(*(x.to(gpu) for x in cache))
    table = torch.arange(cache[0].shape[0], dtype=torch.int32, device=gpu).expand(2, -1).contiguous()
    lens, cu = torch.tensor([n, n - 3], dtype=torch.int32, device=gpu), torch.tensor([0, 2, 4], dtype=torch.int32, device=gpu)
    got = amd.ops.attention_paged(q.half().to(gpu).expand(4, 2, d).contiguous(), dev, table, lens, cu, scale=scale)
    for row, seen in enumerate((n - 1, n, n - 4, n - 3)):
        want, bound = attend_rows(q, k[:seen], v[:seen], scale, torch.float16, torch.float16)
        for h in range(2):
            _close(got[row:row + 1, h], want, bound)


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("ratio", [-15, -9, 7, -40, 40])
def test_paged_values_of_every_code_at_far_scales(amd, gpu, page, ratio):
    """A row that sees one token alone, of the second page, whose scale is 2^ratio of the first's: every code comes out as it is."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 127) != 127]   # without the two NaN
    d = 64
    for part in range(4):
        v = torch.zeros(2, 1, d, page)
        v8 = v.to(E4M3)
        row = codes[part * d:part * d + d]
        row = torch.cat([row, row[:0].new_zeros(d - len(row))])
        v8.view(torch.uint8)[1, 0, :, 1] = row
        v8.view(torch.uint8)[0, 0, :, 2] = row
        k = torch.full((2, 1, page, d), -448.0)
        k[1, 0, 1] = 448.0
        vs = torch.tensor([[2.0 ** -4], [2.0 ** (ratio - 4)]])
        dev = amd.ops.PagedCache(*(x.to(gpu) for x in (k.to(E4M3), v8, torch.ones(2, 1), vs)))
        got = amd.ops.attention_paged(torch.ones(1, 1, d, dtype=torch.bfloat16, device=gpu), dev, torch.tensor([[0, 1]], dtype=torch.int32, device=gpu),
                                      torch.tensor([page + 2], dtype=torch.int32, device=gpu), scale=1.0)
        # one weight, off by 2^-11 of itself at most against the denominator's: less than half a step of bf16, where codes have 4 bits
        assert torch.equal(got.cpu()[0, 0].double(), row.view(E4M3).double() * 2.0 ** (ratio - 4))


def test_paged_nan_of_later_tokens_beside_far_scales(amd, gpu):
    """Values taken one token at a time (a NaN that some rows do not see) have their page's scale as well."""
    from tests.test_gpu_serving import _check_paged, _cu, _filled
    lens, new = [77, 64], [3, 3]
    c, dev, table = _filled(amd, gpu, lens, 1, 16, 64, seed=6, spread=4.0)
    dev.v.view(torch.uint8)[int(table[0, 4]), 0, 9, 12] = 0x7f   # token 76: the last query token's own
    q = torch.randn(6, 4, 64, generator=_gen(6)).half()
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu)).cpu()
    assert torch.isnan(got[2, :, 9]).all()
    got[2, :, 9] = 0
    k, v, vs = c.tokens(table[0], 77)
    from tests import _serving_ref as ref
    want, bound = ref.attend(q[:3].double(), k, v, 74, 0.125, torch.float16, vmax=vs)
    want[2, :, 9] = 0
    _close(got[:3], want, bound)
    _check_paged(got[3:], q[3:], c, table[1:], lens[1:], new[1:], torch.float16)

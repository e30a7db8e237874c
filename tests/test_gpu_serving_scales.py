"""Attention over pages whose scales are damaged."""
import math

import pytest
import torch

from tests import _serving_ref as ref
from tests.test_gpu_serving import _check_paged, _close, _cu, _filled, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, -math.nan, math.inf])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_paged_rows_that_see_a_damaged_scale_are_nan(amd, gpu, bad, which, page):
    """Single tokens: the sequence with the damaged page is NaN, the others, one of them shorter than a tile, are as ever."""
    lens = [130, 200, 5]
    c, dev, table = _filled(amd, gpu, lens, 2, page, 64, seed=31, spread=1.0)
    getattr(dev, which)[int(table[0, 40 // page]), 1] = bad
    q = torch.randn(3, 4, 64, generator=_gen(32)).half()
    got = amd.ops.attention_paged(q.to(gpu), dev, table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)).cpu()
    assert torch.isnan(got[0, 2:]).all()
    k, v, vs = c.tokens(table[0], 130)
    want, bound = ref.attend(q[:1].double(), k, v, 129, 0.125, torch.float16, vmax=vs)
    _close(got[:1, :2], want[:, :2], bound[:, :2])
    _check_paged(got[1:], q[1:], c, table[1:], lens[1:], [1, 1], torch.float16)


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_paged_rows_before_a_damaged_scale(amd, gpu, which):
    """A chunk: rows in front of the damaged page do not see it.  The first page of the pool, which stands in for pages behind a
    sequence's end, is damaged as well and reaches nobody."""
    lens, new = [100, 70], [60, 3]
    c, dev, table = _filled(amd, gpu, lens, 1, 16, 64, seed=33)
    spare = next(p for p in range(dev.k.shape[0]) if p not in table.flatten().tolist())
    for x in (*dev, c.k, c.v, c.ks, c.vs):   # the spare page becomes the first
        x.view(torch.uint8 if x.element_size() == 1 else x.dtype)[[0, spare]] = x.view(torch.uint8 if x.element_size() == 1 else x.dtype)[[spare, 0]]
    moved = table.clone()
    moved[table == 0] = spare
    getattr(dev, which)[0] = math.nan
    getattr(dev, which)[int(moved[0, 5])] = math.nan   # tokens 80..95, rows 40..
    q = torch.randn(63, 4, 64, generator=_gen(34)).half()
    got = amd.ops.attention_paged(q.to(gpu), dev, moved.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), _cu(new, gpu)).cpu()
    assert torch.isnan(got[40:60]).all()
    k, v, vs = c.tokens(moved[0], 80)
    want, bound = ref.attend(q[:40].double(), k, v, 40, 0.125, torch.float16, vmax=vs)
    _close(got[:40], want, bound)
    _check_paged(got[60:], q[60:], c, moved[1:], lens[1:], new[1:], torch.float16)


def test_paged_scales_from_the_smallest_on(amd, gpu):
    """A scale of 0 and one below 2^-100 count as 2^-100."""
    c, dev, table = _filled(amd, gpu, [90], 1, 16, 64, seed=35)
    q = torch.randn(1, 4, 64, generator=_gen(36)).bfloat16().to(gpu)
    lens = torch.tensor([90], dtype=torch.int32, device=gpu)
    outs = [amd.ops.attention_paged(q, dev._replace(v_scale=torch.full_like(dev.v_scale, s)), table.to(gpu), lens) for s in (2.0 ** -100, 0.0, 1e-40, 2.0 ** -120)]
    assert all(torch.equal(outs[0], x) for x in outs[1:]) and (outs[0] != 0).any()


@pytest.mark.parametrize("bad", [math.nan, -math.nan, math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_append_to_a_page_of_a_damaged_scale(amd, gpu, bad, which):
    """The tokens that the page holds become NaN, the new one and the other head's are what they would be anyway."""
    gen = _gen(37)
    pools = [amd.ops.PagedCache.empty(1, 2, 16, 32, gpu) for _ in range(2)]
    k, v = torch.randn(6, 2, 32, generator=gen).half().to(gpu), torch.randn(6, 2, 32, generator=gen).half().to(gpu)
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    past = lambda n: torch.tensor([n], dtype=torch.int32, device=gpu)   # noqa: E731
    for i, dev in enumerate(pools):
        amd.ops.kv_append(dev, k[:5], v[:5], table, past(0), _cu([5], gpu))
        if i:
            getattr(dev, which + "_scale")[0, 1] = bad
        amd.ops.kv_append(dev, k[5:] * 64, v[5:] * 64, table, past(5))   # (a larger scale than before, so that both ways end at one)
    tokens = [tuple(x.float().cpu() for x in (dev.k, dev.v.transpose(2, 3))) for dev in pools]
    for name, a, b in zip("kv", *tokens):
        if name == which:
            assert torch.isnan(b[0, 1, :5]).all()
            b[0, 1, :5] = a[0, 1, :5]
        assert torch.equal(a, b)
    for a, b in zip(pools[0][2:], pools[1][2:]):
        assert torch.equal(a, b)

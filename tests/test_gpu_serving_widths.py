"""Appending with rotary widths that are no multiple of 16, bit for bit against the restatement (tests/_serving_ref.py)."""
import pytest
import torch

from tests import _serving_ref as ref
from tests.test_gpu_serving import Both, _cu, _gen, _tables

pytestmark = pytest.mark.gpu

# (head_dim, rotary_dim): halves of 20, 10, 12, 9, 63, 15 and 17 channels, and 8 r + 4, 8 r - 1
WIDTHS = [(80, 40), (80, 20), (96, 24), (64, 18), (128, 126), (32, 30), (48, 34), (128, 72), (112, 94)]


@pytest.mark.parametrize("d,rot", WIDTHS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_of_any_even_rotary_width(amd, gpu, d, rot, interleaved, dtype):
    """Chunks that begin and end inside pages, scales that grow, single tokens; two kv heads, three query heads."""
    c = Both(amd, gpu, 2, 8, 2, 16, d, seed=d + rot)
    for i, n in enumerate([[17, 1], [1, 40], [33, 2]]):
        c.append(n, dtype, rot, interleaved, q_heads=3, scale=4.0 ** i)
    for i in range(3):
        c.append([1, 1], dtype, rot, interleaved, q_heads=3, scale=[1.0, 300.0, 0.01][i], single=True)


@pytest.mark.parametrize("page", [32, 64, 128])
def test_append_of_any_even_rotary_width_in_larger_pages(amd, gpu, page):
    c = Both(amd, gpu, 2, 4, 1, page, 80, seed=page)
    c.append([page + 5, 2 * page], torch.float16, 40, False, q_heads=5)
    c.append([page // 2, 3], torch.float16, 40, False, q_heads=5, scale=8.0)
    many = Both(amd, gpu, 1, 1200 // page + 1, 1, page, 96, seed=page + 1)   # more tokens than one workgroup's items of queries
    many.append([1100], torch.bfloat16, 24, True, q_heads=2)


@pytest.mark.parametrize("d,rot", WIDTHS)
def test_append_of_any_even_rotary_width_in_place(amd, gpu, d, rot):
    """q rotated where it stands in a merged product; tables whose first row is left out, so that they begin at 4 bytes."""
    gen = _gen(d * rot)
    for inter in (False, True):
        dev = amd.ops.PagedCache.empty(3, 2, 16, d, gpu)
        qkv = torch.randn(40, 8, d, generator=gen).half()
        x = qkv.to(gpu)
        cos, sin = _tables(41, rot)
        q = x[:, :4]
        got = amd.ops.kv_append(dev, x[:, 4:6], x[:, 6:], torch.tensor([[2, 1, 0]], dtype=torch.int32, device=gpu),
                                torch.zeros(1, dtype=torch.int32, device=gpu), _cu([40], gpu), q=q, cos=cos.to(gpu)[1:], sin=sin.to(gpu)[1:],
                                interleaved=inter, q_out=q)
        assert torch.equal(got.cpu(), ref.rotate(qkv[:, :4], torch.arange(1, 41), cos, sin, inter).half())
        assert torch.equal(x[:, 4:].cpu(), qkv[:, 4:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_any_even_rotary_width_passes_infinities_by(amd, gpu, interleaved):
    """Infinite and NaN channels behind the rotated part stay what they are, and a query without an angle is NaN."""
    gen = _gen(5)
    c = Both(amd, gpu, 1, 1, 1, 16, 80, seed=6)
    k, v = torch.randn(9, 1, 80, generator=gen), torch.randn(9, 1, 80, generator=gen)
    k[0, 0, 40], k[1, 0, 47], k[2, 0, 48], k[3, 0, 79] = float("inf"), float("-inf"), float("nan"), float("inf")
    c.append([9], torch.float16, 40, interleaved, k=k, v=v)
    cos, sin = _tables(3, 40)
    q = torch.randn(5, 2, 80, generator=gen).half()
    dev = amd.ops.PagedCache.empty(1, 1, 16, 80, gpu)
    kv = torch.zeros(5, 1, 80, dtype=torch.float16, device=gpu)
    got = amd.ops.kv_append(dev, kv, kv, torch.zeros(1, 1, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu), _cu([5], gpu),
                            q=q.to(gpu), cos=cos.to(gpu), sin=sin.to(gpu), interleaved=interleaved).cpu()
    assert torch.equal(got[:3], ref.rotate(q[:3], torch.arange(3), cos, sin, interleaved).half()) and torch.isnan(got[3:]).all()

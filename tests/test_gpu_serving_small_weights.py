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

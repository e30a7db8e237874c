"""Output rows of the prompt attention in each wave's place of a workgroup's tile."""
import pytest
import torch

from tests import _serving_ref as ref
from tests.test_gpu_serving import _close, _cu, _gen, _qkv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,dtype", [(16, torch.float16), (64, torch.bfloat16), (72, torch.float16), (96, torch.bfloat16), (104, torch.float16), (128, torch.float16)])
def test_prompt_rows_of_every_wave(amd, gpu, causal, d, dtype):
    """Lengths at which each of the four waves' 32 rows are the last of a tile, whole or in part, after one and after two tiles;
    the output rows lie apart in a wider tensor whose other channels stay."""
    lens = [n + m for n in (0, 128, 256) for m in (1, 32, 33, 64, 90, 96, 97, 128)]
    t = sum(lens)
    x, views = _qkv(_gen(d), t, 4, 2, d, dtype, "merged", gpu)
    wide = torch.full((t, 6, d + 8), 7.0, dtype=dtype, device=gpu)
    out = wide[:, 1:5, :d]
    got = amd.ops.attention_prompt(*views, _cu(lens, gpu), causal=causal, out=out).cpu()
    at = 0
    for n in lens:
        s = x[at:at + n].double()
        _close(got[at:at + n], *ref.attend(s[:, :4], s[:, 4:6], s[:, 6:], 0 if causal else None, d ** -0.5, dtype))
        at += n
    assert (wide[:, 0] == 7.0).all() and (wide[:, 5] == 7.0).all() and (wide[..., d:] == 7.0).all()

"""What the serving operators write is known to torch as written."""
import pytest
import torch

from tests.test_gpu_serving import _cu

pytestmark = pytest.mark.gpu


def test_written_tensors_have_a_new_version(amd, gpu):
    ops = amd.ops
    x = torch.randn(4, 8, 64, dtype=torch.float16, device=gpu)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    cache = ops.PagedCache.empty(4, 2, 16, 64, gpu)
    table, lens = torch.arange(4, dtype=torch.int32, device=gpu).view(4, 1), torch.zeros(4, dtype=torch.int32, device=gpu)
    cos = torch.ones(4, 32, device=gpu)
    out = torch.empty(4, 4, 64, dtype=torch.float16, device=gpu)

    def rises(ts, call):
        was = [t._version for t in ts]
        call()
        assert all(t._version > w for t, w in zip(ts, was))

    rises((out,), lambda: ops.attention_prompt(q, k, v, out=out))
    rises((*cache, out), lambda: ops.kv_append(cache, k, v, table, lens, q=q, cos=cos, sin=cos, q_out=out))
    rises((out,), lambda: ops.attention_paged(q, cache, table, lens + 1, out=out))
    rises((x, q, k), lambda: ops.kv_append(cache, k, v, table, lens, q=q, cos=cos, sin=cos, q_out=q))   # views share their base's
    was = [t._version for t in (x, *cache)]
    ops.attention_prompt(q, k, v)
    ops.attention_paged(q, cache, table, lens + 1)
    ops.token_logprobs(x.view(32, 64), torch.zeros(32, dtype=torch.int64, device=gpu))
    assert was == [t._version for t in (x, *cache)]   # what is only read keeps its own


def test_a_saved_output_that_is_overwritten_is_stale(amd, gpu):
    """Autograd refuses to go back through a tensor that a call has written since."""
    ops = amd.ops
    x = torch.randn(4, 8, 64, dtype=torch.float16, device=gpu)
    out = ops.attention_prompt(x[:, :4], x[:, 4:6], x[:, 6:])
    w = torch.ones((), dtype=torch.float16, device=gpu, requires_grad=True)
    y = (w * out).sum()
    ops.attention_prompt(x[:, :4], x[:, 4:6], x[:, 6:], out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors_are_taken(amd, gpu):
    """Made in inference mode, written in it and out of it."""
    ops = amd.ops
    with torch.inference_mode():
        x = torch.randn(4, 8, 64, dtype=torch.float16, device=gpu)
        cache = ops.PagedCache.empty(4, 2, 16, 64, gpu)
        out = torch.empty(4, 4, 64, dtype=torch.float16, device=gpu)
    table, lens = torch.arange(4, dtype=torch.int32, device=gpu).view(4, 1), torch.zeros(4, dtype=torch.int32, device=gpu)
    cos = torch.ones(4, 32, device=gpu)
    got = []
    for mode in (True, False):
        with torch.inference_mode(mode):
            ops.kv_append(cache, x[:, 4:6], x[:, 6:], table, lens, q=x[:, :4], cos=cos, sin=cos, q_out=out)
            got.append(ops.attention_paged(out, cache, table, lens + 1))
            got.append(ops.attention_prompt(x[:, :4], x[:, 4:6], x[:, 6:], _cu([4], gpu)))
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])

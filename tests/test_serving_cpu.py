"""The serving operators without a GPU: what the C entries refuse before they touch the device (with pointers that lead
nowhere), what they answer without a launch, and what the binding refuses.  No kernel is launched here."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from tests.conftest import ROOT

I64, PTR = ctypes.c_int64, ctypes.c_void_p
FAKE = 1 << 20   # aligned, never read


class Rows(ctypes.Structure):
    _fields_ = [("data", PTR), ("token_stride", I64), ("head_stride", I64)]


class Cache(ctypes.Structure):
    _fields_ = [(n, PTR) for n in ("k_codes", "v_codes", "k_scale", "v_scale")] + [(n, I64) for n in ("n_pages", "n_kv_heads", "page", "head_dim")]


class Prompt(ctypes.Structure):
    _fields_ = [(n, Rows) for n in ("out", "q", "k", "v")] + [(n, I64) for n in ("dtype", "n_tokens", "n_heads", "n_kv_heads", "head_dim")] + [
        ("cu_seqlens", PTR), ("batch", I64), ("causal", I64), ("softmax_scale", ctypes.c_double)]


class Append(ctypes.Structure):
    _fields_ = [("cache", Cache)] + [(n, Rows) for n in ("k", "v", "q", "q_out")] + [
        ("dtype", I64), ("n_tokens", I64), ("n_heads", I64), ("block_table", PTR), ("table_width", I64), ("past_lens", PTR), ("cu_seqlens", PTR),
        ("batch", I64), ("cos", PTR), ("sin", PTR), ("max_pos", I64), ("rotary_dim", I64), ("interleaved", I64)]


class Paged(ctypes.Structure):
    _fields_ = [("cache", Cache), ("out", Rows), ("q", Rows), ("dtype", I64), ("n_tokens", I64), ("n_heads", I64), ("block_table", PTR),
                ("table_width", I64), ("seq_lens", PTR), ("cu_seqlens", PTR), ("batch", I64), ("softmax_scale", ctypes.c_double), ("workspace", PTR),
                ("workspace_bytes", I64)]


class Logprobs(ctypes.Structure):
    _fields_ = [("logits", PTR), ("dtype", I64), ("n_rows", I64), ("row_stride", I64), ("vocab", I64), ("tokens", PTR), ("ignore_index", I64),
                ("logprob", PTR), ("entropy", PTR), ("top", I64), ("top_logprob", PTR), ("top_token", PTR)]


STRUCTS = {Prompt: "gq_attention_prompt", Append: "gq_kv_append", Paged: "gq_attention_paged", Logprobs: "gq_token_logprobs"}


def _prompt():
    a = Prompt(dtype=0, n_tokens=40, n_heads=4, n_kv_heads=2, head_dim=64, cu_seqlens=FAKE, batch=3, causal=1, softmax_scale=0.125)
    for r, heads in ((a.out, 4), (a.q, 4), (a.k, 2), (a.v, 2)):
        r.data, r.token_stride, r.head_stride = FAKE, heads * 64, 64
    return a


def _cache():
    return Cache(FAKE, FAKE, FAKE, FAKE, 9, 2, 16, 64)


def _append():
    a = Append(cache=_cache(), dtype=1, n_tokens=3, n_heads=4, block_table=FAKE, table_width=4, past_lens=FAKE, batch=3, cos=FAKE, sin=FAKE,
               max_pos=100, rotary_dim=64)
    for r, heads in ((a.k, 2), (a.v, 2), (a.q, 4), (a.q_out, 4)):
        r.data, r.token_stride, r.head_stride = FAKE, heads * 64, 64
    return a


def _paged():
    a = Paged(cache=_cache(), dtype=0, n_tokens=3, n_heads=4, block_table=FAKE, table_width=4, seq_lens=FAKE, batch=3, softmax_scale=0.125)
    for r in (a.out, a.q):
        r.data, r.token_stride, r.head_stride = FAKE, 256, 64
    return a


def _logprobs():
    return Logprobs(logits=FAKE, dtype=2, n_rows=5, row_stride=1000, vocab=1000, tokens=FAKE, ignore_index=-100, logprob=FAKE, entropy=FAKE, top=3,
                    top_logprob=FAKE, top_token=FAKE)


def _set(a, path, value):
    *owner, last = path.split(".")
    for name in owner:
        a = getattr(a, name)
    setattr(a, last, value)


def _call(a):
    from gptq_v2_amd import _lib
    lib = _lib.load()
    name = STRUCTS[type(a)]
    return getattr(lib, name)(ctypes.addressof(a), None), name, lib


def _refused(a, code=-1):
    rc, name, lib = _call(a)
    assert rc == code, (name, rc)
    assert lib.gq_last_error().decode().startswith(name)


def test_the_structs_of_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "gptq_amd.h"\nint main(void) { printf("%zu %zu %zu %zu", ' +
                   ", ".join(f"sizeof({n}_args)" for n in STRUCTS.values()) + "); return 0; }\n")
    exe = str(tmp_path / "sizes")
    subprocess.check_call(["gcc", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src), "-o", exe])
    assert [int(x) for x in subprocess.check_output([exe]).split()] == [ctypes.sizeof(s) for s in STRUCTS] == [168, 264, 200, 96]


@pytest.mark.parametrize("path,value", [
    ("dtype", 2), ("dtype", -1), ("dtype", 1 << 32), ("head_dim", 0), ("head_dim", 60), ("head_dim", 136), ("head_dim", 1 << 40), ("n_heads", 0), ("n_heads", 3),
    ("n_heads", -4), ("n_heads", 1 << 33), ("n_kv_heads", 0), ("n_kv_heads", -2), ("n_tokens", -1), ("n_tokens", 1 << 30), ("batch", -1), ("batch", 1 << 24),
    ("cu_seqlens", None), ("softmax_scale", 0.0), ("softmax_scale", -1.0), ("softmax_scale", math.nan), ("softmax_scale", math.inf), ("softmax_scale", 3e38),
    ("softmax_scale", 1e-60), ("out.data", None), ("q.data", None), ("k.data", None), ("v.data", None), ("out.data", FAKE + 8), ("q.data", FAKE + 2), ("k.data", FAKE + 4),
    ("v.data", FAKE + 8), ("q.token_stride", 260), ("q.head_stride", 68), ("k.token_stride", 132), ("v.head_stride", 4), ("out.head_stride", 68), ("k.token_stride", 56),
    ("v.token_stride", 0), ("v.token_stride", (1 << 23) + 8), ("k.token_stride", -128), ("out.token_stride", 0), ("out.token_stride", 192), ("out.head_stride", 0),
    ("out.head_stride", 56),
])
def test_prompt_attention_refusals(path, value):
    a = _prompt()
    _set(a, path, value)
    _refused(a)


@pytest.mark.parametrize("path,value", [
    ("dtype", 2), ("cache.head_dim", 24), ("cache.head_dim", 144), ("cache.head_dim", 0), ("cache.page", 0), ("cache.page", 8), ("cache.page", 48), ("cache.page", 256),
    ("cache.n_kv_heads", 0), ("cache.n_kv_heads", -1), ("cache.n_kv_heads", 1 << 17), ("cache.n_pages", -1), ("n_tokens", -1), ("n_tokens", 4), ("batch", -3), ("batch", 2),
    ("table_width", -1), ("n_heads", 0), ("n_heads", 1 << 20), ("rotary_dim", -16), ("rotary_dim", 8), ("rotary_dim", 80), ("rotary_dim", 0), ("max_pos", 0), ("max_pos", -1),
    ("cos", None), ("sin", None), ("cos", FAKE + 4), ("k.data", None), ("v.data", None), ("q_out.data", None), ("k.data", FAKE + 8), ("q.data", FAKE + 8),
    ("cache.k_codes", None), ("cache.v_codes", FAKE + 8), ("cache.k_scale", None), ("cache.v_scale", None), ("block_table", None), ("past_lens", None),
    ("k.token_stride", 132), ("v.head_stride", 65), ("q.token_stride", 4), ("q_out.head_stride", 60), ("q_out.token_stride", 0), ("q_out.head_stride", 8),
])
def test_append_refusals(path, value):
    a = _append()
    _set(a, path, value)
    _refused(a)


@pytest.mark.parametrize("path,value", [
    ("dtype", 2), ("cache.head_dim", 24), ("cache.head_dim", 144), ("cache.head_dim", 1 << 33), ("cache.page", 8), ("cache.page", 1 << 34), ("cache.n_kv_heads", 3),
    ("cache.n_kv_heads", 0), ("cache.n_pages", 0), ("cache.n_pages", -1), ("cache.n_pages", 1 << 31), ("n_tokens", -1), ("n_tokens", 4), ("batch", 2), ("batch", -1),
    ("table_width", -1), ("table_width", 1 << 26), ("n_heads", 0), ("n_heads", 6), ("n_heads", 1 << 32), ("softmax_scale", 0.0), ("softmax_scale", math.nan),
    ("softmax_scale", 3e38), ("out.data", None), ("q.data", None), ("seq_lens", None), ("block_table", None), ("cache.k_codes", None), ("cache.v_codes", None),
    ("cache.k_scale", None), ("cache.v_scale", None), ("cache.k_codes", FAKE + 4), ("q.data", FAKE + 8), ("out.data", FAKE + 8), ("q.token_stride", 4),
    ("out.head_stride", 60), ("out.token_stride", 0), ("out.head_stride", 0),
])
def test_paged_attention_refusals(path, value):
    a = _paged()
    _set(a, path, value)
    _refused(a)


def test_paged_attention_wants_its_workspace():
    """A long table is cut into runs: the call says what it needs, one byte less or no pointer is refused."""
    from gptq_v2_amd import _lib
    need = _lib.load().gq_attention_paged_workspace(3, 3, 0, 4, 2, 64, 16, 4096)
    assert need > 0 and need % 16 == 0
    a = _paged()
    a.table_width = 4096
    _refused(a, -4)
    a.workspace, a.workspace_bytes = FAKE, need - 1
    _refused(a, -4)
    a.workspace_bytes = -1
    _refused(a, -4)
    a.workspace, a.workspace_bytes = FAKE + 8, need
    _refused(a)
    ws = _lib.load().gq_attention_paged_workspace
    assert ws(3, 3, 0, 4, 2, 64, 16, 4) == 0 and ws(0, 3, 0, 4, 2, 64, 16, 4096) == 0 and ws(3, 3, 0, 4, 3, 64, 16, 4096) == 0
    assert ws(3, 3, 0, 4, 2, 64, 24, 4096) == 0 and ws(-3, 3, 0, 4, 2, 64, 16, 4096) == 0


@pytest.mark.parametrize("path,value", [
    ("dtype", 3), ("dtype", -1), ("n_rows", -1), ("n_rows", 1 << 40), ("vocab", 0), ("vocab", -5), ("vocab", (1 << 30) + 1), ("row_stride", 999), ("row_stride", 0),
    ("top", -1), ("top", 33), ("top", 1 << 33), ("logits", None), ("tokens", None), ("logprob", None), ("entropy", None), ("top_logprob", None), ("top_token", None),
    ("logits", FAKE + 2), ("tokens", FAKE + 4), ("top_token", FAKE + 4), ("logprob", FAKE + 2), ("entropy", FAKE + 1), ("top_logprob", FAKE + 2),
])
def test_token_logprobs_refusals(path, value):
    a = _logprobs()
    _set(a, path, value)
    _refused(a)


def test_calls_without_work_need_no_pointers():
    """No tokens, no sequences or no rows: 0 without a launch."""
    p, k, g, lp = _prompt(), _append(), _paged(), _logprobs()
    for a in (p, k, g):
        a.n_tokens = a.batch = 0
    lp.n_rows = 0
    for r in (p.out, p.q, p.k, p.v, k.k, k.v, g.q, g.out):
        r.data = None
    lp.logits = lp.tokens = lp.logprob = lp.top_token = None
    for a in (p, k, g, lp):
        assert _call(a)[0] == 0
    for name in STRUCTS.values():
        from gptq_v2_amd import _lib
        assert getattr(_lib.load(), name)(None, None) == -1


def test_the_wrappers_want_gpu_tensors_and_tensors():
    from gptq_v2_amd import ops
    q, k = torch.zeros(4, 4, 64).half(), torch.zeros(4, 2, 64).half()
    cache = ops.PagedCache.empty(4, 2, 16, 64, "cpu")
    assert cache.k.shape == (4, 2, 16, 64) and cache.v.shape == (4, 2, 64, 16) and cache.k.dtype == torch.float8_e4m3fn
    table, lens = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    for call in (lambda: ops.attention_prompt(q, k, k), lambda: ops.kv_append(cache, k, k, table, lens), lambda: ops.attention_paged(q, cache, table, lens),
                 lambda: ops.token_logprobs(torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: ops.attention_prompt(q.numpy(), k, k), lambda: ops.kv_append(cache, None, k, table, lens), lambda: ops.attention_paged(None, cache, table, lens),
                 lambda: ops.token_logprobs([0.0], torch.zeros((), dtype=torch.int64)), lambda: ops._serving.attention_prompt(q, k)):
        with pytest.raises(TypeError):
            call()


def test_the_binding_belongs_to_the_library():
    """The binding refuses a library of another interface version; the one it was loaded with stays bound."""
    from gptq_v2_amd import _lib, ops
    with pytest.raises(ImportError, match="version"):
        ops._serving.bind(0, 0, 0, 0, 0, _lib.load().gq_version() + 1, _lib.check)
    ops._load_binding()

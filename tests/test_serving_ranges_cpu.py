"""The serving operators' requirements over the ranges they are made for, without a GPU: no call gets as far as a launch."""
import importlib.util
import os
import random

import pytest

from tests.conftest import ROOT
from tests.test_serving_cpu import _append, _call, _logprobs, _paged, _prompt, _refused, _set

CODES = {"f16": 0, "bf16": 1, "f32": 2}


def _cases():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _up_to_the_last(a, field, value):
    """The entry's last check of the arguments is the alignment of pointers: a call that ends there has passed the others."""
    _set(a, field, value)
    rc, name, lib = _call(a)
    assert rc == -1 and "aligned" in lib.gq_last_error().decode(), (name, rc, lib.gq_last_error())


def _as_struct(case):
    rows = lambda r, heads, d: (setattr(r, "token_stride", heads * d), setattr(r, "head_stride", d))   # noqa: E731
    op, code = case["op"], CODES[case["dtype"]]
    if op == "prompt":
        a, lens = _prompt(), [int(n) for n in case["lens"].split(",")]
        a.dtype, a.n_tokens, a.batch, a.n_heads, a.n_kv_heads, a.head_dim = code, sum(lens), len(lens), case["hq"], case["hkv"], case["d"]
        for r, h in ((a.out, case["hq"]), (a.q, case["hq"]), (a.k, case["hkv"]), (a.v, case["hkv"])):
            rows(r, h, case["d"])
        return a, "v.data"
    if op == "logprobs":
        a = _logprobs()
        a.dtype, a.n_rows, a.vocab, a.row_stride, a.top = code, case["rows"], case["vocab"], case["vocab"], case["top"]
        return a, "tokens"
    a = _append() if op == "append" else _paged()
    a.dtype, a.n_heads, a.batch, a.cu_seqlens = code, case["hq"], case["batch"], a.block_table
    a.cache.page, a.cache.head_dim, a.cache.n_kv_heads = case["page"], case["d"], case["hkv"]
    if op == "append":
        a.n_tokens, a.rotary_dim, a.interleaved = case["batch"] * case["new"], case["rot"], case["interleaved"]
        a.table_width = -(-(case["past"] + case["new"]) // case["page"])
        for r, h in ((a.k, case["hkv"]), (a.v, case["hkv"]), (a.q, case["hq"]), (a.q_out, case["hq"])):
            rows(r, h, case["d"])
        return a, "k.data"
    a.n_tokens, a.table_width = case["batch"] * case["nq"], -(-case["ctx"] // case["page"])
    for r in (a.out, a.q):
        rows(r, case["hq"], case["d"])
    return a, "q.data"


def test_every_drawn_case_is_taken():
    """Sizes, types, widths and strides of the measured cases and of thousands drawn from their ranges."""
    cases, rng = _cases(), random.Random(20)
    widths = set()
    for case in cases.listed() + [cases.draw(rng) for _ in range(4000)]:
        a, last = _as_struct(case)
        _up_to_the_last(a, last, (1 << 20) + 4)
        widths.add((case.get("d"), case.get("rot")))
    assert (80, 40) in widths


@pytest.mark.parametrize("head_dim,rotary_dim", [(80, 40), (80, 20), (96, 24), (64, 18), (128, 126), (32, 30), (128, 34)])
def test_even_rotary_widths_are_taken(head_dim, rotary_dim):
    a = _append()
    a.cache.head_dim, a.rotary_dim = head_dim, rotary_dim
    for r, heads in ((a.k, 2), (a.v, 2), (a.q, 4), (a.q_out, 4)):
        r.token_stride, r.head_stride = heads * head_dim, head_dim
    a.cos += 4   # a table's rows are no multiple of 16 bytes there
    _up_to_the_last(a, "sin", (1 << 20) + 2)


@pytest.mark.parametrize("rotary_dim", [1, 2, 14, 17, 63, 66])
def test_other_rotary_widths_are_refused(rotary_dim):
    a = _append()
    a.rotary_dim = rotary_dim
    _refused(a)

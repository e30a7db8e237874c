"""The package with and without the binding of the serving operators; no GPU."""
import importlib.util
import os
import subprocess
import sys

import pytest

from tests.conftest import ROOT


def _build_module():
    spec = importlib.util.spec_from_file_location("build_script", os.path.join(ROOT, "gptq_v2_amd", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_package_imports_without_the_binding():
    """Quantisation needs the library alone; a serving operator says what is missing and how to build it."""
    code = """
import sys
sys.modules["gptq_v2_amd._serving_binding"] = None    # an import of it fails
import torch, gptq_v2_amd as amd
assert amd.GPTQ and amd.QuantLinear and amd.ops.words_per_row(64, 4) > 0
for _ in range(2):
    try:
        amd.ops.token_logprobs(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int64))
    except ImportError as e:
        assert "gptq_v2_amd/build.py" in str(e) and "_serving_binding" in str(e), e
    else:
        raise AssertionError("no error")
"""
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


def test_the_binding_is_loaded_by_the_first_call():
    code = """
import sys, torch, gptq_v2_amd as amd
assert "gptq_v2_amd._serving_binding" not in sys.modules
try:
    amd.ops.token_logprobs(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int64))
except ValueError as e:
    assert "GPU" in str(e)
assert "gptq_v2_amd._serving_binding" in sys.modules and "attention_paged" in vars(amd.ops._serving)
"""
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


def test_the_binding_is_built_again_for_another_torch(tmp_path, monkeypatch):
    b = _build_module()
    monkeypatch.setattr(b, "BINDING", str(tmp_path / "binding.so"))
    monkeypatch.setattr(b, "STAMP", str(tmp_path / "stamp"))
    ran = []

    def run(cmd):
        ran.append(cmd)
        open(b.BINDING, "w").close()

    b._build_binding(False, run)
    b._build_binding(False, run)
    assert len(ran) == 1 and ran[0][0] == "g++"
    import torch
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    b._build_binding(False, run)
    b._build_binding(False, run)
    assert len(ran) == 2
    b._build_binding(True, run)
    os.remove(b.BINDING)
    b._build_binding(False, run)
    assert len(ran) == 4


def test_a_failing_binding_leaves_the_library(tmp_path, monkeypatch):
    """The library is linked before the binding's failure is raised."""
    b = _build_module()
    monkeypatch.setattr(b, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib" / "x.so"))
    monkeypatch.setattr(b, "_hipcc", lambda: "hipcc")
    ran = []
    monkeypatch.setattr(b.subprocess, "check_call", lambda cmd: ran.append(cmd))

    def fail(force, run):
        raise RuntimeError("no g++")

    monkeypatch.setattr(b, "_build_binding", fail)
    with pytest.raises(RuntimeError, match="no g"):
        b.build(force=True, verbose=False)
    assert ran[-1][-len(b.SOURCES) - 1] == b.LIB and len(ran) == len(b.SOURCES) + 1


def _wrappers():
    """Each operator as a function of its differentiable inputs (CPU tensors: the next check would refuse them)."""
    import torch
    from gptq_v2_amd import ops
    table, lens = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    cache = ops.PagedCache.empty(4, 2, 16, 64, "cpu")
    q, k, cos = torch.zeros(4, 4, 64).half(), torch.zeros(4, 2, 64).half(), torch.zeros(9, 32)
    return {
        "prompt q": (q, lambda x: ops.attention_prompt(x, k, k)), "prompt k": (k, lambda x: ops.attention_prompt(q, x, k)),
        "prompt v": (k, lambda x: ops.attention_prompt(q, k, x)), "append k": (k, lambda x: ops.kv_append(cache, x, k, table, lens)),
        "append q": (q, lambda x: ops.kv_append(cache, k, k, table, lens, q=x, cos=cos, sin=cos)),
        "append cos": (cos, lambda x: ops.kv_append(cache, k, k, table, lens, cos=x, sin=cos)),
        "append sin": (cos, lambda x: ops.kv_append(cache, k, k, table, lens, cos=cos, sin=x)),
        "paged q": (q, lambda x: ops.attention_paged(x, cache, table, lens)),
        "logits": (torch.zeros(4, 9), lambda x: ops.token_logprobs(x, torch.zeros(4, dtype=torch.int64))),
    }


@pytest.mark.parametrize("name", ["prompt q", "prompt k", "prompt v", "append k", "append q", "append cos", "append sin", "paged q", "logits"])
def test_tensors_that_carry_a_derivative_are_refused(name):
    import torch
    from torch.autograd import forward_ad
    x, call = _wrappers()[name]
    with pytest.raises(RuntimeError, match="no backward"):
        call(x.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        call(x.clone().requires_grad_())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward derivative"):
                call(dual)
        with pytest.raises(ValueError, match="GPU"):
            call(forward_ad.unpack_dual(dual).primal)

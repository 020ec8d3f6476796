"""The embedding encoder's operators and their build at the edges, without a GPU: what is refused and what is not."""
import ctypes

import pytest

from rag_service_amd import _lib
from test_encoder_refusals import NULL, ODD, P, attention, lib, norm, quantize, refused  # noqa: F401


# ---- attention: hints do not say what there is -----------------------------------------------------------------------

def test_packed_queries_are_there_whatever_the_hint_says(lib):  # noqa: F811
    """max_q = 0 with queries in the packed rows: there is work, so the arguments are looked at (it was taken for nothing to
    do, and the results left as they were)."""
    refused(lib, attention(lib, qo=P, total_q=4, max_q=0, q=NULL), _lib.RR_E_INVALID, "q is null")
    refused(lib, attention(lib, qo=P, total_q=4, max_q=0, out=ODD), _lib.RR_E_INVALID, "aligned")
    assert attention(lib, qo=P, total_q=0, max_q=7, q=NULL, out=NULL) == _lib.RR_OK
    # the workspace asked for with this hint is what the call wants
    need = lib.rr_cross_attention_workspace(1, 2, 2, 2, 16, 0, 4096)
    assert need == lib.rr_cross_attention_workspace(1, 2, 2, 2, 16, 1, 4096) > 0
    refused(lib, attention(lib, qo=P, total_q=4, max_q=0, max_k=4096, ks=(65536, 16, 16), vs=(65536, 16, 16)),
            _lib.RR_E_INVALID, "workspace")


def test_packed_keys_are_checked_whatever_the_hint_says(lib):  # noqa: F811
    """max_k = 0 with keys in the packed rows: the kernels read them, so null and misaligned keys are refused."""
    for change, word in (({"k": NULL}, "k is null"), ({"v": NULL}, "v is null"), ({"k": ODD}, "aligned")):
        refused(lib, attention(lib, ko=P, total_k=4, max_k=0, **change), _lib.RR_E_INVALID, word)


# ---- norm: gates -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("gate_rows,rows_per_gate", [(0, 2 ** 63 - 1), (0, 2 ** 63 - 3), (0, 4), (1, 3), (-1, 2 ** 63 - 1)])
def test_gate_rows_are_counted_without_overflow(lib, gate_rows, rows_per_gate):  # noqa: F811
    """A gate of too few rows for 4 rows, also where rows + rows_per_gate passes 2^63."""
    refused(lib, norm(lib, gate=P, gate_rows=gate_rows, rows_per_gate=rows_per_gate), _lib.RR_E_INVALID, "gate rows")


# ---- the build ---------------------------------------------------------------------------------------------------------

def test_every_object_follows_the_headers_it_includes():
    """A header that a unit includes, directly or through others, is a prerequisite of its object: make would rebuild it
    (asked without building: -n, the header taken as new)."""
    import os
    import re
    import subprocess
    csrc = os.path.join(_lib.PKG_ROOT, "csrc")
    where = [csrc, _lib.PKG_ROOT + "/../include"]                # (as the Makefile spells it)

    def headers(path, seen):
        for name in re.findall(r'^#include "([^"]+\.h)"', open(path).read(), flags=re.M):
            at = next((os.path.join(d, name) for d in where if os.path.exists(os.path.join(d, name))), None)
            if at and at not in seen:
                seen.add(at)
                headers(at, seen)
        return seen

    units = [f for f in sorted(os.listdir(csrc)) if f.endswith((".hip", ".cpp"))]
    assert len(units) >= 12
    needs = {f: headers(os.path.join(csrc, f), set()) for f in units}
    for header in sorted(set().union(*needs.values())):
        told = subprocess.run(["make", "-n", "-C", _lib.PKG_ROOT, "-W", header], capture_output=True, text=True).stdout
        for unit in (f for f in units if header in needs[f]):
            assert f"csrc/{unit}" in told, f"{unit} is not rebuilt when {os.path.basename(header)} changes"


@pytest.fixture
def fake_tree(tmp_path):
    """The Makefile and the sources in a folder of their own, and a compiler that only makes the file it is asked for."""
    import os
    import shutil
    import subprocess
    pkg = tmp_path / "pkg"
    pkg.mkdir()
    (pkg / "rag_service_amd").mkdir()
    shutil.copy(os.path.join(_lib.PKG_ROOT, "Makefile"), pkg / "Makefile")
    os.symlink(os.path.join(_lib.PKG_ROOT, "csrc"), pkg / "csrc")
    os.symlink(os.path.join(_lib.REPO_ROOT, "include"), tmp_path / "include")
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && touch "$2"; shift; done\n')
    cc.chmod(0o755)

    def make(python):
        return subprocess.run(["make", "-C", str(pkg), f"HIPCC={cc}", f"CXX={cc}", f"PYTHON={python}"], capture_output=True,
                              text=True)
    return pkg, make


def test_make_without_torch_builds_the_library(fake_tree):
    """The retriever needs no torch: where there is none, make builds the library, says what it leaves out and succeeds."""
    import sys
    pkg, make = fake_tree
    for none in (sys.executable + " -I -S", "/no/such/python"):
        r = make(none)
        assert r.returncode == 0, r.stdout + r.stderr
        assert (pkg / "librag_retrieval.so").exists() and not (pkg / "rag_service_amd" / "_torch_ops.so").exists()
        assert "torch" in r.stdout and "not built" in r.stdout
    r = make(sys.executable)
    assert r.returncode == 0 and (pkg / "rag_service_amd" / "_torch_ops.so").exists(), r.stdout + r.stderr


def test_build_makes_what_is_missing(tmp_path, monkeypatch):
    """build(): make runs if the library is missing, or the torch side where there is a torch; not if nothing is."""
    import importlib.util
    import subprocess
    ran = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: ran.append(cmd))
    lib_at, ops_at = tmp_path / "librag_retrieval.so", tmp_path / "_torch_ops.so"
    monkeypatch.setattr(_lib, "LIB_PATH", str(lib_at))
    monkeypatch.setattr(_lib, "TORCH_OPS_PATH", str(ops_at), raising=False)
    there = object()
    for have_lib, have_ops, torch, want in ((0, 0, there, 1), (1, 0, there, 1), (1, 1, there, 0), (0, 1, there, 1), (1, 0, None, 0),
                                            (0, 0, None, 1)):
        for p, have in ((lib_at, have_lib), (ops_at, have_ops)):
            p.touch() if have else p.unlink(missing_ok=True)
        monkeypatch.setattr(importlib.util, "find_spec", lambda name: torch)
        ran.clear()
        assert _lib.build() == str(lib_at)
        assert len(ran) == want, (have_lib, have_ops, torch)
    _lib.build(force=True)
    assert len(ran) == want + 1


# ---- the torch side: what it would drop ---------------------------------------------------------------------------------

def each_op(x):
    """Every operator on x, as calls."""
    import torch
    from rag_service_amd import ops
    n, k = x.shape
    w, s, q = torch.zeros(n, k, dtype=torch.int8), torch.ones(n), x.view(1, n, 1, k)
    return [lambda: ops.quantize_rows(x), lambda: ops.linear_int8(x, w, s), lambda: ops.block_norm(x),
            lambda: ops.cross_attention(q, q, q)]


def test_wrappers_refuse_what_they_would_drop():
    """A tangent, a recording, a bit that says the values are negated: none of them goes through these operators, so a tensor that
    has one is refused as one that asks for a gradient is (here the first operand, before its device is looked at)."""
    import torch
    import torch.autograd.forward_ad as fwd
    from rag_service_amd import ops
    x = torch.zeros(4, 8)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in each_op(dual):
            with pytest.raises(ValueError, match="forward"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward"):
                call()
        with pytest.raises(ValueError, match="GPU only"):            # its primal part is a tensor like any other
            ops.quantize_rows(fwd.unpack_dual(dual).primal)
    for call in each_op(torch._neg_view(x)):
        with pytest.raises(ValueError, match="negat"):
            call()
    for i in range(4):
        with pytest.raises(ValueError, match="trace"):
            torch.jit.trace(lambda t: each_op(t)[i](), x)
    from torch.fx.experimental.proxy_tensor import make_fx
    for i in range(4):
        with pytest.raises(ValueError, match="trace"):
            make_fx(lambda t: each_op(t)[i]())(x)


def test_inline_asm_of_the_encoder_units_is_hazard_free():
    """The audit of test_abi's test_inline_asm_loads_are_hazard_free (tools/check_asm_loads.py) on every kernel of the encoder's
    units: their inline-asm loads go to LDS, and nothing of the vector unit is written in inline asm."""
    import os
    import re
    import subprocess
    import sys
    pkg = _lib.PKG_ROOT
    sys.path.insert(0, os.path.join(_lib.REPO_ROOT, "tools"))
    from check_asm_loads import check
    csrc = os.path.join(pkg, "csrc")
    newest = max(os.path.getmtime(os.path.join(csrc, f)) for f in os.listdir(csrc) if f.startswith("rr_encoder"))
    with_loads = {"linear": 0, "norm": 0, "attn": 0}
    for unit in with_loads:
        s_file = os.path.join(pkg, "build", f"rr_encoder_{unit}-hip-amdgcn-amd-amdhsa-gfx950.s")
        if not os.path.exists(s_file) or os.path.getmtime(s_file) < newest:
            subprocess.check_call(["make", "-C", pkg, "-j8"], stdout=subprocess.DEVNULL)
        text = open(s_file).read()
        syms = re.findall(r"^(_ZN2rr3enc\w+kernel\w+):", text, flags=re.M)
        assert len(syms) >= 20, (unit, len(syms))
        lines = text.split("\n")
        for sym in syms:
            n_asm, bad = check(lines, sym)
            assert not bad, (sym, bad[:5])
            with_loads[unit] += n_asm > 0
    assert with_loads["norm"] == 0 and with_loads["linear"] >= 20 and with_loads["attn"] >= 10, with_loads

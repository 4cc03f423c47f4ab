"""The build recipe (CPU only, the compiler cross-compiles): a changed header makes the library stale, the entry point always compiles,
and packed FP32 arithmetic is left out -- checked in the recipe's commands and in the assembly of the one source with vectorisable
float code."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "osmo-tetra_amd")


def _recipe():
    spec = importlib.util.spec_from_file_location("tetra_build_recipe", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_every_hip_source_is_compiled_without_packed_fp32(tmp_path, monkeypatch):
    m = _recipe()
    monkeypatch.setattr(m, "OBJ", str(tmp_path))
    monkeypatch.setattr(m, "LIB", str(tmp_path / "lib.so"))
    cmds = []
    monkeypatch.setattr(m.subprocess, "check_call", lambda cmd: cmds.append(list(cmd)))
    m.build(force=True)
    hip = [c for c in cmds if any(a.endswith(".hip") for a in c)]
    assert len(hip) == len(m.HIP_SRCS)
    for c in hip:
        i = c.index("-packed-fp32-ops")
        assert c[i - 3:i] == ["-Xclang", "-target-feature", "-Xclang"], c


def test_float_front_end_has_no_packed_fp32(tmp_path):
    m = _recipe()
    hipcc = shutil.which("hipcc") or os.path.join(m.ROCM, "bin", "hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc here")
    out = str(tmp_path / "front.s")
    subprocess.check_call([hipcc] + m.HIP_FLAGS + ["-I" + os.path.join(ROOT, "include"), "-I" + m.CSRC, "--cuda-device-only", "-S",
                                                   os.path.join(m.CSRC, "tg_k_front.hip"), "-o", out], stderr=subprocess.DEVNULL)
    text = open(out).read()
    assert "k_float_to_bits" in text
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32.*", text)


def test_every_included_header_makes_the_library_stale():
    m = _recipe()
    named = {os.path.basename(h) for h in m.HEADERS}
    for f in os.listdir(m.CSRC):
        for inc in re.findall(r'^#include "(.*?)"', open(os.path.join(m.CSRC, f)).read(), re.M):
            assert inc in named, (f, inc)


def test_entry_point_compiles_also_where_a_library_is_built(monkeypatch):
    import __graft_entry__ as g
    import osmo_tetra_amd as T
    asked = []
    monkeypatch.setattr(T, "build_library", lambda **kw: asked.append(kw))
    monkeypatch.setattr(g.subprocess, "check_call", lambda *a, **kw: 0)
    monkeypatch.setattr(g, "_check_adapter", lambda: None)
    T.lib()
    g.build()
    assert asked == [{"force": True}]

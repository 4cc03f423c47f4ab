"""Rules on the sources themselves (CPU only): GPU code writes memory through vector stores.  A store, an atomic or a write-back
through the scalar data cache appears in no source, script or build file, comments included; documents may record that it was
measured once and rejected."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIRS = ["include", "oracle", "osmo-tetra_amd", "tests", "tools"]
TEXT = (".hip", ".h", ".c", ".cpp", ".s", ".py", ".sh")

SCALAR_CACHE_WRITE = re.compile(r"(?:\b|amdgcn_)s_(?:(?:buffer_|scratch_)?store_|(?:buffer_)?atomic_|dcache_(?:wb|discard))", re.I)


def _sources():
    for f in sorted(os.listdir(ROOT)):
        if f.endswith(TEXT):
            yield f
    for top in DIRS:
        for d, sub, files in os.walk(os.path.join(ROOT, top)):
            sub[:] = sorted(s for s in sub if s not in ("build", "__pycache__", "_ref"))
            for f in sorted(files):
                if f.endswith(TEXT) or f == "Makefile":
                    yield os.path.relpath(os.path.join(d, f), ROOT)


@pytest.mark.parametrize("line", ["s_store_dwordx4 s[0:3], s[4:5], 0", "S_STORE_DWORD", "s_buffer_store_dword", "s_scratch_store_dword",
                                  "s_atomic_add", "s_buffer_atomic_swap", "s_dcache_wb", "s_dcache_wb_vol", "s_dcache_discard_x2",
                                  "__builtin_amdgcn_s_dcache_wb()"])
def test_pattern_finds(line):
    assert SCALAR_CACHE_WRITE.search(line)


@pytest.mark.parametrize("line", ["s_load_dwordx4", "s_dcache_inv", "global_store_dwordx4", "global_atomic_add", "buffer_store_dword",
                                  "cls_store_x", "reads_atomic_counter"])
def test_pattern_passes(line):
    assert not SCALAR_CACHE_WRITE.search(line)


def test_no_writes_through_the_scalar_cache():
    bad, seen = [], 0
    for rel in _sources():
        if rel == os.path.join("tests", os.path.basename(__file__)):
            continue
        seen += 1
        with open(os.path.join(ROOT, rel), encoding="utf-8", errors="replace") as fh:
            bad += ["%s:%d" % (rel, i) for i, ln in enumerate(fh, 1) if SCALAR_CACHE_WRITE.search(ln)]
    assert seen > 50, seen
    assert not bad, bad

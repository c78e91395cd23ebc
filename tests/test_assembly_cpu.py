"""Distances between instructions that the ISA asks of software, where inline assembly leaves them to this repository."""
from __future__ import annotations

import os
import re
import shutil

import pytest

from conftest import dpa_mod
from gfx950_assembly import assembly_of, kernels_of, m0_too_close

has_hipcc = pytest.mark.skipif(not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="no hipcc")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    made = {}

    def get(source):
        if source not in made:
            made[source] = kernels_of(assembly_of(source, tmp_path_factory.mktemp("assembly")))
        return made[source]
    return get


def test_the_check_of_m0_finds_what_is_too_close():
    text = """_Zk:
	s_mov_b32 m0, s1
	s_cbranch_scc1 .LBB0_2
	s_nop 0
.LBB0_2:
	global_load_lds_dwordx4 v[0:1], off
	s_mov_b32 m0, s2
	global_load_lds_dwordx4 v[0:1], off
	s_endpgm
.Lfunc_end0:
"""
    assert len(m0_too_close(kernels_of(text)["_Zk"])) == 1
    assert not m0_too_close(kernels_of(text.replace("s2", "s2\n\ts_nop 0"))["_Zk"])


def test_every_load_to_lds_waits_for_m0_in_the_sources():
    asm = 0
    for path in sorted(dpa_mod("build").CSRC_DIR.iterdir()):
        if path.suffix not in (".hip", ".hpp"):
            continue
        for n, line in enumerate(path.read_text().splitlines(), 1):
            if re.search(r"_load_lds_\w+ %", line):
                asm += 1
                assert re.search(r"m0, %\d\\n\\ts_nop 0\\n\\t\w+_load_lds_", line), f"{path.name}:{n}: {line}"
    assert asm >= 6


@has_hipcc
@pytest.mark.parametrize("source", ["igemm", "mxfp4_gemm"])
def test_loads_to_lds_wait_for_m0(kernels, source):
    loads = 0
    for name, kernel in kernels(source).items():
        loads += sum(c.to_lds for c in kernel.code)
        assert not (bad := m0_too_close(kernel)), f"{name}: {bad[0]} (of {len(bad)})"
    assert loads > 100

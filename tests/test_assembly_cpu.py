"""Distances between instructions that the ISA asks of software, where inline assembly leaves them to this repository."""
from __future__ import annotations

import os
import re
import shutil

import pytest

from conftest import dpa_mod
from gfx950_assembly import assembly_of, kernels_of, m0_too_close, products_too_close

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


def test_the_check_of_products_finds_what_is_too_close():
    text = """_Zk:
	v_mov_b32_e32 v4, 0
	s_cbranch_scc1 .LBB0_2
	s_nop 1
.LBB0_2:
	v_mfma_scale_f32_16x16x128_f8f6f4 v[2:5], v[6:9], v[10:13], v[2:5], v1, v80 cbsz:4 blgp:4
	s_nop 9
	v_add_f32_e32 v7, v2, v3
	s_endpgm
.Lfunc_end0:
"""
    bad = products_too_close(kernels_of(text)["_Zk"])
    assert len(bad) == 2 and "v_mov" in bad[0] and "v_add" in bad[1]
    text = text.replace("s_nop 9", "s_nop 15").replace("s_cbranch_scc1 .LBB0_2", "s_nop 0")
    assert not products_too_close(kernels_of(text)["_Zk"])


@has_hipcc
def test_matrix_instructions_of_the_product_keep_their_distance(kernels):
    """They are inline assembly, to whose operands the compiler keeps no distance."""
    found = {n: k for n, k in kernels("mxfp4_gemm").items() if "mxfp4_gemm_kernel" in n}
    assert len(found) >= 13 and all(any(c.matrix for c in k.code) for k in found.values())
    bad = {n: lines for n, k in found.items() if (lines := products_too_close(k))}
    assert not bad, "\n".join(f"{n}: {lines[0]} (of {len(lines)})" for n, lines in bad.items())

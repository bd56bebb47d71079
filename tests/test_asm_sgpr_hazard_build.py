"""The SGPR hazard scan over what the build compiles: its own flags, and every source that issues LDS-DMA from inline asm.

A vector memory instruction that takes an SGPR pair as its base needs five wait states behind a vector instruction that wrote the pair
(v_readlane, v_readfirstlane), and an LDS-DMA one behind the write of M0 that it reads; hipcc does not pad that inside an asm string."""
import os
import re
import subprocess

import pytest

from block_transformer_amd import build
from test_asm_sgpr_hazard import HIPCC, _scan


SOURCES = [s for s in build.SOURCES if "global_load_lds_dwordx4" in open(os.path.join(build.CSRC, s)).read()]


@pytest.fixture(scope="module", params=SOURCES)
def kernels(request, tmp_path_factory):
    """(source, {kernel: its instructions})"""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "out.s"
    subprocess.run([HIPCC] + build.FLAGS + ["--cuda-device-only", "-S", "-o", str(out), os.path.join(build.CSRC, request.param)],
                   check=True, capture_output=True, timeout=900)
    found = {}
    for body in re.split(r"\n(?=_ZN2bt\S+:)", out.read_text())[1:]:
        if "s_endpgm" in body:
            found[body[:body.index(":")]] = body[:body.rindex("s_endpgm")]
    return request.param, found


def test_no_valu_written_sgpr_base_within_five_wait_states(kernels):
    source, found = kernels
    seen = 0
    for name, body in found.items():
        total, hazards = _scan(body)
        assert not hazards, (name, hazards[:3])
        seen += total >= 8
    assert seen >= {"gemm.hip": 12, "quant.hip": 8}.get(source, 1), (source, seen)      # it really found the kernels and their loads


def test_no_packed_fp32_arithmetic(kernels):
    for name, body in kernels[1].items():
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", body), name


def test_no_dma_right_behind_its_m0(kernels):
    for name, body in kernels[1].items():
        ins = [l.strip() for l in body.split("\n")]
        ins = [l for l in ins if l and not l.startswith((";", ".")) and not l.endswith(":")]
        for before, dma in zip(ins, ins[1:]):
            assert not (" lds" in dma or "load_lds" in dma) or not re.match(r"s_\w+ m0,", before), (name, before, dma)

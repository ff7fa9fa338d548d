"""CPU check that the kernels' inline assembly has the wait states that the hardware leaves to software (tests/wait_states.py), in the
assembly that the library's build flags give.  A missing one is a stale address now and then, which no run has to show."""
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess

import pytest

from tests.wait_states import missing
from transformer_amd import build as B

SOURCES = sorted(os.path.basename(s) for s in glob.glob(os.path.join(B.CSRC, "*.hip")))


def assembly(src):
    cmd = [B.HIPCC, *B.FLAGS, *B.FILE_FLAGS.get(src, []), "--offload-device-only", "-S", os.path.join(B.CSRC, src), "-o", "-"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


@pytest.fixture(scope="module")
def assemblies():
    with cf.ThreadPoolExecutor(max_workers=8) as ex:
        return dict(zip(SOURCES, ex.map(assembly, SOURCES)))


@pytest.mark.skipif(not shutil.which(B.HIPCC) and not os.path.exists(B.HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src", SOURCES)
def test_no_wait_state_is_missing(assemblies, src):
    found = missing(assemblies[src])
    assert not found, f"{src}: {len(found)} places, the first: {found[:3]}"


LOAD = ";;#ASMSTART\n\ts_mov_b32 m0, s9\n{nop}\tbuffer_load_dwordx4 v1, s[4:7], 0 offen lds\n;;#ASMEND\n"
MFMA = "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[32:47]\n"
MAX = ";;#ASMSTART\n\tv_max3_f32 {to}, {a}, v61, v62\n;;#ASMEND\n"


def kernel(*lines):
    return "kernel:\n" + "".join(lines) + "\ts_endpgm\n.Lfunc_end0:\n"


@pytest.mark.parametrize("lines,places", [
    # a descriptor from vector instructions: 5 wait states, M0: 1
    (("\tv_readlane_b32 s4, v3, 0\n", LOAD.format(nop="")), 2),
    (("\tv_readlane_b32 s4, v3, 0\n", LOAD.format(nop="\ts_nop 0\n")), 1),
    (("\tv_readlane_b32 s4, v3, 0\n", LOAD.format(nop="\ts_nop 2\n")), 1),
    (("\tv_readlane_b32 s4, v3, 0\n", LOAD.format(nop="\ts_nop 3\n")), 0),
    (("\tv_readlane_b32 s4, v3, 0\n", "\ts_nop 4\n", LOAD.format(nop="\ts_nop 0\n")), 0),
    (("\tv_readfirstlane_b32 s10, v3\n", LOAD.format(nop="\ts_nop 0\n")), 0),
    # a scalar instruction writes it anew
    (("\tv_readlane_b32 s4, v3, 0\n", "\ts_mov_b32 s4, s11\n", LOAD.format(nop="\ts_nop 0\n")), 0),
    # along a branch, and around a loop
    (("\tv_readlane_b32 s7, v3, 0\n", "\ts_cbranch_scc1 .LBB0_2\n", "\ts_nop 7\n", ".LBB0_2:\n", LOAD.format(nop="\ts_nop 0\n")), 1),
    (("\ts_nop 0\n", ".LBB0_1:\n", LOAD.format(nop="\ts_nop 0\n"), "\tv_readlane_b32 s5, v3, 0\n", "\ts_cbranch_vccnz .LBB0_1\n"), 1),
    (("\tv_cmp_lt_i32_e64 s[6:7], v0, v1\n", "\tglobal_load_dword v0, v1, s[6:7]\n"), 1),
    # results of matrix instructions in inline assembly
    ((MFMA, MAX.format(to="v60", a="v3")), 1),
    ((MFMA, "\ts_nop 10\n", MAX.format(to="v60", a="v3")), 1),
    ((MFMA, "\ts_nop 11\n", MAX.format(to="v60", a="v3")), 0),
    ((MFMA, MAX.format(to="v15", a="v60")), 1),
    ((MFMA, MAX.format(to="v40", a="v60")), 1),
    ((MFMA, "\ts_nop 7\n", MAX.format(to="v40", a="v60")), 0),
    ((MFMA, MAX.format(to="v60", a="v17")), 0),
    ((MFMA, "\tv_add_f32_e32 v3, v3, v3\n", MAX.format(to="v60", a="v3")), 0),
])
def test_what_is_looked_for(lines, places):
    assert len(missing(kernel(*lines))) == places

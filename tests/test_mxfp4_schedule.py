"""The MXFP4 tile kernel's waits against the order of its loads, stores and LDS reads (no GPU): tests/mxfp4_schedule.cpp
replays them with the kernel's own counts for every tile shape and ring, one to five slabs and tiles, and the generated
code has to hold the wait that tiles of one slab need."""
import os
import re
import shutil
import subprocess

import pytest
from test_codegen import CSRC, FLAGS, HIPCC

HERE = os.path.dirname(os.path.abspath(__file__))
# units of 64 rows and columns a tile, slabs of its ring, template arguments of the kernel that runs it
SHAPES = [(4, 4, 2, "4ELi4ELi1E"), (1, 4, 3, "4ELi4ELi1E"), (2, 4, 2, "2ELi4ELi0E"), (2, 3, 3, "2ELi3ELi0E"),
          (2, 2, 4, "2ELi2ELi0E"), (1, 2, 4, "1ELi2ELi0E")]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("schedule") / "schedule")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", out,
                    os.path.join(HERE, "mxfp4_schedule.cpp")], check=True, timeout=300)
    return out


def test_reads_lie_behind_their_loads(program):
    r = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(r.stdout.split()[-1]) > 500


def test_single_slab_wait_in_the_generated_code(program, tmp_path):
    """Kernels whose ring has more than two slabs wait for the bias and gate before the epilogue: the count, then a barrier."""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    asm = str(tmp_path / "gemm.s")
    subprocess.run([HIPCC, *FLAGS, "-o", asm, os.path.join(CSRC, "mxfp4_gemm.hip")], check=True, capture_output=True,
                   timeout=900)
    with open(asm) as f:
        text = f.read()
    for fm, fn, ring, args in SHAPES:
        for epi in range(4):
            count = int(subprocess.run([program, str(fm), str(fn), str(ring), str(int(epi == 3))], check=True,
                                       capture_output=True, text=True).stdout)
            assert (count < 0) == (ring == 2)
            names = re.findall(rf"^(_ZN\S*mxfp4_gemm_tilesILb[01]ELi{epi}ELi{args}\S*):", text, re.M)
            assert len(names) == 2, (args, epi)
            for name in names:
                body = text[text.index("\n" + name + ":"):]
                body = body[: body.index(".Lfunc_end")]
                if count >= 0:
                    assert re.search(rf"s_waitcnt vmcnt\({count}\)\n(\s*;.*\n)*\s*s_barrier", body), (name, count)

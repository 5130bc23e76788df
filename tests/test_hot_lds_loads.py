"""Loads straight into LDS of the kernels on hot pages (compiled here, no GPU).

Such a load takes its LDS address from m0, and needs a wait state behind the
instruction that writes m0: without one it may still see the previous load's
address.  Inside an asm statement the compiler neither adds the wait state nor
knows that m0 is overwritten, so the compiled code must show both: something
between the write and the load, and no other use of m0.  Nor does it know that
a load inside asm reads a scalar base, which needs five wait states behind a
vector instruction (v_readfirstlane) that wrote it, whatever the compiler puts
in front of the asm; behind a scalar instruction, which waits for a vector
instruction's result by itself, it needs none.
"""
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "vlx-tee_amd"))
import build as B  # noqa: E402  (vlx-tee_amd/build.py: the library's compiler flags)

HIPCC = shutil.which("hipcc") or ("/opt/rocm/bin/hipcc" if Path("/opt/rocm/bin/hipcc").exists() else None)
pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
SOURCES = ("ztcp_attention", "ztcp_mass")


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    d = tmp_path_factory.mktemp("asm")

    def compile_one(name):
        out = d / (name + ".s")
        cmd = [HIPCC, *B.HIPCC_FLAGS, "--cuda-device-only", "-S", "-I", str(ROOT / "include"),
               str(ROOT / "vlx-tee_amd" / "csrc" / (name + ".hip")), "-o", str(out)]
        subprocess.run(cmd, check=True, capture_output=True)
        lines = (re.split(r"[;/]{1,2}", x, maxsplit=1)[0].strip() for x in out.read_text().splitlines())
        return [x for x in lines if x and not x.startswith(".")]

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        return dict(zip(SOURCES, pool.map(compile_one, SOURCES)))


@pytest.mark.parametrize("name", SOURCES)
def test_a_load_waits_for_its_address(listings, name):
    lines = listings[name]
    loads = [i for i, x in enumerate(lines) if x.startswith("global_load_lds")]
    assert loads
    for i in loads:
        assert lines[i - 2].startswith("s_mov_b32 m0,") and re.match(r"s_nop|s_mov_b64", lines[i - 1]), lines[i - 3:i + 1]


@pytest.mark.parametrize("name", SOURCES)
def test_nothing_else_uses_m0(listings, name):
    lines = listings[name]
    writes = [i for i, x in enumerate(lines) if re.search(r"\bm0\b", x)]
    loads = [i for i, x in enumerate(lines) if x.startswith("global_load_lds")]
    assert loads and len(writes) == len(loads)
    assert all(lines[i].startswith("s_mov_b32 m0,") for i in writes)


@pytest.mark.parametrize("name", SOURCES)
def test_a_load_waits_for_its_scalar_base(listings, name):
    lines = listings[name]
    bases = {i: m[1] for i, x in enumerate(lines) if (m := re.match(r"global_load_lds\S*\s+v\S+,\s*(s\[\S+\])", x))}
    assert bases
    for i, base in bases.items():
        assert re.match(r"s_mov_b64 " + re.escape(base) + ",", lines[i - 1]), lines[i - 2:i + 1]

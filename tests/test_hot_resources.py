"""Register and scratch budget of the kernels on hot pages (compiled here, no GPU).

The append, decoding and eviction kernels keep all they work on in registers.
Of the kernels for chunks those for vectors of more than 64 elements fill a
wave's registers; what they keep in scratch memory is written before their loop
over tiles, read back a few words at a time, and stays small.
"""
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

from test_kernel_resources import _kernels

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "vlx-tee_amd"))
import build as B  # noqa: E402  (vlx-tee_amd/build.py: the library's compiler flags)

HIPCC = shutil.which("hipcc") or ("/opt/rocm/bin/hipcc" if Path("/opt/rocm/bin/hipcc").exists() else None)
pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")

# kernel name fragment -> registers a wave may use (512 / waves per SIMD), bytes of scratch
BUDGET = {
    "13append_kernelILi0ELi16E": (128, 0), "13append_kernelILi1ELi64ELi2E": (128, 0),
    "10few_kernelILi1ELi64ELi1E": (168, 0), "10few_kernelILi1ELi128ELi1E": (256, 0),
    "10few_kernelILi1ELi128ELi2E": (512, 0), "10few_kernelILi1ELi256ELi1E": (512, 0),
    "11many_kernelILi1ELi64E": (256, 0), "11many_kernelILi1ELi128E": (256, 160), "11many_kernelILi1ELi256E": (512, 256),
    "15join_few_kernel": (128, 0), "16join_many_kernel": (128, 0),
    "15mass_few_kernelILi1ELi64E": (168, 0), "15mass_few_kernelILi1ELi128E": (256, 0),
    "15mass_few_kernelILi1ELi256ELi1E": (256, 0),
    "16mass_many_kernelILi1ELi64E": (256, 0), "16mass_many_kernelILi1ELi128E": (256, 64),
    "16mass_many_kernelILi1ELi256E": (512, 0),
    "12evict_kernelILi256E": (128, 0), "12evict_kernelILi1024E": (128, 0),
}


@pytest.fixture(scope="module")
def metadata(tmp_path_factory):
    d = tmp_path_factory.mktemp("asm")

    def compile_one(name):
        out = d / (name + ".s")
        cmd = [HIPCC, *B.HIPCC_FLAGS, "--cuda-device-only", "-S", "-I", str(ROOT / "include"),
               str(ROOT / "vlx-tee_amd" / "csrc" / (name + ".hip")), "-o", str(out)]
        subprocess.run(cmd, check=True, capture_output=True)
        return _kernels(out.read_text())

    with ThreadPoolExecutor(4) as pool:
        parts = list(pool.map(compile_one, ["ztcp_append", "ztcp_attention", "ztcp_mass", "ztcp_evict"]))
    return {k: v for p in parts for k, v in p.items()}


@pytest.mark.parametrize("frag", sorted(BUDGET))
def test_registers_and_scratch_fit(metadata, frag):
    hits = {n: m for n, m in metadata.items() if frag in n}
    assert hits, frag
    registers, scratch = BUDGET[frag]
    for name, m in hits.items():
        assert m["private_segment_fixed_size"] <= scratch, (name, m)
        assert m["vgpr_count"] <= registers, (name, m)   # both kinds of registers


# registers that the chunk kernels spill: kernel<dtype, head_dim, whole tiles, drafted trees>
SPILLS = {"11many_kernelILi%dELi64ELb0ELb0E": 0, "11many_kernelILi%dELi64ELb1ELb0E": 0, "11many_kernelILi%dELi128ELb0ELb0E": 30,
          "11many_kernelILi%dELi128ELb1ELb0E": 19, "11many_kernelILi%dELi256ELb0ELb0E": 70, "11many_kernelILi%dELi256ELb1ELb0E": 40}


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("frag", sorted(SPILLS))
def test_chunk_kernels_spill_no_more(metadata, frag, dtype):
    """Scratch that spills share does not tell their number: reads of it in a chunk's loop are time."""
    hits = [m for n, m in metadata.items() if frag % dtype in n]
    assert len(hits) == 1 and hits[0]["vgpr_spill_count"] <= SPILLS[frag], hits


def test_only_kernels_that_are_launched(metadata):
    """Contexts' pieces of drafted trees have a join of their own."""
    assert not any("join_tree_kernel" in n for n in metadata)

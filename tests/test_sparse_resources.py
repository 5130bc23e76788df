"""Register and scratch budget, and loads straight to LDS, of the kernels for page tables, drafted trees and selected pages
(compiled here, no GPU).

Kernels that work in passing (tables, bounds, selection) keep all in registers.  The tree's are the chunk kernels of paged
attention with a mask; the block kernel of selected pages runs at the registers that let two workgroups share a compute unit, and
keeps a few words in scratch memory for it.  What a load straight to LDS needs around it is said in test_hot_lds_loads.py."""
import re
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
LDS_LOADS = ("ztcp_tree", "ztcp_selected")

# kernel name fragment -> registers a wave may use (512 / waves per SIMD), bytes of scratch
BUDGET = {
    "11plan_kernelILi256E": (128, 0), "11plan_kernelILi1024E": (128, 0), "11rows_kernel": (128, 0),
    "20release_count_kernel": (128, 0), "14release_kernel": (128, 0), "18release_sum_kernel": (128, 0),
    "13bounds_kernel": (128, 0), "12score_kernelILi1ELi64E": (128, 0), "12score_kernelILi1ELi128E": (168, 0),
    "12score_kernelILi1ELi256E": (512, 0), "18score_chunk_kernelILi1ELi64E": (128, 0), "18score_chunk_kernelILi1ELi128E": (168, 0),
    "18score_chunk_kernelILi1ELi256E": (512, 0), "15pick_few_kernel": (128, 0), "11pick_kernelILi1ELi1024E": (128, 0),
    "11pick_kernelILi1ELi256E": (128, 0),
    "10few_kernelILi1ELi128ELi1ELb1E": (256, 0), "10few_kernelILi1ELi256ELi1ELb1E": (512, 0),
    "11many_kernelILi1ELi64ELb1ELb1E": (256, 0), "11many_kernelILi1ELi128ELb1ELb1E": (256, 160),
    "11many_kernelILi1ELi256ELb1ELb1E": (512, 256),
    "15selected_kernelILi1ELi64E": (168, 0), "15selected_kernelILi1ELi128E": (256, 0), "15selected_kernelILi1ELi256E": (512, 0),
    "12block_kernelILi1ELi64ELb1ELi1E": (128, 0), "12block_kernelILi1ELi128E": (128, 160), "12block_kernelILi1ELi256E": (256, 0),
    "20join_selected_kernel": (128, 0), "16join_tree_kernel": (128, 0),
}


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    d = tmp_path_factory.mktemp("asm")

    def compile_one(name):
        out = d / (name + ".s")
        subprocess.run([HIPCC, *B.HIPCC_FLAGS, "--cuda-device-only", "-S", "-I", str(ROOT / "include"),
                        str(ROOT / "vlx-tee_amd" / "csrc" / (name + ".hip")), "-o", str(out)], check=True, capture_output=True)
        return out.read_text()

    names = ["ztcp_tables", "ztcp_select", *LDS_LOADS]
    with ThreadPoolExecutor(4) as pool:
        return dict(zip(names, pool.map(compile_one, names)))


@pytest.mark.parametrize("frag", sorted(BUDGET))
def test_registers_and_scratch_fit(listings, frag):
    hits = {n: m for text in listings.values() for n, m in _kernels(text).items() if frag in n}
    assert hits, frag
    registers, scratch = BUDGET[frag]
    for name, m in hits.items():
        assert m["private_segment_fixed_size"] <= scratch, (name, m)
        assert m["vgpr_count"] <= registers, (name, m)   # both kinds of registers


@pytest.mark.parametrize("name", LDS_LOADS)
def test_loads_to_lds_wait_for_their_address_and_base(listings, name):
    lines = (re.split(r"[;/]{1,2}", x, maxsplit=1)[0].strip() for x in listings[name].splitlines())
    lines = [x for x in lines if x and not x.startswith(".")]
    loads = [i for i, x in enumerate(lines) if x.startswith("global_load_lds")]
    writes = [i for i, x in enumerate(lines) if re.search(r"\bm0\b", x)]
    assert loads and len(writes) == len(loads) and all(lines[i].startswith("s_mov_b32 m0,") for i in writes)
    for i in loads:
        assert lines[i - 2].startswith("s_mov_b32 m0,") and re.match(r"s_nop|s_mov_b64", lines[i - 1]), lines[i - 3:i + 1]
        base = re.match(r"global_load_lds\S*\s+v\S+,\s*(s\[\S+\])", lines[i])
        assert not base or re.match(r"s_mov_b64 " + re.escape(base[1]) + ",", lines[i - 1]), lines[i - 2:i + 1]


def test_only_kernels_that_are_launched(listings):
    """Chunks' pieces of paged attention have a join of their own."""
    assert not any("join_many_kernel" in n for n in _kernels(listings["ztcp_tree"]))

"""Into what pieces attention of drafted trees cuts contexts: the host's copy of the function that the kernels call, over work
of any size (no GPU).  A piece is a multiple of 128 tokens, no context has more pieces than there is room for, and a piece is
never longer than the longest context needs."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "vlx-tee_amd"))
import build as B  # noqa: E402  (vlx-tee_amd/build.py: the library's compiler flags)

HIPCC = shutil.which("hipcc") or ("/opt/rocm/bin/hipcc" if Path("/opt/rocm/bin/hipcc").exists() else None)
pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")

CHECK = """
#include "{header}"
constexpr bool holds(int64_t work, int resident, int longest, int splits) {{
    const int64_t n = tree_piece_tokens(work, resident, longest, splits);
    return n > 0 && n % 128 == 0 && n < longest + 128ll && (longest + n - 1) / n <= splits;
}}
constexpr bool all_hold(int resident) {{
    for (int splits : {{2, 7, 8, 64}})
        for (int64_t longest = 1; longest <= (1ll << 31) - 1024; longest = longest * 3 + 5)
            for (int bits = 0; bits < 62; ++bits)
                for (int64_t work : {{1ll << bits, (1ll << bits) / 3 * 2 + 1, -(1ll << bits)}})
                    if (!holds(work, resident, (int)longest, splits)) return false;
    return holds(1ll << 47, resident, 2147482624, 8);
}}
static_assert(all_hold(512) && all_hold(256));
"""


def test_pieces_of_any_amount_of_work(tmp_path):
    src = tmp_path / "pieces.hip"
    src.write_text(CHECK.format(header=ROOT / "vlx-tee_amd" / "csrc" / "ztcp_attend.h"))
    got = subprocess.run([HIPCC, *B.HIPCC_FLAGS, "--cuda-host-only", "-fsyntax-only", "-fconstexpr-steps=100000000", str(src)],
                         capture_output=True, text=True)
    assert got.returncode == 0, got.stderr[-3000:]

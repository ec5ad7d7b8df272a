"""No two CTAs that fit on one SM ask for more tensor memory than it has. An allocation that waits for another kernel's
columns can wait for good: two kernels on two streams, met on several SMs, may each hold what the other's cluster waits for.
The products' shared memory and columns are read from the header that the kernels are built from. No GPU needed."""
from __future__ import annotations

import re
import shutil
import subprocess
from itertools import combinations_with_replacement
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "kernelopt_b200" / "csrc"
PER_SM, PER_CTA, COLUMNS = 228 * 1024, 1024, 512   # shared memory of an SM, the system's share of a CTA, tensor memory

PROGRAM = """
#include <cstdio>
#include "ko_mx_cfg.h"
template <bool F4, int BN> void slice() {
  std::printf("slice_%s_%d %u %u\\n", F4 ? "f4" : "f8", BN, komx::SliceCfg<F4, BN>::kSmem, komx::SliceCfg<F4, BN>::kCols);
}
template <bool F4> void forms() {
  slice<F4, 16>(); slice<F4, 32>(); slice<F4, 64>(); slice<F4, 128>();
  std::printf("pair_%s_128 %u 512\\n", F4 ? "f4" : "f8", komx::PairCfg<F4, 128>::kSmem);
  std::printf("pair_%s_256 %u 512\\n", F4 ? "f4" : "f8", komx::PairCfg<F4, 256>::kSmem);
}
int main() { forms<true>(); forms<false>(); }
"""


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    cxx = shutil.which("g++") or pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("residency")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", f"-I{CSRC}", str(d / "p.cpp"), "-o", str(d / "p")], check=True)
    lines = subprocess.run([str(d / "p")], check=True, capture_output=True, text=True).stdout.split("\n")
    found = {n: (int(s), int(c)) for n, s, c in (line.split() for line in lines if line)}
    # the fp32-grade kernels: what the attention at head dim 32 and every GEMM have at least
    floor = 120 * 1024
    found["attention"] = found["gemm"] = (floor, COLUMNS)
    return found


def test_ctas_that_share_an_sm_share_its_tensor_memory(forms):
    assert len(forms) == 14
    for n in (2, 3):
        for group in combinations_with_replacement(sorted(forms), n):
            if sum(forms[g][0] + PER_CTA for g in group) <= PER_SM:
                assert sum(forms[g][1] for g in group) <= COLUMNS, group
    # the slices are made to share an SM with each other
    for a, b in combinations_with_replacement([f for f in forms if f.startswith("slice")], 2):
        assert forms[a][0] + forms[b][0] + 2 * PER_CTA <= PER_SM, (a, b)


def test_the_fp32_kernels_keep_their_floor():
    """The floor that the test above takes for the attention and the GEMM is the one that they are built with."""
    assert re.search(r"kWholeTmemSmem = 120 \* 1024;", (CSRC / "ko_residency.h").read_text())
    for name, use in (("ko_attention.cu", "kSmemNeed > ko::kWholeTmemSmem ? kSmemNeed : ko::kWholeTmemSmem;"),
                      ("ko_gemm.cu", "static_assert(kSmemBytes >= ko::kWholeTmemSmem")):
        assert use in (CSRC / name).read_text(), name

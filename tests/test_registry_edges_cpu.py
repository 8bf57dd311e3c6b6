"""The quantised registry at the ends of what its calls allow, as far as that goes without a
GPU."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "voice-detect.cpp_b200" / "csrc"

BATCHES = r"""
#include "batches.h"
#include <climits>
#include <cstdio>

int main() {
    const int totals[] = {0, 1, 127, 128, 129, 65535, 65536, 65537, 200000, INT_MAX - 65536,
                          INT_MAX - 65535, INT_MAX - 65534, INT_MAX - 254, INT_MAX - 1, INT_MAX};
    for (const int size : {128, 65408, 65536})
        for (const int total : totals) {
            vdb::Batches b{total, size};
            long long done = 0;
            int a, c;
            for (int first, n; b.next(first, n);) {
                if (first != done || n <= 0 || n > size || (n < size && done + n != total)) {
                    std::printf("total %d size %d: first %d n %d\n", total, size, first, n);
                    return 1;
                }
                done += n;
            }
            if (done != total || b.next(a, c)) return 2;
        }
    std::printf("ok\n");
    return 0;
}
"""


def test_batches_cover_counts_up_to_the_largest(tmp_path):
    """Each count is taken whole, in order and once, to the last one before 2^31; no step of the
    walk leaves its type (checked by the compiler's overflow trap)."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(BATCHES)
    try:
        subprocess.run(["g++", "-O2", "-std=c++17", "-ftrapv", f"-I{CSRC}", str(src), "-o",
                        str(exe)], check=True, capture_output=True, text=True)
    except FileNotFoundError:
        pytest.skip("no host C++ compiler")
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr

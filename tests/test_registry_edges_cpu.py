"""The quantised registry at the ends of what its calls allow, as far as that goes without a
GPU: the batches of queries, and refusals made before any CUDA call."""
import subprocess
from pathlib import Path

import pytest

import vd_b200 as vd
from test_registry_cpu import FAKE, _args, _refused

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


@pytest.mark.parametrize("off", [1, 2, 3])
def test_pointers_off_their_types_alignment_are_refused(off):
    """A load or a store there would fault; every call says so before it launches anything."""
    L, bad = vd.lib(), FAKE + off

    # each call is made only with a pointer that it refuses: the addresses are not memory
    def clear(r=_args(), slots=None):
        return L.vdb_registry_clear(r, slots, 0, 1, None)

    def write(r=_args(), x=FAKE, t=0, slots=None):
        return L.vdb_registry_write(r, x, t, 256, slots, 0, 1, None)

    def read(r=_args(), x=FAKE, t=0, slots=None):
        return L.vdb_registry_read(r, slots, 0, 1, x, t, 256, None)

    def score(r=_args(), x=FAKE, t=0, out=FAKE):
        return L.vdb_registry_score(r, 9, x, t, 256, 1, out, 9, None, 0, None)

    def posterior(r=_args(), x=FAKE, t=0, labels=FAKE, lp=FAKE, ent=FAKE, lse=FAKE, idx=FAKE,
                  alt=FAKE):
        return L.vdb_registry_posterior(r, 9, x, t, 256, 1, 30.0, labels, 5, lp, ent, lse, idx,
                                        alt, FAKE, 1 << 30, None)

    def refused(calls, **kw):
        for call in calls:
            _refused(call(**kw), f"vdb_registry_{call.__name__}", "alignment")

    for field in ("scale", "owner"):
        r = _args(**{field: bad})
        refused((clear, write, read, score, posterior), r=r)
        assert L.vdb_registry_posterior_work(r, 9, 1, 5) == -1
    refused((clear, write, read), slots=bad)
    for t in (0, 1, 2):
        if t == 0 or off != 2:
            refused((write, read, score, posterior), x=bad, t=t)
    refused((score,), out=bad)
    for name in ("labels", "lp", "ent", "lse", "idx", "alt"):
        refused((posterior,), **{name: bad})

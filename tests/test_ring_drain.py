"""What a producer waits for before its block leaves (csrc/mbar.cuh, ring_drain): a model of the barriers of a
ring on the host, for every number of copies issued and taken."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

MODEL = r"""
#include <cuda.h>
#include <cstdio>
#include <vector>
#include "mbar.cuh"

// A `full` barrier: a copy issued into its stage completes the barrier's phase when it lands. A wait for a parity
// returns at once if the phase in progress has the other one; else it lasts until that phase completes, which
// it does if a copy is on its way and never if none is.
struct Full {
    uint32_t phase = 0;
    bool in_flight = false;
};

int main() {
    int bad = 0;
    for (uint32_t stages = 1; stages <= 8; stages++)
        for (uint32_t issued = 0; issued <= 4 * stages; issued++)
            for (uint32_t landed = issued > stages ? issued - stages : 0; landed <= issued; landed++) {
                std::vector<Full> ring(stages);
                uint32_t stage = 0, phase = 0;  // as the producers walk
                for (uint32_t i = 0; i < issued; i++) {
                    Full &f = ring[stage];
                    if (f.in_flight) { f.in_flight = false; f.phase ^= 1; }  // taken before it is filled again
                    f.in_flight = true;
                    if (i < landed) { f.in_flight = false; f.phase ^= 1; }
                    if (++stage == stages) { stage = 0; phase ^= 1; }
                }
                uint32_t stuck = 0;
                lyth::ring_drain(stage, phase, stages, [&](uint32_t s, uint32_t parity) {
                    Full &f = ring[s];
                    if (f.phase != parity) return;                              // complete already
                    if (f.in_flight) { f.in_flight = false; f.phase ^= 1; }      // lands while we wait
                    else stuck++;                                               // would run out
                });
                uint32_t left = 0;
                for (const Full &f : ring) left += f.in_flight;
                if (left || stuck) {
                    if (bad++ < 5) std::printf("stages %u issued %u landed %u: %u in flight, %u waits run out\n", stages, issued, landed, left, stuck);
                }
            }
    std::printf("%d\n", bad);
    return bad != 0;
}
"""


def test_no_copy_in_flight_and_no_wait_for_none(tmp_path):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "model.cu", tmp_path / "model"
    src.write_text(MODEL)
    subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "lyth_b200", "csrc"), "-o", str(exe), str(src)], check=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr

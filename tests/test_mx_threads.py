"""What the launchers keep per process, when several threads make a process's first calls at once. The
host code is compiled against a stand-in for the driver's lookup, so no GPU is needed."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

LOOKUP = r"""
#include <cuda.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include <cuda_runtime.h>

static std::atomic<int> lookups{0};
// The driver's lookup, slow enough that every thread arrives before it is over.
static cudaError_t slow_lookup(const char *, void **p, unsigned long long, cudaDriverEntryPointQueryResult *q) {
    lookups++;
    std::this_thread::sleep_for(std::chrono::milliseconds(200));
    *p = reinterpret_cast<void *>(0x1000);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
#define cudaGetDriverEntryPoint slow_lookup
#include "mbar.cuh"

int main() {
    std::atomic<int> waiting{0}, missing{0};
    std::vector<std::thread> threads;
    for (int i = 0; i < 8; i++)
        threads.emplace_back([&] {
            for (waiting++; waiting < 8;) std::this_thread::yield();
            if (!lyth::tensor_map_encoder()) missing++;
        });
    for (auto &t : threads) t.join();
    std::printf("missing %d lookups %d\n", missing.load(), lookups.load());
    return missing != 0 || lookups != 1;
}
"""


def test_tensor_map_lookup_by_threads_at_once(tmp_path):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "lookup.cu", tmp_path / "lookup"
    src.write_text(LOOKUP)
    subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "lyth_b200", "csrc"), "-o", str(exe), str(src)], check=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


FIRST = """
import threading
import torch
import lyth_b200 as lb

fmt, k = lb.MX_FP4, 512
cuda = torch.device("cuda")
gen = torch.Generator(device=cuda).manual_seed(0)


def operand(rows):
    codes, scales = lb.mx_empty(fmt, rows, k, cuda)
    return codes.random_(0, 256, generator=gen), scales.random_(120, 134, generator=gen)


a, b = operand(300), operand(WIDTH)
out = [torch.zeros(300, WIDTH, device=cuda) for _ in range(9)]
torch.cuda.synchronize()
meet, failed = threading.Barrier(8), []


def work(c):
    try:
        meet.wait()
        lb.matmul_mx(fmt, *a, *b, c, stream=0)
    except BaseException as e:
        failed.append(e)


threads = [threading.Thread(target=work, args=(c,)) for c in out[1:]]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not failed, failed
lb.matmul_mx(fmt, *a, *b, out[0], stream=0)
torch.cuda.synchronize()
assert bool(out[0].any()) and all(torch.equal(c, out[0]) for c in out[1:])
print("OK")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("n", [400, 20000])  # single SMs and CTA pairs
def test_products_as_the_first_calls_of_eight_threads(cuda, n):
    r = subprocess.run([sys.executable, "-c", FIRST.replace("WIDTH", str(n))], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("OK"), r.stdout + r.stderr


NO_CONTEXT = """
import threading
import torch
import lyth_b200 as lb

cuda = torch.device("cuda")
codes, scales = lb.mx_empty(lb.MX_FP8, 128, 512, cuda)
codes.fill_(0x38), scales.fill_(127)
c, d = torch.zeros(128, 128, device=cuda), torch.zeros(128, 256, device=cuda)
a, b = torch.ones(128, 64, dtype=torch.bfloat16, device=cuda), torch.ones(64, 256, dtype=torch.bfloat16, device=cuda)
torch.cuda.synchronize()
failed = []


def work(call):
    try:
        call()
    except BaseException as e:
        failed.append(e)


for call in (lambda: lb.matmul_mx(lb.MX_FP8, codes, scales, codes, scales, c, stream=0), lambda: lb.matmul_bf16(a, b, d, stream=0)):
    t = threading.Thread(target=work, args=(call,))
    t.start()
    t.join()
assert not failed, failed
torch.cuda.synchronize()
assert bool((c == 512).all()) and bool((d == 64).all())
print("OK")
"""


@pytest.mark.gpu
def test_products_on_threads_that_have_no_context(cuda):
    # a thread whose first CUDA work is the product: the tensor map is made before the runtime has set it up
    r = subprocess.run([sys.executable, "-c", NO_CONTEXT], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("OK"), r.stdout + r.stderr

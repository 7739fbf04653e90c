"""Host-side parts of the dense operators, compiled into a small program (CPU only): what is found out once a device, when threads'
first calls meet; what a launch plan asks of an SM."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG, REPO

PROGRAM = r"""
#include "dense.h"
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
using namespace glmx;

struct Table { int n[16]; };

int main()
{
    static PerDevice<Table> tables;
    std::atomic<int> fills{0}, wrong{0}, failed{0};
    // slow, in two steps, as a table that is read before it is complete would show
    auto fill = [&](int device) {
        return [&, device](Table& t) {
            ++fills;
            for (int i = 0; i < 16; ++i) { t.n[i] = device + i; std::this_thread::sleep_for(std::chrono::milliseconds(1)); }
            for (int i = 0; i < 16; ++i) t.n[i] *= 2;
            return cudaSuccess;
        };
    };
    std::vector<std::thread> threads;
    for (int k = 0; k < 24; ++k)
        threads.emplace_back([&, k] {
            const int device = k % 3;
            const Table* t = nullptr;
            if (tables.get(device, &t, fill(device)) != cudaSuccess) { ++failed; return; }
            for (int i = 0; i < 16; ++i) wrong += t->n[i] != 2 * (device + i);
        });
    for (auto& t : threads) t.join();
    std::printf("fills %d wrong %d failed %d\n", fills.load(), wrong.load(), failed.load());
    // an error is reported and not kept; devices out of range are errors
    const Table* t = nullptr;
    const int first = tables.get(7, &t, [](Table&) { return cudaErrorNotReady; }) == cudaErrorNotReady, none = t == nullptr;
    const int again = tables.get(7, &t, fill(7)) == cudaSuccess && t->n[1] == 16;
    const int range = tables.get(-1, &t, fill(0)) == cudaErrorInvalidDevice && tables.get(64, &t, fill(0)) == cudaErrorInvalidDevice;
    std::printf("error %d %d %d range %d\n", first, none, again, range);
    return 0;
}
"""


def run(tmp_path, source):
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc")
    if not nvcc:
        pytest.skip("no nvcc")
    src, exe = tmp_path / "host.cu", tmp_path / "host"
    src.write_text(source)
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                    "-I" + os.path.join(REPO, "include"), "-I" + os.path.join(PKG, "csrc"), str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout


def test_once_a_device(tmp_path):
    out = run(tmp_path, PROGRAM).splitlines()
    assert out == ["fills 3 wrong 0 failed 0", "error 1 1 1 range 1"]


PLANS = r"""
#include "gemm_tc.cuh"
#include <cstdio>
using namespace glmx;

int main()
{
    // an SM: 228 KB of shared memory, of which each CTA takes 1 KB more than it asks for, and 512 columns of tensor memory
    const int SM = 228 * 1024;
    int cost[600] = {};                                    // least shared memory of a CTA with so many columns
    auto put = [&](int cols, int bytes) { if (!cost[cols] || bytes < cost[cols]) cost[cols] = bytes; };
    for (int bn = 64; bn <= 256; bn += 64) put(512, pair_smem(bn) + 1024);
    ColsCapacity cap;
    for (int i = 0; i < 2; ++i)
        for (int s = 0; s <= 8; ++s) cap.n[i][s] = s ? (i ? 148 : 296) / s : 0;
    int most = 0;
    for (int gated = 0; gated < 2; ++gated)
        for (int M = 1; M <= 3000; M += M < 300 ? 1 : 37)
            for (int N : { 8, 64, 136, 1000, 6144, 65536 })
                for (int nk : { 1, 2, 3, 5, 8, 17, 24, 96, 512 })
                {
                    const ColsPlan p = cols_plan(M, N, gated, nk, cap);
                    if (p.us > 1e29) continue;
                    put(cols_tmem(p), cols_smem(p) + 1024);
                    if (cols_smem(p) > most) most = cols_smem(p);
                }
    // the most columns that CTAs which fit an SM together can want
    static int best[SM / 256 + 1];
    for (int b = 1; b <= SM / 256; ++b)
        for (int c = 32; c <= 512; c *= 2)
            if (cost[c] && cost[c] <= b * 256)
            {
                const int left = (b * 256 - cost[c]) / 256;
                if (best[left] + c > best[b]) best[b] = best[left] + c;
            }
    std::printf("columns %d launchable %d\n", best[SM / 256], most <= COLS_SMEM1);
    return 0;
}
"""


def test_ctas_that_fit_an_sm_fit_its_tensor_memory(tmp_path):
    """Else clusters of two streams could each hold what the other waits for."""
    assert run(tmp_path, PLANS).split() == ["columns", "512", "launchable", "1"]

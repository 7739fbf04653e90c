"""Host-side parts of the dense operators, compiled into a small program (CPU only): what is found out once a device, when threads'
first calls meet."""
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

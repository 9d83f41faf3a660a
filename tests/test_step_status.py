"""The words that device code reports through (csrc/status.hpp), in a host
program: a second thread stands for a kernel that is still running while the
host takes the word. The last code of each of its bursts has to be seen."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_HARNESS = r"""
#include "status.hpp"
#include <atomic>
#include <cstdio>
#include <thread>
int main() {
    uint32_t word = 0;
    const uint32_t bursts = 200000;
    std::atomic<uint32_t> seen{0};
    std::atomic<bool> lost{false};
    std::thread device([&] {
        for (uint32_t b = 1; b <= bursts && !lost; ++b) {
            __atomic_store_n(&word, 2 * b, __ATOMIC_RELAXED);
            for (volatile uint32_t wait = 0; wait < b % 64; wait = wait + 1) {}
            __atomic_store_n(&word, 2 * b + 1, __ATOMIC_RELAXED);
            // the host takes the word on and on: 2 s without the code are a loss
            for (uint64_t spins = 0; seen.load() < 2 * b + 1; ++spins) {
                if (spins > 2000) std::this_thread::sleep_for(std::chrono::milliseconds(1));
                if (spins > 4000) { lost = true; break; }
            }
        }
        seen = 0xFFFFFFFFu;
    });
    while (seen.load() != 0xFFFFFFFFu) {
        const uint32_t st = mmhip::take_status(&word);
        if (st) {
            uint32_t was = seen.load();
            while (was != 0xFFFFFFFFu && was < st && !seen.compare_exchange_weak(was, st)) {}
        }
    }
    device.join();
    if (lost) puts("a report was lost");
    return lost ? 1 : 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_no_report_is_lost(tmp_path):
    src, exe = tmp_path / "status.cpp", tmp_path / "status"
    src.write_text(_HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-pthread", "-I",
                    os.path.join(ROOT, "mobile-moe.zig_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr

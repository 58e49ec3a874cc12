"""csrc/lds_limit.h by itself, compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "lds_limit.h"
#include <chrono>
#include <cstdio>
#include <thread>

int main() {
    // One thread sets 64 and, in the middle of that, lets another that wants 128 go on for as long as it can: what holds
    // in the end, and at the second's launch, must be 128.
    static LdsLimit lim;
    std::atomic<size_t> attribute{0}, at_launch{0};
    std::atomic<bool> inside{false}, done{false};
    std::thread second([&] {
        while (!inside) std::this_thread::yield();
        lim.raise(0, 128, [&](size_t want) { attribute = want; return true; });
        done = true;
        std::this_thread::sleep_for(std::chrono::milliseconds(600));
        at_launch = attribute.load();
    });
    lim.raise(0, 64, [&](size_t want) {
        inside = true;
        for (int i = 0; i < 300 && !done; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
        attribute = want;
        return true;
    });
    second.join();
    if (attribute != 128 || at_launch != 128) { std::printf("lowered to %zu\n", (size_t)at_launch); return 1; }
    // set once, and only for more; a failure is not noted
    int calls = 0;
    auto count = [&](size_t) { ++calls; return true; };
    lim.raise(0, 100, count);
    lim.raise(0, 128, count);
    if (calls != 0) { std::printf("set again\n"); return 1; }
    if (lim.raise(1, 50, [](size_t) { return false; })) { std::printf("failure not told\n"); return 1; }
    lim.raise(1, 50, count);
    lim.raise(-1, 50, count);
    lim.raise(LdsLimit::MAX_DEV, 50, count);
    if (calls != 3) { std::printf("%d calls\n", calls); return 1; }
    return 0;
}
"""


def test_a_limit_is_never_lowered_between_another_calls_setting_and_its_launch(tmp_path):
    source, program = tmp_path / "limit.cpp", tmp_path / "limit"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "onmf_ontf_ndl_amd", "csrc"), str(source),
                    "-o", str(program)], check=True, timeout=100)
    run = subprocess.run([str(program)], stdout=subprocess.PIPE, text=True, timeout=60)
    assert run.returncode == 0, run.stdout

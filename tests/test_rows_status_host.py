"""Who hears of a wait that ran out in the operators without a handle: the host side, compiled by itself, without a GPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = r"""
#include <cassert>
#include <cstdint>
#include <thread>
#include <vector>
#include "pmoe_status.h"
int main()
{
    auto stream = [](uintptr_t i) { return (const void *)i; };
    pmoe::FailureCounts c;
    assert(!c.news(0, stream(1), 0) && !c.news(0, stream(2), 0));
    // stream 1 asks first: stream 2, whose wait it may have been, hears of it all the same, and each only once
    assert(c.news(0, stream(1), 3) && !c.news(0, stream(1), 3));
    assert(c.news(0, stream(2), 3) && !c.news(0, stream(2), 3));
    assert(c.news(0, stream(1), 4) && c.news(0, stream(2), 5) && c.news(0, stream(1), 5));
    // a stream that has never asked hears of what was before; the default stream is one of them; devices are apart
    assert(c.news(0, nullptr, 5) && !c.news(0, nullptr, 5) && !c.news(1, stream(1), 0) && c.news(1, stream(1), 1));
    // many threads at once: one of those that ask on a stream hears of a failure
    std::vector<int> heard(8, 0);
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; t++)
        threads.emplace_back([&, t] {
            for (unsigned i = 0; i < 1000; i++) heard[t] += c.news(2, stream(10 + t % 2), 1);
        });
    for (auto &t : threads) t.join();
    int even = 0, odd = 0;
    for (int t = 0; t < 8; t++) (t % 2 ? odd : even) += heard[t];
    assert(even == 1 && odd == 1);
    return 0;
}
"""


def test_every_stream_hears_of_a_failure_once(tmp_path):
    source, program = tmp_path / "status.cpp", tmp_path / "status"
    source.write_text(MAIN)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-pthread", "-I", os.path.join(ROOT, "paramecia_b200", "csrc"), str(source), "-o", str(program)])
    subprocess.check_call([str(program)], timeout=60)

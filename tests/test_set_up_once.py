"""CPU: a kernel's set-up on a device (csrc/set_up_once.h) with fakes of the calls that it makes: what fails is not
remembered as done, and no thread passes before it is done."""
import os
import re
import subprocess

from tests.conftest import ROOT

CSRC = os.path.join(ROOT, "seedvr2_ncnn_b200", "csrc")

PROGRAM = r"""
#include "set_up_once.h"
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>

static int failures = 0;
#define EXPECT(x) do { if (!(x)) { failures++; std::printf("line %d: %s\n", __LINE__, #x); } } while (0)

enum Error { kSuccess = 0, kBad = 7 };

int main()
{
    // a kernel with other registers than its split assumes is refused by every call, not by the first alone
    {
        std::atomic<uint64_t> done{0};
        int registers = 167, calls = 0;
        auto check = [&] { calls++; return registers == 168 ? 0 : -3; };
        for (int i = 0; i < 3; i++) EXPECT(s2::set_up_once(done, 0, check) == -3);
        EXPECT(calls == 3);
        registers = 168; // (a passing failure of a call is not kept either)
        EXPECT(s2::set_up_once(done, 0, check) == 0);
        EXPECT(s2::set_up_once(done, 0, check) == 0);
        EXPECT(calls == 4);
    }
    // each device for itself; numbers without a bit each time
    {
        std::atomic<uint64_t> done{0};
        int calls = 0;
        auto ok = [&] { calls++; return kSuccess; };
        for (int i = 0; i < 2; i++)
            for (int d : {0, 1, 63}) EXPECT(s2::set_up_once(done, d, ok) == kSuccess);
        EXPECT(calls == 3);
        for (int d : {-1, 64, 65}) EXPECT(s2::set_up_once(done, d, ok) == kSuccess);
        EXPECT(s2::set_up_once(done, 64, ok) == kSuccess);
        EXPECT(calls == 7);
        EXPECT(s2::set_up_once(done, 2, [] { return kBad; }) == kBad);
    }
    // threads that come while the first is at it do not pass before the attribute is set
    for (int round = 0; round < 20; round++)
    {
        std::atomic<uint64_t> done{0};
        std::atomic<int> limit{0}, early{0};
        std::vector<std::thread> threads;
        for (int i = 0; i < 8; i++)
            threads.emplace_back([&] {
                const int r = s2::set_up_once(done, 0, [&] {
                    std::this_thread::sleep_for(std::chrono::milliseconds(2));
                    limit.store(1);
                    return 0;
                });
                if (r != 0 || limit.load() != 1) early++;
            });
        for (auto& t : threads) t.join();
        EXPECT(early.load() == 0);
    }
    return failures != 0;
}
"""


def test_set_up_once(tmp_path):
    src, exe = tmp_path / "set_up.cpp", tmp_path / "set_up"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-pthread", "-I", CSRC, str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_register_splits_are_checked_through_it():
    """A kernel that moves registers between its warps (setmaxnreg) assumes how many it was launched with; the check
    of that stands inside the set-up."""
    split = checked = 0
    for f in sorted(os.listdir(CSRC)):
        if not f.endswith(".cu"):
            continue
        text = open(os.path.join(CSRC, f)).read()
        split += "setmaxnreg.inc" in text
        for m in re.finditer(r"\.numRegs", text):
            at = text.rfind("set_up_current_device(", 0, m.start())
            assert at >= 0 and "});" not in text[at:m.start()], f
            checked += 1
    assert checked == split == 2

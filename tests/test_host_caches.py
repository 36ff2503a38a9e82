"""The engine's per-device caches under concurrent calls, on the host: built with the thread
sanitizer, which reports an unsynchronised access whichever way the threads happen to run."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gemmkit_b200", "csrc")

PROGRAM = r"""
#include "gk_once.h"
#include <stdio.h>
#include <thread>
#include <vector>

static int first(int dev) {
    static gk::PerDevice<int> cache;
    return cache.get(dev, [dev] { return 100 + dev; });
}

static std::atomic<int> tries{0};
static int* pointer(int dev) {
    static gk::PerDevice<int*> cache;
    static int value[64];
    return cache.get(dev, [dev]() -> int* { return tries++ < 3 ? nullptr : &value[dev]; });
}

int main() {
    std::atomic<int> wrong{0};
    std::vector<std::thread> all;
    for (int t = 0; t < 8; ++t)
        all.emplace_back([&] {
            for (int i = 0; i < 2000; ++i)
                if (first(i % 64) != 100 + i % 64) ++wrong;
        });
    for (auto& t : all) t.join();
    // a look-up that fails is tried again
    for (int i = 0; i < 3; ++i) wrong += pointer(5) != nullptr;
    wrong += pointer(5) == nullptr || pointer(5) != pointer(5) || tries != 4;
    printf("wrong %d\n", wrong.load());
    return wrong.load() != 0;
}
"""


def test_per_device_cache_is_free_of_races(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    src, exe = tmp_path / "once.cc", tmp_path / "once"
    src.write_text(PROGRAM)
    flags = ["-std=c++17", "-O1", "-g", "-pthread", f"-I{CSRC}", str(src), "-o", str(exe)]
    probe = tmp_path / "probe.cc"
    probe.write_text("int main() { return 0; }\n")
    tsan = subprocess.run([gxx, "-fsanitize=thread", str(probe), "-o", str(tmp_path / "probe")],
                          capture_output=True).returncode == 0 and \
        subprocess.run([str(tmp_path / "probe")], capture_output=True).returncode == 0
    subprocess.run([gxx, *(["-fsanitize=thread"] if tsan else []), *flags], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "wrong 0" in out.stdout, out.stdout + out.stderr[-2000:]


def test_no_cache_is_a_plain_static_array():
    """What a function keeps per device for all threads is a PerDevice (or guarded by a mutex or an
    atomic of its own)."""
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        for m in re.finditer(r"\n    static (?!__device__|PerDevice|gk::PerDevice)[\w: \*]+ (\w+)\[64\]",
                             text):
            head = text[:m.start()]
            body = text[m.start():m.start() + 400]
            scope = head[head.rindex("\n}"):] if "\n}" in head else head
            guarded = "lock_guard" in body or "lock_guard" in scope
            assert "thread_local" in m.group(0) or guarded, f"{name}: {m.group(1)}"

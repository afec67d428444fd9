"""CPU: the rule by which calls refuse buffers that overlap, against every byte."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "overlap.hpp"
#include <cstdio>
#include <random>
#include <set>
using sili::Rows;
static std::set<long> bytes(const Rows &r) {
    std::set<long> s;
    for (long i = 0; i < r.n; ++i)
        for (long w = 0; w < (long)r.width; ++w) s.insert((long)r.p + i * (long)r.pitch + w);
    return s;
}
int main() {
    std::mt19937 rng(1);
    auto in = [&](long lo, long hi) { return std::uniform_int_distribution<long>(lo, hi)(rng); };
    long both[2] = {0, 0};
    for (int t = 0; t < 100000; ++t) {
        const long pitch = in(-9, 9);
        Rows x{(const void *)(1000 + in(0, 60)), in(0, 5), in(0, 8), pitch}, y{(const void *)(1000 + in(0, 60)), in(0, 5), in(0, 8), t % 3 ? pitch : in(-9, 9)};
        if (t % 7 == 0) y.pitch = -x.pitch;
        bool common = false;
        const auto s = bytes(y);
        for (long b : bytes(x)) common |= s.count(b) != 0;
        const bool got = sili::meet(x, y), exact = x.n <= 1 || y.n <= 1 || x.pitch == y.pitch || x.pitch == -y.pitch;
        if (got != sili::meet(y, x) || (common && !got) || (exact && got != common)) {
            printf("x %ld %ld %ld %ld y %ld %ld %ld %ld: %d %d\n", (long)x.p, (long)x.n, (long)x.width, (long)x.pitch, (long)y.p, (long)y.n,
                   (long)y.width, (long)y.pitch, got, common);
            return 1;
        }
        ++both[got];
    }
    const void *low = (const void *)4096;
    if (sili::meet({nullptr, 4, 4, 4}, {nullptr, 4, 4, 4})) return 2;
    if (!sili::meet({low, INT64_MAX, INT64_MAX, INT64_MAX}, {(const void *)~0ul, 1, 1, 0})) return 3;
    if (sili::meet({low, INT64_MAX, 1, INT64_MIN}, {(const void *)8192, INT64_MAX, 1, INT64_MAX})) return 4;
    return both[0] > 1000 && both[1] > 1000 ? 0 : 5;
}
"""


def test_against_every_byte(tmp_path):
    src, exe = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-int-to-pointer-cast", f"-I{ROOT}/sili__new_amd/csrc", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)

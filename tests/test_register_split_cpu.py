"""CPU: a kernel whose warps trade registers is launched only where the compiler gave it as many as they draw."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "register_split.h"
using mxb200::RegisterSplit;
constexpr RegisterSplit split{4, 72, 8, 216};
static_assert(split.needed() == 168);
static_assert(split.served_by(168) && split.served_by(255));
// 128 x 72 + 256 x 216 registers from a block of 384 x 160: the last warps would wait for some that nobody has
static_assert(!split.served_by(160) && !split.served_by(167) && !split.served_by(128));
static_assert(RegisterSplit{4, 40, 8, 121}.needed() == 94);  // rounded up
static_assert(RegisterSplit{}.needed() == 0 && RegisterSplit{}.served_by(32));
static_assert(!RegisterSplit{4, 96, 8, 64}.served_by(80));  // "down" from less than it leaves
int main() {}
"""


def test_what_a_split_needs(tmp_path):
    src = tmp_path / "split.cpp"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-fsyntax-only", "-I",
                           os.path.join(ROOT, "nanochat_cpp_b200", "csrc"), str(src)])

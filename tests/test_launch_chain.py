"""Which attention launches may overlap the ones before them (csrc/launch_chain.h), on the CPU: decided by layers and by what the launches
read and write."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "titan_engine_b200", "csrc")

PROGRAM = r"""
#include "launch_chain.h"
#include <cstdio>
using tk::MemRange;
static char x[400];
static int bad = 0;
static void want(bool got, bool yes, const char* what) { if (got != yes) { std::printf("%s: %d\n", what, got); bad = 1; } }
int main() {
    const MemRange q{x, 100}, a{x + 100, 100}, b{x + 200, 100}, none{nullptr, 0};
    tk::LaunchChain c;
    want(c.add(true, 0, {q}, a), false, "the first has nothing to overlap");
    want(c.add(true, 1, {q}, b), true, "another layer");
    want(c.add(true, 2, {q, none}, a), true, "a third; its output is written after the wait");
    want(c.add(true, 0, {q}, b), false, "the first layer again, two launches later");
    want(c.add(true, 1, {q}, a), true, "a new chain: only the last launch is in it");
    want(c.add(true, 2, {b}, MemRange{x + 300, 100}), false, "reads the output of the launch before the last");
    want(c.add(true, 3, {MemRange{x + 399, 1}}, a), false, "reads the last byte of the last output");
    want(c.add(true, 4, {MemRange{x + 200, 100}}, b), true, "begins where the output ends");
    want(c.add(true, 5, {q, MemRange{x + 90, 11}}, a), false, "the second input reaches into an output");
    want(c.add(false, 6, {q}, a), false, "not allowed");
    want(c.add(true, 5, {q}, a), true, "... which began a new chain");
    c.clear();
    want(c.add(true, 7, {q}, a), false, "cleared");
    want(c.add(true, 8, {none}, none), true, "empty ranges meet nothing");
    return bad;
}
"""


def test_layers_and_ranges(tmp_path):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    (tmp_path / "chain.cpp").write_text(PROGRAM)
    exe = str(tmp_path / "chain")
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(tmp_path / "chain.cpp"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout

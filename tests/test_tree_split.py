"""That the cases of tests/tree_cases.py reach the kernels that they are for: the library's own rule is asked, through a compiled caller of it
(tests/cpp/tree_split.cpp)."""
import os
import subprocess

import pytest

import nunchi_amd
import tree_cases
from conftest import ROOT


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    """sizes -> (column groups of the shared positions, of the own ones, parts of either)."""
    exe = str(tmp_path_factory.mktemp("cpp") / "tree_split")
    lib = os.path.dirname(nunchi_amd.LIB_PATH)
    r = subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", exe, os.path.join(ROOT, "tests", "cpp", "tree_split.cpp"),
                        nunchi_amd.LIB_PATH, f"-Wl,-rpath,{lib}", "-L/opt/rocm/lib", "-Wl,-rpath,/opt/rocm/lib", "-Wl,-rpath-link,/opt/rocm/lib"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def ask(*sizes):
        r = subprocess.run([exe, *(str(x) for s in sizes for x in s)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return [tuple(int(x) for x in line.split()) for line in r.stdout.splitlines()]

    return ask


def test_cases_reach_their_kernels(split):
    cases = tree_cases.cases()
    got = split(*(tree_cases.sizes_of(c) for c in cases))
    assert len(got) == len(cases)
    wrong = [(tree_cases.name(c), g) for c, g in zip(cases, got) if g[:2] != c["kernel"]]
    assert not wrong
    assert all((g[2] > 0) == (c["kernel"][0] > 0) for c, g in zip(cases, got))


def test_every_kernel_has_cases():
    want = {(D, k) for D in tree_cases.DIMS for k in [(0, 1), (0, 2), (1, 1), (2, 1), (2, 2)] + ([(0, 4)] if D <= 64 else [])}
    have = {(c["D"], c["kernel"]) for c in tree_cases.cases()}
    assert have == want
    assert {(c["D"], c["kernel"]) for c in tree_cases.cases() if c["window"]} == want

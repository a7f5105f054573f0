"""The size that a library workspace grows to
(arclight_amd/csrc/workspace_growth.hpp, compiled by the host's compiler):
twice the one before it, or what the call needs where that much is not free."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
MB = 1 << 20


@pytest.fixture(scope="module")
def grow(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path_factory.mktemp("workspace_growth") / "probe")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-o", exe, os.path.join(HERE, "csrc", "workspace_growth.cpp")], check=True)

    def run(*a):
        out = subprocess.run([exe, *map(str, a)], capture_output=True, text=True, check=True).stdout.split()
        return int(out[0]), [int(x) for x in out[1:]]
    return run


@pytest.mark.parametrize("bytes_, held, free, got, asked", [
    (1000, 0, 1 << 40, 20 * MB, [20 * MB]),
    (30 * MB, 20 * MB, 1 << 40, 40 * MB, [40 * MB]),
    (90 * MB, 20 * MB, 1 << 40, 90 * MB, [90 * MB]),
    (2100 * MB, 2000 * MB, 3000 * MB, 2100 * MB, [4000 * MB, 2100 * MB]),     # fits, though twice the size does not
    (1000, 0, 5 * MB, 1000, [20 * MB, 1000]),
    (2100 * MB, 2000 * MB, 2000 * MB, 0, [4000 * MB, 2100 * MB]),
    (90 * MB, 20 * MB, 80 * MB, 0, [90 * MB]),                                # not asked for twice
    (5000 * MB, 0, 5000 * MB, 5000 * MB, [5000 * MB]),                        # past 32 bits
])
def test_grow(grow, bytes_, held, free, got, asked):
    assert grow(bytes_, held, free) == (got, asked)

"""The walk of attention's blocks over units and stages, run on the host from the
kernel's own source: every stage of every unit once, producers and consumers in step;
with lengths that change while the call runs it still ends, in bounds."""
import os
import subprocess

import pytest

from conftest import REPO


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("walk") / "kv4_walk_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall", "-Wextra", "-Werror",
                    "-I", os.path.join(REPO, "mini-rust-inference_b200", "csrc"),
                    os.path.join(REPO, "tests", "kv4_walk_check.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("seed", range(4))
def test_walk(walk, seed):
    r = subprocess.run([walk, str(seed), "2000"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr

"""The ring of tiles of the attention over 8-bit pages (csrc/ring8.h), run on
the CPU with copies that land in any order (tests/cpp/ring8_model.cpp): no
warp takes a tile before it has landed, no copy overwrites one that is still read."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    to = str(tmp_path_factory.mktemp("ring8") / "ring8_model")
    subprocess.run(["g++", "-std=c++20", "-O2", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "tinyllama-engine_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "ring8_model.cpp"), "-o", to], check=True)
    return lambda *how: subprocess.run([to, *how], capture_output=True, text=True, timeout=300)


def test_every_tile_is_met_in_its_lap(model):
    r = model()
    assert r.returncode == 0, r.stdout
    assert r.stdout.count(": ok") == len(r.stdout.splitlines()) >= 10


def test_the_model_sees_a_wait_for_the_barrier_alone(model):
    """Parity alone: a warp that never met the stage's tile of the lap before takes it for the next one."""
    r = model("plain")
    assert r.returncode == 1 and "one team, 8 rows: early" in r.stdout and "three teams: early" in r.stdout, r.stdout

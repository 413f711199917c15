"""How the attention kernel deals out its work, for random batches (wild tables among them), on the host: the
probe includes the very code that the kernels run."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("dealing") / "kv_dealing_probe")
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", out,
                        os.path.join(HERE, "kv_dealing_probe.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return out


@pytest.mark.parametrize("seed", range(4))
def test_every_tile_once_and_every_part_found(probe, seed):
    r = subprocess.run([probe, str(seed + 11), "40"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.startswith("ok 40 cases"), (r.returncode, r.stdout[-500:], r.stderr[-1500:])


def test_lengths_end_with_the_table_and_below_32_bits(tmp_path):
    out = str(tmp_path / "kv_rows_probe")
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", out,
                        os.path.join(HERE, "kv_rows_probe.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok 10\n", (r.stdout, r.stderr)

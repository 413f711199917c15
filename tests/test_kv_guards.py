"""What the key/value cache kernels' shared code makes of unusual but legal calls and of wild tables, on the host: the probes
include the very code that the kernels run."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def build(name, where):
    out = str(where / name)
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", out,
                        os.path.join(HERE, name + ".cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return out


def run(*args):
    r = subprocess.run([str(a) for a in args], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.startswith("ok "), (r.returncode, r.stdout[-500:], r.stderr[-1500:])
    return r.stdout


@pytest.fixture(scope="module")
def phases(tmp_path_factory):
    return build("kv_phases_probe", tmp_path_factory.mktemp("phases"))


@pytest.mark.parametrize("seed", range(4))
def test_streams_know_every_phase_of_the_barriers_they_wait_for(phases, seed):
    run(phases, seed + 1, 150)


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    return build("kv_search_probe", tmp_path_factory.mktemp("search"))


@pytest.mark.parametrize("seed", range(4))
def test_a_row_is_only_looked_for_where_its_sequence_has_it(search, seed):
    run(search, seed + 1, 300)


def test_tile_numbers_stay_within_32_bits(tmp_path):
    run(build("kv_totals_probe", tmp_path))


def test_a_row_sees_all_keys_its_mask_leaves_it(tmp_path):
    run(build("kv_seen_probe", tmp_path))


def test_no_report_is_lost_between_a_look_at_the_status_and_its_clearing(tmp_path):
    if not os.path.exists("/usr/local/cuda/include/cuda_runtime.h"):
        pytest.skip("CUDA headers not present")
    csrc = os.path.join(os.path.dirname(HERE), "torpor_b200", "csrc")
    exe = str(tmp_path / "kv_status_probe")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-pthread", "-o", exe, os.path.join(HERE, "kv_status_probe.cpp"),
                        *(os.path.join(csrc, f) for f in ("engine.cpp", "engine_swap.cpp", "engine_share.cpp", "pool.cpp", "evictor.cpp", "scheduler.cpp",
                                                          "controller.cpp", "kv_cache.cpp")),
                        "-I/usr/local/cuda/include", "-L/usr/local/cuda/lib64", "-lcudart", "-lrt", "-ldl"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60,
                       env=dict(os.environ, LD_LIBRARY_PATH="/usr/local/cuda/lib64:" + os.environ.get("LD_LIBRARY_PATH", "")))
    assert r.returncode == 0 and r.stdout == "ok 4096\n", (r.stdout, r.stderr)


def test_a_workspace_holds_the_lists_there_are(tmp_path):
    run(build("kv_workspace_probe", tmp_path))

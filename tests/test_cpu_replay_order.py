"""The replay program's use of streams and graphs, on a runtime that only keeps account of order (no GPU needed)."""
import importlib.util
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def ordering(tmp_path_factory):
    spec = importlib.util.spec_from_file_location("hom_build_flags", REPO / "hands-on-mlir_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    out = tmp_path_factory.mktemp("replay")
    build._compile(build.CSRC / "bert_replay.cpp", out / "replay.o", False)
    cuda = Path(build._nvcc()).resolve().parents[1] / "include"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{cuda}", f"-I{build.INCLUDE}", "-o", str(out / "ordering"),
                    str(REPO / "tests" / "replay_stub" / "ordering.cpp"), str(out / "replay.o")], check=True)
    return out / "ordering"


@pytest.mark.parametrize("scenario", ["default_stream", "deferred_layernorm", "options", "host_buffers", "callers_stream"])
def test_every_call_comes_after_the_one_before(ordering, scenario):
    run = subprocess.run([str(ordering), scenario], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout + run.stderr


@pytest.mark.parametrize("scenario", ["new_weights", "new_constants"])
def test_no_graph_outlives_its_weights(ordering, scenario):
    run = subprocess.run([str(ordering), scenario], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout + run.stderr

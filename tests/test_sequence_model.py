"""The sequence operators' kernels on the CPU model (tools/hipemu): the gpu-marked tests of the operators without a GPU, and the
first of them under the model's lane-level race detector."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EMU = os.path.join(ROOT, "tools", "hipemu")


def run(build, tests, *extra):
    env = dict(os.environ, DALI_AMD_HIPEMU=build)
    env.pop("LD_PRELOAD", None)
    cmd = [sys.executable, "-m", "pytest", "-q", "-m", "gpu", "-p", "no:cacheprovider", *extra, *tests]
    out = subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=1500)
    tail = "\n".join(out.stdout.splitlines()[-40:]) + out.stderr[-2000:]
    assert out.returncode == 0 and " passed" in out.stdout, tail
    return out.stdout + out.stderr


@pytest.mark.parametrize("tests", ["test_gpu_sequence.py", "test_gpu_sequence_use.py"])
def test_gpu_tests_pass_on_the_cpu_model(tests):
    subprocess.check_call(["make", "-s", "-j8", "-C", EMU])
    run("1", ["tests/" + tests], "-n", "4")


def test_kernels_are_race_free_on_the_cpu_model():
    subprocess.check_call(["make", "-s", "-j8", "-C", EMU, "RACE=1"])
    text = run("race", ["tests/test_gpu_sequence.py"], "-s", "-p", "no:xdist", "-k",
               "packed or per_channel or in_place or long_and_split or sizes or outside or one_token or together")
    assert "race at" not in text and "racecheck:" not in text, text[-4000:]

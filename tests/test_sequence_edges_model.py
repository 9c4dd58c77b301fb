"""test_gpu_sequence_edges.py on the CPU model of the kernels (tools/hipemu)."""
import subprocess

from tests.test_sequence_model import EMU, run


def test_edges_on_the_cpu_model():
    subprocess.check_call(["make", "-s", "-j8", "-C", EMU])
    run("1", ["tests/test_gpu_sequence_edges.py"], "-n", "4")

"""What each make target asks for (dry runs: nothing is built)."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustyllm_b200", "csrc")


def dry(*args):
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], capture_output=True, text=True)


def test_the_c_library_asks_for_no_python():
    r = dry("librq", "PYTHON=/nowhere/python3")
    assert r.returncode == 0, r.stderr
    assert "librq.so" in r.stdout and "rq_llama.cu" in r.stdout and "rq_torch" not in r.stdout
    assert "/nowhere" not in r.stdout + r.stderr


def test_everything_is_the_library_and_the_binding():
    r = dry()
    assert r.returncode == 0, r.stderr
    assert "librq.so" in r.stdout and "rq_torch.cpp" in r.stdout

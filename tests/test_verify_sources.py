"""What the results of the verification of drafts cannot show, or only at sizes that a test has no time for: no GPU needed."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNEL = os.path.join(ROOT, "spy_amd", "csrc", "sample_verify.hip")


def test_requests_are_shared_out_in_64_bits(tmp_path):
    """The counters that the threads of a launch set to 0: each once, and nothing in front of the array, in launches of up to 2^32 - 1 threads too."""
    out = str(tmp_path / "launch_index")
    subprocess.check_call(["g++", "-O2", "-std=c++20", "-o", out, os.path.join(ROOT, "tests", "host", "launch_index.cpp")])
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
    kernel = open(KERNEL).read()
    assert kernel.count("for (int64_t i = launch_first(blockIdx.x, SM_THREADS, threadIdx.x); i < a.n_seq; i += launch_step(gridDim.x, SM_THREADS)) a.arrived[i] = 0;") == 1
    assert not re.search(r"blockIdx\.x \* SM_THREADS|gridDim\.x \* SM_THREADS", kernel)

"""What the results of the verification of drafts do not show, and its limits: no GPU needed."""
import os
import re
import shutil
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


def test_sums_of_parts_are_stored_before_their_workgroup_is_counted(tmp_path):
    """The workgroup that is counted last reads the sums of all: the wave that counts has stored its workgroup's sums itself and has waited for the stores.  A release of one wave waits for
    that wave's stores alone, and a barrier does not wait for those of the others."""
    flags = re.search(r"^HIPFLAGS \?= ((?:.*\\\n)*.*)$", open(os.path.join(ROOT, "spy_amd", "csrc", "Makefile")).read(), re.M).group(1)
    flags = [f for f in flags.replace("\\\n", " ").replace("$(ARCH)", "gfx950").replace("$(PRELOAD)", "").split() if f != "-Wall"]
    out = str(tmp_path / "verify.s")
    subprocess.run([shutil.which("hipcc") or "/opt/rocm/bin/hipcc"] + flags + ["-w", "--cuda-device-only", "-S", "-o", out, KERNEL], check=True, capture_output=True, timeout=300)
    text = open(out).read()
    code = re.search(r"^_Z18verify_draw_kernel\w+:.*?^\.Lfunc_end", text, re.M | re.S).group(0).split("\n")
    count = [i for i, line in enumerate(code) if re.search(r"\bglobal_atomic_add\b", line)]
    sums = [i for i, line in enumerate(code) if re.search(r"\bglobal_store_dwordx2\b.* sc1\b", line)]
    assert len(count) == 1 and len(sums) == 1 and sums[0] < count[0], (sums, count)
    between = "\n".join(code[sums[0]:count[0]])
    assert "s_barrier" not in between and re.search(r"s_waitcnt vmcnt\(0\)", between), between


def test_differences_of_probabilities_are_off_by_what_the_header_says(tmp_path):
    """2^-50 of the larger probability and 2^-60; 2^-60 alone would not be true."""
    out = str(tmp_path / "verify_share")
    subprocess.check_call(["g++", "-O2", "-std=c++20", "-ffp-contract=off", "-o", out, os.path.join(ROOT, "tests", "host", "verify_share.cpp")])
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    worst, steps = map(float, r.stdout.split())
    assert 0 < worst <= 1 and 10 < steps < 1024, r.stdout
    header = open(os.path.join(ROOT, "include", "spy_hip.h")).read()
    assert "p - q by 2^-50 of the larger of them and 2^-60 more" in header
    assert open(KERNEL).read().count("verify_more(w, one_p, ") == 1


def test_how_many_requests_a_call_takes():
    """2^20 - 1, as the header says: the next one's workgroups would be 2^32 threads."""
    from spy_amd import _lib as H
    from tests.test_serving_more_args import verify
    assert verify(n_seq=1 << 20) == H.EINVAL
    assert verify(n_seq=(1 << 20) - 1, room=1 << 20) == H.ENOSPACE
    assert "n_seq below 2^20" in open(os.path.join(ROOT, "include", "spy_hip.h")).read()

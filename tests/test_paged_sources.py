"""What the results of attention over pages cannot show: how often its kernels ask for what they need."""
import os
import re
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_chunks_ask_once_for_each_piece_of_a_tile(tmp_path):
    """A wave requests 16 bytes per lane to LDS: hd / 32 times for K and as often for V^T of a tile, in the three places that do (the first tile, a tile beside the
    products, a tile of a wave without rows)."""
    flags = re.search(r"^HIPFLAGS \?= ((?:.*\\\n)*.*)$", open(os.path.join(ROOT, "spy_amd", "csrc", "Makefile")).read(), re.M).group(1)
    flags = [f for f in flags.replace("\\\n", " ").replace("$(ARCH)", "gfx950").replace("$(PRELOAD)", "").split() if f != "-Wall"]
    out = str(tmp_path / "attn.s")
    subprocess.run([shutil.which("hipcc") or "/opt/rocm/bin/hipcc"] + flags + ["-w", "--cuda-device-only", "-S", "-o", out, os.path.join(ROOT, "spy_amd", "csrc", "paged_attn.hip")],
                   check=True, capture_output=True, timeout=300)
    asked, kernel = {}, None
    for line in open(out):
        name = re.match(r"(_Z\w+):", line)
        if name:
            kernel = re.match(r"_Z17attn_mixed_kernelILi(\d+)ELb(\d)", name.group(1))
        if kernel and "global_load_lds_dwordx4" in line:
            asked[kernel.groups()] = asked.get(kernel.groups(), 0) + 1
    assert asked == {(str(hd), str(f32)): 3 * 2 * hd // 32 for hd in (64, 128, 256) for f32 in (0, 1)}

"""What the native sources are compiled with, and what the library as built must not hold.  CPU only: make's dry runs and the
disassembly of the code built here."""
import os
import re
import shutil
import subprocess
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "esc_gnn_amd", "csrc")
NOPK = "-Xclang -target-feature -Xclang -packed-fp32-ops"


@pytest.mark.parametrize("target", ["all", "stamps", "both_exp", "escat_route.s"])
@pytest.mark.parametrize("how", ["plain", "command line", "environment"])
def test_every_compile_line_turns_packed_fp32_off(target, how):
    """also where CFLAGS are the caller's"""
    env = {k: v for k, v in os.environ.items() if k not in ("CFLAGS", "MAKEFLAGS", "MFLAGS")}
    cmd = ["make", "-n", "-B", "-C", CSRC, target]
    flags = "-O1 -g -std=c++17 -fPIC --offload-arch=gfx950"
    if how == "command line":
        cmd.append("CFLAGS=" + flags)
    if how == "environment":
        env["CFLAGS"] = flags
    r = subprocess.run(cmd, env=env, capture_output=True, text=True, check=True)
    lines = [l for l in r.stdout.splitlines() if ".hip" in l and "hipcc" in l]
    assert len(lines) >= (20 if target in ("all", "stamps") else 1)
    assert all(NOPK in l for l in lines)
    if how != "plain" and target != "escat_route.s":
        assert all("-O1 -g" in l for l in lines)

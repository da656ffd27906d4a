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


# ------------------------------------------------------------------ the library as built
LLVM = "/opt/rocm/llvm/bin"
PACKED = re.compile(r"\s*v_pk_(?:add|mul|fma)_f32\b")
SHIFT = re.compile(r"\s*v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S* v\[\d+:\d+\], v(\d+),")
LABEL = re.compile(r"[0-9a-f]+ <([^>]+)>:$")


def scan(lines, registers):
    """what a disassembly must not hold.  registers: kernel -> VGPRs it has.  A 64-bit shift whose amount lies in the last VGPR of a
    kernel's allocation (of 8 at a time) has shifted by another amount on this card; code outside the kernels may run under each of them"""
    ends = {k: {(n + 7) // 8 * 8 - 1} for k, n in registers.items()}
    every = set().union(*ends.values())
    name, packed, shifts, seen = "", [], [], 0
    for l in lines:
        m = LABEL.match(l)
        if m:
            name = m.group(1)
        elif PACKED.match(l):
            packed.append((name, l.strip()))
        else:
            m = SHIFT.match(l)
            if m:
                seen += 1
                if int(m.group(1)) in ends.get(name, every):
                    shifts.append((name, l.strip()))
    return packed, shifts, seen


def test_the_scan_finds_what_it_looks_for():
    text = ["0000000000001900 <kern>:", "\tv_pk_fma_f32 v[0:1], v[2:3], v[4:5], v[6:7]   // 0", "\tv_lshrrev_b64 v[16:17], v15, v[10:11]  // 1",
            "\tv_lshlrev_b64 v[16:17], v14, 1  // 2", "\tv_lshlrev_b64 v[16:17], 3, v[15:16]  // 3", "\tv_pk_fma_f16 v0, v1, v2, v3  // 4",
            "0000000000002900 <helper>:", "\tv_ashrrev_i64 v[2:3], v23, v[4:5]  // 5"]
    packed, shifts, seen = scan(text, {"kern": 16, "other": 24})
    assert [n for n, _ in packed] == ["kern"] and [n for n, _ in shifts] == ["kern", "helper"] and seen == 3
    assert [n for n, _ in scan(text, {"kern": 9})[1]] == ["kern"]                    # (it gets 16)
    assert [n for n, _ in scan(text, {"kern": 17})[1]] == ["helper"] and scan(text, {"kern": 25})[1] == []


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-objdump")), reason="no llvm-objdump")
def test_the_library_as_built(tmp_path):
    """no packed fp32 instruction, no 64-bit shift by the last VGPR, in any kernel"""
    from concurrent.futures import ThreadPoolExecutor
    shutil.copy(os.path.join(ROOT, "esc_gnn_amd", "libescat.so"), tmp_path / "lib.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    objects = sorted(p for p in tmp_path.iterdir() if "gfx950" in p.name)
    units = [u for u in os.listdir(CSRC) if u.endswith(".hip")]
    assert len(objects) >= len(units) - 1                                           # (a unit of host code alone may have none)

    def one(path):
        notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        registers, name = {}, None
        for l in notes.splitlines():
            m = re.match(r"\s*\.symbol:\s+'?([^\s']+)\.kd'?$", l)
            if m:
                name = m.group(1)
            m = re.match(r"\s*\.vgpr_count:\s+(\d+)", l)
            if m:
                registers[name] = int(m.group(1))
        with subprocess.Popen([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", str(path)], stdout=subprocess.PIPE, text=True) as p:
            found = scan((l.rstrip("\n") for l in p.stdout), registers)
        assert p.returncode == 0
        return found, len(registers)
    with ThreadPoolExecutor(8) as ex:
        results = list(ex.map(one, objects))
    assert sum(k for _, k in results) > 300 and sum(f[2] for f, _ in results) > 100          # the scan saw kernels and shifts
    for (packed, shifts, _), _ in results:
        assert not packed, packed[:5]
        assert not shifts, shifts[:5]

"""CPU check of the compiled 256 x 256 product of the linear: its MFMAs, their order and their waits are written down in
assembly that the compiler does not see into, so what it placed around them is verified on the gfx950 assembly:
no vector instruction writes an operand of an MFMA less than two wait states before it, nothing but MFMAs touches an
accumulator until they have retired, nothing spills.  hipcc cross-compiles without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ppl.pmx_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-Xclang",
         "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S"]


def registers(text):
    out = set()
    for kind, lo, hi, one_kind, one in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        if kind:
            out |= {(kind, i) for i in range(int(lo), int(hi) + 1)}
        else:
            out.add((one_kind, int(one)))
    return out


def findings(body):
    """Of one kernel's instructions."""
    ins = [line.split(";")[0].strip() for line in body.split("\n")]
    labels, kept = {}, []
    for line in ins:
        if line.endswith(":"):
            labels[line[:-1]] = len(kept)
        elif line and not line.startswith("."):
            kept.append(line)
    ins = kept
    at = [i for i, line in enumerate(ins) if line.startswith("v_mfma")]
    found = []
    for i in at:
        operands = set().union(*(registers(t) for t in ins[i].split(None, 1)[1].split(",")[1:]))
        states, j = 0, i - 1
        while j >= 0 and states < 2:
            before = ins[j]
            if before.startswith("s_nop"):
                states += int(before.split()[1]) + 1
            else:
                if before.startswith("v_") and not before.startswith("v_mfma") and \
                        registers(before.split(None, 1)[1].split(",")[0]) & operands:
                    found.append("{} just before {}".format(before, ins[i]))
                states += 1
            j -= 1
    for line in ins[at[0]:at[-1]]:
        if not line.startswith("v_mfma") and any(k == "a" for k, _ in registers(line)):
            found.append("accumulator touched: " + line)
    states, i = 0, at[-1] + 1                       # past the loop's end
    while i < len(ins) and not any(k == "a" for k, _ in registers(ins[i])):
        line = ins[i]
        states += int(line.split()[1]) + 1 if line.startswith("s_nop") else 1
        i = labels[line.split()[1]] if line.startswith("s_branch") else i + 1
    if states < 12:
        found.append("{} wait states before the accumulators are read".format(states))
    found += ["spill: " + line for line in ins if line.startswith("scratch_")]
    found += ["packed fp32: " + line for line in ins if re.match(r"v_pk_(add|mul|fma)_f32", line)]
    return len(at), found


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_large_product_assembly_is_hazard_free(tmp_path):
    out = tmp_path / "linear_gemm.s"
    r = subprocess.run([HIPCC, *FLAGS, os.path.join(CSRC, "linear_gemm.hip"), "-o", str(out)], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    kernels = re.findall(r"^(_ZN\S*linear_gemm_wide_kernel\S*):[^\n]*\n(.*?)^\.Lfunc_end", out.read_text(), re.S | re.M)
    assert len(kernels) == 8                        # two types, four layouts
    for name, body in kernels:
        assert findings(body) == (128, []), name
        # what the counted waits count: 16 loads per k-tile, straight to LDS, and no other access to memory
        loop = [line.strip() for line in body[body.index("v_mfma"):body.rindex("v_mfma")].split("\n")]
        loads = [line for line in loop if line.startswith(("buffer_", "global_", "flat_"))]
        assert len(loads) == 16 and all("lds" in line for line in loads), name


def test_the_check_finds_what_it_looks_for():
    good = ["v_mfma_f32_16x16x32_f16 a[0:3], v[0:3], v[4:7], a[0:3]"] * 4 + ["s_nop 11", "v_accvgpr_read_b32 v1, a0"]
    assert findings("\n".join(good)) == (4, [])
    assert findings("\n".join(good[:4] + ["s_nop 9"] + good[5:]))[1] == ["10 wait states before the accumulators are read"]
    for line, what in (("v_mov_b32_e32 v5, v9", "just before"), ("v_accvgpr_write_b32 a9, v1", "accumulator touched"),
                       ("scratch_store_dword off, v1, s0", "spill"), ("v_pk_fma_f32 v[8:9], v[8:9], v[8:9], v[8:9]", "packed")):
        assert any(what in f for f in findings("\n".join(good[:2] + [line] + good[2:]))[1]), line

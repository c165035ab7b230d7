#!/usr/bin/env python3
"""Compiles a source with the compiler's resource-usage remarks and fails if one of its matrix kernels spills registers in a
variant of the usual shapes: the main loop of those variants sits at the edge of the scalar and vector register budgets, and a
variant that spills a few scalar registers runs 1.5-2.5 % slower.  The general-shape variants (grouped GEMM: last template
argument true; gate_up_kernel: rows of x that a wave does not keep) may spill scalar registers; no variant may spill vector
registers.  Usage: make -C csrc check-spills"""
import re
import subprocess
import sys

KERNELS = ("grouped_gemm_mfma_kernel", "i8_gemm_kernel", "fp4_tile_kernel", "fp4_few_rows_kernel", "fp4_f32_kernel", "gate_up_kernel",
           "gate_up_fp4_kernel", "down_kernel", "swiglu8_fwd_kernel", "swiglu8_bwd_kernel")
GENERAL = (r"Lb1EEEv13MoeGemmParams$", r"gate_up_kernelI\d+Num\w+?Li\d+ELb0E")

cmd = sys.argv[1:]
out = subprocess.run(cmd, capture_output=True, text=True)
text = out.stdout + out.stderr
name, bad, seen = None, [], 0
for line in text.splitlines():
    m = re.search(r"Function Name: (\S+)", line)
    if m:
        name = m.group(1)
        continue
    m = re.search(r"(SGPRs|VGPRs) Spill: (\d+)", line)
    if m and name and any(k in name for k in KERNELS):
        seen += 1
        general = any(re.search(g, name) for g in GENERAL)
        if int(m.group(2)) > 0 and (m.group(1) == "VGPRs" or not general):
            bad.append(f"{name}: {m.group(1)} spill {m.group(2)}")
if out.returncode != 0 or seen == 0:
    sys.stderr.write(text[-2000:])
    sys.exit("check-spills: the compile failed or printed no resource usage")
if bad:
    sys.exit("check-spills: register spills in hot kernel variants:\n  " + "\n  ".join(bad))
print(f"check-spills: {seen // 2} kernel variants, no spills in the variants of the usual shapes")

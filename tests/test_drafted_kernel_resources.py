"""Registers and LDS of the drafted step's kernels, from the compiler's own report
on this repository's sources (no GPU needed)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "qwen35-cpu_amd")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def _report(source, tmp_path):
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++20", "-fPIC", "-Xclang", "-target-feature",
                        "-Xclang", "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"),
                        "-I" + os.path.join(PKG, "csrc"), "-Rpass-analysis=kernel-resource-usage", "-c",
                        os.path.join(PKG, "csrc", source), "-o", str(tmp_path / "out.o")],
                       stderr=subprocess.PIPE, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    out = {}
    for part in r.stderr.split("Function Name: ")[1:]:
        out[part.split()[0]] = {k: int(re.search(re.escape(k) + r"[^:\n]*: (\d+)", part).group(1))
                                for k in ("VGPRs", "VGPRs Spill", "ScratchSize", "LDS Size")}
    return out


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_tree_attention_keeps_its_registers(tmp_path):
    """Two wavefronts to a SIMD (256 registers) and nothing spilled in any head
    dimension; one workgroup's LDS fits a CU."""
    kernels = {k: v for k, v in _report("tree.hip", tmp_path).items() if "tree_" in k}
    assert len([k for k in kernels if "tree_attention_kernel" in k]) == 3
    for name, use in kernels.items():
        assert use["VGPRs"] <= 256 and use["VGPRs Spill"] == 0 and use["ScratchSize"] == 0, (name, use)
        assert use["LDS Size"] <= 160 * 1024, (name, use)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_sampling_keeps_its_registers(tmp_path):
    """The slices, which the stream of logits runs through, spill nothing. The
    pick's scratch is its call of the seldom settling of many keys: no more than
    the 444 bytes a lane it was measured with."""
    kernels = _report("draw.hip", tmp_path)
    slices = [v for k, v in kernels.items() if "draw_slices_kernel" in k]
    pick = [v for k, v in kernels.items() if "draw_pick_kernel" in k]
    assert len(slices) == 1 and len(pick) == 1
    assert slices[0]["VGPRs Spill"] == 0 and slices[0]["ScratchSize"] == 0, slices
    assert pick[0]["VGPRs"] <= 128 and pick[0]["VGPRs Spill"] <= 10 and pick[0]["ScratchSize"] <= 448, pick

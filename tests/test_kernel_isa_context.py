"""Static checks on the generated gfx950 code of the cache, attention and log probability kernels (no GPU needed).

Their tiles live in registers: no kernel may spill vector registers or touch scratch memory.  (Some attention kernels reserve a few
bytes of it beside scalar registers that are kept in lanes of vector registers; no instruction reads or writes them.)
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "nntrain_amd" / "csrc"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.parametrize("source,kernels", [("attention_kernels.hip", 28), ("log_prob_kernels.hip", 4), ("kv_cache_kernels.hip", 8)])
def test_no_spilled_vector_registers(tmp_path, source, kernels):
    if not Path(HIPCC).exists():
        pytest.skip("hipcc is not installed")
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-S", "--cuda-device-only", "-o", str(out), str(CSRC / source)], check=True, capture_output=True, cwd=CSRC)
    text = out.read_text()
    spills = [int(n) for n in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
    private = [int(n) for n in re.findall(r"\.private_segment_fixed_size:\s+(\d+)", text)]
    assert len(spills) == kernels and not any(spills)
    assert len(private) == kernels and max(private) <= 64
    assert not re.search(r"\bscratch_(load|store)", text)
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)          # (packed FP32 is switched off)

"""CPU check of the compiler's report on the serving kernels (hipcc cross-compiles for
gfx950 here): no kernel keeps values in scratch memory, and every workgroup's LDS
leaves room for the workgroups per CU that the estimate of its time counts on."""
import os
import re
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "cuda_fused_attention_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.parametrize("source", ["fa_serving.hip", "fa_paged.hip"])
def test_serving_kernels_do_not_spill(tmp_path, source):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    sys.path.insert(0, REPO)
    from cuda_fused_attention_amd import _build

    r = subprocess.run([HIPCC, *_build.HIP_FLAGS, f"-I{CSRC}", "--cuda-device-only", "-S", "-x", "hip",
                        "-Rpass-analysis=kernel-resource-usage", os.path.join(CSRC, source), "-o", str(tmp_path / "out.s")],
                       check=True, capture_output=True, text=True)
    names = re.findall(r"Function Name: (\S+)", r.stderr)
    scratch = [int(x) for x in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)]
    lds = [int(x) for x in re.findall(r"LDS Size \[bytes/block\]: (\d+)", r.stderr)]
    vgprs = [int(a) + int(b) for a, b in zip(re.findall(r" VGPRs: (\d+)", r.stderr), re.findall(r" AGPRs: (\d+)", r.stderr))]
    assert len(names) == len(scratch) == len(lds) == len(vgprs) > 0
    assert not any(scratch), dict(zip(names, scratch))
    # (head_dim, waves, groups): workgroups per CU
    per_cu = {(64, 2, 1): 6, (64, 4, 1): 3, (64, 2, 2): 3, (128, 2, 1): 3, (128, 4, 1): 2, (128, 8, 1): 1, (128, 2, 2): 2}
    seen = set()
    for name, bytes_, regs in zip(names, lds, vgprs):
        m = re.search(r"serving_attention_kernelIDF16[b_]Li(\d+)ELi(\d+)ELi(\d+)ELb[01]E", name)
        if not m:
            continue
        dim, waves, groups = (int(x) for x in m.groups())
        n = per_cu[(dim, waves, groups)]
        seen.add((dim, waves, groups))
        assert n * bytes_ <= 160 * 1024, (name, bytes_)
        # 512 registers per lane of a SIMD in pieces of 8; a CU's waves spread over four SIMDs
        per_simd = -(-n * waves * groups // 4)
        assert per_simd * (-(-regs // 8) * 8) <= 512, (name, regs)
    if source == "fa_serving.hip":
        assert seen == set(per_cu)

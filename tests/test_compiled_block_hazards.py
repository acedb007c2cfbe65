"""The hazards of test_compiled_hazards.py, checked in the compiled kernels of the cache
operators."""
import os
import re
import shutil
import subprocess

import pytest
from test_compiled_hazards import CSRC, HIPCC, ROOT, short_mfma_reads, unwaited_lds_results


def test_compiled_kernels_wait_for_mfma_and_lds_results(tmp_path):
    if not shutil.which(HIPCC) and not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm",
                    "-amdgpu-kernarg-preload-count=16", f"-I{os.path.join(ROOT, 'include')}",
                    f"-I{CSRC}", "--offload-device-only", "-S",
                    os.path.join(CSRC, "pd_blocks.hip"), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    text = out.read_text()
    bad, mfmas = {}, 0
    for name in sorted(set(re.findall(r"^(_Z\w*kernel\w*):", text, re.M))):
        body = text[text.index(name + ":"):text.index(".Lfunc_end", text.index(name + ":"))]
        mfmas += body.count("v_mfma")
        found = short_mfma_reads(body.splitlines()) + unwaited_lds_results(body.splitlines())
        if found:
            bad[name] = found[:3]
    assert mfmas >= 200
    assert not bad, bad

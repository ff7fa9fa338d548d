"""CPU check of the serving kernels' register budgets, as tests/test_kernel_resources.py checks the other kernels': what lets a
workgroup's waves be on a CU together, and no scratch."""
import os
import re
import shutil

import pytest

from tests.test_kernel_resources import resources
from transformer_amd import build as B

BUDGETS = {
    # file: [(kernel name regex, max VGPR + AGPR per lane, kernels)]
    "paged_append.hip": [(r"append", 128, 2), (r"read", 128, 2)],
    # 6 waves of a workgroup; 12, or 14 and 16 with a shared key and d_latent 384 and 512; 8
    "paged_decode.hip": [(r"paged_decode16_kernel", 256, 10), (r"paged_decode4_kernelILi(384|512)ELb1E", 128, 2),
                         (r"paged_decode4_kernel", 168, 12), (r"paged_merge_kernel", 128, 22)],
    "sample.hip": [(r"sample_kernel", 128, 6)],
}


@pytest.mark.skipif(not shutil.which(B.HIPCC) and not os.path.exists(B.HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src", sorted(BUDGETS))
def test_kernels_fit_their_register_budgets(src):
    res = resources(os.path.join(B.CSRC, src))
    for pattern, most, count in BUDGETS[src]:
        found = [k for k in res if re.search(pattern, k)]
        assert len(found) == count, f"{src}: {len(found)} kernels match {pattern}"
        for k in found:
            assert res[k]["ScratchSize"] == 0, f"{k} spills {res[k]['ScratchSize']} bytes per lane"
            assert res[k]["VGPRs"] + res[k]["AGPRs"] <= most, f"{k} uses {res[k]} registers per lane, budget {most}"

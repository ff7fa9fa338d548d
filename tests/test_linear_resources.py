"""CPU check of the linear layers' register budgets, as tests/test_kernel_resources.py checks the other kernels': two waves a
SIMD for the tiles (256 registers a lane, the accumulators' among them), and no scratch in any kernel."""
import os
import re
import shutil

import pytest

from tests.test_kernel_resources import resources
from transformer_amd import build as B

BUDGETS = {
    # file: [(kernel name regex, max VGPR + AGPR per lane, kernels)]
    "linear_act.hip": [(r"linear_act_kernel", 256, 15), (r"linear_act_finish_kernel", 256, 15),
                       (r"linear_act_rows_kernel", 256, 24)],
    "gated_linear.hip": [(r"gated_linear_kernel", 256, 9), (r"gated_linear_finish_kernel", 256, 9), (r"gated_linear_bwd_kernel", 256, 3),
                         (r"gated_linear_rows_kernel", 256, 18)],
    "act_grad.hip": [(r"act_grad_kernel", 128, 4), (r"act_grad_sum_kernel", 128, 1)],
    "grad_norm.hip": [(r"grad_norm_kernel", 128, 2), (r"grad_scale_kernel", 128, 2)],
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

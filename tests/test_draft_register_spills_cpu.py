"""Kernels of drafted trees and of the norm with rotation that are to keep within their registers, and what the others spill at most."""

import os
import re

import pytest

from test_register_spills_cpu import NVCC, _spilled


@pytest.mark.parametrize("source,kernels,most", [
    # fp32 rows and rows of drafts; the gradient kernel; forward in bf16 and fp32
    ("draft.cu", {r"verify_drafts_kernelI(f|.*Lb1E)": 4, r"draft_tree_kernel": 1}, {r"verify_drafts_kernelI.*(half|bfloat16)Lb0E": (84, 64)}),
    ("qknorm.cu", {r"qk_norm_rope_bwd_kernel": 6, r"qk_norm_rope_kernelI(f|13__nv_bfloat16)": 4, r"qk_norm_weights_kernel": 3},
     {r"qk_norm_rope_kernelI6__half": (12, 12)}),
    ("paged_keep.cu", {}, {r"keep_path_kernel": (96, 116)}),
])
def test_spills(source, kernels, most, tmp_path):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    spilled = _spilled(source, tmp_path)
    for part, count in kernels.items():
        mine = {k: v for k, v in spilled.items() if re.search(part, k)}
        assert len(mine) == count and {k: v for k, v in mine.items() if v != (0, 0)} == {}
    for part, (stores, loads) in most.items():
        mine = [v for k, v in spilled.items() if re.search(part, k)]
        assert len(mine) == 2 and all(a <= stores and b <= loads for a, b in mine)

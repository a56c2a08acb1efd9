"""Barriers and tensor-memory loads are instructions that all lanes of a warp have to execute together: in the kernels of the layer
of experts a __syncwarp() stands in front of each, whatever lanes did before."""
import os
import re

import pytest

from cutlass_b200.build import CSRC

ALIGNED = re.compile(r"\b(cluster_arrive|cluster_wait|tmem_ld_32x32b_x32|i8_tmem_ld_x16)\(|\"bar\.sync ")
# what may stand between: nothing that lanes do differently
SAME_FOR_ALL = re.compile(r"^(//.*|uint32_t v\[\w+\];|ptx::tc_fence_before\(\);|if constexpr \(.*|else .*|\}?)$")


@pytest.mark.parametrize("name", ["int8_kernel.cuh", "route_kernel.cuh"])
def test_a_warp_is_together_before_it(name):
    lines = [line.strip() for line in open(os.path.join(CSRC, name))]
    seen = 0
    for i, line in enumerate(lines):
        if not ALIGNED.search(line) or line.startswith(("__device__", "static __device__", "//")):
            continue
        seen += 1
        j = i - 1
        while SAME_FOR_ALL.match(lines[j]):
            j -= 1
        assert lines[j].startswith(("__syncwarp();", "ptx::cluster_arrive();")), f"{name}:{i + 1}: {line}  (behind: {lines[j]})"
    assert seen >= 3

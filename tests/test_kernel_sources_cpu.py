"""What the kernels' sources have to say, read as text: no GPU needed."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_aligned_cluster_barriers_bring_their_warps_together():
    """barrier.cluster.*.aligned wants all threads of a warp at the instruction.  Nothing but a __syncwarp() in the same function promises
    that behind a branch or a loop, and no file issues the instruction by another way than those functions."""
    found = 0
    for path in glob.glob(os.path.join(ROOT, "reference_model_b200", "csrc", "*.cu*")):
        text = open(path).read()
        for function in re.split(r"\n(?=__device__|template|__global__)", text):
            first = function.find("barrier.cluster.")
            if first >= 0 and ".aligned" in function[first:first + 60]:
                assert os.path.basename(path) == "ptx_sm100.cuh", path
                assert 0 <= function.find("__syncwarp();") < first, function[:200]
                found += 1
    assert found == 3

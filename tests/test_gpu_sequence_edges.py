"""The sequence operators at the sizes and values where one of their kernels' forms begins or ends."""
import pytest
import torch

import sequence_edges as edges
import sequence_reference as ref
from test_gpu_sequence import BF16, F16, F32, TYPES, on_gpu, rand, scan_inputs, seq  # noqa: F401  (seq: fixture)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("dtype,c,groups", [(F32, 347823, 115941), (BF16, 594811, 84973), (F16, 594811, 84973)])
def test_group_norm_of_very_many_narrow_groups(seq, dtype, c, groups):
    # more column blocks than a block has groups; groups narrower than a vector
    x, w, b = rand(101, 1, 3, 1, c, dtype=dtype), rand(102, c, offset=1.0), rand(103, c)
    _, depth = edges.two_launch_depth(1, 3, c, groups, dtype)
    y, bound = edges.group_norm(x, groups, w, b, 1e-3, depth)
    ref.check(seq.group_norm(x.cuda(), groups, w.cuda(), b.cuda(), eps=1e-3), y, bound)

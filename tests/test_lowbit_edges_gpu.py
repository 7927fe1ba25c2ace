"""Tree attention and 4-bit products at the ends of their ranges, on the sm_100a kernels."""
import pytest
import torch

import lowbit_cases as cases
from kotodama_b200.ops import get_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_units_of_one_tile(fp8, hd):
    """A CTA of the 128-row kernel walks many units of one or two tiles, which one of its softmax groups has alone."""
    ops = get_ops("cuda")
    sizes, lens = cases.ragged(300, 140, 6, 12)
    cases.check_tree(ops, "cuda", 40, 2, hd, sizes, lens, fp8, torch.bfloat16, True, bound=400)
    ops.check_status()

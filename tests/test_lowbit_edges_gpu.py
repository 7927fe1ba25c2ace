"""Tree attention and 4-bit products at the ends of their ranges, on the sm_100a kernels."""
import pytest
import torch

import lowbit_cases as cases
import lowbit_edge_cases as edges
from kotodama_b200.ops import Int4Weight, get_ops
from kotodama_b200.ops.cuda import KernelError

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
HEADS = [4, 10, 32]                  # 12, 30 and 96 rows per KV head: one block of 16 rows, two, the kernel of 128 rows
BOUNDS = [None, 5000]                # a block of threads per unit, the line of tiles


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_units_of_one_tile(fp8, hd):
    """A CTA of the 128-row kernel walks many units of one or two tiles, which one of its softmax groups has alone."""
    ops = get_ops("cuda")
    sizes, lens = cases.ragged(300, 140, 6, 12)
    cases.check_tree(ops, "cuda", 40, 2, hd, sizes, lens, fp8, torch.bfloat16, True, bound=400)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_tiny_queries(fp8, dtype, hd, H, bound):
    edges.check_tree_tiny_queries(get_ops("cuda"), "cuda", fp8, dtype, hd, H, bound=bound)
    get_ops("cuda").check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_large_scores(fp8, dtype, hd, H, bound):
    for power in (12, 40, 100):
        edges.check_tree_large_scores(get_ops("cuda"), "cuda", fp8, dtype, hd, H, power, bound=bound)
    get_ops("cuda").check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_hidden_large_values(fp8, dtype, hd, H, bound):
    for power in (12, 17, 24, 40, 100):
        edges.check_tree_hidden_large(get_ops("cuda"), "cuda", fp8, dtype, hd, H, power, bound=bound)
    get_ops("cuda").check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_large_values_of_unlikely_tokens(fp8, dtype, hd, H, bound):
    for power, where in ((40, 3), (60, 3), (60, 200), (80, 250)):
        edges.check_tree_unlikely_large(get_ops("cuda"), "cuda", fp8, dtype, hd, H, power, where, bound=bound)
    get_ops("cuda").check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_values_of_every_size(hd, H, bound):
    edges.check_tree_wide_values(get_ops("cuda"), "cuda", hd, H, bound=bound)
    get_ops("cuda").check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H", [4, 64])
def test_page_lists_without_columns(fp8, dtype, H):
    ops = get_ops("cuda")
    edges.check_tree_without_pages(ops, "cuda", fp8, dtype, H)
    with pytest.raises(KernelError, match="status 6"):
        ops.check_status()
    ops.check_status()


# ------------------------------------------------------------------ 4-bit products
def test_products_added_to_no_output_are_refused():
    ops = get_ops("cuda")
    for M in (3, 40):
        x, w = cases.int4_case(M, 32, 64, 64, 0)
        w = Int4Weight(w.packed.cuda(), w.scales.cuda(), w.shape, w.group)
        with pytest.raises(KernelError, match="output"):
            ops.gemm_nt(x.cuda(), w, accumulate=True)


@pytest.mark.parametrize("case", edges.INT4_SCALE_CASES, ids=str)
@pytest.mark.parametrize("powers", edges.INT4_SCALE_POWERS)
def test_scales_of_any_size(case, powers):
    ops = get_ops("cuda")
    edges.check_int4_scales(ops, "cuda", torch.bfloat16, *case, *powers)
    ops.check_status()

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


@pytest.mark.parametrize("H,G,hd,sizes,lens,masked,seed,spread,bound", [
    (32, 4, 128, [5, 5], [548, 6], False, 540258, 6.0, 3000),
    (8, 8, 128, [11, 31, 19, 19, 15, 25, 27, 4, 32, 33, 23, 8, 16, 27, 31, 31, 31], [96, 32, 20, 50, 15, 25, 27, 5, 32, 69, 24, 70, 17, 27, 43, 40, 47], True, 267427, 1.0, None)])
def test_elements_without_the_large_tokens(H, G, hd, sizes, lens, masked, seed, spread, bound):
    """Elements in which a row's large tokens hold exact zeros live on its small ones."""
    cases.check_tree(get_ops("cuda"), "cuda", H, G, hd, sizes, lens, True, torch.bfloat16, masked, seed=seed, spread=spread, bound=bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H", [4, 64])
def test_page_lists_without_columns(fp8, dtype, H):
    ops = get_ops("cuda")
    edges.check_tree_without_pages(ops, "cuda", fp8, dtype, H)
    with pytest.raises(KernelError, match="status 6"):
        ops.check_status()
    ops.check_status()


@pytest.mark.parametrize("fp8", [False, True])
def test_a_single_head_or_row_has_any_stride(fp8):
    """Whatever stride a dimension of one has, the call is the dense one's, by the same kernel."""
    ops = get_ops("cuda")
    names = []
    launch = type(ops)._launch

    class Listen(type(ops)):
        def _launch(self, fn, *args):
            names.append(fn)
            return launch(self, fn, *args)

    for H, G, sizes, lens in ((1, 1, [3, 2], [40, 9]), (4, 2, [1], [33]), (1, 1, [1], [20])):
        c = cases.tree_case(H, G, 64, sizes, lens, fp8, torch.bfloat16, 4)
        t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        args = (cases._put(c["k"], "cuda"), cases._put(c["v"], "cuda"), c["table"].cuda(), t(c["lens"]), t(c["cu"]), max(sizes), max(lens), 0.125)
        q, N = c["q"].cuda(), sum(sizes)
        odd = torch.empty(4096, device="cuda", dtype=torch.bfloat16).as_strided(q.shape, (H * 64 if N > 1 else 1003, 64 if H > 1 else 13, 1))
        odd.copy_(q)
        out = torch.empty(4096, device="cuda", dtype=torch.bfloat16).as_strided((N, H * 64), (H * 64 if N > 1 else 1001, 1))
        want = ops.paged_tree_attention(q, *args)
        listen = object.__new__(Listen)
        listen.__dict__ = ops.__dict__
        assert torch.equal(listen.paged_tree_attention(odd, *args, None, out), want)
    assert names == ["kb_tree_attn"] * 3
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

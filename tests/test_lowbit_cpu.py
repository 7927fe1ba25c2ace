"""8-bit paged cache, tree attention and 4-bit weights: the plain PyTorch back end, and what is refused."""
import pytest
import torch

import lowbit_cases as cases
from kotodama_b200.ops import TORCH_OPS, Fp8Pages, Int4Weight


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", cases.APPEND_CASES, ids=str)
def test_append_is_exact(case, dtype):
    cases.check_append(TORCH_OPS, "cpu", dtype, *case)


def test_rows_that_are_not_finite():
    cases.check_append_not_finite(TORCH_OPS, "cpu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", cases.GATHER_CASES, ids=str)
def test_gather_is_exact(case, dtype):
    cases.check_gather(TORCH_OPS, "cpu", dtype, *case)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("case", cases.TREE_CASES + cases.TREE_PLAIN_CASES, ids=str)
def test_tree_attention(case, fp8):
    H, G, hd, sizes, lens, masked = case
    cases.check_tree(TORCH_OPS, "cpu", H, G, hd, sizes, lens, fp8, torch.float32, masked)


@pytest.mark.parametrize("fp8", [False, True])
def test_masked_tokens_that_are_not_finite(fp8):
    cases.check_tree_masked_not_finite(TORCH_OPS, "cpu", fp8, torch.float32)
    cases.check_tree_masked_not_finite(TORCH_OPS, "cpu", fp8, torch.float32, 64, 32, 2)


@pytest.mark.parametrize("fp8", [False, True])
def test_bad_sequences(fp8):
    cases.check_tree_bad_sequences(TORCH_OPS, "cpu", fp8)
    cases.check_tree_bad_sequences(TORCH_OPS, "cpu", fp8, 64, 2)


@pytest.mark.parametrize("case", cases.INT4_QUANT_CASES, ids=str)
def test_quantise_weights(case):
    cases.check_quant_int4(TORCH_OPS, "cpu", *case)


@pytest.mark.parametrize("case", cases.INT4_CASES, ids=str)
def test_products_with_4_bit_weights(case):
    M, N, K, group, stride = case
    cases.check_int4(TORCH_OPS, "cpu", torch.float32, M, N, K, group, stride=stride)


def test_operands_that_are_no_pages_or_weights():
    codes, exps = torch.zeros(2, 1, 16, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 1, 16, dtype=torch.uint8)
    for bad in ((codes, exps[:1]), (codes.float(), exps), (codes, exps.int()), (codes[0], exps[0])):
        with pytest.raises(ValueError):
            Fp8Pages(*bad)
    w = TORCH_OPS.quant_int4(torch.randn(20, 72), 64)
    for bad in ((w.packed, w.scales, (20, 72), 32), (w.packed[:1], w.scales, (20, 72), 64), (w.packed, w.scales.float(), (20, 72), 64),
                (w.packed, w.scales, (20, 70), 64), (w.packed.long(), w.scales, (20, 72), 64), (w.packed, w.scales, (33, 72), 64)):
        with pytest.raises(ValueError):
            Int4Weight(*bad)
    for shape, group in (((4, 12), 64), ((4, 64), 32)):
        with pytest.raises(ValueError):
            TORCH_OPS.quant_int4(torch.randn(*shape), group)


@pytest.mark.parametrize("per", [1, 4])
def test_the_merge_reads_what_the_workers_leave(per):
    """The line of tiles cut into parts, with units of all sizes against all numbers of blocks: every part has a tile, every unit is either
    finished or its partial results are exactly the ones that the merge reads."""
    import random
    rng = random.Random(per)
    for _ in range(4000):
        tiles = [rng.randint(1, rng.choice([2, 9, 60])) for _ in range(rng.randint(1, 7))]
        blocks = rng.randint(1, 25)
        parts = [p for p in cases.tile_parts(sum(tiles), blocks * per) if p[1]]
        assert parts[0][0] == 0 and parts[-1][1] == sum(tiles) and all(a < b for a, b in parts) and all(p[1] == q[0] for p, q in zip(parts, parts[1:]))
        assert cases.written_parts(tiles, blocks, per) == cases.merged_parts(tiles, blocks, per)

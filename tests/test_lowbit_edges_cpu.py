"""Tree attention and 4-bit products at the ends of their ranges: the plain PyTorch back end."""
import pytest
import torch

import lowbit_cases as cases
import lowbit_edge_cases as edges
from kotodama_b200.config import MODEL_PRESETS, ModelConfig
from kotodama_b200.models.llama import KotodamaModel
from kotodama_b200.ops import TORCH_OPS
from kotodama_b200.serve.engine import ServingEngine


@pytest.mark.parametrize("fp8", [False, True])
def test_tiny_queries(fp8):
    edges.check_tree_tiny_queries(TORCH_OPS, "cpu", fp8, torch.float32, 64, 4)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("power", [12, 40, 100])
def test_large_scores(fp8, power):
    edges.check_tree_large_scores(TORCH_OPS, "cpu", fp8, torch.float32, 64, 4, power)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("power", [12, 40, 100])
def test_hidden_large_values(fp8, power):
    edges.check_tree_hidden_large(TORCH_OPS, "cpu", fp8, torch.float32, 64, 4, power)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("power,where", [(40, 3), (60, 200), (80, 250)])
def test_large_values_of_unlikely_tokens(fp8, power, where):
    edges.check_tree_unlikely_large(TORCH_OPS, "cpu", fp8, torch.float32, 64, 4, power, where)


@pytest.mark.parametrize("fp8", [False, True])
def test_page_lists_without_columns(fp8):
    edges.check_tree_without_pages(TORCH_OPS, "cpu", fp8, torch.float32, 4)


# ------------------------------------------------------------------ 4-bit products
def test_products_added_to_no_output_are_refused():
    x, w = cases.int4_case(3, 32, 64, 64, 0)
    with pytest.raises(ValueError, match="output"):
        TORCH_OPS.gemm_nt(x.float(), w, accumulate=True)


@pytest.mark.parametrize("powers", edges.INT4_SCALE_POWERS)
def test_scales_of_any_size(powers):
    edges.check_int4_scales(TORCH_OPS, "cpu", torch.float32, 3, 40, 200, 128, *powers)


# ------------------------------------------------------------------ the engine
@pytest.mark.parametrize("low", [dict(kv_dtype="fp8"), dict(weight_bits=4)], ids=str)
def test_low_bits_on_cuda_are_for_bf16_passes(low):
    """The Llama family's kernels read and write bf16; refused before the GPU is asked for anything."""
    model = KotodamaModel(ModelConfig(**MODEL_PRESETS["smoke"])).eval()
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(ValueError, match="bf16"):
            ServingEngine(model, device="cuda", dtype=dtype, ops=TORCH_OPS, max_batch=1, max_ctx=32, **low)

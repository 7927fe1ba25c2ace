"""The serving engine with an 8-bit cache and 4-bit projections on the sm_100a kernels."""
import copy

import pytest
import torch

from kotodama_b200.config import MODEL_PRESETS, ModelConfig
from kotodama_b200.models.llama import KotodamaModel
from kotodama_b200.ops import TORCH_OPS, get_ops
from kotodama_b200.ops.reference import Int4Weight
from kotodama_b200.serve.engine import SamplingParams, ServingEngine

pytestmark = pytest.mark.gpu


class Plain:
    """The CUDA back end with the low-bit operators' plain forms in their place (on the same device)."""

    def __init__(self, ops):
        self._ops = ops

    def __getattr__(self, name):
        return getattr(self._ops, name)

    def gemm_nt(self, a, b, **kw):
        return (TORCH_OPS if isinstance(b, Int4Weight) else self._ops).gemm_nt(a, b, **kw)

    def qknorm_rope_fwd(self, qkv, *args, append=None, **kw):
        r = self._ops.qknorm_rope_fwd(qkv, *args, **kw)
        (n_q, n_kv, hd), (k_pages, v_pages, slots) = args[5:8], append
        TORCH_OPS.kv_append(r[0][:, n_q * hd:], qkv[:, (n_q + n_kv) * hd:], k_pages, v_pages, slots)
        return r

    def paged_tree_attention(self, *args, **kw):
        return TORCH_OPS.paged_tree_attention(*args, **kw)


def _run(model, prompts, graphs=True, wrap=None, **kw):
    ops = get_ops("cuda")
    eng = ServingEngine(copy.deepcopy(model), device="cuda", dtype=torch.bfloat16, max_batch=4, max_ctx=512, ops=wrap(ops) if wrap else ops,
                        kv_dtype="fp8", weight_bits=4, **kw)
    eng.use_cuda_graphs = graphs
    eng.logit_trace = []
    toks = eng.generate(prompts, SamplingParams(max_new_tokens=8, temperature=0.0))
    rows = {}
    for rids, lg in eng.logit_trace:
        for i, rid in enumerate(rids):
            rows.setdefault(rid, []).append(lg[i])
    ops.check_status()
    return toks, [rows[r] for r in sorted(rows)]


def test_engine_against_plain_forms_and_replayed():
    """Replayed decode graphs give the eager passes' numbers; both agree with the plain forms of the three operators in the same engine
    (every pass rounds to bf16; the bound is the one that the engine's bf16 passes keep against fp32 ones), until a near-tie of two
    tokens parts the histories."""
    torch.manual_seed(0)
    cfg = ModelConfig(**MODEL_PRESETS["smoke"], attn_res=True, attn_res_n_blocks=2)
    model = KotodamaModel(cfg)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (128, 40, 256, 1, 16)]
    graph_t, graph_l = _run(model, prompts)
    eager_t, eager_l = _run(model, prompts, graphs=False)
    assert graph_t == eager_t
    assert all(torch.equal(a, b) for x, y in zip(graph_l, eager_l) for a, b in zip(x, y))
    plain_t, plain_l = _run(model, prompts, graphs=False, wrap=Plain)
    compared = 0
    for gt, pt, gl, pl in zip(graph_t, plain_t, graph_l, plain_l):
        for i in range(8):
            assert float((gl[i] - pl[i]).norm() / pl[i].norm()) < 4e-2, i
            compared += 1
            if gt[i] != pt[i]:
                break
    assert compared >= 15


def test_32_bit_passes_take_the_cache_but_not_the_weights():
    torch.manual_seed(0)
    model = KotodamaModel(ModelConfig(**MODEL_PRESETS["smoke"]))
    with pytest.raises(ValueError, match="bf16"):
        ServingEngine(copy.deepcopy(model), device="cuda", dtype=torch.float32, max_batch=1, max_ctx=32, weight_bits=4)

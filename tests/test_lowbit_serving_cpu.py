"""The serving engine with an 8-bit cache and 4-bit projections, on the plain back end: what it computes, what it refuses."""
import copy

import pytest
import torch

import lisunex_cases
from kotodama_b200.config import MODEL_PRESETS, ModelConfig
from kotodama_b200.models.llama import KotodamaModel
from kotodama_b200.ops import Fp8Pages, TORCH_OPS
from kotodama_b200.ops.reference import TorchOps, quant_pow2_rows
from kotodama_b200.serve.engine import SamplingParams, ServingEngine


def _model():
    torch.manual_seed(0)
    cfg = ModelConfig(**MODEL_PRESETS["smoke"], attn_res=True, attn_res_n_blocks=2)
    return cfg, KotodamaModel(cfg).eval()


def _prompts(cfg):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (5, 17, 33, 16, 1)]


def _logits(eng, prompts, new=9):
    eng.logit_trace = []
    toks = eng.generate(prompts, SamplingParams(max_new_tokens=new, temperature=0.0))
    rows = {}
    for rids, lg in eng.logit_trace:
        for i, rid in enumerate(rids):
            rows.setdefault(rid, []).append(lg[i])
    return toks, [torch.stack(rows[r]) for r in sorted(rows)]


class RoundedCache(TorchOps):
    """The plain back end; what goes to the cache is rounded to what 8 bits hold."""

    def kv_append(self, k, v, k_pages, v_pages, slots):
        def held(t):
            hd = k_pages.shape[-1]
            codes, exps = quant_pow2_rows(t.reshape(t.shape[0], -1, hd))
            return torch.ldexp(codes.float(), exps.to(torch.int32)[..., None] - 127).reshape(t.shape[0], -1)
        super().kv_append(held(k), held(v), k_pages, v_pages, slots)


class DenseWeights(TorchOps):
    """The plain back end; projections keep the values that 4 bits hold, as dense matrices."""

    def decode_weight(self, w):
        return self.quant_int4(w).dense()


@pytest.mark.parametrize("cache", [None, "fp8"])
@pytest.mark.parametrize("bits", [16, 4])
def test_low_bit_engine_computes_with_what_is_held(cache, bits):
    """The engine's logits are those of a 16-bit engine whose cache rows and projections hold the rounded values (fp32 both: 2^-24 per
    operation over sums of at most a few thousand terms)."""
    cfg, model = _model()
    prompts = _prompts(cfg)
    kinds = ([RoundedCache] if cache else []) + ([DenseWeights] if bits == 4 else [])
    plain = type("Plain", tuple(kinds) or (TorchOps,), {})()
    want_t, want = _logits(ServingEngine(copy.deepcopy(model), ops=plain, max_batch=3, max_ctx=128), prompts)
    eng = ServingEngine(copy.deepcopy(model), ops=TORCH_OPS, max_batch=3, max_ctx=128, kv_dtype=cache, weight_bits=bits)
    got_t, got = _logits(eng, prompts)
    assert isinstance(eng.cache.k[0], Fp8Pages) == (cache == "fp8")
    for a, b in zip(got, want):
        assert float((a - b).abs().max()) <= 2.0 ** -11 * float(b.abs().max())
    assert got_t == want_t and len(eng.cache.free) == eng.cache.num_pages


def test_low_bits_change_the_result_by_their_rounding():
    """Against the engine with everything kept: near, but not the same (the options do something)."""
    cfg, model = _model()
    prompts = _prompts(cfg)
    _, want = _logits(ServingEngine(copy.deepcopy(model), max_batch=3, max_ctx=128), prompts, new=2)
    _, got = _logits(ServingEngine(copy.deepcopy(model), max_batch=3, max_ctx=128, kv_dtype="fp8", weight_bits=4), prompts, new=2)
    diff = max(float((a - b).norm() / b.norm()) for a, b in zip(got, want))
    assert 1e-4 < diff < 1.0


def test_refusals():
    cfg, model = _model()
    make = lambda **kw: ServingEngine(copy.deepcopy(model), max_batch=1, max_ctx=32, **kw)
    for kw in (dict(kv_dtype="int8"), dict(kv_dtype="bf16"), dict(weight_bits=8)):
        with pytest.raises(ValueError, match="kv_dtype"):
            make(**kw)
    for kw in (dict(kv_dtype="fp8"), dict(weight_bits=4)):
        with pytest.raises(ValueError, match="one GPU"):
            make(tp=object(), **kw)
        with pytest.raises(ValueError, match="Llama"):
            lisunex_cases.engine(lisunex_cases.weights(lisunex_cases.CONFIGS["one"]), "cpu", torch.float32, **kw)

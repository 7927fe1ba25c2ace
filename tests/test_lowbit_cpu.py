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


def test_products_of_overlapping_rows():
    cases.check_int4_overlapping_rows(TORCH_OPS, "cpu")


def test_quantise_weights_that_are_not_finite():
    cases.check_quant_int4_not_finite(TORCH_OPS, "cpu")


@pytest.fixture(scope="module")
def lib():
    try:
        from kotodama_b200.ops import _build
        return _build.load()
    except Exception as e:                                   # no compiler and no built library
        pytest.skip(f"native library unavailable: {e}")


def test_launchers_refuse_bad_arguments(lib):
    """Refused on the host, before any pointer is looked at."""
    import ctypes
    from kotodama_b200.ops.cuda import _ARGS, _CTYPE
    P = 4096

    def call(name, good, **bad):
        names = list(good)
        assert len(names) == len(_ARGS[name])
        f = getattr(lib, name)
        f.argtypes = [_CTYPE[c] for c in _ARGS[name]] + [ctypes.c_void_p, ctypes.c_void_p]
        status = bad.pop("status", P)
        return f(*[{**good, **bad}[n] for n in names], status, None)

    app = dict(k=P, v=P, ks=128, vs=128, kc=P, ke=P, vc=P, ve=P, slots=P, N=4, n_kv=2, hd=64, slots_n=64, type=0)
    for bad in (dict(N=0), dict(n_kv=0), dict(hd=24), dict(hd=272), dict(hd=0), dict(ks=4), dict(vs=129), dict(slots_n=-1), dict(type=2), dict(type=-1),
                dict(k=P + 8), dict(v=P + 2), dict(kc=P + 8), dict(vc=P + 1), dict(N=2 ** 30, n_kv=4)):
        assert call("kb_kv_append_fp8", app, **bad) == 5, bad
    gat = dict(kc=P, ke=P, vc=P, ve=P, G=2, hd=64, table=P, B=1, width=4, pages=8, seq=P, first=P, cu=P, segs=1, k=P, v=P, total=4, type=0)
    for bad in (dict(G=0), dict(hd=8), dict(hd=264), dict(B=0), dict(segs=0), dict(total=0), dict(type=3), dict(kc=P + 4), dict(k=P + 16), dict(v=P + 2)):
        assert call("kb_kv_gather_fp8", gat, **bad) == 5, bad
    tree = dict(q=P, qs=256, k=P, ke=None, v=P, ve=None, table=P, width=4, pages=8, lens=P, cu=None, B=2, masks=None, out=P, outs=256, N=2, H=4, n_kv=2, hd=64,
                max_q=1, max_ctx=64, scale=0.125, zero=0)
    for bad in (dict(ke=P), dict(ve=P), dict(hd=40), dict(hd=272), dict(H=3), dict(B=0), dict(N=0), dict(width=0), dict(pages=0), dict(type=2)):
        assert call("kb_tree_attn_plain", dict(tree, type=0), **bad) == 5, bad
    for bad in (dict(ke=P), dict(ve=P), dict(hd=80), dict(hd=32), dict(H=3), dict(B=0), dict(N=0), dict(width=0), dict(pages=0), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(qs=252), dict(outs=254), dict(q=P + 8), dict(k=P + 8), dict(out=P + 4), dict(work=P + 8), dict(floats=0),
                dict(max_q=0), dict(max_ctx=0), dict(pages=2 ** 31 - 1), dict(status=None)):
        assert call("kb_tree_attn", dict(tree, work=P, floats=2 ** 40), **bad) != 0, bad
    prod = dict(x=P, xs=128, packed=P, scales=P, c=None, cs=0, y=P, ys=64, M=4, N=64, K=128, group=128)
    for bad in (dict(M=0), dict(N=0), dict(K=0), dict(K=12), dict(group=32), dict(group=256), dict(xs=4), dict(x=P + 8), dict(packed=P + 4), dict(scales=P + 2)):
        assert call("kb_gemm_int4", prod, **bad) == 5, bad

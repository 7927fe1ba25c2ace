"""8-bit paged cache, tree attention and 4-bit weights on the sm_100a kernels."""
import math

import pytest
import torch

import lowbit_cases as cases
from kotodama_b200.ops import Fp8Pages, Int4Weight, get_ops
from kotodama_b200.ops.cuda import KernelError
from kotodama_b200.utils.guard import GuardRegions

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def guarded(f):
    ops = get_ops("cuda")
    with GuardRegions() as g:
        r = f(ops)
        torch.cuda.synchronize()
        assert not g.check()
    return r


# ------------------------------------------------------------------ 8-bit cache
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", cases.APPEND_CASES, ids=str)
def test_append_is_exact(case, dtype):
    guarded(lambda ops: cases.check_append(ops, "cuda", dtype, *case))
    get_ops("cuda").check_status()


def test_append_of_many_rows():
    """Enough rows for the form with several rows per lane group: the same bytes as the plain back end's."""
    from kotodama_b200.ops import TORCH_OPS
    ops = get_ops("cuda")
    n, n_kv, hd = 20011, 4, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    k = (torch.randn(n, n_kv * hd, device="cuda", generator=g) * torch.exp(torch.randn(n, 1, device="cuda", generator=g))).bfloat16()
    v = torch.randn(n, n_kv * hd, device="cuda", generator=g).bfloat16()
    slots = torch.randperm(n + 5, device="cuda", generator=g)[:n]
    slots[7::100] = -1
    got = [Fp8Pages.zeros(-(-(n + 5) // 16), n_kv, hd, "cuda") for _ in range(2)]
    want = [Fp8Pages.zeros(-(-(n + 5) // 16), n_kv, hd, "cuda") for _ in range(2)]
    ops.kv_append(k, v, *got, slots)
    TORCH_OPS.kv_append(k, v, *want, slots)
    for a, b in zip(got, want):
        assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.exps, b.exps)
    ops.check_status()


def test_rows_that_are_not_finite():
    cases.check_append_not_finite(get_ops("cuda"), "cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", cases.GATHER_CASES, ids=str)
def test_gather_is_exact(case, dtype):
    guarded(lambda ops: cases.check_gather(ops, "cuda", dtype, *case))
    get_ops("cuda").check_status()


def test_indices_out_of_range_are_reported():
    ops = get_ops("cuda")
    k = torch.randn(3, 64, device="cuda").bfloat16()
    kp, vp = Fp8Pages.zeros(2, 1, 64, "cuda"), Fp8Pages.zeros(2, 1, 64, "cuda")
    ops.kv_append(k, k, kp, vp, torch.tensor([0, 32, 5], device="cuda"))         # slot 32 of 32
    with pytest.raises(KernelError, match="status 6"):
        ops.check_status()
    t = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    x, _ = ops.kv_gather(kp, vp, t(0, 9)[None], t(0), t(0), t(0, 20), 20)          # page 9 of 2
    with pytest.raises(KernelError, match="status 6"):
        ops.check_status()
    assert bool((x[16:] == 0).all()) and bool((x[0] != 0).any())
    ops.check_status()


# ------------------------------------------------------------------ tree attention
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("case", cases.TREE_CASES + cases.TREE_PLAIN_CASES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bound", [None, 5000])          # how long contexts may be: a block of threads per unit, or the line of tiles and a merge
def test_tree_attention(case, fp8, dtype, bound):
    H, G, hd, sizes, lens, masked = case
    guarded(lambda ops: cases.check_tree(ops, "cuda", H, G, hd, sizes, lens, fp8, dtype, masked, bound=bound))
    get_ops("cuda").check_status()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,G,hd,n,most,rows", [(16, 4, 128, 45, 700, 3), (8, 2, 64, 200, 90, 1), (8, 1, 128, 30, 500, 20), (24, 2, 64, 21, 300, 64), (12, 4, 128, 25, 600, 13),
                                                (16, 4, 128, 45, 1500, 3), (8, 2, 64, 300, 90, 1), (4, 2, 64, 9, 2100, 4), (12, 4, 128, 25, 1700, 13),
                                                (12, 1, 128, 1, 9000, 64)])
@pytest.mark.parametrize("bound", [None, 9000])
def test_ragged_batches(H, G, hd, n, most, rows, fp8, bound):
    """Many sequences per block of threads and many blocks per sequence, empty ones among them, on both tensor-core kernels."""
    sizes, lens = cases.ragged(n, most, rows, 7 * n + rows) if n > 1 else ([rows], [most])
    guarded(lambda ops: cases.check_tree(ops, "cuda", H, G, hd, sizes, lens, fp8, torch.bfloat16, rows > 1, bound=bound))
    get_ops("cuda").check_status()


@pytest.mark.parametrize("fp8", [False, True])
def test_calls_that_take_the_plain_kernel(fp8):
    """More sequences than the tensor-core kernels' lists hold, scales that are not positive, query and output rows that are not aligned."""
    ops = get_ops("cuda")
    guarded(lambda ops: cases.check_tree(ops, "cuda", 2, 1, 64, [1] * 1100, [1 + i % 37 for i in range(1100)], fp8, torch.bfloat16, False))
    c = cases.tree_case(4, 2, 64, [3, 2], [40, 9], fp8, torch.bfloat16, 3)
    dense = [cases._dense(c[n]) for n in ("k", "v")]
    for scale in (0.0, -0.25):
        want, mass = cases.plain_tree(c["q"], *dense, c["table"].tolist(), c["lens"], c["cu"], scale, None)
        err = (cases.run_tree(ops, "cuda", c, None, scale).cpu().double().view(5, 4, 64) - want).abs()
        assert bool((err <= cases.tree_tolerance(c, want, mass, abs(scale))).all())
    good = cases.run_tree(ops, "cuda", c, None, 0.125)
    want, mass = cases.plain_tree(c["q"], *dense, c["table"].tolist(), c["lens"], c["cu"], 0.125, None)
    room = torch.zeros(5, 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    room[:, 1:] = c["q"].view(5, -1).cuda()
    odd = torch.zeros(5, 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    args = (cases._put(c["k"], "cuda"), cases._put(c["v"], "cuda"), c["table"].cuda(), t(c["lens"]), t(c["cu"]), 3, 40, 0.125)
    a = ops.paged_tree_attention(room[:, 1:].view(5, 4, 64), *args)
    ops.paged_tree_attention(c["q"].cuda(), *args, None, odd[:, 1:])
    for got in (good, a, odd[:, 1:]):
        assert bool(((got.cpu().double().view(5, 4, 64) - want).abs() <= cases.tree_tolerance(c, want, mass, 0.125)).all())
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", [4, 10, 32])                # 12, 30 and 96 rows per KV head: the three forms of the kernel
@pytest.mark.parametrize("bound", [None, 5000])
def test_masked_tokens_that_are_not_finite(fp8, dtype, hd, H, bound):
    cases.check_tree_masked_not_finite(get_ops("cuda"), "cuda", fp8, dtype, hd, H, 2, bound)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H", [4, 16, 64])
@pytest.mark.parametrize("empty", [0, 230])
def test_bad_sequences(fp8, H, empty):
    ops = get_ops("cuda")
    cases.check_tree_bad_sequences(ops, "cuda", fp8, H, 2, empty)
    with pytest.raises(KernelError, match="status 6"):
        ops.check_status()
    ops.check_status()


# ------------------------------------------------------------------ 4-bit weights
@pytest.mark.parametrize("case", cases.INT4_QUANT_CASES, ids=str)
def test_quantise_weights(case):
    cases.check_quant_int4(get_ops("cuda"), "cuda", *case)


@pytest.mark.parametrize("case", cases.INT4_CASES, ids=str)
def test_products_with_4_bit_weights(case):
    M, N, K, group, stride = case
    guarded(lambda ops: cases.check_int4(ops, "cuda", torch.bfloat16, M, N, K, group, stride=stride))
    get_ops("cuda").check_status()


@pytest.mark.parametrize("case", cases.INT4_LARGE_CASES, ids=str)
def test_products_in_every_form(case):
    M, N, K, group, stride = case
    guarded(lambda ops: cases.check_int4(ops, "cuda", torch.bfloat16, M, N, K, group, stride=stride))
    get_ops("cuda").check_status()


def test_products_of_overlapping_rows():
    guarded(lambda ops: cases.check_int4_overlapping_rows(ops, "cuda"))


def test_a_single_row_has_any_stride():
    ops = get_ops("cuda")
    x, w = cases.int4_case(1, 40, 136, 64, 3)
    w = Int4Weight(w.packed.cuda(), w.scales.cuda(), w.shape, w.group)
    row = x.cuda().as_strided((1, 136), (1001, 1))
    assert torch.equal(ops.gemm_nt(row, w), ops.gemm_nt(x.cuda(), w))
    got = []
    for k in (x[:, :128].cuda(), row[:, :128]):
        kp, vp = Fp8Pages.zeros(1, 2, 64, "cuda"), Fp8Pages.zeros(1, 2, 64, "cuda")
        ops.kv_append(k, k, kp, vp, torch.tensor([7], device="cuda"))
        got.append((kp.codes.view(torch.uint8), kp.exps, vp.codes.view(torch.uint8), vp.exps))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and bool(got[0][0][0, :, 7].any())


def test_quantise_weights_that_are_not_finite():
    cases.check_quant_int4_not_finite(get_ops("cuda"), "cuda")


def test_one_token_repeats_bit_by_bit():
    """A token's result does not depend on the tokens beside it within a form, nor on the run."""
    ops = get_ops("cuda")
    x, w = cases.int4_case(64, 272, 4160, 64, 2)
    x, w = x.cuda(), Int4Weight(w.packed.cuda(), w.scales.cuda(), w.shape, w.group)
    for rows in ((8, 1), (16, 9), (32, 17), (64, 33)):
        full = ops.gemm_nt(x[: rows[0]], w)
        assert torch.equal(ops.gemm_nt(x[: rows[0]], w), full) and torch.equal(ops.gemm_nt(x[: rows[1]], w), full[: rows[1]])


# ------------------------------------------------------------------ refusals
def test_refusals():
    ops = get_ops("cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    kp, vp = Fp8Pages.zeros(2, 1, 64, "cuda"), Fp8Pages.zeros(2, 1, 64, "cuda")
    k = torch.randn(3, 64, device="cuda").bfloat16()
    s = torch.arange(3, device="cuda")
    for call in (lambda: ops.kv_append(k.half(), k.half(), kp, vp, s), lambda: ops.kv_append(k, k, kp, vp, s.int()),
                 lambda: ops.kv_append(k, k, kp, vp, s[:2]), lambda: ops.kv_append(k[:, :32], k[:, :32], kp, vp, s),
                 lambda: ops.kv_append(k, k, kp, Fp8Pages.zeros(3, 1, 64, "cuda"), s), lambda: ops.kv_append(k, k, kp, vp.codes, s),
                 lambda: ops.kv_append(k, k.float(), kp, vp, s), lambda: ops.kv_append(k, k, kp, vp, s.cpu()),
                 lambda: ops.kv_gather(kp, vp, i32(0)[None], i32(0), i32(0), i32(0, 4), 4, torch.float16),
                 lambda: ops.kv_gather(kp, vp, i32(0)[None], i32(0), i32(0, 0), i32(0, 4), 4),
                 lambda: ops.kv_gather(kp, vp, i32(0)[None].long(), i32(0), i32(0), i32(0, 4), 4)):
        with pytest.raises(KernelError):
            call()
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    good = dict(q=q, k_pages=kp, v_pages=vp, page_table=i32(0)[None], ctx_lens=i32(8), cu_seqlens=i32(0, 2), max_q=2, max_ctx=8, scale=0.1)
    ops.paged_tree_attention(**good)
    page = torch.zeros(2, 1, 16, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (dict(q=q.half()), dict(q=q[:, :, :32]), dict(q=q.transpose(0, 1)), dict(v_pages=page), dict(k_pages=page), dict(ctx_lens=i32(8, 8)),
                dict(cu_seqlens=i32(0, 1, 2)), dict(cu_seqlens=torch.tensor([0, 2], device="cuda")), dict(masks=s[:1]), dict(masks=i32(1, 1)),
                dict(page_table=i32(0)), dict(out=q.view(2, 128).float()), dict(out=torch.empty(3, 128, device="cuda", dtype=torch.bfloat16)),
                dict(k_pages=page.float(), v_pages=page.float()), dict(ctx_lens=torch.tensor([8], dtype=torch.int32))):
        with pytest.raises(KernelError):
            ops.paged_tree_attention(**{**good, **bad})
    w = ops.quant_int4(torch.randn(32, 128, device="cuda"))
    x = torch.randn(2, 128, device="cuda").bfloat16()
    for call in (lambda: ops.gemm_nt(x.float(), w), lambda: ops.gemm_nt(x[:, :64], w), lambda: ops.gemm_nt(x.t().contiguous().t(), w),
                 lambda: ops.gemm_nt(torch.randn(2, 132, device="cuda").bfloat16()[:, :128], w), lambda: ops.gemm_nt(x, w, out=x),
                 lambda: ops.gemm_nt(x, w, residual=x), lambda: ops.gemm_nt(x, w, out=x[:, :32], residual=x[:, :32], accumulate=True),
                 lambda: ops.gemm_nt(x, Int4Weight(w.packed.cpu(), w.scales.cpu(), (32, 128), 128))):
        with pytest.raises(KernelError):
            call()
    ops.check_status()


# ------------------------------------------------------------------ together, captured, on another stream
def verification_step(ops, seed=0):
    """What a server does to verify drafted tokens: 4-bit projections, 8-bit append, tree attention over the cache, 4-bit output
    projection.  Returns a function that runs it on given inputs, and the inputs."""
    H, G, hd, D, sizes, lens = 8, 2, 128, 512, [4, 1, 7], [37, 200, 64]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    wqkv, wo = ops.quant_int4(rand((H + 2 * G) * hd, D) / 20), ops.quant_int4(rand(D, H * hd) / 20)
    kp, vp = Fp8Pages.zeros(24, G, hd, "cuda"), Fp8Pages.zeros(24, G, hd, "cuda")
    table = torch.arange(24, device="cuda", dtype=torch.int32).flip(0).view(3, 8)
    table = torch.cat([table, table.new_zeros(3, 6)], 1)
    table[1, :13] = torch.randperm(13, device="cuda", generator=g).int()                   # its own pages: 0 .. 12
    table[0, :8], table[2, :8] = torch.arange(13, 21, device="cuda").int(), torch.tensor([21, 22, 23, 13 + 4, 13 + 5, 0, 0, 0], device="cuda").int()
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 4, 5, 12], dtype=torch.int32, device="cuda")
    slot = lambda b, t: int(table[b, t // 16]) * 16 + t % 16
    old = [slot(b, t) for b in range(3) for t in range(lens[b] - sizes[b])]
    new = torch.tensor([slot(b, t) for b in range(3) for t in range(lens[b] - sizes[b], lens[b])], device="cuda")
    rows = rand(len(old), 2 * G * hd).bfloat16()
    ops.kv_append(rows[:, : G * hd], rows[:, G * hd:], kp, vp, torch.tensor(old, device="cuda"))
    masks = cases.signed(cases.tree_masks(sizes, 3)).cuda()

    def run(x):
        qkv = ops.gemm_nt(x, wqkv)
        ops.kv_append(qkv[:, H * hd:(H + G) * hd], qkv[:, (H + G) * hd:], kp, vp, new)
        o = ops.paged_tree_attention(qkv[:, : H * hd].view(-1, H, hd), kp, vp, table, ctx, cu, 8, 256, 1 / math.sqrt(hd), masks)
        return ops.gemm_nt(o, wo, residual=x)

    def plain(x):
        f = torch.float64
        dense = [w.dense().to(f) for w in (wqkv, wo)]
        qkv = (x.to(f) @ dense[0].t()).bfloat16()
        o, _ = cases.plain_tree(qkv[:, : H * hd].reshape(-1, H, hd).cpu(), cases.plain_values(kp), cases.plain_values(vp), table.tolist(), lens,
                                cu.tolist(), 1 / math.sqrt(hd), [m & (1 << 64) - 1 for m in masks.tolist()])
        return o.reshape(12, -1).bfloat16().to(f) @ dense[1].t().cpu() + x.to(f).cpu()

    return run, plain, [rand(12, D).bfloat16() for _ in range(3)]


@pytest.mark.parametrize("H", [4, 64])                   # 6 and 96 rows per KV head: both tensor-core kernels, with partial results and a merge
def test_long_contexts_captured_on_two_streams(H):
    ops = get_ops("cuda")
    runs = []
    for seed in (0, 1):
        c = cases.tree_case(H, 2, 64, [3, 1, 2], [3000, 40, 1700], True, torch.bfloat16, seed)
        t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        q, args = c["q"].cuda(), (cases._put(c["k"], "cuda"), cases._put(c["v"], "cuda"), c["table"].cuda(), t(c["lens"]), t(c["cu"]), 3, 3000, 0.125)
        runs.append((q, args, ops.paged_tree_attention(q, *args), ops.paged_tree_attention(-q, *args)))
    graphs = []
    for q, args, _, _ in runs:
        x, g = q.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g), ops.dependent_launch():
            y = ops.paged_tree_attention(x, *args)
        graphs.append((x, g, y))
    streams = [torch.cuda.Stream() for _ in runs]
    for sign in (1, -1, 1):
        for (x, g, _), (q, *_), st in zip(graphs, runs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                x.copy_(q * sign)
                g.replay()
        torch.cuda.synchronize()
        for (_, _, y), (_, _, plus, minus) in zip(graphs, runs):
            assert torch.equal(y, plus if sign > 0 else minus)
    ops.check_status()


def test_operands_on_the_host_are_refused():
    """They agree on their device, and it is not a GPU."""
    ops = get_ops("cuda")
    x, w = cases.int4_case(3, 32, 64, 64, 0)
    with pytest.raises(KernelError, match="GPU"):
        ops.gemm_nt(x, w)
    c = cases.tree_case(2, 1, 64, [1], [3], True, torch.bfloat16, 0)
    with pytest.raises(KernelError, match="GPU"):
        cases.run_tree(ops, "cpu", c, None, 0.125)
    with pytest.raises(KernelError, match="GPU"):
        ops.kv_append(x, x, Fp8Pages.zeros(1, 1, 64, "cpu"), Fp8Pages.zeros(1, 1, 64, "cpu"), torch.arange(3))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)
    with pytest.raises(KernelError, match="GPU"):
        ops.kv_gather(c["k"], c["v"], i32(0)[None], i32(0), i32(0), i32(0, 2), 2)


# ------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.parametrize("fp8", [False, True])
def test_caches_of_more_than_4_gigabytes(fp8):
    """The last pages of a large cache give what the pages of a small one give, bit by bit."""
    ops = get_ops("cuda")
    n_kv, hd, few, many = 8, 128, 6, 280_000 if fp8 else 140_000
    assert many * n_kv * 16 * hd * (1 if fp8 else 2) > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(6)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    k, v, slots = rand(90, n_kv * hd), rand(90, n_kv * hd), torch.randperm(few * 16, device="cuda", generator=g)[:90]
    table = torch.tensor([[3, 0, 5], [1, 4, 2]], dtype=torch.int32, device="cuda")
    t = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    got = []
    for pages in (few, many):
        at = pages - few
        new = (lambda: Fp8Pages.zeros(pages, n_kv, hd, "cuda")) if fp8 else (lambda: torch.zeros(pages, n_kv, 16, hd, device="cuda", dtype=torch.bfloat16))
        kp, vp = new(), new()
        ops.kv_append(k, v, kp, vp, slots + at * 16)
        out = list(ops.kv_gather(kp, vp, table + at, t(0, 1), t(2, 0), t(0, 44, 92), 92))
        for H in (16, 64):                            # 6, 24, 24 and 96 rows per KV head
            for rows in (3, 12):
                q = torch.randn(2 * rows, H, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(H + rows)).bfloat16()
                for bound in (48, 5000):              # a block of threads per unit, the line of tiles
                    out.append(ops.paged_tree_attention(q, kp, vp, table + at, t(46, 33), t(0, rows, 2 * rows), rows, bound, 0.09))
        got.append(out)
        del kp, vp
    assert all(torch.equal(a, b) for a, b in zip(*got)) and bool((got[0][0] != 0).any())
    ops.check_status()


def test_weights_of_more_than_4_gigabytes():
    """The last rows of a large weight give what they give alone."""
    ops = get_ops("cuda")
    N, K = 140_000, 65_536
    g = torch.Generator(device="cuda").manual_seed(8)
    packed = torch.randint(-2 ** 31, 2 ** 31 - 1, (N // 16, K // 64, 32, 4), device="cuda", dtype=torch.int32, generator=g)
    scales = (torch.rand(N // 16, K // 128, 8, 2, device="cuda", generator=g) + 0.5).bfloat16()
    assert packed.numel() * 4 > 1 << 32
    whole, end = Int4Weight(packed, scales, (N, K), 128), Int4Weight(packed[-8:].clone(), scales[-8:].clone(), (128, K), 128)
    for M in (4, 40):
        x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
        a, b = ops.gemm_nt(x, whole)[:, -128:].double(), ops.gemm_nt(x, end).double()
        # both round sums over 65536 inputs (fp32, in differing order) to bf16: half a step each
        assert float((a - b).norm() / b.norm()) < 2 * 2.0 ** -8
    ops.check_status()


def test_verification_step():
    ops = get_ops("cuda")
    run, plain, xs = verification_step(ops)
    for x in xs:
        got = run(x)
        want = plain(x)                              # reads the cache that run() wrote
        # roundings to bf16 on the way (projection, attention, output): half a step each of the magnitudes they weigh
        assert float((got.cpu().double() - want).norm() / want.norm()) < 3 * 2.0 ** -8
    ops.check_status()


def test_captured_and_replayed_on_another_stream():
    """The step in a graph: replayed on new inputs it gives what the eager call gives; two graphs replayed in turn do not disturb one another."""
    ops = get_ops("cuda")
    steps = [verification_step(ops, s) for s in (0, 1)]
    want = [[run(x).clone() for x in xs] for run, _, xs in steps]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [run(xs[0]) for run, _, xs in steps]
    side.synchronize()
    assert all(torch.equal(a, w[0]) for a, w in zip(again, want))
    graphs = []
    for run, _, xs in steps:
        x = xs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g), ops.dependent_launch():
            y = run(x)
        graphs.append((g, x, y))
    streams = [torch.cuda.Stream() for _ in steps]
    for i in range(3):
        for (g, x, _), (_, _, xs), st in zip(graphs, steps, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                x.copy_(xs[i])
                g.replay()
        torch.cuda.synchronize()
        for (_, _, y), w in zip(graphs, want):
            assert torch.equal(y, w[i])
    ops.check_status()

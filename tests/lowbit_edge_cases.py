"""Checks of tree attention and 4-bit products at the ends of their number ranges, on either back end, against the plain float64
forms of ``lowbit_cases``."""
import math

import torch

import lowbit_cases as cases
from kotodama_b200.ops import Fp8Pages, Int4Weight

F64 = torch.float64
PAGE = cases.PAGE


def compare_tree(ops, device, c, masks, scale, bound=None):
    """The call's rows against the plain form within the tolerance of the operator's roundings; returns them."""
    N, H, hd = c["q"].shape
    dense = [cases._dense(c[n]) for n in ("k", "v")]
    want, mass = cases.plain_tree(c["q"], *dense, c["table"].tolist(), c["lens"], c["cu"], scale, masks)
    got = cases.run_tree(ops, device, c, masks, scale, max_ctx=bound).cpu().to(F64).view(N, H, hd)
    tol = cases.tree_tolerance(c, want, mass, scale)
    err = (got - want).abs()
    assert bool((err <= tol).all()), (err / tol).nan_to_num(math.inf).amax((1, 2)).tolist()
    return got


# ------------------------------------------------------------------ query rows of zeros, scales that are nearly zero
def check_tree_tiny_queries(ops, device, fp8, dtype, hd, H, G=2, bound=None):
    """A row of zeros gives the mean of what it sees; rows of numbers near the types' lower end and scales near it nearly so.  Masks hide
    drafted tokens, and the contexts end inside a tile and inside a page."""
    masks = [1, 3, 5, 11, 21, 33, 1, 3]
    c = cases.tree_case(H, G, hd, [6, 2], [70, 33], fp8, dtype, 21)
    q = c["q"] = c["q"].clone()
    q[0] = 0.0
    q[2, 0] = 0.0
    q[2, 1:] *= 2.0 ** -126
    q[3] *= 2.0 ** -124
    q[4] *= 2.0 ** -110
    q[7] = 0.0
    compare_tree(ops, device, c, masks, 1.0 / math.sqrt(hd), bound)
    compare_tree(ops, device, c, None, 1.0 / math.sqrt(hd), bound)
    for scale in (1e-30, 1e-38, 1e-42):
        compare_tree(ops, device, c, masks, scale, bound)


# ------------------------------------------------------------------ scores of any size
def scaled_token(pages, page, off, power):
    """The pages with the numbers of one token (all heads) times 2^power."""
    if isinstance(pages, Fp8Pages):
        r = Fp8Pages(pages.codes.clone(), pages.exps.clone())
        r.exps[page, :, off] = (r.exps[page, :, off].int() + power).to(torch.uint8)
        return r
    r = pages.clone()
    r[page, :, off] = (r[page, :, off].to(F64) * 2.0 ** power).to(r.dtype)
    return r


def check_tree_large_scores(ops, device, fp8, dtype, hd, H, power, G=2, bound=None):
    """A drafted token whose keys are 2^power times the others' takes everything in the rows that see it with a positive score and nothing
    where the score is negative; the rows that do not see it do not notice, wherever it lies against the tiles."""
    masks = [1, 3, 5, 11, 21, 33, 1, 3]
    for lens in ([70, 33], [38, 131], [640, 130]):
        c = cases.tree_case(H, G, hd, [6, 2], lens, fp8, dtype, 31, spread=0.25)
        at = lens[0] - 6 + 1                                            # drafted token 1: rows 1 and 3 see it
        c["k"] = scaled_token(c["k"], int(c["table"][0, at // PAGE]), at % PAGE, power)
        hit = compare_tree(ops, device, c, masks, 0.1, bound)
        if power < 30:
            continue
        # (the tolerance above grows with the scores; a score of 2^power leaves one token or none, and no rounding but the result's)
        k, v = (cases._dense(c[n])[int(c["table"][0, at // PAGE]), :, at % PAGE] for n in ("k", "v"))
        for row in (1, 3):
            for h in range(H):
                if float(k[h * G // H] @ c["q"][row, h].to(F64)) > 0:
                    want = v[h * G // H]
                    assert bool(((hit[row, h] - want).abs() <= 2.0 ** -7 * want.abs()).all()), (row, h)


# ------------------------------------------------------------------ values of any size
def check_tree_hidden_large(ops, device, fp8, dtype, hd, H, power, G=2, bound=None):
    """A drafted token with finite values of 2^power times the others' does not reach the rows that do not see it, wherever it lies
    against the tiles."""
    masks = [1, 3, 5, 11, 21, 33, 1, 3]
    for lens in ([70, 33], [38, 131], [640, 130]):
        c = cases.tree_case(H, G, hd, [6, 2], lens, fp8, dtype, 31, spread=0.25)
        at = lens[0] - 6 + 1                                            # drafted token 1: rows 1 and 3 see it
        page, off = int(c["table"][0, at // PAGE]), at % PAGE
        c["v"] = scaled_token(c["v"], page, off, power)
        compare_tree(ops, device, c, masks, 0.1, bound)


def check_tree_unlikely_large(ops, device, fp8, dtype, hd, H, power, where, G=2, bound=None):
    """A seen token whose probability is nearly zero and whose values are huge weighs just their product."""
    lens = [400, 37]
    c = cases.tree_case(H, G, hd, [6, 2], lens, fp8, dtype, 41, spread=0.25)
    c["q"] = (c["q"].float().abs() + 0.5).to(dtype)
    page, off = int(c["table"][0, where // PAGE]), where % PAGE
    c["v"] = scaled_token(c["v"], page, off, power)
    if fp8:
        c["k"] = Fp8Pages(c["k"].codes.clone(), c["k"].exps.clone())
        c["k"].codes[page, :, off] = torch.tensor(-256.0).to(torch.float8_e4m3fn)
        c["k"].exps[page, :, off] = 127 - 6                             # -4
    else:
        c["k"] = c["k"].clone()
        c["k"][page, :, off] = -4.0
    compare_tree(ops, device, c, [1, 3, 5, 11, 21, 33, 1, 3], 0.125 * (64 / hd), bound)


def check_tree_wide_values(ops, device, hd, H, G=2, bound=None):
    """Values of every size from token to token."""
    cases.check_tree(ops, device, H, G, hd, [6, 0, 2, 9], [700, 5, 33, 300], True, torch.bfloat16, True, seed=3, spread=7.0, bound=bound)


# ------------------------------------------------------------------ a page list without columns
def check_tree_without_pages(ops, device, fp8, dtype, H):
    """Sequences have rows and no page lists: zero rows, in a given output too; what lies behind the last sequence is left."""
    G, hd = 2, 64
    pages = Fp8Pages.zeros(1, G, hd, device) if fp8 else torch.ones(1, G, PAGE, hd, device=device, dtype=dtype)
    q = torch.ones(5, H, hd, device=device, dtype=dtype)
    t = lambda *a: torch.tensor(a, dtype=torch.int32, device=device)
    table = torch.zeros(2, 0, dtype=torch.int32, device=device)
    for lens in ((3, 0), (40, 0)):
        out = torch.full((5, H * hd), 7.0, device=device, dtype=dtype)
        args = (q, pages, pages, table, t(*lens), t(0, 3, 3), 3, 40, 0.1)
        got = ops.paged_tree_attention(*args, None, out)
        assert got is out and bool((out[:3] == 0).all()) and bool((out[3:] == 7).all())
        assert bool((ops.paged_tree_attention(*args) == 0).all())


# ------------------------------------------------------------------ 4-bit products
def check_int4_scales(ops, device, dtype, M, N, K, group, scale_power, x_power):
    """Scales near the upper and below the lower end of bf16's normal numbers count as what they are."""
    x, w = cases.int4_case(M, N, K, group, 3)
    x = (x.to(F64) * 2.0 ** x_power).to(dtype)
    w = Int4Weight(w.packed, (w.scales.to(F64) * 2.0 ** scale_power).to(torch.bfloat16), w.shape, group)
    assert bool(torch.isfinite(w.scales).all()) and bool((w.scales != 0).all())
    want = x.to(F64) @ cases.plain_int4(w)[0].t()
    got = ops.gemm_nt(x.to(device), Int4Weight(w.packed.to(device), w.scales.to(device), w.shape, group)).cpu().to(F64)
    held = 143 * (x.to(F64).abs() @ (w.scales.to(F64).permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:N].repeat_interleave(group, 1)[:, :K]).t())
    tol = 2.0 ** -8 * want.abs() + 8 * 2.0 ** -22 * held if dtype == torch.bfloat16 else 2.0 ** -20 * held
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).nan_to_num(math.inf).max())


INT4_SCALE_CASES = [(3, 40, 200, 128), (16, 96, 512, 64), (20, 130, 1032, 128), (64, 48, 768, 64), (100, 100, 1000, 128)]
INT4_SCALE_POWERS = [(124, -100), (122, -60), (-128, 100), (-130, 60)]

"""Checks of the 8-bit paged cache, tree attention and 4-bit weights that run on either back end, against plain float64
implementations that share nothing with the framework's code."""
import math

import torch

from kotodama_b200.ops import Fp8Pages, Int4Weight

PAGE = 16
F64 = torch.float64


# ------------------------------------------------------------------ plain implementations
def _e4m3_table():
    """All finite e4m3 numbers by code, from the format's definition."""
    vals = []
    for code in range(256):
        s, e, m = code >> 7, (code >> 3) & 15, code & 7
        v = math.ldexp(m / 8, -6) if e == 0 else math.ldexp(1 + m / 8, e - 7)
        vals.append(math.nan if e == 15 and m == 7 else -v if s else v)
    return torch.tensor(vals, dtype=F64)


E4M3 = _e4m3_table()


def plain_quantise(x):
    """Float64 rows -> (codes as uint8, exponents as uint8): smallest power of two from 2^-126 with amax <= 448 * 2^e, nearest code,
    ties to the even one, signs of zeros kept."""
    x = x.to(F64).cpu()
    codes = torch.zeros(x.shape, dtype=torch.uint8)
    exps = torch.zeros(x.shape[:-1], dtype=torch.uint8)
    grid = E4M3[:127]                                              # the non-negative numbers in order
    for at in torch.cartesian_prod(*[torch.arange(n) for n in x.shape[:-1]]).reshape(-1, x.ndim - 1).tolist():
        row = x[tuple(at)]
        if not torch.isfinite(row).all():
            codes[tuple(at)], exps[tuple(at)] = 127, 255
            continue
        e = -126
        while float(row.abs().max()) > 448.0 * 2.0 ** e:
            e += 1
        y = (row * 2.0 ** -e).abs()
        d = (y[:, None] - grid[None, :]).abs()
        best = d.amin(-1, keepdim=True)
        near = d == best
        pick = torch.where(near.sum(-1) > 1, (near & (torch.arange(127) % 2 == 0)[None, :]).int().argmax(-1), near.int().argmax(-1))
        codes[tuple(at)] = (pick + 128 * torch.signbit(row).long()).to(torch.uint8)
        exps[tuple(at)] = e + 127
    return codes, exps


def plain_values(pages: Fp8Pages):
    """Float64 numbers of 8-bit pages."""
    c = E4M3[pages.codes.cpu().view(torch.uint8).long()]
    return c * torch.exp2(pages.exps.cpu().to(F64) - 127)[..., None]


def plain_tree(q, kd, vd, table, ctx_lens, cu, scale, masks):
    """Float64 tree attention over dense page values; returns the rows and, per element, sum_j p_j |v_j|."""
    N, H, hd = q.shape
    G = kd.shape[1]
    out, mass = torch.zeros(N, H, hd, dtype=F64), torch.zeros(N, H, hd, dtype=F64)
    for b, n in enumerate(ctx_lens):
        for i in range(cu[b + 1] - cu[b]):
            row = cu[b] + i
            prefix = n - (cu[b + 1] - cu[b])
            toks = [t for t in range(n) if t < prefix or (masks[row] >> (t - prefix) & 1 if masks is not None else t - prefix <= i)]
            toks = [t for t in toks if 0 <= table[b][t // PAGE] < kd.shape[0]]
            if not toks:
                continue
            page = torch.tensor([table[b][t // PAGE] for t in toks])
            off = torch.tensor([t % PAGE for t in toks])
            k, v = kd[page, :, off], vd[page, :, off]                 # [toks, G, hd]
            for h in range(H):
                s = (k[:, h * G // H] @ q[row, h].to(F64)) * scale
                p = torch.softmax(s, 0)
                out[row, h] = p @ v[:, h * G // H]
                mass[row, h] = p @ v[:, h * G // H].abs()
    return out, mass


def plain_int4(weight: Int4Weight):
    """Float64 values of a 4-bit weight, read word by word."""
    N, K = weight.shape
    words = weight.packed.cpu().to(torch.int64) & 0xFFFFFFFF
    scales = weight.scales.cpu().to(F64)
    w = torch.zeros(-(-N // 16) * 16, -(-K // 64) * 64, dtype=F64)
    c = torch.zeros_like(w)
    nibble = {(0, 0): 0, (0, 1): 4, (0, 2): 2, (0, 3): 6, (1, 0): 1, (1, 1): 5, (1, 2): 3, (1, 3): 7}
    n = torch.arange(words.shape[0])[:, None] * 16                     # all row tiles at once
    for half in range(2):
        for r in range(8):
            for lane in range(4):
                for j in range(4):
                    for i in range(4):
                        k = torch.arange(words.shape[1]) * 64 + 16 * lane + 4 * j + i
                        code = (words[:, :, 4 * r + lane, j] >> (4 * nibble[half, i])) & 15
                        g = (k // weight.group).clamp_max(scales.shape[1] - 1)
                        c[n + half * 8 + r, k] = code.to(F64)
                        w[n + half * 8 + r, k] = (code.to(F64) - 8) * scales[:, g, r, half]
    return w[:N, :K], c


# ------------------------------------------------------------------ 8-bit cache
def cache_rows(n, n_kv, hd, dtype, seed):
    """Rows whose sizes differ by many powers of two, with an all-zero row, numbers on rounding ties and, at the borders of the
    exponent, rows whose largest number is 448 or 1.75 times a power of two."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, n_kv, hd, generator=g) * torch.exp2(torch.randint(-30, 30, (n, n_kv, 1), generator=g).float())
    x[0, 0] = 0.0
    if n > 1:
        x[1, 0] = torch.linspace(-448, 448, hd).round()               # exactly representable largest, many ties
        x[1, -1, 0] = 448.0 * 2 ** 7
        x[n - 1, 0] = torch.linspace(-1.75, 1.75, hd)
        x[n - 1, -1] = x[n - 1, -1].sign() * 1e-40 if dtype == torch.float32 else x[n - 1, -1]
    return x.reshape(n, n_kv * hd).to(dtype)


def check_append(ops, device, dtype, n, n_kv, hd, pages, strided, seed=0):
    """Every code and exponent is exactly the definition's; slots that are not named keep their bytes; negative slots are dropped."""
    k, v = cache_rows(n, n_kv, hd, dtype, seed), cache_rows(n, n_kv, hd, dtype, seed + 1)
    g = torch.Generator().manual_seed(seed + 2)
    slots = torch.randperm(pages * PAGE, generator=g)[:n]
    slots[::5] = -1
    pads = 24 if strided else 0
    wide = lambda x: torch.cat([x, torch.full((n, pads), 7.0, dtype=dtype)], 1).to(device)[:, : n_kv * hd]
    kp, vp = Fp8Pages.zeros(pages, n_kv, hd, device), Fp8Pages.zeros(pages, n_kv, hd, device)
    for p in (kp, vp):
        p.codes.view(torch.uint8).fill_(0x5A)
        p.exps.fill_(99)
    ops.kv_append(wide(k), wide(v), kp, vp, slots.to(device))
    for x, p in ((k, kp), (v, vp)):
        codes = torch.full((pages, n_kv, PAGE, hd), 0x5A, dtype=torch.uint8)
        exps = torch.full((pages, n_kv, PAGE), 99, dtype=torch.uint8)
        wc, we = plain_quantise(x.view(n, n_kv, hd))
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                codes[s // PAGE, :, s % PAGE], exps[s // PAGE, :, s % PAGE] = wc[i], we[i]
        assert torch.equal(p.codes.view(torch.uint8).cpu(), codes)
        assert torch.equal(p.exps.cpu(), exps)
    return kp, vp


APPEND_CASES = [(1, 1, 64, 1, False), (7, 3, 128, 2, True), (40, 2, 80, 4, False), (19, 5, 16, 3, True), (33, 1, 256, 3, False)]


def check_append_not_finite(ops, device):
    """A row with an infinity or a NaN reads back as NaN; its neighbours do not notice."""
    n, n_kv, hd = 4, 2, 64
    k = torch.randn(n, n_kv * hd, generator=torch.Generator().manual_seed(3))
    k[1, 5], k[2, hd + 1], k[3, 0] = math.inf, math.nan, -math.inf
    kp, vp = Fp8Pages.zeros(1, n_kv, hd, device), Fp8Pages.zeros(1, n_kv, hd, device)
    ops.kv_append(k.to(device), k.to(device), kp, vp, torch.arange(n, device=device))
    x = plain_values(kp)[0, :, :n].transpose(0, 1)
    bad = torch.zeros(n, n_kv, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = bad[3, 0] = True
    assert torch.equal(torch.isnan(x).all(-1), bad) and torch.equal(torch.isnan(x).any(-1), bad)
    t = lambda *a: torch.tensor(a, dtype=torch.int32, device=device)
    rows, _ = ops.kv_gather(kp, vp, t(0)[None], t(0), t(0), t(0, n), n)
    assert torch.equal(torch.isnan(rows).all(-1).cpu(), bad)


def check_gather(ops, device, dtype, n_kv, hd, lens, seed=0):
    """Reading back is exact: fp32 holds every code times its power, bf16 rounds nothing within its range."""
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // PAGE) for n in lens) + 2
    codes = torch.randint(0, 256, (2, pages, n_kv, PAGE, hd), generator=g, dtype=torch.uint8)
    codes[(codes & 127) == 127] = 0                                   # no NaN codes here
    exps = torch.randint(127 - 100, 127 + 100, (2, pages, n_kv, PAGE), generator=g, dtype=torch.uint8)
    kp, vp = (Fp8Pages(codes[i].view(torch.float8_e4m3fn).to(device), exps[i].to(device)) for i in range(2))
    order = torch.randperm(pages, generator=g)
    table = torch.zeros(len(lens), max(-(-n // PAGE) for n in lens), dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // PAGE)
        table[b, :m] = order[at:at + m].int()
        at += m
    # segments in another order than the sequences, beginning inside a page, one of them empty
    seq = list(range(len(lens)))[::-1] + [0]
    first = [min(3, lens[b] - 1) if i % 2 else 0 for i, b in enumerate(seq)]
    count = [lens[b] - f for b, f in zip(seq, first)]
    count[-1] = 0
    cu = [0]
    for n in count:
        cu.append(cu[-1] + n)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    k, v = ops.kv_gather(kp, vp, table.to(device), t(seq), t(first), t(cu), cu[-1], dtype)
    for got, p in ((k, kp), (v, vp)):
        full = plain_values(p)
        want = torch.cat([torch.stack([full[table[b, j // PAGE], :, j % PAGE] for j in range(f, f + n)])
                          for b, f, n in zip(seq, first, count) if n])
        assert got.dtype == dtype and torch.equal(got.cpu().to(F64), want)


GATHER_CASES = [(1, 64, [1]), (3, 128, [5, 40, 16]), (2, 80, [33, 17]), (5, 16, [100]), (1, 256, [31, 1, 2])]


# ------------------------------------------------------------------ tree attention
def tree_masks(sizes, seed, empty=()):
    """One 64-bit mask per row: a random tree per sequence (each row sees its ancestors and itself); rows in ``empty`` see none."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        seen = []
        for i in range(n):
            parent = int(torch.randint(0, i, (1,), generator=g)) if i else -1
            seen.append((seen[parent] if i else 0) | 1 << i)
        out += seen
    for i in empty:
        out[i] = 0
    return out


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


def tree_case(H, G, hd, sizes, lens, fp8, dtype, seed, stale=True, spread=1.0):
    """Inputs of one call on the host: scattered pages whose unused places hold infinities, NaNs and large numbers."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // PAGE) for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1]) + 1), -5, dtype=torch.int32)      # entries behind a sequence's pages are no pages
    kd = torch.randn(pages, G, PAGE, hd, generator=g)
    vd = torch.randn(pages, G, PAGE, hd, generator=g) * torch.exp2(4 * spread * torch.randn(pages, G, PAGE, 1, generator=g))
    used = torch.zeros(pages, PAGE, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        for i in range(need[b]):
            table[b, i] = order[at]
            used[order[at], : min(PAGE, n - i * PAGE)] = True
            at += 1
    if stale:
        junk = torch.tensor([math.inf, -math.inf, math.nan, 3e38])[torch.randint(0, 4, vd.shape, generator=g)]
        gone = ~used[:, None, :, None].expand_as(vd)
        kd, vd = torch.where(gone, junk, kd), torch.where(gone, junk, vd)
    q = 2.0 * torch.randn(sum(sizes), H, hd, generator=g)
    cu = [0]
    for n in sizes:
        cu.append(cu[-1] + n)
    c = dict(q=q.to(dtype), table=table, lens=list(lens), cu=cu, sizes=list(sizes))
    if fp8:
        for name, x in (("k", kd), ("v", vd)):
            codes, exps = Fp8Pages.zeros(pages, G, hd, "cpu").codes, torch.zeros(pages, G, PAGE, dtype=torch.uint8)
            flat = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).to(torch.bfloat16).float()
            e = torch.ceil(torch.log2(flat.abs().amax(-1).to(F64).clamp_min(1e-30) / 448)).clamp(-126, 127)
            codes = (flat.to(F64) * torch.exp2(-e)[..., None]).clamp(-448, 448).float().to(torch.float8_e4m3fn)
            exps = (e + 127).to(torch.uint8)
            if stale:
                bad = ~used[:, None, :].expand_as(exps)
                exps = torch.where(bad, torch.full_like(exps, 255), exps)
                codes.view(torch.uint8)[bad] = 0x7F
            c[name] = Fp8Pages(codes, exps)
    else:
        c["k"], c["v"] = kd.to(dtype), vd.to(dtype)
    return c


def _dense(p):
    return plain_values(p) if isinstance(p, Fp8Pages) else p.cpu().to(F64)


def _put(p, device):
    return Fp8Pages(p.codes.to(device), p.exps.to(device)) if isinstance(p, Fp8Pages) else p.to(device)


def run_tree(ops, device, c, masks, scale, tail=0, out=None, decode=False, max_ctx=None):
    q = torch.cat([c["q"], torch.full((tail, *c["q"].shape[1:]), math.nan, dtype=c["q"].dtype)]) if tail else c["q"]
    m = None
    if masks is not None:
        m = signed(masks + [-1 & (1 << 64) - 1] * tail).to(device)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return ops.paged_tree_attention(q.to(device), _put(c["k"], device), _put(c["v"], device), c["table"].to(device), t(c["lens"]),
                                    None if decode else t(c["cu"]), max(c["sizes"] + [1]), max_ctx or max(c["lens"] + [1]), scale, m, out)


def tree_tolerance(c, want, mass, scale):
    """Per element.  bf16: the probabilities and the result are rounded once each (half a step, 2^-8, of what they weigh), and the
    exponent of a score carries its fp32 sum's error.  fp32: only sums."""
    hd = c["q"].shape[-1]
    big = float(c["q"].to(F64).norm(dim=-1).max()) * max(float(_dense(p)[torch.isfinite(_dense(p)).all(-1)].norm(dim=-1).max()) for p in (c["k"],)) * scale
    sums = 2.0 ** -23 * (hd + 8) ** 0.5 * big + 2.0 ** -23 * (max(c["lens"]) + 32)     # |error of a score| + error of the sums over tokens
    if c["q"].dtype == torch.float32:
        return 4 * sums * mass + 2.0 ** -23 * want.abs() + 1e-30
    return (2.0 ** -8 + 4 * sums) * mass + 2.0 ** -8 * want.abs() + 1e-30


def check_tree(ops, device, H, G, hd, sizes, lens, fp8, dtype, masked, seed=0, spread=1.0, bound=None):
    c = tree_case(H, G, hd, sizes, lens, fp8, dtype, seed, spread=spread)
    empty = [i for i in (1,) if masked and sum(sizes) > 2]
    masks = tree_masks(sizes, seed + 1, empty) if masked else None
    scale = 1.0 / math.sqrt(hd)
    want, mass = plain_tree(c["q"], _dense(c["k"]), _dense(c["v"]), c["table"].tolist(), c["lens"], c["cu"], scale, masks)
    tol = tree_tolerance(c, want, mass, scale)
    got = run_tree(ops, device, c, masks, scale, tail=3, max_ctx=bound).cpu()
    N = c["q"].shape[0]
    assert got.shape == (N + 3, H * hd) and torch.equal(got[N:], torch.zeros_like(got[N:]))
    err = (got[:N].to(F64).view(N, H, hd) - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), (err / tol).amax((1, 2)).tolist())
    kept = torch.full((N + 3, H * hd + 8), 5.0, dtype=dtype, device=device)         # a given output: strided, rows behind the last are left
    run_tree(ops, device, c, masks, scale, tail=3, out=kept[:, : H * hd], max_ctx=bound)
    assert torch.equal(kept[:N, : H * hd].cpu(), got[:N]) and bool((kept[N:] == 5).all()) and bool((kept[:, H * hd:] == 5).all())
    if max(sizes) == 1 and min(sizes) == 1 and not masked:
        assert torch.equal(run_tree(ops, device, c, None, scale, decode=True, max_ctx=bound).cpu(), got[:N])


TREE_CASES = [  # heads, kv heads, head size, rows per sequence, tokens per sequence, masks
    (1, 1, 64, [1], [1], False), (4, 2, 128, [1, 1, 1], [1, 17, 300], False), (6, 2, 128, [5, 0, 3], [5, 9, 128], True),
    (3, 1, 64, [64], [64], True), (8, 8, 64, [2, 7], [130, 63], True), (24, 8, 128, [8], [301], True), (5, 1, 128, [13, 1], [257, 129], True),
    (16, 2, 128, [33], [65], False), (12, 4, 64, [16, 16], [1023, 31], True), (8, 1, 128, [64, 64], [640, 66], True),
    (24, 2, 64, [3, 1, 6], [900, 3, 128], True), (64, 1, 128, [1, 2], [129, 384], False),
]
TREE_PLAIN_CASES = [(2, 1, 80, [3, 1], [40, 7], True), (3, 3, 16, [1], [200], False), (4, 2, 256, [9], [77], True)]


def check_tree_masked_not_finite(ops, device, fp8, dtype=torch.bfloat16, hd=128, H=4, G=2, bound=None):
    """A drafted token whose keys or values are not finite reaches the rows that see it and no other; of its values, in a row that sees
    it, only the dimensions that are not finite are lost."""
    sizes, lens = [6, 2], [70, 33]
    masks = [1, 3, 5, 11, 21, 33, 1, 3]
    c = tree_case(H, G, hd, sizes, lens, fp8, dtype, 11)
    clean = run_tree(ops, device, c, masks, 0.1, max_ctx=bound).cpu()
    prefix = lens[0] - sizes[0]
    page, off = int(c["table"][0, (prefix + 1) // PAGE]), (prefix + 1) % PAGE      # drafted token 1: rows 1 and 3 see it
    for name in ("k", "v"):
        for what in (math.nan, math.inf):
            d = {**c, "k": _put(c["k"], "cpu"), "v": _put(c["v"], "cpu")}
            if fp8:
                d[name] = Fp8Pages(c[name].codes.clone(), c[name].exps.clone())
                d[name].codes.view(torch.uint8)[page, :, off] = 0x7F
                d[name].exps[page, :, off] = 255
            else:
                d[name] = c[name].clone()
                d[name][page, :, off] = what
            got = run_tree(ops, device, d, masks, 0.1, max_ctx=bound).cpu()
            hit = [1, 3]
            rest = [0, 2, 4, 5, 6, 7]
            assert torch.equal(got[rest], clean[rest]), (name, what)
            assert not bool(torch.isfinite(got[hit]).all(-1).any()), (name, what)
    if not fp8:
        d = {**c, "v": c["v"].clone()}
        d["v"][page, :, off, 3] = math.inf
        got = run_tree(ops, device, d, masks, 0.1, max_ctx=bound).cpu().view(-1, H, hd)
        want, mass = plain_tree(c["q"], _dense(c["k"]), _dense(c["v"]), c["table"].tolist(), lens, c["cu"], 0.1, masks)
        tol = tree_tolerance(c, want, mass, 0.1)
        dims = [i for i in range(hd) if i != 3]
        assert torch.equal(got[[0, 2, 4, 5, 6, 7]], clean.view(-1, H, hd)[[0, 2, 4, 5, 6, 7]])
        assert bool((got[hit][..., 3] == math.inf).all())
        assert bool(((got[hit].to(F64) - want[hit]).abs() <= tol[hit])[..., dims].all())


def check_tree_bad_sequences(ops, device, fp8, H=4, G=2, empty=0):
    """Sequences that break the rules get zero rows, tokens on pages that are not there are not seen; the other sequences are as ever.
    ``empty``: so many sequences without rows behind them (which are then too many for a block of threads each)."""
    hd = 64
    c = tree_case(H, G, hd, [2, 3, 1, 2], [40, 2, 50, 90], fp8, torch.bfloat16, 5)      # 3 rows in 2 tokens
    c["lens"] = list(c["lens"]) + [0] * empty
    c["cu"] = list(c["cu"]) + [c["cu"][-1]] * empty
    c["table"] = torch.cat([c["table"], torch.zeros(empty, c["table"].shape[1], dtype=c["table"].dtype)])
    c["table"][2, 1] = c["k"].shape[0]                              # page past the cache: tokens 16 .. 31 of sequence 2
    c["table"][2, 2] = -1
    got = run_tree(ops, device, c, None, 0.125, max_ctx=60).cpu().view(-1, H, hd)        # sequence 3 is longer than 60
    bad = [2, 3, 4, 6, 7]
    assert bool((got[bad] == 0).all())
    want, mass = plain_tree(c["q"], _dense(c["k"]), _dense(c["v"]), c["table"].tolist(), [40, 0, 50, 0], [0, 2, 2, 3, 3], 0.125, None)
    # sequences 0 and 2 alone: their rows sit at 0, 1 and 5
    ref, m = torch.zeros_like(want), torch.zeros_like(mass)
    ref[[0, 1]], m[[0, 1]] = want[[0, 1]], mass[[0, 1]]
    w2, m2 = plain_tree(c["q"][5:6], _dense(c["k"]), _dense(c["v"]), [c["table"][2].tolist()], [50], [0, 1], 0.125, None)
    ref[5], m[5] = w2[0], m2[0]
    good = [0, 1, 5]
    assert bool(((got[good].to(F64) - ref[good]).abs() <= tree_tolerance(c, ref, m, 0.125)[good]).all())


# ------------------------------------------------------------------ 4-bit weights
def check_quant_int4(ops, device, N, K, group, seed=0):
    """Codes and scales against their definition; the words hold them where the format says."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(N, K, generator=g) * torch.exp2(torch.randint(-6, 6, (N, 1), generator=g).float())
    w[0, : min(K, group)] = 0.0
    q = ops.quant_int4(w.to(device), group)
    assert q.shape == (N, K) and q.group == group
    got, codes = plain_int4(q)
    for n in range(N):
        for k0 in range(0, K, group):
            x = w[n, k0:k0 + group].to(F64)
            s = float((x.float().abs().max() / 7).to(torch.bfloat16))
            c = torch.round(x / s) if s else torch.zeros_like(x)
            near = ((x / s - torch.floor(x / s)) - 0.5).abs() < 1e-6 if s else torch.zeros_like(x, dtype=torch.bool)   # within fp32's division of a tie
            off = (got[n, k0:k0 + group] - s * c).abs()
            assert bool(((off == 0) | (near & (off <= s))).all())
    assert bool((codes[N:] == 8).all()) and bool((codes[:, K:] == 8).all())
    assert torch.equal(q.dense().cpu().to(F64), got)


INT4_QUANT_CASES = [(16, 64, 64), (5, 72, 128), (33, 200, 64), (17, 136, 128)]


def int4_case(M, N, K, group, seed, stride=0):
    g = torch.Generator().manual_seed(seed)
    nt, kb, ng = -(-N // 16), -(-K // 64), -(-K // group)
    packed = torch.randint(-2 ** 31, 2 ** 31, (nt, kb, 32, 4), generator=g).to(torch.int32)
    if K % 64:                                                        # inputs past the matrix have code 8
        lane = torch.arange(32) % 4
        for j in range(4):
            for i, (lo, hi) in enumerate(((0, 4), (16, 20), (8, 12), (24, 28))):
                past = (kb - 1) * 64 + 16 * lane + 4 * j + i >= K
                w = packed[:, -1, :, j].to(torch.int64) & 0xFFFFFFFF
                for s in (lo, hi):
                    w = torch.where(past, (w & ~(15 << s)) | 8 << s, w)
                packed[:, -1, :, j] = (w - ((w >> 31) << 32)).to(torch.int32)
    scales = (torch.rand(nt, ng, 8, 2, generator=g) + 0.1).to(torch.bfloat16)
    x = torch.randn(M, K + stride, generator=g).to(torch.bfloat16)
    return x, Int4Weight(packed, scales, (N, K), group)


def check_int4(ops, device, dtype, M, N, K, group, seed=0, stride=0):
    x, w = int4_case(M, N, K, group, seed, stride)
    x = x.to(dtype)
    wd = Int4Weight(w.packed.to(device), w.scales.to(device), w.shape, group)
    dense, _ = plain_int4(w)
    xd = x.to(device)[:, :K]
    want = x[:, :K].to(F64) @ dense.t()
    # fp32: a group's accumulator holds numbers of up to 143 |x|, and each of its steps (16 inputs) cuts at 2^-22 of them; then sums over
    # groups.  The result is rounded once: half a step.
    held = 143 * (x[:, :K].to(F64).abs() @ (w.scales.to(F64).permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:N].repeat_interleave(group, 1)[:, :K]).t())
    tol = 2.0 ** -8 * want.abs() + 8 * 2.0 ** -22 * held if dtype == torch.bfloat16 else 2.0 ** -20 * held
    ok = lambda got, ref, t: bool(((got.cpu().to(F64) - ref).abs() <= t).all())
    got = ops.gemm_nt(xd, wd)
    assert got.shape == (M, N) and got.dtype == dtype and ok(got, want, tol), float(((got.cpu().to(F64) - want).abs() / tol).max())
    g = torch.Generator().manual_seed(seed + 9)
    res = torch.randn(M, N, generator=g).to(dtype)
    both = want + res.to(F64)
    tol2 = tol + 2.0 ** -8 * (want.abs() + both.abs()) if dtype == torch.bfloat16 else tol + 2.0 ** -23 * both.abs()
    assert ok(ops.gemm_nt(xd, wd, residual=res.to(device)), both, tol2)
    wide = torch.full((M, N + 8), 3.0, dtype=dtype, device=device)
    wide[:, :N] = res.to(device)
    ops.gemm_nt(xd, wd, out=wide[:, :N], accumulate=True)
    assert ok(wide[:, :N], both, tol2) and bool((wide[:, N:] == 3).all())
    row = res[:1].expand(M, N)
    assert ok(ops.gemm_nt(xd, wd, residual=res[:1].to(device)), want + row.to(F64), tol + 2.0 ** -8 * (want.abs() + (want + row.to(F64)).abs()))


INT4_CASES = [(1, 16, 64, 64, 0), (1, 1, 8, 128, 0), (3, 40, 200, 128, 8), (8, 96, 512, 128, 0), (9, 33, 520, 64, 0), (17, 130, 1032, 128, 16),
              (33, 64, 64, 128, 0), (64, 48, 768, 64, 0), (65, 100, 1000, 128, 0), (130, 70, 136, 64, 8)]

# every form of the two product kernels: row tiles per block of threads (1 to 4 at a time, steps of unequal size), rings that turn over,
# inputs shared by clusters and not, one block left over, several portions of tokens
INT4_LARGE_CASES = [(4, 2501, 136, 64, 0), (8, 5001, 200, 128, 0), (1, 9500, 72, 64, 8), (7, 16500, 192, 128, 0), (2, 40, 8200, 128, 0), (5, 64, 4160, 64, 0),
                    (16, 2500, 648, 128, 0), (12, 5000, 136, 64, 0), (9, 12001, 264, 128, 0), (11, 48, 8232, 128, 0), (10, 96, 5000, 64, 8),
                    (40, 9990, 1032, 128, 0), (20, 130, 8200, 128, 0), (64, 200, 8264, 64, 0), (100, 128, 2056, 128, 0), (300, 100, 1352, 128, 8),
                    (130, 1000, 968, 64, 0), (1000, 272, 456, 128, 0), (17, 13, 24, 64, 0), (33, 1, 8, 128, 0)]


def check_int4_overlapping_rows(ops, device):
    """Rows of x that are one row, and rows that overlap."""
    x, w = int4_case(24, 40, 136, 64, 5)
    dense, _ = plain_int4(w)
    wd = Int4Weight(w.packed.to(device), w.scales.to(device), w.shape, w.group)
    flat = x.to(device).reshape(-1)
    for rows in (x[:1].to(device).expand(24, 136), flat.as_strided((24, 136), (8, 1))):
        want = rows.cpu().to(F64) @ dense.t()
        held = 143 * 1.1 * rows.cpu().to(F64).abs().sum(1, keepdim=True)
        err = (ops.gemm_nt(rows, wd).cpu().to(F64) - want).abs()
        assert bool((err <= 2.0 ** -8 * want.abs() + 8 * 2.0 ** -22 * held).all())


def check_quant_int4_not_finite(ops, device):
    """A group that holds an infinity or a NaN has a scale that is not finite; all others are as without it."""
    w = torch.randn(33, 256, generator=torch.Generator().manual_seed(4))
    clean = plain_int4(ops.quant_int4(w.to(device), 64))[0]
    for what in (math.nan, math.inf, -math.inf):
        d = w.clone()
        d[9, 70] = what
        q = ops.quant_int4(d.to(device), 64)
        got = plain_int4(q)[0]
        bad = torch.zeros(33, 256, dtype=torch.bool)
        bad[9, 64:128] = True
        assert torch.equal(got[~bad], clean[~bad]) and not bool(torch.isfinite(q.scales.cpu()).all())


def ragged(n, most, rows, seed):
    """Lengths and rows of ``n`` sequences: empty ones, single tokens, long ones, in no order."""
    g = torch.Generator().manual_seed(seed)
    sizes = torch.randint(0, rows + 1, (n,), generator=g).tolist()
    lens = [s + (int(torch.randint(0, most, (1,), generator=g)) if i % 3 else 0) for i, s in enumerate(sizes)]
    return sizes, [max(a, 1) for a in lens]


def tile_parts(total, workers):
    """The line of ``total`` tiles as the tensor-core kernels cut it (integer arithmetic of the kernels)."""
    parts = min(workers, total)
    return [(total * c // parts, total * (c + 1) // parts) if c < parts else (0, 0) for c in range(workers)]


def written_parts(tiles, blocks, per):
    """What the workers leave for each unit (``tiles``: tiles per unit): slots of partial results, or None where the unit is finished.  A block
    whose ``per`` > 1 parts lie in one unit leaves one."""
    total, workers = sum(tiles), blocks * per
    parts = tile_parts(total, workers)
    out, s0 = [], 0
    for t in tiles:
        slots, finished = [], False
        for c in range(blocks):
            mine = parts[c * per:(c + 1) * per]
            lo, hi = mine[0][0], mine[-1][1]
            if per > 1 and hi > 0 and lo >= s0 and hi <= s0 + t:
                if (lo, hi) == (s0, s0 + t):
                    finished = True
                else:
                    slots.append(2 * c * per + (lo == s0))
                continue
            for w, (a, b) in enumerate(mine):
                a, b = max(a, s0), min(b, s0 + t)
                if a < b:
                    if (a, b) == (s0, s0 + t):
                        finished = True
                    else:
                        slots.append(2 * (c * per + w) + (a == s0))
        assert not (finished and slots)
        out.append(None if finished else slots)
        s0 += t
    return out


def merged_parts(tiles, blocks, per):
    """What the merge kernel reads for each unit, in its arithmetic."""
    total = sum(tiles)
    parts = min(blocks * per, total)
    out, s0 = [], 0
    for t in tiles:
        first, last = ((s0 + 1) * parts - 1) // total, ((s0 + t) * parts - 1) // total
        ca, cb = first // per, last // per

        def whole(c):
            return (c + 1) * per <= parts and total * c * per // parts >= s0 and total * (c + 1) * per // parts <= s0 + t

        wa, wb = whole(ca), whole(cb)
        if (wa and ca == cb and s0 == total * ca * per // parts and s0 + t == total * (ca + 1) * per // parts) or (first == last and not wa):
            out.append(None)
        else:
            head = 1 if wa else min(last, ca * per + per - 1) - first + 1
            mid = cb - ca - 1 if cb > ca else 0
            n = head + mid + ((1 if wb else last - cb * per + 1) if cb > ca else 0)
            js = [first + k if k < head else (ca + 1 + k - head) * per if k < head + mid else cb * per + k - head - mid for k in range(n)]
            out.append([2 * j + (j == first) for j in js])
        s0 += t
    return out

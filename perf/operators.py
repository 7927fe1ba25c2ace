"""Measured cases of the serving operators that keep the cache in 8 bits and the weights in 4.

Four operators, each with a plain form in elementary torch operations and the framework's call:

* ``append``  quantises the keys and values of new tokens while they are written into the paged cache
  (``ops.kv_append`` on ``Fp8Pages``): e4m3 codes with one power-of-two scale per (token, KV head);
* ``gather``  reads cached rows back as packed bf16 rows (``ops.kv_gather`` on ``Fp8Pages``);
* ``tree``    attention of the drafted tokens of several sequences over the paged cache, bf16 or 8-bit: a row sees its
  sequence's prefix and the drafted tokens its mask names (``ops.paged_tree_attention``); one token is plain decoding;
* ``int4``    products with 4-bit weights and one scale per group of inputs (``ops.gemm_nt`` on ``Int4Weight``).

Layouts.  A cache page holds 16 tokens: codes ``[pages, kv heads, 16, head size]``, exponents ``[pages, kv heads, 16]`` (biased by
127, as an 8-bit power of two).  4-bit weights ``[N, K]`` are stored as ``[N/16, K/64, 32, 4]`` 32-bit words: word ``j`` of lane
``l = 4 r + c`` holds inputs ``16 c + 4 j .. + 3`` of the block's rows ``r`` (nibbles 0, 4, 2, 6) and ``r + 8`` (nibbles 1, 5, 3, 7); scales
``[N/16, groups, 8, 2]`` hold rows ``r`` and ``r + 8`` side by side.  A weight is ``scale * (code - 8)``.
"""
import math

import torch

own = False
PAGE = 16


def listed():
    return [
        # one decode step of a full batch: 64 new tokens, rows of a fused q | k | v product
        {"name": "append-decode-64", "op": "append", "tokens": 64, "kv": 8, "hd": 128, "heads": 32},
        # a packed prefill pass, odd length
        {"name": "append-prefill-8191", "op": "append", "tokens": 8191, "kv": 8, "hd": 128, "heads": 32},
        # a context that a portion of a prompt continues, heads of 64
        {"name": "gather-2-ctx1000", "op": "gather", "batch": 2, "ctx": 1000, "kv": 2, "hd": 64},
        # the contexts of a packed pass over several sequences
        {"name": "gather-16-ctx4096", "op": "gather", "batch": 16, "ctx": 4096, "kv": 8, "hd": 128},
        # one request of the smallest preset with eight drafted tokens: latency
        {"name": "tree-1x8-ctx301", "op": "tree", "batch": 1, "rows": 8, "ctx": 301, "heads": 4, "kv": 2, "hd": 128, "fp8": True},
        # plain decoding of a full batch on the 8-bit cache
        {"name": "tree-64x1-ctx2048-fp8", "op": "tree", "batch": 64, "rows": 1, "ctx": 2048, "heads": 24, "kv": 8, "hd": 128, "fp8": True},
        # verification of drafted trees, bf16 cache
        {"name": "tree-16x16-ctx4000-bf16", "op": "tree", "batch": 16, "rows": 16, "ctx": 4000, "heads": 32, "kv": 8, "hd": 128, "fp8": False},
        # one long document with the largest tree: few rows, a long axis
        {"name": "tree-1x64-ctx131000-fp8", "op": "tree", "batch": 1, "rows": 64, "ctx": 131000, "heads": 32, "kv": 8, "hd": 128, "fp8": True},
        # one token through the fused q | k | v projection of the 8b preset
        {"name": "int4-1x6144x4096", "op": "int4", "m": 1, "n": 6144, "k": 4096, "group": 128},
        # eight requests through the fused gate | up projection of the 8b preset
        {"name": "int4-8x28672x4096", "op": "int4", "m": 8, "n": 28672, "k": 4096, "group": 128},
        # a full batch through the down projection, fine groups
        {"name": "int4-64x4096x14336", "op": "int4", "m": 64, "n": 4096, "k": 14336, "group": 64},
        # odd sizes: the feed-forward of the smallest preset cut raggedly
        {"name": "int4-3x1405x1000", "op": "int4", "m": 3, "n": 1405, "k": 1000, "group": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "tree", "tree", "int4", "int4"])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 8191), "kv": kv, "hd": hd, "heads": kv * group}
    if op == "gather":
        batch = _log(rng, 1, 32)
        return {"op": op, "batch": batch, "ctx": min(_log(rng, 1, 32000), 65536 // batch), "kv": kv, "hd": hd}
    if op == "tree":
        batch = _log(rng, 1, 64)
        rows = rng.choice([1, 1, 2, 5, 8, 16, 23, 32, 64])
        ctx = min(rows + _log(rng, 1, 120000), 131000 // max(1, batch * kv * rows * group // 2048 + 1), 262000 // batch)
        return {"op": op, "batch": batch, "rows": rows, "ctx": max(ctx, rows), "heads": kv * group, "kv": kv, "hd": hd, "fp8": rng.random() < 0.5}
    k = 8 * _log(rng, 8, 1792)
    n = _log(rng, 16, min(28672, 100_000_000 // k))
    return {"op": op, "m": _log(rng, 1, 64), "n": n, "k": k, "group": rng.choice([64, 128])}


def _lengths(case):
    """Ragged contexts: the longest first, the others down to half of it, none shorter than the drafted rows."""
    ctx, least = case["ctx"], case.get("rows", 1)
    return [max(least, ctx - (ctx // 2) * ((37 * b) % case["batch"]) // case["batch"]) for b in range(case["batch"])]


def _bytes_per_row(case):
    return case["hd"] + 1 if case.get("fp8", True) else 2 * case["hd"]


def work(case):
    op = case["op"]
    if op == "append":
        rows = 2 * case["tokens"] * case["kv"]
        return {"bytes": rows * (2 * case["hd"] + case["hd"] + 1) + 8 * case["tokens"], "flops": 2 * rows * case["hd"]}
    if op == "gather":
        rows = 2 * sum(_lengths(case)) * case["kv"]
        return {"bytes": rows * (case["hd"] + 1 + 2 * case["hd"]), "flops": rows * case["hd"]}
    if op == "tree":
        lens = _lengths(case)
        seen = sum(n - case["rows"] + (case["rows"] + 1) / 2 for n in lens) * case["rows"]
        q = case["batch"] * case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 2 * sum(lens) * case["kv"] * _bytes_per_row(case) + 4 * q, "flops": 4 * seen * case["heads"] * case["hd"]}
    m, n, k = case["m"], case["n"], case["k"]
    groups = -(-k // case["group"])
    return {"bytes": n * k // 2 + 2 * n * groups + 2 * m * (n + k), "flops": 2 * m * n * k}


def _quantise(x):
    """``x[..., hd]`` -> e4m3 codes and biased exponents: the smallest power of two that brings the row into the type's range."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    k = torch.where(m <= 0.875, e - 9, e - 8).clamp(-126, 127)      # 448 = 0.875 * 2^9
    k = torch.where(m == 0, torch.full_like(k, -126), k)
    codes = torch.ldexp(x, -k[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, (k + 127).to(torch.uint8)


def _value(codes, exps):
    return torch.ldexp(codes.float(), exps.to(torch.int32)[..., None] - 127)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    rand = lambda *s: torch.randn(*s, device=dev, generator=g)
    op = case["op"]
    if op == "append":
        n, kv, hd, heads = case["tokens"], case["kv"], case["hd"], case["heads"]
        qkv = (rand(n, (heads + 2 * kv) * hd) * torch.exp(0.5 * rand(n, 1))).to(torch.bfloat16)
        pages = -(-n // PAGE) + 3
        slots = torch.randperm(pages * PAGE, device=dev, generator=g)[:n]
        code = lambda: torch.zeros(pages, kv, PAGE, hd, device=dev, dtype=torch.float8_e4m3fn)
        exp = lambda: torch.full((pages, kv, PAGE), 127, device=dev, dtype=torch.uint8)
        return {"case": case, "k": qkv[:, heads * hd:(heads + kv) * hd], "v": qkv[:, (heads + kv) * hd:], "slots": slots,
                "kc": code(), "ke": exp(), "vc": code(), "ve": exp()}
    if op == "int4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        nt, kb, ng = -(-n // 16), -(-k // 64), -(-k // group)
        x = rand(m, k).to(torch.bfloat16)
        codes = (rand(nt * 16, kb * 64) * 2.5).round().clamp(-8, 7).to(torch.int32) + 8
        codes[n:] = 8                                                # rows and inputs that are not there weigh nothing
        codes[:, k:] = 8
        scales = (torch.rand(nt * 16, ng, device=dev, generator=g) + 0.5) / (3.0 * math.sqrt(k))
        scales[n:] = 0
        # [nt, half, 8 rows, kb, 4 lanes, 4 words, 4 inputs] -> nibble positions of the words
        c = codes.view(nt, 2, 8, kb, 4, 4, 4).permute(0, 3, 2, 4, 5, 1, 6)      # nt, kb, r, c, j, half, input
        shift = torch.tensor([[0, 16, 8, 24], [4, 20, 12, 28]], device=dev)
        words = (c.to(torch.int64) << shift).sum((-1, -2))
        packed = (words - ((words >> 31) << 32)).to(torch.int32).reshape(nt, kb, 32, 4).contiguous()
        scales = scales.to(torch.bfloat16).view(nt, 2, 8, ng).permute(0, 3, 2, 1).contiguous()
        return {"case": case, "x": x, "packed": packed, "scales": scales}
    lens = _lengths(case)
    batch, kv, hd = case["batch"], case["kv"], case["hd"]
    need = [-(-n // PAGE) for n in lens]
    total = sum(need)
    order = torch.randperm(total + 2, device="cpu", generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros(batch, max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    # keys as a normalised and rotated projection leaves them, values of differing size from token to token
    k = rand(total + 2, kv, PAGE, hd)
    v = rand(total + 2, kv, PAGE, hd) * torch.exp(0.7 * rand(total + 2, kv, PAGE, 1))
    state = {"case": case, "table": table.to(dev), "ctx": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if case.get("fp8", True):
        state["kc"], state["ke"] = _quantise(k.to(torch.bfloat16))
        state["vc"], state["ve"] = _quantise(v.to(torch.bfloat16))
    else:
        state["k"], state["v"] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    if op == "gather":
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        state.update(cu=torch.tensor(cu, dtype=torch.int32, device=dev), seq=torch.arange(batch, dtype=torch.int32, device=dev),
                     first=torch.zeros(batch, dtype=torch.int32, device=dev), total=cu[-1])
        return state
    rows = case["rows"]
    state["q"] = (2.0 * rand(batch * rows, case["heads"], hd)).to(torch.bfloat16)
    state["cu"] = torch.arange(batch + 1, dtype=torch.int32, device=dev) * rows
    # a drafted tree per sequence: every token after the first continues one of the tokens before it
    parents = torch.rand(batch, rows, generator=torch.Generator().manual_seed(seed + 1)).tolist()
    masks = []
    for b in range(batch):
        seen = []
        for i in range(rows):
            seen.append((seen[int(parents[b][i] * i)] if i else 0) | 1 << i)
        masks += [s - (1 << 64) if s >> 63 else s for s in seen]
    state["masks"] = torch.tensor(masks, dtype=torch.int64, device=dev)
    return state


def _ops():
    from kotodama_b200.ops import get_ops
    return get_ops("cuda")


def _fp8(codes, exps):
    from kotodama_b200.ops import Fp8Pages
    return Fp8Pages(codes, exps)


def run(s):
    return {"append": _append, "gather": _gather, "tree": _tree, "int4": _int4}[s["case"]["op"]](s)


def _append(s):
    if own:
        _ops().kv_append(s["k"], s["v"], _fp8(s["kc"], s["ke"]), _fp8(s["vc"], s["ve"]), s["slots"])
    else:
        kv, hd = s["kc"].shape[1], s["kc"].shape[3]
        page, off = s["slots"] // PAGE, s["slots"] % PAGE
        codes, exps = _quantise(s["k"].reshape(-1, kv, hd))
        s["kc"].view(torch.uint8)[page, :, off] = codes.view(torch.uint8)
        s["ke"][page, :, off] = exps
        codes, exps = _quantise(s["v"].reshape(-1, kv, hd))
        s["vc"].view(torch.uint8)[page, :, off] = codes.view(torch.uint8)
        s["ve"][page, :, off] = exps
    return {"k": s["kc"], "k_exp": s["ke"], "v": s["vc"], "v_exp": s["ve"]}


def _gather(s):
    if own:
        k, v = _ops().kv_gather(_fp8(s["kc"], s["ke"]), _fp8(s["vc"], s["ve"]), s["table"], s["seq"], s["first"], s["cu"], s["total"])
        return {"k": k, "v": v}
    row = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    seg = torch.searchsorted(s["cu"], row, right=True) - 1
    t = s["first"][seg] + row - s["cu"][seg]
    page = s["table"][s["seq"][seg].long(), (t // PAGE).long()].long()
    off = (t % PAGE).long()
    pick = lambda codes, exps: _value(codes.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn), exps[page, :, off]).to(torch.bfloat16)
    return {"k": pick(s["kc"], s["ke"]), "v": pick(s["vc"], s["ve"])}


def _tree(s):
    case = s["case"]
    rows, heads, kv, hd, batch, ctx = (case[x] for x in ("rows", "heads", "kv", "hd", "batch", "ctx"))
    scale = 1.0 / math.sqrt(hd)
    if own:
        if case["fp8"]:
            k, v = _fp8(s["kc"], s["ke"]), _fp8(s["vc"], s["ve"])
        else:
            k, v = s["k"], s["v"]
        return _ops().paged_tree_attention(s["q"], k, v, s["table"], s["ctx"], s["cu"], rows, ctx, scale, s["masks"])
    at = s["table"].long()
    if case["fp8"]:
        k = _value(s["kc"].view(torch.uint8)[at].view(torch.float8_e4m3fn), s["ke"][at])
        v = _value(s["vc"].view(torch.uint8)[at].view(torch.float8_e4m3fn), s["ve"][at])
    else:
        k, v = s["k"][at].float(), s["v"][at].float()
    k = k.transpose(1, 2).reshape(batch, kv, -1, hd)                 # [B, kv, T, hd]
    v = v.transpose(1, 2).reshape(batch, kv, -1, hd)
    t = torch.arange(k.shape[2], device="cuda")
    prefix = (s["ctx"].long() - rows)[:, None, None]                 # tokens in front of the drafted ones
    draft = t[None, None, :] - prefix                                # [B, 1, T]
    bit = (s["masks"].view(batch, rows, 1) >> draft.clamp(0, 63)) & 1
    seen = (draft < 0) | ((draft < rows) & (bit == 1))               # [B, rows, T]
    q = s["q"].float().view(batch, rows, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, hd)
    p = (q @ k.transpose(2, 3) * scale).view(batch, kv, rows, heads // kv, -1)
    p.masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    o = (p.view(batch, kv, rows * (heads // kv), -1) @ v).view(batch, kv, rows, heads // kv, hd)
    return o.permute(0, 2, 1, 3, 4).reshape(batch * rows, heads * hd).to(torch.bfloat16)


def _int4(s):
    case = s["case"]
    n, k, group = case["n"], case["k"], case["group"]
    if own:
        from kotodama_b200.ops import Int4Weight
        return _ops().gemm_nt(s["x"], Int4Weight(s["packed"], s["scales"], (n, k), group))
    nt, kb = s["packed"].shape[:2]
    shift = torch.tensor([[0, 16, 8, 24], [4, 20, 12, 28]], device="cuda", dtype=torch.int32)
    c = (s["packed"].view(nt, kb, 8, 4, 4, 1, 1) >> shift) & 15      # nt, kb, r, c, j, half, input
    w = (c.permute(0, 5, 2, 1, 3, 4, 6).reshape(nt * 16, kb * 64) - 8)[:n, :k].float()
    scale = s["scales"].float().permute(0, 3, 2, 1).reshape(nt * 16, -1)[:n]
    w *= scale.repeat_interleave(group, 1)[:, :k]
    return (s["x"].float() @ w.t()).to(torch.bfloat16)


def _e4m3(v):
    """Nearest e4m3 number, ties to even, of float64 values within the type's range."""
    a = v.abs()
    e = torch.floor(torch.log2(a.clamp_min(2.0 ** -60))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return torch.sign(v) * torch.round(a / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "append":
        out = {}
        for name in ("k", "v"):
            rows = s[name].to(f64).reshape(case["tokens"], case["kv"], case["hd"])
            top = rows.abs().amax(-1, keepdim=True)
            power = torch.floor(torch.log2(top / 448.0)) - 1.0           # at most the one wanted: counted up from there
            for _ in range(3):
                power = torch.where(448.0 * torch.exp2(power) < top, power + 1.0, power)
            full = s[name + "c"].to(f64)
            for h in range(case["kv"]):
                full[s["slots"] // PAGE, h, s["slots"] % PAGE] = _e4m3(rows[:, h] / torch.exp2(power[:, h]))
            out[name], out[name + "_exp"] = full, None
        return out
    if op == "int4":
        n, k, group = case["n"], case["k"], case["group"]
        y = torch.empty(case["m"], n, dtype=f64, device="cuda")
        x = s["x"].to(f64)
        for r in range(16):                                          # one row of every block at a time
            half, lane = r // 8, r % 8
            words = s["packed"][:, :, 4 * lane:4 * lane + 4].to(torch.int64) & 0xFFFFFFFF       # nt, kb, c, j
            cols = [(words >> (4 * half + at)) % 16 for at in (0, 16, 8, 24)]
            w = torch.stack(cols, -1).flatten(1)[:, :k].to(f64) - 8.0
            part = torch.zeros(x.shape[0], w.shape[0], dtype=f64, device="cuda")
            for g in range(-(-k // group)):
                cut = slice(g * group, min(k, (g + 1) * group))
                part += (x[:, cut] @ w[:, cut].t()) * s["scales"][:, g, lane, half].to(f64)
            rows = y[:, r::16]
            rows.copy_(part[:, : rows.shape[1]])
        return y
    lens = _lengths(case)

    def rows_of(b, n, what):
        pages = s["table"][b, : -(-n // PAGE)].long()
        if what in s:
            x = s[what][pages].to(f64)
        else:
            x = s[what + "c"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(f64) * torch.exp2(s[what + "e"][pages].to(f64) - 127)[..., None]
        return x.permute(0, 2, 1, 3).reshape(-1, case["kv"], case["hd"])[:n]

    if op == "gather":
        return {w: torch.cat([rows_of(b, n, w) for b, n in enumerate(lens)]) for w in ("k", "v")}
    rows, heads, kv, hd = (case[x] for x in ("rows", "heads", "kv", "hd"))
    out = torch.empty(case["batch"] * rows, heads, hd, dtype=f64, device="cuda")
    for b, n in enumerate(lens):
        mine = slice(b * rows, (b + 1) * rows)
        seen = torch.ones(rows, n, dtype=torch.bool, device="cuda")
        for j in range(rows):
            seen[:, n - rows + j] = (s["masks"][mine] >> j) & 1 == 1
        k, v = rows_of(b, n, "k"), rows_of(b, n, "v")
        for h in range(heads):
            score = s["q"][mine, h].to(f64) @ k[:, h * kv // heads].t() / math.sqrt(hd)
            out[mine, h] = torch.softmax(score.masked_fill(~seen, float("-inf")), -1) @ v[:, h * kv // heads]
    return out.view(case["batch"] * rows, heads * hd)

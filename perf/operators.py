"""The operators a program needs that serves with trees of drafted tokens over a quantised K/V cache.

Five kinds of case, each through the public entry points of rapier_amd:

  prep     per-head norm, rotary positions with three axes, K and V written to the cache in its type; the written rows read back
  convert  a range of fp16 cache rows quantised into a cache and read back (a prompt parked after its ingest)
  tree     attention of drafted tokens (a tree by ancestor masks, or a chain) behind a context, over an fp16 / I8 / I4 cache
  compact  the accepted path's cache rows moved to the front of the draft
  logits   biases, penalties for repeated tokens and grammar masks, per column (tree node)

Sizes are those of the 9B configuration and of the benchmark's contexts, with ragged ones around them.  The quantised caches
are made here in their documented layout: codes [kv head][position][dims] (I8: code + 128 in a byte; I4: code + 8 in a nibble,
dims 2k and 2k + 1 of eight at bits 4k and 16 + 4k of a little-endian word), then the scales [kv head][position][32-dim block],
a byte b standing for the fp16 number with the bits b << 7.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e7
VOCAB = 248320
BITS = {"i8": 8, "i4": 4}
QMAX = {"i8": 127, "i4": 7}
SMAX = {"i8": 512.0, "i4": 8192.0}


def listed():
    return [
        # the new rows of one decoded token: the smallest step that writes the cache
        {"name": "prep_1tok_i8", "kind": "prep", "ktype": "i8", "vtype": "i8", "n_head": 16, "n_kv": 4, "head_dim": 256, "n_rot": 64,
         "ntok": 1, "ctx": 4096, "layout": "text"},
        # a prompt with image patches (positions of time, height and width), ingested in one go
        {"name": "prep_image_999tok_i8_i4", "kind": "prep", "ktype": "i8", "vtype": "i4", "n_head": 16, "n_kv": 4, "head_dim": 256,
         "n_rot": 64, "ntok": 999, "ctx": 4001, "layout": "image"},
        # the cache rows of a 4K prompt, after an fp16 ingest
        {"name": "convert_4k_i8", "kind": "convert", "type": "i8", "n_kv": 4, "head_dim": 256, "rows": 4001, "src": "f16"},
        # the same behind the longest context of the benchmark, at four bits
        {"name": "convert_64k_i4", "kind": "convert", "type": "i4", "n_kv": 4, "head_dim": 256, "rows": 65501, "src": "f16"},
        # one decoded token behind a long context: bound by the cache
        {"name": "decode_64k_i4", "kind": "tree", "ktype": "i4", "vtype": "i4", "n_head": 16, "n_kv": 4, "head_dim": 256, "ntok": 1,
         "ctx": 65501, "tree": False},
        # a tree of eight drafted tokens behind the same
        {"name": "tree_8tok_64k_i8", "kind": "tree", "ktype": "i8", "vtype": "i8", "n_head": 16, "n_kv": 4, "head_dim": 256, "ntok": 8,
         "ctx": 65501, "tree": True},
        # the widest tree over the engine's fp16 cache, 4K tokens into a text
        {"name": "tree_64tok_4k_f16", "kind": "tree", "ktype": "f16", "vtype": "f16", "n_head": 16, "n_kv": 4, "head_dim": 256, "ntok": 64,
         "ctx": 4001, "tree": True},
        # a prompt chunk over a mixed cache: the most arithmetic
        {"name": "chunk_999tok_8k_i8_i4", "kind": "tree", "ktype": "i8", "vtype": "i4", "n_head": 16, "n_kv": 4, "head_dim": 256,
         "ntok": 999, "ctx": 8001, "tree": False},
        # an accepted path over the fp16 caches of eight layers
        {"name": "compact_8layers_f16", "kind": "compact", "type": "f16", "n_kv": 4, "head_dim": 256, "caches": 16, "ntok": 16, "path": 5,
         "ctx": 4001},
        # the longest path over one layer's quantised caches
        {"name": "compact_path31_i4", "kind": "compact", "type": "i4", "n_kv": 4, "head_dim": 256, "caches": 2, "ntok": 64, "path": 31,
         "ctx": 65501},
        # the logits of one decoded token: penalties over a long history, some biases
        {"name": "logits_1col", "kind": "logits", "vocab": VOCAB, "ncols": 1, "history": 4001, "window": 0, "biases": 37, "grammar": False},
        # the logits of a tree's nodes under a grammar
        {"name": "logits_16col_grammar", "kind": "logits", "vocab": VOCAB, "ncols": 16, "history": 1999, "window": 256, "biases": 300,
         "grammar": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _types(rng):
    return rng.choice([("f16", "f16"), ("i8", "i8"), ("i8", "i8"), ("i8", "i4"), ("i4", "i4")])


def _heads(rng):
    n_kv, group, head_dim = rng.choice([(4, 4, 256), (4, 4, 256), (2, 4, 256), (8, 4, 128), (2, 8, 128), (3, 2, 256), (1, 5, 128)])
    return {"n_head": n_kv * group, "n_kv": n_kv, "head_dim": head_dim}


def draw(rng):
    kind = rng.choice(["prep", "convert", "tree", "tree", "tree", "compact", "logits", "logits"])
    h = _heads(rng)
    if kind == "prep":
        kt, vt = rng.choice([("f16", "f16"), ("i8", "i8"), ("i8", "i4")])
        return {"kind": kind, "ktype": kt, "vtype": vt, **h, "n_rot": rng.choice([64, 64, h["head_dim"]]), "ntok": _log(rng, 1, 999),
                "ctx": _log(rng, 1, 65501), "layout": rng.choice(["text", "tree", "image"])}
    if kind == "convert":
        return {"kind": kind, "type": rng.choice(["i8", "i4"]), "n_kv": h["n_kv"], "head_dim": h["head_dim"],
                "rows": _log(rng, 1, 65501 * 1024 // (h["n_kv"] * h["head_dim"]) // 2), "src": rng.choice(["f16", "f32"])}
    if kind == "tree":
        kt, vt = _types(rng)
        tree = rng.random() < 0.6
        ntok = rng.choice([1, 2, _log(rng, 3, 64), _log(rng, 3, 64)]) if tree else rng.choice([1, 2, _log(rng, 3, 999)])
        ctx = _log(rng, 1, min(65501, 999 * 8001 // ntok * 8 // h["n_head"]))
        return {"kind": kind, "ktype": kt, "vtype": vt, **h, "ntok": ntok, "ctx": ctx, "tree": tree}
    if kind == "compact":
        ntok = rng.randint(4, 64)
        return {"kind": kind, "type": rng.choice(["f16", "i8", "i4"]), "n_kv": h["n_kv"], "head_dim": h["head_dim"],
                "caches": 2 * rng.choice([1, 1, 2, 4]), "ntok": ntok, "path": rng.randint(1, ntok // 2), "ctx": _log(rng, 1, 65501)}
    return {"kind": kind, "vocab": _log(rng, 999, VOCAB), "ncols": rng.choice([1, 1, 2, rng.randint(3, 64)]), "history": _log(rng, 1, 20001),
            "window": rng.choice([0, 64, _log(rng, 1, 4096)]), "biases": rng.choice([0, _log(rng, 1, 300)]), "grammar": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std + mean


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantise(x, type_):
    """float rows [..., dims] -> (codes in float64, scales in float64), decided in 64 bits (codes lie next to borders)"""
    b = x.double().unflatten(-1, (-1, 32))
    t = b.abs().amax(-1, keepdim=True) / QMAX[type_]
    exponent = torch.frexp(t).exponent.long() - 4   # four significant bits, but for the grid's smallest numbers
    step = ((exponent.clamp_min(-17) + 1023) << 52).view(torch.float64)
    s = (torch.ceil(t / step) * step).clamp_max(SMAX[type_])
    q = torch.round(b / torch.where(s > 0, s, torch.ones_like(s))).clamp(-QMAX[type_], QMAX[type_])
    return q, s


def _value(x, type_):
    """the float64 values a cache of the type holds for the rows x"""
    if type_ == "f16":
        return x.to(torch.float32).to(torch.float16).double()
    q, s = _quantise(x, type_)
    return (q * s).flatten(-2)


def _cache(x, type_):
    """rows [positions, kv heads, dims] -> a cache of the type in its layout"""
    if type_ == "f16":
        return x.to(torch.float16).contiguous()
    x = x.transpose(0, 1).contiguous()
    codes, scales = [], []
    for head in x:   # by head: the 64-bit steps of a long cache are large
        q, s = _quantise(head, type_)
        q = q.flatten(-2).to(torch.int32) + (QMAX[type_] + 1)
        if type_ == "i4":
            e = q.unflatten(-1, (-1, 4, 2))   # groups of eight dims: [k][parity]
            k = torch.arange(4, device=q.device, dtype=torch.int32) * 4
            q = ((e[..., 0] << k) | (e[..., 1] << (k + 16))).sum(-1)
            q = torch.stack([(q >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2)
        codes.append(q.to(torch.uint8).reshape(-1))
        scales.append((s.flatten(-2).to(torch.float16).view(torch.int16) >> 7).to(torch.uint8).reshape(-1))
    return torch.cat(codes + scales)


def _rows_of(cache, type_, first, n, n_kv, head_dim, max_ctx):
    """rows [first, first + n) of a cache: float32 [kv head][n][dims]"""
    if type_ == "f16":
        return cache[first:first + n].transpose(0, 1).float().contiguous()
    width = head_dim * BITS[type_] // 8
    codes = cache[:n_kv * max_ctx * width].view(n_kv, max_ctx, width)[:, first:first + n]
    scales = cache[n_kv * max_ctx * width:].view(n_kv, max_ctx, head_dim // 32)[:, first:first + n]
    s = (scales.to(torch.int16) << 7).view(torch.float16).float().repeat_interleave(32, -1)
    if type_ == "i4":
        w = codes.to(torch.int32).unflatten(-1, (-1, 4))
        k = torch.arange(4, device=codes.device, dtype=torch.int32) * 4
        low, high = w[..., 0] | (w[..., 1] << 8), w[..., 2] | (w[..., 3] << 8)
        codes = torch.stack([(low.unsqueeze(-1) >> k) & 15, (high.unsqueeze(-1) >> k) & 15], -1).flatten(-3)
    return (codes.float() - (QMAX[type_] + 1)) * s


def _bytes(type_, max_ctx, n_kv, head_dim):
    return n_kv * max_ctx * (head_dim * BITS[type_] // 8 + head_dim // 32)


def _empty_cache(type_, max_ctx, n_kv, head_dim):
    if type_ == "f16":
        return torch.zeros(max_ctx, n_kv, head_dim, dtype=torch.float16, device="cuda")
    return torch.zeros(_bytes(type_, max_ctx, n_kv, head_dim), dtype=torch.uint8, device="cuda")


def _tree(rng, n):
    """ancestor masks (own bit set) of a random tree of n nodes in an order with parents first, as int64 bit patterns"""
    masks, depth = [], []
    for i in range(n):
        p = int(rng.integers(max(-1, i - 12), i)) if i else -1
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return [m - (1 << 64) if m >> 63 else m for m in masks], depth


def _axis_positions(rng, case):
    n, ctx = case["ntok"], case["ctx"]
    if case["layout"] == "text":
        return [[ctx + t for t in range(n)]] * 3
    if case["layout"] == "tree":
        return [[ctx + d for d in _tree(rng, n)[1]]] * 3
    w = max(1, int(math.sqrt(n)))
    return [[ctx] * n, [ctx + t // w for t in range(n)], [ctx + t % w for t in range(n)]]


def _sections(n_rot):
    half = n_rot // 2
    a = half // 3
    return (half - 2 * a, a, a)


def _capacity(case):
    return (case["ctx"] + case["ntok"] + 63) // 64 * 64


def prepare(case, seed):
    c, g, rng = case, _gen(seed), np.random.default_rng(seed)
    s = {"case": c, "handle": _handle(c)}
    if c["kind"] == "convert":
        n, kv, hd = c["rows"], c["n_kv"], c["head_dim"]
        s["src"] = _normal(g, n, kv, hd)
        if c["src"] == "f16":
            s["src"] = s["src"].to(torch.float16)
        s["cache"] = _empty_cache(c["type"], n, kv, hd)
        s["out"] = torch.empty(n, kv, hd, dtype=torch.float16, device="cuda")
        return s
    if c["kind"] == "logits":
        v, n, h = c["vocab"], c["ncols"], c["history"]
        s["logits"] = _normal(g, n, v, std=3.0)
        # a text's tokens repeat: ranks of a heavy-tailed distribution
        s["history"] = torch.from_numpy((np.minimum(rng.zipf(1.3, h), v) - 1).astype(np.int32)).cuda()
        s["history_len"] = _ints(h)
        s["draft"] = torch.from_numpy((np.minimum(rng.zipf(1.3, n), v) - 1).astype(np.int32)).cuda()
        s["masks"] = torch.tensor(_tree(rng, n)[0], dtype=torch.int64, device="cuda")
        ids = rng.choice(v, min(c["biases"], v), replace=False).astype(np.int32)
        s["bias_ids"], s["bias_vals"] = torch.from_numpy(ids).cuda(), _normal(g, len(ids), std=5.0)
        s["allow"] = None
        if c["grammar"]:
            s["allow"] = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), generator=g, device="cuda").to(torch.int32)
        s["out"] = torch.empty_like(s["logits"])
        return s
    kv, hd, n, ctx = c["n_kv"], c["head_dim"], c["ntok"], c["ctx"]
    rows = _capacity(c)
    s["rows"], s["pos"] = rows, _ints(ctx)
    if c["kind"] == "compact":
        # sources behind the destinations, so that another pass over the same state finds the same rows
        src = np.sort(rng.choice(np.arange(c["path"], n), c["path"], replace=False))
        s["path"], s["count"] = torch.from_numpy(src.astype(np.int32)).cuda(), _ints(c["path"])
        s["caches"] = [_empty_cache(c["type"], rows, kv, hd) for _ in range(c["caches"])]
        for k in range(c["caches"]):
            x = _normal(g, n, kv, hd)
            if c["type"] == "f16":
                s["caches"][k][ctx:ctx + n] = x.to(torch.float16)
                continue
            width = hd * BITS[c["type"]] // 8
            small = _cache(x, c["type"])
            for at, per in ((0, width), (n * kv * width, hd // 32)):
                whole = s["caches"][k][at // n * rows:at // n * rows + kv * rows * per].view(kv, rows, per)
                whole[:, ctx:ctx + n] = small[at:at + kv * n * per].view(kv, n, per)
        s["out"] = [torch.empty(c["path"], kv, hd, dtype=torch.float16, device="cuda") for _ in s["caches"]]
        return s
    nh = c["n_head"]
    width = 2 * nh * hd + 2 * kv * hd
    s["q3"] = _normal(g, n, width)
    s["y"] = torch.empty(n, nh, hd, device="cuda")
    if c["kind"] == "prep":
        s["qn"], s["kn"] = _normal(g, hd, mean=1.0, std=0.1), _normal(g, hd, mean=1.0, std=0.1)
        s["axis_pos"] = torch.tensor(_axis_positions(rng, c), dtype=torch.int32, device="cuda")
        s["k"], s["v"] = (_empty_cache(c[t], rows, kv, hd) for t in ("ktype", "vtype"))
        s["krows"], s["vrows"] = (torch.empty(n, kv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    s["q"] = _normal(g, n, nh, hd)
    s["k"], s["v"] = (_cache(_normal(g, rows, kv, hd), c[t]) for t in ("ktype", "vtype"))
    s["masks"] = torch.tensor(_tree(rng, n)[0], dtype=torch.int64, device="cuda") if c["tree"] else None
    if s["handle"]:
        s["nsub"], need = s["handle"]
        s["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    return s


def _handle(c):
    """what a program settles once for its sizes: the split of the context and the workspace that it needs"""
    if not own or c["kind"] != "tree":
        return None
    import rapier_amd as rmi
    nsub = rmi.gqa_tree_nsub(c["ctx"] + c["ntok"], c["n_head"], c["n_kv"], c["head_dim"], c["ntok"])
    return nsub, rmi.gqa_tree_workspace_bytes(_capacity(c), c["n_head"], c["n_kv"], c["head_dim"], c["ntok"], nsub)


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    return _kernels(state) if own else _plain(state)


def _kernels(s):
    import rapier_amd as rmi
    c = s["case"]
    types = {"f16": rmi.KV_F16, "i8": rmi.KV_I8, "i4": rmi.KV_I4}
    if c["kind"] == "logits":
        rmi.logits_process(s["logits"], c["vocab"], c["ncols"], c["vocab"], s["out"], c["vocab"], s["history"], s["history_len"], c["history"],
                           c["window"], s["draft"], s["masks"], c["ncols"], 1.15, 0.25, 0.125, s["bias_ids"], s["bias_vals"],
                           s["bias_ids"].numel(), s["allow"], (c["vocab"] + 31) // 32)
        return s["out"]
    kv, hd = c["n_kv"], c["head_dim"]
    if c["kind"] == "convert":
        n = c["rows"]
        rmi.kv_write(types[c["type"]], s["src"], kv * hd, s["cache"], 0, n, kv, hd, n)
        rmi.kv_read(types[c["type"]], s["cache"], s["out"], kv * hd, 0, n, kv, hd, n)
        return s["out"]
    rows, ctx, n = s["rows"], c["ctx"], c["ntok"]
    if c["kind"] == "compact":
        rmi.kv_compact(types[c["type"]], s["caches"], s["pos"], s["path"], s["count"], c["path"], kv, hd, rows)
        if c["type"] == "f16":
            return [x[ctx:ctx + c["path"]] for x in s["caches"]]
        for cache, out in zip(s["caches"], s["out"]):
            rmi.kv_read(types[c["type"]], cache, out, kv * hd, ctx, c["path"], kv, hd, rows)
        return s["out"]
    nh, width = c["n_head"], s["q3"].shape[1]
    kt, vt = types[c["ktype"]], types[c["vtype"]]
    if c["kind"] == "prep":
        rmi.attn_prep_axes(s["q3"], width, s["qn"], s["kn"], kt, s["k"], vt, s["v"], s["pos"], s["axis_pos"], s["y"], nh, kv, hd, c["n_rot"],
                           THETA, 1.0, 0.0, _sections(c["n_rot"]), True, EPS, n, rows)
        rmi.kv_read(kt, s["k"], s["krows"], kv * hd, ctx, n, kv, hd, rows)
        rmi.kv_read(vt, s["v"], s["vrows"], kv * hd, ctx, n, kv, hd, rows)
        return {"q": s["y"], "k": s["krows"], "v": s["vrows"]}
    rmi.gqa_tree_decode(s["q"], kt, s["k"], vt, s["v"], s["pos"], s["masks"], s["q3"], width, s["y"], nh * hd, None, 0, s["ws"], nh, kv, hd, n,
                        rows, s["nsub"], 1.0 / math.sqrt(hd))
    return s["y"]


def _plain(s):
    c = s["case"]
    if c["kind"] == "logits":
        v, n = c["vocab"], c["ncols"]
        bit = ((s["masks"].unsqueeze(1) >> torch.arange(n, device="cuda")) & 1).bool()   # [column][draft token]
        at = torch.arange(c["history"], device="cuda")
        first = c["history"] + bit.sum(1, keepdim=True) - c["window"] if c["window"] > 0 else torch.zeros(n, 1, dtype=torch.int64, device="cuda")
        order = bit.cumsum(1) - 1 + c["history"]   # the place of a path's token in the column's text
        ids = torch.cat([s["history"], s["draft"]]).long().expand(n, -1)
        seen = torch.cat([(at >= first), bit & (order >= first)], 1).float()
        count = torch.zeros(n, v, device="cuda").scatter_add_(1, ids, seen)
        x = s["logits"].clone()
        x[:, s["bias_ids"].long()] += s["bias_vals"]
        x = torch.where(count > 0, torch.where(x > 0, x / 1.15, x * 1.15), x)
        x = x - count * 0.125 - (count > 0).float() * 0.25
        if s["allow"] is not None:
            word = s["allow"].repeat_interleave(32, 1)[:, :v]
            ok = (word >> (torch.arange(v, device="cuda", dtype=torch.int32) % 32)) & 1
            x = x.masked_fill(ok == 0, -math.inf)
        return x
    kv, hd = c["n_kv"], c["head_dim"]
    if c["kind"] == "convert":
        return torch.cat([_value(x, c["type"]).to(torch.float16) for x in s["src"].split(16384)])
    n, ctx = c["ntok"], c["ctx"]
    if c["kind"] == "compact":
        out = []
        for cache in s["caches"]:
            x = _rows_of(cache, c["type"], ctx, n, kv, hd, s["rows"])[:, s["path"].long()].to(torch.float16).transpose(0, 1).contiguous()
            if c["type"] == "f16":
                cache[ctx:ctx + c["path"]] = x
            out.append(x)
        return out
    nh = c["n_head"]
    if c["kind"] == "prep":
        half = c["n_rot"] // 2
        i = torch.arange(half, device="cuda")
        _, s1, s2 = _sections(c["n_rot"])
        axis = torch.where((i % 3 == 1) & (i < 3 * s1), 1, torch.where((i % 3 == 2) & (i < 3 * s2), 2, 0))
        angle = s["axis_pos"].double()[axis].t() * torch.exp(i.double() * (-2.0 * math.log(THETA) / c["n_rot"]))
        cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)   # [token][1][pair]

        def normed(x, w):   # in 64 bits: the rows are quantised after it, next to borders
            x = x.double()
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
            a, b = x[..., :half], x[..., half:2 * half]
            return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1).float()

        q = s["q3"][:, :2 * nh * hd].view(n, nh, 2, hd)[:, :, 0]
        k, v = s["q3"][:, 2 * nh * hd:].view(n, 2, kv, hd).unbind(1)
        return {"q": normed(q, s["qn"]), "k": _value(normed(k, s["kn"]), c["ktype"]).to(torch.float16),
                "v": _value(v, c["vtype"]).to(torch.float16)}
    group = nh // kv
    k = _rows_of(s["k"], c["ktype"], 0, ctx + n, kv, hd, s["rows"])
    v = _rows_of(s["v"], c["vtype"], 0, ctx + n, kv, hd, s["rows"])
    q = s["q"].view(n, kv, group, hd).permute(1, 0, 2, 3).reshape(kv, n * group, hd)
    score = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv, n, group, ctx + n) / math.sqrt(hd)
    j = torch.arange(n, device="cuda")
    seen = ((s["masks"].unsqueeze(1) >> j) & 1).bool() if c["tree"] else j.unsqueeze(1) >= j
    score[..., ctx:] = score[..., ctx:].masked_fill(~seen.unsqueeze(1), -math.inf)
    score -= score.amax(-1, keepdim=True)
    score = score.exp_()
    o = torch.matmul(score.view(kv, n * group, ctx + n), v).view(kv, n, group, hd) / score.sum(-1, keepdim=True)
    gate = s["q3"][:, :2 * nh * hd].view(n, nh, 2, hd)[:, :, 1]
    return o.permute(1, 0, 2, 3).reshape(n, nh, hd) / (1 + torch.exp(-gate))


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _grid(type_):
    """every scale, in order: (8 + m) 2^(e - 18), or m 2^-17 for e = 0"""
    g = [math.ldexp(m if e == 0 else 8 + m, -17 if e == 0 else e - 18) for e in range(31) for m in range(8)]
    return torch.tensor([x for x in g if x <= SMAX[type_]], dtype=torch.float64, device="cuda")


def _held(x, type_):
    """what a cache of the type holds for float64 rows: the smallest scale that reaches the block's maximum, by search"""
    if type_ == "f16":
        return x.to(torch.float16).double()
    grid, m = _grid(type_), QMAX[type_]
    out = torch.empty_like(x)
    for part, to in zip(x.split(8192), out.split(8192)):
        blocks = part.reshape(-1, 32)
        at = torch.searchsorted(grid * m, blocks.abs().max(1).values).clamp_max(len(grid) - 1)
        s = grid[at].unsqueeze(1)
        q = torch.where(s > 0, blocks / s, 0.0 * blocks)
        to.copy_((q.round().clamp(-m, m) * s).view(part.shape))
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "logits":
        hist, draft, out = s["history"].cpu().numpy(), s["draft"].cpu().numpy(), []
        masks, logits = s["masks"].tolist(), s["logits"].cpu().numpy().astype(np.float64)
        ids, vals = s["bias_ids"].cpu().numpy(), s["bias_vals"].cpu().numpy().astype(np.float64)
        allow = None if s["allow"] is None else np.unpackbits(s["allow"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")
        for col in range(c["ncols"]):
            text = np.concatenate([hist, [draft[j] for j in range(c["ncols"]) if masks[col] >> j & 1]]).astype(np.int64)
            n = np.bincount(text[-c["window"]:] if c["window"] else text, minlength=c["vocab"])
            x = logits[col]
            np.add.at(x, ids, vals)
            hit = n > 0
            x[hit] = np.where(x[hit] > 0, x[hit] / np.float64(np.float32(1.15)), x[hit] * np.float64(np.float32(1.15)))
            x[hit] -= 0.25 + 0.125 * n[hit]
            if allow is not None:
                x[allow[col, :c["vocab"]] == 0] = -math.inf
            out.append(x)
        return torch.from_numpy(np.stack(out))
    kv, hd = c["n_kv"], c["head_dim"]
    if c["kind"] == "convert":
        return _held(s["src"].double(), c["type"])
    n, ctx = c["ntok"], c["ctx"]
    if c["kind"] == "compact":
        out = []
        for cache in s["caches"]:
            rows = _rows_64(cache, c["type"], s["rows"], kv, hd, ctx, ctx + n)
            out.append(torch.stack([rows[:, p] for p in s["path"].tolist()]))
        return out
    nh = c["n_head"]
    if c["kind"] == "prep":
        x = s["q3"].double()
        heads = x[:, :2 * nh * hd].reshape(n, nh, 2 * hd)[..., :hd]
        kv_rows = x[:, 2 * nh * hd:].reshape(n, 2 * kv, hd)
        sec = _sections(c["n_rot"])
        axes = [a if a and i < 3 * sec[a] else 0 for i in range(c["n_rot"] // 2) for a in (i % 3,)]
        freq = torch.tensor([THETA ** (-2.0 * i / c["n_rot"]) for i in range(len(axes))], dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones_like(freq), s["axis_pos"].double()[axes].T * freq).unsqueeze(1)

        def rotated(r, w):
            r = r * w.double() * torch.rsqrt((r * r).sum(-1, keepdim=True) / hd + EPS)
            pair = torch.complex(r[..., :len(axes)].contiguous(), r[..., len(axes):2 * len(axes)].contiguous()) * turn
            return torch.cat([pair.real, pair.imag, r[..., 2 * len(axes):]], -1)

        # the definition rounds a K row to fp32 once, before it is quantised
        return {"q": rotated(heads, s["qn"]), "k": _held(rotated(kv_rows[:, :kv], s["kn"]).float().double(), c["ktype"]),
                "v": _held(kv_rows[:, kv:].contiguous(), c["vtype"])}
    group, total = nh // kv, ctx + n
    out = torch.empty(n, nh, hd, dtype=torch.float64, device="cuda")
    masks = s["masks"].tolist() if c["tree"] else None
    unseen = torch.zeros(n, total, dtype=torch.bool)
    for t in range(n):
        for j in range(n):
            unseen[t, ctx + j] = not masks[t] >> j & 1 if c["tree"] else j > t
    unseen = unseen.cuda()
    for h in range(kv):
        k = _rows_64(s["k"], c["ktype"], s["rows"], kv, hd, 0, total)[h].t().contiguous()
        v = _rows_64(s["v"], c["vtype"], s["rows"], kv, hd, 0, total)[h].contiguous()
        for i in range(h * group, (h + 1) * group):
            w = (s["q"][:, i].double() @ k * hd ** -0.5).masked_fill_(unseen, -math.inf)
            out[:, i] = torch.exp(w - torch.logsumexp(w, 1, keepdim=True)) @ v
    gate = s["q3"][:, :2 * nh * hd].reshape(n, nh, 2 * hd)[..., hd:].double()
    return out * torch.sigmoid(gate)


def _rows_64(cache, type_, max_ctx, n_kv, head_dim, first, last):
    """cache rows in float64 [kv head][rows][dims], decoded code by code"""
    if type_ == "f16":
        return cache[first:last].double().transpose(0, 1)
    per = head_dim * BITS[type_] // 8
    raw, scale = cache[:n_kv * max_ctx * per], cache[n_kv * max_ctx * per:]
    raw = raw.reshape(n_kv, max_ctx, per)[:, first:last].long()
    scale = scale.reshape(n_kv, max_ctx, -1)[:, first:last].long()
    full = torch.tensor([math.ldexp(b % 8 if b < 8 else 8 + b % 8, -17 if b < 8 else b // 8 - 18) for b in range(248)], dtype=torch.float64,
                        device="cuda")
    if type_ == "i4":
        d = torch.arange(head_dim, device="cuda")
        bit = 4 * (d % 8 // 2) + 16 * (d % 2)   # of the word of the dim's eight
        raw = raw[..., d // 8 * 4 + bit // 8] >> (bit % 8) & 15
    return (raw - (QMAX[type_] + 1)).double() * full[scale][..., torch.arange(head_dim, device="cuda") // 32]


def work(case):
    c = case
    if c["kind"] == "logits":
        n, v = c["ncols"], c["vocab"]
        return {"bytes": n * v * 8 + (n * v // 8 if c["grammar"] else 0) + 4 * c["history"] + 8 * c["biases"], "flops": 6 * n * v}
    kv, hd = c["n_kv"], c["head_dim"]

    def row(t):
        return kv * (hd * 2 if t == "f16" else hd * BITS[t] // 8 + hd // 32)

    if c["kind"] == "convert":
        n = c["rows"]
        return {"bytes": n * (kv * hd * ((2 if c["src"] == "f16" else 4) + 2) + 2 * row(c["type"])), "flops": 6 * n * kv * hd}
    if c["kind"] == "compact":
        back = 0 if c["type"] == "f16" else row(c["type"]) + 2 * kv * hd
        return {"bytes": c["caches"] * c["path"] * (2 * row(c["type"]) + back), "flops": 0}
    n, nh = c["ntok"], c["n_head"]
    if c["kind"] == "prep":
        return {"bytes": n * (4 * (nh * hd + 2 * kv * hd) + 4 * nh * hd + 2 * (row(c["ktype"]) + row(c["vtype"])) + 4 * kv * hd),
                "flops": 12 * n * (nh + 2 * kv) * hd}
    keys = c["ctx"] * n + n * (n + 1) // 2   # seen keys of all tokens (a tree's masks leave out some of the draft)
    return {"bytes": (c["ctx"] + n) * (row(c["ktype"]) + row(c["vtype"])) + 12 * n * nh * hd, "flops": 4 * keys * nh * hd}

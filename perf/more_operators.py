"""The operators a program needs that serves several requests at once, their K/V caches in pages of one pool.

Five kinds of case, each through the public entry points of rapier_amd:

  plan    row starts, lengths, slots and positions of a batch's new tokens, and the pages they need, from the requests' lengths
  trim    the pages past the lengths that requests keep (rejected drafts, ended requests), back to the free list
  prep    per-head norm and rotation of new q and k rows, q out in 16 bits, K and V to their slots
  paged   attention of new tokens (single ones, drafts, prompt chunks, or a mix) over their requests' pages
  prompt  causal attention over whole prompts of different lengths, packed row by row, without a cache

Heads and contexts are those of the 9B configuration and of the benchmark, with ragged ones around them.  A page is a cache of
page_size positions in the framework's layout: F16 [position][kv head][dim]; I8 codes (code + 128 in a byte) or I4 codes (code +
8 in a nibble, dims 2k and 2k + 1 of eight at bits 4k and 16 + 4k of a little-endian word) as [kv head][position][dims], then the
scales [kv head][position][32-dim block], a byte b standing for the fp16 number with the bits b << 7.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e7
YARN = {"factor": 4.0, "orig_ctx": 262144.0, "beta_fast": 32.0, "beta_slow": 1.0}
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}
BITS = {"i8": 8, "i4": 4}
QMAX = {"i8": 127, "i4": 7}
SMAX = {"i8": 512.0, "i4": 8192.0}
MODEL = {"n_head": 16, "n_kv": 4, "head_dim": 256}


def listed():
    return [
        # a decode round of 32 requests: one token each, now and then a page
        {"name": "plan_32req_decode", "kind": "plan", "reqs": 32, "page": 64, "ctx": 4096, "new": 1, "mix": "each", "spare": 1.0},
        # a busy round: 999 requests, a few prompts among single tokens, more pages asked for than there are
        {"name": "plan_999req_mixed", "kind": "plan", "reqs": 999, "page": 16, "ctx": 8001, "new": 1999, "mix": "some", "spare": 0.9},
        # the rejected drafts of 32 requests
        {"name": "trim_32req_drafts", "kind": "trim", "reqs": 32, "page": 16, "ctx": 4096, "drop": "draft"},
        # requests that end, among many that go on
        {"name": "trim_999req_ended", "kind": "trim", "reqs": 999, "page": 16, "ctx": 8001, "drop": "some"},
        # the new rows of a decode round, to quantised pages
        {"name": "prep_32tok_i8", "kind": "prep", "qtype": "f16", "ktype": "i8", "vtype": "i8", **MODEL, "n_rot": 64, "pairs": "half",
         "yarn": False, "tokens": 32, "page": 64, "ctx": 4096},
        # a packed prompt batch at far positions, scaled rotation, neighbouring pairs, bf16 q
        {"name": "prep_1999tok_f16_yarn", "kind": "prep", "qtype": "bf16", "ktype": "f16", "vtype": "f16", **MODEL, "n_rot": 64,
         "pairs": "neighbours", "yarn": True, "tokens": 1999, "page": 64, "ctx": 65536},
        # a decode round over 4K contexts of different lengths: bound by the cache
        {"name": "decode_32req_4k_f16", "kind": "paged", "qtype": "f16", "ktype": "f16", "vtype": "f16", **MODEL, "page": 64, "reqs": 32,
         "ctx": 4096, "new": 1, "mix": "each", "gate": True},
        # one request alone behind a long context, in pages of 16 (what is split)
        {"name": "decode_1req_64k_i8", "kind": "paged", "qtype": "bf16", "ktype": "i8", "vtype": "i8", **MODEL, "page": 16, "reqs": 1,
         "ctx": 65501, "new": 1, "mix": "each", "gate": True},
        # a prompt chunk of one request beside the single tokens of 15 others, mixed cache
        {"name": "mixed_999tok_8k_i8_i4", "kind": "paged", "qtype": "f16", "ktype": "i8", "vtype": "i4", **MODEL, "page": 64, "reqs": 16,
         "ctx": 8001, "new": 999, "mix": "first", "gate": True},
        # a short prompt alone: too few rows to fill the card
        {"name": "prompt_500tok_f16", "kind": "prompt", "type": "f16", **MODEL, "reqs": 1, "tokens": 500, "gate": True},
        # a batch of prompts of different lengths, packed
        {"name": "prompt_23req_8001tok_bf16", "kind": "prompt", "type": "bf16", **MODEL, "reqs": 23, "tokens": 8001, "gate": True},
        # a long prompt: the most arithmetic
        {"name": "prompt_8001tok_f16", "kind": "prompt", "type": "f16", **MODEL, "reqs": 1, "tokens": 8001, "gate": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    n_kv, group, head_dim = rng.choice([(4, 4, 256), (4, 4, 256), (2, 4, 256), (8, 4, 128), (2, 8, 128), (3, 3, 256), (1, 5, 128)])
    return {"n_head": n_kv * group, "n_kv": n_kv, "head_dim": head_dim}


def draw(rng):
    kind = rng.choice(["plan", "trim", "prep", "prep", "paged", "paged", "paged", "prompt", "prompt"])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    if kind == "plan":
        mix = rng.choice(["each", "some"])
        return {"kind": kind, "reqs": _log(rng, 1, 999), "page": page, "ctx": _log(rng, 16, 8001), "new": rng.randint(1, 16) if mix == "each" else
                _log(rng, 2, 1999), "mix": mix, "spare": rng.choice([0.8, 1.0, 1.1])}
    if kind == "trim":
        return {"kind": kind, "reqs": _log(rng, 1, 999), "page": page, "ctx": _log(rng, 16, 8001), "drop": rng.choice(["draft", "some"])}
    h = _heads(rng)
    kt, vt = rng.choice([("f16", "f16"), ("f16", "f16"), ("i8", "i8"), ("i8", "i4"), ("i4", "i4")])
    if kind == "prep":
        return {"kind": kind, "qtype": rng.choice(["f16", "bf16"]), "ktype": kt, "vtype": vt, **h, "n_rot": rng.choice([64, 64, h["head_dim"]]),
                "pairs": rng.choice(["half", "neighbours"]), "yarn": rng.random() < 0.5, "tokens": _log(rng, 1, 1999), "page": page,
                "ctx": _log(rng, 2000, 65536)}
    gate = rng.random() < 0.5
    if kind == "paged":
        mix = rng.choice(["each", "each", "first"])
        reqs = _log(rng, 1, 64)
        new = _log(rng, 1, 16) if mix == "each" else _log(rng, 2, 999)
        reqs = min(reqs, 16) if mix == "first" else reqs
        # positions of all requests, and tokens of the longest chunk times its context
        ctx = max(new, _log(rng, 16, min(65501, 32 * 4096 // reqs, 999 * 8001 // new)))
        return {"kind": kind, "qtype": rng.choice(["f16", "bf16"]), "ktype": kt, "vtype": vt, **h, "page": page, "reqs": reqs, "ctx": ctx,
                "new": new, "mix": mix, "gate": gate}
    return {"kind": kind, "type": rng.choice(["f16", "bf16"]), **h, "reqs": rng.choice([1, 1, _log(rng, 2, 40)]), "tokens": _log(rng, 40, 8001),
            "gate": gate}


# ---- sizes of a case --------------------------------------------------------------------------------------------------
def _lengths(case):
    """(past, count) of every request, from the case alone: the work is the same for every seed"""
    c = case
    rng = random.Random("%s %d %d" % (c["kind"], c["reqs"], c.get("ctx", c.get("tokens", 0))))
    n = c["reqs"]
    if c["kind"] == "prompt":
        cuts = sorted(rng.sample(range(1, c["tokens"]), n - 1))
        return [0] * n, [b - a for a, b in zip([0] + cuts, cuts + [c["tokens"]])]
    total = [c["ctx"]] + [rng.randint(c["ctx"] // 4, c["ctx"]) for _ in range(n - 1)]
    if c["kind"] == "trim":
        if c["drop"] == "draft":
            return total, [max(0, t - rng.randint(0, 16)) for t in total]
        return total, [t if rng.random() < 0.8 else 0 for t in total]
    if c["mix"] == "each":
        count = [c["new"]] * n
    elif c["mix"] == "first":
        count = [c["new"]] + [1] * (n - 1)
    else:
        count = [rng.choice([0, 1, 1, 1, 1, 1, 1, rng.randint(1, c["new"])]) for _ in range(n)]
    if c["kind"] == "paged":
        return [max(0, t - k) for t, k in zip(total, count)], [min(t, k) for t, k in zip(total, count)]
    return total, count


def _pages(n, page):
    return (n + page - 1) // page


def _row_bytes(type_, head_dim):
    return head_dim * 2 if type_ == "f16" else head_dim * BITS[type_] // 8 + head_dim // 32


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std + mean


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


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
    """the values a cache of the type holds for the fp32 rows x, in fp16 (which holds them exactly)"""
    if type_ == "f16":
        return x.to(torch.float16)
    q, s = _quantise(x, type_)
    return (q * s).flatten(-2).to(torch.float16)


def _pool(g, type_, n_pages, page, n_kv, head_dim):
    """a pool of pages with rows of normal values, one byte row a page"""
    out = torch.empty(n_pages, page * n_kv * _row_bytes(type_, head_dim), dtype=torch.uint8, device="cuda")
    for at in range(0, n_pages, 4096 // page * 16):   # by pieces: the 64-bit steps of a large pool are large
        to = out[at:at + 4096 // page * 16]
        if type_ == "f16":
            to.copy_(_normal(g, len(to), page, n_kv, head_dim).to(torch.float16).view(torch.uint8).view(len(to), -1))
            continue
        q, s = _quantise(_normal(g, len(to), n_kv, page, head_dim), type_)
        q = q.flatten(-2).to(torch.int32) + (QMAX[type_] + 1)
        if type_ == "i4":
            e = q.unflatten(-1, (-1, 4, 2))   # groups of eight dims: [k][parity]
            k = torch.arange(4, device=q.device, dtype=torch.int32) * 4
            q = ((e[..., 0] << k) | (e[..., 1] << (k + 16))).sum(-1)
            q = torch.stack([(q >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2)
        s = (s.flatten(-2).to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)
        to.copy_(torch.cat([q.to(torch.uint8).flatten(1), s.flatten(1)], 1))
    return out


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c, "handle": _handle(c)}
    if c["kind"] == "prompt":
        past, count = _lengths(c)
        n, nh, kv, hd = c["tokens"], c["n_head"], c["n_kv"], c["head_dim"]
        s["row_start"], s["longest"] = _ints([sum(count[:i]) for i in range(len(count) + 1)]), max(count)
        s["q"], s["k"], s["v"] = (_normal(g, n, h, hd).to(TORCH[c["type"]]) for h in (nh, kv, kv))
        s["y"] = torch.empty_like(s["q"])
        s["gate"] = _normal(g, n, 2 * nh * hd) if c["gate"] else None
        return s
    page = c["page"]
    if c["kind"] == "prep":
        n, nh, kv, hd = c["tokens"], c["n_head"], c["n_kv"], c["head_dim"]
        s["q3"], s["qn"], s["kn"] = _normal(g, n, 2 * nh * hd + 2 * kv * hd), _normal(g, hd, mean=1.0, std=0.1), _normal(g, hd, mean=1.0, std=0.1)
        s["n_pages"] = _pages(n, page) + 3
        s["slot"] = _perm(g, s["n_pages"] * page)[:n].contiguous()
        s["pos"] = torch.randint(0, c["ctx"], (n,), generator=g, device="cuda").to(torch.int32)
        s["k"], s["v"] = (torch.zeros(s["n_pages"], page * kv * _row_bytes(c[t], hd), dtype=torch.uint8, device="cuda") for t in ("ktype", "vtype"))
        s["q"] = torch.empty(n, nh, hd, dtype=TORCH[c["qtype"]], device="cuda")
        s["krows"], s["vrows"] = (torch.empty(n, kv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    past, count = _lengths(c)
    n = len(past)
    if c["kind"] == "paged":
        nh, kv, hd = c["n_head"], c["n_kv"], c["head_dim"]
        total = [a + b for a, b in zip(past, count)]
        need = [_pages(t, page) for t in total]
        s["n_pages"], s["ntok"], s["max_ctx"], s["max_new"] = sum(need) + 2, sum(count), max(total), max(count)
        ids = _perm(g, s["n_pages"])
        s["table"] = torch.full((n, max(need)), -1, dtype=torch.int32, device="cuda")
        starts = [sum(need[:i]) for i in range(n)]
        for i in range(n):
            s["table"][i, :need[i]] = ids[starts[i]:starts[i] + need[i]]
        s["row_start"], s["kv_len"] = _ints([sum(count[:i]) for i in range(n + 1)]), _ints(total)
        s["k"], s["v"] = (_pool(g, c[t], s["n_pages"], page, kv, hd) for t in ("ktype", "vtype"))
        s["q"] = _normal(g, s["ntok"], nh, hd).to(TORCH[c["qtype"]])
        s["y"] = torch.empty_like(s["q"])
        s["gate"] = _normal(g, s["ntok"], 2 * nh * hd) if c["gate"] else None
        if s["handle"]:
            s["split"], bytes_ = s["handle"]
            s["ws"] = torch.empty(max(16, bytes_), dtype=torch.uint8, device="cuda")
        return s
    # plan and trim: table rows filled up to the lengths, the other pages of the pool free, in any order
    order = torch.randperm(n, generator=g, device="cuda").tolist()
    past, count = [past[i] for i in order], [count[i] for i in order]
    held = [_pages(p, page) for p in past]
    s["width"] = _pages(c["ctx"] + c.get("new", 0), page)
    new = sum(_pages(p + k, page) - h for p, k, h in zip(past, count, held)) if c["kind"] == "plan" else 7
    free = max(1, int(new * c.get("spare", 1.0)))
    s["n_pages"] = sum(held) + free
    ids = _perm(g, s["n_pages"])
    s["table"] = torch.full((n, s["width"]), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(s["width"], device="cuda")
    s["table"][column < _ints(held).unsqueeze(1)] = ids[free:]
    s["free"] = torch.full((s["n_pages"],), -1, dtype=torch.int32, device="cuda")
    s["free"][:free] = ids[:free]
    s["n_free"], s["past"], s["count"] = _ints([free]), _ints(past), _ints(count)
    s["status"], s["n_left"] = _ints([0] * n), _ints([0])
    s["row_start"], s["kv_len"] = _ints([0] * (n + 1)), _ints([0] * n)
    s["max_tok"] = sum(count) + 5 if c["kind"] == "plan" else 0   # a few rows of padding
    s["slot"], s["pos"] = _ints([0] * s["max_tok"]), _ints([0] * s["max_tok"])
    return s


def _handle(c):
    """what a program settles once for its sizes: the split of the contexts and the workspace that it needs"""
    if not own or c["kind"] != "paged":
        return None
    import rapier_amd as rmi
    past, count = _lengths(c)
    total = [a + b for a, b in zip(past, count)]
    split = rmi.gqa_paged_split(sum(total), max(total), len(total), sum(count), max(count), c["n_head"], c["n_kv"], c["head_dim"])
    return split, rmi.gqa_paged_workspace_bytes(sum(count), max(total), c["n_head"], c["head_dim"], split)


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    return _kernels(state) if own else _plain(state)


def _kernels(s):
    import rapier_amd as rmi
    c = s["case"]
    types = {"f16": rmi.KV_F16, "i8": rmi.KV_I8, "i4": rmi.KV_I4}
    if c["kind"] == "plan":
        rmi.page_plan(s["past"], s["count"], c["reqs"], c["page"], s["n_pages"], s["free"], s["n_free"], s["table"], s["width"], s["max_tok"],
                      s["row_start"], s["kv_len"], s["slot"], s["pos"], s["n_left"], s["status"])
        return {k: s[k] for k in ("row_start", "kv_len", "slot", "pos", "table", "n_left", "status")}
    if c["kind"] == "trim":
        rmi.page_trim(s["past"], s["count"], c["reqs"], c["page"], s["n_pages"], s["table"], s["width"], s["n_free"], s["free"], s["n_left"])
        return {"free": s["free"], "n_free": s["n_left"]}
    nh, kv, hd = c["n_head"], c["n_kv"], c["head_dim"]
    if c["kind"] == "prep":
        y = YARN if c["yarn"] else {"factor": 1.0, "orig_ctx": 0.0}
        rmi.attn_prep_paged(s["q3"], s["q3"].shape[1], s["qn"], s["kn"], types[c["ktype"]], s["k"], types[c["vtype"]], s["v"], s["slot"], s["pos"],
                            s["q"], nh, kv, hd, c["n_rot"], rmi.ROPE_HALF if c["pairs"] == "half" else rmi.ROPE_NEIGHBOURS, THETA, EPS,
                            c["tokens"], c["page"], s["n_pages"], **y)
        for t, x in (("ktype", "k"), ("vtype", "v")):
            rmi.kv_page_read(types[c[t]], s[x], s["slot"], s[x + "rows"], kv * hd, c["tokens"], kv, hd, c["page"], s["n_pages"])
        return {"q": s["q"], "k": s["krows"], "v": s["vrows"]}
    width = 2 * nh * hd
    if c["kind"] == "paged":
        rmi.gqa_paged_attn(s["q"], types[c["ktype"]], s["k"], types[c["vtype"]], s["v"], s["table"], s["table"].shape[1], s["row_start"],
                           s["kv_len"], s["gate"], width, s["y"], nh * hd, None, 0, s["ws"], c["reqs"], s["ntok"], s["max_new"], s["max_ctx"],
                           nh, kv, hd, c["page"], s["n_pages"], s["split"], 1.0 / math.sqrt(hd))
        return s["y"]
    rmi.gqa_prompt_attn(s["q"], nh * hd, s["k"], kv * hd, s["v"], kv * hd, s["row_start"], s["gate"], width, s["y"], nh * hd, None, 0,
                        c["reqs"], c["tokens"], s["longest"], nh, kv, hd, 1.0 / math.sqrt(hd))
    return s["y"]


def _plan(s):
    c, page, n = s["case"], s["case"]["page"], s["case"]["reqs"]
    past, count = s["past"].long(), s["count"].long()
    total, held = past + count, (past + page - 1) // page
    need = (total + page - 1) // page - held
    upto = need.cumsum(0)
    ok = (need == 0) | (upto <= s["n_free"])
    row_start = torch.cat([count.new_zeros(1), count.cumsum(0)])
    column = torch.arange(s["width"], device="cuda").expand(n, -1) - held.unsqueeze(1)
    taken = (column >= 0) & (column < need.unsqueeze(1)) & ok.unsqueeze(1)
    at = (s["n_free"] - 1 - (upto - need).unsqueeze(1) - column).clamp(0, s["n_pages"] - 1)
    table = torch.where(taken, s["free"][at], s["table"])
    tok = torch.arange(s["max_tok"], device="cuda")
    req = torch.searchsorted(row_start[1:], tok, right=True).clamp_max(n - 1)
    pos = past[req] + tok - row_start[req]
    used = tok < row_start[-1]
    slot = table[req, (pos // page).clamp_max(s["width"] - 1)] * page + pos % page
    return {"row_start": row_start.int(), "kv_len": torch.where(ok, total, 0).int(), "slot": torch.where(used & ok[req], slot, -1).int(),
            "pos": torch.where(used, pos, 0).int(), "table": table, "n_left": s["n_free"] - (need * ok).sum().int(),
            "status": torch.where(ok, 0, 2).int()}


def _trim(s):
    page = s["case"]["page"]
    first, end = (s["count"] + page - 1) // page, (s["past"] + page - 1) // page
    column = torch.arange(s["width"], device="cuda")
    back = s["table"][(column >= first.unsqueeze(1)) & (column < end.unsqueeze(1))]   # in the order of requests, then columns
    free = s["free"].clone()
    place = torch.arange(s["n_pages"], device="cuda") - s["n_free"]
    if len(back):
        free = torch.where((place >= 0) & (place < len(back)), back[place.clamp(0, len(back) - 1)], free)
    return {"free": free, "n_free": s["n_free"] + len(back)}


def _angles(c, pos):
    """the angle of every pair at every position, in 64 bits, and the factor of cos and sin"""
    i = torch.arange(c["n_rot"] // 2, device="cuda", dtype=torch.float64)
    freq, size = torch.exp(i * (-2.0 * math.log(THETA) / c["n_rot"])), 1.0
    if c["yarn"]:
        low, high = (c["n_rot"] * math.log(YARN["orig_ctx"] / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (YARN["beta_fast"], YARN["beta_slow"]))
        low, high = max(0.0, math.floor(low)), min(c["n_rot"] - 1.0, math.ceil(high))
        keep = 1.0 - ((i - low) / max(0.001, high - low)).clamp(0.0, 1.0)
        freq, size = freq / YARN["factor"] * (1 - keep) + freq * keep, 1.0 + 0.1 * math.log(YARN["factor"])
    return pos.double().unsqueeze(1) * freq, size


def _page_values(pool, type_, page, n_kv, head_dim):
    """pages [..., bytes] -> float32 [..., kv head, position, dim]"""
    if type_ == "f16":
        return pool.view(torch.float16).unflatten(-1, (page, n_kv, head_dim)).transpose(-3, -2).float()
    width = head_dim * BITS[type_] // 8
    codes = pool[..., :n_kv * page * width].unflatten(-1, (n_kv, page, width))
    s = pool[..., n_kv * page * width:].unflatten(-1, (n_kv, page, head_dim // 32))
    s = (s.to(torch.int16) << 7).view(torch.float16).float().repeat_interleave(32, -1)
    if type_ == "i4":
        w = codes.to(torch.int32).unflatten(-1, (-1, 4))
        k = torch.arange(4, device=codes.device, dtype=torch.int32) * 4
        low, high = w[..., 0] | (w[..., 1] << 8), w[..., 2] | (w[..., 3] << 8)
        codes = torch.stack([(low.unsqueeze(-1) >> k) & 15, (high.unsqueeze(-1) >> k) & 15], -1).flatten(-3)
    return (codes.float() - (QMAX[type_] + 1)) * s


def _softmax_v(q, k, v, seen):
    """q [..., rows, dims], k and v [..., positions, dims], seen [..., rows, positions], in float32"""
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    score.masked_fill_(~seen, -math.inf)
    score -= score.amax(-1, keepdim=True)
    total = score.exp_().sum(-1, keepdim=True)
    return torch.matmul(score, v) / total


def _gated(c, y, gate):
    """y [tokens, heads, dims] in float32, the gate beside each head's q"""
    if gate is None:
        return y
    return y / (1 + torch.exp(-gate.view(len(y), c["n_head"], 2, c["head_dim"])[:, :, 1]))


def _plain(s):
    c = s["case"]
    if c["kind"] == "plan":
        return _plan(s)
    if c["kind"] == "trim":
        return _trim(s)
    nh, kv, hd = c["n_head"], c["n_kv"], c["head_dim"]
    group = nh // kv
    if c["kind"] == "prep":
        n, half = c["tokens"], c["n_rot"] // 2
        angle, size = _angles(c, s["pos"])
        cos, sin = (size * angle.cos()).unsqueeze(1), (size * angle.sin()).unsqueeze(1)   # [token][1][pair]

        def normed(x, w):   # in 64 bits: the rows are quantised after it, next to borders
            x = x.double()
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
            turned, rest = x[..., :2 * half], x[..., 2 * half:]
            a, b = turned.unflatten(-1, (2, half) if c["pairs"] == "half" else (half, 2)).unbind(-2 if c["pairs"] == "half" else -1)
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -2 if c["pairs"] == "half" else -1).flatten(-2)
            return torch.cat([turned, rest], -1).float()

        q = s["q3"][:, :2 * nh * hd].view(n, nh, 2, hd)[:, :, 0]
        k, v = s["q3"][:, 2 * nh * hd:].view(n, 2, kv, hd).unbind(1)
        return {"q": normed(q, s["qn"]).to(TORCH[c["qtype"]]), "k": _value(normed(k, s["kn"]), c["ktype"]), "v": _value(v, c["vtype"])}
    if c["kind"] == "prompt":
        n = c["tokens"]
        tok = torch.arange(n, device="cuda")
        req = torch.searchsorted(s["row_start"][1:].contiguous(), tok.int(), right=True)
        seen = (req.unsqueeze(1) == req) & (tok.unsqueeze(1) >= tok)
        q = s["q"].float().view(n, kv, group, hd).permute(1, 2, 0, 3).reshape(kv, group, n, hd)
        k, v = (s[x].float().transpose(0, 1).unsqueeze(1).expand(-1, group, -1, -1).contiguous() for x in "kv")
        y = _softmax_v(q, k, v, seen).flatten(0, 1).transpose(0, 1)
        return _gated(c, y, s["gate"]).to(TORCH[c["type"]])
    reqs, new, ctx, start = c["reqs"], s["max_new"], s["max_ctx"], s["row_start"].long()
    k, v = (_page_values(s[x][s["table"].clamp_min(0).long()], c[x + "type"], c["page"], kv, hd).transpose(1, 2).flatten(2, 3)[:, :, :ctx].contiguous()
            for x in "kv")   # [request, kv head, position, dim]
    count = start[1:] - start[:-1]
    j = torch.arange(new, device="cuda")
    row = (start[:-1].unsqueeze(1) + j).clamp_max(s["ntok"] - 1)   # [request][new token]
    last = (s["kv_len"].long() - count).unsqueeze(1) + j
    seen = torch.arange(ctx, device="cuda") <= last.unsqueeze(-1)
    q = s["q"].float()[row].view(reqs, new, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(reqs, kv, new * group, hd)
    y = _softmax_v(q, k, v, seen.repeat_interleave(group, 1).unsqueeze(1))
    y = y.view(reqs, kv, new, group, hd).permute(0, 2, 1, 3, 4).reshape(reqs, new, nh, hd)[j < count.unsqueeze(1)]
    return _gated(c, y, s["gate"]).to(TORCH[c["qtype"]])


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _grid(type_):
    """every scale, in order: (8 + m) 2^(e - 18), or m 2^-17 for e = 0"""
    g = [math.ldexp(m if e == 0 else 8 + m, -17 if e == 0 else e - 18) for e in range(31) for m in range(8)]
    return torch.tensor([x for x in g if x <= SMAX[type_]], dtype=torch.float64, device="cuda")


def _held(x, type_):
    """what a quantised cache holds for float64 rows: the smallest scale that reaches the block's maximum, by search"""
    grid, m = _grid(type_), QMAX[type_]
    blocks = x.reshape(-1, 32)
    at = torch.searchsorted(grid * m, blocks.abs().max(1).values).clamp_max(len(grid) - 1)
    s = grid[at].unsqueeze(1)
    q = torch.where(s > 0, blocks / s, 0.0 * blocks)
    return (q.round().clamp(-m, m) * s).view(x.shape)


def _rows_64(pages, type_, page, n_kv, head_dim):
    """a request's pages [n, bytes] -> float64 [kv head][n page][dim], decoded code by code"""
    if type_ == "f16":
        return pages.view(torch.float16).reshape(-1, n_kv, head_dim).transpose(0, 1).double()
    per = head_dim * BITS[type_] // 8
    raw = pages[:, :n_kv * page * per].reshape(-1, n_kv, page, per).transpose(0, 1).reshape(n_kv, -1, per).long()
    scale = pages[:, n_kv * page * per:].reshape(-1, n_kv, page, head_dim // 32).transpose(0, 1).reshape(n_kv, -1, head_dim // 32).long()
    full = torch.tensor([math.ldexp(b % 8 if b < 8 else 8 + b % 8, -17 if b < 8 else b // 8 - 18) for b in range(248)], dtype=torch.float64,
                        device="cuda")
    d = torch.arange(head_dim, device="cuda")
    if type_ == "i4":
        bit = 4 * (d % 8 // 2) + 16 * (d % 2)   # of the word of the dim's eight
        raw = raw[..., d // 8 * 4 + bit // 8] >> (bit % 8) & 15
    return (raw - (QMAX[type_] + 1)).double() * full[scale][..., d // 32]


def exact(case, seed):
    c = case
    if c["kind"] in ("plan", "trim"):
        return None   # whole numbers
    s = prepare(case, seed)
    nh, kv, hd = c["n_head"], c["n_kv"], c["head_dim"]
    if c["kind"] == "prep":
        n, half = c["tokens"], c["n_rot"] // 2
        freq, size = [THETA ** (-2.0 * i / c["n_rot"]) for i in range(half)], 1.0
        if c["yarn"]:
            f = YARN["factor"]
            edge = [c["n_rot"] * math.log(YARN["orig_ctx"] / (YARN[b] * 2 * math.pi)) / (2 * math.log(THETA)) for b in ("beta_fast", "beta_slow")]
            low, high = max(0, math.floor(edge[0])), min(c["n_rot"] - 1, math.ceil(edge[1]))
            ramp = [min(1.0, max(0.0, (i - low) / max(0.001, high - low))) for i in range(half)]
            freq, size = [x * (r / f + 1 - r) for x, r in zip(freq, ramp)], 1 + 0.1 * math.log(f)
        freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.full_like(freq, size).expand(n, -1).contiguous(), s["pos"].double()[:, None] * freq).unsqueeze(1)
        at = torch.arange(half, device="cuda")
        a, b = (at, at + half) if c["pairs"] == "half" else (2 * at, 2 * at + 1)

        def rotated(r, w):
            r = r * w.double() * torch.rsqrt((r * r).sum(-1, keepdim=True) / hd + EPS)
            pair = torch.complex(r[..., a], r[..., b]) * turn
            r[..., a], r[..., b] = pair.real, pair.imag
            return r

        x = s["q3"].double()
        heads, rows = x[:, :2 * nh * hd].reshape(n, nh, 2 * hd)[..., :hd], x[:, 2 * nh * hd:].reshape(n, 2 * kv, hd)
        k, v = rotated(rows[:, :kv], s["kn"]), rows[:, kv:].contiguous()
        # a quantised row's codes are those of the row rounded to fp32 once
        return {"q": rotated(heads, s["qn"]), "k": k if c["ktype"] == "f16" else _held(k.float().double(), c["ktype"]),
                "v": v if c["vtype"] == "f16" else _held(v, c["vtype"])}
    start, out = s["row_start"].tolist(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(c["reqs"]):
        rows = slice(start[i], start[i + 1])
        n = start[i + 1] - start[i]
        if n == 0:
            continue
        if c["kind"] == "prompt":
            total, k, v = n, s["k"][rows].double().transpose(0, 1), s["v"][rows].double().transpose(0, 1)
        else:
            total = s["kv_len"].tolist()[i]
            ids = s["table"][i, :_pages(total, c["page"])].long()
            k, v = (_rows_64(s[x][ids], c[x + "type"], c["page"], kv, hd)[:, :total] for x in "kv")
        later = torch.ones(n, total, dtype=torch.bool, device="cuda").triu(total - n + 1)
        for h in range(nh):
            w = (s["q"][rows, h].double() @ k[h * kv // nh].t().contiguous() * hd ** -0.5).masked_fill_(later, -math.inf)
            out[rows, h] = torch.exp(w - torch.logsumexp(w, 1, keepdim=True)) @ v[h * kv // nh].contiguous()
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].reshape(len(out), nh, 2 * hd)[..., hd:].double())
    return out


def work(case):
    c = case
    if c["kind"] == "prep":
        n, nh, kv, hd = c["tokens"], c["n_head"], c["n_kv"], c["head_dim"]
        rows = kv * (_row_bytes(c["ktype"], hd) + _row_bytes(c["vtype"], hd))
        return {"bytes": n * (4 * (nh + 2 * kv) * hd + 2 * nh * hd + 2 * rows + 4 * kv * hd + 8), "flops": 12 * n * (nh + 2 * kv) * hd}
    past, count = _lengths(c)
    n = len(past)
    if c["kind"] == "plan":
        moved = sum(_pages(p + k, c["page"]) - _pages(p, c["page"]) for p, k in zip(past, count)) * min(1.0, c["spare"])
        return {"bytes": int(24 * n + 8 * moved + 8 * sum(count)), "flops": 0}
    if c["kind"] == "trim":
        return {"bytes": 8 * n + 8 * sum(_pages(p, c["page"]) - _pages(k, c["page"]) for p, k in zip(past, count)), "flops": 0}
    nh, kv, hd, rows = c["n_head"], c["n_kv"], c["head_dim"], sum(count)
    keys = sum(p * k + k * (k + 1) // 2 for p, k in zip(past, count))   # seen keys of all tokens
    own_rows = rows * nh * hd * (4 + (4 if c["gate"] else 0))
    if c["kind"] == "prompt":
        return {"bytes": own_rows + 4 * rows * kv * hd, "flops": 4 * keys * nh * hd}
    held = sum(p + k for p, k in zip(past, count)) * kv * (_row_bytes(c["ktype"], hd) + _row_bytes(c["vtype"], hd))
    return {"bytes": own_rows + held, "flops": 4 * keys * nh * hd}

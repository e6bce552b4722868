"""Plain 64-bit restatement of the K/V cache types, the tree attention and the logit processing (numpy on the CPU)."""
import numpy as np

F16, I8, I4 = 0, 1, 2
QMAX = {I8: 127, I4: 7}
TOP = {I8: 192, I4: 224}
NAMES = {F16: "f16", I8: "i8", I4: "i4"}


def scale_values():
    """the fp16 number a scale byte stands for, all 256"""
    return (np.arange(256, dtype=np.uint16) << 7).view(np.float16).astype(np.float64)


def quantise(x, type_):
    """rows [..., dims] -> (codes int [..., dims], scale bytes [..., dims / 32]); the smallest scale by search"""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    grid = scale_values()[:TOP[type_] + 1]
    amax = np.abs(b).max(-1)
    bad = ~np.isfinite(amax)
    sb = np.minimum(np.searchsorted(grid * QMAX[type_], np.where(bad, 0, amax)), TOP[type_])
    s = grid[sb][..., None]
    with np.errstate(all="ignore"):
        q = np.where((s > 0) & ~bad[..., None], np.rint(b / np.where(s > 0, s, 1)), 0)
    q = np.clip(np.nan_to_num(q), -QMAX[type_], QMAX[type_]).astype(np.int64)
    return q.reshape(x.shape), np.where(bad, 255, sb).astype(np.uint8)


def values(codes, sb):
    with np.errstate(all="ignore"):
        return codes * np.repeat(scale_values()[sb], 32, -1)


def held(x, type_):
    """what a cache of the type holds for the rows x, in float64"""
    if type_ == F16:
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16).astype(np.float64)
    return values(*quantise(x, type_))


def encode(x, type_):
    """rows [max_ctx, n_kv, dims] -> the cache's bytes"""
    if type_ == F16:
        with np.errstate(over="ignore"):
            return np.ascontiguousarray(np.asarray(x, np.float32).astype(np.float16)).view(np.uint8).reshape(-1)
    q, sb = quantise(np.swapaxes(x, 0, 1), type_)
    u = (q + QMAX[type_] + 1).astype(np.uint32)
    if type_ == I8:
        codes = u.astype(np.uint8).reshape(-1)
    else:
        e = u.reshape(u.shape[:-1] + (-1, 4, 2))
        k = 4 * np.arange(4, dtype=np.uint32)
        codes = ((e[..., 0] << k) | (e[..., 1] << (k + 16))).sum(-1).astype("<u4").view(np.uint8).reshape(-1)
    return np.concatenate([codes, sb.reshape(-1)])


def decode(raw, type_, max_ctx, n_kv, hd):
    """the cache's bytes -> values [max_ctx, n_kv, dims] in float64"""
    raw = np.asarray(raw, np.uint8)
    if type_ == F16:
        return raw.view(np.float16).astype(np.float64).reshape(max_ctx, n_kv, hd)
    per = hd if type_ == I8 else hd // 2
    codes, sb = raw[:n_kv * max_ctx * per], raw[n_kv * max_ctx * per:].reshape(n_kv, max_ctx, hd // 32)
    if type_ == I8:
        q = codes.astype(np.int64).reshape(n_kv, max_ctx, hd) - 128
    else:
        d = np.arange(8)
        shift = 4 * (d // 2) + 16 * (d % 2)
        w = codes.view("<u4").astype(np.int64)
        q = ((w[:, None] >> shift) & 15).reshape(n_kv, max_ctx, hd) - 8
    return np.swapaxes(values(q, sb), 0, 1)


def tree_masks(rng, n, reach=6):
    """ancestor bit masks (own bit set) and depths of a random tree in an order with parents first"""
    masks, depth = [], []
    for i in range(n):
        p = int(rng.integers(max(-1, i - reach), i)) if i else -1
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return masks, depth


def attention(q, k, v, base, masks, scale, gate=None):
    """q [ntok, n_head, hd], k / v [positions, n_kv, hd] float64, masks: list of ints or None (chain).
    Returns y and, per token and head, a bound of fp32 arithmetic's error: (hd + 8) 2^-24 relative to the sum of |q k| in
    every score, twice that in a weight relative to the softmax's sum, one rounding per visible position in its sums, and
    2^-20 for the base-2 exponent (its rounded argument, |s| < 2^4 here) and the gate."""
    ntok, nh, hd = q.shape
    G = nh // k.shape[1]
    y, bound = np.zeros((ntok, nh, hd)), np.zeros((ntok, nh, 1))
    for t in range(ntok):
        seen = list(range(base))
        seen += [base + j for j in range(ntok) if (j <= t if masks is None else masks[t] >> j & 1)]
        for h in range(nh):
            if not seen:
                continue
            kk, vv = k[seen, h // G], v[seen, h // G]
            s = kk @ q[t, h] * scale
            w = np.exp(s - s.max())
            y[t, h] = w @ vv / w.sum()
            a = (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
            bound[t, h] = (2 * (hd + 8) * 2.0 ** -24 * a + len(seen) * 2.0 ** -24 + 2.0 ** -20) * np.abs(vv).max()
    if gate is not None:
        y = y / (1 + np.exp(-gate))
    return y, bound


def logits(x, hist, window, draft, masks, rep, pres, freq, bias_ids, bias_vals, allow):
    """x [ncols, n]; hist: the used part; masks: list of ints; allow: uint32 [ncols, words] or None"""
    x = np.array(x, np.float64)
    n = x.shape[1]
    last = {}
    for i, b in zip(bias_ids, bias_vals):
        last[int(i)] = float(b)
    for i, b in last.items():
        if 0 <= i < n:
            x[:, i] += b
    for c in range(x.shape[0]):
        text = list(hist) + [draft[j] for j in range(len(draft)) if masks[c] >> j & 1]
        if window > 0:
            text = text[-window:]
        ids = np.array([i for i in text if 0 <= i < n], np.int64)
        m = np.bincount(ids, minlength=n)
        hit = m > 0
        v = x[c, hit]
        x[c, hit] = np.where(v > 0, v / rep, v * rep) - (m[hit] * freq + pres)
        if allow is not None:
            bits = np.unpackbits(allow[c].view(np.uint8), bitorder="little")[:n]
            x[c, bits == 0] = -np.inf
    return x

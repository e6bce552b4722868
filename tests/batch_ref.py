"""Plain 64-bit restatements of the page plan, the prep into pages and the attention of a batch (numpy on the CPU)."""
import numpy as np

from . import kv_ref

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # a rounding's largest error, relative


def pages(n, page):
    return -(-n // page)


def plan(past, count, page, n_pages, free, n_free, table, max_tok):
    """row by row: (row_start, kv_len, slot, pos, n_left, status, table)"""
    n, width = table.shape
    table = table.copy()
    row_start, kv_len, status = [0], [], []
    slot, pos = [-1] * max_tok, [0] * max_tok
    wanted, taken = 0, 0
    for i in range(n):
        c = max(0, int(count[i]))
        first, row_start = row_start[-1], row_start + [row_start[-1] + c]
        good = past[i] >= 0 and count[i] >= 0 and past[i] + count[i] <= min(width * page, 1 << 30) and row_start[-1] <= max_tok
        need = pages(past[i] + count[i], page) - pages(past[i], page) if good else 0
        wanted += need
        ok = good and (need == 0 or wanted <= n_free)
        status.append(0 if ok else 2 if good else 1)
        kv_len.append(past[i] + count[i] if ok else 0)
        if ok:
            for k in range(need):
                table[i, pages(past[i], page) + k] = free[n_free - 1 - (wanted - need + k)]
            taken += need
        for k in range(min(c, max(0, max_tok - first))):
            p = past[i] + k
            pos[first + k] = p
            if ok and 0 <= table[i, p // page] < n_pages:
                slot[first + k] = table[i, p // page] * page + p % page
    return [min(r, max_tok) for r in row_start], kv_len, slot, pos, n_free - taken, status, table


def trim(length, keep, page, n_pages, table, n_free, free):
    free = list(free)
    at = n_free
    for i in range(len(length)):
        if 0 <= keep[i] <= length[i]:
            for c in range(pages(keep[i], page), min(pages(length[i], page), table.shape[1])):
                if at < n_pages:
                    free[at] = table[i, c]
                    at += 1
    return at, free


def rotated(x, w, pos, n_rot, neighbours, eps, base, factor=1.0, orig=0.0, ext=1.0, attn=1.0, fast=32.0, slow=1.0):
    """rows x [tokens, heads, dims]: normed with weights w (None: not), pairs turned at pos; plain NEOX or YaRN angles"""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w
    half = n_rot // 2
    i = np.arange(half, dtype=np.float64)
    base = np.float64(np.float32(base))
    freq, size = base ** (-2.0 * i / max(n_rot, 1)), 1.0
    if factor > 1:
        dim = [n_rot * np.log(orig / (b * 2 * np.pi)) / (2 * np.log(base)) for b in (fast, slow)]
        low, high = max(0.0, np.floor(dim[0])), min(n_rot - 1.0, np.ceil(dim[1]))
        ramp = (1 - np.clip((i - low) / max(0.001, high - low), 0, 1)) * ext
        freq = freq / factor * (1 - ramp) + freq * ramp
        size = attn * (1 + 0.1 * np.log(factor)) if ext else attn
    angle = np.asarray(pos, np.float64)[:, None, None] * freq
    c, s = size * np.cos(angle), size * np.sin(angle)
    a, b = (2 * np.arange(half), 2 * np.arange(half) + 1) if neighbours else (np.arange(half), np.arange(half) + half)
    y = x.copy()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def attention(q, k, v, first, scale, gate, weight_step, out_step):
    """One request's new tokens: q [n, heads, hd] at positions first + 0 .. n - 1 over k / v [positions, kv heads, hd].  Returns y
    and a bound of the kernel's error.  fp32 scores and sums: kv_ref.attention's terms; a weight is rounded to 16 bits once
    (weight_step relative; fp16's smallest weights lie 2^-33 below a row's largest, absolutely), so is the result (out_step)."""
    n, nh, hd = q.shape
    G = nh // k.shape[1]
    y, bound = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    for h in range(nh):
        kk, vv = k[:, h // G], v[:, h // G]
        for t in range(n):
            seen = first + t + 1
            if seen <= 0:
                continue
            with np.errstate(all="ignore"):
                s = kk[:seen] @ q[t, h] * scale
                w = np.exp(s - s.max())
                y[t, h] = w @ vv[:seen] / w.sum()
                a = (np.abs(kk[:seen]) @ np.abs(q[t, h])).max() * scale
                top = np.abs(vv[:seen]).max()
                bound[t, h] = (2 * (hd + 8) * 2.0 ** -24 * a + seen * (2.0 ** -24 + 2.0 ** -33) + 2.0 ** -20 + weight_step) * top
    if gate is not None:
        y = y / (1 + np.exp(-gate))
    return y, bound + out_step * (np.abs(y) + bound) + 2.0 ** -25


class Pool:
    """pages of K or V rows in a type's layout, as raw bytes"""

    def __init__(self, type_, n_pages, page, n_kv, hd, fill=None, rng=None):
        self.type, self.n_pages, self.page, self.n_kv, self.hd = type_, n_pages, page, n_kv, hd
        per = len(kv_ref.encode(np.zeros((page, n_kv, hd)), type_))
        if fill is None:
            self.raw = rng.integers(0, 256, (n_pages, per), dtype=np.uint8)   # what unwritten memory may hold
        else:
            self.raw = np.full((n_pages, per), fill, np.uint8)

    def write(self, ids, rows):
        """rows [positions, n_kv, hd] to the pages ids in order; the rest of the last page keeps its bytes"""
        for j, at in enumerate(range(0, len(rows), self.page)):
            part = rows[at:at + self.page]
            whole = kv_ref.encode(np.concatenate([part, np.zeros((self.page - len(part),) + part.shape[1:])]), self.type)
            mask = kv_ref_mask(self.type, len(part), self.page, self.n_kv, self.hd)
            self.raw[ids[j]][mask] = whole[mask]

    def read(self, ids, n):
        rows = [kv_ref.decode(self.raw[i], self.type, self.page, self.n_kv, self.hd) for i in ids]
        return np.concatenate(rows)[:n] if rows else np.zeros((0, self.n_kv, self.hd))


def kv_ref_mask(type_, n, page, n_kv, hd):
    """the bytes of a page's first n positions"""
    if type_ == kv_ref.F16:
        m = np.zeros((page, n_kv * hd * 2), bool)
        m[:n] = True
        return m.reshape(-1)
    per = hd if type_ == kv_ref.I8 else hd // 2
    codes, scales = np.zeros((n_kv, page, per), bool), np.zeros((n_kv, page, hd // 32), bool)
    codes[:, :n], scales[:, :n] = True, True
    return np.concatenate([codes.reshape(-1), scales.reshape(-1)])

"""The attention of a batch in 64 bits (torch, on the CPU or the GPU) with an error bound that follows the data: what a kernel may be
off by shrinks with the weights that it sums, so that positions left out of a long context show."""
import torch

from . import batch_ref as ref


def attention(q, k, v, pos, scale, weight_step, out_step, gate=None, depth=None, left_out=None):
    """Rows q [rows, heads, dims] of tokens at positions pos [rows], over k and v [positions, kv heads, dims] (float64).  Returns y and
    a bound of a kernel's error per element.  With w a row's weights over their sum, a the sums of |q k| and u = 2^-24 (fp32):
      scores    exact products, dims additions, the factor, the maximum taken off, the exponential's 2^-23: a weight is off by
                e = (dims + 8) u a + 4 u max a + 2^-22 relative; q of bf16 is brought to fp16 by a power of two, its smallest elements
                lose 2^-38 of a row's largest.  Moves y by at most sum w e |v - y|
      weights   rounded to 16 bits for the product with V (weight_step), not in their sum: sum w |v| weight_step; fp16's smallest lie
                2^-33 below a row's largest, absolutely
      sums      depth additions one after another (the positions, if not given), in the product and in the weights' sum
      result    rounded once (out_step); the gate's sigmoid by 2^-22 and its argument's rounding
    left_out: positions that y does without (a mistake on purpose, for tests of the bound itself)."""
    rows, heads, dims = q.shape
    group = heads // k.shape[1]
    u = 2.0 ** -24
    y, bound = torch.zeros_like(q), torch.zeros_like(q)
    at = torch.arange(len(k), device=q.device)
    for h in range(k.shape[1]):
        kk, vv = k[:, h].contiguous(), v[:, h].contiguous()
        x = q[:, h * group:(h + 1) * group].reshape(rows * group, dims)
        unseen = at > pos.repeat_interleave(group).unsqueeze(1)
        s = (x @ kk.t().contiguous() * scale).masked_fill_(unseen, -torch.inf)
        a = (x.abs() @ kk.abs().t().contiguous() * scale).masked_fill_(unseen, 0.0)
        w = torch.exp(s - s.amax(1, keepdim=True))
        total = w.sum(1, keepdim=True)
        w /= total
        out, size = w @ vv, w @ vv.abs()
        lost = dims * 2.0 ** -38 * x.abs().amax(1, keepdim=True) * kk.abs().max() * scale
        e = w * ((dims + 8) * u * a + 4 * u * a.amax(1, keepdim=True) + 2.0 ** -22 + lost)
        n = (~unseen).sum(1, keepdim=True).double()
        tol = e @ vv.abs() + e.sum(1, keepdim=True) * out.abs() + weight_step * size + 2.0 ** -33 * n / total * vv.abs().max()
        tol += (n if depth is None else depth) * u * (size + out.abs())
        if left_out is not None:
            w[:, left_out] = 0.0
            out = w @ vv / w.sum(1, keepdim=True)
        y[:, h * group:(h + 1) * group] = out.view(rows, group, dims)
        bound[:, h * group:(h + 1) * group] = tol.view(rows, group, dims)
    if gate is not None:
        open_ = torch.sigmoid(gate)
        y = y * open_
        bound = bound * open_ + y.abs() * (2.0 ** -22 + 2 * u * gate.abs())
    return y, bound + out_step * (y.abs() + bound) + 2.0 ** -25


def outside(got, want, bound):
    """how many elements are (NaN is)"""
    return int((~((got - want).abs() <= bound)).sum())


HALF_STEP = ref.HALF_STEP


def marks(n, dims, by):
    """V rows of zeros with a one each: position j's at dim (j // by) % dims"""
    v = torch.zeros(n, dims, dtype=torch.float64)
    j = torch.arange(n)
    v[j, j // by % dims] = 1.0
    return v


def marked(pos, dims, by):
    """how many of the positions up to pos [rows] have their mark at each dim: [rows, dims]"""
    d = torch.arange(dims, device=pos.device)
    n = (pos + 1).unsqueeze(1)   # positions j < n with j // by % dims == d: whole rounds of by dims, and what the last one has
    return n // (by * dims) * by + (n % (by * dims) - d * by).clamp(0, by)

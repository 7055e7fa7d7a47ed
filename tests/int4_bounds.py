"""How far attention over 4-bit rows may be off, relative to the values (test infrastructure)."""
import math

import torch

LOG2E = math.log2(math.e)


def attention(q, k, v, v_codes, v_scales, scale):
    """q [4, D], k / v [n, D] in 64 bits -> out [4, D] and the bound of the error of out apart from its last rounding.
    v_codes [n, D]: the part s c of the values s c + z; v_scales [n, D]: s.  No term is left when all values are zero: everything
    is proportional to v, s c, z or the largest s.

    * logits: fp32 sums of 128 products and of the zeros' share, each step good to 2^-23 of the largest partial sum
    * probabilities are at most 2^13, the largest of a warp 2^11 at least.  Rounding to fp16: 2^-11 of p; 2^-25 below 2^-14, which is 2^-36
      of the sum of probabilities
    * p s, with s times a power of two that brings the warp's largest to [2, 4): 2^-11 of p s; 2^-25 below 2^-14, which with codes
      up to 15 is 15 2^-37 of the largest s per key; and a scale itself below 2^-16 of the largest, 15 2^-26 of that.  Scales below 2^-15
      are raised by 2^15 only: 15 2^-51 per key
    * the tensor core's sums, rounded towards zero: 2^-24 of the sum for each 16 keys, 2^-20 for those of the last steps and the zeros, and
      2^-16 of p s for codes whose exponent field lies above them, twice"""
    n = k.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    x = q @ k.T * scale
    p = torch.softmax(x, -1)
    logit = 32 * 2.0 ** -23 * float((q.abs() @ k.abs().T).max()) * abs(scale) * LOG2E + 2.0 ** -20
    half, top = 2.0 ** -11, float(v_scales.max())
    bound = (half + 2 * logit) * (p @ v.abs()) + (half * (1 + half) + 2.0 ** -20 + n * 2.0 ** -28) * (p @ v_codes) \
        + 2.0 ** -20 * (p @ (v - v_codes).abs()) + 2.0 ** -15 * (p @ v_scales) \
        + 15 * top * (2.0 ** -26 + n * 2.0 ** -37) + n * 2.0 ** -36 * float(v.abs().max()) + n * 15 * 2.0 ** -51
    return p @ v, bound


def last_rounding(want, dtype):
    """Half a step of the output's type, its subnormals included."""
    info = torch.finfo(dtype)
    return want.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def sink_rows(n, G, size, gap, seed):
    """Queries [1, 4 G, 128] and rows [2, n, G, 128] of a cache in which row n // 3 has a logit of about `gap` above the largest of
    the others, and values of 0.02 of theirs: an attention sink.  Values are of `size`, each channel with a mean of its own."""
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(G, 128, generator=g)
    u = u / u.norm(dim=-1, keepdim=True)
    q = 128 ** 0.5 * u[:, None] + 0.3 * torch.randn(G, 4, 128, generator=g)
    rows = torch.randn(2, n, G, 128, generator=g)
    rows[1] += torch.randn(G, 128, generator=g)
    rows[0, n // 3] = (gap + 3.7) * u
    rows[1, n // 3] *= 0.02
    rows[1] *= size
    return q.view(1, 4 * G, 128), rows

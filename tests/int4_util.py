"""Plain forms, in 64 bits, of the 4-bit cache and of what is done with it (test infrastructure)."""
import math

import torch

K_PIECES, V_PIECES = 4, 8
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}   # of a rounding, relative


def quantize(x):
    """Rows [..., 128] -> codes int64 [..., 4, 32], parameters fp16 [..., 8]: scales, zeros."""
    x = x.double().unflatten(-1, (4, 32))
    fine = torch.isfinite(x).all(-1)
    least = x.nan_to_num(0.0, 0.0, 0.0).amin(-1)
    zero = torch.where(fine, least.clamp(-65504, 65504), torch.nan).half()
    span = x.nan_to_num(0.0, 0.0, 0.0).amax(-1).clamp(max=65504).float() - zero.float()
    scale = torch.where(fine, (span / 15).clamp(min=0), 0.0).half()
    s, z = scale.double()[..., None], zero.double()[..., None]
    codes = torch.where((s > 0) & fine[..., None], (x - z) / s.clamp(min=1e-300), 0.0).round().clamp(0, 15)
    return codes.long(), torch.cat([scale, zero], -1)


def pack(codes, pieces):
    """codes [..., 4, 32] -> bytes [..., 64] in the order of a K row (4 pieces) or a V row (8)."""
    order = [(g, 32 // pieces * p + i) for p in range(pieces) for g in range(4) for i in range(32 // pieces)]
    flat = torch.stack([codes[..., g, i] for g, i in order], -1)
    return (flat[..., 0::2] + 16 * flat[..., 1::2]).to(torch.uint8)


def unpack(packed, params, pieces, zeros=True):
    """bytes [..., 64] and parameters [..., 8] -> values [..., 128] in 64 bits; without the zeros: scale times code only."""
    order = [32 * g + 32 // pieces * p + i for p in range(pieces) for g in range(4) for i in range(32 // pieces)]
    out = torch.empty(*packed.shape[:-1], 128, dtype=torch.float64, device=packed.device)
    out[..., order[0::2]] = (packed & 15).double()
    out[..., order[1::2]] = (packed >> 4).double()
    out = out * params[..., :4].double().repeat_interleave(32, -1)
    return out + params[..., 4:].double().repeat_interleave(32, -1) if zeros else out


def make_cache(lens, G, page=16, seed=0, device="cuda", spread=1.0, interleaved=True):
    """A paged 4-bit cache of random rows with shuffled pages -> (k, v, kp, vp, block table, K values, V values, the
    codes' part of the V values); the values are those that the cache stands for, [B, G, longest, 128] in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    B, longest = len(lens), max(max(lens), 1)
    per = -(-longest // page)
    total = B * per + 2
    table = torch.randperm(total, generator=g)[:B * per].view(B, per).to(torch.int32)
    rows = torch.randn(2, total, page, G, 128, generator=g) * (1 + spread * torch.rand(2, total, page, G, 1, generator=g))
    rows[..., 5] *= 4                                                # a channel of its own size, as keys have
    kc, kp = quantize(rows[0])
    vc, vp = quantize(rows[1])
    k, v = pack(kc, K_PIECES), pack(vc, V_PIECES)
    params = torch.cat([kp, vp], -1).to(device)
    kp, vp = (params[..., :8], params[..., 8:]) if interleaved else (params[..., :8].contiguous(), params[..., 8:].contiguous())

    def values(packed, par, pieces, zeros=True):
        x = unpack(packed, par, pieces, zeros)[table.long()].flatten(1, 2)[:, :longest]
        return x.transpose(1, 2).contiguous()

    return k.to(device), v.to(device), kp, vp, table.to(device), values(k, kp.cpu(), K_PIECES), \
        values(v, vp.cpu(), V_PIECES), values(v, vp.cpu(), V_PIECES, False)


def attention(q, k, v, v_codes, scale):
    """q [4, D], k / v [n, D] in 64 bits -> out [4, D], log2-sum-exp [4], probabilities [4, n], bound of |error| of out apart from
    its last rounding, bound of the error of a logit in units of log2.  v_codes [n, D]: the part s c of the values s c + z."""
    x = q @ k.T * (scale * math.log2(math.e))
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.full((q.shape[0],), -math.inf), x, torch.zeros_like(q), 0.0
    p = torch.softmax(x * math.log(2), -1)
    lse = torch.logsumexp(x * math.log(2), -1) / math.log(2)
    # fp32 sums of 128 products and of the zeros' share, each product and step good to 2^-23 of the largest partial sum
    logit = 32 * 2.0 ** -23 * float((q.abs() @ k.abs().T).max()) * abs(scale) * 1.45 + 2.0 ** -20
    # A probability is rounded to fp16, p (1 + a), |a| <= 2^-11, and its product with a group's scale again, p s (1 + a) (1 + b):
    # the value's share is off by a p (s c + z) + b p s c.  Where s c and z nearly cancel the second term is the larger one.
    # Below 2^-14 both are rounded to multiples of 2^-24: by 2^-25 of a sum of probabilities that is at least 1.
    half = 2.0 ** -11
    out = (half + 2 * logit) * (p @ v.abs()) + (half * (1 + half) + 2.0 ** -20) * (p @ v_codes) + 2.0 ** -20 * (p @ (v - v_codes).abs()) \
        + 2.0 ** -25 * (v.abs() + 15).sum(0)
    return p @ v, lse, p, out, logit

"""Attention over FP8 rows whose values are small, or differ in size, where few keys take most of the weight (GPU): held to a bound that
is relative to the values."""
import pytest
import torch

from tests.int4_bounds import LOG2E, last_rounding, sink_rows

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _quantise(rows, page=16):
    """[n, G, 128] -> e4m3 pages [pages, page, G, 128], scales [pages, G] fp32 and the values in 64 bits [n, G, 128]."""
    n, G, _ = rows.shape
    pages = -(-n // page)
    padded = torch.zeros(pages * page, G, 128)
    padded[:n] = rows
    padded = padded.unflatten(0, (pages, page))
    scale = (padded.abs().amax((1, 3)) / 448).clamp(min=1e-30)
    stored = (padded / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return stored, scale, (stored.double() * scale.double()[:, None, :, None]).flatten(0, 1)[:n]


def _plain(q, k, v, top):
    """q [4, 128], k / v [n, 128] in 64 bits, top: the largest scale of V -> attention, and the bound of its error but for the last
    rounding.  Probabilities times scales, with a power of two that brings the largest scale to 2^14, are rounded to fp16: 2^-11, and
    2^-25 below 2^-14, times stored values of at most 448.  Sums of 16 keys are rounded towards zero: 2^-23 of the sum."""
    n = k.shape[0]
    x = q @ k.T * SCALE
    p = torch.softmax(x, -1)
    logit = 32 * 2.0 ** -23 * float((q.abs() @ k.abs().T).max()) * SCALE * LOG2E + 2.0 ** -20
    return p @ v, (2.0 ** -11 + 2 * logit + 2.0 ** -20 + n * 2.0 ** -27) * (p @ v.abs()) + n * 448 * top * 2.0 ** -39


def _check(rows, q, dense, splits, batch, heads, what):
    from kascade_b200 import _native as nat
    n, G = rows.shape[1:3]
    (k8, ks, k), (v8, vs, v) = _quantise(rows[0]), _quantise(rows[1])
    table = torch.arange(k8.shape[0], dtype=torch.int32).expand(batch, -1).contiguous().cuda()
    kv = nat.kv_layout_paged(k8.cuda(), v8.cuda(), table, ks.cuda(), vs.cuda())
    q = q.half().cuda().expand(batch, -1, -1).contiguous()
    out = torch.full_like(q, 9.0)
    ws = nat.decode_workspace(batch, 4 * G, splits, q.device)
    if dense:
        stride = -(-n // 4) * 4
        logits, pooled = (torch.zeros(batch, m, stride, device="cuda") for m in (4 * G, G))
        lens, lse = torch.full((batch,), n, dtype=torch.int32, device="cuda"), torch.empty(batch, 4 * G, device="cuda")
        nat.decode_anchor_paged(q, kv, lens, n, SCALE, logits, pooled, out, lse, ws, splits)
    else:
        index = torch.stack([torch.randperm(n, generator=torch.Generator().manual_seed(g)) for g in range(G)]).to(torch.int32)
        nat.decode_sparse_paged(q, kv, index.expand(batch, -1, -1).contiguous().cuda(), None, n, None, SCALE, out, None, ws, splits)
    assert torch.equal(out, out[:1].expand_as(out))
    for g in heads:
        want, bound = _plain(q[0, 4 * g:4 * g + 4].cpu().double(), k[:, g], v[:, g], float(vs.max()))
        off = (out[0, 4 * g:4 * g + 4].cpu().double() - want).abs()
        limit = bound + last_rounding(want, torch.float16)
        assert bool((off <= limit).all()), f"{what}, head {g}: {float((off / limit).max()):.3g} times the bound"


@pytest.mark.parametrize("dense", [True, False], ids=["dense", "rows"])
@pytest.mark.parametrize("size", [1.0, 0.1, 0.01, 0.001])
def test_one_key_dominates(size, dense):
    for gap in (9.0, 12.0):
        q, rows = sink_rows(8192, 8, size, gap, seed=3)
        for batch, splits in ((1, 1), (1, 5), (32, 1)):
            _check(rows, q, dense, splits, batch, (0, 5), f"V of {size}, gap {gap}, {batch} x {splits}")


@pytest.mark.parametrize("order", ["grow", "shrink", "mixed"])
def test_pages_of_all_sizes_in_one_sequence(order):
    g = torch.Generator().manual_seed(17)
    rows = torch.randn(2, 1504, 2, 128, generator=g)
    sizes = torch.logspace(-6, 3, 94)
    sizes = sizes.flip(0) if order == "shrink" else sizes[torch.randperm(94, generator=g)] if order == "mixed" else sizes
    rows[1] *= sizes.repeat_interleave(16)[:, None, None]
    rows[1, 160:176] = 0
    q = torch.randn(1, 8, 128, generator=g) * 2
    for dense in (True, False):
        for splits in (1, 3):
            _check(rows, q, dense, splits, 1, (0, 1), f"{order}, {splits} splits")

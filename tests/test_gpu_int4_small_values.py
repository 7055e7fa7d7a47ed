"""Attention over 4-bit rows whose values are small, or differ in size, where few keys take most of the weight (GPU): held to a bound
that is relative to the values."""
import math

import pytest
import torch

from tests.int4_bounds import attention, last_rounding, sink_rows
from tests.int4_util import K_PIECES, V_PIECES, pack, quantize, unpack

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
SCALE = 128 ** -0.5


class Rows:
    """Rows [2, n, G, 128] (K, V) as a paged 4-bit cache, and the values that it stands for."""

    def __init__(self, rows, page=16, seed=0):
        _, n, G, _ = rows.shape
        pages = -(-n // page)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
        padded = torch.zeros(2, pages * page, G, 128)
        padded[:, :n] = rows
        (kc, self.kp), (vc, self.vp) = quantize(padded[0]), quantize(padded[1])
        self.k, self.v = pack(kc, K_PIECES), pack(vc, V_PIECES)
        self.n, self.table, stored = n, torch.empty(1, pages, dtype=torch.int32), []
        self.table[0] = order.to(torch.int32)
        for x in (self.k, self.v, self.kp, self.vp):
            y = torch.empty_like(x).unflatten(0, (pages, page))
            y[order] = x.unflatten(0, (pages, page))
            stored.append(y.cuda())
        self.stored = stored

    def layout(self, batch, dtype):
        from kascade_b200 import _native as nat
        k, v, kp, vp = self.stored
        return nat.kv_layout_paged(k, v, self.table.expand(batch, -1).contiguous().cuda(), kp, vp, dtype)

    def plain(self, q, g):
        """q [4, 128] of KV head g -> what attention of these queries gives, and its bound."""
        n = self.n
        k, v = unpack(self.k[:n, g], self.kp[:n, g], K_PIECES), unpack(self.v[:n, g], self.vp[:n, g], V_PIECES)
        codes, scales = unpack(self.v[:n, g], self.vp[:n, g], V_PIECES, False), self.vp[:n, g, :4].double().repeat_interleave(32, -1)
        return attention(q.cpu().double(), k, v, codes, scales, SCALE)


def _decode(rows, q, G, splits, dense, batch=1):
    """Attention of q [1, 4 G, 128] over all rows, every sequence of the batch the same -> [batch, 4 G, 128]."""
    from kascade_b200 import _native as nat
    n, H = rows.n, 4 * G
    q = q.expand(batch, -1, -1).contiguous()
    out = torch.full((batch, H, 128), 9.0, dtype=q.dtype, device="cuda")
    ws = nat.decode_workspace(batch, H, splits, q.device)
    kv = rows.layout(batch, q.dtype)
    if dense:
        stride = -(-n // 4) * 4
        logits, pooled = (torch.zeros(batch, m, stride, device="cuda") for m in (H, G))
        lens, lse = torch.full((batch,), n, dtype=torch.int32, device="cuda"), torch.empty(batch, H, device="cuda")
        nat.decode_anchor_paged(q, kv, lens, n, SCALE, logits, pooled, out, lse, ws, splits)
    else:
        index = torch.stack([torch.randperm(n, generator=torch.Generator().manual_seed(g)) for g in range(G)]).to(torch.int32)
        nat.decode_sparse_paged(q, kv, index.expand(batch, -1, -1).contiguous().cuda(), None, n, None, SCALE, out, None, ws, splits)
    return out


def _check(rows, out, q, heads, what):
    for g in heads:
        want, bound = rows.plain(q[0, 4 * g:4 * g + 4], g)
        off = (out[4 * g:4 * g + 4].cpu().double() - want).abs()
        limit = bound + last_rounding(want, q.dtype)
        assert bool((off <= limit).all()), f"{what}, head {g}: {float((off / limit).max()):.3g} times the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dense", [True, False], ids=["dense", "rows"])
@pytest.mark.parametrize("size", [1.0, 0.1, 0.01, 0.001])
def test_one_key_dominates(size, dense, dtype):
    """With 1 and 5 splits of one sequence (16 warps in a CTA), and in batches whose CTAs have 8 and 4 warps."""
    G, n = 8, 8192
    for gap in (9.0, 12.0):
        q, rows = sink_rows(n, G, size, gap, seed=3)
        rows, q = Rows(rows), q.to(dtype).cuda()
        for batch, splits in ((1, 1), (1, 5), (32, 1), (32, 5)):
            out = _decode(rows, q, G, splits, dense, batch)
            assert torch.equal(out, out[:1].expand_as(out))
            _check(rows, out[0], q, (0, 5) if splits == 1 else (7,), f"V of {size}, gap {gap}, {batch} x {splits}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["grow", "shrink", "mixed"])
def test_values_of_all_sizes_in_one_sequence(order, dtype):
    """Rows of 1e-6 to 1e3: the scales' power of two moves many times, or every scale lies far below the first one's."""
    G, n = 2, 1500
    g = torch.Generator().manual_seed(17)
    rows = torch.randn(2, n, G, 128, generator=g)
    sizes = torch.logspace(-6, 3, n)
    sizes = sizes.flip(0) if order == "shrink" else sizes[torch.randperm(n, generator=g)] if order == "mixed" else sizes
    rows[1] *= sizes[:, None, None]
    rows[1, ::7, :, 32:64] = 0                                       # scales of zero
    rows = Rows(rows)
    q = (torch.randn(1, 8, 128, generator=g) * 2).to(dtype).cuda()
    for splits in (1, 3):
        for dense in (True, False):
            _check(rows, _decode(rows, q, G, splits, dense)[0], q, range(G), f"{order}, {splits} splits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [0.0, 1e-5, 3e3])
def test_values_at_the_ends_of_the_range(size, dtype):
    G, n = 1, 700
    g = torch.Generator().manual_seed(19)
    rows = torch.randn(2, n, G, 128, generator=g).clamp(-3, 3)
    rows[1] = (rows[1] + 0.5) * size
    rows = Rows(rows)
    q = torch.randn(1, 4, 128, generator=g).to(dtype).cuda()
    for dense in (True, False):
        _check(rows, _decode(rows, q, G, 2, dense)[0], q, range(G), f"V of {size}")


def test_a_row_that_is_not_a_number_spoils_its_group_only():
    G, n = 1, 200
    g = torch.Generator().manual_seed(23)
    rows = torch.randn(2, n, G, 128, generator=g) * 0.01
    rows[1, 77, 0, 40] = math.inf                                   # group 1
    stored = Rows(rows)
    q = torch.randn(1, 4, 128, generator=g).half().cuda()
    out = _decode(stored, q, G, 1, False)[0].cpu().double()
    want, bound = stored.plain(q[0], 0)
    inside = torch.arange(128) // 32 == 1
    assert bool(out[:, inside].isnan().all())
    k, v = unpack(stored.k[:n, 0], stored.kp[:n, 0], K_PIECES), unpack(stored.v[:n, 0], stored.vp[:n, 0], V_PIECES)[:, ~inside]
    codes = unpack(stored.v[:n, 0], stored.vp[:n, 0], V_PIECES, False)[:, ~inside]
    scales = stored.vp[:n, 0, :4].double().repeat_interleave(32, -1)[:, ~inside]
    want, bound = attention(q[0].cpu().double(), k, v, codes, scales, SCALE)
    assert bool(((out[:, ~inside] - want).abs() <= bound + last_rounding(want, torch.float16)).all())


@pytest.mark.parametrize("dense", [True, False], ids=["dense", "rows"])
def test_calls_repeat_themselves_to_the_last_bit(dense):
    q, rows = sink_rows(5000, 8, 0.1, 9.0, seed=5)
    rows, q = Rows(rows), q.half().cuda()
    first = _decode(rows, q, 8, 6, dense, 4)
    assert all(torch.equal(first, _decode(rows, q, 8, 6, dense, 4)) for _ in range(5))

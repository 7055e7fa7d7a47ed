"""Appends of tokens with positions of their own, on one axis and on several (GPU), against the formulas in 64 bits."""
import math

import pytest
import torch

from tests.int4_util import HALF_STEP, K_PIECES, quantize, unpack

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _turned(x, gain, positions, axes, inv_freq, eps, scale=1.0):
    """x [B, T, heads, 128], positions [A, B, T] -> 64 bits, and a bound of what 32-bit arithmetic may be off by."""
    x = x.double()
    if gain is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * gain.double()
    size = x[..., :64].abs() + x[..., 64:].abs()
    if inv_freq is not None:
        axes = torch.zeros(64, dtype=torch.long) if axes is None else axes.long()
        angle = positions.double().permute(1, 2, 0)[..., axes] * inv_freq.double()
        cos, sin = (scale * f(angle)[:, :, None] for f in (torch.cos, torch.sin))
        x = torch.cat([x[..., :64] * cos - x[..., 64:] * sin, x[..., 64:] * cos + x[..., :64] * sin], -1)
    # a handful of 32-bit roundings, and the angle's own to 32 bits after its reduction (pi 2^-24)
    return x, max(scale, 1.0) * 10 * 2.0 ** -23 * torch.cat([size, size], -1)


def _check(got, want, slack, dtype, what):
    off = (got.cpu().double() - want).abs() - HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -10) - slack
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0            # half a step of fp16's subnormals
    assert bool((off <= tiny).all()), f"{what}: {float(off.max()):.3g} too much"


def _paged(B, capacity, G, page, dtype, seed):
    per = -(-capacity // page)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * per + 2, generator=g)[:B * per].view(B, per).to(torch.int32)
    k, v = (torch.randn(B * per + 2, page, G, 128, generator=g).to(dtype).cuda() for _ in range(2))
    return k, v, table.cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("axes,interleaved", [(None, False), ([16, 24, 24], False), ([24, 20, 20], True), ([32, 32], False)])
def test_positions_on_axes(dtype, norm, axes, interleaved):
    from kascade_b200 import EfficientKascadeStrategy, rope_axis_map
    B, T, H, G, page = 3, 19, 8, 2, 16
    g = torch.Generator().manual_seed(3)
    starts, n_new = [5, 0, 40], [19, 0, 7]
    k, v, table = _paged(B, 64, G, page, dtype, 4)
    k0, v0 = k.cpu().clone(), v.cpu().clone()
    qkv = torch.randn(B, T, H + 2 * G, 128, generator=g).to(dtype).cuda()       # q, k, v are slices of one tensor
    gains = [(1 + 0.1 * torch.randn(128, generator=g)).to(dtype) for _ in range(2)] if norm else [None, None]
    inv_freq = 1000000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    A = 1 if axes is None else len(axes)
    positions = torch.randint(0, 200000, (A, B, T), generator=g)
    row = None if axes is None else rope_axis_map(axes, interleaved)
    if axes is not None:
        assert torch.bincount(row.cpu(), minlength=A).tolist() == axes
    noted = torch.full((B, 50), -7, dtype=torch.int32, device="cuda")
    dev = lambda x: None if x is None else x.cuda()                             # noqa: E731
    q_out = EfficientKascadeStrategy.append_kv(
        qkv[:, :, H:H + G], qkv[:, :, H + G:], k, v, table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
        torch.tensor(n_new, dtype=torch.int32, device="cuda"), query=qkv[:, :, :H], q_norm_weight=dev(gains[0]),
        k_norm_weight=dev(gains[1]), inv_freq=inv_freq.cuda(), rope_scale=1.25,
        positions=(positions[0] if axes is None else positions).cuda(), rope_axes=row, token_positions=noted)
    qkv = qkv.cpu()
    axis_row = None if row is None else row.cpu()
    want_q, slack_q = _turned(qkv[:, :, :H], gains[0], positions, axis_row, inv_freq, 1e-6, 1.25)
    want_k, slack_k = _turned(qkv[:, :, H:H + G], gains[1], positions, axis_row, inv_freq, 1e-6, 1.25)
    noted = noted.cpu()
    touched = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b in range(B):
        n = n_new[b]
        _check(q_out[b, :n], want_q[b, :n], slack_q[b, :n], dtype, "q")
        for t in range(n):
            r = starts[b] + t
            at = int(table[b, r // page]), r % page
            touched[at] = True
            _check(k[at], want_k[b, t], slack_k[b, t], dtype, "k")
            assert torch.equal(v[at].cpu(), qkv[b, t, H + G:])
            if r < 50:
                assert int(noted[b, r]) == int(positions[0, b, t])
                noted[b, r] = -7
    assert bool((noted == -7).all())
    assert torch.equal(k.cpu()[~touched], k0[~touched]) and torch.equal(v.cpu()[~touched], v0[~touched])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [0, 131071, 16777217, 2 ** 31 - 40, -5])
def test_far_positions(dtype, first):
    from kascade_b200 import EfficientKascadeStrategy
    B, T, G = 1, 33, 1
    g = torch.Generator().manual_seed(8)
    k, v, table = _paged(B, 64, G, 16, dtype, 9)
    new = torch.randn(B, T, 2, 128, generator=g).to(dtype)
    inv_freq = 10000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    positions = first + torch.arange(T)[None]
    EfficientKascadeStrategy.append_kv(new[:, :, :1].cuda(), new[:, :, 1:].cuda(), k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"),
                                       inv_freq=inv_freq.cuda(), positions=positions.cuda())
    want, slack = _turned(new[:, :, :1], None, positions[None], None, inv_freq, 1e-6)
    got = k[table[0].long()].flatten(0, 1)[:T]
    _check(got, want[0], slack[0], dtype, f"position {first}")


def test_a_long_append_with_positions():
    """Many CTAs, strided positions (a transposed tensor), a table of an axis that does not exist: clamped, not read beyond."""
    from kascade_b200 import EfficientKascadeStrategy
    T, G, H = 3001, 8, 32
    g = torch.Generator().manual_seed(10)
    k, v, table = _paged(1, T, G, 16, torch.bfloat16, 11)
    qkv = torch.randn(1, T, H + 2 * G, 128, generator=g).bfloat16()
    positions = torch.randint(0, 3000, (1, T, 3), generator=g, dtype=torch.int32).cuda().permute(2, 0, 1)
    axes = torch.tensor([0, 1, 2, 3, -1, 7] + [1] * 58, dtype=torch.int32)
    inv_freq = 500000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    q_out = EfficientKascadeStrategy.append_kv(
        qkv[:, :, H:H + G].cuda(), qkv[:, :, H + G:].cuda(), k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"),
        query=qkv[:, :, :H].cuda(), inv_freq=inv_freq.cuda(), positions=positions, rope_axes=axes.cuda())
    axes = axes.clamp(0, 2)
    want, slack = _turned(qkv[:, :, :H], None, positions.cpu(), axes, inv_freq, 1e-6)
    _check(q_out, want, slack, torch.bfloat16, "q")
    want, slack = _turned(qkv[:, :, H:H + G], None, positions.cpu(), axes, inv_freq, 1e-6)
    _check(k[table[0].long()].flatten(0, 1)[:T], want[0], slack[0], torch.bfloat16, "k")
    assert torch.equal(v[table[0].long()].flatten(0, 1)[:T].cpu(), qkv[0, :, H + G:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("store", ["fp8", "int4"])
def test_positions_into_quantised_caches(dtype, store):
    from kascade_b200 import EfficientKascadeStrategy, int4_kv_cache
    B, T, G, page = 1, 40, 2, 16
    g = torch.Generator().manual_seed(12)
    new = torch.randn(B, T, 2 * G, 128, generator=g).to(dtype)
    positions = torch.randint(0, 9000, (1, B, T), generator=g)
    inv_freq = 500000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")
    if store == "int4":
        k, v, ks, vs = int4_kv_cache(4, G, page)
    else:
        k, v = (torch.zeros(4, page, G, 128, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
        ks, vs = (torch.full((4, G), 0.02, device="cuda") for _ in range(2))
    EfficientKascadeStrategy.append_kv(new[:, :, :G].cuda(), new[:, :, G:].cuda(), k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"),
                                       inv_freq=inv_freq.cuda(), positions=positions.cuda(), k_scale=ks, v_scale=vs)
    want, slack = _turned(new[:, :, :G], None, positions, None, inv_freq, 1e-6)
    rows = lambda x: x[table[0].long()].flatten(0, 1)[:T].cpu()                  # noqa: E731
    if store == "int4":
        got = unpack(rows(k), rows(ks), K_PIECES)
        step = rows(ks)[..., :4].double().repeat_interleave(32, -1)
        # half a step; the zero and the scale are off by half a step of fp16 each, the scale fifteen times
        bound = 0.5 * step + slack[0] + 2.0 ** -11 * (want[0].abs().amax(-1, True) + 15 * step)
        assert bool(((got - want[0]).abs() <= bound * (1 + 1e-6)).all())
        _, par = quantize(new[0, :, G:])
        assert torch.equal(rows(vs), par)
    else:
        got = rows(k).float().double() * 0.02
        bound = 2.0 ** -4 * want[0].abs() + 0.02 * 2.0 ** -10 + HALF_STEP[dtype] * want[0].abs() * 1.1 + slack[0]
        sat = want[0].abs() > 0.02 * 448
        assert bool(((got - want[0]).abs() <= bound)[~sat].all())


def test_refusals_of_positions():
    from kascade_b200 import EfficientKascadeStrategy, _native as nat
    k, v, table = _paged(1, 16, 1, 16, torch.float16, 1)
    new = torch.zeros(1, 2, 1, 128, dtype=torch.float16, device="cuda")
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    freq = torch.ones(64, device="cuda")
    call = lambda **kw: EfficientKascadeStrategy.append_kv(new, new, k, v, table, start, inv_freq=freq, **kw)   # noqa: E731
    pos = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="rope_axes"):
        call(positions=pos[None].expand(3, 1, 2))
    with pytest.raises(ValueError, match="integers"):
        call(positions=pos.float())
    with pytest.raises(ValueError, match="belong to positions"):
        call(rope_axes=torch.zeros(64, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="belong to positions"):
        call(token_positions=pos)
    with pytest.raises(nat.KascadeNativeError, match="positions"):
        call(positions=pos[:, :1])
    with pytest.raises(nat.KascadeNativeError, match="pair_axis"):
        call(positions=pos, rope_axes=torch.zeros(32, dtype=torch.int32, device="cuda"))
    with pytest.raises(nat.KascadeNativeError, match="pair_axis"):
        call(positions=pos, rope_axes=torch.zeros(64, dtype=torch.int64, device="cuda"))
    with pytest.raises(nat.KascadeNativeError, match="token_positions"):
        call(positions=pos, token_positions=torch.zeros(2, 16, dtype=torch.int32, device="cuda"))
    with pytest.raises(nat.KascadeNativeError, match="cpu"):
        call(positions=pos.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,T", [(1, 1, 1), (3, 2, 9), (5, 1, 700)])
def test_odd_numbers_of_query_heads(dtype, H, G, T):
    from kascade_b200 import EfficientKascadeStrategy
    g = torch.Generator().manual_seed(H)
    k, v, table = _paged(2, T, G, 16, dtype, 6)
    q, new = (torch.randn(2, T, n, 128, generator=g).to(dtype).cuda() for n in (H, 2 * G))
    inv_freq = 10000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    positions = torch.randint(0, 100000, (1, 2, T), generator=g)
    gain = (1 + 0.1 * torch.randn(128, generator=g)).to(dtype)
    got = EfficientKascadeStrategy.append_kv(new[:, :, :G], new[:, :, G:], k, v, table, torch.zeros(2, dtype=torch.int32, device="cuda"),
                                             query=q, q_norm_weight=gain.cuda(), inv_freq=inv_freq.cuda(), positions=positions[0].cuda())
    want, slack = _turned(q.cpu(), gain, positions, None, inv_freq, 1e-6)
    _check(got, want, slack, dtype, "q")
    want, slack = _turned(new[:, :, :G].cpu(), None, positions, None, inv_freq, 1e-6)
    k, v, table = k.cpu(), v.cpu(), table.cpu().long()
    for b in range(2):
        for t in range(T):
            at = int(table[b, t // 16]), t % 16
            _check(k[at], want[b, t], slack[b, t], dtype, "k")
            assert torch.equal(v[at], new[b, t, G:].cpu())

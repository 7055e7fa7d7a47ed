"""Rows of a 4-bit cache that are read back (GPU): the ends of fp16's range, and attention over them."""
import math

import pytest
import torch

from tests.int4_bounds import last_rounding
from tests.int4_util import HALF_STEP, K_PIECES, V_PIECES, make_cache, pack, quantize, unpack

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
def test_finite_rows_are_read_back_finite(dtype):
    """A group from -65504 to 65504 has a scale of 8736 (8733.9 rounded to fp16), so its code 15 stands for 65536."""
    from kascade_b200 import EfficientKascadeStrategy as S, int4_kv_cache
    top = 65504.0
    x = torch.zeros(1, 6, 1, 128)
    x[0, 0, 0, 1::2], x[0, 0, 0, ::2] = top, -top
    x[0, 1] = torch.linspace(-top, top, 128)
    x[0, 2] = torch.linspace(0, top, 128)
    x[0, 3] = torch.linspace(-top, 0, 128)
    x[0, 4, 0, :2] = torch.tensor([1e30, -1e30]).clamp(-top, top) if dtype == torch.float16 else torch.tensor([1e30, -1e30])
    x[0, 5, 0, 3] = math.nan
    x = x.to(dtype)
    k, v, kp, vp = int4_kv_cache(1, 1)
    table, zero = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    S.append_kv(x.cuda(), x.cuda(), k, v, table, zero, k_scale=kp, v_scale=vp)
    rows = S.read_kv(k, v, table, zero + 6, 6, k_scale=kp, v_scale=vp, dtype=dtype)
    codes, par = quantize(x[0])
    want = unpack(pack(codes, K_PIECES), par, K_PIECES)[:, 0]
    if dtype == torch.float16:
        want = want.clamp(-top, top)
    for got in rows:
        got = got[0, :, 0].cpu().double()
        assert bool(got[:5].isfinite().all()) and bool(got[5, :32].isnan().all()) and bool((got[5, 32:] == 0).all())
        # one rounding to 32 bits, of numbers up to 2 x 65536, and one to 16
        assert bool(((got - want)[:5].abs() <= HALF_STEP[dtype] * want[:5].abs() + 2.0 ** -24 * 131072 + 2.0 ** -25).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_over_rows_that_were_read_back(dtype):
    """The prefill kernels take them as any 16-bit rows, with as many queries as keys; a later piece's attention is the caller's."""
    from kascade_b200 import EfficientKascadeStrategy
    G, n, scale = 2, 300, 128 ** -0.5
    k, v, kp, vp, table, kf, vf, _ = make_cache([n], G, 16, seed=4)
    strat = EfficientKascadeStrategy([0], "x/y", k=20, tile_size=32, head_mapping=[[0, 1]], register=False)
    key, value = strat.read_kv(k, v, table, torch.tensor([n], device="cuda"), n, k_scale=kp, v_scale=vp, dtype=dtype)
    q = torch.randn(1, 4 * G, n, 128, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()

    class M:
        layer_idx = 0

    out, _ = strat.attention_forward(M(), q, key.transpose(1, 2), value.transpose(1, 2), None, scale)      # [1, n, H, D]
    piece = 77                                                       # the last piece of the prompt, by the caller
    kr, vr = (x[0].transpose(0, 1).cpu().double().repeat_interleave(4, 0) for x in (key, value))           # [H, n, D]
    x = (q[0].cpu().double() @ kr.transpose(1, 2)) * scale
    p = torch.softmax(x.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf), -1)
    want = (p @ vr).transpose(0, 1)
    # probabilities rounded to the type and the sum of them not, logits good to 2^-15, and the last rounding
    bound = (HALF_STEP[dtype] * 2 + 2.0 ** -14) * (p @ vr.abs()).transpose(0, 1) + last_rounding(want, dtype)
    assert bool(((out[0].cpu().double() - want).abs() <= bound).all())
    late = torch.softmax(x[:, -piece:].masked_fill(~torch.ones(piece, n, dtype=torch.bool).tril(n - piece), -math.inf), -1) @ vr
    assert torch.allclose(late.transpose(0, 1), want[-piece:], rtol=1e-12, atol=1e-12)
    # against the values that the rows stand for: rounding them once moves a logit by that much of the products' size
    near = (q[0].cpu().double().abs() @ kr.abs().transpose(1, 2)).max() * scale * HALF_STEP[dtype]
    exact = torch.softmax(((q[0].cpu().double() @ kf[0].repeat_interleave(4, 0).transpose(1, 2)) * scale)
                          .masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf), -1)
    vx = vf[0].repeat_interleave(4, 0)
    assert bool(((exact @ vx).transpose(0, 1) - want).abs().le((2 * near * math.exp(near) + HALF_STEP[dtype] * 2)
                                                                 * (exact @ vx.abs()).transpose(0, 1)).all())

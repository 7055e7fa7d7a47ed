"""Rows of a 4-bit cache that are read back (GPU): the ends of fp16's range."""
import math

import pytest
import torch

from tests.int4_util import HALF_STEP, K_PIECES, pack, quantize, unpack

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

"""The bound that attention over 4-bit rows is held to rejects what it has to reject (CPU)."""
import pytest
import torch

from tests.int4_bounds import attention, last_rounding, sink_rows
from tests.int4_util import K_PIECES, V_PIECES, pack, quantize, unpack


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [9.0, 12.0])
@pytest.mark.parametrize("size", [1.0, 0.1, 0.01, 0.001])
def test_bound_of_attention_with_a_dominating_row(size, gap, dtype):
    n = 4096
    q, rows = sink_rows(n, 1, size, gap, seed=1)
    (kc, kp), (vc, vp) = quantize(rows[0, :, 0]), quantize(rows[1, :, 0])
    k, v = unpack(pack(kc, K_PIECES), kp, K_PIECES), unpack(pack(vc, V_PIECES), vp, V_PIECES)
    codes, scales = unpack(pack(vc, V_PIECES), vp, V_PIECES, False), vp[:, :4].double().repeat_interleave(32, -1)
    q = q[0].to(dtype).double()
    x = (q @ k.T) * 128 ** -0.5
    top = x.topk(2, -1).values
    assert bool(((top[:, 0] - top[:, 1]) > gap - 1.5).all()) and bool((x.argmax(-1) == n // 3).all())
    want, bound = attention(q, k, v, codes, scales, 128 ** -0.5)
    limit = bound + last_rounding(want, dtype)
    assert bool(((want.to(dtype).double() - want).abs() <= limit).all())
    low = torch.softmax(x, -1)
    minima = low @ (v - codes)                                         # what is left where all p s vanish
    others = torch.arange(n) != n // 3
    sink_only = want - low[:, others] @ codes[others]                  # ... of all rows but the sink
    for wrong in (torch.zeros_like(want), 0.9 * want, -want, minima, sink_only):
        share = ((wrong - want).abs() > limit).double().mean()
        assert float(share) > 0.8, f"{float(share):.2f} of the elements are seen to be wrong"


def test_bound_has_no_absolute_term():
    q, rows = sink_rows(300, 1, 1.0, 9.0, seed=2)
    k, zero = rows[0, :, 0].double(), torch.zeros(300, 128, dtype=torch.float64)
    _, bound = attention(q[0].double(), k, zero, zero, zero, 0.1)
    assert float(bound.max()) <= 300 * 15 * 2.0 ** -51

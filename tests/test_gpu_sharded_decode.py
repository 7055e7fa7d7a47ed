"""Decode steps of a sharded strategy whose mapping stays among the rank's own KV heads, against the unsharded one (one GPU: the ranks'
steps need nothing from each other)."""
import pytest
import torch

from tests.gpu_util import assert_close
from tests.int4_util import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own_rows", [False, True], ids=["anchor_rows", "index_rows"])
def test_reuse_layers_read_the_rows_of_the_ranks_own_heads(own_rows):
    from kascade_b200 import EfficientKascadeStrategy
    G, lens = 4, [900, 1500]
    k, v, kp, vp, table, *_ = make_cache(lens, G, 16, seed=7)
    g = torch.Generator().manual_seed(8)
    q = [(torch.randn(2, 4 * G, 128, generator=g)).half().cuda() for _ in range(2)]
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def steps(shard, heads):
        strat = EfficientKascadeStrategy([0], "x/y", k=20, tile_size=32, head_mapping=[[0, 1, 2, 3], [1, 1, 3, 2]], register=False,
                                         shard=shard)
        some = [x[:, :, heads] for x in (k, v, kp, vp)]
        qs = [x.view(2, G, 4, 128)[:, heads].reshape(2, -1, 128) for x in q]
        out = [strat.paged_decode_forward(0, qs[0], some[0], some[1], table, seq, 0.1, 1500, some[2], some[3])]
        rows = None
        if own_rows:
            rows = (strat._dec_idx.clone(), strat._dec_count.clone())
            strat._dec_idx.fill_(0)
        out.append(strat.paged_decode_forward(1, qs[1], some[0], some[1], table, seq, 0.1, 1500, some[2], some[3], index_rows=rows))
        return out

    whole = steps(None, slice(0, 4))
    for rank in (0, 1):
        part = steps((rank, 2), slice(2 * rank, 2 * rank + 2))
        for layer in range(2):
            want = whole[layer].view(2, G, 4, 128)[:, 2 * rank:2 * rank + 2].reshape(2, -1, 128)
            assert_close(part[layer], want.float(), what=f"rank {rank}, layer {layer}")


def test_rows_of_a_smaller_batch_are_refused():
    """A reuse layer whose anchor ran for fewer sequences or heads has no rows of its own."""
    from kascade_b200 import EfficientKascadeStrategy
    k, v, kp, vp, table, *_ = make_cache([200, 300, 250], 2, 16, seed=9)
    strat = EfficientKascadeStrategy([0], "x/y", k=20, tile_size=32, head_mapping=[[0, 1]] * 2, register=False)
    seq, q = torch.tensor([200, 300, 250], dtype=torch.int32, device="cuda"), torch.zeros(3, 8, 128, dtype=torch.float16, device="cuda")
    strat.paged_decode_forward(0, q[:2], k, v, table[:2], seq[:2], 0.1, 300, kp, vp)
    with pytest.raises(RuntimeError, match="2 sequences"):
        strat.paged_decode_forward(1, q, k, v, table, seq, 0.1, 300, kp, vp)
    strat.paged_decode_forward(1, q[:2], k, v, table[:2], seq[:2], 0.1, 300, kp, vp)

"""Reuse layers of decode steps whose head mapping does not fit the index rows at hand are refused before anything is launched (CPU)."""
import pytest
import torch

from kascade_b200 import EfficientKascadeStrategy

MAPPING = [[0, 1, 2, 3, 4, 5, 6, 7], [1, 0, 3, 3, 4, 6, 6, 2], [2, 2, 0, 1, 7, 7, 4, 5]]


def _step(strat, layer, G, rows=False):
    cache, table = torch.zeros(4, 16, G, 128, dtype=torch.float16), torch.zeros(1, 4, dtype=torch.int32)
    index = (torch.zeros(1, G, 8, dtype=torch.int32), torch.zeros(1, G, dtype=torch.int32)) if rows else None
    return strat.paged_decode_forward(layer, torch.zeros(1, 4 * G, 128, dtype=torch.float16), cache, cache, table, torch.tensor([9]), 0.1, 9,
                                      index_rows=index)


def _strategy(shard, mapping=MAPPING):
    return EfficientKascadeStrategy([0], "x/y", k=10, tile_size=32, head_mapping=mapping, register=False, shard=shard)


@pytest.mark.parametrize("rows", [False, True], ids=["anchor_rows", "index_rows"])
def test_rows_of_another_ranks_heads_are_refused(rows):
    with pytest.raises(NotImplementedError, match=r"KV heads \[2\]"):
        _step(_strategy((1, 2)), 1, 4, rows)                          # head 7 reads head 2's rows
    with pytest.raises(ValueError, match="8 KV heads"):
        _step(_strategy((0, 2)), 1, 8, rows)


def test_rows_of_this_ranks_heads_are_numbered_from_its_first():
    assert _strategy((0, 2))._decode_mapping(1, 4, "cpu").tolist() == [1, 0, 3, 3]
    assert _strategy((1, 2))._decode_mapping(2, 4, "cpu").tolist() == [3, 3, 0, 1]
    assert _strategy((0, 1))._decode_mapping(1, 8, "cpu").tolist() == MAPPING[1]
    assert _strategy(None)._decode_mapping(1, 8, "cpu").tolist() == MAPPING[1]


def test_mappings_that_do_not_fit_the_cache_are_refused():
    for mapping in ([[0, 1], [0, 2]], [[0, 1], [-1, 0]], [[0, 1], [0]]):
        with pytest.raises(ValueError, match="does not fit"):
            _strategy(None, mapping)._decode_mapping(1, 2, "cpu")

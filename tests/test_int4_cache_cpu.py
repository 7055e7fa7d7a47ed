"""Host side of the 4-bit cache, of positions on axes and of eviction, without a GPU: arguments, refusals, layouts."""
import pytest
import torch

from tests.int4_util import K_PIECES, V_PIECES, pack, quantize, unpack


def test_rope_axis_map():
    from kascade_b200 import rope_axis_map
    assert rope_axis_map([16, 24, 24], device="cpu").tolist() == [0] * 16 + [1] * 24 + [2] * 24
    row = rope_axis_map([24, 20, 20], interleaved=True, device="cpu").tolist()
    assert row[:60] == [0, 1, 2] * 20 and row[60:] == [0] * 4
    assert rope_axis_map([64], device="cpu").tolist() == [0] * 64
    for bad in ([], [16, 24], [-1, 65], [65]):
        with pytest.raises(ValueError, match="64"):
            rope_axis_map(bad, device="cpu")
    with pytest.raises(ValueError, match="interleaved"):
        rope_axis_map([2, 31, 31], interleaved=True, device="cpu")


def test_an_empty_4bit_cache():
    from kascade_b200 import _native as nat, int4_kv_cache
    k, v, ks, vs = int4_kv_cache(5, 3, page_size=8, device="cpu")
    assert k.shape == v.shape == (5, 8, 3, 64) and k.dtype == torch.uint8
    assert ks.shape == vs.shape == (5, 8, 3, 8) and ks.dtype == torch.float16 and ks.stride() == vs.stride()
    assert vs.data_ptr() - ks.data_ptr() == 16                       # beside each other
    assert nat.is_int4(k) and not nat.is_int4(torch.zeros(1, 16, 2, 128, dtype=torch.uint8))
    with pytest.raises(nat.KascadeNativeError, match="CUDA"):
        nat.kv_layout_paged(k, v, torch.zeros(1, 1, dtype=torch.int32), ks, vs)
    with pytest.raises(nat.KascadeNativeError, match="CUDA"):
        nat.kv_layout_contiguous(k, v, 8, ks, vs)


def test_plain_quantiser_is_its_own_inverse():
    """What the GPU tests hold the kernels to: packing loses nothing, values are within half a step."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(7, 3, 128, generator=g)
    codes, par = quantize(x)
    step = par[..., :4].double().repeat_interleave(32, -1)
    for pieces in (K_PIECES, V_PIECES):
        y = unpack(pack(codes, pieces), par, pieces)
        assert bool(((y - x.double()).abs() <= 0.5 * step + 2.0 ** -10 * x.abs().amax()).all())
    assert not torch.equal(pack(codes, K_PIECES), pack(codes, V_PIECES))


def test_refusals_without_a_gpu():
    from kascade_b200 import EfficientKascadeStrategy as S, _native as nat
    new = torch.zeros(1, 2, 2, 128, dtype=torch.float16)
    cache = torch.zeros(4, 16, 2, 128, dtype=torch.float16)
    table, start = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    freq = torch.ones(64)
    with pytest.raises(ValueError, match="integers"):
        S.append_kv(new, new, cache, cache, table, start, inv_freq=freq, positions=torch.zeros(1, 2))
    with pytest.raises(ValueError, match="integers"):
        S.append_kv(new, new, cache, cache, table, start, inv_freq=freq, positions=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="rope_axes"):
        S.append_kv(new, new, cache, cache, table, start, inv_freq=freq, positions=torch.zeros(2, 1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="belong to positions"):
        S.append_kv(new, new, cache, cache, table, start, token_positions=torch.zeros(1, 64, dtype=torch.int32))
    mass = torch.zeros(1, 64)
    pairs = [(cache, cache)]
    for kw in (dict(budget=0), dict(budget=8, recent=7, sinks=2), dict(budget=8, recent=-1), dict(budget=8, sinks=-1)):
        with pytest.raises(ValueError, match="budget"):
            S.evict_kv(pairs, table, start, mass, **kw)
    with pytest.raises(ValueError, match="one layer"):
        S.evict_kv([], table, start, mass, 8)
    with pytest.raises(ValueError, match="pages"):
        S.evict_kv(pairs, table, start, torch.zeros(1, 65), 8)
    with pytest.raises(ValueError, match="sequences"):
        S.evict_kv(pairs, table, torch.zeros(2, dtype=torch.int32), mass, 8)
    with pytest.raises(nat.KascadeNativeError, match="CUDA"):
        S.evict_kv(pairs, table, start, mass, 8)
    with pytest.raises(nat.KascadeNativeError, match="CUDA"):
        S.prompt_mass(torch.zeros(1, 2, 2, 128), mass)
    codes, par = torch.zeros(4, 16, 2, 64, dtype=torch.uint8), torch.zeros(4, 16, 2, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="pages"):
        S.read_kv(codes, codes, table, start, 65, k_scale=par, v_scale=par)
    with pytest.raises(ValueError, match="sequences"):
        S.read_kv(codes, codes, table, torch.zeros(3, dtype=torch.int32), 5, k_scale=par, v_scale=par)
    strat = S([0], "x/y", k=10, tile_size=32, head_mapping=[[0, 1]] * 2, register=False, shard=(0, 2))
    q = torch.zeros(1, 8, 1, 128, dtype=torch.float16)
    kv = torch.zeros(1, 2, 5, 128, dtype=torch.float16)

    class M:
        layer_idx = 0

    with pytest.raises(NotImplementedError, match="all heads"):
        strat.attention_forward(M(), q, kv, kv, None, 0.1, attention_mass=mass)


def test_c_entry_points_refuse_before_they_launch():
    """Null pointers and impossible sizes are answered with an error by the C functions, whatever the caller."""
    import ctypes as C
    from kascade_b200 import _native as nat
    if torch.cuda.is_available():
        pytest.skip("the library is initialised there: tests of the GPU cover the messages")
    lib = nat.load()
    layout = nat.KvLayout()
    assert lib.kb200_decode_anchor_paged_mass(None, 0, 0, C.byref(layout), None, 0, 0.0, None, None, 0, None, 0, None, None, None,
                                              0, 0, 4, 1, 0, None) != 0
    assert lib.kb200_mass_add_prompt(None, 0, None, None, None, 0, 0, 0, 1, 0, 0, None) != 0
    assert lib.kb200_evict(C.byref(layout), 1, None, None, 0, None, 0, 1, 0, 0, None, None, None, 0, None, 0, 0, 1, 0, None) != 0
    assert lib.kb200_evict_workspace_bytes(2, 5, 3) == 4 * (2 * 8 + 2 * (3 + 6) + 4) and lib.kb200_evict_workspace_bytes(0, 5, 3) == 0
    assert lib.kb200_kv_read(C.byref(layout), None, None, None, 0, 0, 1, None) != 0
    act = nat.ActLayout()
    assert lib.kb200_kv_write_at(C.byref(act), None, C.byref(act), C.byref(act), None, None, C.byref(layout), None, None, 0.0, None, 1.0,
                                 None, 0, 0, 0, 1, None) != 0
    assert b"null pointer" in lib.kb200_last_error()


def test_sharded_strategies_refuse_attention_mass_in_a_paged_step():
    from kascade_b200 import EfficientKascadeStrategy
    strat = EfficientKascadeStrategy([0], "x/y", k=10, tile_size=32, head_mapping=[[0, 1]] * 2, register=False, shard=(0, 2))
    cache, table = torch.zeros(4, 16, 1, 128, dtype=torch.float16), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="all heads"):
        strat.paged_decode_forward(0, torch.zeros(1, 4, 128, dtype=torch.float16), cache, cache, table, torch.tensor([9]), 0.1, 9,
                                   attention_mass=torch.zeros(1, 9))

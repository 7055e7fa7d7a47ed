"""The 4-bit KV cache (GPU): rows quantised on their way in, read back, and attended to, against plain forms in 64 bits."""
import math

import pytest
import torch

from tests.int4_util import HALF_STEP, K_PIECES, V_PIECES, attention, make_cache, pack, quantize, unpack

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _strategy(G=8, pct=10, layers=2, anchors=(0,), mapping=None):
    from kascade_b200 import EfficientKascadeStrategy
    heads = [list(range(G))] * layers if mapping is None else [list(range(G)), mapping]
    return EfficientKascadeStrategy(list(anchors), "x/y", k=pct, tile_size=32, head_mapping=heads, register=False)


def _empty_cache(B, capacity, G, page, seed=0):
    from kascade_b200 import int4_kv_cache
    per = -(-capacity // page)
    total = B * per + 2
    table = torch.randperm(total, generator=torch.Generator().manual_seed(seed))[:B * per].view(B, per).to(torch.int32)
    return (*int4_kv_cache(total, G, page), table.cuda())


def _written(cache, par, table, page, b, rows):
    pages = table[b].cpu().long()
    return torch.stack([cache.cpu()[pages[r // page], r % page] for r in rows]), \
        torch.stack([par.cpu()[pages[r // page], r % page] for r in rows])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,G,page,starts,n_new", [(1, 1, 8, 16, [0], None), (3, 5, 2, 16, [14, 0, 31], [5, 0, 2]),
                                                     (2, 33, 1, 1, [7, 0], None), (2, 19, 3, 64, [60, 1], [19, 19])])
def test_append_quantises_rows(dtype, B, T, G, page, starts, n_new):
    g = torch.Generator().manual_seed(5)
    capacity = max(starts) + T
    k, v, kp, vp, table = _empty_cache(B, capacity, G, page)
    k.fill_(0xA5), v.fill_(0x5A), kp.fill_(7.0), vp.fill_(9.0)
    before = [x.clone() for x in (k, v, kp, vp)]
    new = torch.randn(B, T, 2 * G, 128, generator=g) * 3
    new[..., 7] *= 10
    new = new.to(dtype).cuda()
    count = None if n_new is None else torch.tensor(n_new, dtype=torch.int32, device="cuda")
    strat = _strategy(G)
    assert strat.append_kv(new[:, :, :G], new[:, :, G:], k, v, table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                           count, k_scale=kp, v_scale=vp) is None
    touched = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b in range(B):
        n = T if n_new is None else n_new[b]
        for t in range(n):
            r = starts[b] + t
            touched[int(table[b, r // page]), r % page] = True
        if not n:
            continue
        rows = range(starts[b], starts[b] + n)
        for cache, par, x, pieces in ((k, kp, new[b, :n, :G], K_PIECES), (v, vp, new[b, :n, G:], V_PIECES)):
            got, got_par = _written(cache, par, table, page, b, rows)
            codes, want_par = quantize(x.cpu())
            assert torch.equal(got_par, want_par)
            assert torch.equal(got, pack(codes, pieces))
    for now, was in zip((k, v, kp, vp), before):                     # everything else is as it was
        assert torch.equal(now.cpu()[~touched], was.cpu()[~touched])


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_rows_out_of_the_ordinary(dtype):
    """Constant groups, steps below fp16's least, values at half steps, beyond fp16, infinities and NaN."""
    k, v, kp, vp, table = _empty_cache(1, 16, 1, 16)
    x = torch.zeros(1, 8, 1, 128)
    x[0, 0] = 3.25
    x[0, 1] = torch.arange(128) % 31 / 2.0                           # halves: ties of a step of one
    x[0, 2] = 1e-7 * torch.arange(128)
    x[0, 3] = torch.linspace(-60000, 60000, 128)
    x[0, 4] = torch.linspace(-1e-3, 1e-3, 128)
    x[0, 5, 0, 40] = math.inf
    x[0, 6, 0, 100] = math.nan
    x[0, 7] = 1e30 if dtype == torch.bfloat16 else 65504.0
    x[0, 7, 0, 64:] *= -1
    x = x.to(dtype)
    strat = _strategy(1)
    strat.append_kv(x.cuda(), x.cuda(), k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"), k_scale=kp, v_scale=vp)
    codes, par = quantize(x[0])
    for cache, got_par, pieces in ((k, kp, K_PIECES), (v, vp, V_PIECES)):
        got, p = _written(cache, got_par, table, 16, 0, range(8))
        assert torch.equal(p.nan_to_num(-1.0), par.nan_to_num(-1.0)) and torch.equal(p.isnan(), par.isnan())
        assert torch.equal(got, pack(codes, pieces))
    ko, vo = strat.read_kv(k, v, table, torch.tensor([8], dtype=torch.int32, device="cuda"), 8, k_scale=kp, v_scale=vp, dtype=dtype)
    assert torch.equal(ko[0, 0].cpu(), x[0, 0]) and torch.equal(vo[0, 0].cpu(), x[0, 0])
    assert ko[0, 5, 0, 32:64].isnan().all() and ko[0, 5, 0, :32].isfinite().all() and ko[0, 6, 0, 96:].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_normalises_and_rotates_before_it_quantises(dtype):
    """The rows are those of the module's arithmetic; cos and sin may differ in the last place, which may move a code by one."""
    from oracle.kv_write_oracle import kv_write as oracle_kv_write
    g = torch.Generator().manual_seed(6)
    B, T, H, G = 2, 21, 8, 2
    q, kn, vn = (torch.randn(B, T, n, 128, generator=g).to(dtype) for n in (H, G, G))
    gains = [(1 + 0.1 * torch.randn(128, generator=g)).to(dtype) for _ in range(2)]
    inv_freq = 500000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    k, v, kp, vp, table = _empty_cache(B, 40, G, 16)
    starts = torch.tensor([3, 15], dtype=torch.int32)
    strat = _strategy(G)
    q_out = strat.append_kv(kn.cuda(), vn.cuda(), k, v, table, starts.cuda(), query=q.cuda(), q_norm_weight=gains[0].cuda(),
                            k_norm_weight=gains[1].cuda(), inv_freq=inv_freq.cuda(), k_scale=kp, v_scale=vp)
    ref_k, ref_v = (torch.zeros(k.shape[0], 16, G, 128, dtype=dtype) for _ in range(2))
    ref_q = oracle_kv_write(q, kn, vn, starts.tolist(), None, ref_k, ref_v, table.cpu(), 16, gains[0], gains[1], 1e-6, inv_freq, 1.0)
    assert float((q_out.cpu().float() - ref_q.float()).abs().max()) <= 4 * HALF_STEP[dtype] * float(ref_q.float().abs().max())
    for b in range(B):
        rows = range(int(starts[b]), int(starts[b]) + T)
        got, par = _written(k, kp, table, 16, b, rows)
        want = torch.stack([ref_k[int(table[b, r // 16]), r % 16] for r in rows]).double()
        step = par[..., :4].double().repeat_interleave(32, -1)
        # half a step, a code moved by one, and the row's own last place
        assert bool(((unpack(got, par, K_PIECES) - want).abs() <= 0.51 * step + 4 * HALF_STEP[dtype] * want.abs().amax(-1, True)).all())
        got, par = _written(v, vp, table, 16, b, rows)
        assert torch.equal(got, pack(quantize(vn[b])[0], V_PIECES))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,G,page", [([1], 8, 16), ([33, 0, 17], 2, 16), ([5, 64], 3, 4)])
def test_rows_are_read_back(dtype, lens, G, page):
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, page, seed=3)
    longest = max(lens)
    ko, vo = _strategy(G).read_kv(k, v, table, torch.tensor(lens, device="cuda"), longest, k_scale=kp, v_scale=vp, dtype=dtype)
    assert ko.shape == (len(lens), longest, G, 128) and ko.dtype == dtype
    for got, want in ((ko, kf), (vo, vf)):
        got, want = got.cpu().double(), want.transpose(1, 2).clone()
        for b, n in enumerate(lens):
            want[b, n:] = 0
        # one rounding to 32 bits and one to 16
        assert bool(((got - want).abs() <= (HALF_STEP[dtype] + 2.0 ** -23) * want.abs()).all())


def _check_attention(out, lse, q, kf, vf, vc, rows_of, scale, dtype, what):
    B, H, D = q.shape
    G = kf.shape[1]
    q = q.cpu().double().view(B, G, 4, D)
    for b in range(B):
        for g in range(G):
            rows = rows_of(b, g)
            want, want_lse, _, bound, logit = attention(q[b, g], kf[b, g, rows], vf[b, g, rows], vc[b, g, rows], scale)
            got = out[b].view(G, 4, D)[g].cpu().double()
            off = (got - want).abs() - bound - HALF_STEP[dtype] * want.abs() - 2.0 ** -24
            assert bool((off <= 0).all()), f"{what} b{b} g{g} ({len(rows)} rows): {float(off.max()):.3g} too much"
            if lse is not None:
                got_lse = lse[b].view(G, 4)[g].cpu().double()
                if len(rows):
                    assert float((got_lse - want_lse).abs().max()) <= logit + 2.0 ** -22 * (1 + float(want_lse.abs().max())), what
                else:
                    assert bool((got_lse == -math.inf).all())


def _queries(B, H, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, H, 128, generator=g) * size).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("splits", [1, 3, 16])
@pytest.mark.parametrize("G,page", [(8, 16), (2, 1), (1, 32)])
def test_sparse_decode(dtype, splits, G, page):
    """Rows in any order, empty rows, counts at and around a tile's edge, a head map, strided index tensors."""
    from kascade_b200 import _native as nat
    lens = [700, 33, 1, 260]
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, page, seed=11, interleaved=page != 1)
    B, H, kmax = len(lens), 4 * G, 300
    g = torch.Generator().manual_seed(12)
    rows = torch.zeros(B, G, kmax + 5, dtype=torch.int32)
    counts = torch.zeros(B, G, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(G):
            c = min(n, [300, 0, 17, 16, 15, 128, 1, 255][(b + h) % 8])
            rows[b, h, :c] = torch.randperm(n, generator=g)[:c].to(torch.int32)
            counts[b, h] = c
    head_map = torch.randint(0, G, (G,), generator=g, dtype=torch.int32)
    q = _queries(B, H, dtype, 13)
    out = torch.full((B, H, 128), 9.0, dtype=dtype, device="cuda")
    lse = torch.zeros(B, H, device="cuda")
    kv = nat.kv_layout_paged(k, v, table, kp, vp, dtype)
    ws = nat.decode_workspace(B, H, splits, q.device)
    rd = rows.cuda()[:, :, :kmax]
    nat.decode_sparse_paged(q, kv, rd, counts.cuda(), kmax, head_map.cuda(), 128 ** -0.5, out, lse, ws, splits)
    _check_attention(out, lse, q, kf, vf, vc, lambda b, h: rows[b, head_map[h], :counts[b, head_map[h]]].tolist(), 128 ** -0.5, dtype,
                     f"sparse, {splits} splits")
    if splits <= 3:
        again = torch.empty_like(out)
        nat.decode_sparse_paged_noalloc(q, kv, rd, counts.cuda(), kmax, head_map.cuda(), 128 ** -0.5, again, None, splits)
        assert torch.equal(out, again)
    # without counts every row of the index tensor is used
    full = torch.stack([torch.stack([torch.randperm(33, generator=g)[:33] for _ in range(G)]) for _ in range(2)]).to(torch.int32)
    out = torch.empty(2, H, 128, dtype=dtype, device="cuda")
    kv = nat.kv_layout_paged(k, v, table[:2], kp, vp, dtype)
    nat.decode_sparse_paged(q[:2], kv, full.cuda(), None, 33, None, 0.3, out, None, ws, splits)
    _check_attention(out, None, q[:2], kf[:2], vf[:2], vc[:2], lambda b, h: full[b, h].tolist(), 0.3, dtype, "sparse, no counts")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("splits", [1, 5])
@pytest.mark.parametrize("has_v", [True, False], ids=["kv", "k_only"])
@pytest.mark.parametrize("lens", [[1], [15, 16, 17, 0], [129, 1000], [513, 64, 31]])
def test_dense_decode(dtype, splits, has_v, lens):
    from kascade_b200 import _native as nat
    G = 2
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=21)
    B, H, longest = len(lens), 4 * G, max(lens)
    q = _queries(B, H, dtype, 22)
    stride = -(-longest // 4) * 4
    logits = torch.full((B, H, stride), 77.0, device="cuda")
    pooled = torch.full((B, G, stride), 77.0, device="cuda")
    out = torch.full((B, H, 128), 9.0, dtype=dtype, device="cuda") if has_v else None
    lse = torch.zeros(B, H, device="cuda")
    kv = nat.kv_layout_paged(k, v if has_v else None, table, kp, vp if has_v else None, dtype)
    ws = nat.decode_workspace(B, H, splits, q.device)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    nat.decode_anchor_paged(q, kv, seq, longest, 128 ** -0.5, logits, pooled, out, lse, ws, splits)
    first = pooled.clone()
    mass = torch.rand(B, stride + 3, device="cuda")
    added = mass.clone()
    nat.decode_anchor_paged(q, kv, seq, longest, 128 ** -0.5, logits, pooled.fill_(77.0), out, lse, ws, splits, mass=added)
    assert torch.equal(pooled, first)                                 # the weight's sum changes nothing else
    if has_v:
        _check_attention(out, lse, q, kf, vf, vc, lambda b, h: list(range(lens[b])), 128 ** -0.5, dtype, f"dense, {splits} splits")
    for b, n in enumerate(lens):
        total = torch.zeros(n, dtype=torch.float64)
        for h in range(G):
            _, want_lse, p, _, logit = attention(q[b].cpu().double().view(G, 4, 128)[h], kf[b, h, :n], vf[b, h, :n], vc[b, h, :n], 128 ** -0.5)
            got = lse[b].view(G, 4)[h].cpu().double()
            if n:
                assert float((got - want_lse).abs().max()) <= logit + 2.0 ** -22 * (1 + float(want_lse.abs().max()))
            w = pooled[b, h, :n].cpu().double()
            bound = (2 * logit + 2.0 ** -20) * p.sum(0)
            assert bool(((w - p.sum(0)).abs() <= bound).all())
            assert bool((pooled[b, h, n:].cpu() == 77.0).all()) and bool((logits[b].view(G, 4, -1)[h, :, n:].cpu() == 77.0).all())
            total += w
        want = mass[b, :n].cpu().double() + total
        assert bool(((added[b, :n].cpu().double() - want).abs() <= 2.0 ** -22 * (G + 1) * want).all())
        assert torch.equal(added[b, n:], mass[b, n:])
    assert nat.read_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-4, 300.0], ids=["small", "large"])
def test_decode_of_queries_of_any_size(dtype, size):
    """Very small queries (every row weighs the same) and very large ones (one row takes all)."""
    from kascade_b200 import _native as nat
    lens, G = [200], 2
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=31)
    q = _queries(1, 8, dtype, 32, size)
    q[0, 3] = 0
    q[0, 5, 3] = 3e4                                                 # one element far above the others
    out = torch.empty(1, 8, 128, dtype=dtype, device="cuda")
    rows = torch.arange(200, dtype=torch.int32).expand(1, G, 200).contiguous()
    kv = nat.kv_layout_paged(k, v, table, kp, vp, dtype)
    nat.decode_sparse_paged(q, kv, rows.cuda(), None, 200, None, 128 ** -0.5, out, None, None, 1)
    _check_attention(out, None, q, kf, vf, vc, lambda b, h: list(range(200)), 128 ** -0.5, dtype, f"queries of {size}")


@pytest.mark.parametrize("size", [1e-3, 100.0], ids=["small", "large"])
def test_decode_of_values_of_any_size(size):
    from kascade_b200 import _native as nat
    G, n = 1, 333
    g = torch.Generator().manual_seed(41)
    x = torch.randn(2, 21, 16, G, 128, generator=g) * size
    kc, kp = quantize(x[0])
    vc, vp = quantize(x[1])
    k, v = pack(kc, K_PIECES), pack(vc, V_PIECES)
    table = torch.arange(21, dtype=torch.int32)[None]
    kf, vf, vc = (unpack(p, s, n, z).flatten(0, 1)[None, None, :, 0] for p, s, n, z in ((k, kp, K_PIECES, True), (v, vp, V_PIECES, True),
                                                                                     (v, vp, V_PIECES, False)))
    q = _queries(1, 4, torch.bfloat16, 42, 1.0 / size)
    out = torch.empty(1, 4, 128, dtype=torch.bfloat16, device="cuda")
    rows = torch.randperm(n, generator=g).to(torch.int32).view(1, 1, n)
    kv = nat.kv_layout_paged(k.cuda(), v.cuda(), table.cuda(), kp.cuda(), vp.cuda(), torch.bfloat16)
    nat.decode_sparse_paged(q, kv, rows.cuda(), None, n, None, 0.05, out, None, None, 1)
    _check_attention(out, None, q, kf, vf, vc, lambda b, h: list(range(n)), 0.05, torch.bfloat16, f"values of {size}")


def test_layouts_and_strides_of_a_4bit_cache():
    """A contiguous [B, G, L, 64] cache, one that is a slice of a larger tensor, queries that are a slice: equal results."""
    from kascade_b200 import _native as nat
    lens, G = [150, 150], 2
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=51)
    q_all = _queries(2, 16, torch.float16, 52)
    q = q_all[:, ::2]
    rows = torch.arange(150, dtype=torch.int32, device="cuda").expand(2, G, 150)

    def run(kv):
        out = torch.empty(2, 8, 128, dtype=torch.float16, device="cuda")
        nat.decode_sparse_paged(q, kv, rows, None, 150, None, 0.1, out, None, None, 1)
        return out

    want = run(nat.kv_layout_paged(k, v, table, kp, vp))
    _check_attention(want, None, q, kf, vf, vc, lambda b, h: list(range(150)), 0.1, torch.float16, "paged")
    wide = [torch.zeros(k.shape[0], 16, G + 1, d, dtype=t, device="cuda") for d, t in ((128, torch.uint8), (32, torch.float16))]
    wide[0][:, :, 1:, :64], wide[0][:, :, 1:, 64:] = k, v
    wide[1][:, :, 1:, 8:16], wide[1][:, :, 1:, 16:24] = kp, vp
    assert torch.equal(want, run(nat.kv_layout_paged(wide[0][:, :, 1:, :64], wide[0][:, :, 1:, 64:], table, wide[1][:, :, 1:, 8:16],
                                                     wide[1][:, :, 1:, 16:24])))
    flat = [x[table.long()].flatten(1, 2)[:, :150].transpose(1, 2).contiguous() for x in (k, v, kp, vp)]
    assert torch.equal(want, run(nat.kv_layout_contiguous(flat[0], flat[1], 16, flat[2], flat[3])))


def test_steps_over_a_4bit_cache_through_the_strategy():
    """Anchor and reuse layers select and attend as over the values that the cache stands for."""
    from oracle.kascade_oracle import band_check, pooled_scores_decode, topk_budget
    lens, G, pct = [900, 1500], 2, 20
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=61)
    strat = _strategy(G, pct, mapping=[1, 1])
    seq = torch.tensor(lens, device="cuda")
    q = [_queries(2, 8, torch.bfloat16, 62 + i) for i in range(2)]
    scale = 128 ** -0.5
    mass = torch.zeros(2, 1600, device="cuda")
    out = strat.paged_decode_forward(0, q[0], k, v, table, seq, scale, 1500, kp, vp, mean_seq_len=1200.0, attention_mass=mass)
    _check_attention(out, None, q[0], kf, vf, vc, lambda b, h: list(range(lens[b])), scale, torch.bfloat16, "layer 0")
    idx, cnt = strat._dec_idx.cpu().clone(), strat._dec_count.cpu().clone()
    for b, n in enumerate(lens):
        pooled, _ = pooled_scores_decode(q[0][b:b + 1].float().cpu()[:, :, None], kf[b:b + 1, :, :n].float(), scale)
        assert torch.allclose(mass[b, :n].cpu(), pooled[0].sum(0).float(), rtol=1e-4, atol=1e-7)
        assert bool((mass[b, n:] == 0).all())
        for h in range(G):
            assert int(cnt[b, h]) == topk_budget(pct, n, 32)
            ok, msg = band_check(pooled[0, h], idx[b, h, :cnt[b, h]].tolist(), int(cnt[b, h]), n)
            assert ok, msg
    out = strat.paged_decode_forward(1, q[1], k, v, table, seq, scale, 1500, kp, vp, attention_mass=mass)
    _check_attention(out, None, q[1], kf, vf, vc, lambda b, h: idx[b, 1, :cnt[b, 1]].tolist(), scale, torch.bfloat16, "layer 1")
    # the same rows handed over by the caller; the strategy's own rows stay
    again = _strategy(G, pct, mapping=[1, 1]).paged_decode_forward(1, q[1], k, v, table, seq, scale, 1500, kp, vp,
                                                                   index_rows=(idx.cuda(), cnt.cuda()))
    assert torch.equal(out, again) and torch.equal(strat._dec_idx.cpu(), idx)
    # short sequences are attended to in full
    short = torch.tensor([100, 128], device="cuda")
    strat.paged_decode_forward(0, q[0], k, v, table, short, scale, 128, kp, vp)
    out = strat.paged_decode_forward(1, q[1], k, v, table, short, scale, 128, kp, vp)
    _check_attention(out, None, q[1], kf, vf, vc, lambda b, h: list(range([100, 128][b])), scale, torch.bfloat16, "short")


def test_a_step_over_a_4bit_cache_replays_from_a_cuda_graph():
    from kascade_b200 import rope_axis_map
    lens, G = [700, 41], 2
    k, v, kp, vp, table, _, _, _ = make_cache([n + 1 for n in lens], G, 16, seed=71)
    strat = _strategy(G, 20, mapping=[1, 0])
    g = torch.Generator().manual_seed(72)
    q = torch.randn(2, 1, 8, 128, generator=g).half().cuda()
    new = torch.randn(2, 1, 4, 128, generator=g).half().cuda()
    start = torch.tensor(lens, dtype=torch.int32, device="cuda")
    seq = start + 1
    pos = torch.randint(0, 5000, (3, 2, 1), generator=g, dtype=torch.int32).cuda()
    axes = rope_axis_map([16, 24, 24])
    inv_freq = 10000.0 ** (-torch.arange(0, 128, 2, device="cuda").float() / 128)
    mass = torch.zeros(2, 1024, device="cuda")

    def step():
        qq = strat.append_kv(new[:, :, :2], new[:, :, 2:], k, v, table, start, query=q, inv_freq=inv_freq, k_scale=kp, v_scale=vp,
                             positions=pos, rope_axes=axes)[:, 0]
        outs = [strat.paged_decode_forward(i, qq, k, v, table, seq, 0.09, 701, kp, vp, attention_mass=mass) for i in range(2)]
        return outs + [strat.read_kv(k, v, table, seq, 701, k_scale=kp, v_scale=vp)[0]]

    first = [x.clone() for x in step()]
    once = mass.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    mass.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, outs)) and torch.equal(mass, once)
    new.mul_(0.5)
    graph.replay()
    assert not torch.equal(first[2], outs[2])
    fresh = step()
    assert all(torch.equal(a, b) for a, b in zip(fresh, outs))


def test_refusals_of_the_4bit_cache():
    from kascade_b200 import _native as nat
    k, v, kp, vp, table = _empty_cache(1, 64, 2, 16)
    err = nat.KascadeNativeError
    with pytest.raises(err, match="k_scale"):
        nat.kv_layout_paged(k, v, table)
    with pytest.raises(err, match="v_scale|k_scale"):
        nat.kv_layout_paged(k, v, table, kp)
    with pytest.raises(err, match="float16"):
        nat.kv_layout_paged(k, v, table, kp.float(), vp.float())
    with pytest.raises(err, match="expected"):
        nat.kv_layout_paged(k, v, table, kp[..., :4], vp[..., :4])
    with pytest.raises(err, match="strides"):
        nat.kv_layout_paged(k, v, table, kp, vp.contiguous())
    with pytest.raises(err, match="fp16 or bf16"):
        nat.kv_layout_paged(k, v, table, kp, vp, torch.float32)
    with pytest.raises(err, match="int32"):
        nat.kv_layout_paged(k, v, table.long(), kp, vp)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")
    rows = torch.zeros(1, 2, 16, dtype=torch.int32, device="cuda")
    with pytest.raises(err, match="act_dtype"):
        nat.decode_sparse_paged(q, nat.kv_layout_paged(k, v, table, kp, vp), rows, None, 16, None, 0.1, torch.empty_like(q), None, None, 1)
    new = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(err, match="act_dtype"):
        nat.kv_write(None, None, new, new, torch.zeros(1, dtype=torch.int32, device="cuda"), None, nat.kv_layout_paged(k, v, table, kp, vp))
    odd = torch.zeros(k.shape[0], 16, 2, 72, dtype=torch.uint8, device="cuda")[..., :64]
    with pytest.raises(err, match="16-byte"):
        nat.decode_sparse_paged(q, nat.kv_layout_paged(odd, odd, table, kp, vp, q.dtype), rows, None, 16, None, 0.1, torch.empty_like(q))
    half = torch.zeros(1, 16, 2, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(err, match="not INT4"):
        nat.kv_read(nat.kv_layout_paged(half, half, table), torch.ones(1, dtype=torch.int32, device="cuda"), torch.empty_like(half),
                    torch.empty_like(half))
    strat = _strategy(2)
    with pytest.raises(ValueError, match="pages"):
        strat.read_kv(k, v, table, torch.ones(1, device="cuda"), 65, k_scale=kp, v_scale=vp)
    with pytest.raises(ValueError, match="anchor"):
        strat.paged_decode_forward(0, q, k, v, table, torch.ones(1, device="cuda"), 0.1, 64, kp, vp, index_rows=(rows, rows[..., 0]))
    with pytest.raises(ValueError, match="index_rows"):
        strat.paged_decode_forward(1, q, k, v, table, torch.ones(1, device="cuda"), 0.1, 64, kp, vp, index_rows=(rows, rows))


def test_many_sequences_take_small_ctas():
    """Batches of 6 CTAs per SM and more run with four warps per CTA."""
    from kascade_b200 import _native as nat
    B, G = 112, 8
    lens = [(37 * i) % 90 + 1 for i in range(B)]
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=81)
    q = _queries(B, 4 * G, torch.float16, 82)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rows = torch.arange(90, dtype=torch.int32, device="cuda").expand(B, G, 90)
    counts = seq[:, None].expand(B, G).contiguous()
    out, lse = torch.empty(B, 4 * G, 128, dtype=torch.float16, device="cuda"), torch.empty(B, 4 * G, device="cuda")
    kv = nat.kv_layout_paged(k, v, table, kp, vp)
    nat.decode_sparse_paged(q, kv, rows, counts, 90, None, 128 ** -0.5, out, lse, None, 1)
    _check_attention(out[:20], lse[:20], q[:20], kf[:20], vf[:20], vc[:20], lambda b, h: list(range(lens[b])), 128 ** -0.5, torch.float16,
                     "112 sequences, sparse")
    ws = nat.decode_workspace(B, 4 * G, 2, q.device)
    two = torch.empty_like(out)
    nat.decode_sparse_paged(q, kv, rows, counts, 90, None, 128 ** -0.5, two, None, ws, 2)
    logits, pooled = torch.empty(B, 4 * G, 92, device="cuda"), torch.empty(B, G, 92, device="cuda")
    dense = torch.empty_like(out)
    nat.decode_anchor_paged(q, kv, seq, 90, 128 ** -0.5, logits, pooled, dense, lse, None, 1)
    for x in (two, dense):                                           # other splits and orders of sums: a step of fp16 apart at most
        assert float((x.float() - out.float()).abs().max()) <= 2.0 ** -9 * float(out.abs().max())


def test_rows_of_a_cache_beyond_32_bits():
    """Rows whose byte offsets pass 2^31 and 2^32: written, read back and attended to."""
    from kascade_b200 import _native as nat
    G, page = 2, 16
    strat = _strategy(G)
    stride = 3 * 2 ** 20                                              # bytes from page to page: 1500 pages span 4.7 GB
    pages = 1500
    store = torch.empty(2, pages * stride, dtype=torch.uint8, device="cuda")
    params = torch.empty(2, pages, page, G, 8, dtype=torch.float16, device="cuda")
    k, v = (x.as_strided((pages, page, G, 64), (stride, G * 64, 64, 1)) for x in store)
    table = torch.tensor([[0, 700, 1499, 1400]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(91)
    x = torch.randn(1, 60, 2 * G, 128, generator=g).half()
    strat.append_kv(x[:, :, :G].cuda(), x[:, :, G:].cuda(), k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"), k_scale=params[0],
                    v_scale=params[1])
    n = torch.tensor([60], dtype=torch.int32, device="cuda")
    ko, vo = strat.read_kv(k, v, table, n, 60, k_scale=params[0], v_scale=params[1])
    want = []
    for part, pieces in ((x[0, :, :G], K_PIECES), (x[0, :, G:], V_PIECES)):
        codes, par = quantize(part)
        want.append((unpack(pack(codes, pieces), par, pieces), unpack(pack(codes, pieces), par, pieces, False)))
    for got, (w, _) in zip((ko, vo), want):
        assert bool(((got[0].cpu().double() - w).abs() <= (2.0 ** -11 + 2.0 ** -23) * w.abs()).all())
    q = _queries(1, 4 * G, torch.float16, 92)
    out = torch.empty_like(q)
    rows = torch.arange(60, dtype=torch.int32, device="cuda").expand(1, G, 60)
    nat.decode_sparse_paged(q, nat.kv_layout_paged(k, v, table, params[0], params[1]), rows, None, 60, None, 0.08, out, None, None, 1)
    kf, vf, vc = (y.transpose(0, 1)[None] for y in (want[0][0], want[1][0], want[1][1]))
    _check_attention(out, None, q, kf, vf, vc, lambda b, h: list(range(60)), 0.08, torch.float16, "far pages")


@pytest.mark.parametrize("splits", [1, 7])
@pytest.mark.parametrize("n", [40000, 8191])
def test_sums_over_long_lists_are_not_rounded_one_way(n, splits):
    """All rows weigh the same (queries of zero), so every probability is exact and out is the mean of the values: small, while the
    codes' and the zeros' shares of it are large and opposite.  Sums that are rounded towards zero would drift apart."""
    from kascade_b200 import _native as nat
    k, v, kp, vp, table, kf, vf, vc = make_cache([n], 1, 16, seed=101, spread=0.0)
    q = torch.zeros(1, 4, 128, dtype=torch.float16, device="cuda")
    rows = torch.arange(n, dtype=torch.int32, device="cuda").view(1, 1, n)
    out, lse = torch.empty_like(q), torch.empty(1, 4, device="cuda")
    ws = nat.decode_workspace(1, 4, splits, q.device)
    nat.decode_sparse_paged(q, nat.kv_layout_paged(k, v, table, kp, vp), rows, None, n, None, 1.0, out, lse, ws, splits)
    want = vf[0, 0].mean(0)
    # the output's rounding, and 32-bit sums of either share: steps of 2^-24, at most 8 of them between two that are rounded to nearest
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -21 * (vc[0, 0].mean(0) + (vf - vc)[0, 0].abs().mean(0))
    assert bool(((out[0].cpu().double() - want).abs() <= bound).all())
    assert float((lse.cpu().double() - math.log2(n)).abs().max()) <= 2.0 ** -20 * math.log2(n)


def test_the_same_row_twice():
    """An index row may name a row more than once; it then counts as often."""
    from kascade_b200 import _native as nat
    lens, G = [90], 2
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=71)
    rows = torch.randint(0, 90, (1, G, 257), generator=torch.Generator().manual_seed(72), dtype=torch.int32)
    rows[0, 1] = 89
    q = _queries(1, 4 * G, torch.float16, 73)
    out = torch.empty(1, 4 * G, 128, dtype=torch.float16, device="cuda")
    kv = nat.kv_layout_paged(k, v, table, kp, vp)
    nat.decode_sparse_paged(q, kv, rows.cuda(), None, 257, None, 128 ** -0.5, out, None, nat.decode_workspace(1, 8, 2, q.device), 2)
    _check_attention(out, None, q, kf, vf, vc, lambda b, h: rows[b, h].tolist(), 128 ** -0.5, torch.float16, "repeated rows")


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_kv_heads(dtype):
    """70 KV heads: appended, read back, attended to."""
    from kascade_b200 import _native as nat
    G, B, T = 70, 2, 37
    g = torch.Generator().manual_seed(81)
    k, v, kp, vp, table = _empty_cache(B, T, G, 16)
    new = torch.randn(B, T, 2 * G, 128, generator=g).to(dtype).cuda()
    strat = _strategy(G)
    starts, lens = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.full((B,), T, dtype=torch.int32, device="cuda")
    strat.append_kv(new[:, :, :G], new[:, :, G:], k, v, table, starts, k_scale=kp, v_scale=vp)
    for b in range(B):
        for cache, par, x, pieces in ((k, kp, new[b, :, :G], K_PIECES), (v, vp, new[b, :, G:], V_PIECES)):
            got, got_par = _written(cache, par, table, 16, b, range(T))
            codes, want_par = quantize(x.cpu())
            assert torch.equal(got_par, want_par) and torch.equal(got, pack(codes, pieces))
    key, value = strat.read_kv(k, v, table, lens, T, k_scale=kp, v_scale=vp, dtype=dtype)
    flat = lambda c, p, pieces, zeros=True: torch.stack([                               # noqa: E731
        unpack(*_written(c, p, table, 16, b, range(T)), pieces, zeros) for b in range(B)]).transpose(1, 2)
    kf, vf, vc = flat(k, kp, K_PIECES), flat(v, vp, V_PIECES), flat(v, vp, V_PIECES, False)
    for got, want in ((key, kf), (value, vf)):
        off = (got.cpu().double().transpose(1, 2) - want).abs() - (HALF_STEP[dtype] + 2.0 ** -23) * want.abs() - 2.0 ** -25
        assert bool((off <= 0).all())
    q = _queries(B, 4 * G, dtype, 82)
    out = torch.empty(B, 4 * G, 128, dtype=dtype, device="cuda")
    rows = torch.arange(T, dtype=torch.int32, device="cuda").expand(B, G, T)
    nat.decode_sparse_paged(q, nat.kv_layout_paged(k, v, table, kp, vp, dtype), rows, None, T, None, 0.1, out, None, None, 1)
    _check_attention(out, None, q, kf, vf, vc, lambda b, h: list(range(T)), 0.1, dtype, "70 heads")


def test_two_strategies_on_two_streams():
    """Steps over one cache at once, each strategy with scratch of its own: the results of one after the other."""
    lens, G = [3000, 500], 8
    k, v, kp, vp, table, _, _, _ = make_cache(lens, G, 16, seed=91)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    strats, queries = [_strategy(G) for _ in range(2)], [_queries(2, 4 * G, torch.float16, 92 + i) for i in range(2)]
    masses = [torch.zeros(2, 3000, device="cuda") for _ in range(2)]

    def step(i):
        return [strats[i].paged_decode_forward(layer, queries[i], k, v, table, seq, 128 ** -0.5, 3000, kp, vp, attention_mass=masses[i])
                for layer in (0, 1)]

    alone = []
    for i in range(2):
        alone.append([x.clone() for x in step(i)] + [masses[i].clone()])
        masses[i].zero_()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                masses[i].zero_()
                last = step(i)
                if i == 0:
                    first = last
    torch.cuda.synchronize()
    for got, want, mass in ((first, alone[0], masses[0]), (last, alone[1], masses[1])):
        assert all(torch.equal(x, y) for x, y in zip([*got, mass], want))


@pytest.mark.parametrize("B", [5, 33, 64])
def test_dense_passes_of_ragged_batches_in_many_pieces(B):
    """More CTAs than start at once: the longest sequences come first, equal and empty ones among them."""
    from kascade_b200 import _native as nat
    G, splits = 8, 9
    g = torch.Generator().manual_seed(B)
    lens = [int(x) for x in torch.randint(0, 400, (B,), generator=g)]
    lens[0] = lens[B - 1] = 333
    lens[B // 2] = 0
    k, v, kp, vp, table, kf, vf, vc = make_cache(lens, G, 16, seed=95)
    q = _queries(B, 4 * G, torch.float16, 96)
    stride = 400
    logits, pooled = torch.zeros(B, 4 * G, stride, device="cuda"), torch.zeros(B, G, stride, device="cuda")
    out, lse = torch.empty(B, 4 * G, 128, dtype=torch.float16, device="cuda"), torch.zeros(B, 4 * G, device="cuda")
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv = nat.kv_layout_paged(k, v, table, kp, vp)
    nat.decode_anchor_paged(q, kv, seq, 400, 128 ** -0.5, logits, pooled, out, lse, nat.decode_workspace(B, 4 * G, splits, q.device), splits)
    _check_attention(out, lse, q, kf, vf, vc, lambda b, h: list(range(lens[b])), 128 ** -0.5, torch.float16, f"{B} ragged sequences")
    for b in (0, B // 2, B - 1):
        assert bool((logits[b, :, lens[b]:] == 0).all()) and bool((pooled[b, :, lens[b]:] == 0).all())

"""Collected attention weight and eviction (GPU): whole numbers and moved rows have to be equal, sums are checked in 64 bits."""
import math

import pytest
import torch

from tests.int4_util import K_PIECES, V_PIECES, attention, make_cache, unpack

pytestmark = pytest.mark.gpu


# ---- weight ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,G,L,lens", [(1, 8, 1, None), (1, 8, 33, None), (2, 3, 129, [129, 64]), (3, 8, 1000, [1000, 0, 33]),
                                        (1, 2, 4099, None), (2, 8, 6000, [5999, 300])])
def test_weight_of_a_prompt(B, G, L, lens):
    from kascade_b200 import EfficientKascadeStrategy, _native as nat
    T, stride = -(-L // 32), -(-L // 128) * 128
    g = torch.Generator().manual_seed(L)
    pooled = torch.rand(B, G, T, stride, generator=g).pow_(3)
    pooled[torch.arange(stride)[None, None, None].expand(B, G, T, -1) >= 32 * torch.arange(T)[None, None, :, None]] = math.nan
    wide = torch.rand(B, L + 7, generator=g).cuda()                    # more rows than the prompt, and not contiguous
    mass = wide[:, :L + 3]
    seq = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = EfficientKascadeStrategy.prompt_mass(pooled.cuda(), mass, seq).cpu()
    want = mass.cpu().double()
    for b in range(B):
        for t in range(1, T if lens is None else -(-lens[b] // 32)):
            want[b, :32 * t] += pooled[b, :, t, :32 * t].double().sum(0)
    # positive terms: every addition is good to half a step of the sum so far; sums of up to G T terms, mostly in pieces
    assert bool(((got.double() - want).abs() <= want * 2.0 ** -24 * (G * T + 4)).all())
    assert torch.equal(got[:, 32 * (T - 1):], mass.cpu()[:, 32 * (T - 1):])
    again = EfficientKascadeStrategy.prompt_mass(pooled.cuda(), mass, seq).cpu()
    assert torch.equal(got, again)
    inplace = mass.clone()
    nat.mass_add_prompt(pooled.cuda(), inplace, inplace, seq)
    assert torch.equal(inplace.cpu(), got)


@pytest.mark.parametrize("padding", [None, "left", "right"])
@pytest.mark.parametrize("L", [40, 300])
def test_prompts_and_steps_collect_weight(L, padding):
    """attention_forward(attention_mass=): the anchor layers' probabilities, summed over heads and over later tiles / the step."""
    from kascade_b200 import EfficientKascadeStrategy
    B, G, D = 2, 2, 128
    H = 4 * G
    g = torch.Generator().manual_seed(L)
    q, k, v = (torch.randn(B, n, L, D, generator=g).half().cuda() for n in (H, G, G))
    lens = [L, L] if padding is None else [L, L - 7]
    mask = None
    if padding:
        at = torch.arange(L, device="cuda")
        keep = torch.stack([(at >= L - n) if padding == "left" else (at < n) for n in lens])
        mask = torch.ones(L, L, dtype=torch.bool, device="cuda").tril()[None, None] & keep[:, None, None]
    strat = EfficientKascadeStrategy([0], "x/y", k=20, tile_size=32, head_mapping=[[0, 1]] * 2, register=False)

    class M:
        layer_idx = 0

    mass = torch.zeros(B, L + 9, device="cuda")
    out, _ = strat.attention_forward(M(), q, k, v, mask, D ** -0.5, attention_mass=mass)
    plain, _ = strat.attention_forward(M(), q, k, v, mask, D ** -0.5)
    assert torch.equal(out, plain)
    want = torch.zeros(B, L + 9, dtype=torch.float64)
    for b, n in enumerate(lens):
        s = slice(L - n, L) if padding == "left" else slice(0, n)
        x = q[b, :, s].double() @ k[b, :, s].double().repeat_interleave(4, 0).transpose(1, 2) * D ** -0.5
        x = x.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
        p = torch.softmax(x, -1).cpu()
        later = (torch.arange(n)[:, None] // 32 * 32) > torch.arange(n)[None]
        want[b, :n] = (p * later).sum((0, 1))
    # probabilities of 32-bit logits of fp16 operands, a polynomial exponential of 3e-6
    assert torch.allclose(mass.cpu().double(), want, rtol=5e-5, atol=1e-6)
    before = mass.clone()
    M.layer_idx = 1                                                    # a reuse layer adds nothing
    strat.attention_forward(M(), q, k, v, mask, D ** -0.5, attention_mass=mass)
    assert torch.equal(mass, before)
    M.layer_idx = 0
    one = mask[:, :, -1:] if padding == "left" else None
    if padding == "right":
        return
    strat.attention_forward(M(), q[:, :, -1:], k, v, one, D ** -0.5, attention_mass=mass)
    for b, n in enumerate(lens):
        x = (q[b, :, -1].double().view(G, 4, D) @ k[b, :, L - n:].double().transpose(1, 2)) * D ** -0.5
        want[b, :n] += torch.softmax(x, -1).sum((0, 1)).cpu()
    assert torch.allclose(mass.cpu().double(), want, rtol=5e-5, atol=1e-6)


# ---- eviction --------------------------------------------------------------------------------------------------------
def _plain_evict(lens, mass, positions, budget, recent, sinks):
    """Per sequence: moves [(source, target)], rows left, weight and positions after the moves."""
    B, S = mass.shape
    new_mass, new_pos, moves, left = torch.zeros_like(mass), torch.full((B, S), -1, dtype=torch.int32), [], []
    for b in range(B):
        n = min(lens[b], S)
        pos = [int(positions[b, j]) if positions is not None else j for j in range(n)]
        newest = max(pos, default=-1)
        rank = [(-math.inf if p < sinks or p > newest - recent else (0.0 if math.isnan(mass[b, j]) else -float(mass[b, j])), j)
                for j, p in enumerate(pos)]
        kept = sorted(j for _, j in sorted(rank)[:budget])
        k = len(kept)
        holes = [j for j in range(k) if j not in set(kept)]
        pairs = list(zip([j for j in kept if j >= k], holes))
        src = list(range(k))
        for s, t in pairs:
            src[t] = s
        for t, s in enumerate(src):
            new_mass[b, t], new_pos[b, t] = mass[b, s], pos[s]
        moves.append(pairs)
        left.append(k)
    return moves, left, new_mass, new_pos


def _tables(lens, S, page, seed):
    per = -(-S // page)
    table = torch.randperm(len(lens) * per + 3, generator=torch.Generator().manual_seed(seed))[:len(lens) * per]
    return table.view(len(lens), per).to(torch.int32), len(lens) * per + 3


def _run_evict(lens, S, budget, recent, sinks, G, page, layers, kind, mass, positions, seed=0):
    from kascade_b200 import EfficientKascadeStrategy
    g = torch.Generator().manual_seed(seed)
    table, pages = _tables(lens, S, page, seed)
    caches = []
    for _ in range(layers):
        if kind == "int4":
            params = torch.randn(pages, page, G, 16, generator=g).half().cuda()
            caches.append((*(torch.randint(0, 256, (pages, page, G, 64), generator=g, dtype=torch.uint8).cuda() for _ in range(2)),
                           params[..., :8], params[..., 8:]))
        else:
            caches.append(tuple(torch.randn(pages, page, G, 128, generator=g).to(kind).cuda() for _ in range(2)))
    before = [[x.cpu().clone() for x in c] for c in caches]
    got = EfficientKascadeStrategy.evict_kv(caches, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), mass.cuda(),
                                            budget, recent=recent, sinks=sinks,
                                            token_positions=None if positions is None else positions.cuda())
    moves, left, new_mass, new_pos = _plain_evict(lens, mass, positions, budget, recent, sinks)
    assert got[0].tolist() == left
    assert torch.equal(got[1].cpu().nan_to_num(-1.0), new_mass.nan_to_num(-1.0)) and torch.equal(got[2].cpu(), new_pos)
    for was, now in zip(before, caches):
        for x, y in zip(was, now):
            want = x.clone()
            for b, pairs in enumerate(moves):
                for s, t in pairs:
                    want[int(table[b, t // page]), t % page] = x[int(table[b, s // page]), s % page]
            assert torch.equal(y.cpu(), want)
    return got


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, "int4"], ids=["fp16", "bf16", "int4"])
@pytest.mark.parametrize("lens,S,budget,recent,sinks,G,page", [
    ([1], 1, 1, 0, 0, 8, 16), ([600], 600, 512, 64, 4, 8, 16), ([40, 0, 100, 99, 1], 101, 40, 5, 2, 2, 1),
    ([300, 299], 300, 1, 0, 0, 1, 32), ([300], 320, 299, 299, 0, 3, 16), ([77, 50], 80, 200, 10, 4, 2, 16)])
def test_eviction(kind, lens, S, budget, recent, sinks, G, page):
    g = torch.Generator().manual_seed(budget + S)
    mass = torch.rand(len(lens), S, generator=g).pow(4)
    _run_evict(lens, S, budget, recent, sinks, G, page, 2, kind, mass, None)
    # a cache that rows have left before: rows in any order, equal weights, none at all, NaN
    positions = torch.stack([torch.randperm(S, generator=g) for _ in lens]).to(torch.int32) * 3
    mass = torch.randint(0, 4, (len(lens), S), generator=g).float()
    mass[:, ::7] = math.nan
    _run_evict(lens, S, budget, recent, sinks, G, page, 1, kind, mass, positions, seed=1)


@pytest.mark.parametrize("S,budget", [(5000, 2500), (5000, 4999), (20000, 300), (70000, 35001)])
def test_eviction_of_long_sequences(S, budget):
    g = torch.Generator().manual_seed(S)
    mass = torch.rand(2, S, generator=g).pow(6)
    mass[1] = 0                                                      # ties throughout: the lowest rows stay
    _run_evict([S, S - 3], S, budget, 100, 4, 1, 16, 1, torch.float16, mass, None)


def test_eviction_of_many_layers():
    """More layers than one launch takes."""
    mass = torch.rand(1, 64, generator=torch.Generator().manual_seed(2))
    _run_evict([64], 64, 20, 4, 1, 1, 16, 35, torch.float16, mass, None)


def test_eviction_replays_from_a_cuda_graph():
    from kascade_b200 import EfficientKascadeStrategy
    S = 700
    g = torch.Generator().manual_seed(7)
    table, pages = _tables([S, S], S, 16, 7)
    table = table.cuda()
    cache = tuple(torch.randn(pages, 16, 2, 128, generator=g).half().cuda() for _ in range(2))
    start = [x.clone() for x in cache]
    lens = torch.tensor([S, 400], dtype=torch.int32, device="cuda")
    mass = torch.rand(2, S, generator=g).cuda()
    run = lambda: EfficientKascadeStrategy.evict_kv([cache], table, lens, mass, 256, recent=32)   # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(2):
        mass.copy_(torch.rand(2, S, generator=g))
        for x, y in zip(cache, start):
            x.copy_(y)
        graph.replay()
        replayed = [x.clone() for x in outs] + [x.clone() for x in cache]
        for x, y in zip(cache, start):
            x.copy_(y)
        assert all(torch.equal(a, b) for a, b in zip(replayed, list(run()) + list(cache)))


def test_refusals_of_eviction():
    from kascade_b200 import EfficientKascadeStrategy, _native as nat
    table, pages = _tables([64], 64, 16, 1)
    table = table.cuda()
    lens, mass = torch.tensor([64], dtype=torch.int32, device="cuda"), torch.rand(1, 64, device="cuda")
    cache = tuple(torch.zeros(pages, 16, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    call = lambda caches=(cache,), m=mass, budget=32, **kw: EfficientKascadeStrategy.evict_kv(   # noqa: E731
        list(caches), table, lens, m, budget, **kw)
    fp8 = [x.to(torch.float8_e4m3fn) for x in cache]
    scale = torch.ones(pages, 2, device="cuda")
    with pytest.raises(nat.KascadeNativeError, match="FP8"):
        call([(*fp8, scale, scale)])
    with pytest.raises(nat.KascadeNativeError, match="layer 1"):
        call([cache, tuple(x.bfloat16() for x in cache)])
    with pytest.raises(nat.KascadeNativeError, match="layer 1"):
        call([cache, tuple(torch.zeros(pages, 16, 4, 128, dtype=torch.float16, device="cuda")[:, :, :2] for _ in range(2))])
    with pytest.raises(nat.KascadeNativeError, match="token_positions"):
        call(token_positions=torch.zeros(1, 60, dtype=torch.int32, device="cuda"))
    with pytest.raises(nat.KascadeNativeError, match="mass"):
        call(m=mass.double())
    with pytest.raises(ValueError, match="budget"):
        call(budget=32, recent=30, sinks=3)
    with pytest.raises(ValueError, match="pages"):
        call(m=torch.rand(1, 65, device="cuda"))
    with pytest.raises(ValueError, match="one layer"):
        call([])
    assert bool((cache[0] == 0).all())


def test_a_conversation_in_a_4bit_cache_that_is_kept_short():
    """Append, attend, collect weight, evict, go on: every step against a plain simulation over the rows that are left."""
    from kascade_b200 import EfficientKascadeStrategy, int4_kv_cache
    B, G, H, budget, recent, S = 2, 2, 8, 150, 30, 208
    g = torch.Generator().manual_seed(17)
    scale = 128 ** -0.5
    inv_freq = 10000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    strat = EfficientKascadeStrategy([0], "x/y", k=20, tile_size=32, head_mapping=[[0, 1], [1, 0]], register=False)
    table, pages = _tables([S] * B, S, 16, 18)
    table_d = table.cuda()
    layers = [int4_kv_cache(pages, G) for _ in range(2)]
    lens = torch.tensor([180, 60], dtype=torch.int32)
    mass = torch.zeros(B, S, device="cuda")
    positions = torch.full((B, S), -1, dtype=torch.int32, device="cuda")
    seen = lens.clone()                                             # tokens so far: the next token's position
    prompt = torch.randn(2, B, 180, 2 * G, 128, generator=g).half()
    for (k, v, kp, vp), x in zip(layers, prompt):
        own = torch.arange(180, dtype=torch.int32).expand(B, 180).cuda()
        strat.append_kv(x[:, :, :G].cuda(), x[:, :, G:].cuda(), k, v, table_d, torch.zeros(B, dtype=torch.int32, device="cuda"),
                        lens.cuda(), inv_freq=inv_freq.cuda(), k_scale=kp, v_scale=vp, positions=own, token_positions=positions)
    tokens = [list(range(n)) for n in lens.tolist()]                # what the rows of a cache are, in the simulation
    evictions = 0
    for step in range(25):
        new = torch.randn(2, B, 1, H + 2 * G, 128, generator=g).half()
        before = mass.cpu().double()
        for i, ((k, v, kp, vp), x) in enumerate(zip(layers, new)):
            x = x.cuda()
            q = strat.append_kv(x[:, :, H:H + G], x[:, :, H + G:], k, v, table_d, lens.cuda(), query=x[:, :, :H], k_scale=kp,
                                v_scale=vp, inv_freq=inv_freq.cuda(), positions=seen[:, None].cuda(), token_positions=positions)
            out = strat.paged_decode_forward(i, q[:, 0], k, v, table_d, (lens + 1).cuda(), scale, int(lens.max()) + 1, kp, vp,
                                             attention_mass=mass)
            if i == 0:
                for b in range(B):
                    n = int(lens[b]) + 1
                    rows = table[b, torch.arange(n) // 16].long(), torch.arange(n) % 16
                    kf, vf, vc = (unpack(c.cpu()[rows], s.cpu()[rows], p, z) for c, s, p, z in ((k, kp, K_PIECES, True), (v, vp, V_PIECES, True),
                                                                                            (v, vp, V_PIECES, False)))
                    for h in range(G):
                        want, _, p, bound, _ = attention(q[b, 0].cpu().double().view(G, 4, 128)[h], kf[:, h], vf[:, h], vc[:, h], scale)
                        off = (out[b].view(G, 4, 128)[h].cpu().double() - want).abs()
                        assert bool((off <= bound + 2.0 ** -11 * want.abs() + 2.0 ** -24).all())
                        before[b, :n] += p.sum(0)
        lens, seen = lens + 1, seen + 1
        for b in range(B):
            tokens[b].append(int(seen[b]) - 1)
        assert torch.allclose(mass.cpu().double(), before, rtol=1e-4, atol=1e-6)
        assert [positions[b, :int(lens[b])].tolist() for b in range(B)] == tokens
        if int(lens.max()) >= 190:
            evictions += 1
            m, p = mass.cpu(), positions.cpu()
            new_lens, mass, positions = strat.evict_kv(layers, table_d, lens.cuda(), mass, budget, recent=recent, sinks=4,
                                                       token_positions=positions)
            _, left, want_mass, want_pos = _plain_evict(lens.tolist(), m, p, budget, recent, 4)
            assert new_lens.tolist() == left and torch.equal(mass.cpu(), want_mass) and torch.equal(positions.cpu(), want_pos)
            lens = new_lens.cpu()
            tokens = [want_pos[b, :left[b]].tolist() for b in range(B)]
            assert all(set(range(int(seen[b]) - recent, int(seen[b]))) <= set(t) and set(range(4)) <= set(t)
                       for b, t in enumerate(tokens))
    assert evictions >= 1 and int(lens[1]) == 85


def test_two_evictions_at_once_and_one_after_another():
    """Two calls on two streams have workspaces of their own; a second eviction of what the first left, with other budgets."""
    from kascade_b200 import EfficientKascadeStrategy
    g = torch.Generator().manual_seed(23)
    S, G = 900, 2
    table, pages = _tables([S, S - 100], S, 16, 23)
    masses = [torch.rand(2, S, generator=g) for _ in range(2)]
    caches = [tuple(torch.randn(pages, 16, G, 128, generator=g).half().cuda() for _ in range(2)) for _ in range(2)]
    before = [[x.cpu().clone() for x in c] for c in caches]
    table_d, lens, dev = table.cuda(), torch.tensor([S, S - 100], dtype=torch.int32, device="cuda"), [m.cuda() for m in masses]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st, cache, m, budget in zip(streams, caches, dev, (400, 650)):
        with torch.cuda.stream(st):
            got.append(EfficientKascadeStrategy.evict_kv([cache], table_d, lens, m, budget, recent=7, sinks=2))
    torch.cuda.synchronize()
    for i, budget in enumerate((400, 650)):
        moves, left, want_mass, want_pos = _plain_evict([S, S - 100], masses[i], None, budget, 7, 2)
        assert got[i][0].tolist() == left and torch.equal(got[i][1].cpu(), want_mass) and torch.equal(got[i][2].cpu(), want_pos)
        for x, y in zip(before[i], caches[i]):
            for b, pairs in enumerate(moves):
                for s, t in pairs:
                    x[int(table[b, t // 16]), t % 16] = x[int(table[b, s // 16]), s % 16]
            assert torch.equal(y.cpu(), x)
    # again, from the rows that are left
    again = EfficientKascadeStrategy.evict_kv([caches[0]], table_d, got[0][0], got[0][1], 100, recent=7, sinks=2, token_positions=got[0][2])
    moves, left, want_mass, want_pos = _plain_evict([400, 400], got[0][1].cpu(), got[0][2].cpu(), 100, 7, 2)
    assert again[0].tolist() == left and torch.equal(again[1].cpu(), want_mass) and torch.equal(again[2].cpu(), want_pos)
    for x, y in zip(before[0], caches[0]):
        for b, pairs in enumerate(moves):
            for s, t in pairs:
                x[int(table[b, t // 16]), t % 16] = x[int(table[b, s // 16]), s % 16]
        assert torch.equal(y.cpu(), x)


def test_more_protected_rows_than_the_budget_holds():
    """Rows that share a position (images on several axes) can be more than `recent`: the lowest of them stay."""
    mass = torch.rand(1, 64, generator=torch.Generator().manual_seed(3))
    positions = torch.full((1, 64), 5, dtype=torch.int32)
    positions[0, 40:] = 9
    _run_evict([64], 64, 10, 6, 0, 1, 16, 1, torch.float16, mass, positions)


def test_refusals_of_attention_mass():
    from kascade_b200 import EfficientKascadeStrategy
    strat = EfficientKascadeStrategy([0], "x/y", k=20, tile_size=32, head_mapping=[[0, 1]] * 2, register=False)
    k, v, kp, vp, table, _, _, _ = make_cache([200], 2, 16, seed=1)
    q, lens = torch.zeros(1, 8, 128, dtype=torch.float16, device="cuda"), torch.tensor([200], device="cuda")
    good = torch.zeros(1, 200, device="cuda")
    for bad in (good[:, :199], good.double(), good.cpu(), torch.zeros(2, 200, device="cuda"), torch.zeros(1, 400, device="cuda")[:, ::2], good[0]):
        with pytest.raises(ValueError, match="attention_mass"):
            strat.paged_decode_forward(0, q, k, v, table, lens, 0.1, 200, kp, vp, attention_mass=bad)
    x, kv = torch.zeros(1, 8, 140, 128, dtype=torch.float16, device="cuda"), torch.zeros(1, 2, 140, 128, dtype=torch.float16, device="cuda")

    class M:
        layer_idx = 0

    with pytest.raises(ValueError, match="attention_mass"):
        strat.attention_forward(M(), x, kv, kv, None, 0.1, attention_mass=good[:, :139])


@pytest.mark.parametrize("S", [100, 6000])
@pytest.mark.parametrize("own", [False, True], ids=["in_order", "own_positions"])
def test_infinite_weight_does_not_displace_protected_rows(S, own):
    """Rows of infinite weight stay before others, the lowest first, but never in the place of a protected row."""
    g = torch.Generator().manual_seed(9)
    mass = torch.rand(1, S, generator=g)
    mass[0, 3:60] = math.inf
    mass[0, 61] = -math.inf
    order = torch.randperm(S, generator=g) if own else torch.arange(S)              # the row of each position
    positions = torch.empty(1, S, dtype=torch.int32)
    positions[0, order] = torch.arange(S, dtype=torch.int32)
    from kascade_b200 import EfficientKascadeStrategy
    table, pages = _tables([S], S, 16, 1)
    cache = tuple(torch.zeros(pages, 16, 1, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    lens, weight, at = EfficientKascadeStrategy.evict_kv([cache], table.cuda(), torch.tensor([S], dtype=torch.int32, device="cuda"),
                                                         mass.cuda(), 30, recent=8, sinks=2,
                                                         token_positions=positions.cuda() if own else None)
    protected = {0, 1, *range(S - 8, S)}
    others = [int(positions[0, j]) for j in range(3, 60) if int(positions[0, j]) not in protected][:20]
    assert lens.tolist() == [30]
    assert sorted(at[0, :30].tolist()) == sorted([*protected, *others])
    assert torch.equal(weight[0, :30].cpu(), mass[0, order[at[0, :30].cpu().long()]])


def test_a_budget_beyond_the_rows_keeps_them_all():
    """Also where more rows are protected than there are."""
    lens, mass = [64, 10, 0], torch.rand(3, 64, generator=torch.Generator().manual_seed(4))
    got = _run_evict(lens, 64, 500, 100, 20, 2, 16, 1, torch.float16, mass, None)
    for b, n in enumerate(lens):
        assert got[2][b].tolist() == [*range(n), *[-1] * (64 - n)]


def test_calls_on_nothing():
    """No rows, no sequences, no tokens: results of that size, and no error."""
    from kascade_b200 import EfficientKascadeStrategy as S, int4_kv_cache
    k, v, kp, vp = int4_kv_cache(4, 2)
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")      # noqa: E731
    for B, rows in ((2, 0), (0, 16), (0, 0)):
        lens, mass, at = S.evict_kv([(k, v, kp, vp)], i32(B, 1), i32(B), torch.zeros(B, rows, device="cuda"), 8, recent=4)
        assert lens.tolist() == [0] * B and mass.shape == at.shape == (B, rows)
        key, value = S.read_kv(k, v, i32(B, 1), i32(B), rows, k_scale=kp, v_scale=vp)
        assert key.shape == value.shape == (B, rows, 2, 128)
    mass = torch.rand(1, 5, device="cuda")
    assert torch.equal(S.prompt_mass(torch.zeros(1, 2, 0, 128, device="cuda"), mass), mass)
    assert S.prompt_mass(torch.zeros(0, 2, 1, 128, device="cuda"), mass[:0]).shape == (0, 5)
    new = torch.zeros(2, 0, 2, 128, dtype=torch.float16, device="cuda")
    q = S.append_kv(new, new, k, v, i32(2, 1), i32(2), query=torch.zeros(2, 0, 8, 128, dtype=torch.float16, device="cuda"),
                    k_scale=kp, v_scale=vp, positions=i32(2, 0))
    assert q.shape == (2, 0, 8, 128) and not bool(k.any())


def test_weight_of_a_prompt_replays_from_a_cuda_graph():
    from kascade_b200 import EfficientKascadeStrategy as S
    g = torch.Generator().manual_seed(2)
    pooled, mass = torch.rand(2, 2, 5, 256, generator=g).cuda(), torch.rand(2, 160, generator=g).cuda()
    lens = torch.tensor([160, 70], dtype=torch.int32, device="cuda")
    S.prompt_mass(pooled, mass, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = S.prompt_mass(pooled, mass, lens)
    for _ in range(2):
        pooled.copy_(torch.rand(2, 2, 5, 256, generator=g))
        mass.copy_(torch.rand(2, 160, generator=g))
        lens.copy_(torch.tensor([33, 160], dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, S.prompt_mass(pooled, mass, lens))

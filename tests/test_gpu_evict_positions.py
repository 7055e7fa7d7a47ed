"""Eviction where rows share token positions, as the patches of an image or a video frame do, or have none (GPU)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain(mass, pos, budget, recent, sinks):
    """Rows that stay, of one sequence."""
    n, newest = len(pos), max(pos)
    first = [0 <= p < sinks for p in pos]
    last = [p > newest - recent for p in pos]
    weight = [0.0 if math.isnan(m) else m for m in mass]
    if sum(f or r for f, r in zip(first, last)) <= budget or sum(p == newest for p in pos) > budget:
        rank = [(0 if first[j] or last[j] else 1, 0 if first[j] or last[j] else -weight[j], j) for j in range(n)]
    else:
        front = set([j for j in range(n) if first[j]][:sinks])
        rank = [(0, 0, j) if j in front else (1, newest - pos[j], j) if last[j] else (2, -weight[j], j) for j in range(n)]
    return sorted(j for *_, j in sorted(rank)[:budget])


def _run(mass, positions, budget, recent, sinks):
    """One layer of one head whose rows hold their own numbers -> the rows that are left in each sequence, checked against the plain form."""
    from kascade_b200 import EfficientKascadeStrategy
    B, S = mass.shape
    per = -(-S // 16)
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(1)).view(B, per).to(torch.int32)
    cache = torch.zeros(2, B * per, 16, 1, 128, dtype=torch.bfloat16)
    rows = torch.arange(per * 16)
    for b in range(B):                                              # two digits of the row's number, exact in bf16
        cache[:, table[b].long()[rows // 16], rows % 16, 0, 0] = (rows // 256).to(torch.bfloat16)
        cache[:, table[b].long()[rows // 16], rows % 16, 0, 1] = (rows % 256).to(torch.bfloat16)
    cache = cache.cuda()
    lens = torch.full((B,), S, dtype=torch.int32, device="cuda")
    new, weight, at = EfficientKascadeStrategy.evict_kv([(cache[0], cache[1])], table.cuda(), lens, mass.cuda(), budget, recent=recent,
                                                        sinks=sinks, token_positions=positions.cuda())
    left = []
    for b in range(B):
        n = int(new[b])
        want = _plain(mass[b].tolist(), positions[b].tolist(), budget, recent, sinks)
        for x in cache.cpu():
            row = x[table[b].long()[rows // 16], rows % 16, 0, :2].double()
            got = (row[:n, 0] * 256 + row[:n, 1]).long()
            assert sorted(got.tolist()) == want
        assert torch.equal(at[b, :n].cpu(), positions[b][got]) and bool((at[b, n:] == -1).all())
        assert torch.equal(weight[b, :n].cpu().nan_to_num(-1.0), mass[b][got].nan_to_num(-1.0))
        left.append(want)
    return left


@pytest.mark.parametrize("S", [300, 6000])
def test_a_frame_of_one_position_followed_by_text(S):
    """The last tokens stay, whatever the number of patches in the positions that are protected with them."""
    g = torch.Generator().manual_seed(S)
    frame = S // 3
    positions = torch.cat([torch.arange(20), 20 + torch.arange(S - 60) // frame, 24 + torch.arange(40)])[None].to(torch.int32)
    mass = torch.rand(2, S, generator=g).pow(4)
    positions = torch.cat([positions, positions[:, torch.randperm(S, generator=g)]])       # and in any order
    for left, pos in zip(_run(mass, positions, 90, 64, 4), positions):
        kept = pos[left].tolist()
        assert set(range(24, 64)) <= set(kept) and {0, 1, 2, 3} <= set(kept) and len(kept) == 90


@pytest.mark.parametrize("S", [300, 5000])
def test_first_positions_that_are_shared(S):
    """A video at the start: its frames do not displace the newest rows."""
    g = torch.Generator().manual_seed(S + 1)
    positions = torch.cat([torch.arange(S - 30) // (S // 5), 5 + torch.arange(30)])[None].to(torch.int32)
    mass = torch.rand(1, S, generator=g)
    mass[0, 7] = math.inf
    mass[0, 8] = math.nan
    mass[0, 9] = -0.0
    left = _run(mass, positions, S // 4, 20, 4)[0]
    assert set(range(S - 20, S)) <= set(left) and set(range(4)) <= set(left) and 7 in left
    left = _run(mass, positions, 25, 20, 4)[0]
    assert left == [0, 1, 2, 3, *([7] if 7 in left else []), *range(S - 20, S)]


def test_a_newest_position_beyond_the_budget():
    """All protected rows count alike then."""
    positions = torch.cat([torch.arange(50), torch.full((50,), 50)])[None].to(torch.int32)
    assert _run(torch.rand(1, 100), positions, 40, 10, 2)[0] == [0, 1, *range(41, 79)]


def test_rows_without_a_position_are_not_the_first_ones():
    mass = torch.arange(100).float()[None]
    positions = torch.arange(100, dtype=torch.int32)[None].clone()
    positions[0, 10:60] = -1
    assert _run(mass, positions, 20, 3, 0)[0] == [*range(80, 100)]
    assert _run(mass, positions, 20, 3, 12)[0] == [*range(10), *range(90, 100)]
    # none was noted, or all are negative: the newest of them is the newest
    assert _run(mass, torch.full((1, 100), -1, dtype=torch.int32), 20, 3, 5)[0] == [*range(20)]
    assert _run(-mass, -1 - torch.arange(100, dtype=torch.int32).flip(0)[None], 20, 5, 5)[0] == [*range(15), *range(95, 100)]


def test_running_numbers_on_an_axis_of_their_own():
    """What evict_kv counts by need not be an axis that the rotation uses."""
    from kascade_b200 import EfficientKascadeStrategy as S, rope_axis_map
    T, G = 96, 2
    g = torch.Generator().manual_seed(5)
    new = torch.randn(1, T, 2 * G, 128, generator=g).half().cuda()
    grid = torch.stack([torch.arange(T) // 48, torch.arange(T) // 8 % 6, torch.arange(T) % 8]).to(torch.int32)[:, None].cuda()
    inv = (1e4 ** (-torch.arange(0, 128, 2).float() / 128)).cuda()
    table, start = torch.arange(6, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda")
    sections = (16, 24, 24)
    caches, noted = [], []
    for number in (False, True):
        k, v = (torch.zeros(6, 16, G, 128, dtype=torch.float16, device="cuda") for _ in range(2))
        at = torch.full((1, T), -1, dtype=torch.int32, device="cuda")
        running = torch.arange(T, dtype=torch.int32, device="cuda")[None, None]
        S.append_kv(new[:, :, :G], new[:, :, G:], k, v, table, start, inv_freq=inv, token_positions=at,
                    positions=torch.cat([running, grid]) if number else grid,
                    rope_axes=rope_axis_map(sections) + 1 if number else rope_axis_map(sections))
        caches.append((k, v))
        noted.append(at)
    assert all(torch.equal(x, y) for x, y in zip(*caches))
    assert torch.equal(noted[0], grid[:1, 0]) and noted[1][0].tolist() == list(range(T))
    _, _, left = S.evict_kv([caches[1]], table, torch.tensor([T], device="cuda"), torch.zeros(1, T, device="cuda"), 20, recent=10, sinks=2,
                            token_positions=noted[1])
    assert sorted(left[0, :20].tolist()) == [*range(10), *range(86, 96)]


def test_rows_that_sequences_share():
    """The same weight and positions for all sequences, as broadcast tensors; the C entry takes no overlapping rows."""
    from kascade_b200 import EfficientKascadeStrategy as S, _native as nat
    B, rows = 3, 70
    mass, pos = torch.rand(1, rows, generator=torch.Generator().manual_seed(2)), torch.randperm(rows, generator=torch.Generator().manual_seed(3))
    left = _run(mass.expand(B, -1), pos.to(torch.int32).expand(B, -1), 20, 5, 2)
    assert left[0] == left[1] == left[2]
    k, v = (torch.zeros(B * 5, 16, 1, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    table, lens = torch.arange(B * 5, dtype=torch.int32, device="cuda").view(B, 5), torch.full((B,), rows, dtype=torch.int32, device="cuda")
    shared = mass.cuda().expand(B, -1)
    assert S.evict_kv([(k, v)], table, lens, shared, 20)[0].tolist() == [20] * B
    layout, lib = nat.kv_layout_paged(k, v, table), nat.load()
    at = torch.zeros(B, rows, dtype=torch.int32, device="cuda")
    new, out_m, out_p = torch.zeros_like(lens), torch.zeros(B, rows, device="cuda"), torch.zeros_like(at)
    size = lib.kb200_evict_workspace_bytes(B, rows, 20)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    own = mass.cuda().expand(B, -1).contiguous()
    for m, p in ((rows - 1, rows), (rows, rows - 1), (0, rows)):
        rc = lib.kb200_evict((nat.KvLayout * 1)(layout), 1, lens.data_ptr(), own.data_ptr(), m, at.data_ptr(), p, 20, 0, 0, new.data_ptr(),
                             out_m.data_ptr(), out_p.data_ptr(), rows, ws.data_ptr(), size, B, 1, rows, None)
        assert rc != 0 and b"overlap" in lib.kb200_last_error()
    assert not bool(new.any())

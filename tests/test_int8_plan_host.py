"""The split-KV chunk of an INT8 step's prompt chunks: the shortest of a few schedules, found at a cost near that of a 16-bit step's plan."""
import heapq
import random
import time

import pytest

from titan_engine_b200 import PagedKVCache

SMS = 148                                                   # of a handle without a device


def _cache(H, Hkv, ctx, new, dtype="int8", D=128):
    pages = [(a + b + 15) // 16 for a, b in zip(ctx, new)]
    c = PagedKVCache(1, H, Hkv, D, sum(pages), len(ctx), max(pages), dtype=dtype, io_dtype="bf16", max_step_tokens=max(sum(new), 64), host_only=True)
    seqs = [c.seq_alloc() for _ in ctx]
    for s, n in zip(seqs, ctx):
        c.reserve(s, n)
    return c, seqs


def _chunks(H, Hkv, ctx, new, workspace_rows):
    """Every item dealt to the least loaded SM, longest first, for each size that is considered; the first of the shortest schedules."""
    G = H // Hkv
    tpt = 256 // G
    big = [i for i, n in enumerate(new) if n * G > 16]
    tiles = [(ctx[i] + min(new[i], (t + 1) * tpt) + 63) // 64 for i in big for t in range(-(-new[i] // tpt))]
    share = max(4, -(-sum(tiles) * Hkv // SMS))
    fair = share
    if len(tiles) * Hkv <= 8 * SMS:
        best = None
        for cap in (max(tiles), share, share * 3 // 4, share // 2, share // 3, share // 4):
            cap = max(4, cap)
            cost = sorted((min(cap, b - at) + 6 + (10 if b > cap else 0) for b in tiles for at in range(0, b, cap) for _ in range(Hkv)), reverse=True)
            load = [0] * SMS
            for x in cost:
                heapq.heapreplace(load, load[0] + x)
            if best is None or max(load) < best:
                best, fair = max(load), cap
    small_rows = 0                                          # (no sequence here is left to the decode kernel)
    assert len(big) == len(new)
    for shrink in range(10):
        ct = [min(-(-(a + b) // 64) * 64, (fair * 64) << shrink, 32768) for a, b in zip(ctx, new)]
        rows = sum(-(-(a + b) // t) * b for a, b, t in zip(ctx, new, ct) if -(-(a + b) // t) > 1)
        if small_rows + rows <= max(workspace_rows, 4096) or shrink > 8:
            return ct


@pytest.mark.parametrize("seed", range(12))
def test_chunk_is_that_of_the_shortest_schedule(seed):
    r = random.Random(seed)
    Hkv, G = r.choice([1, 2, 3, 4, 8, 32]), r.choice([1, 2, 4, 8, 16])
    n = r.choice([1, 1, 2, 5, 9, 40])
    ctx = [r.randint(0, r.choice([50, 2000, 20000])) for _ in range(n)]
    new = [r.randint(17 if G == 1 else 16 // G + 1, r.choice([40, 600, 3000])) for _ in range(n)]
    c, seqs = _cache(G * Hkv, Hkv, ctx, new)
    c.step_begin(seqs, new)
    _, ct, n_decode = c.step_prefill_plan()
    rows = -(-c.cfg.num_pages * 16 // 128) + 2 * n          # what the handle's workspace holds
    assert n_decode == 0 and ct.tolist() == _chunks(G * Hkv, Hkv, ctx, new, rows)


@pytest.mark.parametrize("H,Hkv,ctx,new", [(32, 8, [0, 700, 1400, 2843, 500, 90, 2000, 1], [1024] * 8),
                                           (16, 4, [0, 1500, 700, 33, 1200, 900, 64, 1111, 400], [24, 492, 100, 350, 77, 200, 410, 61, 300])])
def test_plan_costs_no_more_than_a_16_bit_one(H, Hkv, ctx, new):
    """Twice as much and more while the schedules were simulated item by item."""
    best = {}
    for dtype in ("int8", "bf16"):
        c, seqs = _cache(H, Hkv, ctx, new, dtype)
        best[dtype] = 1.0
        for _ in range(60):
            t = time.perf_counter()
            c.step_begin(seqs, new)
            best[dtype] = min(best[dtype], time.perf_counter() - t)
            for s, n in zip(seqs, ctx):
                c.truncate(s, n)
    assert best["int8"] < 1.4 * best["bf16"], best

"""The paged-cache operators where they are likeliest to go wrong: waits that take
long, maxima that rise within a tile, V scales of every size, long tails of small
weights. Plain 64-bit implementations and bounds are those of test_gpu_kv_ops."""

import math

import pytest

from test_gpu_kv_ops import (PATTERNS, QMAX, attend_bound, attend_plain, check_attention, dense, make_cache,
                             run_attention)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------- waits

@pytest.mark.parametrize("page", [16, 24, 1])
@pytest.mark.parametrize("store", ["fp16", "e4m3"])
def test_loading_warps_wait_for_rows_made_again(cuda, store, page):
    """Rows made again token by token keep the loading warps waiting for a stage by the long form of a wait, which lanes
    leave at different times, in front of the places where all loading threads meet: by boxes, by rows and by codes."""
    torch = cuda
    counts, lens = [600, 300, 40], [2500, 3100, 900]

    def edit(k, v, ks, vs, table, q):
        for s, length in enumerate(lens):  # seen by each chunk's last query alone
            at = int(table[s, (length - 1) // page]), (length - 1) % page
            (v if vs is None else vs)[at] = math.nan

    got = run_attention(torch, "fp16", store, 128, 2, 4, page, counts, lens, seed=41, edit=edit)
    o, lse, want, wl, mag, dot = got[:6]
    last = torch.zeros(sum(counts), dtype=torch.bool, device="cuda")
    last[[sum(counts[:s + 1]) - 1 for s in range(len(counts))]] = True
    assert torch.isnan(o[last]).all()
    # The plain form's products of a zero weight and a NaN are not this operator's: its values come from a clean cache.
    clean = run_attention(torch, "fp16", store, 128, 2, 4, page, counts, lens, seed=41)
    check_attention(torch, (o[~last], lse[~last]) + tuple(x[~last] for x in clean[2:6]), 128, max(lens), store in QMAX)


# ----------------------------------------------------- maxima within a tile

@pytest.mark.parametrize("q_type, store", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "int8")])
@pytest.mark.parametrize("dim, step", [(128, 32), (128, 8), (64, 32)])
@pytest.mark.parametrize("pattern", ["chunk", "prefill", "mixed"])
def test_attention_rises_within_tiles(cuda, pattern, dim, step, q_type, store):
    """Scores whose exponentials rise by about 2^12 every few tokens: the running maximum is passed several times within
    each tile of 128 keys, weights already made and sums follow each time; over codes V's scales rise from tile to tile
    as well."""
    torch = cuda
    counts, lens = PATTERNS[pattern]
    page = 16

    def edit(k, v, ks, vs, table, q):
        q.copy_(q.abs() * 0.25 + 0.5)
        for s, length in enumerate(lens):
            for j in range(length):
                at = int(table[s, j // page]), j % page
                # sqrt(dim) * 0.7 * level: 8.4 more for each step, and down again after sixteen.
                level = (j // step) % 16 * 12.0 / math.sqrt(dim)
                if ks is None:
                    k[at] = (k[at].float() * 0.02 + level).to(k.dtype)
                else:
                    k[at] = torch.full_like(k[at].float(), 96.0).to(k.dtype)
                    ks[at] = max(level, 0.02) / 96.0
                    vs[at] *= 2.0 ** (j // 128 % 8)

    got = run_attention(torch, q_type, store, dim, 2, 4, page, counts, lens, seed=43, edit=edit)
    check_attention(torch, got, dim, max(lens), store in QMAX)

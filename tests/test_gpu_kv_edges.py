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

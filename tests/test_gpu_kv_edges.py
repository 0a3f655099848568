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


# ------------------------------------------------------- V scales of any size

@pytest.mark.parametrize("q_type, store", [("bf16", "e4m3"), ("fp16", "int8"), ("fp16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("pattern", ["verify", "chunk", "prefill", "mixed"])
@pytest.mark.parametrize("small", [2.0 ** -6, 2.0 ** -26])
def test_attention_ignores_masked_scales_of_any_size(cuda, pattern, q_type, store, small):
    """A V scale of 2^119 at the chunk's last token, 2^132 (2^152) times the others': more than an exponent's range away,
    in the same tile of keys as some rows' ends and in a later one than others'. Rows that do not see it are as exact
    as without."""
    torch = cuda
    if q_type == "fp16" and small < 2.0 ** -10:
        small *= 2.0 ** 12  # fp16 holds no smaller results
    counts, lens = PATTERNS[pattern]
    page, kw = 16, dict(seed=45)

    def shrink(k, v, ks, vs, table, q):
        vs.mul_(small)

    def edit(k, v, ks, vs, table, q):
        shrink(k, v, ks, vs, table, q)
        for s, length in enumerate(lens):
            if length:
                vs[int(table[s, (length - 1) // page]), (length - 1) % page] = 2.0 ** 119

    clean = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, edit=shrink, **kw)
    o, lse = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, edit=edit, **kw)[:2]
    tol, tol_l = attend_bound(torch, o.dtype, True, clean[2], clean[4], clean[5], max(lens), 128)
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half of its smallest step
    at = 0
    for n in counts:
        rows = slice(at, at + max(0, n - 1))
        assert ((o[rows].double() - clean[2][rows]).abs() <= tol[rows]).all()
        far = torch.where(torch.isinf(clean[3][rows]), 0.0, (lse[rows].double() - clean[3][rows]).abs())
        assert (far <= tol_l[rows] + clean[3][rows].abs().nan_to_num(posinf=0) * 2.0 ** -23).all()
        at += n


def scales_bound(torch, o, want, mag, dot, longest):
    """attend_bound, and what V scales that differ by more than 2^14 cost on top: 2^-11 of the row's largest magnitude."""
    tol, tol_l = attend_bound(torch, o.dtype, True, want, mag, dot, longest, 128)
    tol = tol + 2.0 ** -11 * mag.amax(2, keepdim=True)
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return tol, tol_l


@pytest.mark.parametrize("q_type, store", [("bf16", "e4m3"), ("fp16", "int8"), ("fp16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("pattern", ["chunk", "prefill", "mixed", "short"])
@pytest.mark.parametrize("window", [0, 90])
def test_attention_scales_of_any_size_in_chunks(cuda, pattern, q_type, store, window):
    """V scales over a hundred powers of two, all of them seen."""
    torch = cuda
    counts, lens = PATTERNS[pattern]

    def edit(k, v, ks, vs, table, q):
        g = torch.Generator(device="cuda").manual_seed(3)
        vs *= torch.exp2(torch.randint(-60, 41, vs.shape, generator=g, device="cuda").float())

    o, lse, want, wl, mag, dot, _ = run_attention(torch, q_type, store, 128, 2, 4, 16, counts, lens, seed=29, edit=edit,
                                                  window=window)
    tol, tol_l = scales_bound(torch, o, want, mag, dot, max(lens))
    # A value that may be off by tol may be anything from want - tol to want + tol: past the type's largest, infinity.
    on = want.abs() + tol < torch.finfo(o.dtype).max
    off = (o.double() - want).abs()
    assert (off[on] <= tol[on]).all(), f"worst {(off / tol)[on].max().item():.2f} of the bound"


@pytest.mark.parametrize("ratio", [14, 20, 24, 40, 90])
@pytest.mark.parametrize("q_type, store", [("bf16", "e4m3"), ("fp16", "int8")])
@pytest.mark.parametrize("pattern", ["decode", "verify", "chunk", "mixed"])
def test_attention_far_scale_of_small_weight(cuda, pattern, q_type, store, ratio):
    """Each sequence's first token, which all of it see, has a V scale 2^ratio times the mean of all (with those planted
    before it, so they grow from sequence to sequence) and a weight of about e^-90: as long as that is the smaller, the
    others' values are the result, whatever kernel takes the call."""
    torch = cuda
    counts, lens = PATTERNS[pattern]

    def edit(k, v, ks, vs, table, q):
        q.copy_(q.abs())
        k.copy_(k.float().abs().to(k.dtype))
        for s, length in enumerate(lens):
            b = int(table[s, 0])
            k[b, 0] = torch.full_like(k[b, 0].float(), -96.0).to(k.dtype)
            ks[b, 0] = 10.0 / 96.0
            vs[b, 0] = vs.mean() * 2.0 ** ratio

    for hints in (True, False):
        o, _, _, _, _, _, (cache, q, table, _, _) = run_attention(torch, q_type, store, 128, 2, 4, 16, counts, lens, seed=30,
                                                                  edit=edit, hints=hints)
        # A value is code * scale in fp32: the last sequence's first token of four (ratio 40) has 448 * 4.4e36 = 2e39, an
        # infinity there, and so have its rows.
        values = dense(torch, cache.value, cache.value_scale).float().double()
        want, wl, mag, dot = attend_plain(torch, q, dense(torch, cache.key, cache.key_scale), values, lens, counts, table,
                                          16, 1 / math.sqrt(128))
        tol, tol_l = scales_bound(torch, o, want, mag, dot, max(lens))
        # Rows that see the first token alone have it whole, and fp16 does not hold it then.
        on = want.abs() + tol < torch.finfo(o.dtype).max
        off = (o.double() - want).abs()
        assert (off[on] <= tol[on]).all(), f"worst {(off / tol)[on].max().item():.2f} of the bound"


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("pattern", ["decode", "decode_long", "verify", "chunk", "mixed"])
@pytest.mark.parametrize("power", [97, -85, "any"])
def test_attention_scales_near_the_ends(cuda, pattern, store, power):
    """V scales of 2^90 and of 2^-92, which bf16 results hold as well as others, and of every size between 2^-117 and
    2^108: both kernels, with and without the hints that choose between them."""
    torch = cuda
    counts, lens = PATTERNS[pattern]

    def edit(k, v, ks, vs, table, q):
        g = torch.Generator(device="cuda").manual_seed(3)
        vs *= 2.0 ** power if power != "any" else torch.exp2(torch.randint(-110, 115, vs.shape, generator=g,
                                                                           device="cuda").float())

    for hints in (True, False):
        o, lse, want, wl, mag, dot, _ = run_attention(torch, "bf16", store, 128, 2, 4, 16, counts, lens, seed=31, edit=edit,
                                                      hints=hints)
        tol, tol_l = scales_bound(torch, o, want, mag, dot, max(lens))
        if power == "any":
            # Decoding: half of fp16's smallest step, 2^-25 of the row's largest weight times scale, for each code.
            tol = tol + max(lens) * 2.0 ** -25 * mag.amax(2, keepdim=True) * 4
        off = (o.double() - want).abs()
        assert (off <= tol).all(), f"worst {(off / tol).max().item():.2f} of the bound"
        seen = ~torch.isinf(wl)
        assert ((lse.double() - wl).abs()[seen] <= (tol_l + wl.abs() * 2.0 ** -23)[seen]).all()


# ----------------------------------------------------- small weights, many

@pytest.mark.parametrize("q_type, store", [("fp16", "fp16"), ("fp16", "int8"), ("bf16", "e4m3"), ("fp16", "e4m3"),
                                           ("bf16", "bf16")])
@pytest.mark.parametrize("pattern", ["decode", "decode_long", "verify", "chunk", "mixed"])
def test_attention_small_weights_beside_a_strong_one(cuda, pattern, q_type, store):
    """Every 32nd token takes almost all the weight and has a V of zero: the result is what the others add up to, each
    with a weight of 20.5 * 2^-24 (about) of it. In fp16 units of the largest that would be 20 or 21 of the smallest
    steps; with the weights taken 2^5 up, 656."""
    torch = cuda
    counts, lens = PATTERNS[pattern]
    dim, weight = 128, 20.5 * 2.0 ** -24

    def edit(k, v, ks, vs, table, q):
        q.fill_(1.0)
        strong = -math.log(weight) / math.sqrt(dim)
        if ks is None:
            k.zero_(), v.fill_(1.0)
        else:
            k.zero_(), v.copy_(torch.full_like(v.float(), 96.0).to(v.dtype))
            ks.fill_(strong / 96.0), vs.fill_(1.0 / 96.0)
        for s, length in enumerate(lens):
            for j in range(0, length, 32):
                at = int(table[s, j // 16]), j % 16
                k[at] = torch.full_like(k[at].float(), strong if ks is None else 96.0).to(k.dtype)
                v[at] = torch.zeros_like(v[at].float()).to(v.dtype)

    o, lse, want, wl, mag, dot, _ = run_attention(torch, q_type, store, dim, 2, 4, 16, counts, lens, seed=33, edit=edit)
    tol, _ = attend_bound(torch, o.dtype, store in QMAX, want, mag, dot, max(lens), dim)
    # Half of fp16's smallest step beside weights of 656 of them; the strong key's rounding moves these by 0.4 % at most.
    tol = tol + mag / (2 * 650)
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = (o.double() - want).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max().item():.2f} of the bound"


# ------------------------------------------------------------- given scales

@pytest.mark.parametrize("dim", [64, 20])
@pytest.mark.parametrize("store", ["e4m3", "int8"])
def test_write_given_scales_of_both_sides(cuda, store, dim):
    """K and V by scales of their own, one for each block: rounded by them, saturated beyond, NaN kept (int8: 0); rows
    of 16-byte pieces and odd ones."""
    torch = cuda
    from pegaflow_b200 import KVCache, kv_write

    t = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}[store]
    k, v = (torch.zeros((4, 16, 2, dim), dtype=t, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(7)
    scales = [torch.exp2(torch.randint(-5, 3, (4, 1, 1), generator=g, device="cuda").float()) * 1.3 for _ in range(2)]
    cache = KVCache(k, v, *scales)
    x = torch.randn((2, 9, 2, dim), generator=g, device="cuda") * 60
    x[:, 3, 1, 5] = math.nan
    x[:, 4, 0, 7], x[:, 4, 0, 8] = math.inf, -math.inf
    slots = torch.randperm(64, generator=g, device="cuda")[:9]
    kv_write(cache, x[0], x[1], slots, given_scales=True)
    q = QMAX[store]
    for codes, s, y in ((k, scales[0], x[0]), (v, scales[1], x[1])):
        want = (y * (1.0 / s[slots // 16])).clamp(-q, q)  # both fp32 operations are correctly rounded; a NaN stays
        got = codes[slots // 16, slots % 16].float()
        if store == "int8":
            want = want.round().nan_to_num(0.0)
        else:
            want = want.to(t).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("dim", [64, 20])
@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -140])
def test_write_given_scales_without_an_inverse(cuda, store, dim, scale):
    """A scale that is not set yet (zero), or so small that 1 / scale is infinite: zeros stay zeros, which a product with
    an infinity would make NaN, and other values saturate."""
    torch = cuda
    from pegaflow_b200 import KVCache, kv_write

    t = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}[store]
    k, v = (torch.zeros((2, 16, 2, dim), dtype=t, device="cuda") for _ in range(2))
    cache = KVCache(k, v, *[torch.full((2, 1, 1), scale, device="cuda") for _ in range(2)])
    x = torch.zeros((3, 2, dim), device="cuda")
    x[1, 0, 3], x[1, 1, 4], x[2, 0, 0] = 5.0, -7.0, 0.25
    kv_write(cache, x, -x, torch.tensor([1, 17, 30], device="cuda"), given_scales=True)
    q = QMAX[store] * math.copysign(1.0, scale)
    for codes, y in ((k, x), (v, -x)):
        got = torch.stack([codes[0, 1], codes[1, 1], codes[1, 14]]).float()
        assert torch.equal(got, y.sign() * q)


# ----------------------------------------------------------------- gradients

def test_results_that_require_a_gradient(cuda):
    """Outputs that autograd follows are refused, and are written under no_grad()."""
    torch = cuda
    from pegaflow_b200 import chunk_attention, kv_read

    cache, k, v, ks, vs = make_cache(torch, "bf16", 2, 16, 2, 64, fill=5)
    table, starts = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    x = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros_like(x).requires_grad_()
    for call in (lambda: kv_read(cache, table, starts, out=(x, y)), lambda: chunk_attention(x, cache, table, starts, lens, out=y),
                 lambda: chunk_attention(y, cache, table, starts, lens)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    with torch.no_grad():
        kv_read(cache, table, starts, out=(x, y))
        assert torch.equal(y, v[1, :3])


# ------------------------------------------------------- weights in 16 bits

@pytest.mark.parametrize("q_type, store", [("bf16", "bf16"), ("fp16", "fp16"), ("fp16", "e4m3"), ("fp16", "int8")])
@pytest.mark.parametrize("dim, heads, group", [(128, 2, 4), (64, 3, 1), (80, 1, 4)])
@pytest.mark.parametrize("pattern", ["one", "decode", "decode_long", "verify"])
def test_attention_decoding_keeps_the_weights(cuda, pattern, dim, heads, group, q_type, store):
    """When decoding, what the rounding of a weight to 16 bits leaves has a product of its own: the result is off by its
    own rounding, and by 2^-8 of 2^-8 (fp16: 2^-11 of 2^-11) of the weighted magnitudes."""
    torch = cuda
    counts, lens = PATTERNS[pattern]
    o, lse, want, wl, mag, dot, _ = run_attention(torch, q_type, store, dim, heads, group, 16, counts, lens, seed=51)
    u, quantised = torch.finfo(o.dtype).eps / 2, store in QMAX
    tol, _ = attend_bound(torch, o.dtype, quantised, want, mag, dot, max(lens), dim)
    tol = tol - (u - u * u) * mag * 1.01
    if o.dtype == torch.float16:
        # The rest of a small weight is rounded to half of fp16's smallest step, 2^-25, beside a largest weight (times V
        # scale, of 1 to 2) of 2^5 at least, and values of 448 codes; results to half of the smallest step.
        tol = tol + 2.0 ** -25 + max(lens) * 2.0 ** -30 * 2 * mag.amax(2, keepdim=True)
    off = (o.double() - want).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max().item():.2f} of the bound"

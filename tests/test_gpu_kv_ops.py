"""The paged-cache operators on the GPU against plain 64-bit implementations.

Tolerances are derived from the roundings each operator makes (u = half a step
of a type, relative: eps / 2), element by element; see `attend_bound`.
"""

import math
import random

import pytest

pytestmark = pytest.mark.gpu

QMAX = {"e4m3": 448.0, "int8": 127.0}


def types(torch):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn,
            "int8": torch.int8}


def make_cache(torch, store, blocks, page, heads, dim, layout="kv_first", fill=None):
    """(KVCache, K view, V view, K scales, V scales), zeros or seeded values."""
    from pegaflow_b200 import KVCache

    t = types(torch)[store]
    if layout == "token_major":
        k, v = (torch.zeros((blocks, page, heads, dim), dtype=t, device="cuda") for _ in range(2))
    elif layout == "blocks_first":
        both = torch.zeros((blocks, 2, page, heads, dim), dtype=t, device="cuda")
        k, v = both[:, 0], both[:, 1]
    elif layout == "heads_first":  # [blocks, heads, page, dim], seen as [blocks, page, heads, dim]
        both = torch.zeros((2, blocks, heads, page, dim), dtype=t, device="cuda").transpose(2, 3)
        k, v = both[0], both[1]
    else:
        both = torch.zeros((2, blocks, page, heads, dim), dtype=t, device="cuda")
        k, v = both[0], both[1]
    ks = vs = None
    if store in QMAX:
        s = torch.zeros((2, blocks, page, heads), device="cuda")
        ks, vs = s[0], s[1]
    if fill is not None:
        g = torch.Generator(device="cuda").manual_seed(fill)
        for view, s in ((k, ks), (v, vs)):
            x = torch.randn((blocks, page, heads, dim), generator=g, device="cuda")
            if s is not None:
                s.copy_(x.abs().amax(3) / QMAX[store])
                x = x / s[..., None]
                x = x.round() if store == "int8" else x
                x = x.clamp(-QMAX[store], QMAX[store])
            view.copy_(x.to(t))
    return KVCache(k, v, ks, vs), k, v, ks, vs


def dense(torch, view, scale):
    x = view.double()
    return x if scale is None else x * scale.double()[..., None]


# ------------------------------------------------------------------- kv_write

def check_row(torch, store, x, codes, scale):
    """One side of a written cache against the formula: [n, heads, dim] rows."""
    x64 = x.double()
    if store not in QMAX:
        assert torch.equal(codes, x.to(codes.dtype))  # one rounding to the type, to nearest
        return
    want = torch.clamp(x64.abs().amax(2) / QMAX[store], min=2.0 ** -126)
    # One fp32 division.
    assert ((scale.double() - want).abs() <= want * 2.0 ** -24).all()
    # Codes are what the documented fp32 steps give, bit for bit: both operations are correctly rounded.
    y = (x.float() * (1.0 / scale)[..., None]).clamp(-QMAX[store], QMAX[store])
    assert torch.equal(codes.float(), y.round() if store == "int8" else y.to(codes.dtype).float())
    # And near the value: half a step of the code, plus three fp32 roundings of at most 448 codes.
    back, s = codes.double() * scale.double()[..., None], scale.double()[..., None]
    half = s * 0.5 if store == "int8" else torch.maximum(x64.abs() * 2.0 ** -4, s * 2.0 ** -10)
    assert ((back - x64).abs() <= half * (1 + 2.0 ** -20) + s * QMAX[store] * 3 * 2.0 ** -24).all()


@pytest.mark.parametrize("layout", ["kv_first", "blocks_first", "token_major", "heads_first"])
@pytest.mark.parametrize("store, dtype", [("e4m3", "bf16"), ("int8", "fp16"), ("e4m3", "fp32"), ("int8", "fp32"),
                                          ("bf16", "bf16"), ("fp16", "fp32")])
@pytest.mark.parametrize("n, heads, dim, page", [(1, 1, 128, 16), (37, 5, 80, 1), (129, 3, 64, 24), (300, 8, 128, 16),
                                                 (7, 2, 256, 32), (9, 3, 20, 4), (5, 2, 1, 3)])
def test_write(cuda, store, dtype, n, heads, dim, page, layout):
    torch = cuda
    from pegaflow_b200 import kv_write

    blocks = -(-n // page) + 3
    cache, k, v, ks, vs = make_cache(torch, store, blocks, page, heads, dim, layout, fill=1)
    before = [x.clone() for x in (k, v, ks, vs) if x is not None]
    g = torch.Generator(device="cuda").manual_seed(n * dim)
    # K and V as slices of one projection; row strengths over many powers of two.
    kv = torch.randn((n, 2, heads, dim), generator=g, device="cuda")
    kv *= torch.exp2(torch.randint(-12, 5, (n, 2, heads, 1), generator=g, device="cuda").float())
    kv = kv.to(types(torch)[dtype])
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:n]
    slots[::5] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv_write(cache, kv[:, 0], kv[:, 1], slots, status=status)
    assert status.item() == 0
    on = slots >= 0
    b, o = slots[on] // page, slots[on] % page
    for i, (view, s) in enumerate(((k, ks), (v, vs))):
        check_row(torch, store, kv[:, i][on], view[b, o], s[b, o] if s is not None else None)
    # Everything else is as it was.
    for x, was in zip([x for x in (k, v, ks, vs) if x is not None], before):
        x[b, o] = 0 if x.dtype != torch.float8_e4m3fn else x[b, o]
        was[b, o] = x[b, o]
        assert torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x,
                           was.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else was)


@pytest.mark.parametrize("store", ["e4m3", "int8"])
def test_write_extremes(cuda, store):
    """Zeros, the smallest and largest values, NaN and infinities: a row with one of the last two reads back as NaN,
    others are not touched by it."""
    torch = cuda
    from pegaflow_b200 import kv_read, kv_write

    cache, k, v, ks, vs = make_cache(torch, store, 2, 16, 1, 64)
    x = torch.randn((8, 1, 64), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    x[0] = 0
    x[1] = 1e-45
    x[2] *= 1e-38
    x[3] = 3e38 * x[3].sign()
    x[4, 0, 5] = math.nan
    x[5, 0, 63] = math.inf
    x[6, 0, 0] = -math.inf
    slots = torch.arange(8, device="cuda")
    kv_write(cache, x, -x, slots)
    key, value = kv_read(cache, torch.zeros((1, 2), dtype=torch.int32, device="cuda"),
                         torch.tensor([0, 8], dtype=torch.int32, device="cuda"), 8, dtype=torch.float32)
    assert torch.isnan(key[4:7]).all() and torch.isnan(value[4:7]).all()
    for got, want in ((key, x), (value, -x)):
        good = [0, 1, 2, 3, 7]
        s = torch.clamp(want[good].double().abs().amax(2, keepdim=True) / QMAX[store], min=2.0 ** -126)
        half = s * 0.5 if store == "int8" else torch.maximum(want[good].double().abs() * 2.0 ** -4, s * 2.0 ** -10)
        tol = half * (1 + 2.0 ** -20) + s * QMAX[store] * 4 * 2.0 ** -24 + 2.0 ** -149
        assert ((got[good].double() - want[good].double()).abs() <= tol).all()
    assert (ks[0, 0, 0] == 2.0 ** -126) and (key[0] == 0).all()


def test_write_given_scales_and_bad_slots(cuda):
    torch = cuda
    from pegaflow_b200 import KVCache, kv_write
    from pegaflow_b200.kv import BAD_BLOCK

    k = torch.zeros((4, 16, 2, 64), dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    scale = torch.tensor([0.5, 0.25, 1.0, 2.0], device="cuda").view(4, 1, 1)  # one for each block
    cache = KVCache(k, v, scale, scale)
    x = torch.randn((6, 2, 64), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 100
    slots = torch.tensor([3, 17, 64, 50, 2 ** 62, -5], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv_write(cache, x, x, slots, given_scales=True, status=status)
    assert status.item() == BAD_BLOCK
    codes = k.view(torch.float8_e4m3fn).float()
    for t, slot in ((0, 3), (1, 17), (3, 50)):
        s = scale[slot // 16, 0, 0]
        want = (x[t] * (1.0 / s)).clamp(-448, 448).to(torch.float8_e4m3fn).float()  # saturates
        assert torch.equal(codes[slot // 16, slot % 16], want)
    assert (codes != 0).any(dim=3).any(dim=2).sum() == 3
    assert torch.equal(scale.flatten(), torch.tensor([0.5, 0.25, 1.0, 2.0], device="cuda"))


# -------------------------------------------------------------------- kv_read

@pytest.mark.parametrize("layout", ["kv_first", "blocks_first", "heads_first"])
@pytest.mark.parametrize("store, dtype", [("e4m3", "bf16"), ("int8", "fp16"), ("e4m3", "fp32"), ("bf16", "bf16"),
                                          ("fp16", "fp32"), ("int8", "bf16")])
@pytest.mark.parametrize("lens, heads, dim, page", [([1], 1, 128, 16), ([0, 33, 0, 7, 1], 5, 80, 16),
                                                    ([100, 3], 8, 128, 1), ([65, 64, 63], 3, 20, 24),
                                                    ([31], 2, 256, 64)])
def test_read(cuda, store, dtype, lens, heads, dim, page, layout):
    torch = cuda
    from pegaflow_b200 import kv_read

    need = [-(-n // page) for n in lens]
    blocks = sum(need) + 4
    cache, k, v, ks, vs = make_cache(torch, store, blocks, page, heads, dim, layout, fill=7)
    r = random.Random(dim)
    order = r.sample(range(blocks), blocks)
    table = torch.full((len(lens), max(need) + 2), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[sum(need[:s]):sum(need[:s]) + n], dtype=torch.int32)
    starts = torch.tensor([3 + sum(lens[:s]) for s in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    total = sum(lens) + 8
    t = types(torch)[dtype]
    # Strided outputs: the middle of wider rows.
    wide = torch.full((2, total, heads, dim + 16), 9.0, dtype=t, device="cuda")
    out = (wide[0, :, :, 8:8 + dim], wide[1, :, :, 8:8 + dim])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv_read(cache, table.cuda(), starts, out=out, status=status)
    assert status.item() == 0
    for got, view, s in ((out[0], k, ks), (out[1], v, vs)):
        x = view.float() if s is None else view.float() * s[..., None]  # one fp32 product, then one rounding
        at = 3
        for i, n in enumerate(lens):
            pos = torch.arange(n)
            want = x[table[i, pos // page].long().cuda(), (pos % page).cuda()].to(t)
            assert torch.equal(got[at:at + n], want)
            at += n
        assert (got[:3] == 9).all() and (got[at:] == 9).all()  # rows outside the sequences
    assert (wide[..., :8] == 9).all() and (wide[..., 8 + dim:] == 9).all()
    # New tensors take the same values.
    key, value = kv_read(cache, table.cuda(), starts, total, dtype=t)
    assert torch.equal(key[3:at], out[0][3:at]) and torch.equal(value[3:at], out[1][3:at])


def test_read_bad_blocks(cuda):
    torch = cuda
    from pegaflow_b200 import kv_read
    from pegaflow_b200.kv import BAD_BLOCK, BAD_LENGTH

    cache, k, v, ks, vs = make_cache(torch, "e4m3", 4, 8, 2, 64, fill=2)
    table = torch.tensor([[1, 4], [-1, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 12, 20], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    key, _ = kv_read(cache, table, starts, 20, dtype=torch.float32, status=status)
    assert status.item() == BAD_BLOCK
    assert torch.equal(key[:8], k[1].float() * ks[1][..., None]) and (key[8:] == 0).all()
    status.zero_()
    starts = torch.tensor([0, 17, 20], dtype=torch.int32, device="cuda")  # one past the two blocks of its row
    kv_read(cache, torch.tensor([[1, 2], [3, 0]], dtype=torch.int32, device="cuda"), starts, 20, status=status)
    assert status.item() == BAD_LENGTH


# ------------------------------------------------------------------ attention

def attend_plain(torch, q, k, v, lens, counts, table, page, scale, causal=True, window=0, bad=()):
    """The formula in 64 bits. k and v: [blocks, page, heads, dim] as values. Returns the output, the log-sums, and for
    the bounds the weighted magnitudes sum_j w_j |v_j| and the largest sum_d |q_d k_jd| of each row."""
    n_heads, dim = q.shape[1], q.shape[2]
    heads = k.shape[2]
    group = n_heads // heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    dot = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    at = 0
    for s, (n, length) in enumerate(zip(counts, lens)):
        if n and length > 0:
            pos = torch.arange(length, device=q.device)
            blk = table[s].to(q.device)[pos // page].long()
            keep = (blk >= 0) & (blk < k.shape[0])
            blk = blk.clamp(0, k.shape[0] - 1)
            kk, vv = k[blk, pos % page], v[blk, pos % page]  # [length, heads, dim]
            qq = q[at:at + n].double().view(n, heads, group, dim)
            p = torch.arange(n, device=q.device) + length - n
            seen = keep[None, :].expand(n, -1)
            if causal:
                seen = seen & (pos[None, :] <= p[:, None])
            if window:
                seen = seen & (pos[None, :] > p[:, None] - window)
            sc = torch.einsum("nhgd,lhd->nhgl", qq, kk) * scale
            sc = torch.where(seen[:, None, None, :], sc, -math.inf)
            ab = torch.einsum("nhgd,lhd->nhgl", qq.abs(), kk.abs()) * abs(scale)
            dot[at:at + n] = torch.where(seen[:, None, None, :], ab, 0.0).amax(3).view(n, n_heads)
            top = sc.amax(3, keepdim=True)
            w = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
            l = w.sum(3, keepdim=True)
            w = torch.where(l > 0, w / l, 0.0)
            # Tokens that no query sees take no part, whatever they hold.
            vs = torch.where(seen.any(0)[:, None, None], vv, 0.0)
            out[at:at + n] = torch.einsum("nhgl,lhd->nhgd", w, vs).reshape(n, n_heads, dim)
            mag[at:at + n] = torch.einsum("nhgl,lhd->nhgd", w, vs.abs()).reshape(n, n_heads, dim)
            lse[at:at + n] = (top + l.log()).view(n, n_heads)
        at += n
    return out, lse, mag, dot


def attend_bound(torch, dtype, quantised, out, mag, dot, longest, dim):
    """How far an output element may be: its own rounding (u of the output's type); the roundings to 16 bits in front
    of the second product, and the scores' error, both times sum_j w_j |v_j|. Those roundings: the weight's (u of the
    type; over an 8-bit cache fp16's, and for a bf16 output V's scale and V times it too, 2^-11 each). A score is a sum
    of dim products (exact) in fp32, an addition off by at most 2^-23 (accumulation may truncate), then two products:
    e = (dim + 4) 2^-23 max_j sum_d |q_d k_jd|. It moves a weight, and the sum it is divided by, by exp(e) each. The
    exponential is off by 2^-21, the sums of `longest` terms by 2^-23 an addition in tiles of 128 at most that are then
    added up."""
    u_out = torch.finfo(dtype).eps / 2
    u_p = torch.finfo(dtype).eps / 2 if not quantised else 2.0 ** -11 * (3 if dtype == torch.bfloat16 else 1)
    e = (dim + 4) * 2.0 ** -23 * dot[..., None]
    sums = (128 + longest / 128 + 64) * 2.0 ** -23
    return u_out * out.abs() + (u_p + 2 * torch.expm1(e) + 2 * sums + 2.0 ** -20) * mag * 1.01 + 1e-30, \
        e[..., 0] * 1.01 + sums + 2.0 ** -20


def run_attention(torch, q_type, store, dim, heads, group, page, counts, lens, layout="kv_first", window=0, causal=True,
                  scale=None, seed=0, spread=1.0, hints=True, table_pad=0, edit=None):
    from pegaflow_b200 import chunk_attention

    need = [max(0, -(-n // page)) for n in lens]
    blocks = sum(need) + 3
    cache, k, v, ks, vs = make_cache(torch, store, blocks, page, heads, dim, layout, fill=seed + 1)
    r = random.Random(seed)
    order = r.sample(range(blocks), blocks)
    table = torch.full((len(lens), max(need + [1]) + table_pad), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[sum(need[:s]):sum(need[:s]) + n], dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    n = sum(counts)
    t = types(torch)[q_type]
    q = (torch.randn((n, 2, heads * group, dim), generator=g, device="cuda") * spread).to(t)[:, 1]  # strided
    if edit:
        edit(k, v, ks, vs, table, q)
    q_start = torch.tensor([sum(counts[:s]) for s in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    sc = 1 / math.sqrt(dim) if scale is None else scale
    more = dict(max_q=max(counts), max_kv=max(lens)) if hints else {}
    o, lse = chunk_attention(q, cache, table.cuda(), q_start, kv_len, scale=scale, causal=causal, window=window,
                             return_lse=True, **more)
    want, wl, mag, dot = attend_plain(torch, q, dense(torch, k, ks), dense(torch, v, vs), lens, counts, table, page, sc,
                                      causal, window)
    return o, lse, want, wl, mag, dot, (cache, q, table, q_start, kv_len)


def check_attention(torch, got, dim, longest, quantised):
    o, lse, want, wl, mag, dot = got[:6]
    tol, tol_l = attend_bound(torch, o.dtype, quantised, want, mag, dot, longest, dim)
    off = (o.double() - want).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max().item():.2f} of the bound, {off.max().item():.3g}"
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse), empty) and (o[empty] == 0).all()
    off = torch.where(empty, 0.0, (lse.double() - wl).abs() - wl.abs() * 2.0 ** -23)
    assert (off <= tol_l).all(), f"lse {(off / tol_l).max().item():.2f} of the bound"


PATTERNS = {
    # name: (new tokens, cached tokens with them)
    "one": ([1], [1]),
    "decode": ([1, 1, 1, 1], [1000, 1, 129, 64]),
    "decode_long": ([1, 1], [9000, 4097]),
    "verify": ([3, 4, 1, 4], [300, 4, 777, 128]),
    "chunk": ([200], [713]),
    "prefill": ([300, 1, 77], [300, 1, 77]),
    "mixed": ([1, 150, 0, 17, 1], [2000, 400, 55, 17, 3]),
    "short": ([5, 9, 3], [0, 4, 2]),  # fewer cached tokens than queries: the first see nothing
}


@pytest.mark.parametrize("pattern", sorted(PATTERNS))
@pytest.mark.parametrize("q_type, store", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "int8"),
                                           ("bf16", "int8"), ("fp16", "e4m3")])
@pytest.mark.parametrize("dim, heads, group, page", [(128, 2, 4, 16), (64, 3, 1, 32), (80, 1, 5, 24), (128, 1, 16, 1),
                                                     (16, 2, 3, 7), (96, 2, 8, 128)])
def test_attention(cuda, pattern, q_type, store, dim, heads, group, page):
    torch = cuda
    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, q_type, store, dim, heads, group, page, counts, lens, seed=dim + page)
    check_attention(torch, got, dim, max(lens), store in QMAX)


@pytest.mark.parametrize("layout", ["blocks_first", "token_major", "heads_first"])
@pytest.mark.parametrize("store", ["bf16", "e4m3"])
@pytest.mark.parametrize("pattern", ["decode", "mixed"])
def test_attention_layouts(cuda, pattern, store, layout):
    torch = cuda
    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "bf16", store, 128, 2, 4, 16, counts, lens, layout=layout, seed=4, table_pad=5)
    check_attention(torch, got, 128, max(lens), store in QMAX)


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [2, 8, 32, 64, 256, 384, 100])
@pytest.mark.parametrize("dim", [16, 48, 80, 112, 128])
def test_attention_block_sizes(cuda, dim, page, store):
    """Blocks that are part of a tile of keys, a whole number of them or neither, heads of every width."""
    torch = cuda
    counts, lens = [70, 1, 33], [900, 300, 33]
    got = run_attention(torch, "bf16", store, dim, 2, 4, page, counts, lens, seed=dim + page)
    check_attention(torch, got, dim, max(lens), store in QMAX)


@pytest.mark.parametrize("heads, group", [(1, 128), (1, 40), (3, 17), (12, 1)])
@pytest.mark.parametrize("pattern", ["decode", "verify", "mixed"])
@pytest.mark.parametrize("store", ["fp16", "int8"])
def test_attention_groups(cuda, pattern, heads, group, store):
    torch = cuda
    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "fp16", store, 64, heads, group, 16, counts, lens, seed=group)
    check_attention(torch, got, 64, max(lens), store in QMAX)


@pytest.mark.parametrize("n_q", [1, 20])
def test_attention_many_sequences(cuda, n_q):
    """More sequences than some of a grid's axes have room for; each its own block."""
    torch = cuda
    from pegaflow_b200 import chunk_attention

    n, page, dim = 70_000 if n_q == 1 else 5_000, 32, 64
    cache, k, v, ks, vs = make_cache(torch, "bf16", n, page, 1, dim, fill=4)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((n * n_q, 1, dim), generator=g, device="cuda").bfloat16()
    lens = torch.randint(n_q, page + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(n, 1)
    starts = torch.arange(n + 1, device="cuda", dtype=torch.int32) * n_q
    o = chunk_attention(q, cache, order, starts, lens, max_q=n_q, max_kv=page)
    keys, values = k[order[:, 0].long(), :, 0].double(), v[order[:, 0].long(), :, 0].double()
    qq = q.view(n, n_q, dim).double()
    s = torch.einsum("nid,njd->nij", qq, keys) / math.sqrt(dim)
    pos = lens[:, None] - n_q + torch.arange(n_q, device="cuda")
    seen = torch.arange(page, device="cuda") <= pos[:, :, None]
    w = torch.where(seen, s, -math.inf).softmax(2)
    want, mag = torch.einsum("nij,njd->nid", w, values), torch.einsum("nij,njd->nid", w, values.abs())
    dot = torch.einsum("nid,njd->nij", qq.abs(), keys.abs()).amax(2) / math.sqrt(dim)
    tol, _ = attend_bound(torch, o.dtype, False, want, mag, dot, page, dim)
    assert ((o.view(n, n_q, dim).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("window", [1, 2, 100, 129, 5000])
@pytest.mark.parametrize("pattern", ["decode_long", "verify", "mixed", "prefill", "short"])
@pytest.mark.parametrize("store", ["fp16", "int8"])
def test_attention_windows(cuda, pattern, window, store):
    torch = cuda
    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "fp16", store, 64, 2, 4, 16, counts, lens, window=window, seed=window)
    check_attention(torch, got, 64, max(lens), store in QMAX)


@pytest.mark.parametrize("pattern", ["decode", "mixed", "short"])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_not_causal(cuda, pattern, window):
    torch = cuda
    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "bf16", "bf16", 128, 2, 4, 16, counts, lens, causal=False, window=window, seed=9)
    check_attention(torch, got, 128, max(lens), False)


@pytest.mark.parametrize("spread, scale", [(30.0, None), (1.0, 0.0), (1.0, -0.5), (0.001, None)])
@pytest.mark.parametrize("pattern", ["decode", "chunk"])
def test_attention_score_ranges(cuda, pattern, spread, scale):
    """Scores of hundreds (weights of one token, maxima that keep rising), of zero, negated."""
    torch = cuda
    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "bf16", "bf16", 128, 2, 4, 16, counts, lens, spread=spread, scale=scale, seed=12)
    check_attention(torch, got, 128, max(lens), False)


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
@pytest.mark.parametrize("pattern", ["decode", "mixed", "prefill"])
def test_attention_rising_scores(cuda, pattern, store):
    """Keys that grow along the sequence: every tile raises the maximum by far."""
    torch = cuda
    counts, lens = PATTERNS[pattern]

    def edit(k, v, ks, vs, table, q):
        q.copy_(q.abs())
        for s in range(table.shape[0]):
            for i, b in enumerate(table[s].tolist()):
                if b < 0:
                    continue
                k[b] = k[b].float().abs().to(k.dtype)
                if ks is not None:
                    ks[b] *= 0.02 * i
                else:
                    k[b] *= 0.02 * i

    got = run_attention(torch, "bf16", store, 128, 2, 4, 16, counts, lens, seed=13, edit=edit)
    check_attention(torch, got, 128, max(lens), store in QMAX)


@pytest.mark.parametrize("store", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("pattern", ["decode", "prefill", "mixed"])
def test_attention_ignores_what_is_masked(cuda, pattern, bad, store):
    """Whatever the cache holds behind a sequence's end, in other blocks, in front of the window or at tokens that a
    query does not see, its row does not change: NaN and infinities at the chunk's last token reach that token alone."""
    torch = cuda
    counts, lens = PATTERNS[pattern]
    q_type = "fp16" if store == "fp16" else "bf16"
    page, clean = 16, {}

    def plant(edit_last):
        def edit(k, v, ks, vs, table, q):
            used = {(int(table[s, j // page]), j % page) for s, n in enumerate(lens) for j in range(n)}
            last = {(int(table[s, (n - 1) // page]), (n - 1) % page) for s, n in enumerate(lens)}
            for b in range(k.shape[0]):
                for o in range(page):
                    if (b, o) not in used or (edit_last and (b, o) in last):
                        for x, s in ((k, ks), (v, vs)):
                            if s is not None:
                                s[b, o] = bad
                            else:
                                x[b, o] = bad
        return edit

    kw = dict(seed=21)
    clean = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, **kw)
    dirty = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, edit=plant(False), **kw)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    check_attention(torch, clean, 128, max(lens), store in QMAX)
    o, lse = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, edit=plant(True), **kw)[:2]
    at = 0
    for n in counts:
        if n > 1:  # all but the chunk's last query
            rows = slice(at, at + n - 1)
            tol, tol_l = attend_bound(torch, o.dtype, store in QMAX, clean[2][rows], clean[4][rows], clean[5][rows],
                                      max(lens), 128)
            assert ((o[rows].double() - clean[2][rows]).abs() <= tol).all()
            assert ((lse[rows].double() - clean[3][rows]).abs() <= tol_l + clean[3][rows].abs() * 2.0 ** -23).all()
        at += n


@pytest.mark.parametrize("q_type, store", [("bf16", "e4m3"), ("fp16", "int8"), ("fp16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("pattern", ["verify", "chunk", "prefill", "mixed"])
@pytest.mark.parametrize("window", [0, 70])
def test_attention_ignores_masked_scales(cuda, pattern, q_type, store, window):
    """A V scale 2^60 times the others', at the chunk's last token and (with a window) in front of it: rows that do not
    see it are as exact as without."""
    torch = cuda
    counts, lens = PATTERNS[pattern]
    page, kw = 16, dict(seed=23, window=window)

    def edit(k, v, ks, vs, table, q):
        for s, (n, length) in enumerate(zip(counts, lens)):
            at = {length - 1} | ({max(0, length - n - 69)} if window and n > 1 else set())
            for j in at:
                vs[int(table[s, j // page]), j % page] *= 2.0 ** 60

    clean = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, **kw)
    o, lse = run_attention(torch, q_type, store, 128, 2, 4, page, counts, lens, edit=edit, **kw)[:2]
    tol, tol_l = attend_bound(torch, o.dtype, True, clean[2], clean[4], clean[5], max(lens), 128)
    at = 0
    for n, length in zip(counts, lens):
        # With a window the planted token is the first that query 0 sees: it alone, of those in front of the last.
        rows = slice(at + (1 if window and length - n - 69 >= 0 else 0), at + n - 1)
        if not window or length - n - 69 >= 0:
            assert ((o[rows].double() - clean[2][rows]).abs() <= tol[rows]).all()
            assert ((lse[rows].double() - clean[3][rows]).abs() <= tol_l[rows] + clean[3][rows].abs() * 2.0 ** -23).all()
        at += n


@pytest.mark.parametrize("q_type, store", [("bf16", "e4m3"), ("fp16", "int8")])
@pytest.mark.parametrize("pattern", ["decode", "decode_long", "verify"])
def test_attention_scales_of_any_size(cuda, pattern, q_type, store):
    """V scales over a hundred powers of two: what is far below a row's largest is off by half of fp16's smallest step
    of that, 2^-25, for each code."""
    torch = cuda
    counts, lens = PATTERNS[pattern]

    def edit(k, v, ks, vs, table, q):
        g = torch.Generator(device="cuda").manual_seed(3)
        vs *= torch.exp2(torch.randint(-60, 41, vs.shape, generator=g, device="cuda").float())

    o, lse, want, wl, mag, dot, (cache, q, table, q_start, kv_len) = run_attention(
        torch, q_type, store, 128, 2, 4, 16, counts, lens, seed=29, edit=edit)
    tol, tol_l = attend_bound(torch, o.dtype, True, want, mag, dot, max(lens), 128)
    # The largest weight times scale is at most 2^9 of the unit that the steps are of, and at least 1; a row's largest
    # magnitude has a code of 448 or 127 (a cache row's largest) next to it.
    tol = tol + max(lens) * 2.0 ** -25 * mag.amax(2, keepdim=True) * 4
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half of its smallest step
    big = torch.finfo(o.dtype).max
    on = want.abs() < big
    assert ((o.double() - want).abs()[on] <= tol[on]).all()
    assert ((lse.double() - wl).abs() <= tol_l + wl.abs() * 2.0 ** -23).all()


def test_attention_waits_for_rows_made_again(cuda):
    """A NaN that only the last query sees, after a long context: the rows beside it are made again token by token,
    which takes longer than a wait's limit, and the call neither gives up nor changes them."""
    torch = cuda
    from pegaflow_b200 import KVCache, chunk_attention

    heads, group, dim, page, n, length = 8, 4, 128, 16, 2048, 34816
    g = torch.Generator(device="cuda").manual_seed(31)
    buf = torch.randn((2, length // page, page, heads, dim), generator=g, device="cuda").half()
    cache = KVCache(buf[0], buf[1])
    table = torch.randperm(length // page, generator=g, device="cuda").int()[None]
    q = torch.randn((n, heads * group, dim), generator=g, device="cuda").half()
    args = (q, cache, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
            torch.tensor([length], dtype=torch.int32, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    clean = chunk_attention(*args, status=status)
    buf[1, table[0, -1].long(), -1] = math.nan
    dirty = chunk_attention(*args, status=status)
    assert status.item() == 0
    assert torch.isnan(dirty[-1]).all()
    # Both are within the bound of the formula: u |o| and, for weights in fp16, u times the mean magnitude, at most the
    # largest value there is.
    u = 2.0 ** -11
    off = (dirty[:-1].double() - clean[:-1].double()).abs()
    assert (off <= 2 * (u * clean[:-1].double().abs() + u * 6.5 + 2.0 ** -12)).all()


def test_attention_nan_query(cuda):
    """A NaN in one query reaches its own row alone."""
    torch = cuda
    counts, lens = PATTERNS["mixed"]
    clean = run_attention(torch, "bf16", "bf16", 128, 2, 4, 16, counts, lens, seed=2)

    def edit(k, v, ks, vs, table, q):
        q[40, 3, 7] = math.nan

    o = run_attention(torch, "bf16", "bf16", 128, 2, 4, 16, counts, lens, seed=2, edit=edit)[0]
    assert torch.isnan(o[40, 3]).all()
    o[40, 3] = clean[0][40, 3]
    assert torch.equal(o, clean[0])


@pytest.mark.parametrize("pattern", ["decode", "decode_long", "mixed"])
@pytest.mark.parametrize("store", ["bf16", "int8"])
def test_attention_without_hints(cuda, pattern, store):
    """No hints, wrong hints and wide tables change the split, never the result beyond its bound."""
    torch = cuda
    from pegaflow_b200 import chunk_attention

    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "bf16", store, 128, 2, 4, 16, counts, lens, hints=False, seed=6, table_pad=300)
    check_attention(torch, got, 128, max(lens), store in QMAX)
    cache, q, table, q_start, kv_len = got[6]
    for more in (dict(max_q=1, max_kv=1), dict(max_q=7, max_kv=200), dict(max_q=4096), dict(max_kv=100000)):
        o, lse = chunk_attention(q, cache, table.cuda(), q_start, kv_len, return_lse=True, **more)
        check_attention(torch, (o, lse) + got[2:6], 128, max(lens), store in QMAX)


@pytest.mark.parametrize("pattern", ["decode", "mixed"])
def test_attention_bad_blocks_and_lengths(cuda, pattern):
    torch = cuda
    from pegaflow_b200 import chunk_attention
    from pegaflow_b200.kv import BAD_BLOCK, BAD_LENGTH

    counts, lens = PATTERNS[pattern]

    def edit(k, v, ks, vs, table, q):
        table[0, 3], table[0, 10], table[0, 40] = -7, k.shape[0], 2 ** 31 - 1

    got = run_attention(torch, "bf16", "bf16", 128, 2, 4, 16, counts, lens, seed=8, edit=edit)
    check_attention(torch, got, 128, max(lens), False)
    cache, q, table, q_start, kv_len = got[6]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    chunk_attention(q, cache, table.cuda(), q_start, kv_len, status=status)
    assert status.item() == BAD_BLOCK
    status.zero_()
    # A length that its table row does not hold: the tokens that it holds are seen.
    table[0, 3], table[0, 10], table[0, 40] = 0, 0, 0
    kv_len[0] = table.shape[1] * 16 + 5
    chunk_attention(q, cache, table.cuda(), q_start, kv_len, status=status)
    assert status.item() & BAD_LENGTH


@pytest.mark.parametrize("pattern", ["decode", "mixed"])
def test_attention_leaves_other_rows(cuda, pattern):
    """Rows behind the last sequence and in front of the first, and what lies between strided rows, stay."""
    torch = cuda
    from pegaflow_b200 import chunk_attention

    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "bf16", "bf16", 128, 2, 4, 16, counts, lens, seed=3)
    cache, q, table, q_start, kv_len = got[6]
    n = q.shape[0]
    wide_q = torch.zeros((n + 9, 8, 128), dtype=q.dtype, device="cuda")
    wide_q[4:4 + n] = q
    room = torch.full((n + 9, 8, 2, 128), 5.0, dtype=q.dtype, device="cuda")
    out = room[:, :, 0]
    chunk_attention(wide_q, cache, table.cuda(), q_start + 4, kv_len, out=out, max_q=max(counts), max_kv=max(lens))
    assert torch.equal(out[4:4 + n], got[0])
    assert (out[:4] == 5).all() and (out[4 + n:] == 5).all() and (room[:, :, 1] == 5).all()


@pytest.mark.parametrize("pattern", ["decode", "decode_long", "mixed", "chunk"])
def test_attention_repeats(cuda, pattern):
    """The same call gives the same bits, alone and with another call on another stream beside it."""
    torch = cuda
    from pegaflow_b200 import chunk_attention

    counts, lens = PATTERNS[pattern]
    got = run_attention(torch, "bf16", "e4m3", 128, 2, 4, 16, counts, lens, seed=5)
    cache, q, table, q_start, kv_len = got[6]
    table = table.cuda()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        o, lse = chunk_attention(q, cache, table, q_start, kv_len, return_lse=True, max_q=max(counts), max_kv=max(lens))
        o2, lse2 = chunk_attention(q, cache, table, q_start, kv_len, return_lse=True, max_q=max(counts),
                                   max_kv=max(lens), stream=other.cuda_stream)
        other.synchronize()
        for a, b in ((o, got[0]), (o2, got[0]), (lse, got[1]), (lse2, got[1])):
            assert torch.equal(a, b)


def test_attention_far_offsets(cuda):
    """A cache whose block offsets pass 32 bits, in elements and in bytes: 2.4 GiB a side of codes."""
    torch = cuda
    from pegaflow_b200 import KVCache, chunk_attention, kv_read, kv_write

    page, heads, dim, blocks = 16, 8, 128, 300_000  # 4.9 billion codes a side
    t = torch.empty((2, blocks, page, heads, dim), dtype=torch.uint8, device="cuda")
    s = torch.empty((2, blocks, page, heads), device="cuda")
    cache = KVCache.from_tensor(t, s)
    n = 40
    ids = torch.tensor([blocks - 1, 150_000, blocks - 2], device="cuda")
    pos = torch.arange(n, device="cuda")
    slots = ids[pos // page] * page + pos % page
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((n, 2, heads, dim), generator=g, device="cuda", dtype=torch.float32).bfloat16()
    kv_write(cache, x[:, 0], x[:, 1], slots)
    table = ids.to(torch.int32).view(1, 3)
    k, v = kv_read(cache, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, dtype=torch.float32)
    for got, want in ((k, x[:, 0]), (v, x[:, 1])):
        s = want.double().abs().amax(2, keepdim=True) / 448
        tol = torch.maximum(want.double().abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20) + s * 448 * 4 * 2.0 ** -24
        assert ((got.double() - want.double()).abs() <= tol).all()
    for n_q in (1, 30):
        q = torch.randn((n_q, 32, dim), generator=g, device="cuda").bfloat16()
        o, lse = chunk_attention(q, cache, table, torch.tensor([0, n_q], dtype=torch.int32, device="cuda"),
                                 torch.tensor([n], dtype=torch.int32, device="cuda"), return_lse=True, max_q=n_q)
        local = torch.arange(3).view(1, 3)
        kk, vv = (torch.zeros((3, page, heads, dim), dtype=torch.float64, device="cuda") for _ in range(2))
        kk.view(-1, heads, dim)[:n], vv.view(-1, heads, dim)[:n] = k.double(), v.double()
        plain = attend_plain(torch, q, kk, vv, [n], [n_q], local, page, 1 / math.sqrt(dim))
        check_attention(torch, (o, lse) + plain, dim, n, True)


# ------------------------------------------------------------------- together

@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_write_save_load_attend(cuda, store):
    """A prompt's K and V are written, its blocks saved to the host pool and loaded into other blocks, and a chunk and
    then single tokens attend over them: what a restored prefix is for."""
    torch = cuda
    import numpy as np

    from pegaflow_b200 import Executor, KVCache, Layout, LoadSpec, PinnedBuffer, SaveSpec, chunk_attention, kv_write

    blocks, page, heads, dim, group = 64, 16, 4, 128, 4
    prefix, chunk = 400, 50
    t = torch.zeros((2, blocks, page, heads, dim), dtype=types(torch)[store], device="cuda")
    parts = [t]
    if store in QMAX:
        parts.append(torch.zeros((2, blocks, page, heads), device="cuda"))
    cache = KVCache.from_tensor(*parts)
    g = torch.Generator(device="cuda").manual_seed(11)
    total = prefix + chunk + 3
    kv = torch.randn((total, 2, heads, dim), generator=g, device="cuda").bfloat16()
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(1))
    src, dst = ids[:25], ids[25:54]  # 400 tokens; 29 blocks hold all
    pos = torch.arange(total)

    def slots(blk, lo, hi):
        p = pos[lo:hi]
        return (blk[p // page] * page + p % page).cuda()

    kv_write(cache, kv[:prefix, 0], kv[:prefix, 1], slots(src, 0, prefix))
    ex, pools, loads = Executor(0), [], []
    torch.cuda.synchronize()
    for x in parts:
        lay = Layout.from_tensor(x)
        pool = PinnedBuffer(2 * 25 * lay.bytes_per_block)
        ex.save([SaveSpec(lay, src.numpy(), pool.ptr, pool.ptr + 25 * lay.bytes_per_block)])
        ks = np.arange(25, dtype=np.uint64) * lay.bytes_per_block + pool.ptr
        loads.append(LoadSpec(lay, dst[:25].numpy(), ks, ks + 25 * lay.bytes_per_block))
        pools.append(pool)
    for x in parts:
        x[:, src.cuda()] = 0  # the prefix is evicted
    torch.cuda.synchronize()
    ex.load(loads)
    table = dst.to(torch.int32).view(1, -1)
    done = prefix
    for n in (chunk, 1, 1, 1):
        kv_write(cache, kv[done:done + n, 0], kv[done:done + n, 1], slots(dst, done, done + n))
        done += n
        q = torch.randn((n, heads * group, dim), generator=g, device="cuda").bfloat16()
        o, lse = chunk_attention(q, cache, table.cuda(), torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                 torch.tensor([done], dtype=torch.int32, device="cuda"), return_lse=True)
        plain = attend_plain(torch, q, dense(torch, cache.key, cache.key_scale),
                             dense(torch, cache.value, cache.value_scale), [done], [n], table, page, 1 / math.sqrt(dim))
        check_attention(torch, (o, lse) + plain, dim, done, store in QMAX)
        # And what the cache holds is what was written, as near as its type.
        exact = attend_plain(torch, q, kv[:done, 0].double().view(1, done, heads, dim),
                             kv[:done, 1].double().view(1, done, heads, dim), [done], [n],
                             torch.zeros((1, 1), dtype=torch.int32), done, 1 / math.sqrt(dim))
        if store == "bf16":
            check_attention(torch, (o, lse) + exact, dim, done, False)


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
def test_captured_steps(cuda, store):
    """A decode step (write, read, attend) captured once and replayed over growing sequences, and a second graph of a
    chunk between its replays."""
    torch = cuda
    from pegaflow_b200 import chunk_attention, kv_read, kv_write

    blocks, page, heads, dim, group = 40, 16, 2, 128, 4
    cache, k, v, ks, vs = make_cache(torch, store, blocks, page, heads, dim, fill=3)
    table = torch.arange(blocks, dtype=torch.int32).view(2, 20)
    dev = table.cuda()
    lens = torch.tensor([100, 7], dtype=torch.int32, device="cuda")
    x = torch.zeros((2, 2, heads, dim), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((2, heads * group, dim), dtype=torch.bfloat16, device="cuda")
    qc = torch.zeros((64, heads * group, dim), dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    one, many = (torch.tensor(s, dtype=torch.int32, device="cuda") for s in ([0, 1, 2], [0, 40, 64]))

    def step():
        kv_write(cache, x[:, 0], x[:, 1], slots)
        return chunk_attention(q, cache, dev, one, lens, max_q=1, return_lse=True)

    def chunk():
        return chunk_attention(qc, cache, dev, many, lens, max_q=40, return_lse=True), \
            kv_read(cache, dev, many, 64, dtype=torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), chunk()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = step()
    with torch.cuda.graph(g2):
        out2, read = chunk()
    g = torch.Generator(device="cuda").manual_seed(4)
    for i in range(4):
        lens += 1
        at = lens.long() - 1
        slots.copy_(dev[torch.arange(2, device="cuda"), at // page].long() * page + at % page)
        for t in (x, q, qc):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        g1.replay()
        g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        values = dense(torch, k, ks), dense(torch, v, vs)
        for out, query, counts in ((out1, q, [1, 1]), (out2, qc, [40, 24])):
            plain = attend_plain(torch, query, *values, lens.tolist(), counts, table, page, 1 / math.sqrt(dim))
            check_attention(torch, tuple(out) + plain, dim, 128, store in QMAX)
        pos = torch.arange(40, device="cuda")
        assert torch.equal(read[0][:40].double(), values[0][dev[0, pos // page].long(), pos % page].float().double())


def test_other_device_current(cuda):
    """Tensors of device 0 while device 1 is the current one."""
    torch = cuda
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    counts, lens = PATTERNS["mixed"]
    got = run_attention(torch, "bf16", "e4m3", 128, 2, 4, 16, counts, lens, seed=5)
    from pegaflow_b200 import chunk_attention

    cache, q, table, q_start, kv_len = got[6]
    table = table.cuda()
    with torch.cuda.device(1):
        o = chunk_attention(q, cache, table, q_start, kv_len)
        assert torch.cuda.current_device() == 1
    torch.cuda.synchronize(0)
    assert torch.equal(o, chunk_attention(q, cache, table, q_start, kv_len))

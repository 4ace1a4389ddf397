"""The 8-bit key/value cache on the GPU against its definition in 64 bits (kv8_ref): appending, reading back, attention of the
newest tokens, selecting blocks, and all of them together as a serving loop uses them."""
import numpy as np
import pytest
import torch

import cuda_ltc_b200 as ltc
from kv8_ref import VALUES, Cache, decode_tolerances, encode
from util import bf16_round, randn

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def device_cache(ref: Cache, layout="bhsd", bounds=True):
    """The reference's cache on the GPU; layout bshd: heads inside tokens, with a gap behind each token."""
    B, H, S, D = ref.k.shape

    def codes(c):
        t = torch.from_numpy(c).cuda()
        if layout == "bshd":
            t = torch.nn.functional.pad(t.transpose(1, 2), (0, 0, 0, 1)).contiguous()[:, :, :H].transpose(1, 2)
        return t.view(torch.float8_e4m3fn)
    f32 = lambda s: torch.from_numpy(s.astype(np.float32)).cuda()  # noqa: E731
    return ltc.Kv8Cache(codes(ref.k), codes(ref.v), f32(ref.ks), f32(ref.vs),
                        torch.from_numpy(ref.bounds.copy()).cuda() if bounds else None, ref.block)


def ints(x):
    return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def same_codes(got, want):
    """Equal as values: NaN is NaN whatever its sign, and zero is zero."""
    a, b = VALUES[got.view(torch.uint8).cpu().numpy()], VALUES[want]
    return np.array_equal(a, b, equal_nan=True)


def check_cache(cache, ref, bounds=True):
    for name, got, want in (("k", cache.k, ref.k), ("v", cache.v, ref.v)):
        assert same_codes(got, want), name
    assert np.array_equal(cache.k_scale.cpu().numpy(), ref.ks) and np.array_equal(cache.v_scale.cpu().numpy(), ref.vs)
    if bounds:
        assert np.array_equal(cache.bounds.cpu().numpy(), ref.bounds)


def filled(B, H, S, D, block, seed, spread=4.0):
    """A cache in use: every block written at its own size, nothing of it special."""
    ref = Cache.empty(B, H, S, D, block)
    r = np.random.default_rng(seed)
    for x, codes, scale in ((0, ref.k, ref.ks), (1, ref.v, ref.vs)):
        codes[:] = encode(r.standard_normal((B, H, S, D)) * 60)
        scale[:] = 2.0 ** np.floor(r.uniform(-6 - spread / 2, -6 + spread / 2, scale.shape))
    for j in range(ref.ks.shape[2]):
        live = VALUES[ref.k[:, :, j * block:(j + 1) * block]]
        ref.bounds[:, :, j, 0], ref.bounds[:, :, j, 1] = np.floor(live.min(2) / 4), np.ceil(live.max(2) / 4)
    return ref


# ---- append ------------------------------------------------------------------------------------
APPENDS = [
    # B, H, S, D, block, n, kv_len, new_len
    (1, 1, 64, 32, 16, 1, [1], None),                              # the first token
    (3, 2, 200, 64, 64, 1, [65, 128, 200], None),                  # a new block, a full one, the last place
    (2, 4, 333, 128, 32, 333, [333, 333], None),                   # a whole odd cache
    (4, 2, 300, 64, 128, 130, [130, 257, 131, 300], None),         # from 0, 127, 1, 170
    (5, 3, 150, 32, 16, 40, [40, 57, 7, 0, 150], [40, 17, 7, 0, 33]),
    (2, 2, 100, 64, 32, 20, [10, 115], None),                      # positions before the cache and behind it
    (3, 1, 64, 128, 64, 5, [-3, 2000000000, 69], [5, 5, 9]),       # nowhere at all; more than there are
    (2, 1, 1000, 64, 64, 17, [500, 17], [-2, 3]),
    (1, 2, 4100, 128, 16, 4099, [4100], None),
    (2, 2, 130, 128, 128, 3, [128, 130], None),
]


@pytest.mark.parametrize("layout", ["bhsd", "bshd", "odd"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "x".join(map(str, c[:6])))
def test_append(ctx, case, dtype, layout):
    B, H, S, D, block, n, kv_len, new_len = case
    ref = filled(B, H, S, D, block, 1)
    cache = device_cache(ref, "bhsd" if layout == "odd" else layout)
    # sizes around the scales that are there: some blocks grow, some keep theirs
    k, v = (bf16_round(randn((B, H, n, D), 5 + i) * 2.0 ** np.random.default_rng(7 + i).integers(-3, 4, (B, H, n, 1)))
            for i in range(2))
    tk, tv = (torch.from_numpy(x).cuda().to(DT[dtype]) for x in (k, v))
    if layout == "bshd":
        tk, tv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (tk, tv))
    if layout == "odd":                                             # rows that start on any element
        tk, tv = (torch.nn.functional.pad(t, (1, 2)).contiguous()[..., 1:1 + D] for t in (tk, tv))
    ref.append(k, v, kv_len, new_len)
    for _ in range(2):                                              # the same tokens again change nothing
        ctx.kv8_append(cache, tk, tv, ints(kv_len), new_len=ints(new_len))
        check_cache(cache, ref)


@pytest.mark.parametrize("block", [16, 64, 128])
def test_append_token_by_token(ctx, block):
    """Scales that grow under tokens which were written before, by one power and by many, over several blocks."""
    B, H, S, D = 2, 3, 150, 64
    ref = Cache.empty(B, H, S, D, block, fill=0x7f)                 # (NaN everywhere: nothing of it may count)
    cache = device_cache(ref)
    r = np.random.default_rng(3)
    for t in range(S):
        size = 2.0 ** r.choice([-8.0, -2.0, 0.0, 0.0, 1.0, 3.0], (B, H, 1, 1))
        k, v = (bf16_round(r.standard_normal((B, H, 1, D)) * size) for _ in range(2))
        ref.append(k, v, [t + 1] * B)
        ctx.kv8_append(cache, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints([t + 1] * B))
    check_cache(cache, ref)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_of_special_values(ctx, dtype):
    B, H, S, D, block = 1, 6, 64, 64, 32
    ref = Cache.empty(B, H, S, D, block, fill=0xff)
    cache = device_cache(ref)
    x = bf16_round(randn((B, H, 40, D), 1))
    x[0, 0, 3, 5], x[0, 0, 3, 6], x[0, 0, 9, 7] = np.inf, -np.inf, np.nan
    x[0, 1] = 0.0
    x[0, 1, :, 0] = -0.0
    x[0, 2] = bf16_round(x[0, 2] * np.float32(1e38))
    x[0, 3] = bf16_round(x[0, 3] * np.float32(1e-36))               # below the smallest scale's range: subnormal codes
    x[0, 4] = np.nan
    x[0, 5] = bf16_round(np.float32(2.0 ** -133) * np.round(x[0, 5] * 4))
    for i, length in ((slice(0, 20), 20), (slice(20, 40), 40)):
        ref.append(x[:, :, i], -x[:, :, i], [length])
        ctx.kv8_append(cache, torch.from_numpy(x[:, :, i]).cuda().to(DT[dtype]), -torch.from_numpy(x[:, :, i]).cuda().to(DT[dtype]),
                       ints([length]))
        check_cache(cache, ref)
    got, _ = ctx.kv8_read(cache, dtype=torch.float32, count=40)
    assert torch.isnan(got[0, 4]).all()
    # what the codes stand for, as far as fp32 goes: an infinity has become 448 * 2^120, which is above 2^128
    with np.errstate(over="ignore"):
        assert np.array_equal(got.cpu().numpy(), ref.values()[0][:, :, :40].astype(np.float32), equal_nan=True)


def test_append_without_bounds_and_at_the_largest_magnitudes(ctx):
    """448 * 2^e fits the scale 2^e, the next number above it does not."""
    for top, e in ((448.0, 0), (np.nextafter(np.float32(448), np.float32(1000)), 1), (1.75, -8), (1.7500001, -7)):
        ref = Cache.empty(1, 1, 16, 32, 16)
        cache = device_cache(ref, bounds=False)
        x = np.zeros((1, 1, 1, 32), np.float32)
        x[0, 0, 0, 31] = -top
        ref.append(x, x, [1])
        ctx.kv8_append(cache, torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda(), ints([1]))
        check_cache(cache, ref, bounds=False)
        assert cache.k_scale.item() == 2.0 ** e


# ---- read --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", [
    # B, H, S, D, block, start, count, kv_len, layout
    (2, 3, 100, 64, 32, 0, None, None, "bhsd"), (3, 2, 257, 128, 64, 3, 250, [0, 1, 257], "bshd"),
    (1, 1, 1, 32, 16, 0, 1, [1], "bhsd"), (2, 2, 1000, 32, 128, 999, 1, [1000, 999], "bhsd"),
    (2, 1, 300, 64, 16, 17, 129, [-5, 2000000000], "bshd"), (1, 2, 5000, 128, 16, 1, 4999, [4097], "bhsd"),
    (1, 2, 64, 128, 64, 64, 0, None, "bhsd")], ids=lambda c: "x".join(map(str, c[:7])))
def test_read(ctx, case, dtype):
    B, H, S, D, block, start, count, kv_len, layout = case
    ref = filled(B, H, S, D, block, 2, spread=30.0)
    ref.k[0, 0, S // 2, 3] = 0x7f
    cache = device_cache(ref, layout)
    n = S - start if count is None else count
    live = np.arange(start, start + n)[None] < np.asarray(kv_len if kv_len is not None else [S] * B)[:, None]
    want = [np.where(live[:, None, :, None], x[:, :, start:start + n], 0.0) for x in ref.values()]
    got = ctx.kv8_read(cache, kv_len=ints(kv_len), start=start, count=count, dtype=DT[dtype])
    out = [torch.full((B, n + 2, H, D + 3), 7.0, device="cuda", dtype=DT[dtype]) for _ in range(2)]      # odd rows, a border
    views = [o[:, 1:n + 1, :, 1:D + 1].transpose(1, 2) for o in out]
    ctx.kv8_read(cache, kv_len=ints(kv_len), start=start, count=n, dtype=DT[dtype], out_k=views[0], out_v=views[1])
    for g, w, x, o in zip(got, want, views, out):
        assert g.dtype == DT[dtype] and np.array_equal(g.double().cpu().numpy(), w, equal_nan=True)
        assert np.array_equal(x.double().cpu().numpy(), w, equal_nan=True)
        x.zero_()
        assert o.double().sum().item() == 7.0 * (o.numel() - x.numel())


# ---- decode ------------------------------------------------------------------------------------
def check_decode(ctx, ref, cache, q, dtype, **kw):
    o, lse = ctx.kv8_decode(q, cache, **{k: ints(v) if k in ("kv_len", "new_len", "blocks") else
                                         torch.from_numpy(v).cuda() if k == "keep_mask" else v for k, v in kw.items()})
    names = dict(score_clamp="clamp")
    o_ref, lse_ref, *rest = ref.decode(q.double().cpu().numpy(), **{names.get(k, k): v for k, v in kw.items()})
    to, tl = decode_tolerances(o_ref, lse_ref, *rest, dtype == "bf16")
    err = np.abs(o.double().cpu().numpy() - o_ref)
    assert o.dtype == DT[dtype] and (err <= to).all(), (np.nanmax(err), np.nanmax(err / to))
    got = lse.double().cpu().numpy()
    fin = np.isfinite(lse_ref)
    assert np.array_equal(got[~fin], lse_ref[~fin])
    assert (np.abs(got[fin] - lse_ref[fin]) <= tl[fin]).all(), np.abs(got[fin] - lse_ref[fin]).max()
    return o, lse


DECODES = [
    # B, H, G, Sq, S, D, block, kv_len, layout
    (1, 1, 1, 1, 1, 32, 16, [1], "bhsd"),
    (3, 2, 1, 1, 100, 64, 32, [0, 1, 100], "bhsd"),
    (4, 2, 4, 1, 333, 128, 64, [17, 64, 65, 333], "bshd"),
    (2, 3, 3, 1, 1000, 64, 16, [999, 16], "bhsd"),
    (2, 2, 8, 2, 700, 128, 128, [700, 1], "bshd"),          # a sequence shorter than its queries
    (1, 2, 7, 5, 515, 64, 64, [515], "bhsd"),               # 35 rows
    (1, 1, 16, 4, 260, 32, 32, [259], "bhsd"),              # 64 rows
    (2, 1, 1, 40, 300, 128, 16, [300, 41], "bhsd"),         # a chunk of a prompt
    (150, 2, 1, 1, 70, 64, 64, None, "bhsd"),               # more pairs than SMs
    (1, 1, 2, 1, 9000, 64, 64, [8999], "bhsd"),             # one pair: its keys over many CTAs
    (1, 8, 4, 1, 4097, 128, 64, [4097], "bshd"),
    (40, 8, 1, 1, 600, 64, 32, "spread", "bhsd"),
    (5, 16, 2, 1, 1300, 32, 128, "spread", "bhsd"),
    (2, 1, 1, 3, 64, 64, 16, [2000000000, -7], "bhsd"),     # lengths behind the capacity and below zero
    (8, 8, 4, 1, 900, 128, 64, "spread", "bhsd"),           # clusters of six CTAs a pair
    (16, 8, 1, 1, 500, 128, 32, "spread", "bshd"),          # of three
]


def lengths(kv_len, B, S):
    if kv_len != "spread":
        return kv_len
    edges = [0, 1, 15, 16, 17, 63, 64, 65, S // 2, S - 1, S]
    return [min(edges[i % len(edges)], S) for i in range(B)]


def queries(B, Hq, Sq, D, dtype, seed, scale=1.0):
    """As a projection leaves them: [B, Sq, Hq, D] seen as [B, Hq, Sq, D]."""
    q = torch.from_numpy(randn((B, Sq, Hq, D), seed, scale)).cuda().to(DT[dtype])
    return q.transpose(1, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", DECODES, ids=lambda c: "x".join(map(str, c[:7])))
def test_decode(ctx, case, dtype):
    B, H, G, Sq, S, D, block, kv_len, layout = case
    ref = filled(B, H, S, D, block, 4)
    check_decode(ctx, ref, device_cache(ref, layout), queries(B, H * G, Sq, D, dtype, 6), dtype, kv_len=lengths(kv_len, B, S))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_decode_masks_and_lengths_that_leave_rows_empty(ctx, D, dtype):
    B, H, G, Sq, S, block = 4, 2, 3, 4, 210, 32
    ref = filled(B, H, S, D, block, 8)
    r = np.random.default_rng(1)
    mask = (r.random((B, Sq, S)) < 0.5).astype(np.float32)
    mask[0, 1], mask[1, :, :150], mask[2, 2, 5:], mask[2, 2, 3] = 0.0, 0.0, 0.0, np.nan     # (NaN is not zero: visible)
    kw = dict(kv_len=[210, 160, 4, 33], new_len=[4, 3, 4, 0], keep_mask=mask)
    cache, q = device_cache(ref), queries(B, H * G, Sq, D, dtype, 2)
    o, lse = check_decode(ctx, ref, cache, q, dtype, **kw)
    assert (o[3] == 0).all() and torch.isinf(lse[3]).all() and (o[1, :, 3] == 0).all() and (o[0, :, 1] == 0).all()
    check_decode(ctx, ref, cache, q, dtype, causal=False, score_clamp=0.5, scale=0.3, **kw)
    check_decode(ctx, ref, cache, q, dtype, causal=False, kv_len=[210, 160, 4, 33])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,block", [(32, 64), (64, 16), (128, 32), (128, 128)])
def test_decode_over_listed_blocks(ctx, D, block, dtype):
    """Blocks in any order, none (-1, and behind the last), the last short one, one listed twice."""
    B, H, G, Sq, S = 3, 2, 4, 2, 777
    ref = filled(B, H, S, D, block, 9)
    nb = -(-S // block)
    r = np.random.default_rng(2)
    blocks = np.stack([[r.permutation(nb + 2)[:7] - 1 for _ in range(H)] for _ in range(B)]).astype(np.int32)
    blocks[0, 0, 2] = blocks[0, 0, 0] = nb - 1
    blocks[1, 1] = -1
    blocks[1, 0, 3], blocks[2, 0, 1] = 2 ** 31 - 1, -2 ** 31
    cache, q = device_cache(ref, "bshd"), queries(B, H * G, Sq, D, dtype, 3)
    mask = (r.random((B, Sq, S)) < 0.7).astype(np.float32)
    o, lse = check_decode(ctx, ref, cache, q, dtype, kv_len=[777, 500, 770], blocks=blocks)
    assert (o[1, G:] == 0).all() and torch.isinf(lse[1, G:]).all()
    check_decode(ctx, ref, cache, q, dtype, kv_len=[777, 500, 770], blocks=blocks, keep_mask=mask)
    check_decode(ctx, ref, cache, q, dtype, blocks=np.arange(nb, dtype=np.int32)[None, None].repeat(B, 0).repeat(H, 1))
    check_decode(ctx, ref, cache, q, dtype, blocks=blocks[:, :, :1].copy(), causal=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_does_not_see_what_is_hidden(ctx, dtype):
    """NaN and the largest codes behind the length, under the mask and in blocks that are not listed."""
    B, H, G, Sq, S, D, block = 2, 2, 2, 2, 300, 64, 32
    ref = filled(B, H, S, D, block, 5)
    mask = np.ones((B, Sq, S), np.float32)
    mask[:, :, 40:77] = 0.0
    for codes in (ref.k, ref.v):
        codes[:, :, 40:77] = 0x7f
        codes[0, :, 201:] = 0xff
        codes[1, :, 299] = 0xff
    ref.vs[0, :, 7:], ref.ks[0, :, 7:] = np.nan, np.inf
    check_decode(ctx, ref, device_cache(ref), queries(B, H * G, Sq, D, dtype, 2), dtype, kv_len=[201, 299], keep_mask=mask)
    blocks = np.array([[[0, 3, 5, 6], [4, 0, 5, -1]]] * 2, dtype=np.int32)
    ref.ks[:, :, 1:3], ref.vs[:, :, 1:3] = np.nan, np.nan
    check_decode(ctx, ref, device_cache(ref), queries(B, H * G, Sq, D, dtype, 2), dtype, kv_len=[201, 299], blocks=blocks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_shows_nan_and_infinity_that_are_seen(ctx, dtype):
    B, H, S, D, block = 3, 1, 200, 64, 64
    ref = filled(B, H, S, D, block, 5)
    ref.k[0, 0, 17, 3] = 0x7f
    ref.v[1, 0, 150, 9] = 0x7f
    o, lse = ctx.kv8_decode(queries(B, 2, 1, D, dtype, 2), device_cache(ref))
    assert torch.isnan(o[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isnan(o[1, :, :, 9]).all() and torch.isfinite(o[1, :, :, :9]).all() and torch.isfinite(lse[1:]).all()
    assert torch.isfinite(o[2]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_of_values_of_very_different_size(ctx, dtype):
    """Scales from 2^-100 to 2^20 side by side, queries of any size: no score or weight may leave fp16 on its way."""
    B, H, G, S, D, block = 2, 2, 2, 256, 64, 16
    ref = filled(B, H, S, D, block, 5)
    r = np.random.default_rng(0)
    ref.vs[:] = 2.0 ** np.round(r.uniform(-100, 20, ref.vs.shape))
    ref.vs[1, 1] = 2.0 ** -100
    ref.ks[:] = 2.0 ** np.round(r.uniform(-60, -10, ref.ks.shape))
    ref.k[:, :, 48:64], ref.v[:, :, 48:64] = 0, 0
    q = queries(B, H * G, 1, D, dtype, 3)
    q[0] *= 2.0 ** 40
    q[1, 0] *= 2.0 ** -30
    q[1, 1, 0, 3] *= 2.0 ** 20
    q[1, 2] = 0
    check_decode(ctx, ref, device_cache(ref), q, dtype, scale=2.0 ** -38)


def test_decode_into_given_outputs_of_any_layout(ctx):
    B, H, G, Sq, S, D = 2, 2, 2, 3, 130, 64
    ref = filled(B, H, S, D, 64, 5)
    cache, q = device_cache(ref), queries(B, H * G, Sq, D, "bf16", 2)
    want, lse = ctx.kv8_decode(q, cache)
    big = torch.full((B, Sq + 2, H * G, D + 3), 5.0, device="cuda", dtype=torch.bfloat16)
    out = big[:, 1:-1, :, 1:D + 1].transpose(1, 2)
    lse2 = torch.empty_like(lse)
    odd = torch.nn.functional.pad(q, (1, 0))[..., 1:]                       # rows that start on any element
    got = ctx.kv8_decode(odd, cache, out=out, lse=lse2)
    assert got[0] is out and got[1] is lse2 and torch.equal(out, want) and torch.equal(lse, lse2)
    out.zero_()
    assert big.double().sum().item() == 5.0 * (big.numel() - out.numel())


def test_decode_and_read_of_shared_keys(ctx):
    """Sequences (or heads) that share their keys through a stride of zero: a common prompt."""
    B, H, S, D = 3, 2, 500, 64
    one = filled(1, H, S, D, 64, 5)
    cache = device_cache(one)
    q = queries(B, 2 * H, 1, D, "bf16", 2)
    rows = lambda t: t.expand(B, *t.shape[1:]).contiguous()  # noqa: E731
    shared = ltc.Kv8Cache(cache.k.expand(B, H, S, D), cache.v.expand(B, H, S, D), rows(cache.k_scale), rows(cache.v_scale), None, 64)
    length = ints([500, 64, 333])
    got = ctx.kv8_decode(q, shared, kv_len=length)
    own = ltc.Kv8Cache(*(rows(t.view(torch.uint8)).view(torch.float8_e4m3fn) for t in cache[:2]), shared.k_scale, shared.v_scale, None, 64)
    want = ctx.kv8_decode(q, own, kv_len=length)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(ctx.kv8_read(shared, kv_len=length)[0], ctx.kv8_read(own, kv_len=length)[0])
    heads = shared._replace(k=own.k[:, :1].expand(B, H, S, D), k_scale=own.k_scale[:, :1].expand(B, H, -1).contiguous())
    got = ctx.kv8_decode(q, heads, kv_len=length)
    want = ctx.kv8_decode(q, heads._replace(k=rows(heads.k.contiguous())), kv_len=length)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ltc.LtcaError):                               # tokens that share a key are no cache
        ctx.kv8_decode(q, shared._replace(k=own.k[:, :, :1].expand(B, H, S, D)), kv_len=length)


# ---- select ------------------------------------------------------------------------------------
SELECTS = [
    # B, H, G, Sq, S, D, block, kv_len, count, first, last
    (1, 1, 1, 1, 1, 32, 16, [1], 1, 0, 1), (2, 2, 4, 1, 1000, 64, 16, [1000, 17], 5, 1, 1),
    (3, 1, 3, 2, 5000, 128, 64, [5000, 0, 64], 16, 1, 2), (2, 2, 1, 4, 777, 128, 32, None, 30, 0, 0),
    (1, 2, 8, 1, 20000, 64, 16, [19985], 100, 2, 3), (4, 8, 2, 1, 300, 32, 128, [300, 129, 128, 1], 2, 1, 1),
    (1, 1, 2, 1, 640, 64, 32, [2000000000], 64, 0, 64), (1, 3, 5, 5, 4100, 64, 16, [4099], 256, 0, 1),
    (2, 1, 1, 1, 300, 64, 16, [-4, 300], 3, 3, 0),
    (2, 2, 2, 1, 300000, 32, 16, [300000, 270001], 77, 1, 1),       # more blocks than one CTA goes through
    (1, 1, 40, 1, 2000, 64, 16, [1999], 33, 1, 1),                  # more rows than are in shared memory at once
    (20, 16, 1, 1, 500, 32, 16, None, 2, 1, 1),                     # a CTA alone; no choice is left
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", SELECTS, ids=lambda c: "x".join(map(str, c[:7])))
def test_select(ctx, case, dtype):
    B, H, G, Sq, S, D, block, kv_len, count, first, last = case
    ref = filled(B, H, S, D, block, 11)
    q = queries(B, H * G, Sq, D, dtype, 6)
    out = torch.full((B, H, count), 99, dtype=torch.int32, device="cuda")
    got = ctx.kv8_select(q, device_cache(ref), ints(kv_len), count, first=first, last=last, out=out)
    assert got is out
    assert np.array_equal(got.cpu().numpy(), ref.select(q.double().cpu().numpy(), kv_len, count, None, first, last))


def test_select_breaks_ties_towards_the_lower_index(ctx):
    """Equal bounds throughout, then two sizes of them: the first ones of the larger size, in order; rows that do not count."""
    B, H, S, D, block = 2, 2, 3000, 64, 16
    ref = filled(B, H, S, D, block, 1, spread=0.0)
    ref.bounds[:] = ref.bounds[:1, :1, :1]
    ref.ks[:] = 1.0
    q = queries(B, H, 2, D, "bf16", 6)
    for ks in (1.0, np.where(np.arange(ref.ks.shape[2]) % 7 == 3, 2.0, 1.0)):
        ref.ks[:] = ks
        for new_len in (None, [1, 0]):
            got = ctx.kv8_select(q, device_cache(ref), ints([S, S - 100]), 40, new_len=ints(new_len))
            assert np.array_equal(got.cpu().numpy(), ref.select(q.double().cpu().numpy(), [S, S - 100], 40, new_len))


def test_select_with_special_queries(ctx):
    B, H, S, D, block = 1, 5, 1000, 64, 16
    ref = filled(B, H, S, D, block, 1)
    q = queries(B, H, 1, D, "f32", 6)
    q[0, 0, 0, 3], q[0, 0, 0, 4] = float("nan"), float("inf")
    q[0, 1] = float("nan")
    q[0, 2] = 0.0
    q[0, 3] *= 2.0 ** 90
    q[0, 4] *= 2.0 ** -110
    got = ctx.kv8_select(q, device_cache(ref), None, 9, first=0, last=0)
    qq = q.double().cpu().numpy()
    qq[0, 0, 0, 4] = np.inf
    assert np.array_equal(got.cpu().numpy(), ref.select(qq, None, 9, None, 0, 0))


# ---- together ----------------------------------------------------------------------------------
def test_a_serving_loop(ctx):
    """Prompts of different lengths, then steps of one token: append, select, attend over the selection and over everything.
    The same steps again from a captured graph, whose replays read the lengths that the loop counts up."""
    B, H, G, S, D, block = 3, 2, 4, 400, 64, 16
    cache = ctx.kv8_cache(B, H, S, D, block=block, bounds=True)
    ref = Cache.empty(B, H, S, D, block)
    new = [150, 1, 77]
    k, v = bf16_round(randn((B, H, 150, D), 1)), bf16_round(randn((B, H, 150, D), 2))
    bf16 = lambda x: torch.from_numpy(x).cuda().bfloat16()  # noqa: E731
    ctx.kv8_append(cache, bf16(k), bf16(v), ints(new), new_len=ints(new))
    ref.append(k, v, new, new)
    check_cache(cache, ref)
    length = ints(new)
    qs, ks, vs = (torch.zeros((B, n, 1, D), dtype=torch.bfloat16, device="cuda") for n in (H * G, H, H))

    def step():
        length.add_(1)
        ctx.kv8_append(cache, ks, vs, length)
        blocks = ctx.kv8_select(qs, cache, length, 4)
        return blocks, ctx.kv8_decode(qs, cache, kv_len=length, blocks=blocks), ctx.kv8_decode(qs, cache, kv_len=length)

    graph, graph_out = None, None
    side = torch.cuda.Stream()
    for t in range(40):
        kn, vn, qn = (bf16_round(randn((B, n, 1, D), 10 + 3 * t + i)) for i, n in enumerate((H, H, H * G)))
        qs.copy_(bf16(qn)); ks.copy_(bf16(kn)); vs.copy_(bf16(vn))
        torch.cuda.synchronize()
        if t < 20:
            blocks, sparse, dense = step()
        else:
            if graph is None:
                before = length.clone()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    ctx.set_stream(side)
                    graph_out = step()
                ctx.set_stream(torch.cuda.current_stream())
                assert torch.equal(before, length)
            graph.replay()
            blocks, sparse, dense = graph_out
        torch.cuda.synchronize()
        new = [n + 1 for n in new]
        ref.append(kn, vn, new)
        assert length.tolist() == new
        check_cache(cache, ref)
        want = ref.select(qn, new, 4)
        assert np.array_equal(blocks.cpu().numpy(), want)
        for got, kw in ((sparse, dict(blocks=want)), (dense, {})):
            o_ref, lse_ref, *rest = ref.decode(qn, kv_len=new, **kw)
            to, tl = decode_tolerances(o_ref, lse_ref, *rest, True)
            assert (np.abs(got[0].double().cpu().numpy() - o_ref) <= to).all()
            assert (np.abs(got[1].double().cpu().numpy() - lse_ref) <= tl).all()


def test_prompt_chunk_through_read_and_forward(ctx):
    """The long chunk of a prompt: the cache read back in bf16, then the framework's forward over it."""
    B, H, S, D = 2, 4, 512, 64
    cache = ctx.kv8_cache(B, H, S, D)
    k, v = (torch.from_numpy(randn((B, H, S, D), i, 0.5)).cuda().bfloat16() for i in range(2))
    length = ints([512, 300])
    ctx.kv8_append(cache, k, v, length, new_len=length)
    q = queries(B, H, 200, D, "bf16", 3, 0.5)
    kk, vv = ctx.kv8_read(cache, kv_len=length)
    o, lse = ctx.attn_fwd(q, kk, vv, kv_len=length)
    o2, lse2 = ctx.kv8_decode(q, cache, kv_len=length, causal=False)
    # the same values on both ways; the forward's own bounds against fp32: 2e-3 + a bf16 step, and lse 2e-3
    assert ((o.float() - o2.float()).abs() <= 4e-3 + 2.0 ** -7 * o2.float().abs()).all()
    assert (lse - lse2).abs().max() < 4e-3


def test_calls_on_two_streams_and_contexts(ctx):
    """Two contexts whose calls overlap, one of them split over scratch: both keep their results."""
    B, H, S, D = 1, 1, 30000, 64
    refs = [filled(B, H, S, D, 64, i) for i in range(2)]
    caches = [device_cache(r) for r in refs]
    qs = [queries(B, 2, 1, D, "bf16", 30 + i) for i in range(2)]
    alone = [ctx.kv8_decode(q, c) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [ltc.Context(0, s) for s in streams]
    got = []
    for _ in range(20):
        got.append([x.kv8_decode(q, c) for x, q, c in zip(ctxs, qs, caches)])
    torch.cuda.synchronize()
    for pair in got:
        for (o, lse), (o_ref, lse_ref) in zip(pair, alone):
            assert torch.equal(o, o_ref) and torch.equal(lse, lse_ref)
    for c in ctxs:
        c.close()


def test_two_captured_graphs_of_one_context(ctx):
    """Calls that join their shares through scratch, captured into two graphs and replayed side by side: each graph has scratch of
    its own, which a larger call in between does not take away."""
    B, H, S, D = 2, 2, 20000, 64
    refs = [filled(B, H, S, D, 64, i) for i in range(2)]
    caches = [device_cache(r) for r in refs]
    qs = [queries(B, 2 * H, 1, D, "f32", 30 + i) for i in range(2)]
    want = [ctx.kv8_decode(q, c) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for q, c, s in zip(qs, caches, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ctx.set_stream(s)
            outs.append(ctx.kv8_decode(q, c))
        graphs.append(g)
    ctx.set_stream(torch.cuda.current_stream())
    big = filled(4, 8, 20000, D, 64, 3)
    ctx.kv8_decode(queries(4, 64, 1, D, "f32", 5), device_cache(big))
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("case", [
    # B, H, G, Sq, S, D            fp32 queries over many keys: the sums do not drift
    (4, 4, 2, 1, 16000, 128), (2, 2, 4, 2, 30000, 32), (60, 8, 1, 1, 2000, 64)])
def test_decode_in_fp32_stays_below_1e_6(ctx, case):
    """In the 2-norm over all of the result against 64 bits.  Each fp32 rounding is off by 2^-24 of its sum at most and in either
    direction, so that the roundings of a row's sums add up like the root of their number at most: for 16000 keys in warps that
    take 64 and more of them, 2^-24 sqrt(500) = 1.3e-6 at the very worst of a row, a third of it in the mean of uniform errors;
    the fp16 terms (2^-22) and exponentials (2^-22) come to less."""
    B, H, G, Sq, S, D = case
    ref = filled(B, H, S, D, 64, 12, spread=2.0)
    q = queries(B, H * G, Sq, D, "f32", 6)
    o, _ = ctx.kv8_decode(q, device_cache(ref))
    k, v = (torch.from_numpy(x).cuda() for x in ref.values())
    x = q.double().reshape(B, H, G * Sq, D) @ k.transpose(2, 3) * D ** -0.5
    seen = torch.arange(S, device="cuda")[None] <= S - Sq + torch.arange(Sq, device="cuda")[:, None]
    x = x.view(B, H, G, Sq, S).masked_fill(~seen, -float("inf")).view(B, H, G * Sq, S)
    want = (torch.softmax(x, 3) @ v).view(B, H * G, Sq, D)
    assert ((o.double() - want).norm() / want.norm()).item() < 1e-6


def test_results_repeat_bit_for_bit(ctx):
    ref = filled(3, 4, 3000, 128, 64, 5)
    cache, q = device_cache(ref), queries(3, 16, 2, 128, "f32", 2)
    first = ctx.kv8_decode(q, cache, kv_len=ints([3000, 1234, 7]))
    for _ in range(5):
        again = ctx.kv8_decode(q, cache, kv_len=ints([3000, 1234, 7]))
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_beyond_32_bits(ctx):
    """A cache of more than 2^32 bytes: its last sequence is written, selected from, read and attended to."""
    B, H, S, D, block = 5, 8, 1 << 20, 128, 128
    cache = ctx.kv8_cache(B, H, S, D, block=block, bounds=True)
    k = torch.from_numpy(bf16_round(randn((B, H, 300, D), 1))).cuda().bfloat16()
    length = ints([S, 5, S - 77, 300, S])
    ctx.kv8_append(cache, k, -k, length)
    kk, vv = ctx.kv8_read(cache, start=S - 300, dtype=torch.float32)
    assert (kk[4] - k[4].float()).abs().max() <= 2.0 ** -4 * k[4].float().abs().max() and torch.equal(kk[4], -vv[4])
    # the newest 300 keys, and zeros before them
    nb = S // block
    blocks = torch.arange(nb - 3, nb, dtype=torch.int32, device="cuda").expand(B, H, 3).contiguous()
    q = queries(B, H * 2, 1, D, "f32", 3)
    o, _ = ctx.kv8_decode(q, cache, blocks=blocks)
    tail = torch.cat([torch.zeros_like(kk[4, :, :84]), kk[4]], 1).double()
    x = q[4].double().view(H, 2, D) @ tail.transpose(1, 2) * D ** -0.5
    want = torch.softmax(x, 2) @ -tail
    assert (o[4].double().view(H, 2, D) - want).abs().max() < 1e-4
    o, _ = ctx.kv8_decode(q, cache, kv_len=length)
    most = torch.exp(x).sum(2, keepdim=True) + (S - 384)
    want = (torch.exp(x) @ -tail) / most
    assert (o[4].double().view(H, 2, D) - want).abs().max() < 1e-5
    got = ctx.kv8_select(q, cache, length, 5)
    assert got[4, :, 0].eq(0).all() and got[4, :, -1].eq(nb - 1).all() and set(got[4].unique().tolist()) >= {nb - 3, nb - 2}


# ---- refusals ----------------------------------------------------------------------------------
def test_refusals(ctx):
    cache = ctx.kv8_cache(2, 2, 100, 64)
    k = torch.zeros((2, 2, 4, 64), dtype=torch.bfloat16, device="cuda")
    length = ints([4, 4])
    q = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: ctx.kv8_append(cache, k[:1], k, length), lambda: ctx.kv8_append(cache, k, k.float(), length),
        lambda: ctx.kv8_append(cache, k, k, None), lambda: ctx.kv8_append(cache, k, k, length.long()),
        lambda: ctx.kv8_append(cache, k, k, length[:1]), lambda: ctx.kv8_append(cache, k, k, length, new_len=length.cpu()),
        lambda: ctx.kv8_append(cache, k.cpu(), k, length), lambda: ctx.kv8_append(cache, k.half(), k.half(), length),
        lambda: ctx.kv8_append(cache[:5], k, k, length), lambda: ctx.kv8_append(cache._replace(block=32), k, k, length),
        lambda: ctx.kv8_append(cache._replace(k=cache.k.view(torch.uint8)), k, k, length),
        lambda: ctx.kv8_append(cache._replace(k=cache.k[..., :32]), k, k, length),
        lambda: ctx.kv8_append(cache._replace(k_scale=cache.k_scale.double()), k, k, length),
        lambda: ctx.kv8_append(cache._replace(k=cache.k[:, :1].expand(2, 2, 100, 64)), k, k, length),
        lambda: ctx.kv8_read(cache, start=-1), lambda: ctx.kv8_read(cache, start=50, count=51),
        lambda: ctx.kv8_read(cache, dtype=torch.float16), lambda: ctx.kv8_read(cache, out_k=q),
        lambda: ctx.kv8_decode(q[:, :3], cache), lambda: ctx.kv8_decode(q[..., :32], cache), lambda: ctx.kv8_decode(q.half(), cache),
        lambda: ctx.kv8_decode(q, cache, keep_mask=torch.ones((2, 1, 99), device="cuda")), lambda: ctx.kv8_decode(q, cache, scale=0.0),
        lambda: ctx.kv8_decode(q, cache, blocks=torch.zeros((2, 4, 1), dtype=torch.int32, device="cuda")),
        lambda: ctx.kv8_decode(q, cache, blocks=torch.zeros((2, 2, 0), dtype=torch.int32, device="cuda")),
        lambda: ctx.kv8_decode(q, cache, out=q.float()), lambda: ctx.kv8_decode(q[:, :, :0], cache),
        lambda: ctx.kv8_select(q, cache, length, 4),
        lambda: ctx.kv8_select(q, ctx.kv8_cache(2, 2, 100, 64, bounds=True), length, 1),
        lambda: ctx.kv8_select(q, ctx.kv8_cache(2, 2, 100, 64, bounds=True), length, 0),
        lambda: ctx.kv8_append(ctx.kv8_cache(2, 2, 100, 48), k[..., :48], k[..., :48], length),
        lambda: ctx.kv8_append(ctx.kv8_cache(2, 2, 100, 64, block=24), k, k, length),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ltc.LtcaError, AssertionError, TypeError)):
            call()
            pytest.fail(f"call {i} was not refused")
    ctx.kv8_append(cache, k[:, :, :0], k[:, :, :0], length)          # nothing to do
    assert ctx.kv8_read(cache, count=0)[0].shape == (2, 2, 0, 64)


def test_module_level_calls(ctx):
    cache = ctx.kv8_cache(1, 1, 64, 32, bounds=True)
    k = torch.from_numpy(randn((1, 1, 64, 32), 1)).cuda()
    n = ints([64])
    ltc.kv8_append(cache, k, k, n)
    q = torch.from_numpy(randn((1, 2, 1, 32), 2)).cuda()
    a, b = ltc.kv8_decode(q, cache, n), ctx.kv8_decode(q, cache, kv_len=n)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert ltc.kv8_select(q, cache, n, 3).tolist() == [[[0, -1, -1]]]
    assert torch.equal(ltc.kv8_read(cache, kv_len=n)[0], ctx.kv8_read(cache)[0])

"""The 8-bit decode where its warps share one line of steps and a second kernel joins what they have of a unit: what large calls
take.  Against the definition in 64 bits, every case with a check that the call does take it."""
import ctypes as C

import numpy as np
import pytest
import torch

import cuda_ltc_b200 as ltc
from cuda_ltc_b200 import _lib
from test_kv8_gpu import check_decode, device_cache, filled, ints, queries

pytestmark = pytest.mark.gpu


def workspace(cache, q, blocks=None):
    """Bytes of scratch that a call of these shapes needs: none where the CTAs of a cluster share a unit."""
    B, H, S, D = cache.k.shape
    c = _lib.Kv8CacheParams(B=B, H=H, S=S, D=D, block=cache.block)
    p = _lib.Kv8DecodeParams(Hq=q.shape[1], Sq=q.shape[2], dtype=_lib.LTCA_F32 if q.dtype == torch.float32 else _lib.LTCA_BF16, scale=1.0)
    if blocks is not None:
        p.blocks, p.n_blocks = 256, blocks.shape[2]
    n = C.c_size_t()
    assert _lib.load().ltca_kv8_decode_workspace_bytes(C.byref(c), C.byref(p), C.byref(n)) == 0
    return n.value


def check_line(ctx, ref, cache, q, dtype, **kw):
    assert workspace(cache, q, kw.get("blocks")) > 0
    return check_decode(ctx, ref, cache, q, dtype, **kw)


def ragged(B, S, seed):
    """Lengths of every kind, empty sequences first, last, alone and several in a row."""
    r = np.random.default_rng(seed)
    edges = np.array([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, S // 2, S - 1, S])
    n = np.where(r.random(B) < 0.5, edges[r.integers(0, edges.size, B)], r.integers(0, S + 1, B))
    n[[0, 1, B - 1]] = 0
    n[B // 2:B // 2 + 5] = 0
    return [int(x) for x in n]


DTYPES = ["f32", "bf16"]
MANY = [
    # B, H, G, Sq, S, D, block, layout         more units than the SMs hold at once
    (300, 2, 1, 1, 200, 64, 32, "bhsd"),       # more than 256 sequences: lengths that are not in shared memory, three to a thread
    (160, 4, 3, 1, 150, 32, 16, "bshd"),       # two to a thread
    (129, 4, 1, 2, 133, 128, 64, "bhsd"),
    (300, 1, 16, 1, 100, 128, 128, "bshd"),    # two tiles of eight rows
    (75, 8, 3, 5, 90, 64, 16, "bhsd"),         # 15 rows: a tile that is not full, tokens that begin inside it
    (60, 4, 5, 7, 70, 32, 32, "bhsd"),         # 35 rows: three units a pair, the last of three rows
    (40, 4, 8, 6, 64, 128, 16, "bhsd"),        # 48 rows
]
LONG = [
    # few units, each over many warps
    (1, 1, 1, 1, 9000, 128, 64, "bhsd"), (2, 1, 7, 5, 9100, 128, 16, "bshd"), (3, 2, 3, 4, 9001, 64, 128, "bhsd"),
    (1, 2, 9, 1, 17000, 32, 32, "bhsd"), (4, 2, 1, 3, 20000, 32, 64, "bshd"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", MANY, ids=lambda c: "x".join(map(str, c[:7])))
def test_many_sequences_of_different_lengths(ctx, case, dtype):
    B, H, G, Sq, S, D, block, layout = case
    ref = filled(B, H, S, D, block, 4)
    check_line(ctx, ref, device_cache(ref, layout), queries(B, H * G, Sq, D, dtype, 6), dtype, kv_len=ragged(B, S, 5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", LONG, ids=lambda c: "x".join(map(str, c[:7])))
def test_few_long_sequences(ctx, case, dtype):
    B, H, G, Sq, S, D, block, layout = case
    ref = filled(B, H, S, D, block, 4)
    cache, q = device_cache(ref, layout), queries(B, H * G, Sq, D, dtype, 6)
    # a length of one step beside the longest, an empty sequence between two others, all at once
    for kv_len in ([S, 17, 0, S - 3], [S - 16, 0, S, 1], [1, S, 5, 0]):
        check_line(ctx, ref, cache, q, dtype, kv_len=kv_len[:B])
    check_line(ctx, ref, cache, q, dtype, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,Sq,S,D,block", [(3, 2, 3, 4, 9000, 64, 32), (300, 2, 2, 3, 110, 64, 32), (2, 1, 16, 2, 9000, 128, 64),
                                                (150, 2, 1, 20, 90, 128, 16), (3, 1, 1, 1, 17000, 32, 16), (110, 8, 4, 4, 70, 32, 64)])
def test_masks_and_tokens_that_are_not_there(ctx, B, H, G, Sq, S, D, block, dtype):
    ref = filled(B, H, S, D, block, 8)
    r = np.random.default_rng(1)
    mask = (r.random((B, Sq, S)) < 0.5).astype(np.float32)
    mask[0, 0], mask[1, :, :S - S // 4], mask[2 % B, Sq - 1, 5:] = 0.0, 0.0, 0.0
    mask[B - 1, 0, 3] = np.nan                                        # (not zero: visible)
    kv_len, new_len = ragged(B, S, 2), r.integers(0, Sq + 1, B)
    if B <= 3:
        kv_len = [S, S - 70, 4][:B]
    new_len[0] = Sq
    cache, q = device_cache(ref), queries(B, H * G, Sq, D, dtype, 2)
    check_line(ctx, ref, cache, q, dtype, kv_len=kv_len, new_len=new_len, keep_mask=mask)
    check_line(ctx, ref, cache, q, dtype, kv_len=kv_len, new_len=new_len, causal=False, score_clamp=0.5, scale=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,Sq,S,D,block,n", [
    (2, 2, 4, 1, 12000, 64, 16, 600),           # a list that several windows of 32 entries hold
    (160, 4, 2, 1, 400, 64, 32, 7), (150, 2, 2, 8, 300, 128, 16, 9), (1, 1, 3, 2, 20000, 128, 128, 70),
    (2, 1, 12, 1, 30000, 32, 64, 300), (170, 4, 1, 1, 300, 32, 16, 33)])
def test_listed_blocks(ctx, B, H, G, Sq, S, D, block, n, dtype):
    """Blocks in any order, none of them, some or most of them -1 or behind the last, and short ones at the end."""
    ref = filled(B, H, S, D, block, 9)
    nb = -(-S // block)
    r = np.random.default_rng(2)
    blocks = np.stack([[np.resize(r.permutation(nb + 4) - 2, n) for _ in range(H)] for _ in range(B)]).astype(np.int32)
    blocks[r.random((B, H)) < 0.3, n // 4:] = -1                      # mostly none
    blocks[0, 0, n // 2:] = -1
    blocks[B - 1, H - 1] = -1
    blocks[0, H - 1, n - 1], blocks[B // 2, 0, 0] = 2 ** 31 - 1, -2 ** 31
    kv_len = ragged(B, S, 3) if B > 3 else [S, S - 100][:B]
    cache, q = device_cache(ref, "bshd"), queries(B, H * G, Sq, D, dtype, 3)
    o, lse = check_line(ctx, ref, cache, q, dtype, kv_len=kv_len, blocks=blocks)
    assert (o[B - 1, -G:] == 0).all() and torch.isinf(lse[B - 1, -G:]).all()
    mask = (r.random((B, Sq, S)) < 0.7).astype(np.float32)
    check_line(ctx, ref, cache, q, dtype, kv_len=kv_len, blocks=blocks, keep_mask=mask, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [1, 11])
def test_rows_on_any_element(ctx, G, dtype):
    """Queries and results off their boundaries, beside results of the usual layout, equal bit for bit."""
    B, H, Sq, S, D = 310, 2, 1, 130, 64
    ref = filled(B, H, S, D, 64, 5)
    cache, q = device_cache(ref), queries(B, H * G, Sq, D, dtype, 2)
    kv_len = ragged(B, S, 7)
    want, lse = check_line(ctx, ref, cache, q, dtype, kv_len=kv_len)
    big = torch.full((B, Sq + 2, H * G, D + 3), 5.0, device="cuda", dtype=q.dtype)
    out = big[:, 1:-1, :, 1:D + 1].transpose(1, 2)
    odd = torch.nn.functional.pad(q, (1, 0))[..., 1:]
    got = ctx.kv8_decode(odd, cache, kv_len=ints(kv_len), out=out)
    assert got[0] is out and torch.equal(out, want) and torch.equal(got[1], lse)
    out.zero_()
    assert big.double().sum().item() == 5.0 * (big.numel() - out.numel())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,G,S", [(2, 2, 9000), (300, 2, 300), (300, 12, 200)])
def test_what_is_hidden(ctx, B, G, S, dtype):
    """NaN and the largest codes behind the length, under the mask and in blocks that are not listed."""
    H, Sq, D, block = 2, 2, 64, 32
    ref = filled(B, H, S, D, block, 5)
    mask = np.ones((B, Sq, S), np.float32)
    mask[:, :, 40:77] = 0.0
    kv_len = [S - 99 - (b % 7) for b in range(B)]
    for codes in (ref.k, ref.v):
        codes[:, :, 40:77] = 0x7f
        for b in range(B):
            codes[b, :, kv_len[b]:] = 0xff
    last = (S - 99 + block - 1) // block
    ref.vs[:, :, last:], ref.ks[:, :, last:] = np.nan, np.inf
    cache, q = device_cache(ref), queries(B, H * G, Sq, D, dtype, 2)
    check_line(ctx, ref, cache, q, dtype, kv_len=kv_len, keep_mask=mask)
    nb = -(-S // block)
    blocks = np.tile(np.array([j for j in range(nb) if j not in (1, 2)] + [-1, -1], np.int32), (B, H, 1))
    ref.ks[:, :, 1:3], ref.vs[:, :, 1:3] = np.nan, np.nan
    check_line(ctx, ref, device_cache(ref), q, dtype, kv_len=kv_len, blocks=blocks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_that_is_seen(ctx, dtype):
    B, H, S, D = 4, 1, 9000, 64
    ref = filled(B, H, S, D, 64, 5)
    ref.k[0, 0, 4017, 3] = 0x7f
    ref.v[1, 0, 8150, 9] = 0x7f
    ref.v[2, 0, 8999, 9] = 0x7f                                       # which only the second of two new tokens sees
    cache, q = device_cache(ref), queries(B, 2, 2, D, dtype, 2)
    assert workspace(cache, q) > 0
    o, lse = ctx.kv8_decode(q, cache)
    assert torch.isnan(o[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isnan(o[1, :, :, 9]).all() and torch.isfinite(o[1, :, :, :9]).all() and torch.isfinite(lse[1:]).all()
    assert torch.isfinite(o[2, :, 0]).all() and torch.isnan(o[2, :, 1, 9]).all() and torch.isfinite(o[2, :, 1, 10:]).all()
    assert torch.isfinite(o[3]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,G,S", [(2, 2, 9000), (320, 1, 256), (310, 9, 100)])
def test_values_of_very_different_size(ctx, B, G, S, dtype):
    """Shares whose references lie far apart: scales from 2^-100 to 2^20 side by side, queries of any size."""
    H, D, block = 2, 64, 16
    ref = filled(B, H, S, D, block, 5)
    r = np.random.default_rng(0)
    ref.vs[:] = 2.0 ** np.round(r.uniform(-100, 20, ref.vs.shape))
    ref.vs[1, 1] = 2.0 ** -100
    ref.ks[:] = 2.0 ** np.round(r.uniform(-60, -10, ref.ks.shape))
    ref.k[:, :, 48:64], ref.v[:, :, 48:64] = 0, 0
    q = queries(B, H * G, 1, D, dtype, 3)
    q[0] *= 2.0 ** 40
    q[1, 0] *= 2.0 ** -30
    q[1, -1] = 0
    check_line(ctx, ref, device_cache(ref), q, dtype, scale=2.0 ** -38)


def test_shared_keys(ctx):
    """Sequences, or heads, that share their keys through a stride of zero."""
    B, H, S, D = 301, 2, 200, 64
    one = filled(1, H, S, D, 64, 5)
    c = device_cache(one)
    rows = lambda t: t.expand(B, *t.shape[1:]).contiguous()  # noqa: E731
    shared = ltc.Kv8Cache(c.k.expand(B, H, S, D), c.v.expand(B, H, S, D), rows(c.k_scale), rows(c.v_scale), None, 64)
    own = shared._replace(k=rows(c.k.view(torch.uint8)).view(torch.float8_e4m3fn), v=rows(c.v.view(torch.uint8)).view(torch.float8_e4m3fn))
    q, n = queries(B, 2 * H, 1, D, "bf16", 2), ints(ragged(B, S, 9))
    assert workspace(own, q) > 0
    got, want = ctx.kv8_decode(q, shared, kv_len=n), ctx.kv8_decode(q, own, kv_len=n)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    heads = own._replace(k=own.k[:, :1].expand(B, H, S, D), k_scale=own.k_scale[:, :1].expand(B, H, -1).contiguous())
    got, want = ctx.kv8_decode(q, heads, kv_len=n), ctx.kv8_decode(q, heads._replace(k=heads.k.contiguous()), kv_len=n)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_one_key_among_many_calls(ctx):
    """Lengths of one and none over thousands of sequences: a unit of one step each, and blanks between them."""
    B, H, S, D = 5000, 1, 16, 32
    ref = filled(B, H, S, D, 16, 5)
    kv_len = np.random.default_rng(3).integers(0, 2, B)
    q = queries(B, 1, 1, D, "f32", 2)
    o, lse = check_line(ctx, ref, device_cache(ref), q, "f32", kv_len=kv_len)
    assert (o[torch.from_numpy(kv_len == 0)] == 0).all()
    check_line(ctx, ref, device_cache(ref), q, "f32", kv_len=np.zeros(B, int))


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_bit_for_bit(ctx, dtype):
    ref = filled(301, 2, 300, 64, 64, 5)
    cache, q, n = device_cache(ref), queries(301, 24, 1, 64, dtype, 2), ints(ragged(301, 300, 4))
    assert workspace(cache, q) > 0
    first = ctx.kv8_decode(q, cache, kv_len=n)
    for _ in range(5):
        again = ctx.kv8_decode(q, cache, kv_len=n)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])

"""The 8-bit decode where a weight and the scale of its values say little of what they bring: keys with all of the weight and no value,
values far below their block's scale.  Both plans, against the definition in 64 bits."""
import numpy as np
import pytest

from kv8_ref import VALUES, encode
from test_kv8_gpu import check_decode, device_cache, filled, ints, queries

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16"]
SHAPES = [(2, 2, 2, 300, 64), (2, 1, 9, 9000, 128), (300, 2, 1, 250, 64), (310, 1, 12, 100, 32)]      # B, H, G, S, D


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [3, 70])
@pytest.mark.parametrize("B,H,G,S,D", SHAPES)
def test_a_key_with_all_of_the_weight_and_no_value(ctx, B, H, G, S, D, at, dtype):
    """The result is what the other keys bring, down to 2^-18 of the weights, and has to be right in itself.

    A row's weights p over l and values v: O = sum p v / l.  Off by the scores' error (2^-19 of their size, on the weights and on l) and
    the exponentials' 2^-20; by the weights' own rounding, 2^-11 with bf16 rows, with fp32 rows 2^-22 and no finer than 2^-35 of the
    largest weight, which the key without a value has (its own p is at least l / 2 here); fp32 additions, 2^-23 for each 8 keys."""
    block = 16
    ref = filled(B, H, S, D, block, 5)
    ref.ks[:] = 1.0
    r = np.random.default_rng(1)
    ref.k[:] = encode(r.choice([-0.125, 0.0, 0.125], ref.k.shape))
    ref.vs[:] = 2.0 ** -6
    first = at // block * block
    ref.v[:, :, first:first + block], ref.vs[:, :, at // block] = 0, 2.0 ** 30
    q = queries(B, H * G, 1, D, dtype, 3)
    q[:] = 1.0
    for b in range(B):
        gap = (1, 6, 12, 18)[b % 4]                                    # and log2 S more, so that its weight is most of all
        ref.k[b, :, at] = encode((gap + np.log2(S)) * np.log(2) / np.sqrt(D))
    kv_len = [S - (b % 3) for b in range(B)]
    o, lse = ctx.kv8_decode(q, device_cache(ref), kv_len=ints(kv_len))
    o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
    want, want_lse, size, keys, _ = ref.decode(q.double().cpu().numpy(), kv_len=kv_len)
    k, v = ref.values()
    for b in range(B):
        for h in range(H):
            s = k[b, h, :kv_len[b]].sum(1) * D ** -0.5
            p = np.exp(s - s.max())
            brought = p @ np.abs(v[b, h, :kv_len[b]]) / p.sum()
            most = np.abs(v[b, h, :kv_len[b]]).sum(0) / p.sum()
            for row in range(h * G, (h + 1) * G):
                to = brought * (2 * size[b, row, 0] * 2.0 ** -19 + 2.0 ** -19 + (keys[b, row, 0] / 8 + 64) * 2.0 ** -23 + 2.0 ** -22)
                to = to + (brought * 2.0 ** -11 + 2.0 ** -8 * np.abs(want[b, row, 0]) if dtype == "bf16" else most * 2.0 ** -35)
                err = np.abs(o[b, row, 0] - want[b, row, 0])
                assert (err <= to).all(), (b, row, (err / to).max())
            assert np.abs(lse[b, h * G:(h + 1) * G] - want_lse[b, h * G:(h + 1) * G]).max() < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,S,D", SHAPES)
def test_small_codes_beside_others(ctx, B, H, G, S, D, dtype):
    """Every third block holds the smallest codes at a scale that makes their values the others' equals, another third is nothing at a
    scale of 2^40."""
    block = 16
    ref = filled(B, H, S, D, block, 5)
    r = np.random.default_rng(2)
    nb = ref.vs.shape[2]
    of = np.arange(S) // block
    small, none = of % 3 == 0, of % 3 == 1
    ref.v[:, :, small] = encode(r.choice([-2.0, -1.0, 1.0, 2.0, 3.0], (B, H, int(small.sum()), D)) * 2.0 ** -9)
    ref.v[:, :, none] = 0
    j = np.arange(nb)
    ref.vs[:] = np.where(j % 3 == 0, 2.0 ** 9, np.where(j % 3 == 1, 2.0 ** 40, 2.0 ** -6))
    assert np.abs(VALUES[ref.v[:, :, small]]).max() == 3 * 2.0 ** -9
    check_decode(ctx, ref, device_cache(ref), queries(B, H * G, 1, D, dtype, 3), dtype, kv_len=[S - (b % 5) for b in range(B)])

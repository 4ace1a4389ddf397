"""The 8-bit decode of scores whose last fp32 place is worth more than fp16's range of weights: one key is far ahead, and its values
are the result."""
import numpy as np
import pytest

from kv8_ref import VALUES, decode_tolerances, encode
from test_kv8_gpu import device_cache, filled, ints, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,S,G", [(64, 300, 2), (128, 333, 9), (32, 9000, 1), (64, 9001, 12), (128, 9000, 3)])   # both plans
def test_one_key_far_ahead(ctx, D, S, G, dtype):
    """Key j is c_j in every channel and the query +-2^x: the largest c (the smallest) by a factor of 30/28 (8/4) and more, where an
    fp32 score of D products is off by 2^-17 at most.  The result is that key's values: exact but for their weight's rounding over
    itself, 2^-11 at most with bf16 rows, which bf16 does not show, and 2^-20 with fp32 rows; lse is the score."""
    r = np.random.default_rng(1)
    B, H, length = 6, 2, [S, S, S - 7, S, S - 3, S]
    ahead = [0, S // 2, S - 8, 17, S - 4, S - 1]                      # in the first step, on the way, in the last one
    ref = filled(B, H, S, D, 64, 5)
    ref.ks[:] = 1.0
    c = r.integers(8, 28, (B, H, S)).astype(float)
    for b in range(B):
        c[b, :, ahead[b]] = 30.0 if b % 2 == 0 else 4.0
    ref.k[:] = encode(c)[..., None]
    q = queries(B, H * G, 1, D, dtype, 3)                             # the last row of each head of keys stays an ordinary one
    sizes = r.permutation(np.resize([20, 24, 26, 28, 30, 31, 33, 36, 40, 50, 60], B * H * G)).reshape(B, H, G)
    for b in range(B):
        for h in range(H):
            for g in range(G):
                if g < G - 1 or G == 1:
                    q[b, h * G + g] = 2.0 ** int(sizes[b, h, g]) * (1 if b % 2 == 0 else -1)
    o, lse = ctx.kv8_decode(q, device_cache(ref), kv_len=ints(length))
    o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
    want, want_lse, *rest = ref.decode(q.double().cpu().numpy(), kv_len=length)
    to, tl = decode_tolerances(want, want_lse, *rest, dtype == "bf16")
    for b in range(B):
        for h in range(H):
            for g in range(G):
                row = h * G + g
                if g < G - 1 or G == 1:
                    v = VALUES[ref.v[b, h, ahead[b]]] * ref.vs[b, h, ahead[b] // 64]
                    assert (np.abs(o[b, row, 0] - v) <= (0.0 if dtype == "bf16" else 2.0 ** -20) * np.abs(v)).all(), (b, row, sizes[b, h, g])
                    score = c[b, h, ahead[b]] * float(q[b, row, 0, 0]) * D ** 0.5
                    assert abs(lse[b, row, 0] - score) <= 2.0 ** -17 * abs(score), (b, row, sizes[b, h, g])
                else:
                    assert (np.abs(o[b, row] - want[b, row]) <= to[b, row]).all() and abs(lse[b, row, 0] - want_lse[b, row, 0]) <= tl[b, row, 0]

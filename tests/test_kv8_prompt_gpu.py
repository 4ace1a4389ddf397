"""A prompt's chunk over an 8-bit cache that already holds tokens, read back for the forward: what the forward takes (a key's head for
each head of queries, one causal line for all sequences) and the mask that says the rest."""
import numpy as np
import pytest
import torch

from test_kv8_gpu import device_cache, filled, ints, queries

pytestmark = pytest.mark.gpu


def chunk_mask(kv_len, new_len, n, capacity):
    """1 where key j is at or before the place of new token i of its sequence, [B, n, capacity]."""
    at = (kv_len - new_len)[:, None] + torch.arange(n, device="cuda")
    there = torch.arange(n, device="cuda")[None] < new_len[:, None]
    return ((torch.arange(capacity, device="cuda") <= at[..., None]) & there[..., None]).float()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,H,G,n,S,D", [(3, 2, 4, 100, 400, 64), (4, 1, 2, 33, 257, 128), (2, 2, 1, 64, 300, 32)])
def test_sequences_of_different_lengths_and_shared_heads(ctx, B, H, G, n, S, D, dtype):
    """The forward's own bounds beside the same call of the decode: 2e-3 and a step of bf16 for each of them, lse 2e-3."""
    ref = filled(B, H, S, D, 64, 3, spread=2.0)
    cache = device_cache(ref)
    kv_len, new_len = [S, n + 7, S - 90, n][:B], [n, n, n - 5, n][:B]
    q = queries(B, H * G, n, D, dtype, 4, 0.5)
    kl, nl = ints(kv_len), ints(new_len)
    want, want_lse = ctx.kv8_decode(q, cache, kv_len=kl, new_len=nl)
    kk, vv = (t.repeat_interleave(G, 1) for t in ctx.kv8_read(cache, kv_len=kl, dtype=q.dtype))
    o, lse = ctx.attn_fwd(q, kk, vv, keep_mask=chunk_mask(kl, nl, n, S))
    there = np.arange(n)[None] < np.array(new_len)[:, None]
    for b in range(B):
        i = torch.from_numpy(there[b]).cuda()
        a, w = o[b, :, i].float(), want[b, :, i].float()
        assert ((a - w).abs() <= 4e-3 * ref.values()[1].std() + 4e-3 + 2.0 ** -7 * w.abs()).all()
        assert (lse[b, :, i] - want_lse[b, :, i]).abs().max() < 4e-3
        assert (o[b, :, ~i] == 0).all() and (want[b, :, ~i] == 0).all() and torch.isinf(want_lse[b, :, ~i]).all()


def test_equal_lengths_need_no_mask(ctx):
    """Where all sequences are as long as the keys that are read, the causal line is the forward's."""
    B, H, n, S, D = 2, 3, 50, 200, 64
    cache = device_cache(filled(B, H, S, D, 64, 3, spread=2.0))
    q = queries(B, H, n, D, "bf16", 4, 0.5)
    length = 150
    want, want_lse = ctx.kv8_decode(q, cache, kv_len=ints([length] * B))
    kk, vv = ctx.kv8_read(cache, count=length)
    o, lse = ctx.attn_fwd(q, kk, vv, causal=True)
    assert ((o.float() - want.float()).abs() <= 8e-3 + 2.0 ** -7 * want.float().abs()).all()
    assert (lse - want_lse).abs().max() < 4e-3

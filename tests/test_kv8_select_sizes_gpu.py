"""Selection from few and from very many blocks: where one CTA searches and where a cluster (or a CTA that is a cluster of its own)
does, on both sides of the line between them and up to the most blocks that there is room for.  Scores are whole numbers, so that the
choice is equal to a stable sort's."""
import pytest
import torch

import cuda_ltc_b200 as ltc

pytestmark = pytest.mark.gpu


def a_cache(pairs, blocks, D, seed):
    """Bounds and scales only: one key, seen as all of them."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    code = torch.zeros((1, 1, 1, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).expand(pairs, 1, blocks * 16, D)
    lo = torch.randint(-100, 1, (pairs, 1, blocks, D), device="cuda", generator=g, dtype=torch.int8)
    hi = torch.randint(0, 100, (pairs, 1, blocks, D), device="cuda", generator=g, dtype=torch.int8)
    scale = torch.ones((pairs, 1, blocks), device="cuda")
    q = torch.randint(-127, 128, (pairs, 2, 1, D), device="cuda", generator=g).float()
    q[..., 0] = 127.0                                                 # a step of one
    return ltc.Kv8Cache(code, code, scale, scale, torch.stack([lo, hi], 3), 16), q


def by_sorting(cache, q, live, count, ends):
    """ends: how many of the first and of the last are taken whatever their scores are."""
    lo, hi = cache.bounds[:, 0, :live, 0].float(), cache.bounds[:, 0, :live, 1].float()
    best = torch.full(lo.shape[:2], -float("inf"), device="cuda")
    for g in range(q.shape[1]):
        row = q[:, g, 0, None]
        best = torch.maximum(best, torch.maximum(row * lo, row * hi).sum(2))     # whole numbers below 2^24
    if ends:
        best[:, :ends] = best[:, live - ends:] = float("inf")
    return torch.sort(torch.sort(best, dim=1, descending=True, stable=True)[1][:, :count], dim=1)[0]


@pytest.mark.parametrize("count,ends", [(1, 0), (300, 1), (2500, 3)])
@pytest.mark.parametrize("pairs,blocks,D", [(1, 4095, 64), (1, 4096, 64), (1, 4097, 64), (9, 4096, 32), (9, 4099, 32), (300, 4096, 32), (300, 4200, 32),
                                            (2, 16384, 128), (3, 16385, 64), (1, 49152 * 16 - 5, 32), (1, 49152 * 16, 32)])
def test_both_searches(ctx, pairs, blocks, D, count, ends):
    cache, q = a_cache(pairs, blocks, D, blocks)
    for short in (0, 31):
        n = torch.full((pairs,), (blocks - short) * 16, dtype=torch.int32, device="cuda")
        got = ctx.kv8_select(q, cache, n, count, first=ends, last=ends)
        assert torch.equal(got[:, 0].long(), by_sorting(cache, q, blocks - short, count, ends))


def test_equal_scores_take_the_first(ctx):
    for blocks in (4096, 4097, 20000):
        cache, q = a_cache(2, blocks, 32, 1)
        cache.bounds[:] = cache.bounds[:, :, :1]
        got = ctx.kv8_select(q, cache, None, 77, first=0, last=1)
        assert got[:, 0].tolist() == [list(range(76)) + [blocks - 1]] * 2


def test_more_blocks_than_there_is_room_for(ctx):
    cache, q = a_cache(1, 49152 * 16 + 1, 32, 1)
    with pytest.raises(ltc.LtcaError, match="too many"):
        ctx.kv8_select(q, cache, None, 4)

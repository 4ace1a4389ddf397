"""The 8-bit key/value cache in numpy, from its definition and in 64 bits: what the kernels' results are compared with."""
import numpy as np


def _table():
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[127] = np.nan
    return np.concatenate([v, -v])


VALUES = _table()                                   # of the 256 codes
_MIDS = (VALUES[:126] + VALUES[1:127]) / 2


def encode(x):
    """Codes of the e4m3 values nearest to x (64 bits), ties to the even code, saturating; NaN is 127."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(x)
    i = np.searchsorted(_MIDS, a, side="left")
    tie = (i < 126) & (a == _MIDS[np.minimum(i, 125)])
    i = np.where(tie & (i % 2 == 1), i + 1, i)
    c = np.where(np.signbit(x), i + 128, i)
    return np.where(np.isnan(x), 127, c).astype(np.uint8)


def pow2_down_to(x, top, e_max):
    """Exponent of the smallest power of two, from 2^-100 on, by which the largest finite magnitude comes down to top."""
    a = np.abs(np.asarray(x, dtype=np.float64))
    a = a[np.isfinite(a)]
    amax = a.max() if a.size else 0.0
    e = -100
    while e < e_max and amax > top * 2.0 ** e:
        e += 1
    return e


class Cache:
    """codes [B,H,S,D] uint8, scales [B,H,nb], bounds [B,H,nb,2,D] int8."""

    def __init__(self, k, v, ks, vs, bounds, block):
        self.k, self.v, self.ks, self.vs, self.block = k, v, ks, vs, block
        self.bounds = bounds

    @classmethod
    def empty(cls, B, H, S, D, block, fill=0):
        nb = -(-S // block)
        codes = lambda: np.full((B, H, S, D), fill, dtype=np.uint8)  # noqa: E731
        return cls(codes(), codes(), np.ones((B, H, nb)), np.ones((B, H, nb)), np.zeros((B, H, nb, 2, D), np.int8), block)

    def copy(self):
        return Cache(self.k.copy(), self.v.copy(), self.ks.copy(), self.vs.copy(), self.bounds.copy(), self.block)

    def append(self, k, v, kv_len, new_len=None):
        B, H, n, D = k.shape
        S, bs = self.k.shape[2], self.block
        for b in range(B):
            m = n if new_len is None else min(max(int(new_len[b]), 0), n)
            first = int(kv_len[b]) - m
            lo, hi = max(first, 0), min(int(kv_len[b]), S)
            for j in range(lo // bs, -(-hi // bs)) if lo < hi else ():
                r0, r1 = max(lo, j * bs), min(hi, (j + 1) * bs)
                for h in range(H):
                    for x, codes, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                        new = x[b, h, r0 - first:r1 - first].astype(np.float64)
                        s = 2.0 ** pow2_down_to(new, 448.0, 120)
                        if r0 > j * bs:
                            old = scale[b, h, j]
                            s = max(s, old)
                            if s > old:
                                codes[b, h, j * bs:r0] = encode(VALUES[codes[b, h, j * bs:r0]] * (old / s))
                        scale[b, h, j] = s
                        codes[b, h, r0:r1] = encode(np.clip(new / s, -448, 448))
                    live = VALUES[self.k[b, h, j * bs:r1]]
                    self.bounds[b, h, j, 0] = np.floor(np.where(np.isnan(live), -448.0, live).min(0) / 4)
                    self.bounds[b, h, j, 1] = np.ceil(np.where(np.isnan(live), 448.0, live).max(0) / 4)

    def values(self):
        at = np.arange(self.k.shape[2]) // self.block
        return VALUES[self.k] * self.ks[:, :, at, None], VALUES[self.v] * self.vs[:, :, at, None]

    def decode(self, q, kv_len=None, new_len=None, scale=None, causal=True, keep_mask=None, clamp=0.0, blocks=None):
        """out, lse and, for each row, a bound on |scale| sum |q k| over its keys and the number of its keys."""
        B, Hq, Sq, D = q.shape
        H, S = self.k.shape[1:3]
        scale = D ** -0.5 if scale is None else scale
        k, v = self.values()
        o, lse = np.zeros((B, Hq, Sq, D)), np.full((B, Hq, Sq), -np.inf)
        size, keys, most = np.zeros((B, Hq, Sq)), np.zeros((B, Hq, Sq)), np.zeros((B, Hq, Sq))
        for b in range(B):
            length = S if kv_len is None else int(kv_len[b])
            n = Sq if new_len is None else min(max(int(new_len[b]), 0), Sq)
            for hq in range(Hq):
                h = hq // (Hq // H)
                if blocks is None:
                    at = np.arange(S)
                else:
                    nb = -(-S // self.block)
                    at = np.concatenate([np.arange(j * self.block, min((j + 1) * self.block, S))
                                         for j in blocks[b, h] if 0 <= j < nb] + [np.zeros(0, int)]).astype(int)
                for i in range(n):
                    seen = at < length
                    if causal:
                        seen &= at <= length - n + i
                    if keep_mask is not None:
                        seen &= keep_mask[b, i, at] != 0
                    j = at[seen]
                    if j.size == 0:
                        continue
                    row = q[b, hq, i].astype(np.float64)
                    s = scale * (k[b, h, j] @ row)
                    if clamp > 0:
                        s = np.minimum(s, clamp)
                    m = s.max()
                    p = np.exp(s - m)
                    o[b, hq, i] = p @ v[b, h, j] / p.sum()
                    lse[b, hq, i] = m + np.log(p.sum())
                    size[b, hq, i] = scale * (np.abs(k[b, h, j]) @ np.abs(row)).max()
                    size[b, hq, i] += scale * D * 2.0 ** -4 * np.abs(row).max() * np.abs(k[b, h, j]).max()
                    keys[b, hq, i], most[b, hq, i] = j.size, np.abs(v[b, h, j]).max()
        return o, lse, size, keys, most

    def select(self, q, kv_len, count, new_len=None, first=1, last=1):
        B, Hq, Sq, D = q.shape
        H, S = self.k.shape[1:3]
        out = np.full((B, H, count), -1, dtype=np.int32)
        for b in range(B):
            blocks = -(-min(max(S if kv_len is None else int(kv_len[b]), 0), S) // self.block)
            n = Sq if new_len is None else min(max(int(new_len[b]), 0), Sq)
            for h in range(H):
                score = [-np.inf] * blocks
                for g in range(Hq // H):
                    for i in range(n):
                        row = q[b, h * (Hq // H) + g, i].astype(np.float64)
                        step = 2.0 ** pow2_down_to(row, 127.0, 121)
                        whole = np.clip(np.round(np.where(np.isnan(row), 0.0, row) / step), -127, 127).astype(np.int64)
                        lo, hi = (self.bounds[b, h, :blocks, x].astype(np.int64) for x in (0, 1))
                        sums = np.maximum(whole * lo, whole * hi).sum(1)
                        score = [max(a, int(x) * step * self.ks[b, h, j]) for j, (a, x) in enumerate(zip(score, sums))]
                for j in range(blocks):
                    if j < first or j >= blocks - last:
                        score[j] = np.inf
                best = sorted(sorted(range(blocks), key=lambda j: (-score[j], j))[:count])
                out[b, h, :len(best)] = best
        return out


def decode_tolerances(o, lse, size, keys, most, bf16):
    """How far out and lse may be from 64 bits on the same codes.

    A score: q in 22 bits (two fp16 terms; bf16's 8 fit one), each term no finer than 2^-25 of the row's largest (the second
    part of `size`, whose 2^-4 makes 2^-24 of it per channel), products exact, at most D/16 + 8 fp32 roundings of 2^-23 of the
    partial sums: 2^-19 of `size` covers them.  The weights move by that much relatively, the result by twice that times the
    largest value; exponentials add 2^-21, the sums over the keys one fp32 rounding for each 8 of them.  With bf16 results the
    weights have fp16's 11 bits (2^-11) and the result half a step of bf16 (2^-8)."""
    ds = size * 2.0 ** -19
    sums = (keys / 8 + 64) * 2.0 ** -23
    to = most * (2 * ds + 2.0 ** -20 + sums + (2.0 ** -11 if bf16 else 0.0))
    to = to[..., None] + (2.0 ** -8 if bf16 else 2.0 ** -23) * np.abs(o) + 1e-37
    return to, ds + 2.0 ** -20 + sums + 2.0 ** -22 * np.abs(np.where(np.isfinite(lse), lse, 0.0))

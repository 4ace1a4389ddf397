"""The table that tells the 8-bit decode's joining kernel which warps have shares of a unit: an entry that was never written becomes
neither an address nor a number of turns.  No GPU needed."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_ltc_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "kv8_shares.h"
int main() {
    const int32_t odd[] = {INT32_MIN, INT32_MIN + 1, -2000000000, -3, -1, 0, 1, 2, 5, 6, 7, 8, 100, 2367, 2368, 2369, 1 << 20, 0x3f800000,
                           0x7fc00000, INT32_MAX - 1, INT32_MAX};
    const int32_t sizes[] = {0, 1, 2, 7, 8, 2368, INT32_MAX};
    int wrong = 0, taken = 0;
    for (int32_t first : odd)
        for (int32_t more : odd)
            for (int32_t warps : sizes) {
                // in 64 bits: both are numbers of warps, and the last of them is one
                const bool want = first >= 0 && more >= 0 && (int64_t)first + more < warps;
                const bool got = ltca::shares_are_there(first, more, warps);
                wrong += want != got;
                taken += got;
            }
    printf("%d %d\n", wrong, taken);
}
"""


def test_only_warps_that_there_are(tmp_path):
    src = tmp_path / "s.cpp"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-fsanitize=undefined", "-I", CSRC, str(src), "-o", str(tmp_path / "s")])
    wrong, taken = map(int, subprocess.check_output([str(tmp_path / "s")]).split())
    assert wrong == 0 and taken > 50


def test_the_join_asks_before_it_forms_an_address():
    with open(os.path.join(CSRC, "kv8_decode.cu")) as f:
        text = f.read()
    join = text[text.index("kv8_decode_join_kernel("):text.index("struct Plan")]
    read, asked = join.index("a.shares["), join.index("shares_are_there(who.x, who.y, a.warps)")
    used = [m.start() for m in re.finditer(r"who\.[xy]", join) if not asked <= m.start() <= asked + 60]
    assert read < asked < min(used)


def _workspace(B, H, G, Sq, S, D, dtype, n_blocks=0):
    import ctypes as C
    from cuda_ltc_b200 import _lib
    c = _lib.Kv8CacheParams(B=B, H=H, S=S, D=D, block=64)
    p = _lib.Kv8DecodeParams(Hq=H * G, Sq=Sq, dtype=dtype, scale=1.0)
    if n_blocks:
        p.blocks, p.n_blocks = 256, n_blocks
    n = C.c_size_t()
    assert _lib.load().ltca_kv8_decode_workspace_bytes(C.byref(c), C.byref(p), C.byref(n)) == 0
    return n.value


def test_scratch_is_what_the_header_says():
    """W R (D + 4) 8 bytes for at most W = 1184 .. 2368 warps and R rows of a tile, and 8 for each head of keys and tile of 8 or 16 rows;
    both in pieces of 256."""
    seen = []
    for D in (32, 64, 128):
        for rows in ((1, 1), (3, 2), (8, 1), (4, 4), (5, 7), (16, 64)):
            for B, H, S in ((1, 1, 1), (1, 8, 100000), (300, 2, 64), (16, 8, 32768), (4096, 8, 1024), (1, 1, 1 << 30)):
                for dtype in (0, 1):
                    R = rows[0] * rows[1]
                    n = _workspace(B, H, *rows, S, D, dtype)
                    tiles = -(-R // (8 if R <= 8 else 16))
                    warps = 1184 if R > 8 and D == 128 else 1776 if R > 8 or D == 128 else 2368
                    most = warps * min(R, 8 if R <= 8 else 16) * (D + 4) * 8
                    assert n <= most + 256 + B * H * tiles * 8 + 256, (D, rows, B, H, S, n)
                    if S * B > 300000:
                        assert n >= most, (D, rows, B, H, S, n)
                    seen.append(n)
    assert min(seen) == 0
    assert 6.5e5 < _workspace(16, 8, 1, 1, 32768, 32, 1) < 7.5e5 and 2.0e7 < _workspace(16, 8, 16, 1, 32768, 128, 1) < 2.1e7


def test_four_times_a_score_bounds_the_products():
    """What the selection's score says of a block: its bounds are quarters of codes.  Blocks of different keys, whose bounds no single key
    reaches, and one block of 16 equal keys along the query, which the score itself does not bound."""
    import numpy as np
    import kv8_ref
    r = np.random.default_rng(0)
    B, H, S, D, block = 1, 1, 320, 64, 16
    ref = kv8_ref.Cache.empty(B, H, S, D, block)
    k = r.standard_normal((B, H, S, D)).astype(np.float32)
    q = r.standard_normal(D)
    k[:, :, -block:] = q * 100
    ref.append(k, k, [S])
    step = 2.0 ** kv8_ref.pow2_down_to(q, 127.0, 121)
    whole = np.round(q / step)
    keys = ref.values()[0][0, 0].reshape(-1, block, D)
    for j in range(S // block):
        lo, hi = ref.bounds[0, 0, j].astype(float)
        score = np.maximum(whole * lo, whole * hi).sum() * ref.ks[0, 0, j] * step
        most, rounding = (keys[j] @ q).max(), 0.5 * step * np.abs(keys[j]).sum(1).max()
        assert most <= 4 * score + rounding
    assert most > score + rounding

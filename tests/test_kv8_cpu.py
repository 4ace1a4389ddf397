"""The 8-bit cache's C ABI without a GPU: struct layouts, the size query, and what the entry points refuse before they touch
a device (a zeroed block stands for a context there: the checks write their text into it and nothing else)."""
import ctypes as C
import os
import subprocess
import textwrap

import numpy as np
import pytest

import kv8_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from cuda_ltc_b200.build import build_library
    build_library()
    from cuda_ltc_b200 import _lib
    return _lib.load()


def _strides(H, S, D):
    from cuda_ltc_b200 import _lib
    return _lib.Strides(H * S * D, S * D, D)


def _cache(**kw):
    from cuda_ltc_b200 import _lib
    c = _lib.Kv8CacheParams(B=2, H=4, S=100, D=64, block=32, k=4096, v=8192, k_scale=64, v_scale=64, bounds=64)
    c.k_strides = c.v_strides = _strides(4, 100, 64)
    for k, v in kw.items():
        if k in ("k_seq", "v_head"):
            setattr(getattr(c, k[0] + "_strides"), k[2:], v)
        else:
            setattr(c, k, v)
    return c


def _calls():
    """name: (parameter class, valid fields)"""
    from cuda_ltc_b200 import _lib
    st = _strides(4, 8, 64)
    q = dict(Hq=8, Sq=1, dtype=1, q=64, q_strides=st)
    return {
        "ltca_kv8_append": (_lib.Kv8AppendParams, dict(n=8, dtype=1, k=64, v=64, k_strides=st, v_strides=st, kv_len=64)),
        "ltca_kv8_read": (_lib.Kv8ReadParams, dict(start=10, n=8, dtype=1, k=64, v=64, k_strides=st, v_strides=st)),
        "ltca_kv8_decode": (_lib.Kv8DecodeParams, dict(q, o=64, o_strides=st, scale=0.125)),
        "ltca_kv8_select": (_lib.Kv8SelectParams, dict(q, count=4, first=1, last=1, blocks=64)),
    }


def test_struct_layouts_match_the_header(tmp_path):
    from cuda_ltc_b200 import _lib
    names = {"ltca_kv8_cache": _lib.Kv8CacheParams, "ltca_kv8_append_params": _lib.Kv8AppendParams,
             "ltca_kv8_read_params": _lib.Kv8ReadParams, "ltca_kv8_decode_params": _lib.Kv8DecodeParams,
             "ltca_kv8_select_params": _lib.Kv8SelectParams}
    lines, want = [], []
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(C.sizeof(py))
        for f, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(py, f).offset)
    src = tmp_path / "s.c"
    src.write_text(textwrap.dedent('#include <stdio.h>\n#include "ltc_attn.h"\nint main(void) {\n%s\nreturn 0; }\n') % "\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    assert list(map(int, subprocess.check_output([str(tmp_path / "s")]).split())) == want


BAD_CACHES = [
    (dict(B=0), -1, b"shape"), (dict(H=0), -1, b"shape"), (dict(S=0), -1, b"shape"), (dict(S=2 ** 30 + 1), -2, b"capacity"), (dict(D=48), -2, b"head_dim"),
    (dict(D=256), -2, b"head_dim"), (dict(block=8), -2, b"tokens"), (dict(block=48), -2, b"tokens"),
    (dict(bounds=72), -1, b"bounds"), (dict(B=1 << 20, H=1 << 12), -1, b"B * H"),
]
BAD_CALLS = [
    ("ltca_kv8_append", dict(n=-1), {}, -1, b"negative"), ("ltca_kv8_append", dict(dtype=2), {}, -1, b"dtype"),
    ("ltca_kv8_append", dict(kv_len=None), {}, -1, b"kv_len"), ("ltca_kv8_append", dict(v=None), {}, -1, b"needs"),
    ("ltca_kv8_append", {}, dict(k=None), -1, b"null"), ("ltca_kv8_append", {}, dict(v_scale=None), -1, b"null"),
    ("ltca_kv8_append", {}, dict(k=4104), -1, b"16-byte"), ("ltca_kv8_append", {}, dict(k_seq=72), -1, b"16-byte"),
    ("ltca_kv8_append", {}, dict(v_head=0), -1, b"share memory"),
    ("ltca_kv8_read", dict(start=-1), {}, -1, b"range"), ("ltca_kv8_read", dict(start=93), {}, -1, b"range"),
    ("ltca_kv8_read", dict(n=2 ** 31 - 1), {}, -1, b"range"), ("ltca_kv8_read", dict(k=None), {}, -1, b"null"),
    ("ltca_kv8_read", dict(dtype=-1), {}, -1, b"dtype"),
    ("ltca_kv8_decode", dict(Hq=6), {}, -1, b"heads"), ("ltca_kv8_decode", dict(Hq=0), {}, -1, b"heads"),
    ("ltca_kv8_decode", dict(Sq=0), {}, -1, b"no queries"), ("ltca_kv8_decode", dict(scale=0.0), {}, -1, b"scale"),
    ("ltca_kv8_decode", dict(scale=float("nan")), {}, -1, b"scale"), ("ltca_kv8_decode", dict(o=None), {}, -1, b"null"),
    ("ltca_kv8_decode", dict(blocks=64, n_blocks=0), {}, -1, b"empty list"),
    ("ltca_kv8_decode", dict(workspace=64), {}, -1, b"256-byte"), ("ltca_kv8_decode", dict(Sq=1 << 20), {}, -2, b"rows"),
    ("ltca_kv8_decode", {}, dict(v=None), -1, b"null"),
    ("ltca_kv8_select", dict(count=0), {}, -1, b"blocks"), ("ltca_kv8_select", dict(first=3, last=2), {}, -1, b"blocks"),
    ("ltca_kv8_select", dict(first=-1), {}, -1, b"blocks"), ("ltca_kv8_select", dict(blocks=None), {}, -1, b"null"),
    ("ltca_kv8_select", {}, dict(bounds=None), -1, b"keeps bounds"), ("ltca_kv8_select", dict(q=None), {}, -1, b"null"),
]


def _refused(lib, name, cache, fields):
    params, valid = _calls()[name]
    ctx = C.create_string_buffer(1 << 14)
    rc = getattr(lib, name)(C.addressof(ctx), C.byref(cache), C.byref(params(**{**valid, **fields})))
    return rc, lib.ltca_last_error(C.addressof(ctx))


@pytest.mark.parametrize("name", ["ltca_kv8_append", "ltca_kv8_read", "ltca_kv8_decode", "ltca_kv8_select"])
def test_bad_caches_are_refused(lib, name):
    for fields, code, text in BAD_CACHES:
        rc, err = _refused(lib, name, _cache(**fields), {})
        assert rc == code and text in err, (fields, rc, err)
    params, valid = _calls()[name]
    p = params(**valid)
    ctx = C.create_string_buffer(1 << 14)
    assert getattr(lib, name)(None, C.byref(_cache()), C.byref(p)) == -1
    assert getattr(lib, name)(C.addressof(ctx), None, C.byref(p)) == -1
    assert getattr(lib, name)(C.addressof(ctx), C.byref(_cache()), None) == -1


@pytest.mark.parametrize("case", BAD_CALLS, ids=lambda c: "-".join([c[0][9:], *c[1], *c[2]]))
def test_bad_calls_are_refused(lib, case):
    name, fields, cache, code, text = case
    rc, err = _refused(lib, name, _cache(**cache), fields)
    assert rc == code and text in err, (rc, err)


def test_nothing_to_do_is_no_error(lib):
    assert _refused(lib, "ltca_kv8_append", _cache(), dict(n=0, k=None, v=None))[0] == 0
    assert _refused(lib, "ltca_kv8_read", _cache(), dict(n=0, k=None, v=None))[0] == 0


def test_size_query_takes_any_arguments(lib):
    from cuda_ltc_b200 import _lib
    n = C.c_size_t(1)
    q = lambda c, **kw: lib.ltca_kv8_decode_workspace_bytes(C.byref(c), C.byref(_lib.Kv8DecodeParams(  # noqa: E731
        **{**_calls()["ltca_kv8_decode"][1], **kw})), C.byref(n))
    assert q(_cache()) == 0
    for bad in (dict(Hq=0), dict(Hq=5), dict(Sq=0), dict(Sq=-5), dict(dtype=7)):
        assert q(_cache(), **bad) == 0 and n.value == 0
    assert q(_cache(B=0)) == 0 and n.value == 0
    assert lib.ltca_kv8_decode_workspace_bytes(None, None, C.byref(n)) == -1


def test_reference_rounds_to_the_nearest_code():
    """Half a step of e4m3 is 2^-4 of the value (2^-10 for the smallest); ties go to the even code; 448 is the last."""
    x = np.concatenate([np.linspace(-500, 500, 20001), np.random.default_rng(0).standard_normal(10000) * 2.0 ** -8])
    y = kv8_ref.VALUES[kv8_ref.encode(x)]
    assert (np.abs(y - np.clip(x, -448, 448)) <= np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** -10)).all()
    assert kv8_ref.encode([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 449.0, 1e9]).tolist() == [
        kv8_ref.encode(16.0), kv8_ref.encode(20.0), 0, 2, 126, 126]
    import torch
    t = torch.from_numpy(x).float().clamp(-448, 448).to(torch.float8_e4m3fn)
    assert np.array_equal(kv8_ref.encode(x.astype(np.float32)), t.view(torch.uint8).numpy())

"""Pointers between two elements: the 8-bit cache's entry points refuse them before they touch a device, where a kernel would fault.
No GPU needed."""
import pytest

from test_kv8_cpu import _cache, _refused, lib  # noqa: F401


def _cases():
    words = dict(ltca_kv8_append=["kv_len", "new_len"], ltca_kv8_read=["kv_len"],
                 ltca_kv8_decode=["lse", "keep_mask", "kv_len", "new_len", "blocks"], ltca_kv8_select=["kv_len", "new_len", "blocks"])
    tensors = dict(ltca_kv8_append=["k", "v"], ltca_kv8_read=["k", "v"], ltca_kv8_decode=["q", "o"], ltca_kv8_select=["q"])
    for name in words:
        for f in words[name]:
            for by in (1, 2, 3):
                more = dict(n_blocks=2) if name == "ltca_kv8_decode" else {}
                yield name, {f: 64 + by, **more}, {}, b"4-byte"
        for f in tensors[name]:
            yield name, {f: 65}, {}, b"elements (2"                   # bf16
            for by in (1, 2, 3):
                yield name, {f: 64 + by, "dtype": 0}, {}, b"elements (4"
        for f in ("k_scale", "v_scale"):
            yield name, {}, {f: 66}, b"4-byte"


@pytest.mark.parametrize("case", list(_cases()), ids=lambda c: "-".join([c[0][9:], *map(str, {**c[1], **c[2]}.items())]))
def test_pointers_between_elements_are_refused(lib, case):  # noqa: F811
    name, fields, cache, text = case
    rc, err = _refused(lib, name, _cache(**cache), fields)
    assert rc == -1 and text in err, (rc, err)

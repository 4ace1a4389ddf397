"""Source-level rule of kernels whose waits are bounded: what a wait reads in shared memory (its barrier, the block's abort word) is
set by one thread or a few and read by others, so that a barrier of the whole block stands between the two.  No GPU needed."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_ltc_b200", "csrc")


def _kernels():
    """(kernel, body) of every __global__ function that sets up a barrier."""
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__\s+void\b", text):
            i = text.index("{", m.end())
            depth, j = 1, i + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[j], 0)
                j += 1
            if "mbar_init(" in text[i:j]:
                yield re.search(r"(\w+_kernel)\s*\(", text[m.end():i]).group(1), text[i + 1:j - 1]


KERNELS = dict(_kernels())


def _outermost(body):
    """The body with everything inside braces blanked out."""
    out, depth = [], 0
    for ch in body:
        depth -= ch == "}"
        out.append(ch if depth == 0 else " ")
        depth += ch == "{"
    return "".join(out)


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_barriers_and_abort_words_are_set_before_the_block_goes_on(name):
    body = KERNELS[name]
    set_up = max(m.end() for m in re.finditer(r"mbar_init\(|\babort\w* = 0|_abort = 0", body))
    used = min(m.start() for m in re.finditer(r"mbar_wait\w*\(|mbar_try_wait\(|mbar_arrive\w*\(|tma_load\w*\(", body))
    assert set_up < used
    # a barrier that every thread reaches, whatever the arguments are
    assert re.search(r"__syncthreads\(\);", _outermost(body)[set_up:used]), name


def test_the_rule_sees_the_kernels():
    assert {"kv8_decode_kernel", "attn_fwd_sm100_kernel", "gemm_bf16_sm100_kernel"} <= set(KERNELS)

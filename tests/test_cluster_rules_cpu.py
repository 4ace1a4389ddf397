"""Source-level rule: the opt-in to clusters of more than eight CTAs stands where a file's largest cluster needs it, and nowhere else.
No GPU needed."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_ltc_b200", "csrc")


def test_wide_clusters_are_opted_into_where_they_occur():
    seen = {}
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        largest = [int(n) for n in re.findall(r"constexpr int kMax\w*Cluster = (\d+)", text)]
        if largest:
            seen[name] = max(largest)
            assert ("cudaFuncAttributeNonPortableClusterSizeAllowed" in text) == (max(largest) > 8), name
    assert seen == {"attn_decode.cu": 16, "kv8_decode.cu": 8, "kv8_select.cu": 16}

"""Refusals of the cache operators at the ends of their ranges, where buffers
meet, and what their workspace queries look at.  No GPU needed."""
import pytest
from test_cache_ops import ARG, refused


@pytest.mark.parametrize("call", ["prompt", "tree", "weights"])
@pytest.mark.parametrize("kw,text", [(dict(cap=2.4e38), "cap"), (dict(cap=3.4e38), "cap"), (dict(cap=2.0 ** 126 * 1.01), "cap"),
                                     (dict(scale=2.4e38), "scale"), (dict(scale=1e-39), "scale"), (dict(cap=1e-45), "cap")])
def test_scores_out_of_range(call, kw, text):
    """Factors whose product with log2(e), or whose reciprocal, fp32 does not hold."""
    refused(call, ARG, text, **kw)


@pytest.mark.parametrize("call", ["prompt", "tree", "weights"])
@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** 126])
def test_scores_at_the_ends(call, size):
    refused(call, ARG, "null context", cap=size, scale=size)


def test_prompt_query_rows():
    """2^29 query rows of a KV head are 2^22 tiles of 768 threads; twice as many pass a grid."""
    wide = dict(q_stride=1 << 18, out_stride=1 << 18, kv_heads=1, k_stride=128, v_stride=128, n=1 << 22)
    refused("prompt", ARG, "rows", heads=256, **wide)
    refused("prompt", ARG, "null context", heads=128, **wide)

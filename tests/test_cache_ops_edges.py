"""Refusals of the cache operators at the ends of their ranges, where buffers
meet, and what their workspace queries look at.  No GPU needed."""
import ctypes as C

import numpy as np
import pytest
from test_cache_ops import ARG, keep, prompt, refused

from rapidocrvl_amd import lib


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


def memory(at, outer, inner, blocks, rows, width):
    """The floats of `blocks` blocks of `rows` rows, by address / 4."""
    return {at + b * outer + r * inner + i for b in range(blocks) for r in range(rows) for i in range(width)}


def keep_answer(**kw):
    L = lib.load()
    rc = L.pocr_cache_keep(None, C.byref(keep(**kw)), None)
    assert rc == ARG
    return L.pocr_last_error().decode()


@pytest.mark.parametrize("seed", range(20))
@pytest.mark.parametrize("alike", [True, False], ids=["one-stride", "two-strides"])
def test_keep_overlap_of_interleaved_rows(seed, alike):
    """Source and destination anywhere in one pool: refused where they share memory and, strides being alike, only there."""
    rng = np.random.default_rng(seed)
    far = dict(v=1 << 30, v_out=1 << 31, kv_heads=1, head_dim=64, max_keep=3)
    for _ in range(40):
        caches, rows, rows_out = (int(x) for x in rng.integers(1, 5, 3))
        inner = 64 + 4 * int(rng.integers(0, 40))
        outer = max(4, rows * inner + 4 * int(rng.integers(-40, 200))) if rng.random() < 0.7 else 4 * int(rng.integers(1, 60))
        inner2, outer2 = (inner, outer) if alike else (64 + 4 * int(rng.integers(0, 40)), 4 * int(rng.integers(1, 300)))
        src, dst = 1 << 20, (1 << 20) + 4 * int(rng.integers(-500, 500))
        if src == dst:
            continue
        text = keep_answer(k=4 * src, k_out=4 * dst, caches=caches, max_rows=rows, max_rows_out=rows_out, k_cache_stride=outer,
                           k_stride=inner, k_out_cache_stride=outer2, k_out_stride=inner2, **far)
        a = memory(src, outer, inner, caches, rows, 64)
        b = memory(dst, outer2, inner2, caches, rows_out, 64)
        if a & b:
            assert "overlaps" in text
        elif alike or min(a) > max(b) or min(b) > max(a):
            assert "null context" in text


def test_keep_from_slot_to_slot():
    """A pool [layer][slot][row]: all layers of one slot into the next; then one row further, into the source's last."""
    slot = 100 * 256
    pool = {n: 4 * slot for n in ("k_cache_stride", "v_cache_stride", "k_out_cache_stride", "v_out_cache_stride")}
    for shift, text in ((0, "null context"), (-256, "overlaps")):
        refused("keep", ARG, text, k=1 << 30, k_out=(1 << 30) + 4 * (slot + shift), v=1 << 34, v_out=(1 << 34) + 8 * slot, **pool)


def test_keep_interleaved_side_buffers():
    """Weights of source and destination row by row in one buffer [cache][KV head][2][100]."""
    out = dict(k_out=1 << 30, v_out=1 << 31, side_stride=200, side_out_stride=200)
    refused("keep", ARG, "null context", weights=1 << 20, weights_out=(1 << 20) + 400, **out)
    refused("keep", ARG, "overlaps", weights=1 << 20, weights_out=(1 << 20) + 396, **out)


# K, V, weights and positions at places of their own, in place and elsewhere, and lists
APART = dict(k=1 << 30, v=1 << 31, k_out=1 << 30, v_out=1 << 31, rows=1 << 20, counts=1 << 21, first=1 << 22)
SIDES = dict(weights=1 << 23, weights_out=1 << 23, positions=1 << 24, positions_out=1 << 24)
ELSEWHERE = dict(k_out=1 << 32, v_out=1 << 33)
CACHE = 4 << 16  # bytes from cache to cache


def answer_behind_the_context(args, want):
    """The answer to a call with a context, which is never looked into: refused before the device, or the device's own error."""
    L = lib.load()
    if L.pocr_device_count() > 0:
        pytest.skip("a call that was not refused would run")
    ctx = C.create_string_buffer(4096)
    rc = L.pocr_cache_keep(C.cast(ctx, C.c_void_p), C.byref(args), None)
    msg = L.pocr_last_error().decode()
    assert rc == want, msg
    return msg


@pytest.mark.parametrize("kw,text", [
    (dict(v=1 << 30, v_out=1 << 30), "destination of K overlaps V"),
    (dict(v=(1 << 30) + 1024 * 99, v_out=(1 << 30) + 1024 * 99), "destination of K overlaps V"),
    (dict(v=(1 << 30) + 2 * CACHE, v_out=(1 << 30) + 2 * CACHE), "destination of K overlaps V"),
    (dict(SIDES, positions=1 << 23, positions_out=1 << 23), "destination of weights overlaps positions"),
    (dict(SIDES, weights=(1 << 31) + 64, weights_out=(1 << 31) + 64), "destination of V overlaps weights"),
    (dict(rows=(1 << 30) + 512), "destination of K overlaps rows"),
    (dict(counts=(1 << 31) + CACHE), "destination of V overlaps counts"),
    (dict(SIDES, first=(1 << 23) + 4 * 599), "destination of weights overlaps first"),
    (dict(ELSEWHERE, k_out=(1 << 31) + 1024 * 99), "destination of K overlaps V"),
    (dict(ELSEWHERE, v_out=(1 << 32) + CACHE), "destination of V overlaps K"),
    (dict(ELSEWHERE, v_out=1 << 32), "destination of V overlaps K"),  # two sources, one destination
    (dict(ELSEWHERE, **dict(SIDES, weights_out=1 << 25, positions_out=1 << 25)), "destination of positions overlaps weights")])
def test_keep_destinations_meet_nothing_else(kw, text):
    assert text in answer_behind_the_context(keep(**{**APART, **kw}), ARG)


@pytest.mark.parametrize("kw", [{}, SIDES, ELSEWHERE, dict(v=(1 << 30) + 1024 * 100, v_out=(1 << 30) + 1024 * 100),
                                dict(v=(1 << 30) + 512, v_out=(1 << 30) + 512, kv_heads=1), dict(ELSEWHERE, v=1 << 30, v_out=1 << 32)])
def test_keep_buffers_side_by_side(kw):
    """K and V behind each other in each cache, row by row, and one buffer as both."""
    answer_behind_the_context(keep(**{**APART, **kw}), lib.POCR_ERR_DEVICE)


def test_outputs_that_overlap_themselves():
    """Two sequences' or caches' rows in one place; rows that alternate are in places of their own."""
    refused("tree", ARG, "two sequences", out_seq_stride=2048 * 4)
    refused("tree", ARG, "two sequences", out_seq_stride=2044, out_stride=3 * 2048)
    refused("tree", ARG, "null context", out_seq_stride=2048 * 5)
    refused("tree", ARG, "null context", out_seq_stride=2048, out_stride=3 * 2048)


@pytest.mark.parametrize("kw", [dict(ELSEWHERE, k_out_cache_stride=256 * 99),
                                dict(ELSEWHERE, v_out_cache_stride=256, v_out_stride=512),
                                dict(k_cache_stride=256 * 99, k_out_cache_stride=256 * 99)])
def test_keep_caches_that_overlap(kw):
    assert "caches of the destination" in answer_behind_the_context(keep(**{**APART, **kw}), ARG)


@pytest.mark.parametrize("kw", [dict(ELSEWHERE, v_out_cache_stride=256, v_out_stride=768),
                                dict(k_cache_stride=256 * 100, k_out_cache_stride=256 * 100)])
def test_keep_caches_that_touch_or_alternate(kw):
    answer_behind_the_context(keep(**{**APART, **kw}), lib.POCR_ERR_DEVICE)


@pytest.mark.parametrize("shape", [dict(n=64, rows_before=9000), dict(n=300, rows_before=5000), dict(n=7, rows_before=5000),
                                   dict(n=2000, rows_before=100), dict(n=1, rows_before=0), dict(n=128, rows_before=8000)])
def test_prompt_workspace_of_shapes_alone(shape):
    """What the query names without pointers is enough with them, spans or none."""
    L = lib.load()
    need = L.pocr_prompt_attention_workspace(C.byref(prompt(q=None, k=None, v=None, out=None, workspace=None, **shape)))
    spans = dict(row_begin=4096, row_end=4096)
    assert L.pocr_prompt_attention_workspace(C.byref(prompt(**spans, **shape))) == need
    for kw in ({}, spans):
        refused("prompt", ARG, "null context", workspace_bytes=need, **kw, **shape)

"""The cache operators on the device against their definitions in 64 bits
(cache_ops_f64.py, with the derivation of the bounds)."""
import threading

import cache_ops_f64 as ref
import numpy as np
import pytest

from rapidocrvl_amd import lib

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32
SENTINEL = F32(-77.25)  # what untouched places hold


def alibi(heads):
    return np.array([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], F32)


def spans_of(kind, n, rows0, rng):
    """(begin, end) of n rows behind rows0, or None for plain causal rows."""
    rows, i = rows0 + n, np.arange(n)
    if kind == "causal":
        return None
    if kind == "prefix":
        p = max(1, (2 * n) // 3)
        return np.zeros(n, I32), np.where(i < p, rows0 + p, rows0 + i + 1).astype(I32)
    if kind == "docs":
        cuts = np.sort(rng.choice(np.arange(0, n + 1), min(4, n)))
        begin = np.array([max([0] + [rows0 + c for c in cuts if c <= t]) for t in i])
        return begin.astype(I32), (rows0 + i + 1).astype(I32)
    if kind == "window":
        return (rows0 + i - 20).astype(I32), (rows0 + i + 1).astype(I32)  # negative at the start: row 0
    if kind == "holes":  # every third row sees nothing, ends past the cache are cut to it
        b, e = rng.integers(0, rows, n), rng.integers(0, rows + 9, n)
        e = np.where(i % 3 == 1, b - rng.integers(0, 2, n) * 5, np.maximum(e, b + 1))
        return b.astype(I32), e.astype(I32)
    raise AssertionError(kind)


def visible(spans, n, rows0):
    rows = rows0 + n
    j, i = np.arange(rows), np.arange(n)[:, None]
    if spans is None:
        return j <= rows0 + i
    return (j >= np.maximum(spans[0], 0)[:, None]) & (j < np.minimum(spans[1], rows)[:, None])


def prompt_case(hip, rng, n, rows0, heads, kvh, hd, spans, cap=0.0, slopes=None, scale=0.0, pad=0, q=None, k=None, v=None):
    """Device buffers and arguments; row strides `pad` floats wider than the rows."""
    rows = rows0 + n
    q = rng.standard_normal((n, heads * hd + pad)).astype(F32) * 3 if q is None else q
    k = rng.standard_normal((rows, kvh * hd + pad)).astype(F32) * F32(0.64) if k is None else k
    v = rng.standard_normal((rows, kvh * hd + pad)).astype(F32) * F32(0.64) if v is None else v
    out = np.full((n, heads * hd + pad), SENTINEL, F32)
    a = lib.PromptArgs(q=hip.up(q), k=hip.up(k), v=hip.up(v), out=hip.up(out), lse=hip.up(np.zeros((n, heads), F32)),
                       row_begin=None if spans is None else hip.up(spans[0]),
                       row_end=None if spans is None else hip.up(spans[1]),
                       slopes=None if slopes is None else hip.up(slopes), n=n, rows_before=rows0, heads=heads, kv_heads=kvh,
                       head_dim=hd, scale=scale, cap=cap, q_stride=q.shape[1], k_stride=k.shape[1], v_stride=v.shape[1],
                       out_stride=out.shape[1])
    need = lib.prompt_attention_workspace(a)
    a.workspace, a.workspace_bytes = hip.raw(need), need
    return a, q, k, v


def check_prompt(hip, a, q, k, v, spans, slopes=None, rows=None):
    """All rows of the call, or those in `rows`, against the definition."""
    n, heads, kvh, hd, rows0 = a.n, a.heads, a.kv_heads, a.head_dim, a.rows_before
    out, lse = hip.down(a.out, (n, a.out_stride)), hip.down(a.lse, (n, heads))
    assert np.all(out[:, heads * hd:] == SENTINEL)
    seen = visible(spans, n, rows0)
    scale = float(a.scale) or float(F32(1 / np.sqrt(hd)))
    dist = np.abs(rows0 + np.arange(n)[:, None] - np.arange(rows0 + n))
    at = np.arange(n) if rows is None else rows
    for h in range(heads):
        g = h // (heads // kvh)
        o, e, _, ob, eb, _ = ref.attention(q[at, h * hd:(h + 1) * hd], k[:, g * hd:(g + 1) * hd], v[:, g * hd:(g + 1) * hd],
                                           seen[at], scale, float(a.cap),
                                           None if slopes is None else np.full(len(at), slopes[h], np.float64), dist[at])
        ref.close(out[at, h * hd:(h + 1) * hd], o, ob, f"out of head {h}")
        ref.close(lse[at, h], e, eb, f"lse of head {h}")


SHAPES = [(1, 0), (1, 1), (1, 31), (1, 32), (1, 33), (1, 700), (2, 0), (5, 64), (15, 0), (16, 16), (17, 15), (31, 1), (33, 95),
          (64, 0), (65, 3), (130, 0), (257, 40)]


@pytest.mark.parametrize("n,rows0", SHAPES)
@pytest.mark.parametrize("heads,kvh,hd", [(16, 2, 128), (4, 2, 64)])
def test_prompt_causal(ctx, rng, n, rows0, heads, kvh, hd):
    with ref.Hip() as hip:
        a, q, k, v = prompt_case(hip, rng, n, rows0, heads, kvh, hd, None)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


@pytest.mark.parametrize("heads,kvh,hd", [(1, 1, 128), (8, 8, 64), (7, 1, 128), (6, 2, 64), (24, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("n,rows0", [(1, 40), (9, 0), (70, 13)])
def test_prompt_head_groups(ctx, rng, heads, kvh, hd, n, rows0):
    with ref.Hip() as hip:
        a, q, k, v = prompt_case(hip, rng, n, rows0, heads, kvh, hd, None, pad=12)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


@pytest.mark.parametrize("kind", ["prefix", "docs", "window", "holes"])
@pytest.mark.parametrize("n,rows0", [(1, 0), (3, 50), (48, 0), (100, 77), (219, 0)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (25.0, True)], ids=["plain", "cap-bias"])
def test_prompt_spans(ctx, rng, kind, n, rows0, cap, bias):
    with ref.Hip() as hip:
        spans = spans_of(kind, n, rows0, rng)
        slopes = alibi(4) if bias else None
        a, q, k, v = prompt_case(hip, rng, n, rows0, 4, 2, 64 if n % 2 else 128, spans, cap, slopes, pad=4)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans, slopes)


@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (50.0, True), (0.01, False), (1e6, False)])
@pytest.mark.parametrize("n,rows0", [(1, 1000), (40, 300)])
def test_prompt_scores(ctx, rng, cap, bias, n, rows0):
    """Capped scores over the whole curve of the tanh, biases of near and far rows."""
    with ref.Hip() as hip:
        slopes = alibi(16) if bias else None
        q = rng.standard_normal((n, 2048)).astype(F32) * np.logspace(-3, 2.3, n * 2048).reshape(n, 2048).astype(F32)
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 2, 128, None, cap, slopes, scale=0.1, q=q)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None, slopes)


@pytest.mark.parametrize("n,rows0", [(1, 4000), (600, 900)])
def test_prompt_long(ctx, rng, n, rows0):
    with ref.Hip() as hip:
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 2, 128, None)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None, rows=np.unique([0, n // 3, n // 2, max(0, n - 65), n - 1]))


@pytest.mark.parametrize("n,rows0", [(1, 90), (50, 60)])
def test_prompt_wide_ranges(ctx, rng, n, rows0):
    """Rows of very different size in one block: large and tiny keys, values and queries, zeros."""
    with ref.Hip() as hip:
        rows = rows0 + n
        size = np.exp2(rng.integers(-14, 15, rows)).astype(F32)[:, None]
        k = rng.standard_normal((rows, 256)).astype(F32) * size[rng.permutation(rows)] * F32(2.0 ** -8)
        v = rng.standard_normal((rows, 256)).astype(F32) * size
        q = rng.standard_normal((n, 2048)).astype(F32) * np.exp2(rng.integers(-12, 3, (n, 1))).astype(F32)
        k[rows // 2], v[rows // 3], q[n // 2, :128] = 0.0, 0.0, 0.0
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 2, 128, None, q=q, k=k, v=v)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -60, 2.0 ** 60, 2.0 ** 100])
def test_prompt_far_scales(ctx, rng, scale):
    """Operands of far exponents: products and sums in fp32's range, operands outside fp16's."""
    with ref.Hip() as hip:
        n, rows0 = 20, 50
        q = rng.standard_normal((n, 256)).astype(F32) * F32(3 / scale)
        k = rng.standard_normal((70, 128)).astype(F32) * F32(scale)
        v = rng.standard_normal((70, 128)).astype(F32) * F32(scale)
        a, q, k, v = prompt_case(hip, rng, n, rows0, 2, 1, 128, None, q=q, k=k, v=v)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, F32(3e38)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_prompt_masked_values_do_not_leak(ctx, rng, bad, where):
    """Non-finite (and the largest) keys and values behind the mask: rows that
    do not see them are exact, rows that see a NaN or an infinite value are not finite."""
    with ref.Hip() as hip:
        n, rows0, at = 45, 30, 52  # row 52 of 75: tokens 22 and later see it
        k = rng.standard_normal((75, 256)).astype(F32)
        v = rng.standard_normal((75, 256)).astype(F32)
        (k if where == "k" else v)[at, 5] = bad  # KV head 0
        a, q, k, v = prompt_case(hip, rng, n, rows0, 4, 2, 128, None, k=k, v=v)
        ctx.prompt_attention(a)
        out = hip.down(a.out, (n, 512))
        clean_k, clean_v = k.copy(), v.copy()
        (clean_k if where == "k" else clean_v)[at, 5] = 0.0
        check_rows = np.arange(at - rows0)
        check_prompt(hip, a, q, clean_k, clean_v, None, rows=check_rows)
        for h in (2, 3):  # heads of KV head 1 see no bad value at all
            o, _, _, ob, _, _ = ref.attention(q[:, h * 128:(h + 1) * 128], clean_k[:, 128:], clean_v[:, 128:],
                                              visible(None, n, rows0), float(F32(128 ** -0.5)))
            ref.close(out[:, h * 128:(h + 1) * 128], o, ob)
        if np.isnan(bad) or (where == "v" and np.isinf(bad)):
            assert not np.isfinite(out[at - rows0:, :256]).all(1).any()


@pytest.mark.parametrize("where", ["q", "k"])
@pytest.mark.parametrize("n", [1, 45])
def test_prompt_nan_passes_the_cap(ctx, rng, n, where):
    """A capped score of NaN is NaN: its row is not finite."""
    with ref.Hip() as hip:
        q = rng.standard_normal((n, 256)).astype(F32)
        k = rng.standard_normal((n + 30, 128)).astype(F32)
        (q if where == "q" else k)[0, 5] = np.nan
        a, q, k, v = prompt_case(hip, rng, n, 30, 2, 1, 128, None, cap=9.0, q=q, k=k)
        ctx.prompt_attention(a)
        out = hip.down(a.out, (n, 2, 128))
        assert not np.isfinite(out[:, 0] if where == "k" else out[:1, 0]).all(-1).any()


@pytest.mark.parametrize("size", [0.01, 0.5, 4.0, 60.0])
@pytest.mark.parametrize("n", [1, 70])
def test_prompt_caps_of_all_sizes(ctx, rng, n, size):
    """Scores far below their cap, around it and far above it."""
    with ref.Hip() as hip:
        q = rng.standard_normal((n, 256)).astype(F32) * F32(size)
        a, q, k, v = prompt_case(hip, rng, n, 50, 2, 1, 128, None, cap=3.0, q=q)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


def test_prompt_rows_that_see_nothing_read_nothing(ctx, rng):
    """A whole prompt of padding: zeros and -inf, whatever the cache holds."""
    with ref.Hip() as hip:
        n = 37
        spans = (np.full(n, 9, I32), np.full(n, 9, I32))
        bad = np.full((n, 128), np.nan, F32)
        a, q, k, v = prompt_case(hip, rng, n, 0, 2, 1, 128, spans, k=bad, v=bad)
        ctx.prompt_attention(a)
        assert np.all(hip.down(a.out, (n, 256)) == 0.0) and np.all(hip.down(a.lse, (n, 2)) == -np.inf)


@pytest.mark.parametrize("edge", [2 ** 31 - 1, -2 ** 31])
def test_prompt_extreme_spans(ctx, rng, edge):
    with ref.Hip() as hip:
        n = 20
        spans = (np.where(np.arange(n) % 2, -2 ** 31, edge).astype(I32), np.where(np.arange(n) % 4 < 2, 2 ** 31 - 1, edge).astype(I32))
        a, q, k, v = prompt_case(hip, rng, n, 7, 2, 1, 64, spans)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans)


# Prompts of many tiles take another way: images of the rows, laid out once, and
# shares that the device cuts (from 8 tiles of 128 query rows and 2,400 steps of
# a tile and 32 keys: 840 tokens of 16 heads over one KV head, 105 tiles of up to
# 28 steps).


@pytest.mark.parametrize("kind", ["causal", "prefix", "docs", "window", "holes"])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (12.0, False), (25.0, True)], ids=["plain", "cap", "cap-bias"])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_many_tiles(ctx, rng, kind, cap, bias, hd):
    with ref.Hip() as hip:
        n, rows0 = 840, 37
        spans = spans_of(kind, n, rows0, rng)
        slopes = alibi(16) if bias else None
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 1, hd, spans, cap, slopes, pad=4)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans, slopes, rows=np.unique(np.r_[0:20, 20:820:11, 820:840]))


@pytest.mark.parametrize("n,rows0,heads,kvh", [(900, 0, 21, 3), (64, 10000, 16, 1), (1100, 0, 64, 4), (700, 5000, 5, 5)],
                         ids=["groups-of-7", "few-tiles-long", "uncut", "group-of-1"])
@pytest.mark.parametrize("kind", ["causal", "docs"])
def test_prompt_many_tiles_shapes(ctx, rng, n, rows0, heads, kvh, kind):
    with ref.Hip() as hip:
        spans = spans_of(kind, n, rows0, rng)
        a, q, k, v = prompt_case(hip, rng, n, rows0, heads, kvh, 64, spans)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans, rows=np.unique(np.r_[0:5, 5:n - 5:23, n - 5:n]))


def test_prompt_many_tiles_all_rows(ctx, rng):
    """No row is left out or written twice, whatever its tile's shares."""
    with ref.Hip() as hip:
        n = 803
        spans = spans_of("holes", n, 0, rng)
        a, q, k, v = prompt_case(hip, rng, n, 0, 16, 1, 64, spans)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans)


def test_prompt_many_tiles_wide_ranges(ctx, rng):
    """Rows of very different size in one step, and of one size in the next."""
    with ref.Hip() as hip:
        n, rows0 = 830, 30
        rows = rows0 + n
        size = np.exp2(np.where(np.arange(rows) // 96 % 2, rng.integers(-14, 15, rows), 3)).astype(F32)[:, None]
        k = rng.standard_normal((rows, 64)).astype(F32) * size * F32(2.0 ** -8)
        v = rng.standard_normal((rows, 64)).astype(F32) * size
        q = rng.standard_normal((n, 1024)).astype(F32) * np.exp2(rng.integers(-12, 3, (n, 1))).astype(F32)
        k[rows // 2], v[rows // 3], q[n // 2, :128] = 0.0, 0.0, 0.0
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 1, 64, None, q=q, k=k, v=v)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None, rows=np.unique(np.r_[0:830:7, 829]))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_prompt_many_tiles_masked_values_do_not_leak(ctx, rng, bad, where):
    with ref.Hip() as hip:
        n, at = 840, 500
        k = rng.standard_normal((n, 64)).astype(F32)
        v = rng.standard_normal((n, 64)).astype(F32)
        (k if where == "k" else v)[at, 5] = bad
        a, q, k, v = prompt_case(hip, rng, n, 0, 16, 1, 64, None, k=k, v=v)
        ctx.prompt_attention(a)
        out = hip.down(a.out, (n, 1024))
        (k if where == "k" else v)[at, 5] = 0.0
        check_prompt(hip, a, q, k, v, None, rows=np.unique(np.r_[0:at:9, at - 20:at]))
        if np.isnan(bad) or where == "v":
            assert not np.isfinite(out[at:].reshape(-1, 16, 64)).all(-1).any()


@pytest.mark.parametrize("edge", [2 ** 31 - 1, -2 ** 31])
def test_prompt_many_tiles_extreme_spans(ctx, rng, edge):
    with ref.Hip() as hip:
        n = 840
        i = np.arange(n)
        spans = (np.where(i % 2, -2 ** 31, edge).astype(I32), np.where(i % 4 < 2, 2 ** 31 - 1, edge).astype(I32))
        spans[0][300:600] = spans[1][300:600] = edge  # whole tiles that see nothing
        a, q, k, v = prompt_case(hip, rng, n, 7, 16, 1, 64, spans)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans, rows=np.unique(np.r_[0:840:13, 838:840]))


def test_prompt_many_tiles_captured_and_replayed(ctx, rng):
    """A graph cuts its tiles by the spans that each replay finds, an eager call of another workspace between."""
    with ref.Hip() as hip:
        s = hip.stream()
        n, rows0 = 820, 20
        spans = spans_of("causal", n, rows0, rng) or (np.zeros(n, I32), (rows0 + 1 + np.arange(n)).astype(I32))
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 1, 64, spans)
        b, bq, bk, bv = prompt_case(hip, rng, 810, 0, 16, 1, 64, None)
        hip.sync()
        g = hip.capture(s, lambda: ctx.prompt_attention(a, s))
        rows = np.unique(np.r_[0:n:17, n - 1])
        for kind in ("causal", "docs", "holes", "window", "docs"):
            spans = spans_of(kind, n, rows0, rng) or (np.zeros(n, I32), (rows0 + 1 + np.arange(n)).astype(I32))
            hip.write(a.row_begin, spans[0])
            hip.write(a.row_end, spans[1])
            k[:] = rng.standard_normal(k.shape) * 0.64
            hip.write(a.k, k)
            hip.replay(g, s)
            check_prompt(hip, a, q, k, v, spans, rows=rows)
            ctx.prompt_attention(b, s)
            hip.sync()
            check_prompt(hip, b, bq, bk, bv, None, rows=rows[rows < 810])


# ---------------------------------------------------------------------------
# drafted trees
# ---------------------------------------------------------------------------


def random_trees(rng, seqs, n):
    i = np.arange(n)
    return np.where(rng.random((seqs, n)) < 0.5, i - 1, np.floor(rng.random((seqs, n)) * (i + 1)) - 1).astype(I32)


class Tree:
    """Buffers of one tree call; cache rows behind the drafted ones hold NaN."""

    def __init__(self, hip, rng, lens, counts, n, heads, kvh, hd, parents=None, cap=0.0, slopes=None, positions=None,
                 room=0, pad=0, take=None, side=0):
        self.hip, self.lens, self.parents, self.slopes, self.take = hip, np.asarray(lens, I32), parents, slopes, take
        s = len(lens)
        self.counts = np.full(s, n, I32) if counts is None else np.asarray(counts, I32)
        self.max_rows = int(max(np.max(np.clip(self.lens, 0, None)) + n, n)) + room
        self.q = rng.standard_normal((s, n, heads * hd + pad)).astype(F32) * 3
        self.k = np.full((s, self.max_rows, kvh * hd + pad), np.nan, F32)
        self.v = np.full((s, self.max_rows, kvh * hd + pad), np.nan, F32)
        for x in range(s):
            e = min(max(int(self.lens[x]), 0), self.max_rows - self.counts[x].clip(0, n)) + self.counts[x].clip(0, n)
            self.k[x, :e] = rng.standard_normal((e, kvh * hd + pad)) * 0.64
            self.v[x, :e] = rng.standard_normal((e, kvh * hd + pad)) * 0.64
        self.side = side or self.max_rows
        self.weights = rng.random((s, kvh, self.side)).astype(F32)
        self.positions = positions(s, kvh, self.side) if positions else None
        out = np.full((s, n, heads * hd + pad), SENTINEL, F32)
        self.a = lib.TreeArgs(q=hip.up(self.q), k=hip.up(self.k), v=hip.up(self.v), lens=hip.up(self.lens),
                              counts=None if counts is None else hip.up(self.counts),
                              parents=None if parents is None else hip.up(parents),
                              slopes=None if slopes is None else hip.up(slopes),
                              positions=None if self.positions is None else hip.up(self.positions),
                              out=hip.up(out), lse=hip.up(np.full((s, n, heads), SENTINEL, F32)), weights=hip.up(self.weights),
                              take=None if take is None else hip.up(np.asarray(take, np.uint64)), seqs=s, n=n,
                              max_rows=self.max_rows, heads=heads, kv_heads=kvh, head_dim=hd, cap=cap, side_stride=side,
                              q_seq_stride=self.q[0].size, q_stride=self.q.shape[2], k_seq_stride=self.k[0].size,
                              k_stride=self.k.shape[2], v_seq_stride=self.v[0].size, v_stride=self.v.shape[2],
                              out_seq_stride=self.q[0].size, out_stride=self.q.shape[2])
        need = lib.tree_attention_workspace(self.a)
        self.a.workspace, self.a.workspace_bytes = hip.raw(need), need

    def expect(self, s):
        """Per head: (out, lse, p, bounds) of sequence s's tokens, and its rows."""
        a, hd = self.a, self.a.head_dim
        count = int(self.counts[s].clip(0, a.n))
        length = min(max(int(self.lens[s]), 0), self.max_rows - count)
        par = self.parents[s] if self.parents is not None else np.arange(a.n) - 1
        sees = ref.ancestors(par, count)
        seen = np.concatenate([np.ones((count, length), bool), sees[:count, :count]], 1)
        depth = sees.sum(1) - 1
        for h in range(a.heads):
            g = h // (a.heads // a.kv_heads)
            if self.positions is None:
                pos = np.concatenate([np.arange(length), length + depth[:count]])
            else:
                pos = self.positions[s, g, :length + count].astype(np.int64)
            dist = np.abs(pos[length:][:, None] - pos)
            slope = None if self.slopes is None else np.full(count, self.slopes[h], np.float64)
            yield h, count, length, ref.attention(
                self.q[s, :count, h * hd:(h + 1) * hd], self.k[s, :length + count, g * hd:(g + 1) * hd],
                self.v[s, :length + count, g * hd:(g + 1) * hd], seen, float(F32(hd ** -0.5)), float(a.cap), slope, dist)

    def check(self):
        a, hd = self.a, self.a.head_dim
        out = self.hip.down(a.out, self.q.shape)
        lse = self.hip.down(a.lse, (a.seqs, a.n, a.heads))
        for s in range(a.seqs):
            count = int(self.counts[s].clip(0, a.n))
            assert np.all(out[s, count:] == SENTINEL) and np.all(lse[s, count:] == SENTINEL)
            assert np.all(out[s, :, a.heads * hd:] == SENTINEL)
            for h, _, _, (o, e, _, ob, eb, _) in self.expect(s) if count else ():
                ref.close(out[s, :count, h * hd:(h + 1) * hd], o, ob, f"out {s} {h}")
                ref.close(lse[s, :count, h], e, eb, f"lse {s} {h}")

    def check_weights(self, times=1):
        a = self.a
        got = self.hip.down(a.weights, self.weights.shape)
        want, bound = self.weights.astype(np.float64), np.zeros(self.weights.shape)
        for s in range(a.seqs):
            count = int(self.counts[s].clip(0, a.n))
            taken = np.array([self.take is None or bool(int(self.take[s]) >> t & 1) for t in range(count)])
            for h, _, length, (_, _, p, _, eb, pb) in self.expect(s) if count else ():
                g = h // (a.heads // a.kv_heads)
                want[s, g, :length + count] += times * p[taken].sum(0)
                # the given lse carries its own error, the sum of rows and heads 8 steps and a rounding each time
                bound[s, g, :length + count] += times * (pb + p * (eb[:, None] + 2.0 ** -21))[taken].sum(0)
        bound += want * 2 * times * ref.U + 1e-38
        untouched = np.ones(got.shape, bool)
        for s in range(a.seqs):
            c = int(self.counts[s].clip(0, a.n))
            untouched[s, :, :min(max(int(self.lens[s]), 0), self.max_rows - c) + c] = False
        assert np.array_equal(got[untouched], self.weights[untouched])
        ref.close(got, want, bound, "weights")


TREES = [([0], None, 1), ([0], None, 5), ([1], None, 1), ([31], None, 1), ([32], None, 2), ([33], None, 7), ([500], None, 16),
         ([700], None, 64), ([3, 90, 0, 257], [4, 0, 2, 6], 6), ([64, 63, 65], [33, 1, 17], 33), ([300] * 5, None, 9)]


@pytest.mark.parametrize("lens,counts,n", TREES)
@pytest.mark.parametrize("heads,kvh,hd", [(16, 2, 128), (4, 2, 64), (3, 3, 128)])
def test_tree_attention_and_weights(ctx, rng, lens, counts, n, heads, kvh, hd):
    with ref.Hip() as hip:
        t = Tree(hip, rng, lens, counts, n, heads, kvh, hd, random_trees(rng, len(lens), n))
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("heads,kvh,hd", [(7, 1, 128), (8, 8, 64), (24, 2, 64), (40, 1, 128)])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_tree_head_groups(ctx, rng, heads, kvh, hd, n):
    with ref.Hip() as hip:
        t = Tree(hip, rng, [77, 5], None, n, heads, kvh, hd, pad=8, room=13, side=150)
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        ctx.cache_weights(t.a)
        t.check_weights(times=2)


@pytest.mark.parametrize("cap", [0.0, 18.0])
@pytest.mark.parametrize("moved", [False, True], ids=["rows", "positions"])
@pytest.mark.parametrize("n", [1, 11])
def test_tree_bias_cap_take(ctx, rng, cap, moved, n):
    """Distances by tree depth, or by the positions of rows that moved; only some tokens count."""
    def positions(s, kvh, side):
        return np.sort(rng.integers(0, 4 * side, (s, kvh, side)), 2).astype(I32)

    with ref.Hip() as hip:
        t = Tree(hip, rng, [130, 0, 41], [n, n, 1], n, 16, 2, 128, random_trees(rng, 3, n), cap, alibi(16),
                 positions if moved else None, take=[0b10110101101, 2 ** 64 - 1, 0])
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("seqs,room", [(1, 0), (40, 20), (90, 20)], ids=["32-keys", "64-keys", "96-keys"])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (18.0, True)], ids=["plain", "cap-bias"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [9, 33])
def test_weights_of_many_rows(ctx, rng, seqs, room, cap, bias, hd, n):
    """More than 64 query rows, by workgroups of 32, 64 and 96 cache rows; lengths that end anywhere in them."""
    with ref.Hip() as hip:
        lens = rng.integers(0, 70, seqs)
        t = Tree(hip, rng, lens, rng.integers(0, n + 1, seqs), n, 16, 2, hd, random_trees(rng, seqs, n), cap,
                 alibi(16) if bias else None, room=room)
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


def test_tree_long(ctx, rng):
    with ref.Hip() as hip:
        t = Tree(hip, rng, [5000, 2100], [12, 3], 12, 4, 2, 128, random_trees(rng, 2, 12))
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


def test_tree_numbers_out_of_range(ctx, rng):
    """Lengths, counts and parents that the host would refuse are forced into range on the device."""
    with ref.Hip() as hip:
        n = 6
        parents = np.array([[7, -5, 2, 2 ** 31 - 1, -2 ** 31, 4], [-1, 0, 0, 1, 9, 4]], I32)
        t = Tree(hip, rng, [-9, 40], [-2 ** 31, 2 ** 31 - 1], n, 4, 2, 64, parents)
        t.lens[1] = 2 ** 31 - 1  # forced to max_rows - n, which the buffers hold
        hip.write(t.a.lens, t.lens)
        ctx.tree_attention(t.a)
        ctx.cache_weights(t.a)
        t.check()
        t.check_weights()


def test_tree_no_drafts_anywhere(ctx, rng):
    with ref.Hip() as hip:
        t = Tree(hip, rng, [10, 20], [0, 0], 3, 4, 2, 128)
        ctx.tree_attention(t.a)
        ctx.cache_weights(t.a)
        t.check()
        t.check_weights()


def test_tree_is_repeatable(ctx, rng):
    """The same call gives the same bits."""
    with ref.Hip() as hip:
        t = Tree(hip, rng, [900, 333], None, 13, 16, 2, 128, random_trees(rng, 2, 13))
        ctx.tree_attention(t.a)
        first = hip.down(t.a.out, t.q.shape)
        for _ in range(5):
            hip.write(t.a.out, np.zeros_like(t.q))
            ctx.tree_attention(t.a)
            assert np.array_equal(hip.down(t.a.out, t.q.shape), first)


def test_tree_weights_of_rows_without_lse(ctx, rng):
    """A row whose lse is -inf adds nothing."""
    with ref.Hip() as hip:
        t = Tree(hip, rng, [50], None, 2, 2, 1, 128)
        hip.write(t.a.lse, np.full((1, 2, 2), -np.inf, F32))
        ctx.cache_weights(t.a)
        assert np.array_equal(hip.down(t.a.weights, t.weights.shape), t.weights)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_tree_bad_draft_stays_in_its_branch(ctx, rng, bad, where):
    with ref.Hip() as hip:
        parents = np.array([[-1, 0, 0, 1, 2, 3]], I32)  # token 2's branch: 2 and 4
        t = Tree(hip, rng, [40], None, 6, 2, 1, 128, parents)
        x = t.k if where == "k" else t.v
        x[0, 42, 77] = bad
        hip.write(t.a.k if where == "k" else t.a.v, x)
        ctx.tree_attention(t.a)
        out = hip.down(t.a.out, t.q.shape)
        x[0, 42, 77] = 0.0
        for h, _, _, (o, _, _, ob, _, _) in t.expect(0):
            for i in (0, 1, 3, 5):
                ref.close(out[0, i, h * 128:(h + 1) * 128], o[i], ob[i])
            for i in (2, 4) if np.isnan(bad) or where == "v" else ():
                assert not np.isfinite(out[0, i, h * 128:(h + 1) * 128]).all()


# ---------------------------------------------------------------------------
# selection and compaction
# ---------------------------------------------------------------------------


def run_select(ctx, hip, weights, lens, budget, sinks, recent, max_rows=None, stream=0):
    c, kvh, side = weights.shape
    max_rows = max_rows or side
    kept = hip.up(np.full((c, kvh, budget), -9, I32))
    counts = hip.up(np.full(c, -9, I32))
    a = lib.SelectArgs(weights=hip.up(weights), lens=hip.up(np.asarray(lens, I32)), kept=kept, counts=counts, caches=c,
                       kv_heads=kvh, max_rows=max_rows, budget=budget, sinks=sinks, recent=recent, side_stride=side)
    ctx.cache_select(a, stream)
    return a


def check_select(hip, a, weights, lens):
    kept = hip.down(a.kept, (a.caches, a.kv_heads, a.budget), I32)
    counts = hip.down(a.counts, a.caches, I32)
    for c in range(a.caches):
        length = min(max(int(lens[c]), 0), a.max_rows)
        assert counts[c] == min(length, a.budget)
        for g in range(a.kv_heads):
            want = ref.select(weights[c, g], length, a.budget, a.sinks, a.recent)
            assert np.array_equal(kept[c, g, :counts[c]], want), (c, g)
            assert np.all(kept[c, g, counts[c]:] == -9)


@pytest.mark.parametrize("rows,budget,sinks,recent", [(1, 1, 0, 0), (2, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (40, 39, 3, 30),
                                                      (64, 10, 0, 0), (65, 64, 4, 8), (100, 30, 10, 20), (1000, 1, 0, 0),
                                                      (1025, 300, 4, 100), (8191, 2000, 0, 512), (8193, 8192, 1, 1),
                                                      (20000, 777, 5, 70), (40000, 39999, 0, 0)])
@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_select(ctx, rng, rows, budget, sinks, recent, kind):
    with ref.Hip() as hip:
        shape = (2, 3, rows + 5)
        w = np.exp(rng.standard_normal(shape) * 3).astype(F32)
        if kind == "ties":
            w = rng.integers(0, 3, shape).astype(F32)
        if kind == "special":
            pick = rng.integers(0, 7, shape)
            for i, x in enumerate([np.nan, np.inf, -np.inf, 0.0, -0.0, F32(1e-42)]):
                w[pick == i] = x
        lens = [rows, max(0, rows - 3)]
        a = run_select(ctx, hip, w, lens, budget, sinks, recent, max_rows=rows)
        check_select(hip, a, w, lens)


def test_select_lengths(ctx, rng):
    """Empty, short, exact and longer caches in one call, and lengths out of range."""
    with ref.Hip() as hip:
        w = rng.random((7, 2, 300)).astype(F32)
        lens = [0, 1, 49, 50, 51, -5, 2 ** 31 - 1]
        a = run_select(ctx, hip, w, lens, 50, 4, 16)
        check_select(hip, a, w, lens)


class Keep:
    def __init__(self, rng, caches, rows, kvh, hd, interleaved=False):
        """K and V of `caches` caches; interleaved: layer by layer, as a sequence holds them."""
        self.c, self.rows, self.kvh, self.hd = caches, rows, kvh, hd
        self.kv = rng.standard_normal((caches, 2, rows, kvh * hd)).astype(F32) if interleaved else \
            rng.standard_normal((2, caches, rows, kvh * hd)).astype(F32)
        self.interleaved = interleaved
        self.weights = rng.random((caches, kvh, rows)).astype(F32)
        self.positions = rng.integers(0, 10000, (caches, kvh, rows)).astype(I32)

    def part(self, kv, x):
        return (kv[:, x] if self.interleaved else kv[x]).reshape(self.c, -1, self.kvh, self.hd)

    def args(self, hip, lists, counts, first, side=True, rows_out=None):
        per_head = lists.ndim == 3
        st = self.kvh * self.hd
        size, cs = self.rows * st, (2 if self.interleaved else 1) * self.rows * st
        base = hip.up(self.kv)
        v = base + 4 * (size if self.interleaved else self.c * size)
        a = lib.KeepArgs(k=base, v=v, rows=hip.up(lists.astype(I32)), counts=hip.up(np.asarray(counts, I32)),
                         first=None if first is None else hip.up(np.asarray(first, I32)), caches=self.c, kv_heads=self.kvh,
                         head_dim=self.hd, max_keep=lists.shape[-1], per_head=int(per_head), max_rows=self.rows,
                         max_rows_out=rows_out or self.rows, k_cache_stride=cs, v_cache_stride=cs, k_stride=st, v_stride=st)
        if side:
            a.weights, a.positions = hip.up(self.weights), hip.up(self.positions)
        if rows_out is None:
            a.k_out, a.v_out, a.weights_out, a.positions_out = a.k, a.v, a.weights, a.positions
            a.k_out_cache_stride = a.v_out_cache_stride = cs
            a.k_out_stride = a.v_out_stride = st
        else:
            n = self.c * rows_out
            a.k_out, a.v_out = hip.up(np.full(n * (st + 4), SENTINEL, F32)), hip.up(np.full(n * st, SENTINEL, F32))
            a.k_out_cache_stride, a.k_out_stride = rows_out * (st + 4), st + 4
            a.v_out_cache_stride, a.v_out_stride = rows_out * st, st
            if side:
                a.weights_out = hip.up(np.full((self.c, self.kvh, rows_out + 3), SENTINEL, F32))
                a.positions_out = hip.up(np.full((self.c, self.kvh, rows_out + 3), -9, I32))
                a.side_out_stride = rows_out + 3
        return a

    def check(self, hip, a, lists, counts, first):
        """Moved rows, and every other place of the destination as it was."""
        rows_out, inplace = a.max_rows_out, a.k_out == a.k
        if inplace:
            got = hip.down(a.k, self.kv.shape)
            k2, v2 = self.part(got, 0), self.part(got, 1)
            want_k, want_v = self.part(self.kv, 0).copy(), self.part(self.kv, 1).copy()
            want_w, want_p = self.weights.copy(), self.positions.copy()
            side = self.rows
        else:
            raw = hip.down(a.k_out, (self.c, rows_out, self.kvh * self.hd + 4))
            assert np.all(raw[..., self.kvh * self.hd:] == SENTINEL)
            k2 = raw[..., :self.kvh * self.hd].reshape(self.c, rows_out, self.kvh, self.hd)
            v2 = hip.down(a.v_out, (self.c, rows_out, self.kvh, self.hd))
            want_k, want_v = (np.full((self.c, rows_out, self.kvh, self.hd), SENTINEL, F32) for _ in range(2))
            side = rows_out + 3
            want_w, want_p = np.full((self.c, self.kvh, side), SENTINEL, F32), np.full((self.c, self.kvh, side), -9, I32)
        for c in range(self.c):
            f = 0 if first is None else min(max(int(first[c]), 0), rows_out)
            n = min(max(int(counts[c]), 0), min(lists.shape[-1], rows_out - f))
            for g in range(self.kvh):
                src = (lists[c, g] if lists.ndim == 3 else lists[c])[:n].clip(0, self.rows - 1)
                want_k[c, f:f + n, g] = self.part(self.kv, 0)[c, src, g]
                want_v[c, f:f + n, g] = self.part(self.kv, 1)[c, src, g]
                want_w[c, g, f:f + n] = self.weights[c, g, src]
                want_w[c, g, f + n:rows_out] = 0.0
                want_p[c, g, f:f + n] = self.positions[c, g, src]
        assert np.array_equal(k2, want_k) and np.array_equal(v2, want_v)
        if a.weights:
            assert np.array_equal(hip.down(a.weights_out, (self.c, self.kvh, side)), want_w)
            assert np.array_equal(hip.down(a.positions_out, (self.c, self.kvh, side), I32), want_p)


def ascending(rng, shape, n, rows):
    """Ascending row lists of length n."""
    flat = [np.sort(rng.choice(rows, n, replace=False)) for _ in range(int(np.prod(shape)))]
    return np.array(flat, I32).reshape(*shape, n)


@pytest.mark.parametrize("place", ["in place", "elsewhere"])
@pytest.mark.parametrize("rows,n", [(1, 1), (9, 4), (64, 64), (300, 65), (700, 600), (3000, 2500)])
@pytest.mark.parametrize("kvh,hd", [(2, 128), (3, 64)])
def test_keep_lists_per_head(ctx, rng, place, rows, n, kvh, hd):
    with ref.Hip() as hip:
        kp = Keep(rng, 3, rows, kvh, hd, interleaved=rows % 2 == 0)
        lists = ascending(rng, (3, kvh), n, rows)
        counts = [n, n // 2, 0]
        a = kp.args(hip, lists, counts, None, rows_out=None if place == "in place" else n + 2)
        ctx.cache_keep(a)
        kp.check(hip, a, lists, counts, None)


@pytest.mark.parametrize("place", ["in place", "elsewhere"])
@pytest.mark.parametrize("n", [1, 6, 64])
def test_keep_accepted_paths(ctx, rng, place, n):
    """Drafted rows behind each cache's end, the accepted ones moved up to it."""
    with ref.Hip() as hip:
        rows, c = 200, 5
        kp = Keep(rng, c, rows, 2, 128)
        lens = np.array([0, 1, 77, 136, 120], I32)
        m = max(1, n // 2)
        lists = lens[:, None] + np.array([np.sort(rng.choice(n, m, replace=False)) for _ in range(c)])
        counts = rng.integers(0, m + 1, c)
        a = kp.args(hip, lists, counts, lens, side=n > 1, rows_out=None if place == "in place" else rows)
        ctx.cache_keep(a)
        kp.check(hip, a, lists, counts, lens)


def test_keep_numbers_out_of_range(ctx, rng):
    """Elsewhere: rows, counts and first are forced into range; in place a bad list moves rows but writes nowhere else."""
    with ref.Hip() as hip:
        kp = Keep(rng, 4, 50, 2, 64)
        lists = rng.integers(-90, 140, (4, 2, 30)).astype(I32)
        lists[0, 0, :2] = [2 ** 31 - 1, -2 ** 31]
        counts, first = [30, 2 ** 31 - 1, -3, 30], [0, -7, 2, 2 ** 31 - 1]
        a = kp.args(hip, lists, counts, first, rows_out=25)
        ctx.cache_keep(a)
        kp.check(hip, a, lists, counts, first)
        b = kp.args(hip, lists, counts, first)
        ctx.cache_keep(b)
        hip.sync()  # the guards around every buffer are checked at the end


# ---------------------------------------------------------------------------
# together, and where the calls run
# ---------------------------------------------------------------------------


def test_draft_verify_accept_evict(ctx, rng):
    """A serving loop's turn: trees verified, the accepted path's rows moved up,
    its weights added, the caches evicted, the next trees verified on what is left."""
    with ref.Hip() as hip:
        seqs, n, heads, kvh, hd = 3, 7, 4, 2, 128
        lens = np.array([150, 97, 60], I32)
        t = Tree(hip, rng, lens, None, n, heads, kvh, hd, random_trees(rng, seqs, n), slopes=alibi(heads), room=20,
                 positions=lambda s, g, side: np.broadcast_to(np.arange(side, dtype=I32), (s, g, side)).copy())
        t.weights[:] = 0.0
        hip.write(t.a.weights, t.weights)
        par = t.parents
        pos = t.positions
        for s in range(seqs):  # drafted rows hold the positions of their depths
            depth = ref.ancestors(par[s], n).sum(1) - 1
            pos[s, :, lens[s]:lens[s] + n] = lens[s] + depth
        hip.write(t.a.positions, pos)
        ctx.tree_attention(t.a)
        t.check()
        paths = []  # from the deepest token to the root
        for s in range(seqs):
            sees = ref.ancestors(par[s], n)
            paths.append(np.flatnonzero(sees[np.argmax(sees.sum(1))]))
        t.take = [sum(1 << int(x) for x in p) for p in paths]
        t.a.take = hip.up(np.array(t.take, np.uint64))
        ctx.cache_weights(t.a)
        t.check_weights()
        m = max(len(p) for p in paths)
        lists = np.array([np.concatenate([lens[s] + p, np.zeros(m - len(p), int)]) for s, p in enumerate(paths)], I32)
        counts = np.array([len(p) for p in paths], I32)
        rows, st = t.max_rows, kvh * hd
        acc = lib.KeepArgs(k=t.a.k, v=t.a.v, k_out=t.a.k, v_out=t.a.v, weights=t.a.weights, weights_out=t.a.weights,
                           positions=t.a.positions, positions_out=t.a.positions, rows=hip.up(lists), counts=hip.up(counts),
                           first=t.a.lens, caches=seqs, kv_heads=kvh, head_dim=hd, max_keep=m, max_rows=rows, max_rows_out=rows,
                           k_cache_stride=rows * st, v_cache_stride=rows * st, k_out_cache_stride=rows * st,
                           v_out_cache_stride=rows * st, k_stride=st, v_stride=st, k_out_stride=st, v_out_stride=st)
        w = hip.down(t.a.weights, t.weights.shape)
        ctx.cache_keep(acc)
        k, v = t.k.copy(), t.v.copy()
        new = lens + counts
        for s, p in enumerate(paths):
            k[s, lens[s]:new[s]], v[s, lens[s]:new[s]] = t.k[s, lens[s] + p], t.v[s, lens[s] + p]
            pos[s, :, lens[s]:new[s]] = pos[s][:, lens[s] + p]
            w[s, :, lens[s]:new[s]] = w[s][:, lens[s] + p]
            w[s, :, new[s]:] = 0.0
        assert np.array_equal(hip.down(t.a.weights, w.shape), w)
        assert np.array_equal(hip.down(t.a.positions, pos.shape, I32), pos)
        # evict to 64 rows in place
        budget = 64
        sel = lib.SelectArgs(weights=t.a.weights, lens=hip.up(new.astype(I32)), kept=hip.up(np.zeros((seqs, kvh, budget), I32)),
                             counts=hip.up(np.zeros(seqs, I32)), caches=seqs, kv_heads=kvh, max_rows=rows, budget=budget,
                             sinks=4, recent=20)
        ctx.cache_select(sel)
        ev = lib.KeepArgs.from_buffer_copy(acc)
        ev.rows, ev.counts, ev.first, ev.max_keep, ev.per_head = sel.kept, sel.counts, None, budget, 1
        ctx.cache_keep(ev)
        left = np.minimum(new, budget)
        for s in range(seqs):
            for g in range(kvh):
                keep = ref.select(w[s, g], int(new[s]), budget, 4, 20)
                cols = slice(g * hd, (g + 1) * hd)
                k[s, :left[s], cols], v[s, :left[s], cols] = k[s, keep, cols].copy(), v[s, keep, cols].copy()
                pos[s, g, :left[s]] = pos[s, g, keep].copy()
        # the next trees on what is left: distances still those of the rows' positions
        nxt = Tree(hip, rng, left, None, n, heads, kvh, hd, random_trees(rng, seqs, n), slopes=alibi(heads),
                   room=rows - int(left.max()) - n, positions=lambda *_: pos)
        fresh_k, fresh_v = nxt.k, nxt.v
        for s in range(seqs):
            k[s, left[s]:left[s] + n], v[s, left[s]:left[s] + n] = fresh_k[s, left[s]:left[s] + n], fresh_v[s, left[s]:left[s] + n]
            pos[s, :, left[s]:left[s] + n] = int(new[s]) + ref.ancestors(nxt.parents[s], n).sum(1) - 1
        dk, dv = hip.down(t.a.k, k.shape), hip.down(t.a.v, v.shape)
        for s in range(seqs):
            assert np.array_equal(dk[s, :left[s]], k[s, :left[s]]) and np.array_equal(dv[s, :left[s]], v[s, :left[s]])
            dk[s, left[s]:left[s] + n], dv[s, left[s]:left[s] + n] = k[s, left[s]:left[s] + n], v[s, left[s]:left[s] + n]
        nxt.k, nxt.v, nxt.positions = k, v, pos
        hip.write(nxt.a.k, dk)
        hip.write(nxt.a.v, dv)
        hip.write(nxt.a.positions, pos)
        ctx.tree_attention(nxt.a)
        nxt.check()


def test_prompt_rows_agree_with_tree_rows(ctx, rng):
    """The last rows of a prompt and a chain of drafted tokens over the same cache are the same attention."""
    with ref.Hip() as hip:
        a, q, k, v = prompt_case(hip, rng, 10, 200, 16, 2, 128, None)
        ctx.prompt_attention(a)
        t = Tree(hip, rng, [200], None, 10, 16, 2, 128)
        hip.write(t.a.q, q)
        hip.write(t.a.k, k)
        hip.write(t.a.v, v)
        t.q, t.k, t.v = q[None], k[None], v[None]
        ctx.tree_attention(t.a)
        check_prompt(hip, a, q, k, v, None)
        t.check()


def test_captured_and_replayed(ctx, rng):
    """A graph of the calls replays on new lengths and values, eager calls between."""
    with ref.Hip() as hip:
        s = hip.stream()
        t = Tree(hip, rng, [300, 180], None, 5, 16, 2, 128, random_trees(rng, 2, 5), room=40)
        eager = Tree(hip, rng, [250], None, 9, 16, 2, 128)
        hip.sync()
        sel_w = rng.random((2, 2, 400)).astype(F32)
        hip.sync()
        lens = hip.up(np.array([400, 30], I32))
        sel = lib.SelectArgs(weights=hip.up(sel_w), lens=lens, kept=hip.up(np.full((2, 2, 64), -9, I32)),
                             counts=hip.up(np.zeros(2, I32)), caches=2, kv_heads=2, max_rows=400, budget=64, sinks=1, recent=7)
        hip.sync()

        def calls():
            ctx.tree_attention(t.a, s)
            ctx.cache_weights(t.a, s)
            ctx.cache_select(sel, s)

        g = hip.capture(s, calls)
        for turn, new in enumerate(([300, 180], [7, 0], [340, 341], [31, 32], [300, 180])):
            t.lens[:] = new
            t.k[:] = rng.standard_normal(t.k.shape) * 0.64
            t.v[:] = rng.standard_normal(t.v.shape) * 0.64
            hip.write(t.a.lens, t.lens)
            hip.write(t.a.k, t.k)
            hip.write(t.a.v, t.v)
            t.weights[:] = turn
            hip.write(t.a.weights, t.weights)
            hip.replay(g, s)
            t.check()
            t.check_weights()
            check_select(hip, sel, sel_w, [400, 30])
            ctx.tree_attention(eager.a, s)
            hip.sync()
            eager.check()


def test_calls_on_two_streams_and_threads(ctx, rng):
    """Calls at once, each with its own workspace, from threads on their own streams."""
    with ref.Hip() as hip:
        trees = [Tree(hip, rng, [700 + 50 * i], None, 6 + i, 16, 2, 128) for i in range(4)]
        streams = [hip.stream() for _ in trees]
        hip.sync()
        errors = []

        def work(t, s):
            try:
                for _ in range(20):
                    ctx.tree_attention(t.a, s)
            except Exception as e:  # reported below
                errors.append(e)

        threads = [threading.Thread(target=work, args=x) for x in zip(trees, streams)]
        for x in threads:
            x.start()
        for x in threads:
            x.join()
        assert not errors
        for t in trees:
            t.check()


def test_far_caches(ctx, rng):
    """Sequences whose caches lie more than 2^31 floats apart."""
    with ref.Hip() as hip:
        t = Tree(hip, rng, [70, 40], None, 4, 4, 2, 64)
        far = 2 ** 31 + 4096
        for name, x in (("k", t.k), ("v", t.v)):
            base = hip.raw(4 * (far + x[0].size))
            hip.write(base, x[0])
            hip.write(base + 4 * far, x[1])
            setattr(t.a, name, base)
        t.a.k_seq_stride = t.a.v_seq_stride = far
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()
        rows, st = t.max_rows, 128
        lists = np.array([[3, 9, 50], [0, 1, 39]], I32)
        keep = lib.KeepArgs(k=t.a.k, v=t.a.v, k_out=t.a.k, v_out=t.a.v, rows=hip.up(lists), counts=hip.up(np.array([3, 3], I32)),
                            caches=2, kv_heads=2, head_dim=64, max_keep=3, max_rows=rows, max_rows_out=rows, k_cache_stride=far,
                            v_cache_stride=far, k_out_cache_stride=far, v_out_cache_stride=far, k_stride=st, v_stride=st,
                            k_out_stride=st, v_out_stride=st)
        ctx.cache_keep(keep)
        for s in range(2):
            got = hip.down(t.a.k + 4 * far * s, (3, st))
            assert np.array_equal(got, t.k[s, lists[s]])


def test_rows_far_apart(ctx, rng):
    """One cache whose rows lie so far apart that its end passes 2^31 floats."""
    with ref.Hip() as hip:
        n, rows0, st = 3, 5, 2 ** 29
        a, q, k, v = prompt_case(hip, rng, n, rows0, 2, 1, 64, None)
        for name, x in (("k", k), ("v", v)):
            base = hip.raw(4 * ((rows0 + n - 1) * st + 64))
            for j in range(rows0 + n):
                hip.write(base + 4 * st * j, x[j])
            setattr(a, name, base)
            setattr(a, name + "_stride", st)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


def test_refusals_touch_nothing(ctx, rng):
    with ref.Hip() as hip:
        t = Tree(hip, rng, [20], None, 2, 4, 2, 64)
        t.a.head_dim = 80
        with pytest.raises(lib.PocrError) as e:
            ctx.tree_attention(t.a)
        assert e.value.code == lib.POCR_ERR_UNSUPPORTED
        assert np.all(hip.down(t.a.out, t.q.shape) == SENTINEL)

"""The cache operators at the ends of the ranges that their header states.
Definitions and bounds: cache_ops_f64.py."""
import ctypes as C

import cache_ops_f64 as ref
import numpy as np
import pytest
from test_gpu_cache_ops import (F32, I32, SENTINEL, Keep, Tree, alibi, ascending, check_prompt, check_select, prompt_case,
                                random_trees, run_select, spans_of, visible)

from rapidocrvl_amd import lib

pytestmark = pytest.mark.gpu


def check_one_hot(out, lse, s, seen, v):
    """Rows whose largest score stands far above the next: their key's value row.

    A score of 22-bit operands is off by at most 2^-15 of the largest (2^-19 of
    the sum of its 64 products' sizes, which stays below 16 times the largest
    score).  Where the next is 2^-12 of that and at least 2^7 further down, its
    weight is below e^-90.  The value row keeps 22 bits (2^-19 with its sums),
    and the logarithm of the sum what the score does."""
    order = np.sort(np.where(seen, s, -np.inf), 1)
    size = np.abs(np.where(seen, s, 0.0)).max(1)
    clear = order[:, -1] - order[:, -2] > np.maximum(size * 2.0 ** -12, 2.0 ** 7)
    assert clear.sum() > len(s) / 2
    at = np.where(seen, s, -np.inf).argmax(1)
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    err = np.abs(out - v[at])[clear]
    assert np.all(err <= np.abs(v[at])[clear] * 2.0 ** -19 + np.abs(v[at]).max(1)[clear, None] * 2.0 ** -28)
    assert np.all(np.abs(lse - order[:, -1]) <= size * 2.0 ** -15)


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 13, 2.0 ** 14, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("n,rows0,heads", [(1, 200, 2), (20, 200, 2), (840, 37, 16)], ids=["few", "tiles", "images"])
def test_prompt_far_scores(ctx, rng, n, rows0, heads, size, bias):
    """Finite scores of 2^24 and far more: a step of fp32 there is more than an exponent of fp16 holds."""
    with ref.Hip() as hip:
        q = (rng.standard_normal((n, heads * 64)) * size).astype(F32)
        k = (rng.standard_normal((rows0 + n, 64)) * size).astype(F32)
        slopes = alibi(heads) if bias else None
        a, q, k, v = prompt_case(hip, rng, n, rows0, heads, 1, 64, None, 0.0, slopes, q=q, k=k)
        ctx.prompt_attention(a)
        out, lse = hip.down(a.out, (n, heads * 64)), hip.down(a.lse, (n, heads))
        dist = rows0 + np.arange(n)[:, None] - np.arange(rows0 + n)
        for h in range(heads):
            s = q[:, h * 64:(h + 1) * 64].astype(np.float64) @ k.T.astype(np.float64) * 0.125
            if bias:
                s -= slopes[h].astype(np.float64) * np.abs(dist)
            check_one_hot(out[:, h * 64:(h + 1) * 64], lse[:, h], s, visible(None, n, rows0), v)


@pytest.mark.parametrize("slope", [2.0 ** 18, 2.0 ** 19, 2.0 ** 20, 2.0 ** 21, 2.0 ** 24])
@pytest.mark.parametrize("n,rows0,heads", [(1, 400, 2), (20, 400, 2), (840, 237, 16)], ids=["few", "tiles", "images"])
def test_prompt_far_biases(ctx, rng, n, rows0, heads, slope):
    """Rows that see none of their nearest 100 keys: all their scores lie far below zero."""
    with ref.Hip() as hip:
        i = np.arange(n)
        spans = np.zeros(n, I32), (rows0 + i - 100).astype(I32)
        slopes = np.full(heads, slope, F32)
        a, q, k, v = prompt_case(hip, rng, n, rows0, heads, 1, 64, spans, 0.0, slopes)
        ctx.prompt_attention(a)
        out, lse = hip.down(a.out, (n, heads * 64)), hip.down(a.lse, (n, heads))
        dist = rows0 + i[:, None] - np.arange(rows0 + n)
        for h in range(heads):
            s = q[:, h * 64:(h + 1) * 64].astype(np.float64) @ k.T.astype(np.float64) * 0.125 - slope * np.abs(dist)
            check_one_hot(out[:, h * 64:(h + 1) * 64], lse[:, h], s, visible(spans, n, rows0), v)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("at", [5, 70, 103], ids=["first", "middle", "last"])
@pytest.mark.parametrize("n,rows0,heads", [(1, 103, 2), (4, 100, 2), (30, 74, 2), (840, 20, 16)],
                         ids=["one", "few", "tiles", "images"])
def test_prompt_bad_values_leave_the_lse(ctx, rng, n, rows0, heads, at, bad):
    """lse is of the scores alone, whatever a visible value row holds; out is not finite there."""
    with ref.Hip() as hip:
        v = rng.standard_normal((rows0 + n, 64)).astype(F32)
        clean = v.copy()
        v[at, 9], clean[at] = bad, 0.0
        a, q, k, v = prompt_case(hip, rng, n, rows0, heads, 1, 64, None, v=v)
        ctx.prompt_attention(a)
        out, lse = hip.down(a.out, (n, heads, 64)), hip.down(a.lse, (n, heads))
        sees = rows0 + np.arange(n) >= at
        assert not np.isfinite(out[sees]).all(-1).any()
        assert np.isfinite(out[~sees]).all()
        for h in range(heads):
            _, e, _, _, eb, _ = ref.attention(q[:, h * 64:(h + 1) * 64], k, clean, visible(None, n, rows0), 0.125)
            ref.close(lse[:, h], e, eb, f"lse of head {h}")


@pytest.mark.parametrize("at", [3, 300, 601], ids=["first", "middle", "draft"])
@pytest.mark.parametrize("n", [2, 20])
def test_tree_bad_values_leave_the_weights(ctx, rng, n, at):
    """The lse that pocr_cache_weights takes stays that of the scores: weights are those of finite values."""
    with ref.Hip() as hip:
        t = Tree(hip, rng, [600, 601], None, n, 4, 2, 128)
        x = t.v.copy()
        x[:, at, 7] = np.nan  # KV head 0
        hip.write(t.a.v, x)
        ctx.tree_attention(t.a)
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("slope", [3e38, -3e38])
@pytest.mark.parametrize("n,heads", [(1, 2), (20, 2), (840, 16)], ids=["few", "tiles", "images"])
def test_prompt_largest_slopes(ctx, rng, n, heads, slope):
    """A slope near fp32's end: a row's own key has no distance and no bias.  Rows see themselves alone."""
    with ref.Hip() as hip:
        i = np.arange(n)
        spans = i.astype(I32), (i + 1).astype(I32)
        a, q, k, v = prompt_case(hip, rng, n, 0, heads, 1, 64, spans, 0.0, np.full(heads, slope, F32))
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans)


@pytest.mark.parametrize("n", [1, 20])
def test_tree_largest_slopes(ctx, rng, n):
    with ref.Hip() as hip:
        t = Tree(hip, rng, [0, 0], None, n, 2, 1, 64, np.full((2, n), -1, I32))  # every token sees itself alone
        t.a.slopes = hip.up(np.full(2, 3e38, F32))
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("cap", [2.0 ** -126, 2.0 ** 126])
@pytest.mark.parametrize("n,heads", [(1, 2), (20, 2), (840, 16)], ids=["few", "tiles", "images"])
def test_prompt_caps_at_the_ends(ctx, rng, n, heads, cap):
    """The least cap makes all scores alike, the largest leaves them as they are."""
    with ref.Hip() as hip:
        a, q, k, v = prompt_case(hip, rng, n, 60, heads, 1, 64, None, cap)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


@pytest.mark.parametrize("n", [1, 20])
def test_tree_positions_of_the_whole_range(ctx, rng, n):
    """Positions further apart than 2^31."""
    def positions(s, kvh, side):
        return rng.integers(-2 ** 31, 2 ** 31, (s, kvh, side)).astype(I32)

    with ref.Hip() as hip:
        t = Tree(hip, rng, [90, 33], None, n, 4, 2, 64, slopes=np.array([1e-9, 2e-9, 4e-10, 1e-9], F32), positions=positions)
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("up,down", [(64, 63), (100, 27), (27, 100)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("n", [1, 20])
def test_prompt_products_that_need_their_scale(ctx, rng, n, cap, up, down):
    """q·k passes fp32's range where scale·q·k does not."""
    with ref.Hip() as hip:
        q = (rng.standard_normal((n, 128)) * 2.0 ** up).astype(F32)
        k = (rng.standard_normal((n + 50, 64)) * 2.0 ** down).astype(F32)
        a, q, k, v = prompt_case(hip, rng, n, 50, 2, 1, 64, None, cap, scale=2.0 ** -126, q=q, k=k)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, None)


def all_calls(ctx, hip, rng):
    """One small call of each operator and of each of its forms, with its check."""
    t, big = Tree(hip, rng, [70], None, 2, 4, 2, 64), Tree(hip, rng, [500], None, 20, 4, 2, 64)
    a, q, k, v = prompt_case(hip, rng, 840, 0, 16, 1, 64, None)
    w = rng.random((2, 2, 100)).astype(F32)
    sel = lib.SelectArgs(weights=hip.up(w), lens=hip.up(np.array([100, 60], I32)), kept=hip.up(np.full((2, 2, 50), -9, I32)),
                         counts=hip.up(np.zeros(2, I32)), caches=2, kv_heads=2, max_rows=100, budget=50, sinks=1, recent=7)
    kp = Keep(rng, 2, 200, 2, 64)
    lists = ascending(rng, (2, 2), 100, 200)
    keep = kp.args(hip, lists, [100, 40], None, rows_out=120)
    return [(ctx.tree_attention, t.a, t.check), (ctx.cache_weights, t.a, t.check_weights),
            (ctx.tree_attention, big.a, big.check), (ctx.cache_weights, big.a, big.check_weights),
            (ctx.prompt_attention, a, lambda: check_prompt(hip, a, q, k, v, None, rows=np.arange(0, 840, 41))),
            (ctx.cache_select, sel, lambda: check_select(hip, sel, w, [100, 60])),
            (ctx.cache_keep, keep, lambda: kp.check(hip, keep, lists, [100, 40], None))]


def test_errors_of_others_are_theirs(ctx, rng):
    """A call that follows an error of the application's own, or one that these
    calls answered themselves (a stream they do not know), succeeds and says so."""
    with ref.Hip() as hip:
        calls = all_calls(ctx, hip, rng)
        hip.sync()
        no_stream = C.create_string_buffer(4096)  # an address that no stream has
        for call, args, check in calls:
            assert hip.rt.hipSetDevice(4711) != 0  # handled, and left behind as the thread's last error
            call(args)
            check()
            with pytest.raises(lib.PocrError) as e:
                call(args, C.addressof(no_stream))
            assert e.value.code == lib.POCR_ERR_ARG
        for call, args, check in all_calls(ctx, hip, rng):
            call(args)
            check()
        hip.rt.hipGetLastError()


@pytest.mark.parametrize("rows_out,first,side", [(1000, 3, False), (1000, 985, True), (360_000_000, 359_999_990, True)],
                         ids=["short", "short-weights", "long-weights"])
def test_keep_longest_lists(ctx, rng, rows_out, first, side):
    """Lists as long as the header allows, few of whose entries are in use; destinations
    whose workgroups pass 2^32 threads and whose weights' tail passes 31 bits with its steps."""
    with ref.Hip() as hip:
        free, total = C.c_size_t(), C.c_size_t()
        assert hip.rt.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
        if free.value < (200 << 30) and rows_out > 1000:
            pytest.skip("needs 200 GiB of device memory")
        count = min(20, rows_out - first)
        src = rng.standard_normal((2, 40, 64)).astype(F32)
        w = rng.random(40).astype(F32)
        pick = np.sort(rng.choice(40, 20, replace=False)).astype(I32)
        a = lib.KeepArgs(k=hip.up(src[0]), v=hip.up(src[1]), k_out=hip.raw(256 * rows_out), v_out=hip.raw(256 * rows_out),
                         rows=hip.raw(4 << 30), counts=hip.up(np.array([20], I32)), first=hip.up(np.array([first], I32)),
                         caches=1, kv_heads=1, head_dim=64, max_keep=2 ** 30, max_rows=40, max_rows_out=rows_out,
                         k_stride=64, v_stride=64, k_out_stride=64, v_out_stride=64)
        hip.write(a.rows, pick)
        at = max(0, first - 5)  # a window of the destination around the moved rows
        size = min(first + count + 5, rows_out) - at
        for p in (a.k_out, a.v_out):
            hip.write(p + 256 * at, np.full((size, 64), SENTINEL, F32))
        tails = {at, rows_out // 3, rows_out - 900} & set(range(rows_out - 899))
        if side:
            a.weights, a.weights_out = hip.up(w), hip.raw(4 * rows_out)
            for t in tails:
                hip.write(a.weights_out + 4 * t, np.full(900, SENTINEL, F32))
        ctx.cache_keep(a)
        for x, p in enumerate((a.k_out, a.v_out)):
            want = np.full((size, 64), SENTINEL, F32)
            want[first - at:first - at + count] = src[x, pick[:count]]
            assert np.array_equal(hip.down(p + 256 * at, (size, 64)), want)
        for t in tails if side else ():
            i = t + np.arange(900)
            moved = w[pick[np.clip(i - first, 0, count - 1)]]
            want = np.where(i < first, SENTINEL, np.where(i < first + count, moved, F32(0.0)))
            assert np.array_equal(hip.down(a.weights_out + 4 * t, 900), want), t


@pytest.mark.parametrize("n,heads", [(1, 2), (16, 2), (20, 16)], ids=["one", "few", "many"])
def test_tree_of_the_largest_bound(ctx, rng, n, heads):
    """max_rows is a bound: lengths far below it, workgroups past 2^32 threads."""
    with ref.Hip() as hip:
        t = Tree(hip, rng, [300], None, n, heads, 1, 64)
        t.a.max_rows, t.a.weights = 2 ** 30, hip.raw(4 << 30)
        hip.write(t.a.weights, t.weights)
        t.a.workspace_bytes = lib.tree_attention_workspace(t.a)
        t.a.workspace = hip.raw(t.a.workspace_bytes)
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


def test_keep_within_a_pool(ctx, rng):
    """Caches of all layers from one slot of a pool [layer][slot][K, V][row] into another; the other slots stay."""
    with ref.Hip() as hip:
        layers, slots, rows, st = 3, 4, 90, 2 * 64
        pool = rng.standard_normal((layers, slots, 2, rows, st)).astype(F32)
        lists = ascending(rng, (layers, 2), 70, rows)
        base, size = hip.up(pool), 4 * rows * st
        at = lambda slot, x: base + (2 * slot + x) * size  # noqa: E731
        a = lib.KeepArgs(k=at(2, 0), v=at(2, 1), k_out=at(1, 0), v_out=at(1, 1), rows=hip.up(lists), counts=hip.up(np.full(layers, 70, I32)),
                         caches=layers, kv_heads=2, head_dim=64, max_keep=70, per_head=1, max_rows=rows, max_rows_out=rows)
        for n in ("k", "v", "k_out", "v_out"):
            setattr(a, n + "_cache_stride", slots * 2 * rows * st)
            setattr(a, n + "_stride", st)
        ctx.cache_keep(a)
        want = pool.copy().reshape(layers, slots, 2, rows, 2, 64)
        src = want.copy()
        for c in range(layers):
            for g in range(2):
                want[c, 1, :, :70, g] = src[c, 2][:, lists[c, g], g]
        assert np.array_equal(hip.down(base, want.shape), want)


@pytest.mark.parametrize("n", [20, 300])
def test_keep_one_buffer_as_k_and_v(ctx, rng, n):
    """Elsewhere it moves to one destination as both; in place, where two workgroups would move each row, it is refused."""
    with ref.Hip() as hip:
        kp = Keep(rng, 2, 400, 2, 64)
        lists = ascending(rng, (2, 2), n, 400)
        a = kp.args(hip, lists, [n, n // 2], None, side=False)
        b = lib.KeepArgs.from_buffer_copy(a)
        a.v = a.v_out = a.k
        with pytest.raises(lib.PocrError) as e:
            ctx.cache_keep(a)
        assert e.value.code == lib.POCR_ERR_ARG
        assert np.array_equal(hip.down(a.k, kp.kv.shape), kp.kv)
        b.v, b.k_out = b.k, hip.up(np.full((2, n, 128), SENTINEL, F32))
        b.v_out, b.max_rows_out, b.k_out_cache_stride, b.v_out_cache_stride = b.k_out, n, n * 128, n * 128
        ctx.cache_keep(b)
        got = hip.down(b.k_out, (2, n, 2, 64))
        for c, count in enumerate((n, n // 2)):
            assert np.all(got[c, count:] == SENTINEL)
            for g in range(2):
                assert np.array_equal(got[c, :count, g], kp.part(kp.kv, 0)[c, lists[c, g, :count], g])


@pytest.mark.parametrize("max_rows", [2048, 2049, 8193, 16384, 16385, 70000])
def test_select_of_short_caches_in_long_buffers(ctx, rng, max_rows):
    """Lengths far below what the buffers hold, on both sides of one and of several tiles, in one call."""
    with ref.Hip() as hip:
        lens = [0, 51, 700, 2048, min(8192, max_rows), min(16384, max_rows), min(16385, max_rows), max_rows]
        w = rng.integers(0, 400, (len(lens), 2, max_rows)).astype(F32)
        for c, length in enumerate(lens):
            w[c, :, length:] = 1e6  # rows behind a cache's end weigh nothing
        a = run_select(ctx, hip, w, lens, 50, 4, 16)
        check_select(hip, a, w, lens)


@pytest.mark.parametrize("seqs,kvh,n,longest", [(140, 2, 1, 600), (300, 1, 3, 1500), (256, 1, 1, 4000)])
def test_tree_many_ragged_sequences(ctx, rng, seqs, kvh, n, longest):
    """Few rows of so many sequences that a tile has at most four shares: lengths from 0 on, sequences without tokens."""
    with ref.Hip() as hip:
        lens = rng.integers(0, longest, seqs)
        lens[:4] = 0, 1, longest - 1, longest
        t = Tree(hip, rng, lens, rng.integers(0, n + 1, seqs), n, 4 * kvh, kvh, 64, random_trees(rng, seqs, n))
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("seqs,kvh,n,longest", [(60, 2, 33, 900), (130, 1, 20, 1300), (90, 2, 33, 900)])
def test_tree_many_ragged_trees(ctx, rng, seqs, kvh, n, longest):
    """More rows: two or three tiles a sequence, of which counts leave some or all without rows, in two, three shares or one."""
    with ref.Hip() as hip:
        lens, counts = rng.integers(0, longest, seqs), rng.integers(0, n + 1, seqs)
        lens[:4], counts[:8] = (0, 1, longest - 1, longest), (n, n, n, n, 0, 1, 2, n)
        t = Tree(hip, rng, lens, counts, n, 8 * kvh, kvh, 64, random_trees(rng, seqs, n), slopes=alibi(8 * kvh))
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("n", [1, 12, 24])
def test_tree_one_long_sequence_among_short_ones(ctx, rng, n):
    with ref.Hip() as hip:
        lens = np.r_[rng.integers(0, 500, 15), 7900]
        t = Tree(hip, rng, lens, None, n, 8, 1, 64, random_trees(rng, 16, n))
        ctx.tree_attention(t.a)
        t.check()
        ctx.cache_weights(t.a)
        t.check_weights()


@pytest.mark.parametrize("n,rows0", [(33, 2000), (64, 8000), (300, 2000), (600, 0)])
@pytest.mark.parametrize("kind", ["causal", "docs"])
def test_prompt_chunks_behind_a_prefix(ctx, rng, n, rows0, kind):
    """Prompts of few tiles whose keys are cut into shares."""
    with ref.Hip() as hip:
        spans = spans_of(kind, n, rows0, rng)
        a, q, k, v = prompt_case(hip, rng, n, rows0, 16, 2, 64, spans)
        ctx.prompt_attention(a)
        check_prompt(hip, a, q, k, v, spans, rows=np.unique(np.r_[0, 1, np.arange(0, n, 17), n - 1]))

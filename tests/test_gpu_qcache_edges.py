"""The attention over caches in 4 or 8 bits at the ends of the ranges that its
header states.  Definitions and bounds: qcache_f64.py."""
import threading

import cache_ops_f64 as base
import numpy as np
import pytest
from test_gpu_qcache import F32, SENTINEL, U, Attend, Rows

from rapidocrvl_amd import lib

pytestmark = pytest.mark.gpu


def heads_of(a, s=0):
    """Head, its query rows, its keys' and values' (step * code, mid), and what each token sees."""
    _, n, rows, heads, kvh, hd = a.shape
    dist = (int(a.lens[s]) - n + np.arange(n))[:, None] - np.arange(rows)
    seen = (dist >= 0) & (dist < (a.window or rows))
    for h in range(heads):
        g = h // (heads // kvh)
        yield h, a.q[s, :, h * hd:(h + 1) * hd].astype(np.float64), *([x[i][s, g] for i in (0, 1)] for x in (a.k, a.v)), seen


def weigh(s, seen, v):
    """Scores that the device has exactly → out, lse and the bounds of their errors, as
    qcache_f64.attention without an error of the scores."""
    va, vb = v
    s = np.where(seen, s, -np.inf)
    m = s.max(1, keepdims=True)
    e = np.exp(s - m)
    total = e.sum(1, keepdims=True)
    p, lse = e / total, m[:, 0] + np.log(total[:, 0])
    steps = (seen.sum(1) / 16 + 32) * U
    d = np.where(seen, (m - np.where(seen, s, m)) * 2 * U + 2 * U, 0.0)
    rows = (p * d).sum(1) + steps
    size = np.abs(va) + np.abs(vb)
    out_err = (p * (d + rows[:, None])) @ size + (p @ size) * (2.0 ** -21 + steps[:, None] + 2 * U) + 1e-38
    out_err += (np.where(seen, size.max(1), 0.0).max(1) * seen.sum(1))[:, None] * 2.0 ** -32
    return p @ (va + vb), lse, out_err, rows + np.abs(lse) * 4 * U + 2 * U


VALUES = {"one": lambda rng, *shape: rng.standard_normal(shape), "large": lambda rng, *shape: rng.uniform(-6e4, 6e4, shape),
          "small": lambda rng, *shape: rng.standard_normal(shape) * 1e-5}


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("far", [21, 22, 23, 25, 26, -22, -23, -25, 40])
@pytest.mark.parametrize("n", [1, 40], ids=["few", "many"])
@pytest.mark.parametrize("hd,bits,bias", [(128, 4, False), (128, 8, False), (64, 4, True), (128, 4, True)])
def test_scores_that_differ_little_far_from_zero(ctx, rng, hd, bits, bias, n, far, values):
    """Scores of 2^far + unit * (16 + t) to the base 2, t from -8 on and up to 5 in later
    blocks, unit a step of fp32 there and 1 or more.  They are exact on the device: the scale
    times log2(e) is 1; a key row's group has the midpoint 16 and the step 1; the sum of the
    query row is the large part, and only its small element meets codes other than zero.  So
    weights are 2^(unit * t), whatever the values' size."""
    with base.Hip() as hip:
        rows, half = 400, 1 << (bits - 1)
        unit = 2.0 ** max(0, abs(far) - 23)
        t = np.where(np.arange(rows) < 200, rng.integers(-8, 1, rows), rng.integers(-8, 6, rows))
        k = np.full((1, 1, rows, hd), 16.0, F32)
        k[0, 0, :, 1] += t
        k[..., 3], k[..., 4] = 16 - half, 16 + half - 1
        q = np.zeros((1, n, 2, hd), F32)
        q[..., 1], q[..., 2] = unit, np.sign(far) * 2.0 ** (abs(far) - 4)
        v = VALUES[values](rng, 1, 1, rows, hd).astype(F32)
        a = Attend(hip, rng, 1, n, rows, 2, 1, hd, bits, q=q.reshape(1, n, -1), k=k, v=v, scale=F32(np.log(2)),
                   slopes=np.zeros(2, F32) if bias else None)
        assert np.array_equal(a.k[1][0, 0, :, :64], np.full((rows, 64), 16.0)) and np.array_equal(a.k[0][0, 0, :, 1], t)
        out, lse = a.run(ctx).got()
        for h, x, (ka, kb), v, seen in heads_of(a):
            o, e, ob, eb = weigh(x @ (ka + kb).T * a.scale, seen, v)
            base.close(out[0, :, h * hd:(h + 1) * hd], o, ob, f"out of head {h}")
            base.close(lse[0, :, h], e, eb, f"lse of head {h}")


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 24, 2.0 ** 40, 2.0 ** 80])
@pytest.mark.parametrize("n,hd,bits", [(1, 128, 4), (20, 128, 4), (70, 128, 8), (20, 64, 8), (70, 64, 4)])
def test_the_one_key_of_far_scores(ctx, rng, n, hd, bits, size, values):
    """Where the largest score stands above the next by more than both errors and 90 (a
    weight of e^-90), out is that key's value row, and lse its score."""
    with base.Hip() as hip:
        rows = 300
        q = (rng.standard_normal((1, n, 2 * hd)) * size).astype(F32)
        v = VALUES[values](rng, 1, 1, rows, hd).astype(F32)
        a = Attend(hip, rng, 1, n, rows, 2, 1, hd, bits, q=q, v=v)
        out, lse = a.run(ctx).got()
        clear = 0
        for h, x, (ka, kb), (va, vb), seen in heads_of(a):
            s = x @ (ka + kb).T * a.scale
            key = np.abs(ka) + np.abs(kb)
            err = np.abs(x) @ key.T * a.scale * (17 * U + 2.0 ** -21) + np.abs(s) * 4 * U
            err = (err + a.scale * 2.0 ** -32 * np.abs(x).max(1)[:, None] * key.sum(1)).max(1)
            s = np.where(seen, s, -np.inf)
            at, two = s.argmax(1), np.sort(s, 1)[:, -2:]
            one = two[:, 1] - two[:, 0] > 2 * err + 90
            clear += one.sum()
            o, w = out[0, :, h * hd:(h + 1) * hd], (va + vb)[at]
            bound = (np.abs(va) + np.abs(vb))[at] * (2.0 ** -21 + 40 * U) + (np.abs(va) + np.abs(vb)).max() * 2.0 ** -32
            assert np.isfinite(o).all() and np.isfinite(lse).all()
            assert np.all((np.abs(o - w) <= bound)[one])
            assert np.all(np.abs(lse[0, :, h] - two[:, 1]) <= err + np.abs(two[:, 1]) * 4 * U + 2 * U + np.log(rows))
        assert clear >= n


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("n,heads", [(8, 2), (15, 2), (40, 2), (24, 8)])
@pytest.mark.parametrize("hd,bits", [(128, 4), (128, 8), (64, 4)])
def test_values_that_a_row_does_not_see_cost_it_nothing(ctx, rng, hd, bits, n, heads, window, cap):
    """Values of about 1e-3, and one row of up to 65504 in the block of the last tokens' own
    rows (no window), or in one that the window of most has left: the other tokens keep
    their precision."""
    with base.Hip() as hip:
        rows = 200
        v = (rng.standard_normal((1, 1, rows, hd)) * 1e-3).astype(F32)
        first = rows - n
        v[0, 0, first - window + 4 if window else rows - 3, 7::64] = 65504.0
        Attend(hip, rng, 1, n, rows, heads, 1, hd, bits, window=window, cap=cap, v=v).run(ctx).check()


def shares(a):
    """Key shares of a call, from its workspace: [tiles of so many rows][share][sums, reference, denominator]."""
    seqs, n, _, heads, kvh, hd = a.shape
    rows = n * (heads // kvh)
    tile = 16 if rows <= 16 else 32 if rows <= 32 else 64
    tiles = -(-rows // tile) * kvh * seqs
    assert a.args.workspace_bytes % (tiles * tile * (hd + 2) * 4) == 0
    return a.args.workspace_bytes // (tiles * tile * (hd + 2) * 4)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,heads,kvh,hd,rows", [
    (1, 4, 2, 64, 1100), (1, 4, 2, 64, 3000), (12, 4, 2, 64, 1100), (12, 8, 8, 64, 3000), (70, 4, 2, 64, 1100), (70, 8, 8, 64, 3000),
    (1, 16, 2, 128, 640), (2, 16, 2, 128, 900), (3, 16, 2, 128, 300), (3, 16, 2, 128, 700), (4, 16, 2, 128, 700),
    (4, 16, 2, 128, 5000), (3, 16, 2, 128, 5000), (6, 16, 2, 128, 200), (20, 4, 1, 128, 1500)])
def test_shares_of_ragged_sequences(ctx, rng, bits, n, heads, kvh, hd, rows):
    """Keys in shares and their join, in every kind of tile; sequences that end before their first or last share."""
    with base.Hip() as hip:
        lens = [rows, rows // 2 + 1, 40, rows - 33, 0]
        a = Attend(hip, rng, 5, n, rows, heads, kvh, hd, bits, lens=lens, counts=[n, n, n, max(1, n - 1), n], pad=4, capacity=rows + 7)
        assert shares(a) > 1
        a.run(ctx).check(np.unique([0, n // 2, n - 2, n - 1])[-4:] % n, [0, heads - 1])


@pytest.mark.parametrize("cap,bias", [(0.0, False), (30.0, True)], ids=["plain", "cap-bias"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,heads,kvh,hd,window", [(1, 16, 2, 128, 700), (1, 4, 2, 64, 2000), (4, 16, 2, 128, 700), (4, 16, 2, 128, 2001),
                                                   (3, 8, 1, 64, 1033), (33, 4, 2, 128, 700)])
def test_shares_of_windows(ctx, rng, bits, n, heads, kvh, hd, window, cap, bias):
    """The first share begins where the window of the tile's first token does, in the middle of a block."""
    with base.Hip() as hip:
        slopes = np.array([2.0 ** (-0.7 * (h + 3)) for h in range(heads)], F32) if bias else None
        a = Attend(hip, rng, 3, n, 5000, heads, kvh, hd, bits, lens=[5000, 4011, 600], window=window, cap=cap, slopes=slopes)
        assert shares(a) > 1
        a.run(ctx).check(np.unique([0, n - 1]), [0, heads - 1])


@pytest.mark.parametrize("seqs,rows,most", [(1, 600, 5), (8, 1100, 9), (40, 1100, 6), (80, 900, 3), (120, 1500, 2)])
def test_few_shares_of_few_rows(ctx, rng, seqs, rows, most):
    """Two to nine shares, the fewer the more sequences there are: joined two or eight at a time."""
    with base.Hip() as hip:
        a = Attend(hip, rng, seqs, 1, rows, 4, 2, 128, 4, lens=rows - 7 * np.arange(seqs))
        assert 1 < shares(a) <= most
        a.run(ctx).check(heads_at=[0, 3])


@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("seqs,kvh,hd,bits", [(130, 2, 64, 4), (33, 8, 128, 4), (33, 8, 128, 8)])
def test_long_caches_of_many_sequences(ctx, rng, seqs, kvh, hd, bits, n):
    """So many (sequence, KV head) pairs that each takes one workgroup, whatever its length."""
    with base.Hip() as hip:
        rows = 1300
        a = Attend(hip, rng, seqs, n, rows, 4 * kvh, kvh, hd, bits, lens=rows - 9 * np.arange(seqs))
        assert shares(a) == 0
        a.run(ctx).check(np.array([0, n - 1]), [0, 4 * kvh - 1])


FORMS = [(2, 1, 300), (2, 1, 2500), (2, 3, 200), (2, 3, 600), (1, 70, 100), (2, 70, 900)]  # each tile, in one launch and in shares


def fresh(a):
    """The same call into buffers that hold nothing but the sentinel."""
    seqs, n, _, heads, _, hd = a.shape
    args = lib.QAttentionArgs.from_buffer_copy(a.args)
    args.out, args.lse = a.hip.up(np.full((seqs, n, heads * hd), SENTINEL, F32)), a.hip.up(np.full((seqs, n, heads), SENTINEL, F32))
    return args


@pytest.mark.parametrize("seqs,n,rows", FORMS)
def test_a_call_without_lse_writes_its_rows_and_no_lse(ctx, rng, seqs, n, rows):
    with base.Hip() as hip:
        a = Attend(hip, rng, seqs, n, rows, 16, 2, 128, 4).run(ctx)
        args = fresh(a)
        lse, args.lse = args.lse, None
        ctx.qcache_attention(args, a.cache.args)
        assert np.all(hip.down(lse, (seqs, n, 16)) == SENTINEL)
        a.args.out = args.out
        a.check(heads_at=[0, 15])


@pytest.mark.parametrize("seqs,n,rows", FORMS)
def test_each_call_writes_the_same(ctx, rng, seqs, n, rows):
    """The same call several times, each into buffers of its own: equal to the last bit."""
    with base.Hip() as hip:
        a = Attend(hip, rng, seqs, n, rows, 16, 2, 128, 4).run(ctx).check(heads_at=[0, 15])
        out, lse = a.got()
        for _ in range(4):
            args = fresh(a)
            ctx.qcache_attention(args, a.cache.args)
            assert np.array_equal(hip.down(args.out, out.shape), out) and np.array_equal(hip.down(args.lse, lse.shape), lse)


def test_threads_write_each_their_own(ctx, rng):
    """Calls from four threads on streams of their own, workspaces of their own, each call
    into buffers of its own: all as when alone."""
    with base.Hip() as hip:
        work = [Attend(hip, rng, 2, n, rows, 16, 2, 128, 4).run(ctx) for n, rows in ((1, 700), (5, 400), (40, 300), (1, 2500))]
        calls = [[fresh(a) for _ in range(8)] for a in work]
        streams = [hip.stream() for _ in work]
        fails = []

        def run(a, args, stream):
            try:
                for x in args:
                    ctx.qcache_attention(x, a.cache.args, stream)
            except Exception as e:  # noqa: BLE001
                fails.append(e)

        threads = [threading.Thread(target=run, args=x) for x in zip(work, calls, streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not fails
        for a, args in zip(work, calls):
            out, lse = a.check(heads_at=[0, 15]).got()
            for x in args:
                assert np.array_equal(hip.down(x.out, out.shape), out) and np.array_equal(hip.down(x.lse, lse.shape), lse)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("hd,rotary,adjacent", [(128, 0, 0), (128, 64, 0), (64, 32, 1)])
def test_norm_of_an_infinite_element(ctx, rng, hd, rotary, adjacent, sign):
    """x / sqrt(mean(x^2) + eps) of a head with an infinity: zeros, and NaN in its own place
    and that of the other element of its pair."""
    with base.Hip() as hip:
        q = rng.standard_normal((1, 3, 2 * hd)).astype(F32)
        q[0, 1, 5] = sign * np.inf
        r = Rows(hip, rng, 1, 3, 2, 1, hd, rotary, 1, norms=True, q=q, adjacent=adjacent)
        ctx.rotate_rows(r.args)
        got = r.got("q")[0]
        bad = np.zeros(hd, bool)
        bad[5] = True
        if rotary:
            bad[4 if adjacent else 5 + rotary // 2] = True
        assert np.array_equal(np.isnan(got[1, :hd]), bad) and np.all(got[1, :hd][~bad] == 0.0)
        assert np.isfinite(np.delete(got.reshape(3, 2, hd).reshape(6, hd), 2, 0)).all()


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("far", [22, -22])
@pytest.mark.parametrize("n,rows", [(1, 400), (1, 1500), (3, 700), (40, 400)])
@pytest.mark.parametrize("hd,bits,bias,window", [(128, 4, False, 0), (128, 8, True, 0), (64, 4, False, 0), (128, 4, True, 250)])
def test_scores_on_both_sides_of_where_far_begins(ctx, rng, hd, bits, bias, window, n, rows, far, values):
    """As above with scores of 2^22 + t (-2^22 + t), t rising by 13 over the rows: references
    pass from near to far (from far to near), in one wave and from share to share."""
    with base.Hip() as hip:
        half = 1 << (bits - 1)
        t = np.clip(np.arange(rows) * 14 // rows - 8 + rng.integers(-1, 2, rows), -8, 5)
        k = np.full((1, 1, rows, hd), 16.0, F32)
        k[0, 0, :, 1] += t
        k[..., 3], k[..., 4] = 16 - half, 16 + half - 1
        q = np.zeros((1, n, 2, hd), F32)
        q[..., 1], q[..., 2] = 1.0, np.sign(far) * 2.0 ** (abs(far) - 4) - 1.0
        v = VALUES[values](rng, 1, 1, rows, hd).astype(F32)
        a = Attend(hip, rng, 1, n, rows, 2, 1, hd, bits, q=q.reshape(1, n, -1), k=k, v=v, scale=F32(np.log(2)),
                   slopes=np.zeros(2, F32) if bias else None, window=window)
        out, lse = a.run(ctx).got()
        for h, x, (ka, kb), v, seen in heads_of(a):
            o, e, ob, eb = weigh(x @ (ka + kb).T * a.scale, seen, v)
            base.close(out[0, :, h * hd:(h + 1) * hd], o, ob, f"out of head {h}")
            base.close(lse[0, :, h], e, eb, f"lse of head {h}")

"""Rotation of rows, caches in 4 or 8 bits and the attention over them, on the
device against their definitions in 64 bits (qcache_f64.py, with the bounds)."""
import threading

import cache_ops_f64 as base
import numpy as np
import pytest
import qcache_f64 as ref

from rapidocrvl_amd import lib

pytestmark = pytest.mark.gpu
F32, I32, U = np.float32, np.int32, 2.0 ** -24
SENTINEL = F32(-77.25)  # what untouched places hold


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------


class Rows:
    """A call's buffers and arguments; rows `pad` floats apart beyond their width."""

    def __init__(self, hip, rng, seqs, n, heads, kvh, hd, rotary=0, axes=3, sections=None, interleaved=0, adjacent=0,
                 norms=False, counts=None, first=None, pad=0, q=None, k=None, v=None, positions=None, theta=500000.0,
                 max_rows=None, cache=None, eps=1e-5):
        self.hip, self.cache = hip, cache
        self.shape = (seqs, n, heads, kvh, hd)
        self.counts = None if counts is None else np.asarray(counts, I32)
        self.first = None if first is None else np.asarray(first, I32)
        self.count = [n if counts is None else min(max(int(c), 0), n) for c in (counts if counts is not None else [n] * seqs)]
        self.max_rows = max_rows or n
        limit = cache.capacity if cache else self.max_rows
        self.at = [0 if first is None else min(max(int(f), 0), limit - c) for f, c in zip(first if first is not None else [0] * seqs, self.count)]
        self.rotary, self.adjacent, self.eps = rotary, adjacent, eps
        a = lib.RowsArgs(seqs=seqs, n=n, heads=heads, kv_heads=kvh, head_dim=hd, eps=eps, max_rows=0 if cache else self.max_rows)
        self.src = {}
        for w, h, x in (("q", heads, q), ("k", kvh, k), ("v", kvh, v)):
            if not h:
                continue
            if x is None:
                x = rng.standard_normal((seqs, n, h * hd)).astype(F32) * F32(2.5 if w == "q" else 0.64)
            full = np.full((seqs, n, h * hd + pad), SENTINEL, F32)
            full[..., :h * hd] = x
            self.src[w] = x
            setattr(a, w, hip.up(full))
            setattr(a, w + "_stride", full.shape[2])
            setattr(a, w + "_seq_stride", full.shape[1] * full.shape[2])
            if cache and w != "q":
                continue
            rows = n if w == "q" else self.max_rows
            setattr(a, w + "_out", hip.up(np.full((seqs, rows, h * hd + pad), SENTINEL, F32)))
            setattr(a, w + "_out_stride", h * hd + pad)
            setattr(a, w + "_out_seq_stride", rows * (h * hd + pad))
        self.pad = pad
        self.norm = {}
        if norms:
            for w in ("q", "k"):
                self.norm[w] = (1 + 0.3 * rng.standard_normal(hd)).astype(F32)
                setattr(a, w + "_norm", hip.up(self.norm[w]))
        self.angle = None
        if rotary:
            half = rotary // 2
            if sections is None:
                each = half // axes - 1 if interleaved else half // axes
                sections = [half - each * (axes - 1)] + [each] * (axes - 1)
            if positions is None:
                positions = rng.integers(0, 3000, (seqs, n, axes)).astype(I32)
            freqs = theta ** (-np.arange(half) * 2.0 / rotary)
            axis = ref.axes_of(half, axes, sections, interleaved)
            self.angle = positions.astype(np.float64)[..., axis] * freqs
            a.positions, a.freqs = hip.up(positions), hip.up(freqs)
            a.rotary_dim, a.axes, a.interleaved, a.adjacent = rotary, axes, interleaved, adjacent
            a.sections[:axes] = [int(x) for x in sections]
        if self.counts is not None:
            a.counts = hip.up(self.counts)
        if self.first is not None:
            a.first = hip.up(self.first)
        self.args = a

    def want(self, w, s):
        """Live rows of one sequence, and each element's bound."""
        n, hd = self.count[s], self.shape[4]
        x = self.src[w][s, :n].reshape(n, self.shape[2 if w == "q" else 3], hd)
        if w == "v":
            return x.reshape(n, x.shape[1] * hd), np.zeros((n, x.shape[1] * hd))
        y = [ref.rotate(x[:, h], self.norm.get(w), self.eps, None if self.angle is None else self.angle[s, :n], self.adjacent)
             for h in range(x.shape[1])]
        y, size = (np.stack(z, 1).reshape(n, x.shape[1] * hd) for z in zip(*y))
        exact = not self.norm.get(w, np.zeros(0)).size and self.angle is None
        return y, np.zeros(y.shape) if exact else np.abs(y) * U * (1 + 2.0 ** -20) + size * 2.0 ** -48 + 2.0 ** -149

    def got(self, w):
        h = self.shape[2] if w == "q" else self.shape[3]
        rows = self.shape[1] if w == "q" else self.max_rows
        return self.hip.down(getattr(self.args, w + "_out"), (self.shape[0], rows, h * self.shape[4] + self.pad))

    def check(self, which):
        for w in which:
            got = self.got(w)
            width = got.shape[2] - self.pad
            assert np.all(got[..., width:] == SENTINEL), w
            for s in range(self.shape[0]):
                at = 0 if w == "q" else self.at[s]
                y, bound = self.want(w, s)
                err = np.abs(got[s, at:at + self.count[s], :width].astype(np.float64) - y)
                assert np.all(err <= bound), (w, s, float((err / np.maximum(bound, 1e-300)).max()))
                rest = np.delete(got[s], slice(at, at + self.count[s]), 0)
                assert np.all(rest == SENTINEL), (w, s)


HEADS = [(16, 2, 128), (4, 2, 64), (8, 8, 64), (7, 1, 128), (1, 1, 64)]


@pytest.mark.parametrize("heads,kvh,hd", HEADS)
@pytest.mark.parametrize("seqs,n", [(1, 1), (1, 5), (3, 1), (2, 67), (16, 3)])
def test_rotate(ctx, rng, heads, kvh, hd, seqs, n):
    with base.Hip() as hip:
        r = Rows(hip, rng, seqs, n, heads, kvh, hd, rotary=hd, pad=4 * (n % 3))
        ctx.rotate_rows(r.args)
        r.check("qkv")


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("hd,rotary,axes,sections,interleaved,adjacent", [
    (128, 128, 1, None, 0, 0), (128, 128, 3, (16, 24, 24), 0, 0), (128, 128, 3, (24, 20, 20), 1, 0), (128, 128, 4, (10, 0, 27, 27), 0, 1),
    (128, 64, 2, (1, 31), 0, 0), (128, 112, 3, None, 0, 0), (128, 16, 1, None, 0, 1), (128, 48, 4, None, 1, 1), (128, 0, 0, None, 0, 0),
    (64, 64, 3, (8, 12, 12), 0, 0), (64, 64, 4, None, 1, 0), (64, 32, 2, None, 1, 1), (64, 16, 1, None, 0, 0), (64, 48, 3, (0, 0, 24), 0, 0)])
def test_rotate_forms(ctx, rng, hd, rotary, axes, sections, interleaved, adjacent, norms):
    with base.Hip() as hip:
        r = Rows(hip, rng, 2, 19, 6, 2, hd, rotary, axes, sections, interleaved, adjacent, norms, counts=[19, 11])
        ctx.rotate_rows(r.args)
        r.check("qkv")


@pytest.mark.parametrize("counts,first", [([4, 0, 9, -3], None), ([9, 40, 1, 2], [0, 5, 30, 100]), (None, [-7, 2, 31, 2 ** 31 - 1])])
def test_rotate_appends(ctx, rng, counts, first):
    """Ragged counts and places out of range: forced into it, nothing else written."""
    with base.Hip() as hip:
        r = Rows(hip, rng, 4, 9, 4, 2, 128, 128, counts=counts, first=first, max_rows=31, pad=8)
        ctx.rotate_rows(r.args)
        r.check("qkv")


@pytest.mark.parametrize("which", ["q", "k", "v", "qk", "kv"])
def test_rotate_some(ctx, rng, which):
    with base.Hip() as hip:
        r = Rows(hip, rng, 2, 21, 5, 3, 64, 64, norms=True)
        for w in "qkv":
            if w not in which:
                setattr(r.args, w, None)
                setattr(r.args, w + "_out", None)
        ctx.rotate_rows(r.args)
        r.check(which)


def test_rotate_in_place(ctx, rng):
    with base.Hip() as hip:
        for kw in (dict(hd=128, rotary=128), dict(hd=128, rotary=96, norms=True), dict(hd=64, rotary=64, adjacent=1)):
            r = Rows(hip, rng, 2, 33, 6, 2, **kw)
            a = r.args
            for w in "qkv":
                setattr(a, w + "_out", getattr(a, w))
            ctx.rotate_rows(a)
            r.check("qkv")


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 24 + 1, 2 ** 31 - 1])
def test_rotate_far_positions(ctx, rng, far):
    """Angles of far and of negative positions: their turn is exact to 2^-20."""
    with base.Hip() as hip:
        pos = np.array([far, -far, 0, far - 1], I32).reshape(1, 4, 1)
        r = Rows(hip, rng, 1, 4, 2, 1, 128, 128, 1, positions=pos)
        ctx.rotate_rows(r.args)
        got = r.got("q")[0]
        for t in range(4):
            y, bound = r.want("q", 0)
            pair = np.abs(r.src["q"][0, t].reshape(2, 2, 64)).sum(1, keepdims=True).repeat(2, 1).reshape(-1)
            slack = pair * (2 * np.pi * 2.0 ** -20 if far > 2 ** 24 + 1 else 2.0 ** -27)
            assert np.all(np.abs(got[t] - y[t]) <= bound[t] + slack), t


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_rotate_bad_values_stay_in_their_head(ctx, rng, bad):
    with base.Hip() as hip:
        for norms in (False, True):
            q = rng.standard_normal((1, 5, 256)).astype(F32)
            q[0, 2, 3] = bad
            r = Rows(hip, rng, 1, 5, 2, 1, 128, 128, norms=norms, q=q)
            ctx.rotate_rows(r.args)
            got = r.got("q")[0]
            assert not np.isfinite(got[2, :128]).all() and np.isfinite(got[2, 128:]).all() and np.isfinite(got[[0, 1, 3, 4]]).all()


def test_rotate_zero_rows_and_eps(ctx, rng):
    """Normed rows of zeros are zeros where eps is not; large and tiny rows have their norm."""
    with base.Hip() as hip:
        q = rng.standard_normal((1, 4, 128)).astype(F32) * np.array([0, 1e30, 1e-25, 1], F32)[:, None]
        r = Rows(hip, rng, 1, 4, 1, 1, 128, 128, norms=True, q=q)
        ctx.rotate_rows(r.args)
        r.check("qk")


# ---------------------------------------------------------------------------
# caches
# ---------------------------------------------------------------------------


class Cache:
    """A cache's buffers, filled with `fill`; content() takes them apart."""

    def __init__(self, hip, seqs, kvh, hd, capacity, bits, seq_pad=0, fill=0xC3):
        self.hip, self.capacity, self.bits = hip, capacity, bits
        self.shape = (seqs, kvh, hd)
        self.seq_rows = kvh * capacity + seq_pad
        self.raw = {}
        for w in "kv":
            self.raw[w] = (hip.up(np.full((seqs * self.seq_rows, hd * bits // 8), fill, np.uint8)),
                           hip.up(np.full((seqs * self.seq_rows, hd // 16), fill, np.uint8)))
        self.args = lib.QCache(k_codes=self.raw["k"][0], v_codes=self.raw["v"][0], k_params=self.raw["k"][1],
                               v_params=self.raw["v"][1], seq_stride=self.seq_rows if seq_pad else 0, seqs=seqs, kv_heads=kvh,
                               head_dim=hd, capacity=capacity, bits=bits)

    def bytes_of(self, w):
        seqs, _, hd = self.shape
        return (self.hip.down(self.raw[w][0], (seqs, self.seq_rows, hd * self.bits // 8), np.uint8),
                self.hip.down(self.raw[w][1], (seqs, self.seq_rows, hd // 32), np.uint16))

    def put(self, w, x):
        """Rows x [seqs][kvh][rows][hd] (fp32) from the definition; → (step * code, mid) of them."""
        seqs, kvh, hd = self.shape
        codes, params = ref.quantise(x, self.bits)
        c, p = self.bytes_of(w)
        c = c[:, :kvh * self.capacity].reshape(seqs, kvh, self.capacity, -1)
        p = p[:, :kvh * self.capacity].reshape(seqs, kvh, self.capacity, -1)
        c[:, :, :x.shape[2]] = ref.pack(codes, w, self.bits)
        p[:, :, :x.shape[2]] = params.view(np.uint16)
        full_c = np.zeros((seqs, self.seq_rows, c.shape[-1]), np.uint8)
        full_p = np.zeros((seqs, self.seq_rows, p.shape[-1]), np.uint16)
        full_c[:, :kvh * self.capacity] = c.reshape(seqs, -1, c.shape[-1])
        full_p[:, :kvh * self.capacity] = p.reshape(seqs, -1, p.shape[-1])
        self.hip.write(self.raw[w][0], full_c)
        self.hip.write(self.raw[w][1], full_p)
        return ref.values(codes, params, self.bits, parts=True)


def check_written(cache, w, rows, at, count):
    """The cache's bytes: fp32 rows [seqs][n][kvh * hd] of live tokens at their places, the rest untouched."""
    seqs, kvh, hd = cache.shape
    codes, params = cache.bytes_of(w)
    touched = np.zeros(codes.shape[:2], bool)
    for s in range(seqs):
        x = rows[s, :count[s]].reshape(count[s], kvh, hd)
        c, p = ref.quantise(x, cache.bits)
        for g in range(kvh):
            i = g * cache.capacity + at[s]
            got_c, got_p = codes[s, i:i + count[s]], params[s, i:i + count[s]]
            bad = np.isnan(p[:, g])
            assert np.array_equal(got_c, ref.pack(c[:, g], w, cache.bits)), (w, s, g)
            assert np.array_equal(got_p[~bad], p[:, g].view(np.uint16)[~bad]) and np.isnan(got_p.view(np.float16)[bad]).all(), (w, s, g)
            touched[s, i:i + count[s]] = True
    assert np.all(codes[~touched] == 0xC3) and np.all(params[~touched] == 0xC3C3), w


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kvh,hd", [(16, 2, 128), (4, 2, 64), (0, 3, 128), (0, 5, 64)])
@pytest.mark.parametrize("seqs,n,counts,first,capacity,pad", [
    (1, 1, None, None, 1, 0), (1, 40, None, None, 43, 0), (3, 1, [1, 1, 1], [0, 8, 12], 13, 5), (4, 9, [9, 0, 4, 77], [2, 3, -5, 900], 31, 0)])
def test_write(ctx, rng, bits, heads, kvh, hd, seqs, n, counts, first, capacity, pad):
    """Codes and parameters to the bit; rows of others, behind and between sequences stay."""
    with base.Hip() as hip:
        cache = Cache(hip, seqs, kvh, hd, capacity, bits, pad)
        r = Rows(hip, rng, seqs, n, heads, kvh, hd, counts=counts, first=first, cache=cache, pad=pad - pad % 4)
        ctx.qcache_write(r.args, cache.args)
        for w in "kv":
            check_written(cache, w, r.src[w], r.at, r.count)
        if heads:
            r.check("q")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kw", [dict(hd=128, rotary=128, sections=(16, 24, 24)), dict(hd=128, rotary=128, norms=True, interleaved=1),
                                dict(hd=128, rotary=64, axes=2, adjacent=1, norms=True), dict(hd=64, rotary=64, norms=True)])
@pytest.mark.parametrize("seqs,n", [(1, 1), (2, 130), (16, 1)])
def test_written_rows_are_the_rotated_ones(ctx, rng, bits, kw, seqs, n):
    """What pocr_rotate_rows gives is what is held, to the bit, and q is the same in both."""
    with base.Hip() as hip:
        hd, capacity = kw["hd"], n + 7
        cache = Cache(hip, seqs, 2, hd, capacity, bits)
        first = rng.integers(0, 8, seqs)
        rot = Rows(hip, rng, seqs, n, 6, 2, max_rows=capacity, first=first, **kw)
        ctx.rotate_rows(rot.args)
        rot.check("qkv")
        a = rot.args
        q = hip.up(np.zeros((seqs, n, 6 * hd), F32))
        k_out, q_out = rot.got("k"), rot.got("q")
        a.k_out, a.v_out, a.q_out = None, None, q
        ctx.qcache_write(a, cache.args)
        k = np.stack([k_out[s, f:f + n] for s, f in enumerate(rot.at)])
        check_written(cache, "k", k, rot.at, rot.count)
        check_written(cache, "v", rot.src["v"], rot.at, rot.count)
        assert np.array_equal(hip.down(q, (seqs, n, 6 * hd)), q_out)


def special_rows(rng, hd):
    """Rows whose groups are what quantisation meets at its ends."""
    x = [rng.standard_normal(hd) * 10.0 ** e for e in (-42, -30, -9, -7, -4, 0, 3, 4, 5, 12, 38)]
    x += [np.zeros(hd), np.full(hd, 0.1), np.full(hd, -7.0), np.full(hd, 1e9), np.full(hd, 3e-8), np.full(hd, -3e38)]
    x += [np.where(np.arange(hd) % 2, 65504.0, -65504.0), np.where(np.arange(hd) % 64, 1.0, 1e6), np.linspace(0, 1, hd) + 1000]
    x += [np.arange(hd) % 16 - 8.0, (np.arange(hd) % 31 - 15) * 0.5, (np.arange(hd) % 64 - 32) * 0.25, np.arange(hd) % 64 * 4.0]
    x += [np.where(np.arange(hd) == 5, 1.0, 0.0), np.where(np.arange(hd) == 5, -0.0, 0.0), rng.integers(-127, 128, hd) / 2.0]
    for bad in (np.nan, np.inf, -np.inf):
        y = rng.standard_normal(hd)
        y[hd - 3] = bad
        x.append(y)
    with np.errstate(over="ignore"):
        return np.array(x).astype(F32)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [64, 128])
def test_write_special_rows(ctx, rng, bits, hd):
    """Subnormal, huge, constant and tied groups, zeros, NaN and infinities."""
    with base.Hip() as hip:
        x = special_rows(rng, hd)
        n = len(x)
        k, v = x.reshape(1, n, hd), x[::-1].reshape(1, n, hd)
        cache = Cache(hip, 1, 1, hd, n, bits)
        r = Rows(hip, rng, 1, n, 0, 1, hd, k=k, v=v, cache=cache)
        ctx.qcache_write(r.args, cache.args)
        check_written(cache, "k", k, r.at, r.count)
        check_written(cache, "v", v, r.at, r.count)


@pytest.mark.parametrize("bits,lo,hi", [
    (8, "-0x1.f4ede0p-1", "0x1.86a352p+0"), (8, "-0x1.84bd1ap+0", "0x1.dd7f78p+0"), (8, "-0x1.cdc304p+0", "0x1.89eff6p+0"),
    (4, "-0x1.fe25a20000000p+0", "0x1.041bee0000000p+0")])
def test_midpoints_are_rounded_twice(ctx, rng, bits, lo, hi):
    """Midpoints whose fp32 lies halfway between two fp16 numbers and whose 64 bits do not."""
    with base.Hip() as hip:
        lo, hi = float.fromhex(lo), float.fromhex(hi)
        x = np.concatenate([[lo, hi], rng.uniform(lo, hi, 62)]).astype(F32).reshape(1, 1, 64)
        cache = Cache(hip, 1, 1, 64, 1, bits)
        r = Rows(hip, rng, 1, 1, 0, 1, 64, k=x, v=x[..., ::-1].copy(), cache=cache)
        ctx.qcache_write(r.args, cache.args)
        for w in "kv":
            check_written(cache, w, r.src[w], r.at, r.count)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("scale", [1e-3, 0.64, 300.0])
def test_values_are_within_half_a_step(ctx, rng, bits, scale):
    with base.Hip() as hip:
        cache = Cache(hip, 1, 2, 128, 200, bits)
        r = Rows(hip, rng, 1, 200, 0, 2, 128, cache=cache, k=(rng.standard_normal((1, 200, 256)) * scale + scale).astype(F32))
        ctx.qcache_write(r.args, cache.args)
        out = hip.up(np.zeros((1, 200, 256), F32))
        ctx.qcache_read(lib.QReadArgs(k_out=out, k_out_seq_stride=200 * 256, k_out_stride=256, n=200), cache.args)
        got, x = hip.down(out, (200, 4, 64)).astype(np.float64), r.src["k"].reshape(200, 4, 64).astype(np.float64)
        step = ref.quantise(r.src["k"].reshape(200, 2, 128), bits)[1][..., :2].astype(np.float64).reshape(200, 4)
        assert np.all(np.abs(got - x) <= step[..., None] * (0.5 + 2.0 ** -18) + np.abs(got) * U)


def read_call(hip, cache, n, seqs, kvh, hd, pad=0, which="kv", **kw):
    out = {w: hip.up(np.full((seqs, n, kvh * hd + pad), SENTINEL, F32)) for w in which}
    a = lib.QReadArgs(n=n, **{k: hip.up(np.asarray(v, I32)) if isinstance(v, (list, np.ndarray)) else v for k, v in kw.items()})
    for w in which:
        setattr(a, w + "_out", out[w])
        setattr(a, w + "_out_stride", kvh * hd + pad)
        setattr(a, w + "_out_seq_stride", n * (kvh * hd + pad))
    return a, out


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kvh,hd", [(2, 128), (3, 64)])
@pytest.mark.parametrize("form", ["all", "ranges", "list", "heads", "k", "v"])
def test_read(ctx, rng, bits, kvh, hd, form):
    """Every value to the bit: the midpoint and step times the code, rounded once."""
    with base.Hip() as hip:
        seqs, capacity, n = 3, 37, 37 if form == "all" else 22
        cache = Cache(hip, seqs, kvh, hd, capacity, bits, seq_pad=6)
        x = {w: rng.standard_normal((seqs, kvh, capacity, hd)).astype(F32) for w in "kv"}
        x["v"][1, 0, 9, 3] = np.nan
        part = {w: cache.put(w, x[w]) for w in "kv"}
        kw, counts = {}, [n] * seqs
        if form == "ranges":
            counts, kw = [22, 7, 0], dict(counts=[50, 7, -1], first=[99, -4, 3])
        elif form in ("list", "heads"):
            shape = (seqs, kvh, n) if form == "heads" else (seqs, n)
            rows = rng.integers(-5, capacity + 5, shape).astype(I32)
            rows[0, ..., :3] = 11  # the same row several times
            counts, kw = [22, 5, 13], dict(counts=[22, 5, 13], rows=rows, per_head=1 if form == "heads" else 0)
        a, out = read_call(hip, cache, n, seqs, kvh, hd, 8, form if form in "kv" else "kv", **kw)
        ctx.qcache_read(a, cache.args)
        for w in out:
            got = hip.down(out[w], (seqs, n, kvh * hd + 8))
            assert np.all(got[..., kvh * hd:] == SENTINEL)
            for s in range(seqs):
                for g in range(kvh):
                    if form == "ranges":
                        at = [15, 0, 3][s] + np.arange(counts[s])
                    elif form in ("list", "heads"):
                        at = np.clip(rows[s, g] if form == "heads" else rows[s], 0, capacity - 1)[:counts[s]]
                    else:
                        at = np.arange(counts[s])
                    a_, b_ = (y[s, g][at] for y in part[w])
                    want = (a_ + b_).astype(F32)  # 19 and 11 bits: exact in 64, rounded once
                    assert np.array_equal(got[s, :counts[s], g * hd:(g + 1) * hd], want, equal_nan=True), (w, s, g)
                assert np.all(got[s, counts[s]:] == SENTINEL)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


class Attend:
    def __init__(self, hip, rng, seqs, n, rows, heads, kvh, hd, bits, lens=None, counts=None, window=0, cap=0.0, slopes=None,
                 scale=0.0, pad=0, capacity=None, q=None, k=None, v=None, q_std=2.0, seq_pad=0):
        self.hip = hip
        self.shape = (seqs, n, rows, heads, kvh, hd)
        self.cache = Cache(hip, seqs, kvh, hd, capacity or rows, bits, seq_pad)
        k = rng.standard_normal((seqs, kvh, rows, hd)).astype(F32) * F32(0.64) if k is None else k
        v = rng.standard_normal((seqs, kvh, rows, hd)).astype(F32) * F32(0.64) + F32(0.2) if v is None else v
        self.k, self.v = self.cache.put("k", k), self.cache.put("v", v)
        self.q = (rng.standard_normal((seqs, n, heads * hd)) * q_std).astype(F32) if q is None else q
        full = np.full((seqs, n, heads * hd + pad), SENTINEL, F32)
        full[..., :heads * hd] = self.q
        self.lens = np.full(seqs, rows, I32) if lens is None else np.asarray(lens, I32)
        self.counts = None if counts is None else np.asarray(counts, I32)
        self.slopes, self.window, self.cap, self.pad = slopes, window, cap, pad
        out = np.full(full.shape, SENTINEL, F32)
        a = lib.QAttentionArgs(q=hip.up(full), out=hip.up(out), lse=hip.up(np.full((seqs, n, heads), SENTINEL, F32)),
                               lens=hip.up(self.lens), counts=None if counts is None else hip.up(self.counts),
                               slopes=None if slopes is None else hip.up(slopes), q_seq_stride=full[0].size, q_stride=full.shape[2],
                               out_seq_stride=full[0].size, out_stride=full.shape[2], n=n, heads=heads, max_rows=rows,
                               window=window, scale=scale, cap=cap)
        self.scale = float(a.scale) or float(F32(1 / np.sqrt(hd)))
        need = lib.qcache_attention_workspace(a, self.cache.args)
        a.workspace, a.workspace_bytes = hip.raw(need), need
        self.args = a

    def run(self, ctx, stream=0):
        ctx.qcache_attention(self.args, self.cache.args, stream)
        return self

    def got(self):
        seqs, n, _, heads, _, hd = self.shape
        return self.hip.down(self.args.out, (seqs, n, heads * hd + self.pad)), self.hip.down(self.args.lse, (seqs, n, heads))

    def check(self, tokens=None, heads_at=None):
        seqs, n, rows, heads, kvh, hd = self.shape
        out, lse = self.got()
        assert np.all(out[..., heads * hd:] == SENTINEL)
        for s in range(seqs):
            count = n if self.counts is None else min(max(int(self.counts[s]), 0), n)
            length = min(max(int(self.lens[s]), 0), rows)
            assert np.all(out[s, count:] == SENTINEL) and np.all(lse[s, count:] == SENTINEL)
            t = np.arange(count) if tokens is None else tokens[tokens < count]
            if not t.size:
                continue
            dist = (length - count + t)[:, None] - np.arange(length)
            seen = dist >= 0
            if self.window:
                seen &= dist < self.window
            for h in range(heads) if heads_at is None else heads_at:
                g = h // (heads // kvh)
                k, v = ((x[0][s, g, :length], x[1][s, g, :length]) for x in (self.k, self.v))
                slope = None if self.slopes is None else np.full(t.size, self.slopes[h], np.float64)
                o, e, ob, eb = ref.attention(self.q[s, t, h * hd:(h + 1) * hd], k, v, seen, self.scale, self.cap, slope, dist)
                base.close(out[s, t, h * hd:(h + 1) * hd], o, ob, f"out of sequence {s}, head {h}")
                base.close(lse[s, t, h], e, eb, f"lse of sequence {s}, head {h}")
        return self


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 300, 1000]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kvh,hd", [(16, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("rows", LENGTHS)
def test_attention_of_one_token(ctx, rng, bits, heads, kvh, hd, rows):
    with base.Hip() as hip:
        Attend(hip, rng, 1, 1, rows, heads, kvh, hd, bits).run(ctx).check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kvh,hd", [(1, 1, 128), (8, 8, 64), (7, 1, 128), (6, 2, 64), (24, 1, 128), (40, 2, 64), (17, 1, 64)])
@pytest.mark.parametrize("seqs,n,rows", [(1, 1, 77), (3, 4, 130), (2, 37, 90)])
def test_attention_of_head_groups(ctx, rng, bits, heads, kvh, hd, seqs, n, rows):
    with base.Hip() as hip:
        Attend(hip, rng, seqs, n, rows, heads, kvh, hd, bits, pad=4, capacity=rows + 3, seq_pad=2).run(ctx).check()


@pytest.mark.parametrize("cap,bias", [(0.0, False), (25.0, True)], ids=["plain", "cap-bias"])
@pytest.mark.parametrize("window", [0, 1, 20, 33, 100])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_attention_windows(ctx, rng, n, window, cap, bias):
    """Ragged sequences: lengths and counts out of range, tokens before the cache's first row."""
    with base.Hip() as hip:
        slopes = np.array([2.0 ** (-2.0 * (h + 1)) for h in range(4)], F32) if bias else None
        Attend(hip, rng, 7, n, 150, 4, 2, 64 if n == 3 else 128, 4 if n == 1 else 8, lens=[150, 99, 0, -4, 1, 2, 4000],
               counts=[n, n + 5, n, 1, 1, n, max(0, n - 2)], window=window, cap=cap, slopes=slopes).run(ctx).check()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 150, 149])
@pytest.mark.parametrize("n", [10, 70])
def test_attention_windows_of_any_size(ctx, rng, n, window):
    """The largest windows with tokens before the cache's first row: positions less the window do not wrap."""
    with base.Hip() as hip:
        Attend(hip, rng, 4, n, 150, 4, 2, 128, 4, lens=[150, 5, 1, 0], window=window).run(ctx).check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("seqs,n,rows", [(1, 1, 9000), (5, 1, 2100), (1, 12, 3000), (1, 200, 1500), (2, 65, 700)])
def test_attention_long(ctx, rng, bits, seqs, n, rows):
    with base.Hip() as hip:
        lens = rows - np.arange(seqs) * (rows // 6)
        at = np.unique([0, n // 3, n // 2, max(0, n - 3), n - 1])
        Attend(hip, rng, seqs, n, rows, 16, 2, 128, bits, lens=lens).run(ctx).check(at, [0, 3, 8, 15])


@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (50.0, True), (0.01, False), (1e6, False)])
@pytest.mark.parametrize("n,rows", [(1, 1000), (40, 300)])
def test_attention_scores(ctx, rng, n, rows, cap, bias):
    """Capped scores over the whole curve of the tanh, biases of near and far rows."""
    with base.Hip() as hip:
        slopes = np.array([2.0 ** (-0.5 * (h + 1)) for h in range(16)], F32) if bias else None
        q = (rng.standard_normal((1, n, 2048)) * np.logspace(-3, 2.3, n * 2048).reshape(1, n, 2048)).astype(F32)
        Attend(hip, rng, 1, n, rows, 16, 2, 128, 4, cap=cap, slopes=slopes, scale=0.1, q=q).run(ctx).check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 30])
def test_attention_of_wide_ranges(ctx, rng, bits, n):
    """Rows of very different sizes side by side, zeros among them."""
    with base.Hip() as hip:
        rows = 140
        size = np.exp2(rng.integers(-12, 13, rows)).astype(F32)[:, None]
        k = rng.standard_normal((1, 2, rows, 128)).astype(F32) * size[rng.permutation(rows)] * F32(2.0 ** -8)
        v = rng.standard_normal((1, 2, rows, 128)).astype(F32) * size
        q = (rng.standard_normal((1, n, 2048)) * np.exp2(rng.integers(-12, 3, (1, n, 1)))).astype(F32)
        k[0, :, rows // 2], v[0, :, rows // 3], q[0, n // 2, :128] = 0.0, 0.0, 0.0
        Attend(hip, rng, 1, n, rows, 16, 2, 128, bits, q=q, k=k, v=v).run(ctx).check()


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_attention_scores_that_climb(ctx, rng, order):
    """The running maximum moves at every row, or never again: scores from -300 to 300."""
    with base.Hip() as hip:
        rows, hd = 400, 128
        line = np.linspace(-300, 300, rows) * np.sqrt(hd) / 16
        k = np.zeros((1, 1, rows, hd), F32)
        k[..., 0] = line if order == "rising" else line[::-1]
        q = np.zeros((1, 3, 2 * hd), F32)
        q[..., 0] = q[..., hd] = 16.0
        Attend(hip, rng, 1, 3, rows, 2, 1, hd, 8, q=q, k=k).run(ctx).check()


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60])
@pytest.mark.parametrize("n", [1, 20])
def test_attention_of_far_scales(ctx, rng, scale, n):
    """Query rows far outside fp16's range, scores back in their usual one."""
    with base.Hip() as hip:
        q = (rng.standard_normal((1, n, 256)) * 2 / scale).astype(F32)
        Attend(hip, rng, 1, n, 90, 2, 1, 128, 4, q=q, scale=F32(scale * 128 ** -0.5)).run(ctx).check()


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 40, 2.0 ** 80])
@pytest.mark.parametrize("n", [1, 20])
def test_attention_of_far_scores(ctx, rng, size, n):
    """Scores so large that one key has all the weight."""
    with base.Hip() as hip:
        q = (rng.standard_normal((1, n, 256)) * size).astype(F32)
        Attend(hip, rng, 1, n, 90, 2, 1, 128, 4, q=q).run(ctx).check()


@pytest.mark.parametrize("bad", [np.nan, np.inf, F32(3e38)])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("n,window", [(1, 20), (40, 0)])
def test_attention_masked_rows_do_not_leak(ctx, rng, bad, where, n, window):
    """NaN, infinite and the largest rows outside what a token sees change nothing; tokens that see a bad one show it."""
    with base.Hip() as hip:
        rows, at = 75, 52  # tokens 17 and later of 40 see row 52; one token's window ends behind it
        x = {w: rng.standard_normal((1, 2, rows, 128)).astype(F32) for w in "kv"}
        x[where][0, 0, at, 5] = bad
        a = Attend(hip, rng, 1, n, rows, 4, 2, 128, 4, window=window, k=x["k"], v=x["v"]).run(ctx)
        first = rows - n
        clean = np.arange(n) if n == 1 else np.arange(at - first)
        if not np.isfinite(bad):
            for y in (a.k if where == "k" else a.v):
                y[0, 0, at, :64] = 0.0  # not seen by the tokens below
        a.check(clean)
        if n > 1 and not np.isfinite(bad):
            out, lse = a.got()
            assert not np.isfinite(out[0, at - first:, :64]).any(-1).any()
            if where == "v":
                a.check(np.arange(n), [2, 3])
                assert np.isfinite(out[0, :, 64:128]).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("n", [1, 20])
def test_attention_bad_queries_stay_in_their_row(ctx, rng, n):
    with base.Hip() as hip:
        q = (rng.standard_normal((1, n, 512)) * 2).astype(F32)
        q[0, 0, 130] = np.nan
        a = Attend(hip, rng, 1, n, 60, 4, 2, 128, 4, q=q).run(ctx)
        out, lse = a.got()
        assert np.isnan(out[0, 0, 128:256]).all() and np.isnan(lse[0, 0, 1])
        a.q[0, 0, 128:256] = 0
        a.check(np.arange(n), [0, 2, 3])
        a.check(np.arange(1, n), [1])


def test_attention_ignores_what_lies_behind_a_sequence(ctx, rng):
    """Rows behind a sequence's length hold anything: NaN parameters, any codes."""
    with base.Hip() as hip:
        for n in (1, 18):
            x = rng.standard_normal((3, 2, 70, 128)).astype(F32)
            x[:, :, 41:] = np.nan
            Attend(hip, rng, 3, n, 70, 16, 2, 128, 4, lens=[41, 30, 18], k=x, v=x).run(ctx).check()


def test_attention_without_lse(ctx, rng):
    with base.Hip() as hip:
        a = Attend(hip, rng, 2, 3, 600, 16, 2, 128, 4)
        a.run(ctx)
        out, _ = a.got()
        a.args.lse = None
        a.run(ctx)
        assert np.array_equal(hip.down(a.args.out, out.shape), out)


def test_attention_is_the_same_each_time(ctx, rng):
    with base.Hip() as hip:
        for n, rows in ((1, 2500), (70, 900)):
            a = Attend(hip, rng, 2, n, rows, 16, 2, 128, 4).run(ctx)
            out, lse = a.got()
            for _ in range(3):
                a.run(ctx)
                again = a.got()
                assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)


def test_long_caches_pass_32_bit_offsets(ctx, rng):
    """The second sequence's rows lie past 2^31 bytes, and so do list entries."""
    with base.Hip() as hip:
        capacity, kvh, hd = 1 << 24, 2, 128
        rows = 2 * kvh * capacity
        bufs = [hip.raw(rows * 64), hip.raw(rows * 64), hip.raw(rows * 8), hip.raw(rows * 8)]
        cache = lib.QCache(k_codes=bufs[0], v_codes=bufs[1], k_params=bufs[2], v_params=bufs[3], seqs=2, kv_heads=kvh,
                           head_dim=hd, capacity=capacity, bits=4)
        n, first = 40, np.array([capacity - 40, capacity - 41], I32)
        k, v = (rng.standard_normal((2, n, 256)).astype(F32) for _ in range(2))
        a = lib.RowsArgs(k=hip.up(k), v=hip.up(v), first=hip.up(first), seqs=2, n=n, kv_heads=kvh, head_dim=hd,
                         k_seq_stride=n * 256, k_stride=256, v_seq_stride=n * 256, v_stride=256)
        ctx.qcache_write(a, cache)
        want = [sum(ref.values(*ref.quantise(x.reshape(2, n, 2, 128), 4), 4, parts=True)) for x in (k, v)]
        r, out = read_call(hip, cache, n, 2, kvh, hd, rows=first[:, None] + np.arange(n, dtype=I32))
        ctx.qcache_read(r, cache)
        for w, y in zip("kv", want):
            assert np.array_equal(hip.down(out[w], (2, n, 2, 128)), y.astype(F32))
        q = rng.standard_normal((2, 1, 2048)).astype(F32)
        o, lse = hip.up(np.zeros((2, 1, 2048), F32)), hip.up(np.zeros((2, 1, 16), F32))
        b = lib.QAttentionArgs(q=hip.up(q), out=o, lse=lse, lens=hip.up(first + n), q_seq_stride=2048, q_stride=2048,
                               out_seq_stride=2048, out_stride=2048, n=1, heads=16, max_rows=capacity, window=n)
        need = lib.qcache_attention_workspace(b, cache)
        b.workspace, b.workspace_bytes = hip.raw(need), need
        ctx.qcache_attention(b, cache)
        got = hip.down(o, (2, 16, 128))
        for s in range(2):
            for h in range(16):
                kk, vv = (ref.values(*ref.quantise(x[s].reshape(n, 2, 128)[:, h // 8], 4), 4, parts=True) for x in (k, v))
                w, _, ob, _ = ref.attention(q[s, :, h * 128:(h + 1) * 128], kk, vv, np.ones((1, n), bool), float(F32(128 ** -0.5)))
                base.close(got[s, h][None], w, ob)


# ---------------------------------------------------------------------------
# calls together
# ---------------------------------------------------------------------------


class Decoder:
    """Prompt, then token by token: rows rotated into a cache, attention over it."""

    def __init__(self, hip, rng, bits, hd=128):
        self.hip, self.hd, self.seqs, self.capacity = hip, hd, 3, 120
        self.cache = Cache(hip, 3, 2, hd, 120, bits)
        self.lens = np.zeros(3, I32)
        self.held = {w: np.zeros((3, 120, 2, hd), F32) for w in "kv"}

    def step(self, ctx, rng, n, counts, stream=0):
        hip, hd = self.hip, self.hd
        start = self.lens[:, None, None] + np.arange(n)[None, :, None] + np.zeros((1, 1, 3), np.int64)
        r = Rows(hip, rng, 3, n, 8, 2, hd, hd, 3, norms=True, counts=counts, first=self.lens, cache=self.cache, positions=start.astype(I32))
        ctx.qcache_write(r.args, self.cache.args, stream)
        self.lens = (self.lens + counts).astype(I32)
        out, lse = hip.up(np.zeros((3, n, 8 * hd), F32)), hip.up(np.zeros((3, n, 8), F32))
        a = lib.QAttentionArgs(q=r.args.q_out, out=out, lse=lse, lens=hip.up(self.lens), counts=r.args.counts,
                               q_seq_stride=n * 8 * hd, q_stride=8 * hd, out_seq_stride=n * 8 * hd, out_stride=8 * hd, n=n, heads=8,
                               max_rows=120)
        need = lib.qcache_attention_workspace(a, self.cache.args)
        a.workspace, a.workspace_bytes = hip.raw(need), need
        ctx.qcache_attention(a, self.cache.args, stream)
        hip.sync()
        # the rows as the device rounded them: y in 64 bits, rounded to fp32
        for s in range(3):
            for w in "kv":
                y = r.want(w, s)[0].astype(F32)
                self.held[w][s, r.at[s]:r.at[s] + counts[s]] = y.reshape(counts[s], 2, hd)
        q = hip.down(r.args.q_out, (3, n, 8 * hd))
        got = hip.down(out, (3, n, 8 * hd))
        for s in range(3):
            length, m = int(self.lens[s]), counts[s]
            seen = np.arange(length) <= (length - m + np.arange(m))[:, None]
            for h in range(8):
                k, v = (ref.values(*ref.quantise(self.held[w][s, :length, h // 4], self.cache.bits), self.cache.bits, parts=True)
                        for w in "kv")
                o, _, ob, _ = ref.attention(q[s, :m, h * hd:(h + 1) * hd], k, v, seen, float(F32(hd ** -0.5)))
                base.close(got[s, :m, h * hd:(h + 1) * hd], o, ob, f"sequence {s}, head {h}")


@pytest.mark.parametrize("bits,hd", [(4, 128), (8, 64)])
def test_a_run_of_the_calls(ctx, rng, bits, hd):
    """A ragged prompt, tokens, a drafted chunk; then what was held is read back."""
    with base.Hip() as hip:
        d = Decoder(hip, rng, bits, hd)
        stream = hip.stream()
        for n, counts in ((50, [50, 33, 7]), (1, [1, 1, 1]), (1, [1, 0, 1]), (6, [6, 2, 5]), (1, [1, 1, 1])):
            d.step(ctx, rng, n, np.array(counts, I32), stream)
        a, out = read_call(hip, d.cache, 120, 3, 2, hd, counts=d.lens)
        ctx.qcache_read(a, d.cache.args, stream)
        for w in "kv":
            got = hip.down(out[w], (3, 120, 2, hd))
            for s in range(3):
                want = ref.values(*ref.quantise(d.held[w][s, :d.lens[s]], bits), bits)
                assert np.array_equal(got[s, :d.lens[s]], want.astype(F32)), w


def test_a_captured_step_follows_its_lengths(ctx, rng):
    """Write, attention and reading back in one graph, replayed on new rows and lengths, with eager calls between."""
    with base.Hip() as hip:
        seqs, capacity, hd = 4, 90, 128
        cache, eager = (Cache(hip, seqs, 2, hd, capacity, 4) for _ in range(2))
        past = {w: rng.standard_normal((seqs, 2, capacity, hd)).astype(F32) for w in "kv"}
        for c in (cache, eager):
            for w in "kv":
                c.put(w, past[w])
        bufs = []
        for c in (cache, eager):
            r = Rows(hip, np.random.default_rng(3), seqs, 1, 16, 2, hd, hd, first=[0] * seqs, cache=c)
            out, lse = hip.up(np.zeros((seqs, 1, 2048), F32)), hip.up(np.zeros((seqs, 1, 16), F32))
            a = lib.QAttentionArgs(q=r.args.q_out, out=out, lse=lse, lens=hip.up(np.zeros(seqs, I32)), q_seq_stride=2048, q_stride=2048,
                                   out_seq_stride=2048, out_stride=2048, n=1, heads=16, max_rows=capacity)
            need = lib.qcache_attention_workspace(a, c.args)
            a.workspace, a.workspace_bytes = hip.raw(need), need
            rd, back = read_call(hip, c, capacity, seqs, 2, hd)
            bufs.append((c, r, a, rd, back))
        stream = hip.stream()

        def calls(b, s):
            c, r, a, rd, _ = b
            ctx.qcache_write(r.args, c.args, s)
            ctx.qcache_attention(a, c.args, s)
            ctx.qcache_read(rd, c.args, s)

        graph = hip.capture(stream, lambda: calls(bufs[0], stream))
        for lens in ([80, 3, 40, 1], [5, 89, 0, 33], [90, 90, 90, 90], [1, 2, 3, 4]):
            k = rng.standard_normal((seqs, 1, 256)).astype(F32)
            for _, r, a, _, _ in bufs:
                hip.write(r.args.k, k)
                hip.write(r.args.first, np.maximum(np.array(lens, I32) - 1, 0))
                hip.write(a.lens, np.array(lens, I32))
            hip.replay(graph, stream)
            calls(bufs[1], stream)
            hip.sync()
            for x, y, shape in ((bufs[0][2].out, bufs[1][2].out, (seqs, 2048)), (bufs[0][2].lse, bufs[1][2].lse, (seqs, 16)),
                                (bufs[0][4]["k"], bufs[1][4]["k"], (seqs, capacity, 256)),
                                (bufs[0][4]["v"], bufs[1][4]["v"], (seqs, capacity, 256))):
                assert np.array_equal(hip.down(x, shape), hip.down(y, shape))


def test_streams_and_threads(ctx, rng):
    """Calls from four threads on streams of their own, workspaces of their own: each as when alone."""
    with base.Hip() as hip:
        work = [Attend(hip, rng, 2, n, rows, 16, 2, 128, 4) for n, rows in ((1, 700), (5, 400), (40, 300), (1, 2500))]
        want = []
        for a in work:
            want.append([x.copy() for x in a.run(ctx).got()])
        streams = [hip.stream() for _ in work]
        fails = []

        def run(a, s):
            try:
                for _ in range(20):
                    a.run(ctx, s)
            except Exception as e:  # noqa: BLE001
                fails.append(e)

        threads = [threading.Thread(target=run, args=(a, s)) for a, s in zip(work, streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not fails
        for a, w in zip(work, want):
            got = a.got()
            assert np.array_equal(got[0], w[0]) and np.array_equal(got[1], w[1])

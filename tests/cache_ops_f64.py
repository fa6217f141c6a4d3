"""The cache operators' definitions in 64 bits (numpy), their error bounds, and
device buffers for the tests, from the HIP runtime the library itself links.

Error bounds (u = 2^-24, half a step of fp32).  A product keeps 22 bits of each
operand and drops the product of the two remainders: 2 * 2^-21 of its size with
truncated remainders; a dot product's sums add at most 17u of the sum of the
products' sizes (4 to 12 accumulations of trees of 5 levels).  Scores: 4u for
the scale and the shift, 8u of the capped score (quotient, tanh, product), 2u
of the bias.  exp of an argument x off by d is off by d relatively, plus 2u|x|
of the argument's own rounding and 2u of the exponential.  Numerator and
denominator of a softmax each carry that, their sums (N/16 + 32)u.
"""
import ctypes as C

import numpy as np

from rapidocrvl_amd import lib

U = 2.0 ** -24
H2D, D2H = 1, 2


def attention(q, k, v, seen, scale, cap=0.0, slope=None, dist=None):
    """One KV head: q [R][hd], k/v [L][hd], seen [R][L], slope [R], dist [R][L]
    → out, lse, p and the bounds of the errors of out, lse and p."""
    q, k = np.asarray(q, np.float64), np.asarray(k, np.float64)
    seen = np.broadcast_to(seen, (q.shape[0], k.shape[0]))
    used = seen.any(0)  # rows no query sees may hold anything
    k = np.where(used[:, None], k, 0.0)
    s = q @ k.T * scale
    err = np.abs(q) @ np.abs(k).T * scale * (17 * U + 2 * 2.0 ** -21) + np.abs(s) * 4 * U
    err += scale * 2.0 ** -32 * (np.abs(q).max(1)[:, None] * np.abs(k).sum(1) + np.abs(q).sum(1)[:, None] * np.abs(k).max(1))
    if cap:
        s = cap * np.tanh(s / cap)
        err = err + np.abs(s) * 8 * U
    if slope is not None:
        s = s - slope[:, None] * dist
        err = err + slope[:, None] * np.abs(dist) * 2 * U + np.abs(s) * U
    s = np.where(seen, s, -np.inf)
    m = s.max(1, keepdims=True) if s.shape[1] else np.full((s.shape[0], 1), -np.inf)
    m0 = np.where(np.isfinite(m), m, 0.0)
    e = np.exp(s - m0)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    with np.errstate(divide="ignore"):
        lse = m0[:, 0] + np.log(total[:, 0])
    lse = np.where(total[:, 0] == 0, -np.inf, lse)
    steps = (seen.sum(1) / 16 + 32) * U
    d = np.where(seen, err + np.abs(np.where(seen, s, 0.0) - m0) * 2 * U + 2 * U, 0.0)
    rows = (p * d).sum(1) + steps  # the denominator's relative error
    lse_err = rows + np.abs(np.where(np.isfinite(lse), lse, 0.0)) * 2 * U + 2 * U
    p_err = p * (d + rows[:, None])
    if v is None:
        return None, lse, p, None, lse_err, p_err
    v = np.where(used[:, None], np.asarray(v, np.float64), 0.0)
    out_err = p_err @ np.abs(v) + (p @ np.abs(v)) * (2 * 2.0 ** -21 + steps[:, None] + 2 * U) + 1e-38
    top = np.abs(v).max(1)
    out_err += (p @ top)[:, None] * 2.0 ** -32 + ((p * top).max(1) * seen.sum(1))[:, None] * 2.0 ** -30
    return p @ v, lse, p, out_err, lse_err, p_err


def close(got, want, bound, what=""):
    """Every value within its bound, and the whole within what independent
    errors of the 64 or more products behind a value leave of it (a quarter)."""
    got = np.asarray(got, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine]), what
    err = np.abs(got - np.where(fine, want, 0.0))[fine]
    bound = np.broadcast_to(bound, want.shape)[fine]
    assert np.all(np.isfinite(err)), what
    worst = float(np.max(err / bound, initial=0.0))
    assert worst <= 1.0, f"{what}: {worst} of the bound"
    if err.size >= 64:
        whole = float(np.linalg.norm(err) / np.linalg.norm(bound))
        assert whole <= 0.25, f"{what}: {whole} of the bound over all"


def ancestors(parents, count):
    """[token][token]: the second is the first or one of its ancestors."""
    n = len(parents)
    sees = np.zeros((n, n), bool)
    for i in range(count):
        a = i
        while a >= 0:
            sees[i, a] = True
            b = int(parents[a])
            a = b if -1 <= b < a else -1
    return sees


def select(weights, length, budget, sinks, recent):
    """Rows of one cache and KV head that stay."""
    if length <= budget:
        return np.arange(length)
    key = np.where(np.isnan(weights[:length]), -np.inf, weights[:length].astype(np.float64))
    nan = np.isnan(weights[:length])
    cand = np.arange(sinks, length - recent)
    order = sorted(cand, key=lambda j: (nan[j], -key[j], j))
    mid = order[:budget - sinks - recent]
    return np.array(sorted(list(range(sinks)) + list(mid) + list(range(length - recent, length))))


class Hip:
    """Device memory, streams and graphs; `guard` bytes behind each buffer are
    checked at the end."""

    GUARD = 4096

    def __init__(self):
        self.rt = lib.load()
        self.rt.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
        self.rt.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        self.rt.hipFree.argtypes = [C.c_void_p]
        self.rt.hipStreamCreateWithFlags.argtypes = [C.POINTER(C.c_void_p), C.c_uint]
        self.rt.hipStreamDestroy.argtypes = [C.c_void_p]
        self.rt.hipStreamSynchronize.argtypes = [C.c_void_p]
        self.rt.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
        self.rt.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
        self.rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
        self.rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
        self.rt.hipGraphExecDestroy.argtypes = [C.c_void_p]
        self.rt.hipGraphDestroy.argtypes = [C.c_void_p]
        self.bufs, self.streams, self.execs = {}, [], []

    def __enter__(self):
        return self

    def __exit__(self, kind, *_):
        self.sync()
        if kind is None:
            self.check_guards()
        for e in self.execs:
            self.rt.hipGraphExecDestroy(e)
        for s in self.streams:
            self.rt.hipStreamDestroy(s)
        for p in self.bufs:
            self.rt.hipFree(p)

    def sync(self):
        assert self.rt.hipDeviceSynchronize() == 0

    def raw(self, nbytes):
        p = C.c_void_p()
        assert self.rt.hipMalloc(C.byref(p), C.c_size_t(nbytes + self.GUARD)) == 0
        self.bufs[p.value] = nbytes
        self.write(p.value + nbytes, np.full(self.GUARD, 0xA5, np.uint8))
        return p.value

    def write(self, ptr, a):
        a = np.ascontiguousarray(a)
        assert self.rt.hipMemcpy(C.c_void_p(ptr), a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes), H2D) == 0

    def up(self, a):
        a = np.ascontiguousarray(a)
        p = self.raw(a.nbytes)
        if a.nbytes:
            self.write(p, a)
        return p

    def down(self, ptr, shape, dtype=np.float32):
        self.sync()
        out = np.zeros(shape, dtype)
        assert self.rt.hipMemcpy(out.ctypes.data_as(C.c_void_p), C.c_void_p(ptr), C.c_size_t(out.nbytes), D2H) == 0
        return out

    def check_guards(self):
        for p, n in self.bufs.items():
            assert np.all(self.down(p + n, self.GUARD, np.uint8) == 0xA5), "a write behind a buffer"

    def stream(self):
        s = C.c_void_p()
        assert self.rt.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        self.streams.append(s)
        return s.value

    def capture(self, stream, calls):
        """A graph of what `calls` queues on the stream."""
        g, e = C.c_void_p(), C.c_void_p()
        assert self.rt.hipStreamBeginCapture(stream, 2) == 0  # relaxed
        try:
            calls()
        finally:
            assert self.rt.hipStreamEndCapture(stream, C.byref(g)) == 0
        assert self.rt.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
        self.rt.hipGraphDestroy(g)
        self.execs.append(e)
        return e

    def replay(self, graph, stream):
        assert self.rt.hipGraphLaunch(graph, stream) == 0
        assert self.rt.hipStreamSynchronize(stream) == 0

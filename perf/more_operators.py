"""Operators of a K/V cache held in 4 or 8 bits as timed cases: the rows' norms and
rotation with several axes, their quantisation as they are written and their
reading back, and the attention over them.

A case is one call (or the few calls that belong together) on device buffers
the program owns, on its stream.  Widths are those of the 0.3B decoder (16
query heads over 2 KV heads of 128) and of smaller or other head groups.
``own`` chooses between the plain forms (elementary torch operations) and the
package's calls.

How a cache row lies in memory (include/pocr_hip.h): of every 64 elements of a
head a step and a midpoint in fp16, [step of each group | midpoint of each],
and codes c from -2^(bits-1) on, stored as c + 2^(bits-1); the value is
midpoint + step * c.  A row's codes are in the order of ``_order``, the lower
half of a byte first.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one page's prompt, rows as the projection leaves them (q | k | v): three axes, the decoder's own sections
        {"name": "rotate_page", "op": "rotate", "seqs": 1, "n": 1345, "heads": 16, "kv_heads": 2, "head_dim": 128,
         "rotary": 128, "axes": 3, "interleaved": False, "adjacent": False, "norms": False, "packed": True},
        # the frames of a video: normed heads, axes that alternate over the frequencies
        {"name": "rotate_video_norm", "op": "rotate", "seqs": 1, "n": 8192, "heads": 16, "kv_heads": 2, "head_dim": 128,
         "rotary": 128, "axes": 3, "interleaved": True, "adjacent": False, "norms": True, "packed": False},
        # one step of a server: 16 sequences' tokens rotated and appended to their caches
        {"name": "write_step16", "op": "write", "seqs": 16, "n": 1, "rows": 1609, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "rotary": 128, "axes": 3, "interleaved": False, "adjacent": False, "norms": False,
         "packed": True, "bits": 4},
        # a long document's prompt into its cache, normed and rotated on the way
        {"name": "write_long", "op": "write", "seqs": 1, "n": 8192, "rows": 0, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "rotary": 128, "axes": 3, "interleaved": False, "adjacent": False, "norms": True,
         "packed": True, "bits": 4},
        # all layers' rows of a page, already rotated, into caches of 8 bits: as many sequences as layers
        {"name": "write_layers8", "op": "write", "seqs": 18, "n": 1345, "rows": 0, "heads": 0, "kv_heads": 2,
         "head_dim": 128, "rotary": 0, "axes": 0, "interleaved": False, "adjacent": False, "norms": False,
         "packed": False, "bits": 8},
        # a page's caches of all layers back to fp32
        {"name": "read_page", "op": "read", "seqs": 18, "n": 1609, "rows": 1609, "listed": False, "kv_heads": 2,
         "head_dim": 128, "bits": 4},
        # the rows that stay of a long document's caches
        {"name": "read_kept8", "op": "read", "seqs": 18, "n": 2048, "rows": 8192, "listed": True, "kv_heads": 2,
         "head_dim": 128, "bits": 8},
        # the smallest call: one token behind a page
        {"name": "attend_token", "op": "attend", "seqs": 1, "n": 1, "rows": 1609, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "bits": 4, "window": 0, "cap": 0.0, "bias": False},
        # one step of 16 sequences behind long documents, ragged
        {"name": "attend_step16_long", "op": "attend", "seqs": 16, "n": 1, "rows": 8192, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "bits": 4, "window": 0, "cap": 0.0, "bias": False},
        # a chunk of a prompt behind a long document: the largest call
        {"name": "attend_chunk", "op": "attend", "seqs": 1, "n": 600, "rows": 8792, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "bits": 4, "window": 0, "cap": 0.0, "bias": False},
        # drafted chains of 5 tokens in 16 sequences, 8 bits, the last 1,024 rows, capped and biased scores
        {"name": "attend_drafts8", "op": "attend", "seqs": 16, "n": 5, "rows": 1609, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "bits": 8, "window": 1024, "cap": 30.0, "bias": True},
        # a text decoder of small heads, 8 sequences' tokens
        {"name": "attend_heads64", "op": "attend", "seqs": 8, "n": 1, "rows": 700, "heads": 4, "kv_heads": 2,
         "head_dim": 64, "bits": 4, "window": 0, "cap": 0.0, "bias": False},
    ]


HEADS = [(16, 2, 128), (16, 2, 128), (4, 2, 64), (8, 8, 64), (12, 4, 128), (32, 8, 128), (7, 1, 128)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rotate", "write", "write", "read", "attend", "attend", "attend"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case = {"op": op, "kv_heads": kv_heads, "head_dim": head_dim}
    wide = max(1, kv_heads * head_dim // 256)
    if op in ("rotate", "write"):
        case["heads"] = heads if op == "rotate" else rng.choice([0, heads])
        case["seqs"] = rng.choice([1, rng.randint(2, 16)])
        case["n"] = rng.choice([1, _log_int(rng, 1, 8192 // (case["seqs"] * wide))])
        rotates = op == "rotate" or rng.random() < 0.7
        case["rotary"] = rng.choice([head_dim, head_dim, head_dim // 2]) if rotates else 0
        case["axes"] = rng.choice([1, 2, 3, 3, 4]) if rotates else 0
        case["interleaved"] = rotates and rng.random() < 0.4
        case["adjacent"] = rotates and rng.random() < 0.3
        case["norms"] = rotates and rng.random() < 0.5
        case["packed"] = case["heads"] > 0 and rng.random() < 0.5
    if op == "write":
        case["rows"] = rng.choice([0, _log_int(rng, 1, 1609)])
    if op == "read":
        case["seqs"] = rng.randint(1, 18)
        case["rows"] = _log_int(rng, 1, 8192 // wide)
        case["n"] = rng.randint(1, min(case["rows"], 2048 // wide))
        case["listed"] = rng.random() < 0.5
    if op == "attend":
        case["heads"] = heads
        case["seqs"] = rng.choice([1, rng.randint(2, 16)])
        case["n"] = rng.choice([1, 1, _log_int(rng, 1, 600 // case["seqs"])])
        case["rows"] = case["n"] + _log_int(rng, 1, (8191 if case["seqs"] > 1 or case["n"] > 1 else 40000) // wide)
        if case["n"] > 1:  # products: no more than the chunk's
            case["rows"] = min(case["rows"], case["n"] + 600 * 16 * 8192 // (case["seqs"] * case["n"] * heads))
        case["window"] = rng.choice([0, 0, _log_int(rng, 1, case["rows"])])
        case["cap"] = rng.choice([0.0, 0.0, round(rng.uniform(15.0, 60.0), 2)])
        case["bias"] = rng.random() < 0.3
    if op != "rotate":
        case["bits"] = rng.choice([4, 4, 8])
    return case


# ---------------------------------------------------------------------------
# inputs: everything from the seed, drawn on the GPU
# ---------------------------------------------------------------------------


def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1009 + part)
    return g


def _up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _scale(case):
    return float(np.float32(1.0 / math.sqrt(case["head_dim"])))


def _lens(case, seed, count, most):
    """Requests of one batch differ in length, as their prompts do."""
    rng = np.random.default_rng([int(seed), 11])
    lens = most - rng.integers(0, 1 + most // 4, count)
    lens[0] = most
    return lens.astype(np.int32)


def _sections(case):
    """Frequencies of each axis: a quarter for time, the rest shared by the
    others; axes that alternate get what keeps their last frequency in range."""
    half, axes = case["rotary"] // 2, case["axes"]
    if axes == 1:
        return [half]
    if case["interleaved"]:
        each = half // axes - 1
        return [half - each * (axes - 1)] + [each] * (axes - 1)
    rest = half - half // 4
    cut = [rest // (axes - 1)] * (axes - 1)
    cut[-1] += rest - sum(cut)
    return [half // 4] + cut


def _axis_of(case):
    """The axis whose position turns each frequency."""
    half, axes, sections = case["rotary"] // 2, case["axes"], _sections(case)
    if not case["interleaved"]:
        return np.repeat(np.arange(axes), sections)
    i = np.arange(half)
    a = i % axes  # axis a > 0 takes frequencies a, a + axes, ... as long as its section lasts
    return np.where(i < axes * np.array(sections)[a], a, 0)


def _positions(case, seed):
    """Text, then an image's grid (or a video's frames) whose rows and columns
    count on from the text, for each sequence behind its cached rows."""
    rng = np.random.default_rng([int(seed), 5])
    s, n, axes = case["seqs"], case["n"], case["axes"]
    i = np.arange(n)
    side = max(1, int(math.sqrt(n / (8 if n > 2000 else 1))))
    grid = np.stack([i // (side * side), i // side % side, i % side, i % 7], -1)[:, :axes]
    start = rng.integers(0, 2000, (s, 1, 1))
    text = (i < 5) | (i >= n - 8)
    pos = np.where(text[:, None], i[:, None], 5 + grid) + start
    return pos.astype(np.int32)


def _freqs(case):
    return 500000.0 ** (-np.arange(case["rotary"] // 2) * 2.0 / case["rotary"])


def _order(what, hd, bits):
    """The element at each place of a row's codes.  K: the 16 lanes of a matrix
    instruction's lane group read 8 codes of each 32 elements; V: a lane's codes
    are 4 neighbours of each group."""
    at = np.arange(hd)
    if what == "k" and bits == 4:
        word, e = at // 8, at % 8
        return 32 * (word % (hd // 32)) + 8 * (word // (hd // 32)) + 2 * (e % 4) + e // 4
    if what == "k":
        unit, e = at // 8, at % 8
        return 32 * (2 * (unit // 8) + unit % 2) + 8 * (unit // 2 % 4) + e
    if hd == 128:
        return 64 * (at % 8 // 4) + 4 * (at // 8) + at % 4
    return at


def _pack(codes, what, bits):
    """Codes [..., hd] from 0 on, in a row's order, as bytes."""
    hd = codes.shape[-1]
    c = codes[..., _up(_order(what, hd, bits))].to(torch.uint8)
    return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)


def _quantised(x, bits):
    """Codes from 0 on [..., hd], steps and midpoints [..., hd / 64] in fp16 of rows x [..., hd]."""
    half = 1 << (bits - 1)
    g = x.clamp(-65504.0, 65504.0).double().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    mid = (((half - 1) * lo + half * hi) / (2 * half - 1)).float().half()
    need = torch.maximum((hi - mid.double()) / (half - 1), (mid.double() - lo) / half)
    step = need.float().half()
    step = torch.where(step.double() < need, (step.view(torch.int16) + 1).view(torch.float16), step)
    inv = torch.where(step > 0, 1.0 / step.double(), 0.0)
    codes = torch.round((g - mid.double()[..., None]) * inv[..., None]).clamp(-half, half - 1)
    return (codes + half).flatten(-2), step, mid


def _cache_of(x, what, bits):
    """A cache's codes and parameters of rows x [seqs][kv heads][rows][hd]."""
    codes, params = [], []
    for s in x:
        c, step, mid = _quantised(s, bits)
        codes.append(_pack(c, what, bits))
        params.append(torch.cat([step, mid], -1))
    return torch.stack(codes), torch.stack(params)


def prepare(case, seed):
    g = _gen(seed, 1)
    st = {"case": case}
    kvh, hd, s = case["kv_heads"], case["head_dim"], case["seqs"]
    kvd = kvh * hd
    if case["op"] in ("rotate", "write"):
        n, qd = case["n"], case["heads"] * hd
        rows = torch.randn((s, n, qd + 2 * kvd), generator=g, device="cuda") * 0.64
        rows[..., :qd] *= 4.0
        part = (lambda a, b: rows[..., a:b]) if case["packed"] else (lambda a, b: rows[..., a:b].contiguous())
        st["q"] = part(0, qd) if case["heads"] else None
        st["k"], st["v"] = part(qd, qd + kvd), part(qd + kvd, qd + 2 * kvd)
        st["counts"] = _up(_lens(case, seed, s, n))
        if case["rotary"]:
            st["positions"], st["freqs"] = _up(_positions(case, seed)), _up(_freqs(case))
            st["axis"] = _up(_axis_of(case))
        if case["norms"]:
            st["q_norm"], st["k_norm"] = (1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
        st["q_out"] = torch.zeros((s, n, qd), device="cuda") if case["heads"] else None
        st["k_out"], st["v_out"] = (torch.zeros((s, n, kvd), device="cuda") for _ in range(2))
    if case["op"] == "write":
        cap = case["rows"] + case["n"]
        st["first"] = _up(_lens(case, seed + 1, s, case["rows"]))
        for w in ("k", "v"):
            st[w + "_codes"] = torch.zeros((s, kvh, cap, hd * case["bits"] // 8), dtype=torch.uint8, device="cuda")
            st[w + "_params"] = torch.zeros((s, kvh, cap, hd // 32), dtype=torch.float16, device="cuda")
    if case["op"] in ("read", "attend"):
        for w in ("k", "v"):
            x = torch.randn((s, kvh, case["rows"], hd), generator=g, device="cuda") * 0.64
            if w == "k":  # some elements of a decoder's keys are offset
                x += torch.randn((kvh, 1, hd), generator=g, device="cuda")
            st[w + "_codes"], st[w + "_params"] = _cache_of(x, w, case["bits"])
            st[w + "_at"] = _up(np.argsort(_order(w, hd, case["bits"])))
        st["lens"] = _up(_lens(case, seed, s, case["rows"]))
    if case["op"] == "read":
        n, rng = case["n"], np.random.default_rng([int(seed), 17])
        st["counts"] = _up(_lens(case, seed, s, n))
        if case["listed"]:
            st["list"] = _up(np.sort(np.argsort(rng.random((s, case["rows"])), 1)[:, :n], 1).astype(np.int32))
        st["k_out"], st["v_out"] = (torch.zeros((s, n, kvd), device="cuda") for _ in range(2))
    if case["op"] == "attend":
        n, qd = case["n"], case["heads"] * hd
        st["q"] = torch.randn((s, n, qd), generator=g, device="cuda") * (8.0 if case["cap"] else 2.0)
        st["counts"] = _up(_lens(case, seed + 1, s, n))
        st["slopes"] = None
        if case["bias"]:
            st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])], device="cuda")
        st["out"] = torch.zeros((s, n, qd), device="cuda")
        st["lse"] = torch.zeros((s, n, case["heads"]), device="cuda")
    st["plan"] = _plan(case, st) if own else None
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _rotated(st, x, norm, dtype):
    """Rows [seqs][n][heads * hd] normed and rotated in `dtype`, rounded to fp32; angles in 64 bits."""
    case = st["case"]
    x = x.to(dtype).unflatten(-1, (-1, case["head_dim"]))
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * norm.to(dtype)
    if case["rotary"]:
        r = case["rotary"]
        angle = (st["positions"][..., st["axis"]].double() * st["freqs"])[:, :, None]
        c, s = torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["adjacent"] else (x[..., :r // 2], x[..., r // 2:r])
        a, b = a * c - b * s, b * c + a * s
        turned = torch.stack([a, b], -1).flatten(-2) if case["adjacent"] else torch.cat([a, b], -1)
        x = torch.cat([turned, x[..., r:]], -1)
    return x.float().flatten(-2)


def _live(st, out, rows):
    """Rows of each sequence's tokens into their places."""
    live = torch.arange(st["case"]["n"], device="cuda") < st["counts"][:, None]
    out.copy_(torch.where(live[..., None], rows, out))
    return out


def _plain_rotate(st):
    return {"q": _live(st, st["q_out"], _rotated(st, st["q"], st.get("q_norm"), torch.float32)),
            "k": _live(st, st["k_out"], _rotated(st, st["k"], st.get("k_norm"), torch.float32)),
            "v": _live(st, st["v_out"], st["v"])}


def _held(x, case):
    """What rows [seqs][n][kv heads * hd] are worth once held in a few bits."""
    codes, step, mid = _quantised(x.unflatten(-1, (-1, case["head_dim"])), case["bits"])
    c = (codes - (1 << (case["bits"] - 1))).unflatten(-1, (-1, 64))
    return (c * step.double()[..., None] + mid.double()[..., None]).flatten(-3).float()


def _plain_write(st):
    case = st["case"]
    k = _rotated(st, st["k"], st.get("k_norm"), torch.float64)  # a code's border is near: all of it in 64 bits
    out = {"k": _live(st, st["k_out"], _held(k, case)), "v": _live(st, st["v_out"], _held(st["v"], case))}
    if case["heads"]:
        out["q"] = _live(st, st["q_out"], _rotated(st, st["q"], st.get("q_norm"), torch.float32))
    return out


def _values(st, w, codes, params):
    """Rows [..., hd] in fp32 of their codes and parameters."""
    bits = st["case"]["bits"]
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    c = (codes[..., st[w + "_at"]].float() - float(1 << (bits - 1))).unflatten(-1, (-1, 64))
    step, mid = params.float().unflatten(-1, (2, -1)).unbind(-2)
    return (c * step[..., None] + mid[..., None]).flatten(-2)


def _plain_read(st):
    case = st["case"]
    out = {}
    for w in ("k", "v"):
        codes, params = st[w + "_codes"], st[w + "_params"]
        if case["listed"]:
            at = st["list"].long()[:, None, :, None].expand(-1, case["kv_heads"], -1, -1)
            codes = torch.gather(codes, 2, at.expand(-1, -1, -1, codes.shape[-1]))
            params = torch.gather(params, 2, at.expand(-1, -1, -1, params.shape[-1]))
        rows = _values(st, w, codes[:, :, :case["n"]], params[:, :, :case["n"]]).transpose(1, 2).flatten(-2)
        out[w] = _live(st, st[w + "_out"], rows)
    return out


def _plain_attend(st):
    case = st["case"]
    s_, n, kvh, hd, rows = case["seqs"], case["n"], case["kv_heads"], case["head_dim"], case["rows"]
    k, v = (_values(st, w, st[w + "_codes"], st[w + "_params"]) for w in ("k", "v"))
    t, j = torch.arange(n, device="cuda"), torch.arange(rows, device="cuda")
    live = t < st["counts"][:, None]
    pos = (st["lens"] - st["counts"])[:, None] + t
    dist = pos[..., None] - j  # [seq][token][row]
    seen = (dist >= 0) & live[..., None]
    if case["window"]:
        seen = seen & (dist < case["window"])
    q = st["q"].reshape(s_, n, kvh, -1, hd).permute(0, 2, 3, 1, 4)  # [seq][kv head][head][token][hd]
    s = torch.matmul(q.reshape(s_, kvh, -1, hd), k.transpose(-1, -2)).view(*q.shape[:4], rows) * _scale(case)
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(kvh, -1, 1, 1) * dist[:, None, None].float()
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(s_, kvh, -1, rows), v).view(*q.shape) / torch.where(total == 0, 1.0, total)
    lse = (m + torch.log(total)).squeeze(-1)
    return {"out": _live(st, st["out"], out.permute(0, 3, 1, 2, 4).flatten(2)),
            "lse": _live(st, st["lse"], lse.permute(0, 3, 1, 2).flatten(2))}


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------

_kept = {}


def _lib():
    from rapidocrvl_amd import lib

    if "ctx" not in _kept:
        _kept["ctx"] = lib.Context(0)
    return lib, _kept["ctx"]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _plan(case, st):
    """The arguments and workspace that a program keeps between its calls."""
    lib, ctx = _lib()
    s, n, kvh, hd = case["seqs"], case["n"], case["kv_heads"], case["head_dim"]
    cache = rows = read = attend = work = None
    if case["op"] != "rotate":
        cache = lib.QCache(k_codes=_ptr(st["k_codes"]), v_codes=_ptr(st["v_codes"]), k_params=_ptr(st["k_params"]),
                           v_params=_ptr(st["v_params"]), seqs=s, kv_heads=kvh, head_dim=hd,
                           capacity=st["k_codes"].shape[2], bits=case["bits"])
    if case["op"] in ("rotate", "write"):
        rows = lib.RowsArgs(q=_ptr(st["q"]), k=_ptr(st["k"]), v=_ptr(st["v"]), q_out=_ptr(st["q_out"]),
                            counts=_ptr(st["counts"]), q_norm=_ptr(st.get("q_norm")), k_norm=_ptr(st.get("k_norm")),
                            k_seq_stride=st["k"].stride(0), k_stride=st["k"].stride(1),
                            v_seq_stride=st["v"].stride(0), v_stride=st["v"].stride(1),
                            seqs=s, n=n, heads=case["heads"], kv_heads=kvh, head_dim=hd, eps=1e-5)
        if case["heads"]:
            rows.q_seq_stride, rows.q_stride = st["q"].stride(0), st["q"].stride(1)
            rows.q_out_seq_stride, rows.q_out_stride = st["q_out"].stride(0), st["q_out"].stride(1)
        if case["rotary"]:
            rows.positions, rows.freqs = _ptr(st["positions"]), _ptr(st["freqs"])
            rows.rotary_dim, rows.axes = case["rotary"], case["axes"]
            rows.sections[:case["axes"]] = _sections(case)
            rows.interleaved, rows.adjacent = case["interleaved"], case["adjacent"]
    if case["op"] == "rotate":
        rows.k_out, rows.v_out, rows.max_rows = _ptr(st["k_out"]), _ptr(st["v_out"]), n
        rows.k_out_seq_stride, rows.k_out_stride = st["k_out"].stride(0), st["k_out"].stride(1)
        rows.v_out_seq_stride, rows.v_out_stride = st["v_out"].stride(0), st["v_out"].stride(1)
    if case["op"] == "write":
        rows.first = _ptr(st["first"])
    if case["op"] in ("write", "read"):
        read = lib.QReadArgs(k_out=_ptr(st["k_out"]), v_out=_ptr(st["v_out"]), rows=_ptr(st.get("list")),
                             counts=_ptr(st["counts"]), first=_ptr(st.get("first")),
                             k_out_seq_stride=st["k_out"].stride(0), k_out_stride=st["k_out"].stride(1),
                             v_out_seq_stride=st["v_out"].stride(0), v_out_stride=st["v_out"].stride(1), n=n)
    if case["op"] == "attend":
        attend = lib.QAttentionArgs(q=_ptr(st["q"]), out=_ptr(st["out"]), lse=_ptr(st["lse"]), lens=_ptr(st["lens"]),
                                    counts=_ptr(st["counts"]), slopes=_ptr(st["slopes"]),
                                    q_seq_stride=st["q"].stride(0), q_stride=st["q"].stride(1),
                                    out_seq_stride=st["out"].stride(0), out_stride=st["out"].stride(1),
                                    n=n, heads=case["heads"], max_rows=case["rows"], window=case["window"],
                                    scale=_scale(case), cap=case["cap"])
        work = torch.empty(max(16, lib.qcache_attention_workspace(attend, cache)), dtype=torch.uint8, device="cuda")
        attend.workspace, attend.workspace_bytes = work.data_ptr(), work.numel()
    return ctx, cache, rows, read, attend, work


def _run_own(st):
    ctx, cache, rows, read, attend, _ = st["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    op = st["case"]["op"]
    if op == "rotate":
        ctx.rotate_rows(rows, stream)
        return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"]}
    if op == "attend":
        ctx.qcache_attention(attend, cache, stream)
        return {"out": st["out"], "lse": st["lse"]}
    if op == "write":
        ctx.qcache_write(rows, cache, stream)
    ctx.qcache_read(read, cache, stream)
    out = {"k": st["k_out"], "v": st["v_out"]}
    if op == "write" and st["case"]["heads"]:
        out["q"] = st["q_out"]
    return out


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "rotate":
        return _plain_rotate(st)
    if op == "write":
        return _plain_write(st)
    if op == "read":
        return _plain_read(st)
    return _plain_attend(st)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    s, n, kvh, hd = case["seqs"], case["n"], case["kv_heads"], case["head_dim"]
    share = 1.0 if s == 1 else 0.88  # live tokens and rows of ragged sequences, about
    tokens = s * n * (share if n > 3 else 1.0)
    held = kvh * (hd * case.get("bits", 0) / 8 + hd / 16)  # one row of K or of V
    if case["op"] == "rotate":
        return {"bytes": 8.0 * tokens * (case["heads"] + 2 * kvh) * hd, "flops": 0.0}
    if case["op"] == "write":  # rows in, q out, the cache written and read, its values out
        return {"bytes": tokens * (8.0 * case["heads"] * hd + 16.0 * kvh * hd + 4.0 * held), "flops": 0.0}
    if case["op"] == "read":
        return {"bytes": tokens * (8.0 * kvh * hd + 2.0 * held), "flops": 0.0}
    rows = case["rows"] * share
    seen = min(rows, case["window"] or rows) - (n / 2 if n > 1 and not case["window"] else 0)
    rows = min(rows, case["window"] + n) if case["window"] else rows
    return {"bytes": s * rows * 2.0 * held + 8.0 * tokens * case["heads"] * hd,
            "flops": 4.0 * hd * case["heads"] * tokens * max(1.0, seen)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_head(x, norm, cos, sin, case):
    """One head's rows [n][hd]: x * norm / rms, then each pair turned by its angle."""
    y = x.double().clone()
    if norm is not None:
        y = y / torch.sqrt((y ** 2).sum(1, keepdim=True) / case["head_dim"] + 1e-5) * norm.double()
    if case["rotary"]:
        half = case["rotary"] // 2
        i = torch.arange(half, device="cuda")
        a, b = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + half)
        z = torch.complex(y[:, a], y[:, b]) * torch.complex(cos, sin)
        y[:, a], y[:, b] = z.real, z.imag
    return y


def _exact_held(x, bits):
    """Values of fp32 rows [n][hd] once held in `bits`, group by group."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    low, top = -(2 ** (bits - 1)), 2 ** (bits - 1) - 1
    for c in range(0, x.shape[1], 64):
        g = torch.clip(x[:, c:c + 64].double(), -65504.0, 65504.0)
        lo, hi = g.min(1, keepdim=True).values, g.max(1, keepdim=True).values
        mid = ((top * lo - low * hi) / (top - low)).to(torch.float32).to(torch.float16).double()
        need = torch.maximum((hi - mid) / top, (lo - mid) / low)
        near = need.to(torch.float32).to(torch.float16)
        above = (near.view(torch.int16) + 1).view(torch.float16)
        step = torch.where(near.double() >= need, near, above).double()
        code = torch.where(step > 0, torch.round((g - mid) * step.reciprocal()), 0.0).clip(low, top)
        out[:, c:c + 64] = mid + step * code
    return out


def _exact_rows(case, st):
    hd, kvh = case["head_dim"], case["kv_heads"]
    out = {w: torch.zeros(st[w].shape, dtype=torch.float64, device="cuda") for w in ("q", "k", "v") if st[w] is not None}
    for s in range(case["seqs"]):
        m = int(st["counts"][s])
        cos = sin = None
        if case["rotary"]:
            at = st["positions"][s, :m].cpu().numpy().astype(np.float64)
            angle = at[:, _axis_of(case)] * _freqs(case)
            cos, sin = _up(np.cos(angle)), _up(np.sin(angle))
        for w, heads in (("q", case["heads"]), ("k", kvh), ("v", kvh)):
            for h in range(heads):
                x = st[w][s, :m, h * hd:(h + 1) * hd]
                y = x.double() if w == "v" else _exact_head(x, st.get(w + "_norm"), cos, sin, case)
                if case["op"] == "write" and w != "q":  # the rounded row is what is held
                    y = _exact_held(y.float(), case["bits"])
                out[w][s, :m, h * hd:(h + 1) * hd] = y
    return out


def _exact_values(st, w, s, g, case):
    """Rows [rows][hd] of one head's cache, element by element place."""
    hd, bits = case["head_dim"], case["bits"]
    raw, params = st[w + "_codes"][s, g].to(torch.int64), st[w + "_params"][s, g].double()
    out = torch.empty((raw.shape[0], hd), dtype=torch.float64, device="cuda")
    for place, d in enumerate(_order(w, hd, bits).tolist()):
        c = raw[:, place] if bits == 8 else (raw[:, place // 2] >> (4 * (place % 2))) % 16
        out[:, d] = params[:, hd // 64 + d // 64] + params[:, d // 64] * (c - 2 ** (bits - 1))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    f64, hd, kvh = torch.float64, case["head_dim"], case["kv_heads"]
    if case["op"] in ("rotate", "write"):
        return {w: x for w, x in _exact_rows(case, st).items()}
    if case["op"] == "read":
        out = {w: torch.zeros((case["seqs"], case["n"], kvh * hd), dtype=f64, device="cuda") for w in ("k", "v")}
        for s in range(case["seqs"]):
            m = int(st["counts"][s])
            at = st["list"][s, :m].long() if case["listed"] else torch.arange(m, device="cuda")
            for g in range(kvh):
                for w in ("k", "v"):
                    out[w][s, :m, g * hd:(g + 1) * hd] = _exact_values(st, w, s, g, case)[at]
        return out
    n, group = case["n"], case["heads"] // kvh
    out = torch.zeros((case["seqs"], n, case["heads"], hd), dtype=f64, device="cuda")
    lse = torch.zeros((case["seqs"], n, case["heads"]), dtype=f64, device="cuda")
    for s in range(case["seqs"]):
        length, m = int(st["lens"][s]), int(st["counts"][s])
        pos = length - m + torch.arange(m, device="cuda")
        j = torch.arange(length, device="cuda")
        seen = j[None] <= pos[:, None]
        if case["window"]:
            seen &= j[None] > pos[:, None] - case["window"]
        for h in range(case["heads"]):
            k, v = (_exact_values(st, w, s, h // group, case)[:length] for w in ("k", "v")) if h % group == 0 else (k, v)
            x = st["q"][s, :m, h * hd:(h + 1) * hd].double() @ k.T * _scale(case)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if st["slopes"] is not None:
                x = x - st["slopes"][h].double() * (pos[:, None] - j[None])
            x = torch.where(seen, x, -math.inf)
            e = torch.logsumexp(x, 1)
            p = torch.where(seen, torch.exp(x - e[:, None]), 0.0)
            out[s, :m, h], lse[s, :m, h] = p @ v, e
    return {"out": out.flatten(2), "lse": lse}

"""Cache operators as timed cases: attention of a prompt's rows with masks,
capped scores and distance biases, attention of drafted token trees, the
accumulated attention weight of cache rows, and the selection and compaction
of the rows that stay.

A case is one call (or the few calls that belong together) on device buffers
the program owns, on its stream.  Widths are those of the 0.3B decoder (16
query heads over 2 KV heads of 128) and of smaller or other head groups.
``own`` chooses between the plain forms (elementary torch operations in 32
bits) and the package's calls.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one page's image prompt: the image rows see each other, the text rows before them
        {"name": "prompt_page", "op": "prompt", "n": 1345, "rows0": 0, "heads": 16, "kv_heads": 2, "head_dim": 128,
         "mask": "prefix", "docs": 1, "cap": 0.0, "bias": False, "packed": True},
        # several requests' prompts packed into one pass, capped scores, ragged lengths, padding rows at the end
        {"name": "prompt_packed", "op": "prompt", "n": 2403, "rows0": 0, "heads": 16, "kv_heads": 2, "head_dim": 128,
         "mask": "docs", "docs": 7, "cap": 30.0, "bias": False, "packed": True},
        # the largest call: a long causal document
        {"name": "prompt_long", "op": "prompt", "n": 8192, "rows0": 0, "heads": 16, "kv_heads": 2, "head_dim": 128,
         "mask": "causal", "docs": 1, "cap": 0.0, "bias": False, "packed": False},
        # one token of a decoder with distance biases and capped scores, behind a page
        {"name": "token_bias_cap", "op": "prompt", "n": 1, "rows0": 1608, "heads": 16, "kv_heads": 2, "head_dim": 128,
         "mask": "causal", "docs": 1, "cap": 30.0, "bias": True, "packed": False},
        # the smallest call: five drafted tokens right behind a short text, heads of 64
        {"name": "tree_short_d64", "op": "tree", "seqs": 1, "n": 5, "rows": 64, "heads": 4, "kv_heads": 2,
         "head_dim": 64, "cap": 0.0, "bias": False},
        # a server's full house: 16 sequences verify up to 12 drafted tokens each behind a page, ragged
        {"name": "tree_page16", "op": "tree", "seqs": 16, "n": 12, "rows": 1609, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "cap": 0.0, "bias": False},
        # a wide tree at the end of a long document
        {"name": "tree_long64", "op": "tree", "seqs": 1, "n": 64, "rows": 8192, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "cap": 30.0, "bias": False},
        # the weights of one decode step of 16 sequences, accumulated
        {"name": "weights_step16", "op": "weights", "seqs": 16, "n": 1, "rows": 1609, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "cap": 0.0, "bias": False},
        # the last 64 rows of a long prompt vote on what stays
        {"name": "weights_window64", "op": "weights", "seqs": 1, "n": 64, "rows": 8192, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "cap": 0.0, "bias": False},
        # all 18 layers of one sequence behind a page fall to 768 rows, each KV head its own
        {"name": "evict_page", "op": "evict", "caches": 18, "rows": 1609, "budget": 768, "sinks": 4, "recent": 256,
         "heads": 16, "kv_heads": 2, "head_dim": 128},
        # and of a long document to a quarter
        {"name": "evict_long", "op": "evict", "caches": 18, "rows": 8192, "budget": 2048, "sinks": 4, "recent": 512,
         "heads": 16, "kv_heads": 2, "head_dim": 128},
        # the accepted path of 12 drafted tokens takes its places, 18 layers of 4 sequences
        {"name": "accept_page", "op": "accept", "caches": 72, "n": 12, "rows": 1609, "heads": 16, "kv_heads": 2,
         "head_dim": 128},
    ]


HEADS = [(16, 2, 128), (16, 2, 128), (4, 2, 64), (8, 8, 64), (12, 4, 128), (32, 8, 128), (7, 1, 128)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "weights", "evict", "accept"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    if op in ("prompt", "tree", "weights"):
        case["cap"] = rng.choice([0.0, 0.0, round(rng.uniform(15.0, 60.0), 2)])
        case["bias"] = rng.random() < 0.3
    if op == "prompt":
        case["n"] = _log_int(rng, 1, 2600)
        case["rows0"] = rng.choice([0, _log_int(rng, 1, 4096)])
        case["mask"] = rng.choice(["causal", "prefix", "docs"]) if case["rows0"] == 0 else "causal"
        case["docs"] = rng.randint(1, min(9, case["n"])) if case["mask"] == "docs" else 1
        case["packed"] = rng.random() < 0.5
    elif op in ("tree", "weights"):
        case["seqs"] = rng.choice([1, rng.randint(2, 16)])
        case["n"] = rng.choice([1, _log_int(rng, 1, 64)])
        case["rows"] = _log_int(rng, 1, 9000 if case["seqs"] == 1 else 3000)
    elif op == "evict":
        case["caches"] = rng.randint(1, 18)
        case["rows"] = _log_int(rng, 40, 9000)
        case["sinks"] = rng.randint(0, 4)
        case["recent"] = rng.randint(0, case["rows"] // 8)
        case["budget"] = case["sinks"] + case["recent"] + rng.randint(1, case["rows"] // 2)
    else:
        case["caches"] = rng.randint(1, 72)
        case["n"] = _log_int(rng, 1, 64)
        case["rows"] = _log_int(rng, 1, 1700)
    return case


# ---------------------------------------------------------------------------
# inputs: everything from the seed, drawn on the GPU
# ---------------------------------------------------------------------------


def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1009 + part)
    return g


def _scale(case):
    return float(np.float32(1.0 / math.sqrt(case["head_dim"])))


def _slopes(case):
    if not case["bias"]:
        return None
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])], device="cuda")


def _q_std(case):
    """Query rows whose scores spread by about 2 against key rows of 0.64; a
    decoder that caps its scores lets them grow further."""
    return 8.0 if case["cap"] else 3.0


def _spans(case, seed):
    """First and end visible row of each prompt row; None for plain causal rows."""
    n, rng = case["n"], np.random.default_rng([int(seed), 7])
    i = np.arange(n)
    if case["mask"] == "causal":
        return None
    if case["mask"] == "prefix":  # five text rows, the image, the question: rows of the image see all of it
        first, last = min(5, n - 1), max(1, n - 8)
        end = np.where((i >= first) & (i < last), last, i + 1)
        return np.zeros(n, np.int32), end.astype(np.int32)
    cuts = np.sort(rng.choice(np.arange(1, n), case["docs"] - 1, replace=False)) if case["docs"] > 1 else np.array([], int)
    starts = np.concatenate([[0], cuts])
    begin = starts[np.searchsorted(starts, i, side="right") - 1]
    end = i + 1
    pad = i >= n - n // 50  # rows behind the last prompt see nothing
    return np.where(pad, 0, begin).astype(np.int32), np.where(pad, 0, end).astype(np.int32)


def _lens(case, seed, count, rows):
    """Requests of one batch differ in length, as their prompts do."""
    rng = np.random.default_rng([int(seed), 11])
    lens = rows - rng.integers(0, 1 + rows // 4, count)
    lens[0] = rows
    return lens.astype(np.int32)


def _trees(case, seed):
    """Drafted trees: mostly runs, with branches; fewer tokens in some sequences."""
    rng = np.random.default_rng([int(seed), 13])
    s, n = case["seqs"], case["n"]
    i = np.arange(n)
    par = np.where(rng.random((s, n)) < 0.7, i - 1, np.floor(rng.random((s, n)) * (i + 1)) - 1).astype(np.int32)
    counts = np.maximum(1, n - rng.integers(0, 1 + n // 3, s)).astype(np.int32)
    counts[0] = n
    return par, counts


def _up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    g = _gen(seed, 1)
    st = {"case": case}
    hd, kvd = case["head_dim"], case["kv_heads"] * case["head_dim"]
    qd = case["heads"] * hd
    if case["op"] == "prompt":
        n, rows = case["n"], case["rows0"] + case["n"]
        if case["packed"] and case["rows0"] == 0:  # one projection's output rows: q | k | v
            qkv = torch.randn((n, qd + 2 * kvd), generator=g, device="cuda") * 0.64
            qkv[:, :qd] *= _q_std(case) / 0.64
            st["q"], st["k"], st["v"] = qkv[:, :qd], qkv[:, qd:qd + kvd], qkv[:, qd + kvd:]
        else:
            st["q"] = torch.randn((n, qd), generator=g, device="cuda") * _q_std(case)
            st["k"] = torch.randn((rows, kvd), generator=g, device="cuda") * 0.64
            st["v"] = torch.randn((rows, kvd), generator=g, device="cuda") * 0.64
        spans = _spans(case, seed)
        st["begin"], st["end"] = (None, None) if spans is None else (_up(spans[0]), _up(spans[1]))
        st["slopes"] = _slopes(case)
        st["out"] = torch.zeros((n, qd), device="cuda")
        st["lse"] = torch.zeros((n, case["heads"]), device="cuda")
    elif case["op"] in ("tree", "weights"):
        s, n = case["seqs"], case["n"]
        par, counts = _trees(case, seed)
        lens = _lens(case, seed, s, case["rows"])
        cap = case["rows"] + n
        st["q"] = torch.randn((s, n, qd), generator=g, device="cuda") * _q_std(case)
        st["k"] = torch.randn((s, cap, kvd), generator=g, device="cuda") * 0.64
        st["v"] = torch.randn((s, cap, kvd), generator=g, device="cuda") * 0.64
        st["lens"], st["parents"], st["counts"] = _up(lens), _up(par), _up(counts)
        st["slopes"] = _slopes(case)
        if case["op"] == "tree":
            st["out"] = torch.zeros((s, n, qd), device="cuda")
            st["lse"] = torch.zeros((s, n, case["heads"]), device="cuda")
        else:
            lse = _rows_softmax(*_tree_scores(st, torch.float64))[1]
            st["lse"] = lse.permute(0, 3, 1, 2).reshape(s, n, -1).float()
            st["weights"] = torch.rand((s, case["kv_heads"], cap), generator=g, device="cuda") * 4.0
    elif case["op"] == "evict":
        c, rows, b = case["caches"], case["rows"], case["budget"]
        st["k"] = torch.randn((c, rows, kvd), generator=g, device="cuda") * 0.64
        st["v"] = torch.randn((c, rows, kvd), generator=g, device="cuda") * 0.64
        st["weights"] = torch.exp(torch.randn((c, case["kv_heads"], rows), generator=g, device="cuda") * 2.0)
        st["lens"] = _up(_lens(case, seed, c, rows))
        st["k2"], st["v2"] = (torch.zeros((c, b, kvd), device="cuda") for _ in range(2))
        st["weights2"] = torch.zeros((c, case["kv_heads"], b), device="cuda")
        st["kept"] = torch.full((c, case["kv_heads"], b), -1, dtype=torch.int32, device="cuda")
        st["counts"] = torch.zeros(c, dtype=torch.int32, device="cuda")
    else:
        c, n = case["caches"], case["n"]
        cap = case["rows"] + n
        st["k"] = torch.randn((c, cap, kvd), generator=g, device="cuda") * 0.64
        st["v"] = torch.randn((c, cap, kvd), generator=g, device="cuda") * 0.64
        lens = _lens(case, seed, c, case["rows"])
        rng = np.random.default_rng([int(seed), 17])
        path = np.sort(np.argsort(rng.random((c, n)), 1)[:, :max(1, n // 2)], 1)  # half the drafted tokens, in order
        st["lens"] = _up(lens)
        st["list"] = _up((lens[:, None] + path).astype(np.int32))
        st["counts"] = _up(np.maximum(1, path.shape[1] - rng.integers(0, 2, c)).astype(np.int32))
    st["plan"] = _plan(case, st) if own else None
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _shape_scores(s, case, slopes, dist):
    """Scaled products → scores; slopes against [..., heads, rows, keys]."""
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    if slopes is not None:
        s = s - slopes.to(s.dtype).view(case["kv_heads"], -1, 1, 1) * dist.to(s.dtype)
    return s


def _rows_softmax(s, seen):
    """Weights and log-sum-exp over the last axis; rows that see nothing: zeros and -inf."""
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total), (m + torch.log(total)).squeeze(-1)


def _plain_prompt(st):
    case = st["case"]
    n, rows, kvh, hd = case["n"], case["rows0"] + case["n"], case["kv_heads"], case["head_dim"]
    q = st["q"].reshape(n, kvh, -1, hd).permute(1, 2, 0, 3)  # [g][h][i][d]
    k = st["k"].reshape(rows, kvh, hd).permute(1, 2, 0)
    v = st["v"].reshape(rows, kvh, hd).permute(1, 0, 2)
    i = torch.arange(n, device="cuda")[:, None] + case["rows0"]
    j = torch.arange(rows, device="cuda")
    seen = j <= i if st["begin"] is None else (j >= st["begin"][:, None]) & (j < st["end"][:, None])
    s = torch.matmul(q, k[:, None]) * _scale(case)
    s = _shape_scores(s, case, st["slopes"], (i - j).abs())
    p, lse = _rows_softmax(s, seen)
    st["out"].copy_(torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).reshape(n, -1))
    st["lse"].copy_(lse.permute(2, 0, 1).reshape(n, -1))
    return {"out": st["out"], "lse": st["lse"]}


def _tree_scores(st, dtype=torch.float32):
    """Scores [seq][kv head][head][token][row] and what each token sees."""
    case = st["case"]
    s_, n, kvh, hd = case["seqs"], case["n"], case["kv_heads"], case["head_dim"]
    cap = case["rows"] + n
    t = torch.arange(n, device="cuda")
    j = torch.arange(cap, device="cuda")
    # node 0 is the cache's end, node a + 1 drafted token a; a path from a node to an ancestor is the only one
    up = (st["parents"].long()[..., None] + 1 == torch.arange(n + 1, device="cuda")).float()
    up = torch.cat([torch.zeros((s_, 1, n + 1), device="cuda"), up], 1) + torch.eye(n + 1, device="cuda")
    reach = torch.linalg.matrix_power(up, 64)[:, 1:, 1:] > 0  # [seq][token][itself or an ancestor]
    depth = reach.sum(-1) - 1
    lens = st["lens"].long()
    a = (j - lens[:, None]).clamp(0, n - 1)  # drafted token of a row
    cached = j < lens[:, None]
    drafted = (j >= lens[:, None]) & (j < lens[:, None] + st["counts"][:, None])
    seen = cached[:, None] | (drafted[:, None] & torch.gather(reach, 2, a[:, None].expand(s_, n, cap)))
    live = t < st["counts"][:, None]
    seen = seen & live[..., None]
    pos_k = torch.where(cached, j, lens[:, None] + torch.gather(depth, 1, a))
    dist = (lens[:, None, None] + depth[..., None] - pos_k[:, None]).abs()[:, None, None]
    q = st["q"].to(dtype).reshape(s_, n, kvh, -1, hd).permute(0, 2, 3, 1, 4)
    k = st["k"].to(dtype).reshape(s_, cap, kvh, hd).permute(0, 2, 3, 1)
    s = torch.matmul(q, k[:, :, None]) * _scale(case)
    return _shape_scores(s, case, st["slopes"], dist), seen[:, None, None]


def _plain_tree(st):
    case = st["case"]
    s_, n, kvh, hd = case["seqs"], case["n"], case["kv_heads"], case["head_dim"]
    p, lse = _rows_softmax(*_tree_scores(st))
    drafted_end = (st["lens"] + st["counts"])[:, None, None, None]
    v = st["v"].reshape(s_, -1, kvh, hd)
    v = torch.where(torch.arange(v.shape[1], device="cuda")[:, None, None] < drafted_end, v, 0.0).permute(0, 2, 1, 3)
    live = (torch.arange(n, device="cuda") < st["counts"][:, None])[..., None]
    st["out"].copy_(torch.where(live, torch.matmul(p, v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(s_, n, -1), st["out"]))
    st["lse"].copy_(torch.where(live, lse.permute(0, 3, 1, 2).reshape(s_, n, -1), st["lse"]))
    return {"out": st["out"], "lse": st["lse"]}


def _plain_weights(st):
    case = st["case"]
    s, seen = _tree_scores(st)
    lse = st["lse"].reshape(case["seqs"], case["n"], case["kv_heads"], -1).permute(0, 2, 3, 1)[..., None]
    p = torch.exp(torch.where(seen, s - lse, -math.inf))
    st["weights"] += p.sum((2, 3))
    return {"weights": st["weights"]}


def _plain_evict(st):
    case = st["case"]
    c, rows, b, kvh, hd = case["caches"], case["rows"], case["budget"], case["kv_heads"], case["head_dim"]
    j = torch.arange(rows, device="cuda")
    lens = st["lens"].long()[:, None, None]
    w = torch.where((j < case["sinks"]) | (j >= lens - case["recent"]), math.inf, st["weights"])
    w = torch.where(j < lens, w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :b]
    kept = torch.sort(order, dim=-1).values
    if kept.shape[-1] < b:  # fewer rows than the budget
        kept = torch.cat([kept, torch.full((c, kvh, b - kept.shape[-1]), rows, device="cuda")], -1)
    counts = lens[:, 0, 0].clamp(max=b)
    live = torch.arange(b, device="cuda") < counts[:, None, None]
    st["counts"].copy_(counts)
    st["kept"].copy_(torch.where(live, kept, st["kept"].long()))
    at = torch.where(live, kept, 0)
    st["weights2"].copy_(torch.where(live, torch.gather(st["weights"], 2, at), 0.0))
    at, live = at.permute(0, 2, 1)[..., None].expand(c, b, kvh, hd), live.permute(0, 2, 1)[..., None]
    k2, v2 = st["k2"].view(c, b, kvh, hd), st["v2"].view(c, b, kvh, hd)
    k2.copy_(torch.where(live, torch.gather(st["k"].view(c, rows, kvh, hd), 1, at), k2))
    v2.copy_(torch.where(live, torch.gather(st["v"].view(c, rows, kvh, hd), 1, at), v2))
    return {n: st[n] for n in ("kept", "counts", "k2", "v2", "weights2")}


def _plain_accept(st):
    case = st["case"]
    c, m = st["list"].shape
    cache = torch.arange(c, device="cuda")[:, None]
    j = torch.arange(m, device="cuda")
    live = j < st["counts"][:, None]
    dst = st["lens"].long()[:, None] + j
    src = torch.where(live, st["list"].long(), dst)
    k, v = st["k"][cache, src], st["v"][cache, src]
    st["k"][cache, dst] = k
    st["v"][cache, dst] = v
    return {"k": st["k"], "v": st["v"]}


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------

_held = {}


def _lib():
    from rapidocrvl_amd import lib

    if "ctx" not in _held:
        _held["ctx"] = lib.Context(0)
    return lib, _held["ctx"]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _work_buffer(nbytes):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device="cuda")


def _plan(case, st):
    """The arguments and workspace that a program keeps between its calls."""
    lib, ctx = _lib()
    heads = {"heads": case["heads"], "kv_heads": case["kv_heads"], "head_dim": case["head_dim"]}
    kvd = case["kv_heads"] * case["head_dim"]
    if case["op"] == "prompt":
        a = lib.PromptArgs(q=_ptr(st["q"]), k=_ptr(st["k"]), v=_ptr(st["v"]), out=_ptr(st["out"]), lse=_ptr(st["lse"]),
                           row_begin=_ptr(st["begin"]), row_end=_ptr(st["end"]), slopes=_ptr(st["slopes"]),
                           n=case["n"], rows_before=case["rows0"], q_stride=st["q"].stride(0),
                           k_stride=st["k"].stride(0), v_stride=st["v"].stride(0), out_stride=st["out"].stride(0),
                           scale=_scale(case), cap=case["cap"], **heads)
        work = _work_buffer(lib.prompt_attention_workspace(a))
        a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
        return ctx, a, work
    if case["op"] in ("tree", "weights"):
        lse = st["lse"].contiguous()  # [seq][token][head], as the attention writes it
        a = lib.TreeArgs(q=_ptr(st["q"]), k=_ptr(st["k"]), v=_ptr(st["v"]), lens=_ptr(st["lens"]),
                         counts=_ptr(st["counts"]), parents=_ptr(st["parents"]), slopes=_ptr(st["slopes"]),
                         out=_ptr(st.get("out")), lse=_ptr(lse),
                         weights=_ptr(st.get("weights")), seqs=case["seqs"], n=case["n"],
                         max_rows=case["rows"] + case["n"], q_seq_stride=st["q"].stride(0), q_stride=st["q"].stride(1),
                         k_seq_stride=st["k"].stride(0), k_stride=kvd, v_seq_stride=st["v"].stride(0), v_stride=kvd,
                         out_seq_stride=st["q"].stride(0), out_stride=st["q"].stride(1), scale=_scale(case),
                         cap=case["cap"], **heads)
        work = None
        if case["op"] == "tree":
            work = _work_buffer(lib.tree_attention_workspace(a))
            a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
        return ctx, a, (work, lse)
    if case["op"] == "evict":
        rows, b = case["rows"], case["budget"]
        s = lib.SelectArgs(weights=_ptr(st["weights"]), lens=_ptr(st["lens"]), kept=_ptr(st["kept"]),
                           counts=_ptr(st["counts"]), caches=case["caches"], kv_heads=case["kv_heads"], max_rows=rows,
                           budget=b, sinks=case["sinks"], recent=case["recent"])
        k = lib.KeepArgs(k=_ptr(st["k"]), v=_ptr(st["v"]), weights=_ptr(st["weights"]), k_out=_ptr(st["k2"]),
                         v_out=_ptr(st["v2"]), weights_out=_ptr(st["weights2"]), rows=_ptr(st["kept"]),
                         counts=_ptr(st["counts"]), caches=case["caches"], kv_heads=case["kv_heads"],
                         head_dim=case["head_dim"], max_keep=b, per_head=1, max_rows=rows, max_rows_out=b,
                         k_cache_stride=rows * kvd, k_stride=kvd, v_cache_stride=rows * kvd, v_stride=kvd,
                         k_out_cache_stride=b * kvd, k_out_stride=kvd, v_out_cache_stride=b * kvd, v_out_stride=kvd)
        return ctx, s, k
    rows = case["rows"] + case["n"]
    k = lib.KeepArgs(k=_ptr(st["k"]), v=_ptr(st["v"]), k_out=_ptr(st["k"]), v_out=_ptr(st["v"]), rows=_ptr(st["list"]),
                     counts=_ptr(st["counts"]), first=_ptr(st["lens"]), caches=case["caches"],
                     kv_heads=case["kv_heads"], head_dim=case["head_dim"], max_keep=st["list"].shape[1], per_head=0,
                     max_rows=rows, max_rows_out=rows, k_cache_stride=rows * kvd, k_stride=kvd,
                     v_cache_stride=rows * kvd, v_stride=kvd, k_out_cache_stride=rows * kvd, k_out_stride=kvd,
                     v_out_cache_stride=rows * kvd, v_out_stride=kvd)
    return ctx, k, None


def _run_own(st):
    op = st["case"]["op"]
    ctx, a, b = st["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "prompt":
        ctx.prompt_attention(a, stream)
        return {"out": st["out"], "lse": st["lse"]}
    if op == "tree":
        ctx.tree_attention(a, stream)
        return {"out": st["out"], "lse": st["lse"]}
    if op == "weights":
        ctx.cache_weights(a, stream)
        return {"weights": st["weights"]}
    if op == "evict":
        ctx.cache_select(a, stream)
        ctx.cache_keep(b, stream)
        return {n: st[n] for n in ("kept", "counts", "k2", "v2", "weights2")}
    ctx.cache_keep(a, stream)
    return {"k": st["k"], "v": st["v"]}


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "prompt":
        return _plain_prompt(st)
    if op == "tree":
        return _plain_tree(st)
    if op == "weights":
        return _plain_weights(st)
    if op == "evict":
        return _plain_evict(st)
    return _plain_accept(st)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------


def _mean_seen(case):
    """Visible (row, key) pairs of a prompt, about."""
    n, rows0 = case["n"], case["rows0"]
    if case["mask"] == "prefix":
        image = max(0, n - 13)
        return image * n + (n - image) * n / 2
    if case["mask"] == "docs":
        return n * n / case["docs"] * 0.7
    return n * rows0 + n * (n + 1) / 2


def work(case):
    hd, kvd, qd = case["head_dim"], case["kv_heads"] * case["head_dim"], case["heads"] * case["head_dim"]
    if case["op"] == "prompt":
        rows = case["n"] + case["rows0"]
        return {"bytes": 4.0 * (2 * case["n"] * qd + 2 * rows * kvd + case["n"] * case["heads"]),
                "flops": 4.0 * hd * case["heads"] * _mean_seen(case)}
    if case["op"] in ("tree", "weights"):
        rows, n, s = case["rows"] * 0.9 + case["n"], case["n"] * 0.85, case["seqs"]
        rows, n = (case["rows"] + case["n"], case["n"]) if s == 1 else (rows, n)
        if case["op"] == "tree":
            return {"bytes": 4.0 * s * (2 * n * qd + 2 * rows * kvd + n * case["heads"]),
                    "flops": 4.0 * hd * case["heads"] * s * n * rows}
        return {"bytes": 4.0 * s * (n * qd + rows * kvd + n * case["heads"] + 2 * rows * case["kv_heads"]),
                "flops": 2.0 * hd * case["heads"] * s * n * rows}
    if case["op"] == "evict":
        c, b = case["caches"], min(case["budget"], case["rows"])
        return {"bytes": 4.0 * c * (case["kv_heads"] * (case["rows"] + 4 * b) + 4 * b * kvd), "flops": 0.0}
    return {"bytes": 4.0 * case["caches"] * max(1, case["n"] // 2) * (4 * kvd + 1), "flops": 0.0}


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence and KV head by KV head
# ---------------------------------------------------------------------------


def _exact_rows(q, k, v, case, slopes, dist, seen):
    """Out and log-sum-exp of the heads of one KV head: q [h][i][d], k/v [j][d]."""
    h, n, hd = q.shape
    s = (q.reshape(h * n, hd) @ k.T).reshape(h, n, -1) * _scale(case)
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if slopes is not None:
        s -= slopes[:, None, None] * dist
    s = torch.where(seen, s, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    out = None if v is None else (p.reshape(h * n, -1) @ v).reshape(h, n, hd)
    return out, lse, p


def _ancestors(parents, count):
    """[token][token]: whether the second is the first or one of its ancestors."""
    sees = np.zeros((len(parents), len(parents)), bool)
    for i in range(count):
        a = i
        while a >= 0:
            sees[i, a] = True
            a = int(parents[a])
    return sees


def exact(case, seed):
    st = prepare(case, seed)
    kvh, hd, f64 = case["kv_heads"], case["head_dim"], torch.float64
    if case["op"] == "prompt":
        n, rows, group = case["n"], case["rows0"] + case["n"], case["heads"] // case["kv_heads"]
        out = torch.zeros((n, kvh, group, hd), dtype=f64, device="cuda")
        lse = torch.zeros((n, kvh, group), dtype=f64, device="cuda")
        j = torch.arange(rows, device="cuda")
        for g in range(kvh):
            k, v = (st[x][:, g * hd:(g + 1) * hd].to(f64) for x in ("k", "v"))
            for i0 in range(0, n, 1024):
                i = torch.arange(i0, min(n, i0 + 1024), device="cuda")
                if st["begin"] is None:
                    seen = j[None] <= (i + case["rows0"])[:, None]
                else:
                    seen = (j[None] >= st["begin"][i][:, None]) & (j[None] < st["end"][i][:, None])
                q = st["q"][i].to(f64).reshape(-1, kvh, group, hd)[:, g].permute(1, 0, 2)
                slopes = None if st["slopes"] is None else st["slopes"].to(f64).view(kvh, group)[g]
                o, e, _ = _exact_rows(q, k, v, case, slopes, ((i + case["rows0"])[:, None] - j[None]).abs(), seen)
                out[i, g], lse[i, g] = o.permute(1, 0, 2), e.T
        return {"out": out.reshape(n, -1), "lse": lse.reshape(n, -1)}
    if case["op"] in ("tree", "weights"):
        group, n = case["heads"] // kvh, case["n"]
        out = torch.zeros((case["seqs"], n, kvh, group, hd), dtype=f64, device="cuda")
        lse = torch.zeros((case["seqs"], n, kvh, group), dtype=f64, device="cuda")
        weights = st["weights"].to(f64) if case["op"] == "weights" else None
        for s in range(case["seqs"]):
            length, count = int(st["lens"][s]), int(st["counts"][s])
            sees = _ancestors(st["parents"][s].tolist(), count)
            depth = torch.from_numpy(sees.sum(1) - 1).cuda()[:count]
            seen = torch.cat([torch.ones((count, length), dtype=torch.bool, device="cuda"),
                              torch.from_numpy(sees[:count, :count]).cuda()], 1)
            pos = torch.cat([torch.arange(length, device="cuda"), length + depth])
            dist = ((length + depth)[:, None] - pos[None]).abs()
            for g in range(kvh):
                k, v = (st[x][s, :length + count, g * hd:(g + 1) * hd].to(f64) for x in ("k", "v"))
                q = st["q"][s, :count].to(f64).reshape(count, kvh, group, hd)[:, g].permute(1, 0, 2)
                slopes = None if st["slopes"] is None else st["slopes"].to(f64).view(kvh, group)[g]
                o, e, p = _exact_rows(q, k, v, case, slopes, dist, seen)
                out[s, :count, g], lse[s, :count, g] = o.permute(1, 0, 2), e.T
                if weights is not None:  # against the rows' given log-sum-exp
                    given = st["lse"][s, :count].to(f64).view(count, kvh, group)[:, g].T
                    weights[s, g, :length + count] += (p * torch.exp(e - given)[..., None]).sum((0, 1))
        if weights is not None:
            return {"weights": weights}
        return {"out": out.reshape(case["seqs"], n, -1), "lse": lse.reshape(case["seqs"], n, -1)}
    return None

"""Refusals of the cache operators: every shape, stride and buffer that their
kernels do not take is answered before any device work.  No GPU needed."""
import ctypes as C

import pytest

from rapidocrvl_amd import lib

P = 4096  # an aligned address that is never read: every call here is refused first


def prompt(**kw):
    a = dict(q=P, k=P, v=P, out=P, workspace=P, workspace_bytes=1 << 40, q_stride=2048, k_stride=256, v_stride=256,
             out_stride=2048, n=7, rows_before=3, heads=16, kv_heads=2, head_dim=128)
    return lib.PromptArgs(**{**a, **kw})


def tree(**kw):
    a = dict(q=P, k=P, v=P, lens=P, out=P, lse=P, weights=P, workspace=P, workspace_bytes=1 << 40, q_seq_stride=1 << 20,
             q_stride=2048, k_seq_stride=1 << 20, k_stride=256, v_seq_stride=1 << 20, v_stride=256,
             out_seq_stride=1 << 20, out_stride=2048, seqs=3, n=5, max_rows=100, heads=16, kv_heads=2, head_dim=128)
    return lib.TreeArgs(**{**a, **kw})


def select(**kw):
    a = dict(weights=P, lens=P, kept=P, counts=2 * P, caches=3, kv_heads=2, max_rows=100, budget=10, sinks=2, recent=3)
    return lib.SelectArgs(**{**a, **kw})


def keep(**kw):
    a = dict(k=P, v=2 * P, k_out=P, v_out=2 * P, rows=P, counts=P, first=P, caches=3, kv_heads=2, head_dim=128,
             max_keep=5, max_rows=100, max_rows_out=100)
    for n in ("k", "v", "k_out", "v_out"):
        a[n + "_cache_stride"], a[n + "_stride"] = 1 << 16, 256
    return lib.KeepArgs(**{**a, **kw})


CALLS = {"prompt": ("pocr_prompt_attention", prompt), "tree": ("pocr_tree_attention", tree),
         "weights": ("pocr_cache_weights", tree), "select": ("pocr_cache_select", select),
         "keep": ("pocr_cache_keep", keep)}
ARG, UNS = lib.POCR_ERR_ARG, lib.POCR_ERR_UNSUPPORTED


def refused(call, want, text, **kw):
    name, make = CALLS[call]
    L = lib.load()
    rc = getattr(L, name)(None, C.byref(make(**kw)), None)
    msg = L.pocr_last_error().decode()
    assert rc == want, (rc, msg)
    assert text in msg and name in msg, msg


@pytest.mark.parametrize("call", CALLS)
def test_whole_arguments_only_lack_a_context(call):
    refused(call, ARG, "null context")


@pytest.mark.parametrize("call", CALLS)
def test_null_arguments(call):
    name, _ = CALLS[call]
    assert getattr(lib.load(), name)(None, None, None) == ARG


BAD_HEADS = [(dict(heads=0), ARG, "heads"), (dict(kv_heads=0), ARG, "heads"), (dict(heads=15), ARG, "heads"),
             (dict(heads=2048, kv_heads=2), ARG, "heads"), (dict(head_dim=96), UNS, "head_dim"),
             (dict(head_dim=0), UNS, "head_dim"), (dict(head_dim=-128), UNS, "head_dim")]
BAD_SCORES = [(dict(scale=-1.0), ARG, "scale"), (dict(scale=float("nan")), ARG, "scale"),
              (dict(scale=float("inf")), ARG, "scale"), (dict(cap=-3.0), ARG, "cap"), (dict(cap=float("nan")), ARG, "cap"),
              (dict(cap=1e-40), ARG, "cap")]


@pytest.mark.parametrize("kw,want,text", BAD_HEADS + BAD_SCORES + [
    (dict(n=0), ARG, "rows"), (dict(n=(1 << 22) + 1), ARG, "rows"), (dict(n=1 << 22, heads=1024, kv_heads=1), ARG, "rows"),
    (dict(rows_before=-1), ARG, "rows before"),
    (dict(rows_before=1 << 30), ARG, "rows before"), (dict(q=None), ARG, "null q"), (dict(k=None), ARG, "null k"),
    (dict(v=None), ARG, "null v"), (dict(out=None), ARG, "null out"), (dict(q=P + 4), ARG, "aligned"),
    (dict(k=P + 8), ARG, "aligned"), (dict(lse=P + 2), ARG, "aligned"), (dict(q_stride=2044), ARG, "q rows"),
    (dict(k_stride=258), ARG, "k rows"), (dict(v_stride=255), ARG, "v rows"), (dict(out_stride=0), ARG, "out rows"),
    (dict(row_begin=P), ARG, "together"), (dict(row_end=P), ARG, "together")])
def test_prompt_refusals(kw, want, text):
    refused("prompt", want, text, **kw)


@pytest.mark.parametrize("call", ["tree", "weights"])
@pytest.mark.parametrize("kw,want,text", BAD_HEADS + BAD_SCORES + [
    (dict(seqs=0), ARG, "sequences"), (dict(seqs=65536), ARG, "sequences"), (dict(n=0), ARG, "tokens"),
    (dict(n=65), ARG, "tokens"), (dict(max_rows=4), ARG, "max_rows"), (dict(max_rows=(1 << 30) + 1), ARG, "max_rows"),
    (dict(lens=None), ARG, "null lens"), (dict(q=None), ARG, "null q"), (dict(k=P + 4), ARG, "aligned"),
    (dict(q_stride=2046), ARG, "q rows"), (dict(k_seq_stride=0), ARG, "k blocks"), (dict(q_seq_stride=6), ARG, "q blocks"),
    (dict(side_stride=99), ARG, "side_stride"), (dict(lens=P + 1), ARG, "aligned"), (dict(positions=P + 2), ARG, "aligned")])
def test_tree_refusals(call, kw, want, text):
    refused(call, want, text, **kw)


@pytest.mark.parametrize("kw,text", [(dict(v=None), "null v"), (dict(out=None), "null out"), (dict(v_stride=12), "v rows"),
                                     (dict(out_seq_stride=-4), "out blocks"), (dict(v_seq_stride=2), "v blocks")])
def test_tree_attention_refusals(kw, text):
    refused("tree", ARG, text, **kw)


@pytest.mark.parametrize("kw,text", [(dict(lse=None), "null lse"), (dict(weights=None), "weights"),
                                     (dict(weights=P + 2), "aligned"), (dict(take=P + 4), "aligned")])
def test_weights_refusals(kw, text):
    refused("weights", ARG, text, **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(caches=0), "caches"), (dict(caches=65536), "caches"), (dict(kv_heads=0), "KV heads"), (dict(max_rows=0), "max_rows"),
    (dict(budget=0), "budget"), (dict(budget=4), "budget"), (dict(sinks=-1), "first"), (dict(recent=-1), "last"),
    (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), "budget"), (dict(side_stride=50), "side_stride"),
    (dict(weights=None), "null"), (dict(lens=None), "null"), (dict(kept=None), "null"), (dict(counts=None), "null"),
    (dict(counts=P), "counts is lens"), (dict(kept=P + 2), "aligned")])
def test_select_refusals(kw, text):
    refused("select", ARG, text, **kw)


OUT = dict(k_out=1 << 30, v_out=1 << 31)  # another place than the source


@pytest.mark.parametrize("kw,text", [
    (dict(caches=0), "caches"), (dict(kv_heads=70000), "KV heads"), (dict(max_keep=0), "max_keep"),
    (dict(max_rows=0), "max_rows"), (dict(max_rows_out=0), "max_rows_out"), (dict(k=None), "null k"),
    (dict(v_out=None), "null v_out"), (dict(k_stride=255), "k rows"), (dict(v_out_stride=128), "v_out rows"),
    (dict(k_cache_stride=0), "k blocks"), (dict(rows=None), "null rows"), (dict(counts=None), "null rows or counts"),
    (dict(weights=P), "their destinations"), (dict(positions_out=P), "their destinations"),
    (dict(first=P + 1), "aligned"), (dict(side_stride=3), "side_stride"), (dict(side_out_stride=99), "side_out_stride"),
    (dict(k_out=1 << 30), "together"), (dict(weights=P, weights_out=4 * P), "together"),
    (dict(positions=P, positions_out=4 * P), "together"), (dict(k_out_stride=512), "in place"),
    (dict(max_rows_out=90), "in place"), (dict(v_out_cache_stride=1 << 17), "in place"),
    (dict(weights=P, weights_out=P, side_out_stride=128), "in place"),
    (dict(k_out=P + 1024, v_out=1 << 31), "overlaps"), (dict(k_out=1 << 30, v_out=2 * P + 16), "overlaps"),
    (dict(weights=P, weights_out=P + 4, **OUT), "overlaps"), (dict(positions=P + 8, positions_out=P, **OUT), "overlaps")])
def test_keep_refusals(kw, text):
    refused("keep", ARG, text, **kw)


def test_keep_overlap_counts_the_destinations_own_stride():
    """Side buffers of other strides: 2,600 floats at the destination, of which the last 200 are the source's first."""
    refused("keep", ARG, "overlaps", weights=1 << 20, weights_out=(1 << 20) - 4 * 2400, side_out_stride=500, **OUT)
    refused("keep", ARG, "null context", weights=1 << 20, weights_out=(1 << 20) - 4 * 2600, side_out_stride=500, **OUT)


def test_keep_head_dim():
    refused("keep", UNS, "head_dim", head_dim=80)


@pytest.mark.parametrize("ask,make", [("pocr_prompt_attention_workspace", prompt), ("pocr_tree_attention_workspace", tree)])
def test_workspace_queries(ask, make):
    fn = getattr(lib.load(), ask)
    assert fn(None) == ARG
    assert fn(C.byref(make(head_dim=100))) == UNS
    assert fn(C.byref(make(n=0))) == ARG
    need = fn(C.byref(make(q=None, k=None, workspace=None)))  # shapes only
    assert 0 <= need < 1 << 32
    big = dict(rows_before=1 << 29) if make is prompt else dict(max_rows=1 << 30, seqs=65535)
    assert fn(C.byref(make(**big))) >= need


@pytest.mark.parametrize("call,ask", [("prompt", "pocr_prompt_attention_workspace"), ("tree", "pocr_tree_attention_workspace")])
def test_short_workspaces(call, ask):
    name, make = CALLS[call]
    shape = dict(rows_before=5000) if call == "prompt" else dict(max_rows=5000)
    need = getattr(lib.load(), ask)(C.byref(make(**shape)))
    if need:
        refused(call, ARG, "workspace", workspace_bytes=need - 1, **shape)
        refused(call, ARG, "workspace", workspace=None, **shape)
        refused(call, ARG, "workspace", workspace=P + 8, **shape)
    refused(call, ARG, "null context", workspace_bytes=need, **shape)


@pytest.mark.parametrize("call", CALLS)
def test_injected_failures_come_after_the_checks(call, monkeypatch):
    name, make = CALLS[call]
    monkeypatch.setenv("POCR_HIP_FAIL_OP", name[5:])
    ctx = C.create_string_buffer(4096)  # never looked into: the injected failure comes first
    rc = getattr(lib.load(), name)(C.cast(ctx, C.c_void_p), C.byref(make()), None)
    assert rc == lib.POCR_ERR_INJECTED and name[5:] in lib.load().pocr_last_error().decode()
    assert getattr(lib.load(), name)(C.cast(ctx, C.c_void_p), None, None) == ARG


def test_argument_structures_match_the_header():
    """Field names and order of lib.py's structures against include/pocr_hip.h."""
    import re

    text = open(lib.HEADER).read()
    for cls, name in ((lib.PromptArgs, "pocr_prompt_args"), (lib.TreeArgs, "pocr_tree_args"),
                      (lib.SelectArgs, "pocr_select_args"), (lib.KeepArgs, "pocr_keep_args")):
        end = text.index("} " + name + ";")
        body = re.sub(r"/\*.*?\*/", "", text[text.rindex("typedef struct {", 0, end) + 16:end], flags=re.S)
        fields = []
        for decl in body.split(";"):
            decl = decl.strip()
            if not decl:
                continue
            kind, rest = re.match(r"(?:const )?(\w+)(.*)", decl, re.S).groups()
            for f in rest.split(","):
                f = f.strip()
                fields.append((f.lstrip("* "), C.c_void_p if f.startswith("*") else
                               {"int64_t": C.c_int64, "int32_t": C.c_int32, "float": C.c_float}[kind]))
        assert fields == [tuple(f) for f in cls._fields_], name

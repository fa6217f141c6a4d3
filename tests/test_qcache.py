"""Refusals of the calls on K/V caches in 4 or 8 bits, and of the rotation of rows:
every shape, stride and buffer that their kernels do not take is answered before
any device work.  No GPU needed."""
import ctypes as C

import pytest

from rapidocrvl_amd import lib

ARG, UNS = lib.POCR_ERR_ARG, lib.POCR_ERR_UNSUPPORTED
# addresses that are never read: every call here is refused first
Q, K, V, QO, KO, VO = (i << 32 for i in range(1, 7))
CODES = [i << 33 for i in range(10, 14)]
SIDE = 1 << 40


def rows(cache=False, **kw):
    a = dict(q=Q, k=K, v=V, q_out=QO, k_out=None if cache else KO, v_out=None if cache else VO, positions=SIDE,
             freqs=SIDE + 4096, q_norm=SIDE + 8192, k_norm=SIDE + 8192, counts=SIDE + 12288, first=SIDE + 16384,
             seqs=3, n=7, heads=16, kv_heads=2, head_dim=128, rotary_dim=128, axes=3, max_rows=50, eps=1e-5)
    for n in ("q", "q_out"):
        a[n + "_seq_stride"], a[n + "_stride"] = 1 << 20, 2048
    for n in ("k", "v", "k_out", "v_out"):
        a[n + "_seq_stride"], a[n + "_stride"] = 1 << 20, 256
    sections = kw.pop("sections", (16, 24, 24))
    r = lib.RowsArgs(**{**a, **kw})
    r.sections[:len(sections)] = sections
    return r


def qcache(**kw):
    a = dict(k_codes=CODES[0], v_codes=CODES[1], k_params=CODES[2], v_params=CODES[3], seqs=3, kv_heads=2, head_dim=128,
             capacity=100, bits=4)
    return lib.QCache(**{**a, **kw})


def read(**kw):
    a = dict(k_out=KO, v_out=VO, counts=SIDE, k_out_seq_stride=1 << 20, k_out_stride=256, v_out_seq_stride=1 << 20,
             v_out_stride=256, n=20)
    return lib.QReadArgs(**{**a, **kw})


def attention(**kw):
    a = dict(q=Q, out=QO, lse=SIDE, lens=SIDE + 65536, counts=SIDE + 69632, workspace=SIDE << 1, workspace_bytes=1 << 40,
             q_seq_stride=1 << 20, q_stride=2048, out_seq_stride=1 << 20, out_stride=2048, n=5, heads=16, max_rows=100)
    return lib.QAttentionArgs(**{**a, **kw})


CACHE = ("bits", "capacity", "seq_stride", "k_codes", "v_codes", "k_params", "v_params")


def call(name, kw):
    c = {k[6:]: v for k, v in kw.items() if k.startswith("cache_")}
    kw = {k: v for k, v in kw.items() if not k.startswith("cache_")}
    L, cache = lib.load(), C.byref(qcache(**c))
    if name == "rotate":
        return L.pocr_rotate_rows(None, C.byref(rows(**kw)), None)
    if name == "write":
        return L.pocr_qcache_write(None, C.byref(rows(True, **kw)), cache, None)
    if name == "read":
        return L.pocr_qcache_read(None, C.byref(read(**kw)), cache, None)
    return L.pocr_qcache_attention(None, C.byref(attention(**kw)), cache, None)


NAMES = {"rotate": "pocr_rotate_rows", "write": "pocr_qcache_write", "read": "pocr_qcache_read",
         "attention": "pocr_qcache_attention"}


def refused(name, want, text, **kw):
    rc = call(name, kw)
    msg = lib.load().pocr_last_error().decode()
    assert rc == want, (rc, msg)
    assert text in msg and NAMES[name] in msg, msg


@pytest.mark.parametrize("name", NAMES)
def test_whole_arguments_only_lack_a_context(name):
    refused(name, ARG, "null context")


@pytest.mark.parametrize("name", NAMES)
def test_null_arguments(name):
    L, c = lib.load(), C.byref(qcache())
    if name == "rotate":
        assert L.pocr_rotate_rows(None, None, None) == ARG
        return
    f = getattr(L, NAMES[name])
    assert f(None, None, c, None) == ARG
    a = {"write": rows(True), "read": read(), "attention": attention()}[name]
    assert f(None, C.byref(a), None, None) == ARG
    assert "null cache" in L.pocr_last_error().decode()


BAD_ROWS = [
    (dict(seqs=0), ARG, "sequences"), (dict(n=0), ARG, "tokens"), (dict(n=(1 << 22) + 1), ARG, "tokens"),
    (dict(head_dim=96), UNS, "head_dim"), (dict(heads=0), ARG, "heads of q"), (dict(heads=1025), ARG, "heads of q"),
    (dict(q=Q + 4), ARG, "aligned"), (dict(k=K + 8), ARG, "aligned"), (dict(q_out=None), ARG, "null q_out"),
    (dict(q=None), ARG, "without q"), (dict(q_stride=2044), ARG, "q rows"), (dict(k_stride=258), ARG, "k rows"),
    (dict(v_seq_stride=0), ARG, "v blocks"), (dict(q_seq_stride=1 << 41), ARG, "stride"),
    (dict(rotary_dim=8), ARG, "rotary_dim"), (dict(rotary_dim=144), ARG, "rotary_dim"), (dict(rotary_dim=-16), ARG, "rotary_dim"),
    (dict(rotary_dim=0), ARG, "positions without"), (dict(positions=None), ARG, "positions"), (dict(freqs=None), ARG, "freqs"),
    (dict(freqs=SIDE + 4100), ARG, "aligned"), (dict(positions=SIDE + 2), ARG, "aligned"), (dict(axes=0), ARG, "axes"),
    (dict(axes=5), ARG, "axes"), (dict(sections=(16, 24, 23)), ARG, "sections"), (dict(sections=(-8, 36, 36)), ARG, "section 0"),
    (dict(axes=2), ARG, "sections"), (dict(sections=(10, 10, 65)), ARG, "section 2"),
    (dict(sections=(16, 24, 24), interleaved=1), ARG, "section 1"), (dict(eps=-1.0), ARG, "eps"),
    (dict(eps=float("nan")), ARG, "eps"), (dict(q_out=K), ARG, "overlaps k"), (dict(q_out=Q + 16), ARG, "overlaps q"),
    (dict(q_out=SIDE), ARG, "side buffer"), (dict(q_out=QO, q_out_seq_stride=2048), ARG, "sequences of q_out overlap"),
]


@pytest.mark.parametrize("name", ["rotate", "write"])
@pytest.mark.parametrize("kw,want,text", BAD_ROWS)
def test_row_refusals(name, kw, want, text):
    if name == "write" and "head_dim" in kw:
        kw = {**kw, "cache_head_dim": kw["head_dim"]}
    refused(name, want, text, **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None, k=None, v=None, q_out=None, k_out=None, v_out=None), "null q, k and v"), (dict(max_rows=6), "max_rows"),
    (dict(max_rows=(1 << 30) + 1), "max_rows"), (dict(kv_heads=0), "heads of k"), (dict(k=None), "k_out without k"),
    (dict(k_out=None), "null k_out"), (dict(v_out=KO), "another destination"), (dict(k_out=K), "overlaps k"),
    (dict(k_out=V), "overlaps v"), (dict(v_out_stride=128), "v_out rows"), (dict(k_out_seq_stride=-4), "k_out blocks")])
def test_rotate_refusals(kw, text):
    refused("rotate", ARG, text, **kw)


def test_rotation_in_place_is_taken():
    refused("rotate", ARG, "null context", q_out=Q, k_out=K, v_out=V, first=None)
    refused("rotate", ARG, "overlaps k", k_out=K)  # elsewhere in the same rows


def test_packed_rows_rotate_in_place():
    """q | k | v rows of one projection: destinations between each other's rows do not meet."""
    at = dict(q=Q, k=Q + 8192, v=Q + 9216, q_out=Q, k_out=Q + 8192, v_out=VO, first=None, max_rows=7)
    for n in ("q", "k", "v", "q_out", "k_out"):
        at[n + "_stride"], at[n + "_seq_stride"] = 2560, 7 * 2560
    refused("rotate", ARG, "null context", **at)
    refused("rotate", ARG, "overlaps", **{**at, "k_out": Q + 8176})


BAD_CACHE = [(dict(cache_bits=6), UNS, "bits"), (dict(cache_capacity=0), ARG, "capacity"),
             (dict(cache_capacity=(1 << 30) + 1), ARG, "capacity"), (dict(cache_seq_stride=199), ARG, "rows apart"),
             (dict(cache_seq_stride=-1), ARG, "rows apart"), (dict(cache_seq_stride=1 << 41), ARG, "stride"),
             (dict(cache_k_codes=None), ARG, "null or not"), (dict(cache_v_codes=CODES[1] + 8), ARG, "aligned"),
             (dict(cache_k_params=CODES[2] + 4), ARG, "aligned"), (dict(cache_v_params=None), ARG, "null or not"),
             (dict(cache_head_dim=32), UNS, "head_dim"), (dict(cache_seqs=0), ARG, "sequences"), (dict(cache_seqs=65536), ARG, "sequences")]


@pytest.mark.parametrize("name", ["write", "read", "attention"])
@pytest.mark.parametrize("kw,want,text", BAD_CACHE)
def test_cache_refusals(name, kw, want, text):
    refused(name, want, text, **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(cache_seqs=4), "a cache of"), (dict(cache_kv_heads=4), "a cache of"), (dict(cache_head_dim=64), "a cache of"),
    (dict(k=None), "null k or v"), (dict(v=None), "null k or v"), (dict(k_out=KO), "k_out and v_out are null"),
    (dict(v_out=VO), "k_out and v_out are null"), (dict(n=101), "101 tokens"), (dict(cache_v_codes=CODES[0]), "another destination"),
    (dict(cache_k_params=K), "the cache overlaps k"), (dict(cache_v_codes=QO + 1024), "another destination"),
    (dict(cache_k_codes=SIDE), "side buffer")])
def test_write_refusals(kw, text):
    refused("write", ARG, text, **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(n=0), "rows"), (dict(k_out=None, v_out=None), "null k_out and v_out"), (dict(rows=SIDE + 4096, first=SIDE + 8192), "rows and first"),
    (dict(rows=SIDE + 2), "aligned"), (dict(k_out_stride=128), "k_out rows"), (dict(v_out=KO), "k_out overlaps v_out"),
    (dict(v_out=CODES[0]), "overlaps the cache"), (dict(k_out=SIDE), "index buffer"), (dict(k_out=KO + 4), "aligned"),
    (dict(k_out_seq_stride=256), "sequences of k_out overlap")])
def test_read_refusals(kw, text):
    refused("read", ARG, text, **kw)


@pytest.mark.parametrize("kw,want,text", [
    (dict(heads=15), ARG, "heads"), (dict(heads=0), ARG, "heads"), (dict(heads=2048), ARG, "heads"), (dict(n=0), ARG, "tokens"),
    (dict(n=1 << 22, heads=16), ARG, "tokens"), (dict(max_rows=0), ARG, "max_rows"), (dict(max_rows=101), ARG, "max_rows"),
    (dict(window=-1), ARG, "window"), (dict(scale=-1.0), ARG, "scale"), (dict(cap=float("nan")), ARG, "cap"),
    (dict(q=None), ARG, "null q"), (dict(out=None), ARG, "null out"), (dict(lens=None), ARG, "null lens"),
    (dict(lse=SIDE + 2), ARG, "aligned"), (dict(q_stride=2046), ARG, "q rows"), (dict(out_seq_stride=2048), ARG, "overlap")])
def test_attention_refusals(kw, want, text):
    refused("attention", want, text, **kw)


@pytest.mark.parametrize("kw,want", [(dict(n=0), ARG), (dict(heads=3), ARG)])
def test_attention_workspace_answers_for_shapes(kw, want):
    L = lib.load()
    assert L.pocr_qcache_attention_workspace(C.byref(attention(**kw)), C.byref(qcache())) == want
    assert L.pocr_qcache_attention_workspace(None, C.byref(qcache())) == ARG
    assert L.pocr_qcache_attention_workspace(C.byref(attention()), None) == ARG
    need = lib.qcache_attention_workspace(attention(q=None, lens=None, q_stride=0), qcache(k_codes=None))
    assert need >= 0
    if need:
        refused("attention", ARG, "workspace", workspace_bytes=need - 1)
        refused("attention", ARG, "workspace", workspace=None)

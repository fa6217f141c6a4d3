"""Into how many workgroups the attention over caches in 4 or 8 bits cuts its keys, as its
workspace tells.  No GPU needed."""
import pytest

from rapidocrvl_amd import lib


@pytest.mark.parametrize("hd,bits,places", [(128, 4, 768), (128, 8, 512), (64, 4, 768), (64, 8, 768)])
@pytest.mark.parametrize("n", [33, 64, 256, 500, 540, 600, 700, 800, 1000])
@pytest.mark.parametrize("seqs,rows", [(1, 2048), (1, 8192), (16, 8192)])
def test_workgroups_of_many_rows_fill_the_device(hd, bits, places, n, seqs, rows):
    """256 CUs hold two or three workgroups each, of 64 rows: a call has no more of them, or
    twice as many that are so much shorter that less is done one after the other."""
    c = lib.QCache(seqs=seqs, kv_heads=2, head_dim=hd, capacity=rows, bits=bits)
    need = lib.qcache_attention_workspace(lib.QAttentionArgs(n=n, heads=16, max_rows=rows), c)
    tiles = -(-n * 8 // 64) * 2 * seqs
    work = need // (64 * (hd + 2) * 4)
    assert work * 64 * (hd + 2) * 4 == need and work % tiles == 0
    shares, blocks, once = max(1, work // tiles), rows // 32, max(1, places // tiles)
    assert shares > 1 or tiles > places // 2
    if work > max(places, 256):
        assert work <= 2 * places and 2 * -(-blocks // shares) < -(-blocks // once)

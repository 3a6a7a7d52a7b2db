"""How many parts the attention over the paged cache asks a workspace for, by its rule: where several workgroups read a sequence's tokens (rows x heads of a group over 16) as many, in powers of two, as
give 256 workgroups at most, or 1024 of at least 1024 tokens each (CPU: no launch)."""
import ctypes as C

import pytest

from qwegn_amd import qwhip


@pytest.mark.parametrize("rows,seqs,kv,shared,d,length,window,parts", [
    (16, 1, 8, 5, 128, 1500, 0, 4), (32, 1, 8, 5, 128, 1500, 0, 2), (64, 1, 8, 5, 128, 1500, 0, 1), (16, 1, 8, 5, 128, 8000, 0, 4), (16, 1, 8, 5, 128, 32768, 0, 32),
    (16, 1, 8, 5, 128, 900, 0, 1), (8, 20, 4, 4, 256, 6000, 1000, 1), (4, 20, 2, 8, 256, 6000, 1000, 2), (32, 3, 4, 6, 64, 6000, 1000, 1), (4, 5, 4, 6, 64, 3000, 0, 4), (8, 1, 1, 5, 128, 4096, 0, 32),
])
def test_parts_of_several_workgroups(rows, seqs, kv, shared, d, length, window, parts):
    lib = qwhip.load()
    cache = qwhip.KvCache(pages=256, bytes=1 << 50, page_count=1 << 20, page_size=64, kv_heads=kv, head_dim=d)
    batch = qwhip.KvBatch(row_start=256, lengths=256, block_table=256, ld_table=(length + 63) // 64, seqs=seqs, max_rows=rows, max_length=length)
    total = rows * seqs
    need = lib.qwhip_kv_attention_workspace_bytes(C.byref(cache), C.byref(batch), kv * shared, total, window)
    assert need == (parts * total * kv * shared * (d + 2) * 4 if parts > 1 else 0)

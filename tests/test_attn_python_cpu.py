"""The Python calls of the operators of include/apus_attn_gcuda.h: what they refuse, and what they hand to the
library.  No GPU is used."""
import pytest
import torch

import apus_gcuda as G


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("nseq", [1, 3])
def test_batch_holds_max_len_to_the_page_table(nseq):
    """A view of a wider table: the last columns are as far apart as the table is wide, and behind the last row's there
    is nothing."""
    wide = ints(nseq, 100)
    for table in (wide, wide[:, 98:], wide[:, :7], ints(nseq, 1), ints(nseq, 0)):
        pages = table.shape[1]
        b = G.Kv4Batch(ints(nseq + 1), ints(nseq), table, 1, 64 * pages)
        # entries that the kernels may read
        last = (nseq - 1) * b.desc.table_stride + -(-b.desc.max_len // 64) if b.desc.max_len else 0
        have = table.untyped_storage().nbytes() // 4 - table.storage_offset()
        assert last <= have
        for bad in (64 * pages + 1, 64 * 100 + 1, -1):
            with pytest.raises(G.GcudaError, match="pages"):
                G.Kv4Batch(ints(nseq + 1), ints(nseq), table, 1, bad)

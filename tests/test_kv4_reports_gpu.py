"""What the operators of include/apus_attn_gcuda.h report of entries out of bounds, and the error word."""
import pytest
import torch

from test_kv4_gpu import Case, bf16, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nseq", [2, 5, 700])
def test_cache_rows_report_every_sequence(gcuda, nseq):
    """A row range or a length out of bounds is reported by append and read, that of a sequence without rows and
    that behind the last row too; the other rows are as ever."""
    c = Case(gcuda, 64, 2, [70] + [0] * (nseq - 1), [3] + [0] * (nseq - 1), seed=1)
    k, v = (bf16(c.g, 3, 2, 64).cuda() for _ in range(2))
    gcuda.kv4_append(c.cache, c.batch, k, v)
    want = [torch.empty_like(k) for _ in range(2)]
    gcuda.kv4_read(c.cache, c.batch, *want)
    assert gcuda.apus_gcuda_kernel_error() == 0
    cu, lens = c.cu.tolist(), list(c.lens)
    bad_range = cu[:-1] + [1 << 30]
    bad_len = lens[:-1] + [-1]
    for cu_, lens_ in ((bad_range, lens), (cu, bad_len)):
        b = c.make_batch(cu_, lens_, max_rows=3, max_len=70)
        gcuda.kv4_append(c.cache, b, k, v)
        assert gcuda.apus_gcuda_kernel_error() == 42
        got = [torch.empty_like(k) for _ in range(2)]
        gcuda.kv4_read(c.cache, b, *got)
        assert gcuda.apus_gcuda_kernel_error() == 42 and gcuda.apus_gcuda_kernel_error() == 0
        assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_error_word_is_the_most_severe_and_clears_all(gcuda):
    """Errors of several operators at once: the largest code is returned, and nothing is left for a later call."""
    g = gen(2)
    c = Case(gcuda, 64, 1, [130, 20], [2, 1], seed=2)
    c.fill_all()
    q = bf16(g, 3, 2, 64).cuda()
    k, v = (bf16(g, 3, 1, 64).cuda() for _ in range(2))
    table = c.table.clone()
    c.table[0, 2] = c.pages.shape[0]
    bad_page = c.make_batch(c.cu, c.lens)
    keep = c.dev
    c.table = table
    bad_len = c.make_batch(c.cu, [130, 1 << 20], max_len=130)
    for first, second in ((bad_page, bad_len), (bad_len, bad_page)):
        gcuda.kv4_append(c.cache, first, k, v)           # 41 in one word, 42 in another
        c.attn(q, 0.1, batch=second)
        assert gcuda.apus_gcuda_kernel_error() == 42
        assert gcuda.apus_gcuda_kernel_error() == 0
        for b in (first, second):                        # both in the same word, in either order
            c.attn(q, 0.1, batch=b)
        assert gcuda.apus_gcuda_kernel_error() == 42
        assert gcuda.apus_gcuda_kernel_error() == 0
    assert keep

"""What the operators of include/apus_attn_gcuda.h refuse, and the index
arithmetic of the 4-bit cache (csrc/kv4_layout.h, compiled for the host): no
GPU is used.  The addresses below are never followed: every call is refused
before anything is launched, or has nothing to do."""
import ctypes as C
import os
import subprocess

import pytest

import apus_gcuda as G
import attn_ref as R
from conftest import PKG

AT = 0x7000_0000_0000      # 16-byte aligned, no memory there


def rows(**kw):
    d = dict(p=AT, rows=4, heads=2, row_stride=256, head_stride=128) | kw
    return G.HeadRows(*(d[n] for n, _ in G.HeadRows._fields_))


def cache(**kw):
    d = dict(pages=AT, num_pages=8, heads=2, dim=128) | kw
    return G.Kv4CacheDesc(*(d[n] for n, _ in G.Kv4CacheDesc._fields_))


def batch(**kw):
    d = dict(cu_rows=AT, kv_len=AT, page_table=AT, table_stride=4, nseq=2, max_rows=3, max_len=256) | kw
    return G.Kv4BatchDesc(*(d[n] for n, _ in G.Kv4BatchDesc._fields_))


def prompt(**kw):
    d = dict(cu_q=AT, cu_k=AT, nseq=2, max_rows=3) | kw
    return G.PromptBatchDesc(*(d[n] for n, _ in G.PromptBatchDesc._fields_))


def refused(rc, *words):
    err = G.apus_gcuda_last_error().decode()
    G.apus_gcuda_clear_error()
    assert rc == -1 and all(w in err for w in words), (rc, err)


BAD_ROWS = [dict(p=0), dict(p=AT + 8), dict(row_stride=260), dict(head_stride=132), dict(row_stride=64), dict(head_stride=64),
            dict(heads=0), dict(rows=1 << 31), dict(heads=70000), dict(row_stride=0), dict(head_stride=0),
            dict(row_stride=1 << 31)]
BAD_CACHE = [dict(dim=96), dict(dim=0), dict(dim=512), dict(heads=0), dict(pages=0), dict(pages=AT + 4),
             dict(num_pages=1 << 31)]
BAD_SCALES = [0.0, -0.5, float("nan"), float("inf")]
BAD_BATCH = [dict(cu_rows=0), dict(kv_len=0), dict(page_table=0), dict(max_len=257), dict(nseq=70000),
             dict(max_rows=1 << 31), dict(table_stride=1 << 31)]


@pytest.mark.parametrize("fn,what", [(G.apus_gcuda_kv4_append_dev, "kv4_append"), (G.apus_gcuda_kv4_read_dev, "kv4_read")])
def test_cache_rows_refused(fn, what):
    good = cache(), batch(), rows(), rows()
    for bad in BAD_CACHE:
        refused(fn(cache(**bad), *good[1:], None), what)
    for bad in BAD_BATCH:
        refused(fn(good[0], batch(**bad), *good[2:], None), what)
    for bad in BAD_ROWS:
        refused(fn(*good[:2], rows(**bad), good[3], None), what)
        refused(fn(*good[:3], rows(**bad), None), what)
    refused(fn(*good[:3], rows(rows=5), None), what, "5")
    refused(fn(*good[:2], rows(heads=1), rows(heads=1), None), what, "heads")
    for i in range(4):
        refused(fn(*(None if i == j else x for j, x in enumerate(good)), None), what)


def test_read_refuses_overlapping_outputs():
    over = rows(row_stride=128, head_stride=128)
    refused(G.apus_gcuda_kv4_read_dev(cache(), batch(), over, rows(), None), "overlap")
    refused(G.apus_gcuda_kv4_read_dev(cache(), batch(), rows(), over, None), "overlap")


def attn(c=None, b=None, q=None, out=None, sel=None, stride=0, pool=0, work=AT, nbytes=1 << 30, scale=0.1):
    return G.apus_gcuda_kv4_attn_dev(c or cache(), b or batch(), q or rows(heads=4, row_stride=512),
                                     out or rows(heads=4, row_stride=512), scale, sel, stride, pool, work, nbytes, None)


def test_attention_refused():
    for bad in BAD_CACHE:
        refused(attn(c=cache(**bad)), "kv4_attn")
        assert G.apus_gcuda_kv4_attn_workspace(cache(**bad), batch(), 4) == 0
        refused(-1, "kv4_attn_workspace")
    for bad in BAD_BATCH:
        refused(attn(b=batch(**bad)), "kv4_attn")
    for bad in BAD_ROWS:
        refused(attn(q=rows(**(dict(heads=4, row_stride=512) | bad))), "kv4_attn")
        refused(attn(out=rows(**(dict(heads=4, row_stride=512) | bad))), "kv4_attn")
    refused(attn(q=rows(heads=3, row_stride=512), out=rows(heads=3, row_stride=512)), "3 query heads over 2")
    refused(attn(out=rows(heads=2)), "out")
    refused(attn(out=rows(heads=4, row_stride=512, rows=3)), "out")
    refused(attn(out=rows(heads=4, row_stride=128)), "overlap")
    for scale in BAD_SCALES:
        refused(attn(scale=scale), "scale")
    refused(attn(sel=AT, stride=8, pool=0), "pools")
    refused(attn(sel=AT, stride=8, pool=129), "pools")
    refused(attn(sel=AT, stride=1 << 31, pool=4), "pools")
    refused(attn(b=batch(max_rows=1 << 30)), "too many")
    refused(attn(b=batch(max_len=(1 << 28) + 64, table_stride=1 << 23)), "positions")
    big = batch(max_len=1 << 16, table_stride=1 << 10)
    need = G.apus_gcuda_kv4_attn_workspace(cache(), big, 4)
    assert need > 0
    refused(attn(b=big, nbytes=need - 1), "workspace", str(need))
    refused(attn(b=big, work=None), "workspace")
    refused(attn(b=big, work=AT + 4), "workspace")


def test_prompt_refused():
    def call(b=None, q=None, k=None, v=None, out=None, dim=128, scale=0.1):
        wide = rows(heads=4, row_stride=512)
        return G.apus_gcuda_prompt_attn_dev(b or prompt(), q or wide, k or rows(), v or rows(), out or wide, dim, scale, None)
    for dim in (0, 32, 96, 512):
        refused(call(dim=dim), "prompt_attn", str(dim))
    for scale in BAD_SCALES:
        refused(call(scale=scale), "scale")
    for bad in (dict(cu_q=0), dict(cu_k=0), dict(nseq=70000), dict(max_rows=1 << 31)):
        refused(call(b=prompt(**bad)), "prompt_attn")
    for bad in BAD_ROWS:
        refused(call(q=rows(**(dict(heads=4, row_stride=512) | bad))), "prompt_attn")
        refused(call(out=rows(**(dict(heads=4, row_stride=512) | bad))), "prompt_attn")
        refused(call(k=rows(**bad)), "prompt_attn")
        refused(call(v=rows(**bad)), "prompt_attn")
    refused(call(k=rows(heads=1)), "prompt_attn")
    refused(call(v=rows(rows=3)), "prompt_attn")
    refused(call(q=rows(heads=3, row_stride=512), out=rows(heads=3, row_stride=512)), "prompt_attn")
    refused(call(out=rows(heads=4, row_stride=512, rows=3)), "prompt_attn")
    refused(call(out=rows(heads=4, row_stride=128)), "overlap")
    refused(G.apus_gcuda_prompt_attn_dev(None, rows(), rows(), rows(), rows(), 128, 0.1, None), "batch")


def test_nothing_to_do():
    """No sequences, no rows: done, without a launch."""
    empty = rows(rows=0, p=0)
    assert G.apus_gcuda_kv4_append_dev(cache(), batch(), empty, empty, None) == 0
    assert G.apus_gcuda_kv4_read_dev(cache(), batch(nseq=0, cu_rows=0), rows(), rows(), None) == 0
    assert attn(b=batch(nseq=0), work=None, nbytes=0) == 0
    assert attn(b=batch(max_rows=0), work=None, nbytes=0) == 0
    assert G.apus_gcuda_kv4_attn_workspace(cache(), batch(nseq=0), 4) == 0
    assert G.apus_gcuda_prompt_attn_dev(prompt(nseq=0), rows(), rows(), rows(), rows(), 128, 0.1, None) == 0
    assert G.apus_gcuda_last_error() == b""


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_workspace_grows_with_the_bounds(dim):
    for nseq in (1, 2, 48, 300):
        for max_rows in (1, 2, 3, 4, 5, 17):
            for max_len in (1, 512, 513, 700, 5000, 131072):
                def need(n, r, m):
                    return G.apus_gcuda_kv4_attn_workspace(cache(heads=8, dim=dim), batch(nseq=n, max_rows=r, max_len=m,
                                                                                          table_stride=4096), 32)
                at = need(nseq, max_rows, max_len)
                assert all(need(*b) >= at for b in ((nseq + 1, max_rows, max_len), (nseq, max_rows + 1, max_len),
                                                    (nseq, max_rows, max_len + 1), (nseq, max_rows, max_len * 2)))


def test_page_bytes():
    for heads, dim in ((1, 64), (8, 128), (64, 256)):
        assert G.apus_gcuda_kv4_page_bytes(heads, dim) == heads * 72 * dim
    assert G.apus_gcuda_kv4_page_bytes(4, 100) == 0
    G.apus_gcuda_clear_error()


def test_python_refusals():
    import torch
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(G.GcudaError):
        G.head_rows(x.float())
    with pytest.raises(G.GcudaError):
        G.head_rows(x.transpose(1, 2))
    with pytest.raises(G.GcudaError):
        G.head_rows(x[0])
    with pytest.raises(G.GcudaError):
        G.Kv4Cache(torch.zeros(3, 2, 100, dtype=torch.uint8))
    with pytest.raises(G.GcudaError):
        G.Kv4Cache(torch.zeros(3, 2, 72 * 128))
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(G.GcudaError):
        G.Kv4Batch(i(3), i(3), i(3, 4), 1, 1)
    with pytest.raises(G.GcudaError):
        G.Kv4Batch(i(3), i(2).long(), i(2, 4), 1, 1)
    with pytest.raises(G.GcudaError):
        G.PromptBatch(i(3), i(4), 1)
    c = G.Kv4Cache(torch.zeros(3, 2, 72 * 128, dtype=torch.uint8))
    with pytest.raises(G.GcudaError):     # tensors in host memory
        G.kv4_append(c, G.Kv4Batch(i(2), i(1), i(1, 4), 1, 1), x, x)
    with pytest.raises(G.GcudaError):     # another head dim
        G.kv4_append(c, G.Kv4Batch(i(2), i(1), i(1, 4), 1, 1), x[..., :64], x[..., :64])


SRC = r"""
#include "kv4_layout.h"
extern "C" {
int k_word(int d, int p, int j, int q) { return kv4_k_word(d, p, j, q); }
int v_word(int d, int p, int g, int jj) { return kv4_v_word(d, p, g, jj); }
size_t block_at(int page, int head, int heads, int dim) { return kv4_block_at(page, head, heads, dim); }
int page_ok(int page, long n) { return kv4_page_ok(page, n); }
void seq(int lo, int hi, int len, long rows, long mr, long ml, int *o) {
    struct Kv4Seq s = kv4_seq(lo, hi, len, rows, mr, ml);
    o[0] = s.row0; o[1] = s.n; o[2] = s.len; o[3] = s.bad;
}
}
"""


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4")
    src, so = d / "l.cpp", d / "l.so"
    src.write_text(SRC)
    subprocess.check_call(["g++", "-O1", "-fsanitize=undefined", "-shared", "-fPIC", "-I", os.path.join(PKG, "csrc"), str(src), "-o",
                           str(so), "-static-libubsan"])
    lib = C.CDLL(str(so))
    lib.block_at.restype = C.c_size_t
    lib.seq.argtypes = [C.c_int, C.c_int, C.c_int, C.c_long, C.c_long, C.c_long, C.c_void_p]
    lib.page_ok.argtypes = [C.c_int, C.c_long]
    return lib


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_words(layout, dim):
    """The kernels' word formulas are the header's, and every code of a row has one place inside it."""
    for p in range(64):
        ks, vs = set(), set()
        for d in range(dim):
            kw, ki, vw, vi = R.word_and_code(dim, p, d)
            assert layout.k_word(dim, p, d // 32, d % 32 // 8) == kw
            assert layout.v_word(dim, p, d % 32 // 4, d // 64) == vw
            ks.add((kw, ki)), vs.add((vw, vi))
        assert ks == vs == {(w, i) for w in range(dim // 8) for i in range(8)}


def test_bounds(layout):
    assert layout.block_at(2 ** 31 - 1, 63, 64, 256) == ((2 ** 31 - 1) * 64 + 63) * 72 * 256
    assert [layout.page_ok(p, 5) for p in (-2 ** 31, -1, 0, 4, 5, 2 ** 31 - 1)] == [0, 0, 1, 1, 0, 0]
    o = (C.c_int * 4)()
    for args, want in (((2, 5, 9, 10, 3, 9), (2, 3, 9, 0)), ((2, 2, 0, 10, 3, 9), (2, 0, 0, 0)),
                       ((2, 6, 9, 10, 3, 9), (0, 0, 9, 1)), ((8, 11, 9, 10, 3, 9), (0, 0, 9, 1)),
                       ((5, 2, 9, 10, 3, 9), (0, 0, 9, 1)), ((-1, 1, 9, 10, 3, 9), (0, 0, 9, 1)),
                       ((2, 5, 10, 10, 3, 9), (2, 3, 0, 1)), ((2, 5, -1, 10, 3, 9), (2, 3, 0, 1)),
                       ((-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1, 10, 3, 9), (0, 0, 0, 1))):
        layout.seq(*args, o)
        assert tuple(o) == want, args

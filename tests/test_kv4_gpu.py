"""The 4-bit key/value cache on the B200: rows quantised as they are written
(apus_gcuda_kv4_append_dev), read back (apus_gcuda_kv4_read_dev) and attended
to (apus_gcuda_kv4_attn_dev), against 64-bit references (attn_ref.py).  Codes
and scales must be equal bit for bit; attention is held elementwise to the
bound that two f16 roundings of a weight (as it is, and times its value's scale)
and its fp32 sums allow."""
import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf16(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


class Case:
    """Sequences of n rows and given lengths over shuffled pages."""

    def __init__(self, gcuda, dim, heads, lens, rows, seed=1, fill=0xff, spare=2, max_rows=None, behind=0):
        self.G, self.dim, self.heads, self.lens, self.rows = gcuda, dim, heads, lens, rows
        self.g = gen(seed)
        need = [-(-n // 64) for n in lens]
        order = torch.randperm(sum(need) + spare, generator=self.g).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        # untouched places hold what cannot be taken for data: scales of 0xffff are NaN
        self.pages = torch.full((sum(need) + spare, heads, 72 * dim), fill, dtype=torch.uint8, device="cuda")
        self.cu = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
        self.total = int(self.cu[-1]) + behind
        self.cache = gcuda.Kv4Cache(self.pages)
        self.max_rows = max_rows or max(rows)
        self.batch = self.make_batch(self.cu, lens)

    def make_batch(self, cu, lens, max_rows=None, max_len=None):
        self.dev = [torch.as_tensor(x, dtype=torch.int32).cuda() for x in (cu, lens, self.table)]
        return self.G.Kv4Batch(*self.dev, max_rows=max_rows or self.max_rows,
                               max_len=max(max(lens), 0) if max_len is None else max_len)

    def fill_all(self, std_k=1.0, std_v=1.0):
        """Every sequence's positions, written by the append under test; what the cache then holds, in 64 bits."""
        starts = torch.tensor([0] + self.lens).cumsum(0)
        n = int(starts[-1])
        k, v = bf16(self.g, n, self.heads, self.dim, std=std_k), bf16(self.g, n, self.heads, self.dim, std=std_v)
        self.write_all(k, v)

    def write_all(self, k, v):
        starts = torch.tensor([0] + self.lens).cumsum(0)
        b = self.make_batch(starts, self.lens, max_rows=max(self.lens))
        self.keep = self.dev
        self.G.kv4_append(self.cache, b, k.cuda(), v.cuda())
        torch.cuda.synchronize()
        self.k, self.v = (R.held(*R.quantise(x)) for x in (k, v))
        ks = R.quantise(k)[1]
        self.offset = 16 * ks.repeat_interleave(32, -1)     # the code's offset: 8 s is added and taken away
        self.most = R.quantise(v)[1].amax(-1)               # each position's largest value scale
        self.starts = starts.tolist()
        self.batch = self.make_batch(self.cu, self.lens)

    def attn(self, q, scale, sel=None, pool=0, out=None, work=None, batch=None):
        G, batch = self.G, batch or self.batch
        heads = q.shape[1]
        if out is None:
            out = torch.full_like(q, 7.0)
        if work is None:
            work = torch.full((max(G.kv4_attn_workspace(self.cache, batch, heads), 1),), 0xff, dtype=torch.uint8,
                              device="cuda")
        G.kv4_attn(self.cache, batch, q, out, scale, work, sel=sel, pool=pool)
        return out

    def check(self, q, got, scale, sel=None, pool=0):
        for i, (n, length) in enumerate(zip(self.rows, self.lens)):
            if not n:
                continue
            r0, k0 = int(self.cu[i]), self.starts[i]
            j = torch.arange(length)[None]
            end = length - n + 1 + torch.arange(n)[:, None]
            seen = j < end
            if sel is not None:
                padded = torch.nn.functional.pad(sel[r0:r0 + n], (0, length // pool + 1))
                seen = seen & ((j >= end - end % pool) | padded.gather(1, (j // pool).expand(n, -1)).bool())
            ref = R.attention(q[r0:r0 + n].double().cpu(), self.k[k0:k0 + length], self.v[k0:k0 + length], scale, seen,
                              self.offset[k0:k0 + length], self.most[k0:k0 + length])
            R.assert_within(got[r0:r0 + n], ref[0], R.bound(*ref, weight=(1 + R.H) ** 2 - 1), f"sequence {i}")
        assert self.G.apus_gcuda_kernel_error() == 0


# ------------------------------------------------------------ rows and codes

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("layout", ["packed", "interleaved", "head_major"])
def test_append_and_read(gcuda, dim, layout):
    """Codes, scales and every other byte of the cache; then the rows read back.  Ragged rows over page borders, an
    empty sequence, a sequence whose first rows stand before position 0, rows behind the last sequence."""
    heads, lens, rows = 3, [70, 0, 1, 200, 5, 129], [9, 0, 1, 137, 8, 2]
    c = Case(gcuda, dim, heads, lens, rows, seed=dim, behind=3)
    both = bf16(c.g, c.total, heads, 2, dim, std=1.0) * (0.2 + torch.rand(heads, 2, dim, generator=c.g)).to(torch.bfloat16)
    both = both.cuda()
    if layout == "packed":
        k, v = both[:, :, 0].contiguous(), both[:, :, 1].contiguous()
    elif layout == "interleaved":
        k, v = both[:, :, 0], both[:, :, 1]
    else:
        k, v = (both[:, :, i].transpose(0, 1).contiguous().transpose(0, 1) for i in (0, 1))
    before = c.pages.cpu()
    gcuda.kv4_append(c.cache, c.batch, k, v)
    torch.cuda.synchronize()
    want = [x.clone() for x in R.split(before, dim)]
    qk, qv = R.quantise(k.cpu()), R.quantise(v.cpu())
    back = torch.zeros(2, c.total, heads, dim)
    for i, (n, length) in enumerate(zip(rows, lens)):
        for t in range(n):
            pos, row = length - n + t, int(c.cu[i]) + t
            if pos < 0:
                continue
            page, off = int(c.table[i, pos // 64]), pos % 64
            want[0][page, :, off], want[1][page, :, off] = qk[0][row], qv[0][row]
            want[2][page, :, off], want[3][page, :, off] = qk[1][row], qv[1][row]
            back[0, row], back[1, row] = R.held(qk[0], qk[1])[row].float(), R.held(qv[0], qv[1])[row].float()
    for g, w in zip(R.split(c.pages.cpu(), dim), want):
        assert torch.equal(g.nan_to_num(-1.0) if g.is_floating_point() else g,
                           w.nan_to_num(-1.0) if w.is_floating_point() else w)
    ok, ov = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    gcuda.kv4_read(c.cache, c.batch, ok, ov)
    torch.cuda.synchronize()
    n = int(c.cu[-1])
    assert torch.equal(ok[:n].cpu(), back[0, :n].to(torch.bfloat16)) and torch.equal(ov[:n].cpu(), back[1, :n].to(torch.bfloat16))
    assert (ok[n:] == 7).all() and (ov[n:] == 7).all()
    assert gcuda.apus_gcuda_kernel_error() == 0


def test_append_special_values(gcuda):
    """Zeros, one large value among zeros, ties between two codes, subnormals, the largest BF16, NaN, infinities."""
    dim = 64
    rows = torch.zeros(12, 1, dim)
    rows[1, 0, 5] = -3.0
    rows[2, 0] = torch.arange(dim) % 15 * 0.5 - 3.5          # s = 0.5: every quotient a code
    rows[3, 0] = torch.arange(dim) % 14 * 0.5 - 3.25         # ties
    rows[3, 0, 31], rows[3, 0, 63] = 3.5, -3.5
    rows[4, 0] = 2.0 ** -133
    rows[5, 0] = torch.arange(dim) * 2.0 ** -133
    rows[6, 0] = torch.finfo(torch.bfloat16).max
    rows[6, 0, ::3] = 1.0
    rows[7, 0, 3] = float("nan")
    rows[8, 0, 40] = float("inf")
    rows[9, 0, 40] = float("-inf")
    rows[9, 0, 3] = 1.5
    rows[10, 0] = -0.0
    rows[11, 0] = torch.randn(dim, generator=gen(3)) * 1e-30
    x = rows.to(torch.bfloat16)
    c = Case(gcuda, dim, 1, [12], [12])
    gcuda.kv4_append(c.cache, c.batch, x.cuda(), x.flip(0).cuda())
    ok, ov = torch.empty_like(x, device="cuda"), torch.empty_like(x, device="cuda")
    gcuda.kv4_read(c.cache, c.batch, ok, ov)
    torch.cuda.synchronize()
    page = int(c.table[0, 0])
    kc, vc, ks, vs = R.split(c.pages.cpu(), dim)
    for codes, scales, src, back in ((kc, ks, x, ok), (vc, vs, x.flip(0), ov)):
        wc, ws = R.quantise(src)
        assert torch.equal(codes[page, 0, :12], wc[:, 0])
        assert torch.equal(scales[page, 0, :12].isnan(), ws[:, 0].isnan())
        assert torch.equal(scales[page, 0, :12].nan_to_num(), ws[:, 0].nan_to_num())
        want = R.held(wc, ws).to(torch.bfloat16)
        assert torch.equal(back.cpu().isnan(), want.isnan()) and torch.equal(back.cpu().nan_to_num(), want.nan_to_num())


# ----------------------------------------------------------------- attention

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,rows", [(2, 4, 1), (3, 1, 4), (1, 16, 1), (2, 3, 7), (1, 1, 1), (1, 8, 6)])
def test_attention(gcuda, dim, heads, group, rows):
    """Lengths around the borders of fragments, units and pages, one position, one row more than positions, an empty
    sequence; untouched places of the cache hold NaN scales."""
    lens = [rows, rows + 15, 63, 64, 65, 0, 300, rows - 1, 1030]
    ns = [rows] * 5 + [0, rows, rows, rows]
    c = Case(gcuda, dim, heads, lens, ns, seed=dim + rows, behind=2)
    c.fill_all()
    q = bf16(c.g, c.total, heads * group, dim, std=2.0).cuda()
    scale = dim ** -0.5
    got = c.attn(q, scale)
    torch.cuda.synchronize()
    n = int(c.cu[-1])
    assert (got[n:] == 7).all()
    c.check(q, got, scale)
    assert torch.equal(got, c.attn(q, scale))


@pytest.mark.parametrize("dim,heads,group,rows,longest", [(128, 1, 8, 1, 20000), (256, 2, 1, 4, 9001), (64, 1, 4, 2, 33333)])
def test_attention_long(gcuda, dim, heads, group, rows, longest):
    """Many chunks of one sequence, beside a short one; a steep softmax."""
    c = Case(gcuda, dim, heads, [longest, 40], [rows, rows], seed=5)
    c.fill_all()
    q = bf16(c.g, c.total, heads * group, dim, std=5.0).cuda()
    scale = dim ** -0.5
    assert gcuda.kv4_attn_workspace(c.cache, c.batch, heads * group) > 0
    c.check(q, c.attn(q, scale), scale)


@pytest.mark.parametrize("std_q,std_k,std_v", [(1e-20, 1.0, 1e-30), (1e15, 1e-15, 1e20), (1.0, 30.0, 1e-5)])
def test_attention_magnitudes(gcuda, std_q, std_k, std_v):
    """Any range of the types: queries and scales far from 1."""
    c = Case(gcuda, 128, 2, [200, 3], [2, 1], seed=6)
    c.fill_all(std_k, std_v)
    q = bf16(c.g, c.total, 4, 128, std=std_q).cuda()
    c.check(q, c.attn(q, 0.1), 0.1)


def test_attention_values_of_very_different_size(gcuda):
    """A position with values 1e12 times the others' that the softmax leaves almost out."""
    c = Case(gcuda, 64, 1, [130], [1], seed=8)
    k, v = bf16(c.g, 130, 1, 64), bf16(c.g, 130, 1, 64)
    v[17] *= 1e12
    k[17] = -4.0
    c.write_all(k, v)
    q = torch.full((1, 2, 64), 1.0, dtype=torch.bfloat16).cuda()
    c.check(q, c.attn(q, 0.125), 0.125)


@pytest.mark.parametrize("dim,pool", [(64, 4), (128, 6), (256, 4), (128, 1), (128, 128), (256, 3)])
def test_attention_selected(gcuda, dim, pool):
    """Pools kept at random, none kept (only the row's incomplete pool is seen, or nothing), all kept, a selection
    shorter than the sequence."""
    heads, group, rows, lens = 2, 2, 3, [5, 700, 64, 1283, 24 * pool if pool < 64 else 256]
    c = Case(gcuda, dim, heads, lens, [rows] * 5, seed=pool)
    c.fill_all()
    q = bf16(c.g, c.total, heads * group, dim, std=2.0).cuda()
    pools = max(lens) // pool - (2 if pool < 64 else 0)
    sel = (torch.rand(c.total, pools, generator=c.g) < 0.07).to(torch.uint8) * 3
    sel[0] = 0
    sel[3:6] = 0
    sel[6] = 1
    sel[12:] = 0
    got = c.attn(q, 0.09, sel.cuda(), pool)
    c.check(q, got, 0.09, sel, pool)
    if pool == 1:
        assert (got[0] == 0).all()           # no pool kept, no incomplete pool


def test_unseen_positions_have_no_influence(gcuda):
    """NaN and infinities at positions that only the later rows of a step see, at positions the selection leaves out,
    and in the rest of the last page."""
    dim, pool = 128, 4
    c = Case(gcuda, dim, 2, [150, 90], [4, 2], seed=11)
    k, v = bf16(c.g, 240, 2, dim), bf16(c.g, 240, 2, dim)
    sel = torch.ones(6, 40, dtype=torch.uint8)
    c.write_all(k, v)
    q = bf16(c.g, 6, 8, dim).cuda()
    plain = c.attn(q, 0.1)
    c.check(q, plain, 0.1)
    k2, v2 = k.clone(), v.clone()
    k2[149], v2[149] = float("nan"), float("inf")     # the last row's own position
    v2[148, 0, 7] = float("nan")
    c.write_all(k2, v2)
    got = c.attn(q, 0.1)
    assert torch.equal(got[:2], plain[:2]) and torch.equal(got[4:], plain[4:])
    assert got[2, :4].isnan()[:, :32].all() and got[3].isnan().all()
    assert torch.equal(got[2, 4:], plain[2, 4:])
    c.write_all(k, v)
    sel[:, 10] = 0
    want = c.attn(q, 0.1, sel.cuda(), pool)
    k2, v2 = k.clone(), v.clone()
    k2[40:44], v2[40:44] = float("inf"), float("nan")
    k2[190:194], v2[190:194] = float("nan"), float("nan")
    c.write_all(k2, v2)
    assert torch.equal(c.attn(q, 0.1, sel.cuda(), pool), want)


def test_seen_nan_is_seen(gcuda):
    c = Case(gcuda, 64, 1, [100], [2], seed=12)
    k, v = bf16(c.g, 100, 1, 64), bf16(c.g, 100, 1, 64)
    k[30, 0, 0] = float("nan")
    c.write_all(k, v)
    q = bf16(c.g, 2, 1, 64).cuda()
    assert c.attn(q, 0.1).isnan().all()
    q[0] = float("nan")
    c.write_all(torch.ones_like(k), v)
    got = c.attn(q, 0.1)
    assert got[0].isnan().all() and got[1].isfinite().all()


def test_strides(gcuda):
    """Queries and outputs with heads outermost, or rows farther apart than their heads need."""
    c = Case(gcuda, 128, 2, [77, 200], [2, 3], seed=13)
    c.fill_all()
    q = bf16(c.g, 5, 6, 128).cuda()
    want = c.attn(q, 0.1)
    c.check(q, want, 0.1)
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(5, 9, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:7] = q
    for x in (major, wide[:, 1:7]):
        assert torch.equal(c.attn(x, 0.1), want)
    out = torch.full((6, 5, 128), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(c.attn(q, 0.1, out=out), want)


# -------------------------------------------------- what the host cannot see

def test_out_of_bounds_entries(gcuda):
    """Page ids, lengths and row ranges out of bounds are not followed; the other sequences are as before."""
    dim, heads = 128, 2
    lens, rows = [200, 130, 70], [2, 2, 2]
    c = Case(gcuda, dim, heads, lens, rows, seed=14)
    c.fill_all()
    q = bf16(c.g, 6, 4, dim).cuda()
    want = c.attn(q, 0.1)
    c.check(q, want, 0.1)
    table = c.table.clone()
    for bad in (-1, c.pages.shape[0], 2 ** 31 - 1, -2 ** 31):
        c.table = table.clone()
        c.table[1, 1] = bad
        b = c.make_batch(c.cu, lens)
        got = c.attn(q, 0.1, batch=b)
        assert gcuda.apus_gcuda_kernel_error() == 41 and gcuda.apus_gcuda_kernel_error() == 0
        assert torch.equal(got[:2], want[:2]) and torch.equal(got[4:], want[4:])
        # its other positions are seen
        k0 = c.starts[1]
        seen = torch.ones(2, 130, dtype=torch.bool)
        seen[:, 64:128] = False
        seen[0, 129] = False
        ref = R.attention(q[2:4].double().cpu(), c.k[k0:k0 + 130], c.v[k0:k0 + 130], 0.1, seen, c.offset[k0:k0 + 130],
                          c.most[k0:k0 + 130])
        R.assert_within(got[2:4], ref[0], R.bound(*ref, weight=(1 + R.H) ** 2 - 1))
        ok = torch.full((6, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        before = c.pages.clone()
        c.table[1, 1], c.table[1, 2] = table[1, 1], bad
        b = c.make_batch(c.cu, lens)
        gcuda.kv4_read(c.cache, b, ok, torch.empty_like(ok))
        assert gcuda.apus_gcuda_kernel_error() == 41
        assert (ok[2:4] == 0).all() and (ok[:2] != 7).any() and (ok[4:] != 7).any()
        gcuda.kv4_append(c.cache, b, ok, ok)
        assert gcuda.apus_gcuda_kernel_error() == 41
        c.pages.copy_(before)
    c.table = table
    for cu, ln, empty in (([0, 2, 4, 6], [200, -5, 70], 1), ([0, 2, 4, 6], [200, 10 ** 9, 70], 1),
                          ([0, 2, 9, 6], lens, None), ([0, 2, 1, 6], lens, None), ([-3, 2, 4, 6], lens, None)):
        b = c.make_batch(cu, ln, max_len=200)
        got = c.attn(q, 0.1, batch=b)
        assert gcuda.apus_gcuda_kernel_error() == 42
        if empty is not None:
            assert (got[2:4] == 0).all() and torch.equal(got[:2], want[:2]) and torch.equal(got[4:], want[4:])


def test_more_rows_than_the_bound(gcuda):
    c = Case(gcuda, 64, 1, [90], [5], seed=15)
    c.fill_all()
    q = bf16(c.g, 5, 1, 64).cuda()
    got = c.attn(q, 0.1, batch=c.make_batch(c.cu, c.lens, max_rows=4))
    torch.cuda.synchronize()
    assert (got == 7).all() and gcuda.apus_gcuda_kernel_error() == 42


def test_large_cache(gcuda):
    """Pages whose bytes lie beyond 32 bits."""
    dim, heads = 256, 64
    per = heads * 72 * dim
    n = (1 << 32) // per + 40
    c = Case(gcuda, dim, 1, [130], [2], seed=16)
    pages = torch.empty(n, heads, 72 * dim, dtype=torch.uint8, device="cuda")
    cache = gcuda.Kv4Cache(pages)
    table = torch.tensor([[n - 1, n - 30, n - 7]], dtype=torch.int32).cuda()
    k, v = bf16(c.g, 130, heads, dim), bf16(c.g, 130, heads, dim)
    cu, ln = torch.tensor([0, 130], dtype=torch.int32).cuda(), torch.tensor([130], dtype=torch.int32).cuda()
    gcuda.kv4_append(cache, gcuda.Kv4Batch(cu, ln, table, max_rows=130, max_len=130), k.cuda(), v.cuda())
    cu2 = torch.tensor([0, 2], dtype=torch.int32).cuda()
    b = gcuda.Kv4Batch(cu2, ln, table, max_rows=2, max_len=130)
    q = bf16(c.g, 2, heads, dim).cuda()
    out = torch.empty_like(q)
    work = torch.empty(max(1, gcuda.kv4_attn_workspace(cache, b, heads)), dtype=torch.uint8, device="cuda")
    gcuda.kv4_attn(cache, b, q, out, 0.06, work)
    torch.cuda.synchronize()
    (hk, hv), (ks, vs) = (R.held(*R.quantise(x)) for x in (k, v)), (R.quantise(x)[1] for x in (k, v))
    seen = torch.arange(130)[None] < torch.tensor([[129], [130]])
    ref = R.attention(q.double().cpu(), hk, hv, 0.06, seen, 16 * ks.repeat_interleave(32, -1), vs.amax(-1))
    R.assert_within(out, ref[0], R.bound(*ref, weight=(1 + R.H) ** 2 - 1))


# ------------------------------------------------------------ graphs, streams

def test_graph_replay(gcuda):
    """Append and attention captured once, replayed as the sequences grow: lengths, rows and pages are read on the
    device."""
    dim, heads, group = 128, 2, 4
    lens = [60, 500]
    c = Case(gcuda, dim, heads, [n + 4 for n in lens], [1, 1], seed=17)
    c.fill_all()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    ln, table = torch.tensor(lens, dtype=torch.int32).cuda(), c.table.cuda()
    b = gcuda.Kv4Batch(cu, ln, table, max_rows=1, max_len=504)
    q = torch.zeros(2, heads * group, dim, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(2, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out = torch.zeros_like(q)
    work = torch.empty(max(1, gcuda.kv4_attn_workspace(c.cache, b, heads * group)), dtype=torch.uint8, device="cuda")
    gcuda.kv4_append(c.cache, b, k, v)
    gcuda.kv4_attn(c.cache, b, q, out, 0.1, work)       # the first call on a device sets the kernels' limits
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gcuda.kv4_append(c.cache, b, k, v)
        gcuda.kv4_attn(c.cache, b, q, out, 0.1, work)
    c.rows, c.cu = [1, 1], torch.tensor([0, 1, 2])
    ks = c.offset / 16
    for i in range(2):                                  # the first call's rows: zeros
        at = c.starts[i] + lens[i] - 1
        c.k[at], c.v[at], ks[at], c.most[at] = 0.0, 0.0, 0.0, 0.0
    for step in range(4):
        lens = [n + 1 for n in lens]
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        nk, nv, nq = bf16(c.g, 2, heads, dim), bf16(c.g, 2, heads, dim), bf16(c.g, 2, heads * group, dim)
        k.copy_(nk), v.copy_(nv), q.copy_(nq)
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            at = c.starts[i] + lens[i] - 1
            (kc, kscale), (vc, vscale) = R.quantise(nk[i]), R.quantise(nv[i])
            c.k[at], c.v[at], ks[at] = R.held(kc, kscale), R.held(vc, vscale), kscale.repeat_interleave(32, -1)
            c.most[at] = vscale.amax(-1)
            s0 = c.starts[i]
            ref = R.attention(nq[i:i + 1].double(), c.k[s0:at + 1], c.v[s0:at + 1], 0.1,
                              torch.ones(1, lens[i], dtype=torch.bool), 16 * ks[s0:at + 1], c.most[s0:at + 1])
            R.assert_within(out[i:i + 1], ref[0], R.bound(*ref, weight=(1 + R.H) ** 2 - 1))


def test_two_streams(gcuda):
    """Calls on two streams at once, each with its own workspace."""
    c = Case(gcuda, 128, 2, [5000, 300], [1, 1], seed=18)
    c.fill_all()
    qs = [bf16(c.g, 2, 8, 128).cuda() for _ in range(2)]
    want = [c.attn(q, 0.1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    n = gcuda.kv4_attn_workspace(c.cache, c.batch, 8)
    works = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(8)] for q in qs]
    torch.cuda.synchronize()
    for i in range(8):
        for s in range(2):
            gcuda.kv4_attn(c.cache, c.batch, qs[s], outs[s][i], 0.1, works[s], stream=streams[s])
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(o, want[s]) for o in outs[s])


def test_selected_with_a_page_out_of_range(gcuda):
    """Selected positions of a page whose id is out of range count as unseen."""
    c = Case(gcuda, 128, 1, [300], [2], seed=19)
    c.fill_all()
    q = bf16(c.g, 2, 2, 128).cuda()
    sel = (torch.rand(2, 75, generator=c.g) < 0.3).to(torch.uint8)
    c.table[0, 2] = c.pages.shape[0]
    got = c.attn(q, 0.1, sel.cuda(), 4, batch=c.make_batch(c.cu, c.lens))
    assert gcuda.apus_gcuda_kernel_error() == 41
    sel[:, 32:48] = 0
    c.check(q, got, 0.1, sel, 4)


@pytest.mark.parametrize("nseq,longest", [(300, 200), (150, 2000)])
def test_many_sequences(gcuda, nseq, longest):
    """More sequences than threads of a block, of very different lengths, some empty, some without rows."""
    g = gen(nseq)
    lens = [int(x) for x in (torch.rand(nseq, generator=g) ** 4 * longest).tolist()]
    rows = [int(x) for x in torch.randint(0, 4, (nseq,), generator=g).tolist()]
    lens[7], rows[8], lens[nseq - 1] = longest, 0, longest
    c = Case(gcuda, 64, 1, lens, rows, seed=20, max_rows=3)
    c.fill_all()
    q = bf16(c.g, c.total, 2, 64, std=2.0).cuda()
    c.check(q, c.attn(q, 0.125), 0.125)


def test_bound_far_above_the_rows(gcuda):
    """max_rows far above the rows that there are, and more columns than the joining kernel has blocks."""
    c = Case(gcuda, 128, 2, [2500, 700, 4000], [3, 40, 1], seed=21, max_rows=5000)
    c.fill_all()
    q = bf16(c.g, c.total, 8, 128, std=2.0).cuda()
    c.check(q, c.attn(q, 0.09), 0.09)


@pytest.mark.parametrize("dim,pool,kept", [(64, 4, 0.3), (128, 100, 0.9), (64, 1, 0.02)])
def test_selected_long(gcuda, dim, pool, kept):
    """More kept positions than one list holds, and a longer way between them than its offsets reach."""
    c = Case(gcuda, dim, 1, [150001], [2], seed=pool)
    c.fill_all()
    q = bf16(c.g, 2, 2, dim, std=2.0).cuda()
    sel = (torch.rand(2, 150001 // pool + 1, generator=c.g) < kept).to(torch.uint8)
    sel[:, 20000 // pool:100000 // pool] = 0
    sel[1, 90000 // pool] = 1
    c.check(q, c.attn(q, 0.1, sel.cuda(), pool), 0.1, sel, pool)


@pytest.mark.parametrize("length", [100, 6000])
def test_seen_nan_with_no_weight(gcuda, length):
    """A value that is NaN reaches the rows that see it however small its weight, in a run of its own too."""
    c = Case(gcuda, 64, 1, [length], [1], seed=22)
    k, v = bf16(c.g, length, 1, 64), bf16(c.g, length, 1, 64)
    q = torch.ones(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    k[10], v[10, 0, 3] = -1000.0, float("nan")
    c.write_all(k, v)
    got = c.attn(q, 1.0)
    assert got[0, 0, :32].isnan().all() and got[0, 0, 32:].isfinite().all()

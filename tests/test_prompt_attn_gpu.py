"""Causal prompt attention over packed sequences (apus_gcuda_prompt_attn_dev)
on the B200, against a 64-bit reference (attn_ref.py): held elementwise to the
bound that one BF16 rounding of a weight and fp32 sums allow."""
import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu


def bf16(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def starts(counts):
    return torch.tensor([0] + counts).cumsum(0).to(torch.int32)


def check(q, k, v, out, rows, keys, scale):
    q0 = k0 = 0
    for i, (n, m) in enumerate(zip(rows, keys)):
        if n:
            seen = torch.arange(m)[None] <= m - n + torch.arange(n)[:, None]
            ref = R.attention(q[q0:q0 + n].double().cuda(), k[k0:k0 + m].double().cuda(), v[k0:k0 + m].double().cuda(),
                              scale, seen.cuda())
            R.assert_within(out[q0:q0 + n], ref[0], R.bound(*ref, weight=R.U), f"sequence {i}")
        q0, k0 = q0 + n, k0 + m


def run(G, q, k, v, rows, keys, scale, out=None, max_rows=None):
    out = torch.full_like(q, 7.0) if out is None else out
    dev = starts(rows).cuda(), starts(keys).cuda()
    G.prompt_attn(G.PromptBatch(*dev, max_rows=max_rows or max(rows)), q, k, v, out, scale)
    torch.cuda.synchronize()
    assert G.apus_gcuda_kernel_error() == 0
    return out


SHAPES = [
    # rows, keys of each sequence
    ([1], [1]), ([5, 1, 64], [5, 1, 64]), ([127, 128, 129], [127, 128, 129]), ([300, 0, 17, 256], [300, 0, 17, 256]),
    ([700], [700]), ([1, 130, 40], [513, 400, 41]), ([128], [385]), ([9, 0, 3], [4, 30, 0]),
]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group", [(2, 4), (3, 1), (1, 7)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_prompt(gcuda, dim, heads, group, shape):
    """Lengths around the tiles' borders, single rows, empty sequences, prefixes, more queries than keys (the first
    see nothing and give zeros), rows behind the last sequence."""
    rows, keys = SHAPES[shape]
    g = torch.Generator().manual_seed(shape * 31 + dim + heads)
    q = bf16(g, sum(rows) + 2, heads * group, dim, std=2.0).cuda()
    k, v = (bf16(g, sum(keys) + 1, heads, dim).cuda() for _ in range(2))
    out = run(gcuda, q, k, v, rows, keys, dim ** -0.5)
    check(q, k, v, out, rows, keys, dim ** -0.5)
    assert (out[sum(rows):] == 7).all()
    if shape == 7:
        assert (out[:5] == 0).all() and (out[9:12] == 0).all()
    assert torch.equal(out, run(gcuda, q, k, v, rows, keys, dim ** -0.5))


@pytest.mark.parametrize("dim,rows,keys,std", [(128, [2050], [2050], 4.0), (64, [1500, 1000], [1500, 3000], 1.0),
                                               (256, [1100], [2300], 3.0), (128, [33] * 40, [33] * 40, 1.0)])
def test_prompt_long(gcuda, dim, rows, keys, std):
    """Many key tiles, a steep softmax (the running maximum rises again and again), many short sequences."""
    g = torch.Generator().manual_seed(dim)
    q = bf16(g, sum(rows), 4, dim, std=std).cuda()
    k, v = (bf16(g, sum(keys), 2, dim).cuda() for _ in range(2))
    ramp = torch.linspace(0.2, 3.0, sum(keys))[:, None, None]
    k = (k.cpu().float() * ramp).to(torch.bfloat16).cuda()
    check(q, k, v, run(gcuda, q, k, v, rows, keys, dim ** -0.5), rows, keys, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_strides(gcuda, dim):
    """Keys and values interleaved in one tensor (as kv_b leaves them), heads outermost, rows farther apart."""
    g = torch.Generator().manual_seed(7)
    rows = [150, 61]
    q = bf16(g, 211, 4, dim).cuda()
    kv = bf16(g, 211, 2, 2, dim).cuda()
    k, v = kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous()
    want = run(gcuda, q, k, v, rows, rows, 0.1)
    check(q, k, v, want, rows, rows, 0.1)
    assert torch.equal(run(gcuda, q, kv[:, :, 0], kv[:, :, 1], rows, rows, 0.1), want)

    def major(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    out = major(torch.full_like(q, 7.0))
    assert torch.equal(run(gcuda, major(q), major(k), major(v), rows, rows, 0.1, out=out), want)
    wide = torch.zeros(211, 7, dim, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:6] = q
    assert torch.equal(run(gcuda, wide[:, 2:6], k, v, rows, rows, 0.1, out=torch.empty_like(q)), want)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_unseen_keys_have_no_influence(gcuda, dim):
    """NaN and infinities at later keys of the same sequence, in neighbouring sequences and behind the last."""
    g = torch.Generator().manual_seed(9)
    rows, keys = [200, 140, 90], [200, 180, 90]
    q = bf16(g, 430, 4, dim).cuda()
    k, v = (bf16(g, 480, 2, dim).cuda() for _ in range(2))
    want = run(gcuda, q, k, v, rows, keys, 0.1)
    check(q, k, v, want, rows, keys, 0.1)
    k2, v2 = k.clone(), v.clone()
    k2[470:], v2[470:] = float("nan"), float("inf")
    assert torch.equal(run(gcuda, q, k2, v2, rows, keys, 0.1), want)
    v2[160, 1, 3], k2[199, 0] = float("nan"), float("inf")     # seen by rows 160.., 199 of the first sequence
    v2[395, 0, 5] = float("-inf")                              # by rows 15.. of the last
    got = run(gcuda, q, k2, v2, rows, keys, 0.1)
    for a, b in ((0, 160), (200, 355)):
        assert torch.equal(got[a:b], want[a:b])
    assert torch.equal(got[160:199, :2], want[160:199, :2])
    assert got[160:200, 2:, 3].isnan().all()
    assert got[199, :2].isnan().all()
    assert (got[355:430, :2, 5] == float("-inf")).all()
    assert torch.equal(got[355:430, 2:], want[355:430, 2:])
    qn = q.clone()
    qn[100, 1] = float("nan")
    got = run(gcuda, qn, k, v, rows, keys, 0.1)
    assert got[100, 1].isnan().all()
    got[100, 1] = want[100, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dim,heads,group", [(64, 4, 8), (128, 4, 8), (256, 16, 2)])
def test_many_items(gcuda, dim, heads, group):
    """Far more blocks of rows than SMs, so that a CTA takes one after the other: over a hundred sequences of 0 to 300
    rows over 0 to 500 keys, and the same with NaN and infinities in every third sequence's last value, which its last
    row alone sees."""
    g = torch.Generator().manual_seed(dim + 1)
    rows = [int(x) for x in torch.randint(0, 301, (110,), generator=g)]
    keys = [n + int(x) for n, x in zip(rows, torch.randint(-20, 200, (110,), generator=g))]
    keys = [max(m, 0) for m in keys]
    rows[40:44], keys[40:44] = [0, 0, 5, 256], [0, 9, 0, 256]
    q = bf16(g, sum(rows) + 3, heads * group, dim).cuda()
    k, v = (bf16(g, sum(keys) + 3, heads, dim).cuda() for _ in range(2))
    out = run(gcuda, q, k, v, rows, keys, dim ** -0.5)
    check(q, k, v, out, rows, keys, dim ** -0.5)
    assert (out[sum(rows):] == 7).all()
    v2, want = v.clone(), out.clone()
    q0, k0 = starts(rows).tolist(), starts(keys).tolist()
    for i in range(0, 110, 3):
        if rows[i] and keys[i]:
            c = i // 3 % 3
            v2[k0[i + 1] - 1, i % heads, 7 * c] = (float("nan"), float("inf"), float("-inf"))[c]
            want[q0[i + 1] - 1, i % heads * group:(i % heads + 1) * group, 7 * c] = (float("nan"), float("inf"), float("-inf"))[c]
    for _ in range(2):
        got = run(gcuda, q, k, v2, rows, keys, dim ** -0.5)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def test_heads_in_parts(gcuda):
    """Sequences whose keys and values do not stay in L2 together: their heads are taken in parts, the last one
    smaller; one before and one behind whose heads are taken together."""
    g = torch.Generator().manual_seed(14)
    rows, keys = [40, 300, 129, 70], [50, 6000, 4100, 70]
    q = bf16(g, sum(rows), 26, 256).cuda()
    k, v = (bf16(g, sum(keys), 13, 256).cuda() for _ in range(2))
    check(q, k, v, run(gcuda, q, k, v, rows, keys, 0.07), rows, keys, 0.07)


@pytest.mark.parametrize("dim", [64, 256])
def test_many_sequences(gcuda, dim):
    """More sequences than are looked up at a time, most of a few rows, some empty; a range out of bounds behind the
    last row is reported."""
    g = torch.Generator().manual_seed(dim + 2)
    rows = [int(x) for x in torch.randint(0, 4, (700,), generator=g)]
    rows[130], rows[500] = 300, 513
    rows[600:] = [0] * 100
    q = bf16(g, sum(rows) + 1, 2, dim).cuda()
    k, v = (bf16(g, sum(rows), 1, dim).cuda() for _ in range(2))
    out = run(gcuda, q, k, v, rows, rows, 0.1)
    check(q, k, v, out, rows, rows, 0.1)
    assert (out[sum(rows):] == 7).all()
    cu, bad = starts(rows).cuda(), starts(rows).cuda()
    bad[700] = 1 << 30
    again = torch.full_like(q, 7.0)
    gcuda.prompt_attn(gcuda.PromptBatch(bad, cu, max_rows=513), q, k, v, again, 0.1)
    torch.cuda.synchronize()
    assert gcuda.apus_gcuda_kernel_error() == 42
    assert torch.equal(again, out)


def test_ranges_out_of_bounds(gcuda):
    g = torch.Generator().manual_seed(10)
    q, k, v = (bf16(g, 100, 2, 64).cuda() for _ in range(3))
    want = run(gcuda, q, k, v, [40, 30, 30], [40, 30, 30], 0.1)
    for cu_q, cu_k, fine in (([0, 40, 70, 101], [0, 40, 70, 100], 70), ([0, 40, 70, 100], [0, 40, 70, 1000], 70),
                             ([0, 40, 70, 60], [0, 40, 70, 100], 70), ([0, 40, 70, 100], [-1, 40, 70, 100], 0)):
        out = torch.full_like(q, 7.0)
        dev = [torch.tensor(x, dtype=torch.int32).cuda() for x in (cu_q, cu_k)]
        gcuda.prompt_attn(gcuda.PromptBatch(*dev, max_rows=40), q, k, v, out, 0.1)
        assert gcuda.apus_gcuda_kernel_error() == 42
        if fine:
            assert torch.equal(out[:fine], want[:fine])
        else:
            assert (out[:40] == 0).all() and torch.equal(out[40:], want[40:])


def test_graph_and_streams(gcuda):
    """Captured once and replayed with other lengths; two streams at once."""
    g = torch.Generator().manual_seed(11)
    q, k, v = (bf16(g, 600, 4, 128).cuda() for _ in range(3))
    cu = starts([200, 400]).cuda()
    b = gcuda.PromptBatch(cu, cu, max_rows=400)
    out = torch.zeros_like(q)
    gcuda.prompt_attn(b, q, k, v, out, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gcuda.prompt_attn(b, q, k, v, out, 0.1)
    for rows in ([300, 300], [399, 1], [250, 350]):
        cu.copy_(starts(rows))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(q, k, v, out, rows, rows, 0.1)
        assert (out[sum(rows):] == 7).all()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.empty_like(q) for _ in range(8)]
    torch.cuda.synchronize()
    for i in range(8):
        gcuda.prompt_attn(b, q, k, v, outs[i], 0.1, stream=streams[i & 1])
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)


# ------------------------------------------------------- the operators together

@pytest.mark.parametrize("dim,heads,group", [(128, 2, 4), (256, 3, 1), (64, 1, 8)])
def test_prompt_cache_decode(gcuda, dim, heads, group):
    """A serving run: two prompts attend to themselves and go into the cache; a second chunk attends to the prefix
    read back from the cache and its own rows; then verify steps of three rows over the cache."""
    G, g = gcuda, torch.Generator().manual_seed(dim)
    first, second, scale = [90, 33], [50, 128], dim ** -0.5
    pages = G.kv4_pages(12, heads, dim)
    cache = G.Kv4Cache(pages)
    table = torch.randperm(12, generator=g).to(torch.int32).reshape(2, 6).cuda()
    held_k, held_v, step = ([torch.zeros(0, heads, dim, dtype=torch.float64) for _ in range(2)] for _ in range(3))
    most = [torch.zeros(0, heads, dtype=torch.float64) for _ in range(2)]      # each position's largest value scale

    def remember(k, v, counts):
        at = 0
        for i, n in enumerate(counts):
            (kc, ks), (vc, vs) = R.quantise(k[at:at + n].cpu()), R.quantise(v[at:at + n].cpu())
            held_k[i], held_v[i] = torch.cat((held_k[i], R.held(kc, ks))), torch.cat((held_v[i], R.held(vc, vs)))
            step[i] = torch.cat((step[i], 16 * ks.repeat_interleave(32, -1)))
            most[i] = torch.cat((most[i], vs.amax(-1)))
            at += n

    def fresh(n):
        return bf16(g, n, heads * group, dim, std=2.0).cuda(), bf16(g, n, heads, dim).cuda(), bf16(g, n, heads, dim).cuda()

    def batch(counts, lens):
        return G.Kv4Batch(starts(counts).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), table, max_rows=max(counts),
                          max_len=max(lens))

    q, k, v = fresh(sum(first))
    check(q, k, v, run(G, q, k, v, first, first, scale), first, first, scale)
    G.kv4_append(cache, batch(first, first), k, v)
    remember(k, v, first)
    # the second chunk: prefix from the cache (whole sequences read), then its own BF16 rows
    pk, pv = (torch.empty(sum(first), heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    G.kv4_read(cache, batch(first, first), pk, pv)
    q, k, v = fresh(sum(second))
    both = [a + b for a, b in zip(first, second)]
    ck, cv = (torch.cat((p[:first[0]], x[:second[0]], p[first[0]:], x[second[0]:])) for p, x in ((pk, k), (pv, v)))
    check(q, ck, cv, run(G, q, ck, cv, second, both, scale), second, both, scale)
    assert torch.equal(pk.cpu(), torch.cat(held_k).to(torch.bfloat16)) and torch.equal(pv.cpu(), torch.cat(held_v).to(torch.bfloat16))
    G.kv4_append(cache, batch(second, both), k, v)
    remember(k, v, second)
    lens, out = both, None
    for _ in range(3):
        lens = [n + 3 for n in lens]
        q, k, v = fresh(6)
        b = batch([3, 3], lens)
        G.kv4_append(cache, b, k, v)
        remember(k, v, [3, 3])
        out = torch.empty_like(q)
        n = G.kv4_attn_workspace(cache, b, heads * group)
        work = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        G.kv4_attn(cache, b, q, out, scale, work)
        torch.cuda.synchronize()
        for i in range(2):
            seen = torch.arange(lens[i])[None] <= lens[i] - 3 + torch.arange(3)[:, None]
            ref = R.attention(q[3 * i:3 * i + 3].double().cpu(), held_k[i], held_v[i], scale, seen, step[i], most[i])
            R.assert_within(out[3 * i:3 * i + 3], ref[0], R.bound(*ref, weight=(1 + R.H) ** 2 - 1))
    assert G.apus_gcuda_kernel_error() == 0

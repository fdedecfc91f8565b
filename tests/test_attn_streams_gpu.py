"""The Python calls of the operators of include/apus_attn_gcuda.h on a stream that the caller gives: tensors that are
dropped before the stream gets to them stay what they are until it is through."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def bf16(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def inputs(G, seed):
    """Everything that the calls read, made anew from the seed."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads, dim, n = 2, 128, 1000
    d = dict(pages=G.kv4_pages(16, heads, dim), table=torch.randperm(16, generator=g, device="cuda").to(torch.int32)[None],
             cu=ints([0, n]), last=ints([0, 2]), lens=ints([n]), k=bf16(g, n, heads, dim), v=bf16(g, n, heads, dim),
             q=bf16(g, 2, 8, dim), pq=bf16(g, n, 4, dim), sel=(torch.rand(2, 250, generator=g, device="cuda") < 0.5).to(torch.uint8))
    d["work"] = torch.empty(G.kv4_attn_workspace(G.Kv4Cache(d["pages"]), G.Kv4Batch(d["last"], d["lens"], d["table"], 2, n), 8),
                            dtype=torch.uint8, device="cuda")
    return d


def calls(G, d, outs, stream):
    n = d["k"].shape[0]
    cache = G.Kv4Cache(d["pages"])
    whole = G.Kv4Batch(d["cu"], d["lens"], d["table"], n, n)
    last = G.Kv4Batch(d["last"], d["lens"], d["table"], 2, n)
    G.kv4_append(cache, whole, d["k"], d["v"], stream=stream)
    G.kv4_read(cache, whole, outs[0], outs[1], stream=stream)
    G.kv4_attn(cache, last, d["q"], outs[2], 0.1, d["work"], stream=stream)
    G.kv4_attn(cache, last, d["q"], outs[3], 0.1, d["work"], sel=d["sel"], pool=4, stream=stream)
    G.prompt_attn(G.PromptBatch(d["cu"], d["cu"], n), d["pq"], d["k"], d["v"], outs[4], 0.1, stream=stream)


def test_tensors_dropped_early(gcuda):
    G = gcuda
    d = inputs(G, 1)
    make = lambda: [torch.zeros_like(d[x]) for x in ("k", "v", "q", "q", "pq")]  # noqa: E731
    want, outs = make(), make()
    calls(G, d, want, None)
    torch.cuda.synchronize()
    d = inputs(G, 1)
    used = [(t.shape, t.dtype, t.data_ptr(), t.data_ptr() + t.nbytes) for t in d.values()]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)              # a fifth of a second and more
    calls(G, d, outs, side)
    d.clear()
    assert not side.query()                         # it has not got to them yet (an allocation may wait for it)
    # the same sizes again: what was dropped is not handed out while the stream waits.  (The addresses tell; that the
    # values are overwritten too depends on whether the device runs both streams' kernels at once.  Zeros: as row
    # ranges, lengths and page ids they are in bounds.)
    again = [torch.zeros(*shape, dtype=dtype, device="cuda") for shape, dtype, _, _ in used for _ in range(4)]
    if not side.query():
        for t in again:
            assert not any(lo < t.data_ptr() + t.nbytes and t.data_ptr() < hi for _, _, lo, hi in used)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert G.apus_gcuda_kernel_error() == 0

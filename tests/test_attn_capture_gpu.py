"""The operators of include/apus_attn_gcuda.h captured into a CUDA graph by a process's first calls, and called after
another entry point of the library has failed."""
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from test_kv4_gpu import Case, bf16

pytestmark = pytest.mark.gpu

CHILD = """
import os, sys
sys.path[:0] = [os.path.join(r"%s", "apus-glm5.3-flash_b200")]
import torch
import apus_gcuda as G

g = torch.Generator(device="cuda").manual_seed(1)
i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
for dim in (64, 128, 256):
    t = lambda n, h: torch.randn(n, h, dim, generator=g, device="cuda").to(torch.bfloat16)
    n, heads = 700, 2
    cache = G.Kv4Cache(G.kv4_pages(11, heads, dim))
    table = torch.arange(11, dtype=torch.int32, device="cuda")[None]
    whole, last = G.Kv4Batch(i([0, n]), i([n]), table, n, n), G.Kv4Batch(i([0, 3]), i([n]), table, 3, n)
    k, v, q, pq = t(n, heads), t(n, heads), t(3, 8), t(n, 4)
    sel = torch.ones(3, 175, dtype=torch.uint8, device="cuda")
    plan = G.PromptBatch(whole.tensors[0], whole.tensors[0], n)
    work = torch.empty(G.kv4_attn_workspace(cache, last, 8), dtype=torch.uint8, device="cuda")
    outs = [torch.empty_like(x) for x in (k, v, q, q, pq)]

    def calls():
        G.kv4_append(cache, whole, k, v)
        G.kv4_read(cache, whole, outs[0], outs[1])
        G.kv4_attn(cache, last, q, outs[2], 0.1, work)
        G.kv4_attn(cache, last, q, outs[3], 0.1, work, sel=sel, pool=4)
        G.prompt_attn(plan, pq, k, v, outs[4], 0.1)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in outs]
    [x.zero_() for x in outs]
    calls()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, outs)) and outs[4].any()
assert G.apus_gcuda_kernel_error() == 0
print("same")
"""


def test_first_calls_captured(gcuda):
    r = subprocess.run([sys.executable, "-c", CHILD % ROOT], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=""))
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout + r.stderr[-2000:]


def test_after_a_failed_call(gcuda):
    """A region of 2^50 bytes is refused; the calls after it succeed and say so."""
    c = Case(gcuda, 64, 1, [70], [2], seed=1)
    c.fill_all()
    q, k = bf16(c.g, 2, 2, 64).cuda(), bf16(c.g, 2, 1, 64).cuda()
    host = torch.zeros(64)

    def fail():
        assert gcuda.apus_gcuda_register_region(host.data_ptr(), 1 << 50) != 0

    fail()
    gcuda.kv4_append(c.cache, c.batch, k, k)
    fail()
    gcuda.kv4_read(c.cache, c.batch, k, k.clone())
    fail()
    c.attn(q, 0.1)
    fail()
    b = gcuda.PromptBatch(c.dev[0], c.dev[0], 2)
    gcuda.prompt_attn(b, q, k, k, torch.empty_like(q), 0.1)
    torch.cuda.synchronize()

"""The operators of include/apus_attn_gcuda.h called from several host threads at once, the process's first calls of
each kernel among them."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CHILD = """
import os, sys, threading
sys.path[:0] = [os.path.join(r"%s", d) for d in ("apus-glm5.3-flash_b200", "tests")]
import torch
import apus_gcuda as G

THREADS, CALLS = 6, 6
shapes = [(64, 2, 4), (128, 2, 2), (256, 1, 2)]


def make(dim, heads, group, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def t(n, h):
        return torch.randn(n, h, dim, generator=g, device="cuda").to(torch.bfloat16)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    rows, lens = [300, 40], [1300, 40]
    cache = G.Kv4Cache(G.kv4_pages(32, heads, dim))
    table = torch.randperm(32, generator=g, device="cuda").to(torch.int32).reshape(1, 32)
    table = torch.cat((table[:, :24], table[:, 24:].repeat(1, 3)))
    whole = G.Kv4Batch(i([0, 1300, 1340]), i(lens), table, 1300, 1300)
    last = G.Kv4Batch(i([0, 2, 3]), i(lens), table, 2, 1300)
    return dict(G=G, cache=cache, whole=whole, last=last, k=t(1340, heads), v=t(1340, heads), q=t(3, heads * group),
                pq=t(340, heads * group), plan=G.PromptBatch(i([0, 300, 340]), i([0, 1300, 1340]), 300))


def run(s):
    G.kv4_append(s["cache"], s["whole"], s["k"], s["v"])
    n = G.kv4_attn_workspace(s["cache"], s["last"], s["q"].shape[1])
    work = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    a, p, rk, rv = (torch.empty_like(x) for x in (s["q"], s["pq"], s["k"], s["v"]))
    G.kv4_attn(s["cache"], s["last"], s["q"], a, 0.1, work)
    G.kv4_read(s["cache"], s["whole"], rk, rv)
    G.prompt_attn(s["plan"], s["pq"], s["k"], s["v"], p, 0.1)
    try:                                    # a refusal in this thread is not seen by the others
        G.prompt_attn(s["plan"], s["pq"], s["k"], s["v"], p, -1.0 - s["id"])
        raise SystemExit("not refused")
    except G.GcudaError as e:
        assert "%%g" %% (-1.0 - s["id"]) in str(e), e
    return [a, p, rk, rv]


torch.cuda.init()
states = [make(*shapes[i %% 3], i) for i in range(THREADS)]
for i, s in enumerate(states):
    s["id"] = i
torch.cuda.synchronize()
out, errors = [[] for _ in states], []
gate = threading.Barrier(THREADS)


def work(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            gate.wait()
            for _ in range(CALLS):
                out[i].append(run(states[i]))
    except BaseException as e:
        errors.append(repr(e))


threads = [threading.Thread(target=work, args=(i,)) for i in range(THREADS)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert not errors, errors
assert G.apus_gcuda_kernel_error() == 0
for i, s in enumerate(states):
    want = run(s)
    torch.cuda.synchronize()
    for got in out[i]:
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
print("same")
"""


def test_threads(gcuda):
    """Six threads, each with a stream, a cache and a workspace of its own: what they get is what one thread gets, and
    each finds its own refusal."""
    env = dict(os.environ, PYTHONPATH="")
    r = subprocess.run([sys.executable, "-c", CHILD % ROOT], capture_output=True, text=True, timeout=300, env=env, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout + r.stderr[-2000:]

"""Attention over a 4-bit key/value cache, and what stands around it, as measured work.

Three operators of a serving step:

* the cache (kind "cache"): new key and value rows are quantised into the pages of a 4-bit cache and the
  same rows are read back as BF16;
* attention over the cache (kind "decode"): the newest rows of every sequence (one token, or the rows of a
  speculative verify step) attend to the sequence's cached positions, all of them or those an indexer kept;
* prompt attention (kind "prompt"): causal attention over packed sequences of different lengths with
  grouped heads, a sequence's queries being the last of its keys' positions.

The cache's layout (include/apus_attn_gcuda.h): pages of 64 positions, [pages][heads][72 * dim] bytes. A head's
block holds the key codes [64][dim / 2], the value codes [64][dim / 2], the key scales [64][dim / 32] and the
value scales [64][dim / 32] in BF16. 32 neighbouring dims share a scale: s = bf16(amax / 7),
code = clamp(rint(x / s), -7, 7) + 8, value = (code - 8) * s. Where a code stands in its row: code_at() below.
"""
import os
import sys

import torch

own = False

PAGE, GROUP = 64, 32


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one verify step's rows (draft depth 3) of one DSA layer: 64 heads of 256
        {"name": "cache_verify_rows", "kind": "cache", "dim": 256, "heads": 64, "rows": 4, "seqs": 1, "before": 517},
        # one chunk of the prompt pass (256 rows) of the same layer
        {"name": "cache_prompt_chunk", "kind": "cache", "dim": 256, "heads": 64, "rows": 256, "seqs": 1, "before": 1280},
        # nine prompts of different lengths that arrive together, 8 heads of 128
        {"name": "cache_ragged_prompts", "kind": "cache", "dim": 128, "heads": 8, "rows": 8191, "seqs": 9, "before": 0},
        # one token of a short chat: latency
        {"name": "decode_one_short", "kind": "decode", "dim": 128, "heads": 8, "group": 4, "rows": 1, "seqs": 1, "longest": 513, "kept": 0, "pool": 0},
        # a verify step (4 rows) of a DSA layer over the whole of a 4096-token prompt and its answer
        {"name": "decode_verify_rows", "kind": "decode", "dim": 256, "heads": 64, "group": 1, "rows": 4, "seqs": 1, "longest": 4363, "kept": 0, "pool": 0},
        # the same step far into a long context, under the indexer's top 2048 (pools of 4 positions)
        {"name": "decode_verify_selected", "kind": "decode", "dim": 256, "heads": 64, "group": 1, "rows": 4, "seqs": 1, "longest": 32771, "kept": 512, "pool": 4},
        # one token of a single long document
        {"name": "decode_one_long", "kind": "decode", "dim": 128, "heads": 8, "group": 8, "rows": 1, "seqs": 1, "longest": 131072, "kept": 0, "pool": 0},
        # a serving batch: 48 sequences of very different lengths
        {"name": "decode_batch", "kind": "decode", "dim": 128, "heads": 8, "group": 4, "rows": 1, "seqs": 48, "longest": 8192, "kept": 0, "pool": 0},
        # one short prompt: latency
        {"name": "prompt_short", "kind": "prompt", "dim": 128, "heads": 8, "group": 4, "rows": 77, "seqs": 1, "before": 0},
        # seven prompts of different lengths, packed
        {"name": "prompt_packed", "kind": "prompt", "dim": 128, "heads": 8, "group": 4, "rows": 4099, "seqs": 7, "before": 0},
        # a 2048-token prompt at the DSA layers' head layout, up to where the indexer still keeps everything
        {"name": "prompt_wide_heads", "kind": "prompt", "dim": 256, "heads": 64, "group": 1, "rows": 2048, "seqs": 1, "before": 0},
        # the second half of a long prompt, over its first half
        {"name": "prompt_long", "kind": "prompt", "dim": 128, "heads": 8, "group": 4, "rows": 8192, "seqs": 1, "before": 4096},
    ]


def spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("cache", "decode", "prompt"))
    dim = rng.choice((64, 128, 256))
    if kind == "cache":
        heads = rng.choice((1, 2, 5, 8, 16, 64))
        rows = spread(rng, 1, 4194304 // (heads * dim))
        return {"kind": kind, "dim": dim, "heads": heads, "rows": rows, "seqs": rng.randint(1, min(rows, 12)), "before": rng.choice((0, spread(rng, 1, 4000)))}
    if kind == "decode":
        heads, group = rng.choice(((1, 8), (2, 7), (4, 16), (8, 4), (8, 8), (16, 1), (64, 1), (3, 5)))
        seqs = spread(rng, 1, 64)
        longest = spread(rng, 16, min(131072, 67108864 // (heads * dim * seqs)))
        pool = rng.choice((0, 0, 4, 6))
        return {"kind": kind, "dim": dim, "heads": heads, "group": group, "rows": min(rng.choice((1, 1, 2, 4, 6)), longest), "seqs": seqs,
                "longest": longest, "kept": spread(rng, 1, 512) if pool else 0, "pool": pool}
    heads, group = rng.choice(((1, 8), (2, 7), (4, 8), (8, 4), (16, 1), (32, 1), (3, 5)))
    rows = spread(rng, 1, min(8192, 8192 * 128 * 32 // (2 * heads * group * dim)))
    return {"kind": kind, "dim": dim, "heads": heads, "group": group, "rows": rows, "seqs": rng.randint(1, min(rows, 16)),
            "before": rng.choice((0, 0, spread(rng, 1, 2048)))}


def parts(total, count, gen):
    """`total` rows cut into `count` sequences of different lengths, one row at least each."""
    if count == 1:
        return [total]
    cuts = (torch.randperm(total - 1, generator=gen)[: count - 1] + 1).sort().values.tolist()
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def lengths(case):
    """The lengths that go with a case, the same for every seed: (rows, positions) of each sequence."""
    gen = torch.Generator().manual_seed(case["dim"] * 131 + case["rows"] * 7 + case["seqs"])
    if case["kind"] == "decode":
        low, high = max(case["rows"], case["longest"] // 16), case["longest"]
        kv = [high] + [int(low + (high - low) * u) for u in torch.rand(case["seqs"] - 1, generator=gen).tolist()]
        return [case["rows"]] * case["seqs"], kv
    rows = parts(case["rows"], case["seqs"], gen)
    return rows, [n + case["before"] for n in rows]


def starts(counts, device):
    return torch.tensor([0] + counts, dtype=torch.int64).cumsum(0).to(torch.int32).to(device)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dim, heads = case["dim"], case["heads"]
    group = case.get("group", 1)
    rows, kv = lengths(case)
    total = sum(rows)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def keys(*shape):
        return (normal(*shape) * (0.6 + 0.9 * torch.rand(shape[-2:], generator=gen, device="cuda"))).to(torch.bfloat16)

    s = {"kind": case["kind"], "dim": dim, "heads": heads, "group": group, "seqs": case["seqs"], "total": total,
         "max_rows": max(rows), "max_len": max(kv), "rows_of": rows, "kv_of": kv, "scale": dim ** -0.5,
         "cu_rows": starts(rows, "cuda"), "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda")}
    if case["kind"] == "prompt":
        s["q"] = (1.5 * normal(total, heads * group, dim)).to(torch.bfloat16)
        s["k"], s["v"] = keys(sum(kv), heads, dim), normal(sum(kv), heads, dim).to(torch.bfloat16)
        s["cu_k"] = starts(kv, "cuda")
        return s
    # the pages of all sequences, in an order of their own
    need = [-(-n // PAGE) for n in kv]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, at = torch.zeros(case["seqs"], max(need), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"] = table.cuda()
    s["pages"] = torch.zeros(sum(need) + 3, heads, 72 * dim, dtype=torch.uint8, device="cuda")
    if case["kind"] == "cache":
        s["k"], s["v"] = keys(total, heads, dim), normal(total, heads, dim).to(torch.bfloat16)
        return s
    for i in range(0, len(order), 256):     # a filled cache
        n = min(256, len(order) - i)
        where = torch.arange(PAGE, device="cuda").repeat(n)
        at = torch.arange(i, i + n, device="cuda").repeat_interleave(PAGE)
        write_rows(s["pages"], dim, at, where, keys(n * PAGE, heads, dim), normal(n * PAGE, heads, dim).to(torch.bfloat16))
    s["q"] = (1.5 * normal(total, heads * group, dim)).to(torch.bfloat16)
    s["pool"] = case["pool"]
    if case["pool"]:
        # the indexer's choice: the best pools of each row, much the same ones for the rows of one step
        pools = max(1, max(kv) // case["pool"])
        liked = normal(case["seqs"], 1, pools) + 0.4 * normal(case["seqs"], case["rows"], pools)
        ends = (s["kv_len"].long()[:, None] - case["rows"] + 1 + torch.arange(case["rows"], device="cuda")) // case["pool"]
        liked = liked.masked_fill(torch.arange(pools, device="cuda") >= ends[..., None], float("-inf"))
        kept = torch.zeros(liked.shape, dtype=torch.uint8, device="cuda")
        kept.scatter_(2, liked.topk(min(case["kept"], pools), dim=2).indices, 1)
        s["sel"] = kept.reshape(total, pools)
    return s


def work(case):
    rows, kv = lengths(case)
    dim, heads, total = case["dim"], case["heads"], sum(rows)
    held = 2 * (dim // 2 + dim // GROUP * 2)                # bytes of one position of one head
    if case["kind"] == "cache":
        return {"bytes": total * heads * (2 * 2 * dim * 2 + 2 * held), "flops": total * heads * dim * 2 * 4}
    group = case["group"]
    if case["kind"] == "decode":
        if case["pool"]:                                    # what one row keeps is read by all
            seen = [min(n, case["kept"] * case["pool"] + case["pool"]) for n in kv]
        else:
            seen = kv
        pairs = sum(n * r for n, r in zip(seen, rows))
        moved = sum(seen) * heads * held + 2 * total * heads * group * dim * 2
        return {"bytes": moved + (total * (max(kv) // case["pool"]) if case["pool"] else 0), "flops": 4 * pairs * heads * group * dim}
    pairs = sum(r * (n - r) + r * (r + 1) // 2 for r, n in zip(rows, kv))
    return {"bytes": 2 * (2 * total * heads * group * dim + 2 * sum(kv) * heads * dim), "flops": 4 * pairs * heads * group * dim}


# ---------------------------------------------------------- the plain forms

def code_at(dim, device):
    """Where the codes of a head's row stand: (keys, values), each [64][dim] with the index of the 4-bit
    code (word * 8 + nibble) of dim d in the row of the page's position p."""
    p = torch.arange(PAGE, device=device)[:, None]
    d = torch.arange(dim, device=device)[None, :]
    j, q, g, jj = d // 32, d % 32 // 8, d % 32 // 4, d // 64
    if dim == 64:
        k, v = q * 2 + j + 0 * p, g + 0 * p
    elif dim == 128:
        k, v = q * 4 + j + 0 * p, (g ^ ((p >> 1 & 1) << 2)) * 2 + jj
    else:
        k, v = ((j >> 2) ^ (p >> 2 & 1)) * 16 + q * 4 + (j & 3), (g ^ ((p & 3) << 1)) * 4 + jj
    return k * 8 + d % 8, v * 8 + (j & 1) * 4 + d % 4


def regions(pages, dim):
    """The four parts of every page: key codes, value codes, key scales, value scales."""
    a, b, c = 32 * dim, 64 * dim, 68 * dim
    groups = dim // GROUP
    return (pages[..., :a].unflatten(-1, (PAGE, dim // 2)), pages[..., a:b].unflatten(-1, (PAGE, dim // 2)),
            pages[..., b:c].view(torch.bfloat16).unflatten(-1, (PAGE, groups)), pages[..., c:].view(torch.bfloat16).unflatten(-1, (PAGE, groups)))


def quantise(x):
    """Codes [rows][heads][dim] and scales [rows][heads][dim / 32] of BF16 rows."""
    f = x.float().unflatten(-1, (-1, GROUP))
    top = f.abs().amax(-1)
    fine = torch.isfinite(f).all(-1)
    s = torch.where(fine, top / torch.full_like(top, 7.0), torch.nan).to(torch.bfloat16)
    by = s.float()[..., None]
    c = torch.where(fine[..., None] & (by > 0), torch.round(f / by).clamp(-7, 7), 0.0) + 8
    return c.to(torch.uint8).flatten(-2), s


def write_rows(pages, dim, page, off, k, v):
    """Quantises rows into the places (page, off) of the cache."""
    kc, vc, ks, vs = regions(pages, dim)
    at = code_at(dim, k.device)

    def put(x, at, to, scales):
        c, s = quantise(x)
        order = at.argsort(-1)[off]                         # the dim that stands at each place of the row
        c = c.gather(-1, order[:, None].expand_as(c)).unflatten(-1, (-1, 2))
        to[page, :, off] = c[..., 0] | c[..., 1] << 4
        scales[page, :, off] = s

    put(k, at[0], kc, ks)
    put(v, at[1], vc, vs)


def values(codes, scales, at):
    """Codes [..., 64][dim / 2] and scales of whole pages as 32-bit values [..., 64][dim]."""
    p = torch.arange(PAGE, device=codes.device)[:, None]
    c = (codes[..., p, at // 2] >> (at % 2 * 4).to(torch.uint8) & 15).float() - 8
    return (c.unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def rows_at(s):
    """(sequence, position) of every row of the batch."""
    n = s["cu_rows"].long().diff()
    seq = torch.repeat_interleave(torch.arange(s["seqs"], device=n.device), n, output_size=s["total"])
    return seq, s["kv_len"].long()[seq] - n[seq] + torch.arange(s["total"], device=n.device) - s["cu_rows"].long()[seq]


def cache_plain(s):
    seq, pos = rows_at(s)
    page, off = s["table"].long()[seq, pos // PAGE], pos % PAGE
    write_rows(s["pages"], s["dim"], page, off, s["k"], s["v"])
    kc, vc, ks, vs = regions(s["pages"], s["dim"])
    at = code_at(s["dim"], page.device)

    def read(codes, scales, at):
        c = codes[page, :, off]
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2).gather(-1, at[off][:, None].expand(-1, c.shape[1], -1)).float() - 8
        return (c.unflatten(-1, (-1, GROUP)) * scales[page, :, off].float()[..., None]).flatten(-2).to(torch.bfloat16)

    return {"k": read(kc, ks, at[0]), "v": read(vc, vs, at[1])}


def softmax_plain(score, seen):
    """Weights over the last axis of the places that are seen; a row that sees none has none."""
    score = torch.where(seen, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    return w / w.sum(-1, keepdim=True).clamp_min(1e-38)


def decode_plain(s):
    dim, heads, group, seqs, R = s["dim"], s["heads"], s["group"], s["seqs"], s["max_rows"]
    kc, vc, ks, vs = regions(s["pages"][s["table"].long()], dim)           # [seqs][pages][heads][64][..]
    at = code_at(dim, kc.device)
    k = values(kc, ks, at[0]).transpose(1, 2).flatten(2, 3)                 # [seqs][heads][positions][dim]
    v = values(vc, vs, at[1]).transpose(1, 2).flatten(2, 3)
    q = s["q"].float().reshape(seqs, R, heads, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)   # [seqs][heads][group * R][dim]
    seen_to = s["kv_len"].long()[:, None] - R + 1 + torch.arange(R, device=q.device)              # [seqs][R]
    j = torch.arange(k.shape[2], device=q.device)
    seen = j < seen_to[..., None]
    if s["pool"]:
        sel = s["sel"].reshape(seqs, R, -1).bool()
        chosen = sel[:, :, (j // s["pool"]).clamp_max(sel.shape[-1] - 1)] & (j // s["pool"] < sel.shape[-1])
        seen = seen & (chosen | (j >= (seen_to - seen_to % s["pool"])[..., None]))
    seen = seen[:, None, None].expand(-1, heads, group, -1, -1).flatten(2, 3)
    w = softmax_plain(q @ k.transpose(-1, -2) * s["scale"], seen)
    out = (w @ v).unflatten(2, (group, R)).permute(0, 3, 1, 2, 4)
    return {"out": out.reshape(s["total"], heads * group, dim).to(torch.bfloat16)}


def prompt_plain(s):
    heads, group = s["heads"], s["group"]
    q = s["q"].float().unflatten(1, (heads, group)).permute(1, 2, 0, 3)     # [heads][group][rows][dim]
    k, v = s["k"].float().transpose(0, 1)[:, None], s["v"].float().transpose(0, 1)[:, None]
    seq, pos = rows_at(s)
    n = s["kv_len"].long()
    k_seq = torch.repeat_interleave(torch.arange(s["seqs"], device=n.device), n, output_size=k.shape[2])
    k_pos = torch.arange(k.shape[2], device=n.device) - s["cu_k"].long()[k_seq]
    seen = (seq[:, None] == k_seq) & (k_pos <= pos[:, None])
    w = softmax_plain(q @ k.transpose(-1, -2) * s["scale"], seen)
    return {"out": (w @ v).permute(2, 0, 1, 3).flatten(1, 2).to(torch.bfloat16)}


# ------------------------------------------------------ the framework's calls

def engine():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "apus-glm5.3-flash_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import apus_gcuda
    return apus_gcuda


def run(s):
    if not own:
        return {"cache": cache_plain, "decode": decode_plain, "prompt": prompt_plain}[s["kind"]](s)
    G = engine()
    if s["kind"] == "prompt":
        batch = s.get("plan")
        if batch is None:       # a program's handle of its batch
            batch = s["plan"] = G.PromptBatch(s["cu_rows"], s["cu_k"], max_rows=s["max_rows"])
        out = torch.empty_like(s["q"])
        G.prompt_attn(batch, s["q"], s["k"], s["v"], out, s["scale"])
        return {"out": out}
    if "plan" not in s:
        s["plan"] = G.Kv4Cache(s["pages"]), G.Kv4Batch(s["cu_rows"], s["kv_len"], s["table"], max_rows=s["max_rows"], max_len=s["max_len"])
    cache, batch = s["plan"]
    if s["kind"] == "cache":
        G.kv4_append(cache, batch, s["k"], s["v"])
        k, v = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        G.kv4_read(cache, batch, k, v)
        return {"k": k, "v": v}
    if "work" not in s:
        s["work"] = torch.empty(G.kv4_attn_workspace(cache, batch, s["q"].shape[1]), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(s["q"])
    G.kv4_attn(cache, batch, s["q"], out, s["scale"], s["work"], sel=s.get("sel"), pool=s["pool"])
    return {"out": out}


# ------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    dim, heads, group = s["dim"], s["heads"], s["group"]
    if case["kind"] == "cache":
        def held(x):
            x = x.double().reshape(s["total"], heads, dim // 32, 32)
            step = (x.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double()
            return ((x / step).nan_to_num(0.0).round().clamp(-7, 7) * step).reshape(s["total"], heads, dim)
        return {"k": held(s["k"]), "v": held(s["v"])}

    def dims_of(kind, p, w):
        """The dims of the eight codes in word w of position p's row."""
        if kind == "v":
            u, jj = w // (dim // 64), w % (dim // 64)
            g = u ^ {64: 0, 128: p // 2 % 2 * 4, 256: p % 4 * 2}[dim]
            return [64 * jj + 32 * (i // 4) + 4 * g + i % 4 for i in range(8)]
        b = min(dim // 32, 4)
        j = w % b + (4 * (w // 16 ^ p // 4 % 2) if dim == 256 else 0)
        return [32 * j + 8 * (w % (4 * b) // b) + i for i in range(8)]

    places = {}
    for kind in "kv" if case["kind"] == "decode" else "":
        eight = torch.tensor([[dims_of(kind, p, w) for w in range(dim // 8)] for p in range(8)], device="cuda")
        places[kind] = eight.flatten(1).repeat(PAGE // 8, 1)

    def held_values(block, kind):
        """One head's pages [pages][72 * dim] as 64-bit values [positions][dim], word by word."""
        n = block.shape[0]
        at, to = (0, 64 * dim) if kind == "k" else (32 * dim, 68 * dim)
        word = block[:, at:at + 32 * dim].contiguous().view(torch.int32).reshape(n, PAGE, dim // 8).long() & 0xFFFFFFFF
        step = block[:, to:to + 4 * dim].contiguous().view(torch.bfloat16).double().reshape(n, PAGE, dim // 32)
        code = torch.stack([word >> 4 * i & 15 for i in range(8)], -1).double() - 8
        out = torch.empty(n, PAGE, dim, dtype=torch.float64, device=block.device)
        out.scatter_(2, places[kind].expand(n, -1, -1), code.flatten(2))
        return (out * step.repeat_interleave(32, -1)).flatten(0, 1)

    out = torch.empty(s["total"], heads * group, dim, dtype=torch.float64, device="cuda")
    row, key = 0, 0
    for i, (r, n) in enumerate(zip(s["rows_of"], s["kv_of"])):
        last = torch.arange(n - r, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hide = j > last
        if case["kind"] == "decode" and s["pool"]:
            pool = s["pool"]
            by = torch.nn.functional.pad(s["sel"][row:row + r], (0, 1))
            whole = (last + 1) // pool * pool
            hide = hide | ((j < whole) & (by.gather(1, (j // pool).clamp_max(by.shape[1] - 1).expand(r, n)) == 0))
        for h in range(heads):
            if case["kind"] == "decode":
                mine = s["pages"][s["table"][i, : -(-n // PAGE)].long(), h]
                k, v = held_values(mine, "k")[:n], held_values(mine, "v")[:n]
            else:
                k, v = s["k"][key:key + n, h].double(), s["v"][key:key + n, h].double()
            q = s["q"][row:row + r, h * group:(h + 1) * group].double()
            x = torch.einsum("rgd,nd->grn", q, k) * s["scale"]
            out[row:row + r, h * group:(h + 1) * group] = torch.einsum("grn,nd->rgd", torch.softmax(x.masked_fill(hide, -torch.inf), -1), v)
        row, key = row + r, key + n
    return {"out": out}

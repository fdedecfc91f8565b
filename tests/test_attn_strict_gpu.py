"""Attention over the 4-bit cache and prompt attention held to more than the elementwise bound, which has to allow for
every rounding pointing the same way: the root mean square of the errors, their bias, and that each visible position,
and no other, takes part with its weight.

Roundings to nearest are off by half a step at most (U = 2^-8 of a BF16 number, H = 2^-11 of an f16 number) and by 1 /
sqrt(3) of that in the root mean square, since they spread evenly over a step.  With values that are independent and of
mean 0, as here, the errors that rounded weights make add up as the output itself does: sum p^2 v^2 against (sum p v)^2
in the mean.  So the relative error of a whole output (root of the sum of squares) is at most
  sqrt(a U^2 + b H^2) / sqrt(3),
a the BF16 roundings (the output's own, and the weight's for prompts), b the f16 roundings of a weight (two over the
cache); the fp32 sums and exponentials add less than 2^-16 at these sizes of scores, and the sample is of thousands of
elements, so 10 % is allowed for chance.  The bias, the factor by which the output is the reference, is off by the mean
of such errors: those of the n outputs are independent, those of the weights at least from row to row and head to head."""
import math

import pytest
import torch

import attn_ref as R
from test_kv4_gpu import Case, bf16, gen
from test_prompt_attn_gpu import run as run_prompt

pytestmark = pytest.mark.gpu


def assert_close(got, want, a, b, rows):
    """got, want [..][dim]; `rows` independent sets of weights."""
    got, want = got.double().cpu(), want.double().cpu()
    out, weights = R.U / math.sqrt(3), math.sqrt((a - 1) * R.U ** 2 + b * R.H ** 2) / math.sqrt(3)
    error = float((got - want).norm() / want.norm())
    assert error <= 1.1 * math.hypot(out, weights) + 2.0 ** -16, error
    factor = float((got * want).sum() / (want * want).sum())
    # six standard deviations of a mean
    assert abs(factor - 1) <= 6 * (out / math.sqrt(want.numel()) + weights / math.sqrt(rows)) + 2.0 ** -16, factor


CACHE = [
    # dim, heads, group, rows, lengths
    (64, 2, 4, 1, [300, 1030, 2000]), (128, 2, 4, 1, [300, 1030, 5003]), (128, 4, 8, 2, [300, 700, 2500]),
    (256, 16, 1, 4, [300, 1030]), (256, 4, 1, 4, [9001]), (64, 4, 4, 2, [33333, 100]), (128, 8, 1, 1, [20000]),
]


@pytest.mark.parametrize("case", range(len(CACHE)))
@pytest.mark.parametrize("std", [0.5, 2.0])
def test_cache_attention(gcuda, case, std):
    dim, heads, group, rows, lens = CACHE[case]
    c = Case(gcuda, dim, heads, lens, [rows] * len(lens), seed=case)
    c.fill_all()
    q = bf16(c.g, c.total, heads * group, dim, std=std).cuda()
    scale = dim ** -0.5
    for pool in (0, 4):
        sel = (torch.rand(c.total, max(lens) // 4 + 1, generator=c.g) < 0.4).to(torch.uint8) if pool else None
        got = c.attn(q, scale, sel if sel is None else sel.cuda(), pool).cpu()
        for i, n in enumerate(lens):
            r0, k0 = int(c.cu[i]), c.starts[i]
            j = torch.arange(n)[None]
            end = n - rows + 1 + torch.arange(rows)[:, None]
            seen = j < end
            if pool:
                seen = seen & ((j >= end - end % pool) | sel[r0:r0 + rows].gather(1, (j // pool).expand(rows, -1)).bool())
            want = R.attention(q[r0:r0 + rows].double().cpu(), c.k[k0:k0 + n], c.v[k0:k0 + n], scale, seen)[0]
            assert_close(got[r0:r0 + rows], want, 1, 2, rows * heads * group)


@pytest.mark.parametrize("dim,heads,group,rows,keys", [(64, 2, 4, [300, 1000], [300, 1500]), (128, 2, 2, [257, 700], [900, 700]),
                                                       (256, 2, 2, [300, 1100], [300, 2300]), (128, 1, 7, [130], [4099])])
@pytest.mark.parametrize("std", [0.5, 2.0])
def test_prompts(gcuda, dim, heads, group, rows, keys, std):
    g = gen(dim + heads)
    q = bf16(g, sum(rows), heads * group, dim, std=std).cuda()
    k, v = (bf16(g, sum(keys), heads, dim).cuda() for _ in range(2))
    got = run_prompt(gcuda, q, k, v, rows, keys, dim ** -0.5)
    q0 = k0 = 0
    for n, m in zip(rows, keys):
        seen = (torch.arange(m)[None] <= m - n + torch.arange(n)[:, None]).cuda()
        want = R.attention(q[q0:q0 + n].double(), k[k0:k0 + m].double(), v[k0:k0 + m].double(), dim ** -0.5, seen)[0]
        assert_close(got[q0:q0 + n], want, 2, 0, n * heads * group)
        q0, k0 = q0 + n, k0 + m


# Every position by itself: with keys of zeros all weights are 1 / (positions seen), and a value of 1 in one dim, zeros
# in the others, shows in that dim's output alone.  A scale of bf16(1 / 7) holds 7 / 7 = 1 to 2^-8 (seven times the
# scale, as a whole number of its steps); the output's rounding adds U, the weight's two f16 roundings 2 H.

@pytest.mark.parametrize("dim,heads,group,rows,length", [(64, 1, 2, 3, 300), (128, 2, 1, 2, 517), (128, 1, 16, 1, 700),
                                                         (256, 2, 1, 4, 1030), (64, 2, 4, 1, 1300), (128, 1, 4, 1, 70)])
@pytest.mark.parametrize("selected", [False, True])
def test_every_position_takes_part(gcuda, dim, heads, group, rows, length, selected):
    c = Case(gcuda, dim, heads, [length], [rows], seed=length)
    k = torch.zeros(length, heads, dim, dtype=torch.bfloat16)
    q = bf16(c.g, rows, heads * group, dim).cuda()
    end = length - rows + 1 + torch.arange(rows)[:, None]
    seen = torch.arange(length)[None] < end
    sel, pool = None, 0
    if selected:
        pool = 3
        sel = (torch.rand(rows, length // pool + 1, generator=c.g) < 0.5).to(torch.uint8)
        j = torch.arange(length)[None]
        seen = seen & ((j >= end - end % pool) | sel.gather(1, (j // pool).expand(rows, -1)).bool())
    count = seen.sum(1)
    for first in range(0, length, dim):
        n = min(dim, length - first)
        v = torch.zeros(length, heads, dim, dtype=torch.bfloat16)
        v[first + torch.arange(n), :, torch.arange(n)] = 1.0
        c.write_all(k, v)
        got = c.attn(q, 0.1, sel if sel is None else sel.cuda(), pool).float().cpu()
        for r in range(rows):
            want = torch.zeros(dim)
            want[:n] = seen[r, first:first + n].float() / count[r]
            assert ((got[r] - want).abs() <= want * (2 * R.U + 2 * R.H + 2.0 ** -12)).all(), (first, r)


@pytest.mark.parametrize("dim,heads,group,rows,keys", [(64, 1, 2, 300, 300), (128, 1, 1, 200, 330), (256, 1, 1, 130, 260),
                                                       (128, 2, 2, 5, 129), (64, 1, 1, 20, 13)])
def test_every_key_takes_part(gcuda, dim, heads, group, rows, keys):
    """The same for prompts: one BF16 rounding of a weight, which is the same for all keys of a row, so that numerator
    and sum may differ by U, and the output's."""
    g = gen(rows)
    q = bf16(g, rows, heads * group, dim).cuda()
    k = torch.zeros(keys, heads, dim, dtype=torch.bfloat16).cuda()
    see = (keys - rows + 1 + torch.arange(rows)).clamp_min(0)
    for first in range(0, keys, dim):
        n = min(dim, keys - first)
        v = torch.zeros(keys, heads, dim, dtype=torch.bfloat16)
        v[first + torch.arange(n), :, torch.arange(n)] = 1.0
        got = run_prompt(gcuda, q, k, v.cuda(), [rows], [keys], 0.1).float().cpu()
        want = torch.zeros(rows, dim)
        want[:, :n] = (first + torch.arange(n)[None] < see[:, None]).float() / see.clamp_min(1)[:, None]
        assert ((got - want[:, None]).abs() <= want[:, None] * (2 * R.U + 2.0 ** -12)).all(), first

"""Attention over the 4-bit cache (apus_gcuda_kv4_attn_dev) over the whole range of its values and scores: what a
position weighs goes by its score alone, however large or small its values are."""
import math

import pytest
import torch

import attn_ref as R
from test_kv4_gpu import Case, bf16, gen

pytestmark = pytest.mark.gpu


def run(gcuda, dim, heads, group, k, v, q, scale=0.125, lens=None, rows=None):
    """The case's attention over all positions, and under a selection that keeps everything, both held to the bound."""
    n = k.shape[0]
    c = Case(gcuda, dim, heads, lens or [n], rows or [q.shape[0]], seed=dim)
    c.write_all(k, v)
    got = c.attn(q, scale)
    c.check(q, got, scale)
    sel = torch.ones(q.shape[0], max(c.lens), dtype=torch.uint8)
    c.check(q, c.attn(q, scale, sel.cuda(), 1), scale, sel, 1)
    return got


def level(g, n, heads, dim, values):
    """Keys of zeros (so every score is the same), values of random signs with the given magnitude at each position."""
    v = torch.where(torch.rand(n, heads, dim, generator=g) < 0.3, -0.5, 1.0) * torch.as_tensor(values)[:, None, None]
    return torch.zeros(n, heads, dim, dtype=torch.bfloat16), v.to(torch.bfloat16)


@pytest.mark.parametrize("dim,heads,group", [(64, 1, 2), (128, 2, 16), (128, 1, 3), (256, 1, 4)])
@pytest.mark.parametrize("large", [1e6, 1e12, 1e20, 1e30])
def test_zero_values_keep_their_weight(gcuda, dim, heads, group, large):
    """Zeros in one unit, in alternation, and in runs of their own, beside large values."""
    for n, zero in ((128, lambda j: j < 32), (96, lambda j: j >= 64), (200, lambda j: j % 2 == 0), (6000, lambda j: j < 3500),
                    (6000, lambda j: j % 3 == 1)):
        g = gen(n)
        j = torch.arange(n)
        k, v = level(g, n, heads, dim, torch.where(zero(j), 0.0, large))
        run(gcuda, dim, heads, group, k, v, bf16(g, 2, heads * group, dim).cuda())


@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (256, 2)])
@pytest.mark.parametrize("small,large", [(1e-20, 1e20), (1e-36, 1.0), (1e-30, 1e30), (1e-3, 1e36)])
def test_small_values_keep_their_weight(gcuda, dim, group, small, large):
    for n, pick in ((128, lambda j: j < 32), (200, lambda j: j % 2 == 0), (6000, lambda j: j < 3500)):
        g = gen(n + dim)
        k, v = level(g, n, 1, dim, torch.where(pick(torch.arange(n)), small, large))
        run(gcuda, dim, 1, group, k, v, bf16(g, 1, group, dim).cuda())


@pytest.mark.parametrize("dim,group", [(64, 1), (128, 16), (256, 2)])
def test_zero_prefix_with_rising_scores(gcuda, dim, group):
    """Zero values whose scores rise step by step (7.9 powers of two above the first ones'), then ordinary values."""
    for n in (200, 3000):
        g = gen(n)
        k, v = bf16(g, 2 * n, 1, dim), bf16(g, 2 * n, 1, dim) * 0.3
        v[:n] = 0.0
        up = torch.zeros(2 * n)
        up[16:] = 7.9 * math.log(2.0) * 8 / dim            # q of ones, scale 1 / 8
        k[:] = up[:, None, None].to(torch.bfloat16)
        run(gcuda, dim, 1, group, k, v, torch.ones(1, group, dim, dtype=torch.bfloat16).cuda())


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 16), (256, 1)])
@pytest.mark.parametrize("power", [-112, -124, -98])
def test_tiny_values_over_a_long_context(gcuda, dim, group, power):
    n = 8192
    g = gen(power + 200)
    k, v = level(g, n, 1, dim, torch.full((n,), 7 * 2.0 ** power))
    v = v.abs()
    got = run(gcuda, dim, 1, group, k, v, bf16(g, 1, group, dim).cuda())
    assert (got > 0).all()


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 16), (256, 1)])
@pytest.mark.parametrize("size", [8e37, 3e38])
def test_largest_values_with_rising_scores(gcuda, dim, group, size):
    """Values at the type's upper end whose weights rise by 7.9 powers of two after the first ones."""
    for n in (100, 3000):
        g = gen(n)
        k, v = level(g, n, 1, dim, torch.full((n,), size))
        k[20:] = torch.tensor(7.9 * math.log(2.0) * 8 / dim).to(torch.bfloat16)
        got = run(gcuda, dim, 1, group, k, v, torch.ones(1, group, dim, dtype=torch.bfloat16).cuda())
        assert got.isfinite().all()


def test_huge_scores(gcuda):
    """Scores of 2^27 and more, where neighbouring fp32 numbers are 8 to 16 apart: the later positions' lie one such
    step above the first ones'.  Whatever the rounding of the scores, an output lies between the values."""
    dim, lens = 64, [40] * 48
    k = torch.zeros(sum(lens), 1, dim)
    v = torch.ones(sum(lens), 1, dim)
    v[:, :, 1] = -1.0
    for i in range(len(lens)):
        k[40 * i:40 * i + 40, 0, :32] = 2.0 ** 22 * (1 + i / 64)          # 2^27 (1 + i / 64) with q of ones
        k[40 * i + 20:40 * i + 40, 0, 32:] = (4 + i % 8) / 32.0           # 4 to 11 more
    c = Case(gcuda, dim, 1, lens, [1] * len(lens), seed=3)
    c.write_all(k.to(torch.bfloat16), v.to(torch.bfloat16))
    q = torch.ones(len(lens), 2, dim, dtype=torch.bfloat16).cuda()
    got = c.attn(q, 1.0)
    torch.cuda.synchronize()
    want = torch.ones(len(lens), 2, dim)
    want[:, :, 1] = -1.0
    # every value is the same: weights of 2^-11 and a BF16 rounding
    assert ((got.float().cpu() - want).abs() <= R.U + 2 * R.H).all()


@pytest.mark.parametrize("dim,group", [(64, 2), (128, 16), (256, 1)])
@pytest.mark.parametrize("power", [6, 12, 16, 20, 24, 30])
def test_large_scores(gcuda, dim, group, power):
    """Scores of about 2^power that differ from position to position: whatever their rounding, equal values come out
    as they are (each weight off by two f16 roundings, the sums by fp32's, the result by a BF16 rounding)."""
    for n in (90, 3000):
        g = gen(power)
        k = bf16(g, n, 1, dim)
        k[:, :, 0] = 7.0
        v = torch.full((n, 1, dim), 3.0e-2)
        v[:, :, 1::2] = -7.0
        c = Case(gcuda, dim, 1, [n], [1], seed=power)
        c.write_all(k, v.to(torch.bfloat16))
        q = bf16(g, 1, group, dim)
        q[:, :, 0] = 2.0 ** power / 7.0
        held = c.v[0, 0].float()
        for sel in (None, torch.ones(1, n, dtype=torch.uint8).cuda()):
            got = c.attn(q.cuda(), 1.0, sel, 0 if sel is None else 1)
            torch.cuda.synchronize()
            assert ((got.float().cpu() - held).abs() <= held.abs() * (R.U + 2 * R.H + 2.0 ** -18)).all()


def test_query_beyond_the_scores(gcuda):
    """A query whose factor passes fp32 makes its rows NaN, whatever the keys' signs; the others are as before."""
    g = gen(4)
    c = Case(gcuda, 128, 1, [70, 700, 20], [2, 1, 1], seed=4)
    k, v = bf16(g, 790, 1, 128).abs(), bf16(g, 790, 1, 128)
    c.write_all(k, v)
    q = bf16(g, 4, 2, 128).cuda()
    want = c.attn(q, 0.1)
    for sign in (1.0, -1.0):
        big = q.clone()
        big[1, 0] = sign * 3e38
        big[2, 1] = big[3, 0] = sign * 3e38
        got = c.attn(big, 0.1)
        torch.cuda.synchronize()
        assert got[1, 0].isnan().all() and got[2, 1].isnan().all() and got[3, 0].isnan().all()
        got[1, 0], got[2, 1], got[3, 0] = want[1, 0], want[2, 1], want[3, 0]
        assert torch.equal(got, want)

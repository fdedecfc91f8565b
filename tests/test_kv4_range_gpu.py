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

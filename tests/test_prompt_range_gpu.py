"""Causal prompt attention (apus_gcuda_prompt_attn_dev) at the ends of its scores' range."""
import pytest
import torch

import attn_ref as R
from test_kv4_gpu import bf16, gen
from test_prompt_attn_gpu import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,group", [(64, 2), (128, 4), (256, 1)])
@pytest.mark.parametrize("power", [6, 12, 18, 24, 30, 36, 48, 90])
def test_large_scores(gcuda, dim, group, power):
    """Scores of about 2^power that differ from key to key, rising and falling: whatever their rounding, equal values come
    out as they are (a weight and the result off by one BF16 rounding each, the sums by fp32's)."""
    for rows, keys in ((150, 150), (40, 600)):
        g = gen(power)
        k = bf16(g, keys, 1, dim)
        k[:, :, 0] = (torch.rand(keys, 1, generator=g) + 1.0).to(torch.bfloat16)
        v = torch.full((keys, 1, dim), 3.0e-2)
        v[:, :, 1::2] = -7.0
        v = v.to(torch.bfloat16)
        q = bf16(g, rows, group, dim)
        q[:, :, 0] = 2.0 ** power
        got = run(gcuda, q.cuda(), k.cuda(), v.cuda(), [rows], [keys], 1.0).float().cpu()
        held = v[0, 0].float()
        assert ((got - held).abs() <= held.abs() * (2 * R.U + 2.0 ** -16)).all(), (rows, keys)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("big", [2.0 ** 40, float("inf")])
def test_large_scores_of_other_rows(gcuda, dim, big):
    """A row's bits do not go by its neighbours' scores, of its own sequence or of the next."""
    g = gen(dim)
    rows, keys = [70, 5, 200], [300, 5, 200]
    q = bf16(g, 275, 2, dim, std=3.0).cuda()
    k, v = (bf16(g, 505, 1, dim).cuda() for _ in range(2))
    want = run(gcuda, q, k, v, rows, keys, 0.1)
    q2 = q.clone()
    at = [3, 40, 71, 90, 274]
    q2[at] = (q2[at].float().sign() * big).to(torch.bfloat16)
    got = run(gcuda, q2, k, v, rows, keys, 0.1)
    keep = [i for i in range(275) if i not in at]
    assert torch.equal(got[keep], want[keep])

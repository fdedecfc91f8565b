"""Plain 64-bit references of the operators of include/apus_attn_gcuda.h, and
the error bounds that their tests use.

A BF16 rounding is off by at most U = 2^-8 of the value, an f16 rounding by
H = 2^-11."""
import numpy as np
import torch

PAGE = 64
U, H = 2.0 ** -8, 2.0 ** -11


def word_and_code(dim, p, d):
    """(key word, key code, value word, value code) of dim d at position p, as the header states them."""
    j, q, g = d // 32, d % 32 // 8, d % 32 // 4
    kw = {64: 2 * q + j, 128: 4 * q + j}.get(dim, 16 * ((j // 4) ^ (p // 4 % 2)) + 4 * q + j % 4)
    vw = {64: g, 128: 2 * (g ^ 4 * (p // 2 % 2)) + d // 64}.get(dim, 4 * (g ^ 2 * (p % 4)) + d // 64)
    return kw, d % 8, vw, 4 * (j % 2) + d % 4


_places = {}


def places(dim):
    """Index of each code (word * 8 + code) by [position][dim], for keys and values."""
    if dim not in _places:
        t = np.array([[word_and_code(dim, p, d) for d in range(dim)] for p in range(PAGE)])
        _places[dim] = t[..., 0] * 8 + t[..., 1], t[..., 2] * 8 + t[..., 3]
    return _places[dim]


def split(pages, dim):
    """Pages (CPU uint8 [n][heads][72 dim]) -> key codes, value codes [n][heads][64][dim] (natural order, 0..15)
    and key, value scales [n][heads][64][dim / 32] (float64)."""
    n, h, _ = pages.shape
    out = []
    for at, place in ((0, places(dim)[0]), (32 * dim, places(dim)[1])):
        b = pages[..., at:at + 32 * dim].reshape(n, h, PAGE, dim // 2)
        codes = torch.stack((b & 15, b >> 4), -1).reshape(n, h, PAGE, dim)
        out.append(codes.gather(-1, torch.from_numpy(place).expand(n, h, -1, -1)))
    for at in (64 * dim, 68 * dim):
        s = pages[..., at:at + 4 * dim].contiguous().view(torch.bfloat16)
        out.append(s.double().reshape(n, h, PAGE, dim // 32))
    return out


def quantise(x):
    """Codes 0..15 [..., dim] and scales [..., dim / 32] of BF16 rows, decided in 64 bits."""
    f = x.double().unflatten(-1, (-1, 32))
    fine = torch.isfinite(f).all(-1)
    s = torch.where(fine, f.abs().amax(-1) / 7, torch.nan).to(torch.bfloat16).double()
    c = torch.where(fine[..., None] & (s[..., None] > 0), torch.round(f / s[..., None]).clamp(-7, 7), 0.0)
    return (c + 8).to(torch.uint8).flatten(-2), s


def held(codes, scales):
    """The 64-bit values that codes and scales stand for."""
    return ((codes.double() - 8).unflatten(-1, (-1, 32)) * scales[..., None]).flatten(-2)


def attention(q, k, v, scale, seen, extra=None, steps=None):
    """Rows q [r][heads][dim] over k, v [n][kv heads][dim] (64 bits), seen [r][n]: (out, spread, slack, floor).
    spread is sum p |v| / sum p; slack bounds the relative error of a weight that fp32 sums of the scores make:
    each of the dim products (and each term of `extra`, [n][kv heads][dim]: further magnitudes that a kernel adds
    and takes away again) takes part in at most dim + 8 additions off by 2^-22 of the running sum.
    floor is what f16's least step adds where `steps`, [n][kv heads], the largest value scale of each position, is
    given.  With 2^E <= steps < 2^(E + 1), p 2^E is held in f16 in a unit in which the largest one of the row is 2^5 at
    least, and the scales divided by 2^E, below 2, too.  Below 2^-14 a rounding is off by 2^-25 at most, so (codes of at
    most 7): 7 * 2 * 2^-30 max(p 2^E) a position for p 2^E, 7 * 2^-30 max(p 2^E) for its product with a scale, and
    7 * 2^-25 p 2^E for the scale."""
    r, heads, dim = q.shape
    if not k.shape[0]:
        return torch.zeros_like(q), torch.zeros_like(q), 0.0, 0.0
    group = heads // k.shape[1]
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    hide = ~seen[:, None, :]
    x = torch.einsum("rhd,nhd->rhn", q, k).masked_fill(hide, -torch.inf) * scale
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0)).masked_fill(hide, 0.0)
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    out = torch.einsum("rhn,nhd->rhd", w, v)
    spread = torch.einsum("rhn,nhd->rhd", w, v.abs())
    mag = k.abs() if extra is None else k.abs() + extra.repeat_interleave(group, 1)
    size = torch.einsum("rhd,nhd->rhn", q.abs(), mag).masked_fill(hide, 0.0).amax(-1, keepdim=True)
    slack = 2 * (dim + 8) * 2.0 ** -22 * abs(scale) * size + k.shape[0] * 2.0 ** -24 + 2.0 ** -20
    floor = 0.0
    if steps is not None:
        held = w * steps.T.repeat_interleave(group, 0)
        floor = 21 * k.shape[0] * 2.0 ** -30 * held.amax(-1, keepdim=True) + 7 * 2.0 ** -25 * held.sum(-1, keepdim=True)
    return out, spread, slack, floor


def bound(out, spread, slack, floor, weight):
    """What a kernel may be off: each weight by its roundings (`weight`, relative) and the scores' slack, the result by
    one BF16 rounding (and by half a step of the smallest BF16 number)."""
    rel = (1 + weight) * (1 + slack) - 1
    return U * out.abs() + (1 + U) * ((rel + slack) * spread + floor) + 2.0 ** -134


def assert_within(got, want, most, what=""):
    off = (got.double().cpu() - want.cpu()).abs()
    most = most.cpu()
    bad = ~(off <= most)
    assert not bad.any(), (what, int(bad.sum()), float((off - most)[bad].max()), bad.nonzero()[:4].tolist())

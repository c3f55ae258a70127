"""Attention over the 8-bit cache where magnitudes differ widely inside a sequence, against float64.

The tolerance of an output element follows from the formula and the number formats, per row, from the keys
that the row sees and nothing else.  With p the exact weights, A = sum_j p_j |v_j| and W = max_j p_j |vs_j|:
  * the score of key j is off by at most d_j (in natural units, all terms times the softmax scale):
    2^-18.8 sum_d |q_d k_jd|: roundings of q (a term split of 22 bits at least), of the scale, of at most
       16 accumulation steps that may truncate, and of the sum's factors;
    2^-30 max|q| sum_d |k_jd|: no element of q is held finer than 2^-30 of the row's largest by either kernel;
    2^-23 max_i sum_d |q_d k_id|: the difference to the running maximum is rounded;
    with 2^-21 for exp2 and the factors after it, a weight is off by the factor 1 + 2 d_j + 2^-21 at most, and
    the output by sum_j p_j |v_j| (2 d_j + 2^-21) plus A times the mean of the same over p;
  * weights times value scales as two fp16 terms 2^-21 A, 16 accumulation steps of a block 2^-19 A, the running
    sums in fp32 (256 + n / 64) 2^-24 A for n keys;
  * a weight's absolute floor: fp16 numbers are at least 2^-25 apart from their rounding and the unit keeps the
    row's largest weight within 2^9 of 2^10, so no weight is held finer than 2^-26 W: 2^-26 W sum_j |code_j|.
"""
import math

import pytest
import torch

from test_gpu_cache import Setup, compare, dev

pytestmark = pytest.mark.gpu


def exact(s, q, heads, scale):
    """Causal outputs and their tolerances, float64 [rows, heads * dim]; a key that a row does not see takes no
    part in either, whatever it holds."""
    out = torch.zeros(s.rows, heads, s.dim, dtype=torch.float64, device=dev())
    tol = torch.zeros_like(out)
    group, row = heads // s.kv, 0
    for b, (new, n) in enumerate(zip(s.news, s.lengths)):
        k, v = s.held(b)
        page, slot = s.where(b)
        codes, vs = s.cache.values[page, :, slot].double().abs(), s.cache.value_scales[page, :, slot].double().abs()
        qb = q[row:row + new].double().view(new, s.kv, group, s.dim)
        for i in range(new):
            seen = max(0, n - new + i + 1)
            if seen == 0:
                continue
            ki, vi = k[:seen], v[:seen]
            t = torch.einsum("hgd,jhd->hgj", qb[i], ki) * scale
            size = torch.einsum("hgd,jhd->hgj", qb[i].abs(), ki.abs()) * abs(scale)
            floor = qb[i].abs().amax(-1)[..., None] * ki.abs().sum(-1).t()[:, None] * abs(scale)
            p = torch.softmax(t, -1)
            d = 2 * (2.0 ** -18.8 * size + 2.0 ** -30 * floor + 2.0 ** -23 * size.amax(-1, keepdim=True)) + 2.0 ** -21
            a = torch.einsum("hgj,jhd->hgd", p, vi.abs())
            w = (p * vs[:seen].t()[:, None]).amax(-1)
            e = torch.einsum("hgj,jhd->hgd", p * d, vi.abs()) + a * (p * d).sum(-1, keepdim=True)
            e += a * (2.0 ** -21 + 2.0 ** -19 + (256 + seen / 64) * 2.0 ** -24)
            e += 2.0 ** -26 * w[..., None] * codes[:seen].sum(0)[:, None]
            out[row + i] = torch.einsum("hgj,jhd->hgd", p, vi).reshape(heads, s.dim)
            tol[row + i] = e.reshape(heads, s.dim)
        row += new
    return out.view(s.rows, -1), tol.view(s.rows, -1)


def run(s, q, scale, **kw):
    got = s.pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, scale, max_new=max(s.news), **kw)
    s.pkg.session.get_session(dev()).sync()
    return got


@pytest.mark.parametrize("share", [0.4, 1.0])
@pytest.mark.parametrize("new", [1, 3, 8, 200])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_of_either_sign(pkg, new, dim, share):
    """k and v are scale * code: a pool of the caller's may hold negative scales."""
    s = Setup(pkg, [new], [500], 2, dim, 16, seed=new + dim)
    q = torch.randn(new, 8 * dim, device=dev(), generator=s.g)
    for t in (s.cache.key_scales, s.cache.value_scales):
        t[torch.rand(t.shape, device=dev(), generator=s.g) < share] *= -1
    want, tol = exact(s, q, 8, 1 / math.sqrt(dim))
    compare(run(s, q, None), want, tol, new)

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


# ---- value scales ---------------------------------------------------------------------------------


@pytest.mark.parametrize("power", [12, 20, 40, 66, 120])
@pytest.mark.parametrize("new,heads,kv,dim", [(8, 1, 1, 128), (8, 4, 2, 64), (5, 2, 1, 128), (200, 4, 2, 128), (200, 2, 2, 64), (3, 40, 1, 128)])
def test_a_token_that_a_row_does_not_see_leaves_its_result_alone(pkg, new, heads, kv, dim, power):
    """The value scales of later new tokens are 2^power times the others."""
    n = 330
    s = Setup(pkg, [new], [n], kv, dim, 16, seed=power + new)
    q = torch.randn(new, heads * dim, device=dev(), generator=s.g)
    page, slot = s.where(0)
    for back in {1, max(1, new // 2)}:  # tokens n - back .. n - 1
        s.cache.value_scales[page[n - back], :, slot[n - back]] *= 2.0 ** power
    want, tol = exact(s, q, heads, 1 / math.sqrt(dim))
    compare(run(s, q, None), want, tol, new)


@pytest.mark.parametrize("value", [math.inf, 3e38])
@pytest.mark.parametrize("new", [8, 200])
def test_the_largest_and_infinite_scales_stay_with_the_rows_that_see_them(pkg, new, value):
    n, dim = 330, 128
    s = Setup(pkg, [new], [n], 1, dim, 64, seed=new)
    q = torch.randn(new, 2 * dim, device=dev(), generator=s.g)
    want, tol = exact(s, q, 2, 1 / math.sqrt(dim))
    page, slot = s.where(0)
    bad = n - new // 2
    s.cache.value_scales[page[bad], 0, slot[bad]] = value
    compare(run(s, q, None), want, tol, bad - (n - new))


@pytest.mark.parametrize("power,below", [(20, 127), (40, 127), (30, 21), (12, 9), (66, 40), (100, 75)])
@pytest.mark.parametrize("new,heads,kv,dim", [(1, 4, 1, 128), (1, 16, 2, 64), (8, 2, 2, 128), (16, 2, 2, 64), (200, 2, 1, 64), (150, 2, 2, 128)])
def test_a_token_of_small_weight_and_large_values(pkg, new, heads, kv, dim, power, below):
    """Tokens that every row sees with a score `below` under the others (in natural units, about) and value scales
    2^power times theirs: from no share in the result to most of it.  They lie in the first block, in the middle
    and in the last."""
    n = 700
    s = Setup(pkg, [new], [n], kv, dim, 32, seed=power + new + dim)
    q = torch.randn(new, heads * dim, device=dev(), generator=s.g)
    q.view(new, heads, dim)[:, :, 0] = 8.0
    page, slot = s.where(0)
    for pos in (5, 300, n - new):
        s.cache.keys[page[pos], :, slot[pos]] = 0
        s.cache.keys[page[pos], :, slot[pos], 0] = -127
        s.cache.key_scales[page[pos], :, slot[pos]] = below / 127
        s.cache.value_scales[page[pos], :, slot[pos]] *= 2.0 ** power
    want, tol = exact(s, q, heads, 0.125)
    compare(run(s, q, 0.125), want, tol, new)


@pytest.mark.parametrize("new", [1, 8, 200])
@pytest.mark.parametrize("dim", [64, 128])
def test_value_scales_spread_over_many_powers(pkg, new, dim):
    """No two tokens alike: scales over 60 powers of two in three sequences, one of them within one page, and zero
    scales among them."""
    s = Setup(pkg, [new, new, new], [700, 300, new + 3], 2, dim, 16, seed=new)
    q = torch.randn(s.rows, 4 * dim, device=dev(), generator=s.g)
    s.cache.value_scales *= torch.exp2(torch.randint(-30, 31, s.cache.value_scales.shape, device=dev(), generator=s.g).float())
    s.cache.value_scales[torch.rand(s.cache.value_scales.shape, device=dev(), generator=s.g) < 0.1] = 0.0
    want, tol = exact(s, q, 4, 1 / math.sqrt(dim))
    compare(run(s, q, None), want, tol, s.rows)


@pytest.mark.parametrize("below", [14, 30, 50])
@pytest.mark.parametrize("new,heads,kv,dim", [(1, 4, 1, 128), (16, 1, 1, 64), (200, 2, 1, 64), (150, 2, 2, 128), (2, 20, 1, 128)])
def test_a_token_with_most_of_the_weight_and_no_values(pkg, new, heads, kv, dim, below):
    """One token scores `below` above the others (in natural units, about), and its values are zeros: what is left of
    the others is all of the result."""
    n = 500
    s = Setup(pkg, [new], [n], kv, dim, 32, seed=below + new)
    q = torch.randn(new, heads * dim, device=dev(), generator=s.g)
    q.view(new, heads, dim)[:, :, 0] = 8.0
    page, slot = s.where(0)
    for pos in (0, 270):
        s.cache.keys[page[pos], :, slot[pos]] = 0
        s.cache.keys[page[pos], :, slot[pos], 0] = 127
        s.cache.key_scales[page[pos], :, slot[pos]] = below / 127
        s.cache.values[page[pos], :, slot[pos]] = 0
        s.cache.value_scales[page[pos], :, slot[pos]] = 0
    want, tol = exact(s, q, heads, 0.125)
    compare(run(s, q, 0.125), want, tol, new)


@pytest.mark.parametrize("news,lengths", [([1, 1], [9000, 5000]), ([160], [6000])])
def test_pieces_of_cut_items_with_scales_that_differ(pkg, news, lengths):
    """Long sequences, whose keys several CTAs share: each piece has a range of scales of its own."""
    s = Setup(pkg, news, lengths, 1, 128, 64, seed=3)
    q = torch.randn(s.rows, 2 * 128, device=dev(), generator=s.g)
    page, slot = s.where(0)
    step = torch.arange(len(page), device=dev()) // 1000
    s.cache.value_scales[page, 0, slot] *= torch.exp2(10.0 * step)
    want, tol = exact(s, q, 2, 1 / math.sqrt(128))
    compare(run(s, q, None), want, tol, s.rows)


# ---- q --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("large", [100.0, 1000.0, 16384.0])
@pytest.mark.parametrize("new,heads,kv,dim", [(1, 8, 1, 128), (1, 8, 2, 64), (2, 8, 1, 128), (16, 1, 1, 64), (60, 2, 1, 128), (60, 4, 2, 64)])
@pytest.mark.parametrize("n", [64, 90])
def test_an_outlier_channel_of_q_on_which_keys_are_small(pkg, new, heads, kv, dim, large, n):
    """One channel of q is `large` times the others, the keys are 0 on it (or one code for a few): the other channels
    decide the scores and have to keep their bits."""
    s = Setup(pkg, [new] * 12, [n] * 12, kv, dim, 16, seed=int(large) + new)
    q = torch.randn(s.rows, heads * dim, device=dev(), generator=s.g)
    q.view(s.rows, heads, dim)[:, :, 7] *= large
    s.cache.keys[..., 7] = 0
    for b in range(6):
        page, slot = s.where(b)
        s.cache.keys[page[1::3], :, slot[1::3], 7] = 1
    want, tol = exact(s, q, heads, 1 / math.sqrt(dim))
    compare(run(s, q, None), want, tol, s.rows)

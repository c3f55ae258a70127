"""The paged 8-bit cache and attention over it, on the GPU against 64-bit arithmetic.

Codes, scales and what is read back are exact by definition and compared for equality.  Attention's
tolerance is derived per output element.  With A = sum_j p_j |v_j| (p the exact weights):
  * a score's error is at most dS = c * scale * sum_d |q_d k_jd|, c = 2^-22 (q as the sum of two
    11-bit terms) + 2^-23 for each of at most 16 accumulation steps that may truncate + 4 * 2^-24
    (scales applied in fp32) < 2^-18.8; weights are off by a factor e^(2 dS) at most, so the
    output by 2 dS A;
  * weights times value scales as two 11-bit terms, exp2 and the scalings: 2^-20 A; the product's 16
    accumulation steps of a block 2^-19 A;
  * the running sums over blocks and the sum of the weights, in fp32: (256 + n / 64) 2^-24 A for n
    keys (a thread adds at most 128 weights of a block one after another, and blocks one by one);
  * fp16 ends: a weight is held in units that put the largest value scale of its block, rounded up to
    a power of two E <= 2 max vs, times the largest p at 2^10 or more, and the low term's spacing never
    falls below 2^-24, so a weight has an absolute error of at most 2^-25 2^-10 E however small it
    is.  With |vc| <= 127 and a sum of weights of at least 1 that is 2^-35 * 2 max vs * 127 per
    key, n times: the only term that does not shrink with A (it shows where one key takes nearly all the
    weight and its value is exactly 0)."""
import math

import numpy as np
import pytest
import torch

from test_gpu_s8_linear import reference_codes

pytestmark = pytest.mark.gpu
C_SCORE = 2.0 ** -18.8


def dev():
    return torch.device("cuda:0")


class Setup:
    """A pool full of plausible values, sequences spread over shuffled pages."""

    def __init__(self, pkg, news, lengths, kv_heads, dim, page, seed=0, pad_rows=0, spare=3):
        g = torch.Generator(device=dev()).manual_seed(seed)
        self.g, self.pkg = g, pkg
        self.news, self.lengths, self.page, self.kv, self.dim = news, lengths, page, kv_heads, dim
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + spare
        order = torch.randperm(pages, device=dev(), generator=g).to(torch.int32)
        self.table = torch.full((len(news), max(need + [1]) + 1), 0, dtype=torch.int32, device=dev())
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.rows = sum(news) + pad_rows
        self.starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device=dev())
        self.lens = torch.tensor(lengths, dtype=torch.int32, device=dev())
        shape = (pages, kv_heads, page, dim)
        codes = [(torch.randn(shape, device=dev(), generator=g) * 42).round_().clamp_(-127, 127).to(torch.int8) for _ in "kv"]
        scales = [torch.exp(0.3 * torch.randn(shape[:3], device=dev(), generator=g)) / 42 for _ in "kv"]
        self.cache = pkg.cache.PagedCache(codes[0], scales[0], codes[1], scales[1])

    def where(self, b, n=None):
        """(pages, slots) of the first n positions of sequence b."""
        pos = torch.arange(self.lengths[b] if n is None else n, device=dev())
        return self.table[b, pos // self.page].long(), pos % self.page

    def held(self, b):
        """Dequantized keys and values of sequence b, float64 [length, kv, dim]."""
        page, slot = self.where(b)
        c = self.cache
        return tuple(x[page, :, slot].double() * s[page, :, slot].double()[..., None]
                     for x, s in ((c.keys, c.key_scales), (c.values, c.value_scales)))

    def unused(self):
        """Mask over [pages, page] of slots that belong to no sequence."""
        free = torch.ones(self.cache.pages, self.page, dtype=torch.bool, device=dev())
        for b in range(len(self.news)):
            page, slot = self.where(b)
            free[page, slot] = False
        return free


def expected(s, q, heads, scale, causal):
    """Exact outputs and their tolerances, float64 [rows, heads * dim]."""
    out = torch.zeros(s.rows, heads, s.dim, dtype=torch.float64, device=dev())
    tol = torch.zeros_like(out)
    group = heads // s.kv
    row = 0
    for b, (new, n) in enumerate(zip(s.news, s.lengths)):
        k, v = s.held(b)
        qb = q[row:row + new].double().view(new, s.kv, group, s.dim)
        if new and n:
            t = torch.einsum("ihgd,jhd->hgij", qb, k) * scale
            size = torch.einsum("ihgd,jhd->hgij", qb.abs(), k.abs()) * abs(scale)
            if causal:
                last = torch.arange(new, device=dev()) + n - new
                hide = torch.arange(n, device=dev())[None] > last[:, None]
                t = t.masked_fill(hide, -math.inf)
                size = size.masked_fill(hide, 0.0)
            p = torch.softmax(t, -1)
            empty = torch.isneginf(t).all(-1, keepdim=True)
            p = torch.where(empty, 0.0, p)
            out[row:row + new] = torch.einsum("hgij,jhd->ihgd", p, v).reshape(new, heads, s.dim)
            a = torch.einsum("hgij,jhd->ihgd", p, v.abs())
            ds = size.amax(-1).permute(2, 0, 1)[..., None] * C_SCORE
            page, slot = s.where(b)
            top = s.cache.value_scales[page, :, slot].double().amax()
            end = n * 2.0 ** -34 * 127 * top
            tol[row:row + new] = (a * (2 * ds + 2.0 ** -20 + 2.0 ** -19 + (256 + n / 64) * 2.0 ** -24) + end).reshape(new, heads, s.dim)
        row += new
    return out.view(s.rows, -1), tol.view(s.rows, -1)


def compare(got, want, tol, rows):
    off = (got[:rows].double() - want[:rows]).abs()
    bad = ~(off <= tol[:rows])
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst "
                                 f"{float((off / tol[:rows].clamp_min(1e-30)).max()):.3g} of the tolerance")


# ---- write and read back ------------------------------------------------------------------------


@pytest.mark.parametrize("news,lengths,kv,dim,page", [
    ([1], [1], 1, 64, 1), ([1] * 9, [3, 64, 65, 1, 128, 200, 7, 8, 9], 8, 128, 64), ([5, 0, 130, 1], [5, 0, 400, 77], 12, 64, 16),
    ([33, 2], [33, 1000], 3, 128, 1024), ([300], [300], 5, 64, 8), ([1000, 500], [1003, 500], 2, 128, 32)])
def test_append_writes_the_definition_and_read_gives_it_back(pkg, news, lengths, kv, dim, page):
    s = Setup(pkg, news, lengths, kv, dim, page, seed=len(news))
    width = kv * dim
    packed = torch.randn(s.rows, 3 * width + 4, device=dev(), generator=s.g) * 3
    packed[0, :dim] = 0.0
    if s.rows > 3:
        packed[2, 5], packed[3, width + 70] = math.nan, math.inf
    k, v = packed[:, :width], packed[:, width:2 * width]  # column slices, as of a packed projection
    before = [t.clone() for t in (s.cache.keys, s.cache.key_scales, s.cache.values, s.cache.value_scales)]
    pkg.cache.append(s.cache, k, v, s.starts, s.lens, s.table)
    want = [t.clone() for t in before]
    row = 0
    for b, (new, n) in enumerate(zip(news, lengths)):
        page_, slot = s.where(b)
        page_, slot = page_[n - new:], slot[n - new:]
        for x, i in ((k, 0), (v, 2)):
            c, sc = reference_codes(x[row:row + new].reshape(-1, dim))if new else (np.zeros((0, dim), np.int8), np.zeros(0, np.float32))
            want[i][page_, :, slot] = torch.from_numpy(c).to(dev()).view(new, kv, dim)
            want[i + 1][page_, :, slot] = torch.from_numpy(sc).to(dev()).view(new, kv)
        row += new
    for got, w in zip((s.cache.keys, s.cache.key_scales, s.cache.values, s.cache.value_scales), want):
        np.testing.assert_array_equal(got.cpu().numpy(), w.cpu().numpy())  # untouched slots among them
    rk, rv = pkg.cache.read(s.cache, s.starts, s.lens, s.table, s.rows)
    row = 0
    for b, (new, n) in enumerate(zip(news, lengths)):
        page_, slot = s.where(b)
        page_, slot = page_[n - new:], slot[n - new:]
        for got, c, sc in ((rk, s.cache.keys, s.cache.key_scales), (rv, s.cache.values, s.cache.value_scales)):
            np.testing.assert_array_equal(got[row:row + new].cpu().numpy(),
                                          (c[page_, :, slot].float() * sc[page_, :, slot][..., None]).reshape(new, width).cpu().numpy())
        row += new
    pkg.session.get_session(dev()).sync()


def test_read_of_whole_sequences_leaves_padding_rows(pkg):
    s = Setup(pkg, [0, 0, 0], [70, 0, 130], 2, 64, 32, seed=3)
    starts = torch.tensor([0, 70, 70, 200], dtype=torch.int32, device=dev())
    out = tuple(torch.full((210, 2 * 64 + 4), -7.0, device=dev())[:, :128] for _ in "kv")
    k, v = pkg.cache.read(s.cache, starts, s.lens, s.table, 210, out=out)
    assert k.data_ptr() == out[0].data_ptr()
    for b, lo in ((0, 0), (2, 70)):
        hk, hv = s.held(b)
        n = s.lengths[b]
        assert torch.equal(k[lo:lo + n].double(), hk.float().double().view(n, -1)) or \
            torch.allclose(k[lo:lo + n].double(), hk.view(n, -1), rtol=2.0 ** -24, atol=0)
        assert torch.allclose(v[lo:lo + n].double(), hv.view(n, -1), rtol=2.0 ** -24, atol=0)
    assert bool((k[200:] == -7).all()) and bool((v[200:] == -7).all())


def test_tokens_without_a_position_are_skipped(pkg):
    """More new tokens than the sequence is long: the first ones have no position."""
    s = Setup(pkg, [5, 2], [3, 2], 2, 64, 16, seed=4)
    k, v = (torch.randn(7, 128, device=dev(), generator=s.g) for _ in "kv")
    free = s.unused()
    before = s.cache.keys.clone()
    pkg.cache.append(s.cache, k, v, s.starts, s.lens, s.table)
    rk, _ = pkg.cache.read(s.cache, s.starts, s.lens, s.table, 7)
    assert bool((rk[:2] == 0).all())
    assert bool(((rk[2:] - k[2:]).abs() <= k[2:].abs().amax() / 127).all())
    keep = free[:, None, :, None].expand_as(before)
    assert torch.equal(s.cache.keys[keep], before[keep])
    pkg.session.get_session(dev()).sync()


# ---- attention ----------------------------------------------------------------------------------

CASES = [
    # news, lengths, heads, kv_heads, dim, page, causal
    ([1], [1], 1, 1, 64, 16, True),
    ([1], [100], 12, 12, 64, 16, True),
    ([1], [129], 8, 8, 128, 64, True),
    ([1, 1, 1, 1, 1], [1, 127, 128, 129, 700], 8, 2, 128, 64, True),
    ([1] * 6, [5, 1000, 0, 333, 64, 2049], 16, 2, 64, 8, True),
    ([2, 1, 3], [300, 2, 3], 5, 1, 128, 32, True),
    ([4, 3], [200, 4000], 8, 2, 128, 128, True),
    ([1, 1], [9000, 6000], 6, 2, 64, 1024, True),
    ([16, 15, 17], [16, 500, 129], 3, 3, 64, 16, True),
    ([1], [600], 32, 1, 128, 64, True),
    ([2], [3000], 20, 1, 64, 64, True),
    ([130], [130], 4, 4, 64, 16, True),
    ([257, 1, 64], [257, 300, 1000], 4, 2, 128, 32, True),
    ([100, 7], [900, 2000], 21, 3, 64, 1, True),
    ([300], [500], 7, 1, 128, 256, True),
    ([600, 1, 5, 0, 40], [700, 1500, 5, 30, 2000], 8, 4, 64, 64, True),
    ([50, 1, 300], [50, 400, 600], 4, 2, 128, 16, False),
    ([1, 3], [130, 70], 8, 8, 64, 16, False),
    ([1000], [1000], 2, 2, 128, 64, True),
]


@pytest.mark.parametrize("news,lengths,heads,kv,dim,page,causal", CASES)
def test_attention(pkg, news, lengths, heads, kv, dim, page, causal):
    s = Setup(pkg, news, lengths, kv, dim, page, seed=sum(lengths) + heads)
    q = torch.randn(s.rows, heads * dim, device=dev(), generator=s.g)
    scale = 1 / math.sqrt(dim)
    want, tol = expected(s, q, heads, scale, causal)
    for bounds in ({}, {"max_new": max(news), "max_length": max(lengths)}):
        got = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, causal=causal, **bounds)
        compare(got, want, tol, s.rows)
    again = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, causal=causal, **bounds)
    assert torch.equal(got, again)
    pkg.session.get_session(dev()).sync()


@pytest.mark.parametrize("news,lengths,heads", [([1, 1], [90, 300], 4), ([40, 200], [90, 300], 2)])
def test_strided_rows_padding_and_large_scores(pkg, news, lengths, heads):
    """Column slices of a packed projection, padding rows left alone, scores up to about 100 (one key
    takes all the weight) and a scale that is not the default."""
    dim = 128
    s = Setup(pkg, news, lengths, 2, dim, 32, seed=8, pad_rows=3)
    packed = torch.randn(s.rows, heads * dim + 260, device=dev(), generator=s.g) * 10
    q = packed[:, 4:4 + heads * dim]
    out = torch.full((s.rows, heads * dim + 8), 5.0, device=dev())[:, :heads * dim]
    want, tol = expected(s, q, heads, 0.1, True)
    got = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, 0.1, out=out)
    compare(got, want, tol, sum(news))
    assert bool((got[sum(news):] == 5.0).all())


@pytest.mark.parametrize("news,lengths", [([1, 1, 1], [40, 129, 500]), ([64, 1, 200], [130, 5, 333]), ([5, 2], [5, 200])])
def test_garbage_outside_the_sequences_is_not_seen(pkg, news, lengths):
    """Slots behind a sequence's end hold NaN scales and arbitrary codes, unused table entries
    nonsense: nothing of it may reach the result."""
    s = Setup(pkg, news, lengths, 2, 64, 16, seed=5)
    q = torch.randn(s.rows, 4 * 64, device=dev(), generator=s.g)
    want, tol = expected(s, q, 4, 0.125, True)
    free = s.unused()[:, None, :].expand_as(s.cache.key_scales)
    for t in (s.cache.key_scales, s.cache.value_scales):
        t[free] = math.nan
    for b, n in enumerate(lengths):
        s.table[b, -(-n // 16):] = -12345
    got = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table)
    compare(got, want, tol, s.rows)
    pkg.session.get_session(dev()).sync()


@pytest.mark.parametrize("new", [8, 200])
@pytest.mark.parametrize("what", ["key", "value"])
def test_non_finite_tokens_reach_only_the_rows_that_see_them(pkg, new, what):
    n = 300
    s = Setup(pkg, [new], [n], 1, 128, 64, seed=6)
    q = torch.randn(new, 2 * 128, device=dev(), generator=s.g)
    bad = n - new // 2  # seen by the later half of the rows only
    page, slot = s.where(0)
    want, tol = expected(s, q, 2, 1 / math.sqrt(128), True)
    (s.cache.key_scales if what == "key" else s.cache.value_scales)[page[bad], 0, slot[bad]] = math.nan
    got = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table)
    first = bad - (n - new)
    compare(got, want, tol, first)
    assert bool(got[first:].isnan().all())


def test_rows_that_see_nothing_are_zero(pkg):
    s = Setup(pkg, [4, 1, 150, 3], [2, 0, 100, 3], 2, 64, 16, seed=7)
    q = torch.randn(s.rows, 4 * 64, device=dev(), generator=s.g)
    want, tol = expected(s, q, 4, 0.125, True)
    got = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table)
    compare(got, want, tol, s.rows)
    assert bool((got[:2] == 0).all()) and bool((got[4] == 0).all()) and bool((got[5:55] == 0).all())


@pytest.mark.parametrize("new", [1, 100])
def test_bad_pages_and_sequences_are_reported_and_touch_nothing_else(pkg, new):
    ex = pkg.exceptions
    news, lengths = [new, new, new], [200, 150, 260]
    s = Setup(pkg, news, lengths, 2, 64, 16, seed=9)
    q = torch.randn(s.rows, 4 * 64, device=dev(), generator=s.g)
    want, tol = expected(s, q, 4, 0.125, True)
    sess = pkg.session.get_session(dev())
    sess.sync()
    # a page of the second sequence that does not exist
    for page in (-1, s.cache.pages, 2 ** 31 - 1):
        table = s.table.clone()
        table[1, 3] = page
        got = pkg.cache.attention(s.cache, q, s.starts, s.lens, table)
        with pytest.raises(ex.InvalidArgumentError, match="0x20"):
            sess.sync()
        compare(got[:new], want[:new], tol[:new], new)
        compare(got[2 * new:], want[2 * new:], tol[2 * new:], new)
        assert bool(got[new:2 * new].isnan().all())
        k, v = (torch.randn(s.rows, 128, device=dev()) for _ in "kv")
        table[1, :] = page
        keep = s.cache.keys.clone(), s.cache.values.clone()
        mine = [s.where(b) for b in (0, 2)]
        pkg.cache.append(s.cache, k, v, s.starts, s.lens, table)
        with pytest.raises(ex.InvalidArgumentError, match="0x20"):
            sess.sync()
        for t, old in zip((s.cache.keys, s.cache.values), keep):
            for pg, sl in mine:
                old[pg, :, sl] = t[pg, :, sl]
            assert torch.equal(t, old)
            t.copy_(old)
        rk, _ = pkg.cache.read(s.cache, s.starts, s.lens, table, s.rows)
        with pytest.raises(ex.InvalidArgumentError, match="0x20"):
            sess.sync()
        assert bool((rk[new:2 * new] == 0).all())
        want, tol = expected(s, q, 4, 0.125, True)  # (the first and third sequences were rewritten)
    # a length beyond the table, a negative one, rows out of order or out of range
    out = torch.full((s.rows, 256), 3.0, device=dev())
    for lens, starts in (([200, 10 ** 6, 260], None), ([200, -5, 260], None), (None, [0, 2 * new, new, 3 * new]),
                         (None, [0, new, 4 * new + 1, 5 * new]), (None, [-3, new, 2 * new, 3 * new])):
        l = s.lens if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev())
        st = s.starts if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev())
        got = pkg.cache.attention(s.cache, q, st, l, s.table, out=out.clone())
        with pytest.raises(ex.InvalidArgumentError, match="0x10"):
            sess.sync()
        if starts is None:
            compare(got[:new], want[:new], tol[:new], new)
            compare(got[2 * new:], want[2 * new:], tol[2 * new:], new)
            assert bool((got[new:2 * new] == 3.0).all())


def test_sequences_beyond_the_stated_bounds_are_reported(pkg):
    ex = pkg.exceptions
    s = Setup(pkg, [3, 40, 1], [50, 80, 400], 1, 64, 16, seed=10)
    q = torch.randn(s.rows, 64, device=dev(), generator=s.g)
    want, tol = expected(s, q, 1, 0.125, True)
    sess = pkg.session.get_session(dev())
    out = torch.full((s.rows, 64), 3.0, device=dev())
    got = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, max_new=4, max_length=100, out=out)
    with pytest.raises(ex.InvalidArgumentError, match="0x10"):
        sess.sync()
    compare(got, want, tol, 3)
    assert bool((got[3:] == 3.0).all())


def test_pool_beyond_four_gigabytes(pkg):
    """Page and slot offsets pass 32 bits."""
    pages, kv, page, dim = 70000, 8, 64, 128
    cache = pkg.cache.PagedCache.empty(pages, page, kv, dim, dev())
    n = 200
    table = torch.tensor([[pages - 1, 3, pages - 2, 40000]], dtype=torch.int32, device=dev())
    g = torch.Generator(device=dev()).manual_seed(1)
    k, v = (torch.randn(n, kv * dim, device=dev(), generator=g) for _ in "kv")
    starts, lens = (torch.tensor(t, dtype=torch.int32, device=dev()) for t in ([0, n], [n]))
    pkg.cache.append(cache, k, v, starts, lens, table)
    rk, rv = pkg.cache.read(cache, starts, lens, table, n)
    for x, r in ((k, rk), (v, rv)):
        c, sc = reference_codes(x.view(-1, dim))
        np.testing.assert_array_equal(r.view(-1, dim).cpu().numpy(), c.astype(np.float32) * sc[:, None])
    for new in (1, 150):
        q = torch.randn(new, 16 * dim, device=dev(), generator=g)
        st = torch.tensor([0, new], dtype=torch.int32, device=dev())
        got = pkg.cache.attention(cache, q, st, lens, table)
        s = Setup.__new__(Setup)
        s.rows, s.news, s.lengths, s.kv, s.dim, s.page, s.cache, s.table = new, [new], [n], kv, dim, page, cache, table
        s.held = lambda b: (rk.double().view(n, kv, dim), rv.double().view(n, kv, dim))
        want, tol = expected(s, q, 16, 1 / math.sqrt(dim), True)
        compare(got, want, tol * 2, new)  # (the values read back carry one more rounding, 2^-24)
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("most", [1, 64])
def test_a_captured_step_follows_the_sequences(pkg, most):
    """One graph, replayed with other lengths, tables and queries: nothing of the capture's
    sequences may be left in it.  A second graph on the same session shares the workspace."""
    kv, heads, dim, page = 2, 8, 64, 16
    news = [most, 1, most]
    s = Setup(pkg, news, [200, 400, 300], kv, dim, page, seed=11)
    q = torch.randn(s.rows, heads * dim, device=dev(), generator=s.g)
    k, v = (torch.randn(s.rows, kv * dim, device=dev(), generator=s.g) for _ in "kv")

    def step():
        pkg.cache.append(s.cache, k, v, s.starts, s.lens, s.table)
        return pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, max_new=most)

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for lengths in ([200, 400, 300], [most, 390, 150], [201, 1, 299]):
        s.lengths = lengths
        s.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        for t in (q, k, v):
            t.normal_(generator=s.g)
        for g, out in zip(graphs, outs):
            out.fill_(math.nan)
            g.replay()
        want, tol = expected(s, q, heads, 0.125, True)
        for out in outs:
            compare(out, want, tol, s.rows)
    pkg.session.get_session(dev()).sync()


def test_many_sequences(pkg):
    """More sequences than a CTA has threads, most of them short, some empty, with and without new tokens."""
    rng = np.random.default_rng(5)
    news = [int(rng.integers(0, 3)) for _ in range(1100)]
    lengths = [n + int(rng.integers(0, 40)) for n in news]
    news[700], lengths[700] = 60, 700
    lengths[1099] = 3000
    s = Setup(pkg, news, lengths, 2, 64, 16, seed=13)
    q = torch.randn(s.rows, 8 * 64, device=dev(), generator=s.g)
    want, tol = expected(s, q, 8, 0.125, True)
    compare(pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table), want, tol, s.rows)
    k, v = (torch.randn(s.rows, 128, device=dev(), generator=s.g) for _ in "kv")
    pkg.cache.append(s.cache, k, v, s.starts, s.lens, s.table)
    rk, rv = pkg.cache.read(s.cache, s.starts, s.lens, s.table, s.rows)
    for x, r in ((k, rk), (v, rv)):
        c, sc = reference_codes(x.view(-1, 64))
        np.testing.assert_array_equal(r.view(-1, 64).cpu().numpy(), c.astype(np.float32) * sc[:, None])
    pkg.session.get_session(dev()).sync()


def test_a_call_without_new_tokens_leaves_everything(pkg):
    s = Setup(pkg, [0, 0], [30, 500], 2, 64, 16, seed=14, pad_rows=5)
    q = torch.randn(5, 4 * 64, device=dev())
    for most in (1, 5):
        out = torch.full((5, 256), 2.0, device=dev())
        pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, max_new=most, out=out)
        assert bool((out == 2.0).all())
    before = s.cache.keys.clone()
    kv = torch.randn(5, 128, device=dev())
    pkg.cache.append(s.cache, kv, kv, s.starts, s.lens, s.table)
    assert torch.equal(s.cache.keys, before)
    pkg.session.get_session(dev()).sync()


def test_graphs_replayed_side_by_side(pkg):
    """Two captured calls with pieces in scratch, replayed on two streams at once."""
    setups, graphs, outs, wants = [], [], [], []
    for seed, news, lengths in ((20, [1, 1], [9000, 7000]), (21, [200], [6000]), (22, [1], [12000])):
        s = Setup(pkg, news, lengths, 2, 128, 64, seed=seed)
        q = torch.randn(s.rows, 8 * 128, device=dev(), generator=s.g)
        wants.append(pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, max_new=max(news)))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table, max_new=max(news)))
        setups.append((s, q))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        assert torch.equal(out, want)
    pkg.session.get_session(dev()).sync()


def test_side_streams(pkg):
    s = Setup(pkg, [1, 90, 2], [500, 300, 7], 2, 128, 16, seed=12)
    q = torch.randn(s.rows, 6 * 128, device=dev(), generator=s.g)
    want = pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append([pkg.cache.attention(s.cache, q, s.starts, s.lens, s.table) for _ in range(3)])
    torch.cuda.synchronize()
    for g in got:
        for t in g:
            assert torch.equal(t, want)


def test_decoder_block_of_the_operators_together(pkg):
    """x -> linear(Wqkv) -> append -> attention -> linear(Wo), a prompt and then single tokens,
    against the same chain in float64 with the codes of the device (which their own tests pin): each
    projection adds one rounding per product term, so 1e-5 normwise is ample for four operators."""
    q8, ch = pkg.quantization, pkg.cache
    heads, kv, dim, page, hidden = 8, 2, 64, 16, 512
    g = torch.Generator(device=dev()).manual_seed(2)
    wqkv, sqkv = q8.quantize_channels(torch.randn(hidden, (heads + 2 * kv) * dim, device=dev(), generator=g) * 0.05)
    wo, so = q8.quantize_channels(torch.randn(heads * dim, hidden, device=dev(), generator=g) * 0.05)
    cache = ch.PagedCache.empty(40, page, kv, dim, dev())
    table = torch.randperm(40, device=dev(), generator=g).to(torch.int32)[:30].view(2, 15).contiguous()
    lengths = [0, 0]
    for news in ([70, 33], [1, 1], [1, 1], [5, 1]):
        lengths = [a + b for a, b in zip(lengths, news)]
        rows = sum(news)
        starts = torch.tensor([0, news[0], rows], dtype=torch.int32, device=dev())
        lens = torch.tensor(lengths, dtype=torch.int32, device=dev())
        x = torch.randn(rows, hidden, device=dev(), generator=g)
        qkv = q8.linear(x, wqkv, sqkv)
        q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], dim=1)
        ch.append(cache, k, v, starts, lens, table)
        o = ch.attention(cache, q, starts, lens, table, max_new=max(news))
        y = q8.linear(o, wo, so)
        # the same in float64
        cx, sx = q8.quantize_tokens(x)
        want_qkv = (cx.double() * sx.double()[:, None]) @ (wqkv.double() * sqkv.double())
        assert float((qkv.double() - want_qkv).norm() / want_qkv.norm()) < 1e-6
        s = Setup.__new__(Setup)
        s.pkg, s.news, s.lengths, s.rows, s.kv, s.dim, s.page, s.cache, s.table = pkg, news, lengths, rows, kv, dim, page, cache, table
        want, tol = expected(s, q, heads, 0.125, True)
        compare(o, want, tol, rows)
        co, sco = q8.quantize_tokens(o)
        want_y = (co.double() * sco.double()[:, None]) @ (wo.double() * so.double())
        assert float((y.double() - want_y).norm() / want_y.norm()) < 1e-5
    pkg.session.get_session(dev()).sync()

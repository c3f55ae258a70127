"""The 8-bit linear layer (one scale per token and channel) on the GPU against 64-bit arithmetic.

Codes and scales are exact by definition (the exact quotient decides every rounding), so they are
compared for equality.  The product's int32 sums are exact; what rounds is sum -> fp32, times the row
scale, the fused multiply-add with column scale and bias: each at most 2^-24 relative to a term no
larger than |sum s w| + |bias|, hence 4 * 2^-24 of that, second-order terms included.  GELU multiplies
an incoming error by at most 1.13 and adds the rounding of erf and of two products: 8 * 2^-24 * |y|."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def reference_codes(x):
    """float32 [R, K] -> (codes, scales), the definition in float64 (whose quotient of two floats
    cannot land on a tie that the exact one misses: they differ by 2^-32 relative at least)."""
    x = x.detach().cpu().numpy()
    amax = np.abs(x).max(axis=-1)
    bad = ~np.isfinite(x).all(axis=-1)
    scales = (amax.astype(np.float64) / 127).astype(np.float32)
    scales[bad] = np.nan
    with np.errstate(all="ignore"):
        q = np.rint(x.astype(np.float64) / scales.astype(np.float64)[..., None])
    q[bad | (scales == 0)] = 0
    return np.clip(q, -127, 127).astype(np.int8), scales


def activations(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g))


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (1, 768), (7, 511), (5, 512), (6, 513), (9, 2048), (3, 2049),
                                       (130, 1000), (2, 8192), (3, 20003)])
def test_codes_and_scales_are_exact(pkg, rows, cols):
    x = activations(rows, cols, rows + cols)
    codes, scales = pkg.quantization.quantize_tokens(x.to(dev()))
    want, want_scales = reference_codes(x)
    assert codes.shape == (rows, cols) and codes.stride(0) % 16 == 0
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(codes.cpu().numpy(), want)


def test_codes_on_and_around_ties(pkg):
    """max 127 makes the scale exactly 1: k + 0.5 ties go to the even code, one ulp either side does not.
    Other maxima put quotients within an ulp of a tie without being one."""
    base = np.arange(-127, 127, dtype=np.float32) + np.float32(0.5)
    rows = [np.concatenate([[np.float32(127)], f]) for f in
            (base, np.nextafter(base, np.float32(1e9)), np.nextafter(base, np.float32(-1e9)))]
    rng = np.random.default_rng(3)
    for m in rng.uniform(0.1, 300, 40).astype(np.float32):
        s = np.float32(np.float64(m) / 127)
        near = (base.astype(np.float64) * np.float64(s)).astype(np.float32)
        near = np.where(np.abs(near) <= m, near, np.float32(0))
        rows.append(np.concatenate([[m], near]))
    x = torch.from_numpy(np.stack(rows).astype(np.float32))
    codes, scales = pkg.quantization.quantize_tokens(x.to(dev()))
    want, want_scales = reference_codes(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(codes.cpu().numpy(), want)


def test_zero_tiny_huge_and_non_finite_rows(pkg):
    x = activations(8, 100, 1)
    x[0] = 0
    x[1] *= 2.0 ** -140  # subnormal values and scale
    x[2] *= 2.0 ** -110
    x[3] *= 2.0 ** 115
    x[4, 7] = math.inf
    x[5, 99] = math.nan
    x[6, 0] = -math.inf
    x[7] = torch.tensor([2.0 ** -149] * 99 + [60 * 2.0 ** -149])  # the scale rounds to 0
    codes, scales = pkg.quantization.quantize_tokens(x.to(dev()))
    want, want_scales = reference_codes(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(codes.cpu().numpy(), want)


def test_quantize_takes_strided_and_batched_rows(pkg):
    wide = activations(12, 900, 2).to(dev())
    for x in (wide[:, 100:700], wide[:, 3:501], wide[::2, :64], wide.view(3, 4, 900)[:, :, 5:55], wide.view(12, 1, 900)):
        codes, scales = pkg.quantization.quantize_tokens(x)
        want, want_scales = reference_codes(x.reshape(-1, x.shape[-1]))
        np.testing.assert_array_equal(codes.reshape(-1, x.shape[-1]).cpu().numpy(), want)
        np.testing.assert_array_equal(scales.reshape(-1).cpu().numpy(), want_scales)
        assert scales.shape == x.shape[:-1]


def operands(m, k, n, seed, pad=True):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    b = torch.randint(-127, 128, (k, n), generator=g, dtype=torch.int8)
    sa = torch.exp(torch.randn(m, generator=g)) * 0.01
    sb = torch.exp(torch.randn(n, generator=g)) * 0.01
    bias = torch.randn(n, generator=g)
    out = []
    for t in (a, b):
        if pad:
            w = torch.zeros(t.shape[0], (t.shape[1] + 15) // 16 * 16, dtype=torch.int8)
            w[:, :t.shape[1]] = t
            out.append(w.to(dev())[:, :t.shape[1]])
        else:
            out.append(t.to(dev()))
    return out[0], sa.to(dev()), out[1], sb.to(dev()), bias.to(dev())


def check(got, a, sa, b, sb, bias, gelu=False):
    sums = (a.double() @ b.double())
    y = sums * sa.double()[:, None] * sb.double()
    tol = 4 * EPS * (y.abs() + (bias.double().abs() if bias is not None else 0))
    if bias is not None:
        y = y + bias.double()
    if gelu:
        tol = 1.13 * tol + 8 * EPS * y.abs()
        y = torch.special.ndtr(y) * y
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol.clamp_min(1e-300)).max())} of the tolerance"


SHAPES = [(1, 16, 16), (1, 768, 768), (3, 1003, 130), (16, 512, 2050), (77, 129, 257), (128, 128, 128), (129, 640, 1001),
          (300, 2000, 96), (513, 384, 777), (257, 4096, 512)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("path", ["auto", "umma", "umma2", "simt"])
def test_product(pkg, m, k, n, path):
    a, sa, b, sb, bias = operands(m, k, n, m + k + n)
    check(pkg.quantization.matmul_scaled(a, sa, b, sb, path=path), a, sa, b, sb, None)
    check(pkg.quantization.matmul_scaled(a, sa, b, sb, bias, path=path), a, sa, b, sb, bias)
    check(pkg.quantization.matmul_scaled(a, sa, b, sb, bias, activation="gelu", path=path), a, sa, b, sb, bias, True)
    pkg.session.get_session(dev()).sync()


@pytest.mark.parametrize("m,k,n", [(1, 16, 16), (1, 5, 3), (3, 33, 130), (16, 768, 768), (8, 1003, 129), (16, 4096, 300), (9, 2000, 1),
                                   (2, 300, 20000)])
def test_few_tokens(pkg, m, k, n):
    a, sa, b, sb, bias = operands(m, k, n, m + k)
    check(pkg.quantization.matmul_scaled(a, sa, b, sb, path="skinny"), a, sa, b, sb, None)
    check(pkg.quantization.matmul_scaled(a, sa, b, sb, bias, activation="gelu", path="skinny"), a, sa, b, sb, bias, True)


def test_nothing_behind_the_operands_is_touched(pkg):
    """Operands that end where their allocation ends, the last row shorter than the pitch: the product may not
    depend on, or read, what would follow (a slice of a packed weight)."""
    wide = torch.randint(-127, 128, (200, 512), dtype=torch.int8, device=dev())
    w = wide[:, 512 - 112 - 32:512 - 32]  # 112 columns, pitch 512
    tall = torch.randint(-127, 128, (30, 256), dtype=torch.int8, device=dev())
    x = tall[:, 48:48 + 200]              # K = 200, pitch 256
    sa, sb = torch.rand(30, device=dev()), torch.rand(112, device=dev())
    for rows in (1, 16, 30):
        check(pkg.quantization.matmul_scaled(x[:rows], sa[:rows].contiguous(), w, sb), x[:rows], sa[:rows], w, sb, None)


@pytest.mark.parametrize("m,k,n", [(5, 63, 61), (70, 130, 100), (1, 1, 1), (200, 33, 17)])
def test_product_of_unaligned_operands(pkg, m, k, n):
    a, sa, b, sb, bias = operands(m, k, n, m, pad=False)
    check(pkg.quantization.matmul_scaled(a, sa, b, sb, bias), a, sa, b, sb, bias)


def test_product_extremes_and_non_finite_scales(pkg):
    m, k, n = 40, 100000, 64  # sums beyond 2^24, up to 1.6e9
    a = torch.full((m, k), 127, dtype=torch.int8, device=dev())
    b = torch.full((k, n), -127, dtype=torch.int8, device=dev())
    sa, sb = torch.full((m,), 0.5, device=dev()), torch.full((n,), 0.25, device=dev())
    sa[3], sb[5] = math.nan, math.inf
    for path in ("auto", "simt"):
        got = pkg.quantization.matmul_scaled(a, sa, b, sb, path=path).cpu()
        assert got[3].isnan().all()
        keep = torch.ones(m, dtype=torch.bool)
        keep[3] = False
        assert (got[keep][:, 5] == -math.inf).all()
        cols = [j for j in range(n) if j != 5]
        np.testing.assert_allclose(got[keep][:, cols].numpy(), -127.0 * 127 * k / 8, rtol=2 * EPS)


def test_batched_rows_and_strided_operands(pkg):
    a, sa, b, sb, bias = operands(60, 256, 320, 9)
    got = pkg.quantization.matmul_scaled(a.view(3, 20, 256), sa.view(3, 20), b, sb, bias)
    assert got.shape == (3, 20, 320)
    check(got.view(60, 320), a, sa, b, sb, bias)
    # a weight that is a column slice of a packed one, on and off a 16-byte boundary
    for lo in (64, 5):
        w, s = b[:, lo:lo + 200], sb[lo:lo + 200].contiguous()
        check(pkg.quantization.matmul_scaled(a, sa, w, s), a, sa, w, s, None)


@pytest.mark.parametrize("m,k,n,gelu", [(1, 768, 768, False), (5, 1003, 514, True), (130, 600, 1000, False), (700, 130, 259, True)])
def test_linear_is_quantize_then_product(pkg, m, k, n, gelu):
    x = activations(m, k, m).to(dev())
    _, _, b, sb, bias = operands(1, k, n, k)
    act = "gelu" if gelu else None
    got = pkg.quantization.linear(x, b, sb, bias, activation=act)
    codes, scales = pkg.quantization.quantize_tokens(x)
    assert torch.equal(got, pkg.quantization.matmul_scaled(codes, scales, b, sb, bias, activation=act))
    check(got, codes, scales, b, sb, bias, gelu)


def test_quantize_channels(pkg):
    w = activations(300, 77, 5)
    codes, scales = pkg.quantization.quantize_channels(w.to(dev()))
    want, want_scales = reference_codes(w.t().contiguous())
    np.testing.assert_array_equal(codes.cpu().numpy(), want.T)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    assert codes.stride(0) % 16 == 0


def test_linear_graphs_replayed_side_by_side(pkg):
    """Each captured call keeps the codes of its own activations."""
    _, _, b, sb, bias = operands(1, 2048, 512, 3)
    graphs, outs, wants = [], [], []
    for m in (3, 16, 300):
        x = activations(m, 2048, m).to(dev())
        wants.append(pkg.quantization.linear(x, b, sb, bias))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.quantization.linear(x, b, sb, bias))
        graphs.append((g, x))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(50):
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        assert torch.equal(out, want)


def test_weights_written_just_before_are_seen(pkg):
    """The few-token product asks for its weights before it waits for the kernel ahead: what an earlier kernel of
    the stream wrote into them has to be there."""
    _, _, b, sb, _ = operands(1, 4096, 2048, 5)
    new = torch.randint(-127, 128, tuple(b.shape), dtype=torch.int8, device=dev())
    x = activations(7, 4096, 6).to(dev())
    codes, scales = pkg.quantization.quantize_tokens(x)
    for w in (new, -new, new // 2) * 4:
        b.copy_(w)
        got = pkg.quantization.linear(x, b, sb)
        check(got, codes, scales, w, sb, None)


def test_linear_in_a_graph_and_on_a_side_stream(pkg):
    _, _, b, sb, bias = operands(1, 512, 640, 3)
    x = activations(20, 512, 4).to(dev())
    want = pkg.quantization.linear(x, b, sb, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.quantization.linear(x, b, sb, bias)
    side.synchronize()
    assert torch.equal(got, want)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.quantization.linear(static, b, sb, bias)
    for seed in (5, 6):
        fresh = activations(20, 512, seed).to(dev())
        static.copy_(fresh)
        graph.replay()
        assert torch.equal(out, pkg.quantization.linear(fresh, b, sb, bias))


@pytest.mark.parametrize("m,path", [(4, "auto"), (200, "umma"), (200, "umma2"), (200, "simt")])
@pytest.mark.parametrize("activation", [None, "gelu"])
def test_results_beyond_the_range_are_infinite(pkg, m, path, activation):
    # 64 * 127 * 127 * 1e20 * 1e20 passes the largest float; gelu(+inf) = inf.  Column 1 is an exact zero.
    a = torch.full((m, 64), 127, dtype=torch.int8, device="cuda")
    b = torch.zeros(64, 16, dtype=torch.int8, device="cuda")
    b[:, 0] = 127
    s = torch.full((m,), 1e20, device="cuda")
    out = pkg.quantization.matmul_scaled(a, s, b, torch.full((16,), 1e20, device="cuda"), activation=activation, path=path)
    assert bool((out[:, 0] == math.inf).all()) and bool((out[:, 1:] == 0).all())

"""The 8-bit linear layer and the cache at the ends of their ranges, on the GPU."""
import pytest
import torch

from test_gpu_cache import Setup

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("m,path", [(1, "skinny"), (16, "auto"), (40, "umma"), (40, "umma2"), (40, "simt")])
def test_the_largest_sums(pkg, m, path):
    """K at its limit, codes of -128 in both operands: 2147467264, or its negative against 127.  One rounding of the
    sum and two products with powers of two: within 2^-24."""
    k = 131071
    a = torch.full((m, k + 1), -128, dtype=torch.int8, device=dev())[:, :k]
    b = torch.full((k, 32), -128, dtype=torch.int8, device=dev())
    b[:, 16:] = 127
    sa, sb = torch.full((m,), 0.5, device=dev()), torch.full((32,), 0.25, device=dev())
    got = pkg.quantization.matmul_scaled(a, sa, b, sb, path=path).double()
    want = torch.full_like(got, 128 * 128 * k / 8)
    want[:, 16:] = -128 * 127 * k / 8
    assert bool(((got - want).abs() <= 2.0 ** -24 * want.abs()).all())
    pkg.session.get_session(dev()).sync()


@pytest.mark.parametrize("m,n,k", [(65536 * 64 + 3, 5, 3), (3, 65536 * 64 + 3, 2)])
def test_operands_off_16_bytes_of_any_length(pkg, m, n, k):
    """More tiles than a grid's second dimension has, on the CUDA-core path: nothing is refused, above all not after
    the tokens have been quantized.  Results as from the same rows and columns in a small call."""
    g = torch.Generator(device=dev()).manual_seed(1)
    x = torch.randn(m, k, device=dev(), generator=g)
    b = torch.randint(-127, 128, (k, n), device=dev(), generator=g).to(torch.int8)
    s = torch.rand(n, device=dev(), generator=g)
    got = pkg.quantization.linear(x, b, s)
    codes, scales = pkg.quantization.quantize_tokens(x)
    for rows, cols in ((slice(0, 70), slice(0, 5)), (slice(m - 70 if m > 70 else 0, m), slice(max(0, n - 5), n))):
        sums = codes[rows].double() @ b[:, cols].double()
        want = sums * scales[rows].double()[:, None] * s[cols].double()
        assert bool(((got[rows, cols].double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all())
    pkg.session.get_session(dev()).sync()


@pytest.mark.parametrize("news,lengths,heads", [([1, 1], [3000, 700], 1), ([1], [9000], 8), ([60, 1], [700, 2000], 2)])
def test_bounds_beyond_the_tensors_shape_the_launch_like_the_tensors(pkg, news, lengths, heads):
    """UINT_MAX for "no bound" at the C entry: same kernels, same cuts, same bits as with the tensors' own extents."""
    s = Setup(pkg, news, lengths, 1, 64, 16, seed=5)
    q = torch.randn(s.rows, heads * 64, device=dev(), generator=s.g)
    capacity = s.table.shape[1] * 16
    scratch = torch.empty(64 << 20, dtype=torch.uint8, device=dev())
    outs, launches = [], []
    for most, longest in ((s.rows, capacity), (2 ** 32 - 1, capacity), (s.rows, 2 ** 32 - 1), (2 ** 32 - 1, 2 ** 32 - 100), (2 ** 31, 2 ** 31)):
        need = pkg.lib.tfccb200_cache_attention_workspace(s.cache._ref, len(news), s.rows, heads, most, longest)
        assert 0 < need <= scratch.numel()
        out = torch.full_like(q, -1.0)
        before = pkg.launch_count()
        st = pkg.lib.tfccb200_cache_attention_f32(
            torch.cuda.current_stream().cuda_stream, s.cache._ref, q.data_ptr(), q.shape[1], out.data_ptr(), q.shape[1], s.starts.data_ptr(),
            s.lens.data_ptr(), s.table.data_ptr(), len(news), s.table.shape[1], s.rows, heads, most, longest, 0.125, 1, scratch.data_ptr(), need, None)
        assert st == 0
        outs.append(out)
        launches.append(pkg.launch_count() - before)
    assert len(set(launches)) == 1
    for out in outs[1:]:
        assert torch.equal(out, outs[0])

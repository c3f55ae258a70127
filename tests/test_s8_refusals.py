"""What the 8-bit linear layer, the cache and its attention refuse, without a GPU: argument classes
at the C entry points (decided before anything touches CUDA) and the Python checks."""
import ctypes as C

import pytest
import torch

EINVAL, EALIGN, EWORKSPACE, EOVERFLOW, EUNSUPPORTED = -1, -2, -3, -4, -5
P = 1 << 20  # an address nobody follows: every call here is refused first


def linear_args(**kw):
    a = dict(stream=None, A=P, lda=64, sa=P, B=P, ldb=64, sb=P, bias=None, C=P, M=4, N=64, K=64, act=0, path=0, status=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,want", [
    ({"A": None}, EINVAL), ({"B": None}, EINVAL), ({"C": None}, EINVAL), ({"sa": None}, EINVAL), ({"sb": None}, EINVAL),
    ({"M": 0}, EINVAL), ({"N": 0}, EINVAL), ({"K": 0}, EINVAL), ({"lda": 63}, EINVAL), ({"ldb": 63}, EINVAL),
    ({"act": 7}, EINVAL), ({"path": 9}, EINVAL), ({"path": 2, "M": 17}, EUNSUPPORTED), ({"path": 2, "lda": 72}, EUNSUPPORTED), ({"K": 133001, "lda": 133008}, EOVERFLOW),
    ({"M": 1 << 20, "N": 1 << 13, "ldb": 1 << 13}, EOVERFLOW), ({"C": P + 2}, EALIGN), ({"sa": P + 1}, EALIGN),
    ({"bias": P + 2}, EALIGN), ({"path": 3, "lda": 72}, EUNSUPPORTED), ({"path": 4, "B": P + 4}, EUNSUPPORTED)])
def test_product_refusals(pkg, kw, want):
    assert pkg.lib.tfccb200_qgemm_scaled_s8(*linear_args(**kw)) == want


@pytest.mark.parametrize("kw,want", [
    ({"src": None}, EINVAL), ({"codes": None}, EINVAL), ({"scales": None}, EINVAL), ({"rows": 0}, EINVAL),
    ({"cols": 0}, EINVAL), ({"ld_src": 9}, EINVAL), ({"ld_codes": 9}, EINVAL), ({"src": P + 2}, EALIGN),
    ({"rows": 1 << 31}, EOVERFLOW)])
def test_quantize_tokens_refusals(pkg, kw, want):
    a = dict(stream=None, src=P, ld_src=10, rows=2, cols=10, codes=P, ld_codes=16, scales=P)
    a.update(kw)
    assert pkg.lib.tfccb200_quantize_tokens_f32(*a.values()) == want


@pytest.mark.parametrize("kw,want", [
    ({"x": None}, EINVAL), ({"ldx": 9}, EINVAL), ({"B": None}, EINVAL), ({"ldb": 9}, EINVAL), ({"act": 3}, EINVAL),
    ({"ws": None}, EWORKSPACE), ({"ws": P + 16}, EWORKSPACE), ({"ws_len": 100}, EWORKSPACE)])
def test_linear_refusals(pkg, kw, want):
    a = dict(stream=None, x=P, ldx=10, B=P, ldb=16, sb=P, bias=None, C=P, M=2, N=10, K=10, act=0, ws=P, ws_len=4096, status=None)
    a.update(kw)
    assert pkg.lib.tfccb200_qlinear_f32(*a.values()) == want
    assert pkg.lib.tfccb200_qlinear_workspace(2, 10) == 256 + 32


def struct(pkg, **kw):
    a = dict(keys=P, key_scales=P, values=P, value_scales=P, pages=10, page_size=16, kv_heads=2, dim=64)
    a.update(kw)
    return pkg.cache._Struct(*a.values())


POOL = [({"keys": None}, EINVAL), ({"value_scales": None}, EINVAL), ({"pages": 0}, EINVAL), ({"kv_heads": 0}, EINVAL),
        ({"dim": 32}, EUNSUPPORTED), ({"dim": 96}, EUNSUPPORTED), ({"page_size": 0}, EUNSUPPORTED),
        ({"page_size": 48}, EUNSUPPORTED), ({"page_size": 2048}, EUNSUPPORTED), ({"keys": P + 8}, EALIGN),
        ({"pages": 1 << 31}, EOVERFLOW)]
CALL = [({"x": None}, EINVAL), ({"starts": None}, EINVAL), ({"lengths": None}, EINVAL), ({"table": None}, EINVAL),
        ({"batch": 0}, EINVAL), ({"width": 0}, EINVAL), ({"rows": 0}, EINVAL), ({"ld": 124}, EINVAL), ({"ld": 130}, EALIGN),
        ({"x": P + 4}, EALIGN), ({"starts": P + 2}, EALIGN), ({"width": 1 << 28}, EOVERFLOW)]


@pytest.mark.parametrize("pool,call,want", [(p, {}, w) for p, w in POOL] + [({}, c, w) for c, w in CALL])
def test_cache_refusals(pkg, pool, call, want):
    lib = pkg.lib
    a = dict(x=P, ld=128, starts=P, lengths=P, table=P, batch=3, width=4, rows=9)
    a.update(call)
    s = C.byref(struct(pkg, **pool))
    rest = [a["starts"], a["lengths"], a["table"], a["batch"], a["width"], a["rows"]]
    for fn in (lib.tfccb200_cache_append_f32, lib.tfccb200_cache_read_f32):
        assert fn(None, s, a["x"], a["ld"], P, 128, *rest, None) == want
        if call and ("x" in call or "ld" in call):
            assert fn(None, s, P, 128, a["x"], a["ld"], *rest, None) == want
    for q, ldq, o, ldo in ((a["x"], a["ld"], P, 128), (P, 128, a["x"], a["ld"])):
        if call and not ("x" in call or "ld" in call) or pool or q == a["x"] or o == a["x"]:
            assert lib.tfccb200_cache_attention_f32(None, s, q, ldq, o, ldo, *rest, 2, 1, 64, 0.1, 1, P, 1 << 40, None) == want


@pytest.mark.parametrize("kw,want", [({"heads": 0}, EINVAL), ({"heads": 3}, EINVAL), ({"max_new": 0}, EINVAL), ({"max_length": 0}, EINVAL)])
def test_attention_refusals(pkg, kw, want):
    a = dict(heads=2, max_new=1, max_length=64)
    a.update(kw)
    assert pkg.lib.tfccb200_cache_attention_f32(None, C.byref(struct(pkg)), P, 256, P, 256, P, P, P, 3, 4, 9, a["heads"], a["max_new"],
                                                a["max_length"], 0.1, 1, P, 1 << 40, None) == want
    assert pkg.lib.tfccb200_cache_attention_workspace(None, 3, 9, 2, 1, 64) == 0


def test_python_checks_refuse_what_is_not_on_a_gpu(pkg):
    ex, q, ch = pkg.exceptions, pkg.quantization, pkg.cache
    x, b = torch.zeros(4, 64), torch.zeros(64, 32, dtype=torch.int8)
    with pytest.raises(ex.InvalidArgumentError, match="CUDA"):
        q.quantize_tokens(x)
    with pytest.raises(ex.InvalidArgumentError, match="invalid tensor a"):
        q.quantize_tokens(torch.zeros(4))
    with pytest.raises(ex.NotImplementedError, match="float32"):
        q.quantize_tokens(x.double())
    with pytest.raises(ex.InvalidArgumentError, match="CUDA"):
        q.linear(x, b, torch.zeros(32))
    with pytest.raises(ex.NotImplementedError, match="int8"):
        q.matmul_scaled(x, torch.zeros(4), b, torch.zeros(32))
    with pytest.raises(ex.InvalidArgumentError, match="invalid tensor w"):
        q.quantize_channels(torch.zeros(3, 4, 5))
    codes, scales = torch.zeros(3, 2, 16, 64, dtype=torch.int8), torch.zeros(3, 2, 16)
    with pytest.raises(ex.InvalidArgumentError, match="CUDA"):
        ch.PagedCache(codes, scales, codes.clone(), scales.clone())
    with pytest.raises(ex.InvalidArgumentError, match="values: expected shape"):
        ch.PagedCache(codes, scales, codes[:2], scales)
    with pytest.raises(ex.NotImplementedError, match="keys: implemented"):
        ch.PagedCache(codes.float(), scales, codes, scales)
    with pytest.raises(ex.InvalidArgumentError, match="pages, kv_heads"):
        ch.PagedCache(codes[0], scales, codes, scales)
    with pytest.raises(ex.InvalidArgumentError, match="PagedCache"):
        ch.append(None, x, x, None, None, None)


# rows whose column counter would pass 32 bits; operands that only the second of linear's two kernels reads
def test_refusals_of_the_largest_and_the_misaligned(pkg):
    lib, big = pkg.lib, 1 << 31
    assert lib.tfccb200_quantize_tokens_f32(None, P, big, 1, big, P, big, P) == EOVERFLOW
    for kw in ({"C": P + 2}, {"sb": P + 2}, {"bias": P + 1}):
        a = dict(stream=None, x=P, ldx=10, B=P, ldb=16, sb=P, bias=None, C=P, M=2, N=10, K=10, act=0, ws=P, ws_len=4096, status=None)
        a.update(kw)
        assert lib.tfccb200_qlinear_f32(*a.values()) == EALIGN
    # 2^24 tiles of 2^23 blocks each
    s = C.byref(struct(pkg, kv_heads=1, page_size=1024))
    assert lib.tfccb200_cache_attention_f32(None, s, P, 256, P, 256, P, P, P, 1, 1 << 20, (1 << 29) - 1, 4, (1 << 29) - 1, 1 << 30,
                                            0.1, 1, P, 1 << 40, None) == EOVERFLOW

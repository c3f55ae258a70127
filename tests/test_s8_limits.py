"""Limits of the 8-bit linear layer and the cache at the C entry points and in Python, without a GPU."""
import pytest

from test_s8_refusals import EOVERFLOW, P, linear_args


@pytest.mark.parametrize("k", [131072, 132105, 133000])
def test_sums_of_codes_of_minus_128_have_to_fit(pkg, k):
    """128 * 128 * 131072 = 2^31."""
    assert pkg.lib.tfccb200_qgemm_scaled_s8(*linear_args(K=k, lda=k // 16 * 16 + 16)) == EOVERFLOW
    args = [None, P, k, P, 64, P, None, P, 2, 64, k, 0, P, 1 << 40, None]
    assert pkg.lib.tfccb200_qlinear_f32(*args) == EOVERFLOW


@pytest.mark.parametrize("kw", [{"M": 1 << 31, "N": 1, "K": 1}, {"M": 0xffffffff, "N": 1, "K": 1}, {"M": 1, "N": 1 << 31, "K": 1, "ldb": 1 << 31}])
@pytest.mark.parametrize("path", [0, 1, 3, 4])
def test_rows_and_columns_that_a_tile_would_carry_past_32_bits(pkg, kw, path):
    assert pkg.lib.tfccb200_qgemm_scaled_s8(*linear_args(**dict(kw, path=path))) == EOVERFLOW


def test_the_attributes_of_a_cache_are_fixed(pkg):
    """Calls go by the addresses that the constructor took: a tensor put in another's place would leave them pointing
    into freed memory."""
    cache = pkg.cache.PagedCache.__new__(pkg.cache.PagedCache)
    for name in ("keys", "key_scales", "values", "value_scales", "pages", "kv_heads", "page_size", "dim", "device"):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(cache, name, None)
        with pytest.raises(AttributeError, match="fixed"):
            delattr(cache, name)

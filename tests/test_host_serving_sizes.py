"""CPU tests of the serving calls' sizes: products beyond 64 bits are refused like other sizes beyond the limits.  C ABI with addresses that are never read."""
import pytest

from test_host_serving import append, packed, paged

BIG = (1 << 62, (1 << 62) + 7, (1 << 63) - 1, 1 << 61, 1 << 33, (1 << 32) + 1)


@pytest.mark.parametrize("tokens", BIG)
def test_more_tokens_than_64_bits_count_heads_of(pkg, tokens):
    for H in (4, 8, 1):
        strides = (64 * H, 64, 64, 64 * H)
        assert packed(pkg, desc=(2, 10, 10, H, 1, 64), tokens=(tokens, 20), strides=strides) == pkg.ERR_TOO_LARGE
        assert paged(pkg, desc=(2, 1, 100, H, 1, 64), tokens=tokens, strides=(64 * H, 64 * H)) == pkg.ERR_TOO_LARGE
        assert append(pkg, dims=(tokens, H, 2, 64, 64), strides=(64 * H, 128, 128)) == pkg.ERR_TOO_LARGE


def test_more_heads_than_64_bits_count(pkg):
    assert append(pkg, dims=(1, 1 << 62, 2, 64, 64)) == pkg.ERR_TOO_LARGE and append(pkg, dims=(1, 4, (1 << 62) + 1, 64, 64)) == pkg.ERR_TOO_LARGE


@pytest.mark.parametrize("stride", [1 << 62, (1 << 63) - 16, 1 << 60, 1 << 41])
def test_strides_beyond_any_memory(pkg, stride):
    for i in range(4):
        strides = [256, 128, 128, 256]
        strides[i] = stride
        assert packed(pkg, strides=strides) == pkg.ERR_TOO_LARGE, i
    for i in range(2):
        strides = [256, 256]
        strides[i] = stride
        assert paged(pkg, strides=strides) == pkg.ERR_TOO_LARGE, i
    assert paged(pkg, cache=(8, 16, stride, 4, 4)) == pkg.ERR_TOO_LARGE
    assert paged(pkg, cache=(8, 16, 2048, 4, stride)) == pkg.ERR_TOO_LARGE
    for i in range(3):
        strides = [256, 128, 128]
        strides[i] = stride
        assert append(pkg, strides=strides) == pkg.ERR_TOO_LARGE, i
    assert append(pkg, cache=(8, 16, stride)) == pkg.ERR_TOO_LARGE


def test_more_sequences_and_heads_than_units(pkg):
    L = pkg.lib()
    assert packed(pkg, desc=((1 << 31) - 1, 10, 10, 1 << 20, 1 << 20, 64), tokens=(1, 20), strides=(1 << 26, 1 << 26, 1 << 26, 1 << 26)) == pkg.ERR_TOO_LARGE
    assert paged(pkg, desc=((1 << 31) - 1, 1, 100, 1 << 20, 1 << 20, 64), tokens=1, strides=(1 << 26, 1 << 26), cache=(8, 16, 1 << 30, 4, 4)) == pkg.ERR_TOO_LARGE
    assert L.fmha_i8_sm100_last_status() == pkg.ERR_TOO_LARGE

"""Arguments at the ends of what the kernels can take (no GPU). fp32 and int32
arrays that are not 4-byte aligned are refused: the kernels read them by the
word, and a misaligned address is a fault of the GPU."""

import pytest

from test_cache_attn_args import A, S, _lib, _shape, decode, evict, shared, weights, window


def decode_acc(acc):
    return _lib()[1].lfm_attention_decode(_shape(), A, 512, A, A, 16384, 4, A, A, 2, 128, 0, 0, acc, A, 512, None)


@pytest.mark.parametrize("call", [
    lambda x: window(lse=A + x), lambda x: weights(lse=A + x), lambda x: weights(acc=A + x), lambda x: decode(sl=A + x),
    lambda x: decode(lens=A + x), lambda x: decode_acc(A + x), lambda x: shared(lens=A + x),
    lambda x: evict(src=(S, 2 * S, 3 * S + x, 4 * S)), lambda x: evict(src=(S, 2 * S, 3 * S, 4 * S + x)),
    lambda x: evict(dst=(5 * S, 6 * S, 7 * S + x, 8 * S)), lambda x: evict(dst=(5 * S, 6 * S, 7 * S, 8 * S + x)),
    lambda x: evict(sl=9 * S + x), lambda x: evict(lens=10 * S + x), lambda x: evict(out=11 * S + x)])
def test_misaligned_words(call):
    for x in (1, 2, 3):
        assert call(x) == 1
        assert "4-byte aligned" in _lib()[1].lfm_ops_error().decode()
    assert call(4) == 1  # aligned: refused only because these are no device pointers
    assert "current device" in _lib()[1].lfm_ops_error().decode()


@pytest.mark.parametrize("call", [window, weights, decode, shared])
def test_scales_whose_powers_of_two_are_no_fp32_number(call):
    """scale * log2 e above fp32's largest, and scales below its smallest normal number."""
    for bad in (3e38, 2.5e38, 1e-39, 1e-45):
        assert call(sh=_shape(scale=bad)) == 1
        assert "scale" in _lib()[1].lfm_ops_error().decode()
    for good in (2.0 ** 127, 2.0 ** -126, 0.0, -0.0, 1.0):
        assert call(sh=_shape(scale=good)) == 1
        assert "current device" in _lib()[1].lfm_ops_error().decode()

"""What the attention entry points refuse before they touch a device."""
import ctypes

import numpy as np
import pytest

import attention_reference as R
from ane_fieldfare_b200 import binding
from ane_fieldfare_b200.binding import FFAttentionConfig


@pytest.mark.parametrize("config,says", [
    ((6, 4, 64, 16, 1, 1), b"multiple of kvHeads"), ((0, 0, 64, 16, 1, 1), b"multiple of kvHeads"), ((130, 2, 64, 16, 1, 1), b"64 query heads"),
    ((4, 2, 96, 16, 1, 1), b"headDim"), ((4, 2, 64, 8, 1, 1), b"pageTokens"), ((4, 2, 64, 48, 1, 1), b"pageTokens"),
    ((4, 2, 64, 512, 1, 1), b"pageTokens"), ((4, 2, 64, 16, 0, 1), b"requests"), ((4, 2, 64, 16, 1, 0), b"rows")])
def test_unsupported_shapes(config, says):
    lib, err, c = binding.load(), ctypes.c_char_p(), FFAttentionConfig(*config)
    assert not lib.ff_attention_create(0, ctypes.byref(c), ctypes.byref(err))
    assert says in err.value
    assert lib.ff_cache_page_bytes(ctypes.byref(c)) == 0


def test_null_handles():
    lib = binding.load()
    err = ctypes.c_char_p()
    assert not lib.ff_attention_create(0, None, ctypes.byref(err)) and b"config" in err.value
    err = ctypes.c_char_p()
    assert not lib.ff_attention(None, None, 0, 0, None, 0, None, 0, None, None, 0, 0, 1.0, 0, 0, None, 0, None, ctypes.byref(err))
    assert b"null attention handle" in err.value
    err = ctypes.c_char_p()
    assert not lib.ff_cache_plan(None, *[None] * 2, 0, None, 0, None, 0, *[None] * 5, 0, None, ctypes.byref(err))
    assert b"null attention handle" in err.value
    lib.ff_attention_destroy(None)


@pytest.mark.parametrize("dim,page,kvHeads", [(64, 16, 1), (128, 64, 8), (256, 256, 2)])
def test_page_bytes_are_codes_and_words_of_keys_and_values(dim, page, kvHeads):
    c = FFAttentionConfig(kvHeads, kvHeads, dim, page, 1, 1)
    assert binding.load().ff_cache_page_bytes(ctypes.byref(c)) == kvHeads * page * 2 * (dim // 2 + dim // 64 * 4)


def test_the_reference_reads_what_it_quantizes():
    """The tests' own statements agree with one another: pages packed by hand, unpacked, give the quantizer's values."""
    rng = np.random.RandomState(0)
    x = R.to_bf16(rng.randn(2, 16, 1, 64))
    codes, scale, low, value = R.quantized(x)
    words = ((scale.astype(np.float32).view(np.uint32) >> 16) | (R.to_bf16(low).astype(np.float32).view(np.uint32) & 0xFFFF0000)).astype(np.uint32)
    parts = []
    for side in range(2):
        c = codes[side, :, 0].astype(np.uint8)
        parts += [(c[:, 0::2] | c[:, 1::2] << 4).reshape(-1), words[side, :, 0].reshape(-1).view(np.uint8)]
    keys, values = R.unpack(np.concatenate(parts).reshape(1, 1, -1), 1, 64, 16)
    assert np.array_equal(keys, value[0]) and np.array_equal(values, value[1])


def test_to_bf16_rounds_once():
    assert R.to_bf16(1 + 2.0 ** -8) == 1.0 and R.to_bf16(1 + 2.0 ** -8 + 2.0 ** -40) == 1 + 2.0 ** -7
    assert R.to_bf16(1 + 3 * 2.0 ** -8) == 1 + 2.0 ** -6 and np.isnan(R.to_bf16(np.nan)) and R.to_bf16(-np.inf) == -np.inf

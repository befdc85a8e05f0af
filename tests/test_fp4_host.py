"""The 4-bit element on the host: sizes and the constant, and the definition that the GPU tests compare with on values worked out by hand."""
import os
import re

import numpy as np
import pytest

import saragossa_amd as skv
from fp4_reference import attention, stored
from saragossa_amd import flags


def test_the_constant_is_the_headers():
    header = open(os.path.join(os.path.dirname(__file__), "..", "include", "saragossa_kv.h")).read()
    assert int(re.search(r"#define SKV_DTYPE_FP4 (\d+)", header).group(1)) == skv.DTYPE_FP4 == 2


@pytest.mark.parametrize("dims,capacity,window,rows", [((16, 2, 256), 32768 + 300, 0, 33072), ((32, 8, 128), 100, 0, 112), ((8, 8, 80), 1024, 0, 1024),
                                                       ((16, 8, 256), 65536, 1024, 1056), ((5, 1, 33), 17, 0, 32), ((8, 2, 512), 64, 0, 64)], ids=str)
def test_layer_bytes(dims, capacity, window, rows):
    """Codes of half a byte and a byte per 32 dims, K and V, of heads padded to 32, 64, 96, 128, 256 or 512 dims: 17 bytes where bf16 has 64.
    The rest of a layer (table, partials, staging rows) is the same as with the other elements, or smaller."""
    padded = next(p for p in (32, 64, 96, 128, 256, 512) if p >= dims[2])
    pools = 2 * rows * dims[1] * padded * 17 // 32
    got = flags.layer_bytes(capacity, *dims, skv.DTYPE_FP4, window)
    other = flags.layer_bytes(capacity, *dims, skv.DTYPE_BF16, window)
    rest = other - 2 * rows * dims[1] * padded * 2
    assert pools < got <= pools + rest + 4096


def test_layer_bytes_refuses_what_a_layer_refuses():
    for bad in [(0, 16, 2, 256), (16, 0, 2, 256), (16, 16, 3, 256), (16, 16, 2, 513)]:
        with pytest.raises(skv.ConfigError):
            flags.layer_bytes(*bad, skv.DTYPE_FP4)
    with pytest.raises(skv.ConfigError):
        flags.layer_bytes(16, 16, 2, 256, 3)


def test_the_definition_by_hand():
    def one(*x):
        row = np.zeros((1, 32), np.float32)
        row[0, :len(x)] = x
        return stored(row, 32)[0, :len(x)].tolist()

    assert one(6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5) == [6, 0, 1, 1, 2, 2, 4, 4]      # 2^0: ties to the even index
    assert one(7, 0.26, -5.1) == [6, 0.5, -6]                                           # 7 is still within 7 * 2^0
    assert one(np.nextafter(np.float32(7), np.float32(8)), 5.1, 1) == [8, 6, 1]        # above it the power is 2
    assert one(3.5, 0.125, 0.126) == [3, 0, 0.25]                                       # 2^-1
    assert one(1.0, np.nan)[0] != one(1.0)[0] and all(np.isnan(one(1.0, np.inf)))
    assert one(0.0, -0.0) == [0.0, 0.0]
    tiny = 2.0 ** -126                                                                  # the smallest power is 2^-125
    assert one(np.float32(tiny)) == [tiny] and one(np.float32(tiny / 4)) == [0.0]


def test_groups_do_not_cross_heads():
    """Heads of 40 dims: groups of 32 and of 8."""
    row = np.zeros((1, 80), np.float32)
    row[0, [0, 35, 40, 75]] = 6, 96, 0.375, 1536
    row[0, [1, 36, 41, 76]] = 1, 16, 0.0625, 256
    assert np.array_equal(stored(row, 40), row)


def test_the_reference_attention_is_a_weighted_mean():
    """Equal keys give every row the same weight, through a window as well."""
    v = np.arange(12, dtype=np.float64).reshape(6, 2)
    q = np.ones((2, 4), np.float32)
    got, tol = attention(q, np.ones((6, 2)), v, (2, 1, 2), window=3)
    assert np.allclose(got[0].reshape(2, 2), v[2:5].mean(0)) and np.allclose(got[1].reshape(2, 2), v[3:6].mean(0))
    assert (tol > 0).all() and (tol < 1e-3).all()

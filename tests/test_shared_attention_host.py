"""Host side of the shared-prefix and bounded-cache operators (no GPU): what
the library's size queries answer to shapes that it does not compute, and the
bookkeeping of caches behind a prefix."""
import ctypes

import pytest

from nki_moe_7013_b200 import _C


@pytest.fixture(scope="module")
def lib():
    from nki_moe_7013_b200.build import build

    build()
    return _C.lib()


@pytest.mark.parametrize("nh,nkv", [(17, 1), (128, 4), (129, 1), (256, 1), (1 << 20, 2)])
def test_sizes_of_unsupported_head_ratios(lib, nh, nkv):
    """More than 16 query heads per KV head: the size queries answer 0, and the
    entry points refuse the shape by name."""
    assert lib.qmoe_attention_weights_workspace_size(1, 4, nh, nkv, 64) == 0
    for P, max_len, weights in ((4096, 64, 0), (0, 4096, 1), (10, 10, 1)):
        assert lib.qmoe_attention_prefix_decode_workspace_size(2, nh, nkv, P, max_len, weights) == 0
    if nh > 65535:
        return
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    p += -p % 256
    f = ctypes.c_float(0.1)
    assert lib.qmoe_attention_weights(p, p, p, p, None, None, 1, 4, nh, nkv, 128, 2, 64, 64, f, p, 1, None, 0, None) == -2
    assert b"query heads per KV head" in lib.qmoe_last_error()
    assert lib.qmoe_attention_prefix_decode(p, p, p, 1, 4096, 0, 4096, p, p, p, None, None, 2, nh, nkv, 128, 2, 64, 64,
                                            f, None, 1, p, None, 0, None) == -2
    assert b"query heads per KV head" in lib.qmoe_last_error()

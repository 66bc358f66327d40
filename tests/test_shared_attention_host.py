"""Host side of the shared-prefix and bounded-cache operators (no GPU): what
the library's size queries answer to shapes that it does not compute, and the
bookkeeping of caches behind a prefix."""
import copy
import ctypes

import pytest
import torch

from nki_moe_7013_b200 import _C
from nki_moe_7013_b200.attention import KVCache, SharedPrefix


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


def _prefix(n=1, rows=8, length=5, slot=0):
    k = torch.zeros(n, 2, rows, 128, dtype=torch.bfloat16)
    return SharedPrefix(k, torch.zeros_like(k), length, slot)


def test_a_cache_stays_behind_its_prefix():
    """Rows behind one prefix are not continued behind another of the same
    length; the same rows by another name are the same prefix."""
    a, b, two = _prefix(), _prefix(), _prefix(n=2)
    c = KVCache(2, 2, 16, 128, device="cpu", track=True)
    c._follow(5, None, 2, a)
    c.lengths = [3, 3]
    c._follow(5, None, 2, a)
    c._follow(5, None, 2, SharedPrefix(a.k.view(a.k.shape), a.v, 5, 0))
    for other in (b, SharedPrefix(a.k, b.v, 5, 0), SharedPrefix(two.k, two.v, 5, 1)):
        with pytest.raises(ValueError, match="another prefix"):
            c._follow(5, None, 2, other)
    fork = copy.deepcopy(c)  # stays behind the prefix, which is not copied
    fork._follow(5, None, 2, a)
    assert fork.behind[0] is a and fork.k.data_ptr() != c.k.data_ptr() and fork.behind is not c.behind
    with pytest.raises(ValueError, match="another prefix"):
        fork._follow(5, None, 2, b)
    c._evicted(2)
    with pytest.raises(ValueError, match="another prefix"):
        c._follow(5, None, 2, b)
    c._follow(5, None, 2, a)
    c.reset()
    c._follow(5, None, 1, two)
    c.lengths[0] = 2
    c._follow(5, None, 2, two)  # the second slot is still empty
    with pytest.raises(ValueError, match="another prefix"):
        c._follow(5, None, 2, SharedPrefix(two.k, two.v, 5, 1))
    # paddings alone hold nothing of a prefix yet
    d = KVCache(1, 2, 16, 128, device="cpu")
    d._follow(5, [2], 1, a)
    d.lengths = [2]
    d._follow(5, None, 1, b)
    d.lengths = [3]
    with pytest.raises(ValueError, match="another prefix"):
        d._follow(5, None, 1, a)


@pytest.mark.parametrize("behind", [False, True])
def test_refused_positions_leave_the_cache_as_it_was(behind):
    """Positions that do not continue the cache: refused before anything runs,
    and paddings of the refused call are not remembered."""
    from nki_moe_7013_b200.attention import Qwen3MoeAttention

    attn = object.__new__(Qwen3MoeAttention)
    object.__setattr__(attn, "cfg", None)
    prefix = _prefix() if behind else None
    x = torch.zeros(2, 4, 8)
    mask = torch.tensor([[1, 1, 1, 1], [0, 0, 1, 1]])
    for lengths in ([0, 0], [4, 4]):
        c = KVCache(2, 2, 16, 128, device="cpu")
        if lengths[0]:
            c._follow(5 if behind else 0, [0, 1], 2, prefix)
            c.lengths, mask = lengths, torch.cat([torch.ones(2, 4, dtype=torch.int64), mask], dim=1)
            mask[1, :4] = torch.tensor([0, 1, 1, 1])
            mask[1, 4:] = 1
            if not behind:
                mask[1, 1] = 0  # without a prefix the paddings may change
        kept = [list(getattr(c, n)) for n in ("pad", "lead", "prefix_len", "offset", "behind")]
        with pytest.raises(ValueError, match="position_ids"):
            Qwen3MoeAttention.forward(attn, x, torch.full((2, 4), 40), c, attention_mask=mask, prefix=prefix)
        assert [getattr(c, n) for n in ("pad", "lead", "prefix_len", "offset", "behind")] == kept

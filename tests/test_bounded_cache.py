"""Host side of shared prefixes and bounded caches (no GPU): the cache's
bookkeeping, and the refusals of the entry points before any launch."""
import ctypes

import pytest
import torch

from nki_moe_7013_b200 import _C, ops
from nki_moe_7013_b200.attention import KVCache


def _cache(n=3, rows=16, track=True):
    return KVCache(n, 2, rows, 128, device="cpu", track=track)


def test_eviction_bookkeeping():
    c = _cache()
    c.lengths, c.pad = [10, 4, 0], [3, 0, 0]
    c._evicted(6)
    assert c.lengths == [6, 4, 0] and c.pad == [0, 0, 0]
    # a new row's position goes on where the tokens stopped
    assert [n + o for n, o in zip(c.lengths, c.offset)] == [10, 4, 0]
    assert c.dropped == [4, 0, 0]
    c.lengths[0] = 9
    c._evicted(6)
    assert c.lengths[0] + c.offset[0] == 13 and c.dropped[0] == 7
    c.reset()
    assert c.offset == c.dropped == c.lengths == [0, 0, 0]


def test_cache_refusals():
    with pytest.raises(ValueError, match="track"):
        _cache(track=False).evict(4)
    for keep, recent in ((-1, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError, match="recent"):
            _cache().evict(keep, recent)
    with pytest.raises(ValueError, match="score_queries"):
        KVCache(1, 2, 8, 128, device="cpu", track=True, score_queries=0)
    c = _cache()
    c.lengths = [5, 5, 5]
    assert (c.as_prefix(1).length, c.as_prefix(1).slot) == (5, 1)
    with pytest.raises(ValueError, match="slot"):
        c.as_prefix(3)
    c.pad[0] = 1
    with pytest.raises(ValueError, match="padded"):
        c.as_prefix(0)
    c.lengths, c.pad = [9, 5, 5], [0, 0, 0]
    c._evicted(4)
    with pytest.raises(ValueError, match="evicted"):
        c.as_prefix(1)


def test_paddings_behind_a_prefix():
    c = _cache()
    c._follow(5, [0, 2, 4], 3)
    assert c.offset == [5, 3, 1] and c.prefix_len == [5, 5, 5] and c.lead == [0, 2, 4]
    c.lengths = [4, 4, 4]  # the third holds paddings alone
    for pads in ([1, 2, 4], [0, 0, 4], [0, 2, 3]):
        with pytest.raises(ValueError, match="first tokens"):
            c._follow(5, pads, 3)
    with pytest.raises(ValueError, match="another prefix"):
        c._follow(6, None, 3)
    assert c.offset == [5, 3, 1] and c.pad == [0, 2, 4]
    c._follow(5, [0, 2, 6], 3)  # its first token comes at row 6, at position 5
    assert c.offset == [5, 3, -1] and c.pad == [0, 2, 6]
    c.lengths = [8, 8, 8]
    c._follow(5, None, 3)
    assert c.offset == [5, 3, -1]
    # without a prefix a row's position is the row
    d = _cache()
    d._follow(0, [0, 2, 4], 3)
    assert d.offset == [0, 0, 0] and d.pad == [0, 2, 4]


def test_a_prefix_is_one_prompt():
    from nki_moe_7013_b200.model import Qwen3MoeModel

    for ids in (torch.zeros(2, 3, dtype=torch.int64), torch.zeros(0, dtype=torch.int64)):
        with pytest.raises(ValueError, match="one prompt"):
            Qwen3MoeModel.prefill_prefix(object.__new__(Qwen3MoeModel), ids)


def test_wrappers_refuse_cpu_tensors():
    k = torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16)
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    w = torch.zeros(2, 2, 16)
    calls = [lambda: ops.attention_prefix_decode(q, k, k, 4, k, k, i, 16),
             lambda: ops.attention_decode_weights(q, k, k, i, 16, w),
             lambda: ops.attention_prefix_prefill(q, k, k, 4, k, k, i, 2, 1),
             lambda: ops.attention_weights(q, torch.zeros(2, 8), k, i, 2, 1, w),
             lambda: ops.kv_evict(k, k, w, w.int(), i, 16, 4)]
    for call in calls:
        with pytest.raises(ValueError, match="no CPU path"):
            call()


@pytest.fixture(scope="module")
def lib():
    from nki_moe_7013_b200.build import build

    build()
    return _C.lib()


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(4096)
    p._keep = buf
    a = ctypes.addressof(buf)
    return a + (-a) % 256


def _decode(lib, p, **kw):
    a = dict(q=p, kp=p, vp=p, n_prefix=1, prefix_max=600, slot=0, P=500, k=p, v=p, kv_len=p, B=2, nh=32, nkv=4, hd=128,
             n_slots=2, max_seq=64, max_len=64, scale=0.1, out=p, ws=p, bytes=1 << 30, cache_slot=None)
    a.update(kw)
    return lib.qmoe_attention_prefix_decode(
        a["q"], a["kp"], a["vp"], a["n_prefix"], a["prefix_max"], a["slot"], a["P"], a["k"], a["v"], a["kv_len"],
        a["cache_slot"], None, a["B"], a["nh"], a["nkv"], a["hd"], a["n_slots"], a["max_seq"], a["max_len"],
        ctypes.c_float(a["scale"]), None, 1, a["out"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), -1), (dict(kv_len=None), -1), (dict(ws=None), -1), (dict(kp=None), -1),
    (dict(hd=64), -2), (dict(nh=30), -1), (dict(nh=128), -2), (dict(nkv=0), -1),
    (dict(P=-1), -1), (dict(P=601), -1), (dict(slot=1), -1), (dict(slot=-1), -1),
    (dict(max_len=65), -1), (dict(max_len=-1), -1), (dict(B=3), -1), (dict(B=-1), -1),
    (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1),
    (dict(bytes=255), -4), (dict(n_slots=0), -1),
])
def test_decode_refusals(lib, p, kw, status):
    assert _decode(lib, p, **kw) == status
    assert b"attention_prefix_decode" in lib.qmoe_last_error()


@pytest.mark.parametrize("name", ["q", "k", "v", "kp", "vp", "out", "ws"])
def test_decode_alignment(lib, p, name):
    assert _decode(lib, p, **{name: p + 8}) == -3


def test_prefill_and_weights_refusals(lib, p):
    f = ctypes.c_float

    def prefill(q=p, kp=p, P=8, q_start=p, B=2, S=4, nh=32, nkv=4, hd=128, n_slots=2, max_seq=64, scale=0.1, out=p):
        return lib.qmoe_attention_prefix_prefill(q, kp, p, 1, 64, 0, P, p, p, q_start, None, None, B, S, nh, nkv, hd,
                                                 n_slots, max_seq, f(scale), out, None, None)

    for kw, st in ((dict(q=None), -1), (dict(q_start=None), -1), (dict(kp=None), -1), (dict(P=65), -1),
                   (dict(S=65), -1), (dict(S=-1), -1), (dict(nh=31), -1), (dict(nh=128), -2), (dict(hd=96), -2),
                   (dict(B=3), -1), (dict(scale=0.0), -1), (dict(out=p + 4), -3), (dict(kp=p + 8), -3)):
        assert prefill(**kw) == st, kw

    def weights(q=p, lse=p, k=p, w=p, B=2, S=4, nh=32, nkv=4, hd=128, max_seq=64, max_len=64, scale=0.1, size=1 << 30):
        return lib.qmoe_attention_weights(q, lse, k, p, None, None, B, S, nh, nkv, hd, 2, max_seq, max_len, f(scale),
                                          w, 1, p, size, None)

    for kw, st in ((dict(q=None), -1), (dict(lse=None), -1), (dict(w=None), -1), (dict(S=65), -1),
                   (dict(max_len=65), -1), (dict(max_len=3), -1), (dict(hd=64), -2), (dict(nh=6), -1),
                   (dict(scale=-0.1), -1), (dict(q=p + 8), -3), (dict(B=3), -1)):
        assert weights(**kw) == st, kw


def test_evict_refusals(lib, p):
    def evict(k=p, w=p, tok=p, n=p, B=2, nkv=4, hd=128, n_slots=2, max_seq=64, max_len=64, keep=8, recent=4, ws=p,
              size=1 << 20):
        return lib.qmoe_kv_evict(k, p, w, tok, n, None, None, B, nkv, hd, n_slots, max_seq, max_len, keep, recent, ws,
                                 size, None)

    for kw, st in ((dict(k=None), -1), (dict(w=None), -1), (dict(tok=None), -1), (dict(n=None), -1),
                   (dict(hd=64), -2), (dict(keep=-1), -1), (dict(recent=9), -1), (dict(recent=-1), -1),
                   (dict(max_len=65), -1), (dict(B=3), -1), (dict(size=16), -4), (dict(k=p + 8), -3),
                   (dict(ws=None), -1)):
        assert evict(**kw) == st, kw


def test_workspace_queries(lib):
    f = lib.qmoe_attention_prefix_decode_workspace_size
    # a short call is one kernel without parts; a long one keeps some
    assert f(0, 32, 4, 100, 100, 0) == 0 and f(2, 32, 4, 100, 100, 0) == 0 and f(2, 32, 4, 1000, 1000, 0) > 0
    assert f(2, 32, 4, 100, 100, 1) == 2 * 32 * 100 * 4
    # the scores of the own rows come on top: one fp32 per row and query head
    assert f(8, 32, 4, 100, 4096, 1) - f(8, 32, 4, 100, 4096, 0) == 8 * 32 * 4096 * 4
    assert lib.qmoe_kv_evict_workspace_size(2, 4, 1000, 10) == 2 * 4 * (2 + 20) * 4
    assert lib.qmoe_kv_evict_workspace_size(2, 4, 5, 10) == 2 * 4 * (2 + 10) * 4

"""Shared-prefix and bounded-cache operators on batches that make a CTA, a
kernel form or a padding meet more than one sequence, against 64 bits."""
import pytest
import torch

from test_shared_attention_gpu import C, HD, _check_weights, _error, _gen, _i32, _randn

pytestmark = pytest.mark.gpu


def _prompt_weights(B, nh, nkv, S, past, pads, accumulate, seed):
    """The totals of a call next to those in 64 bits.  The log-sum-exp handed
    over is the 64-bit one rounded to fp32: off by at most 2^-24 of itself,
    which the score's 136 * 2^-24 * D of _check_weights' second delta covers
    (|lse| <= D + ln L, L <= 4096, and D > 5 for these inputs)."""
    from nki_moe_7013_b200 import ops

    g = _gen(seed)
    G, L = nh // nkv, past + S
    k, q = _randn(g, B, nkv, L + 3, HD), _randn(g, B * S, nh, HD)
    k[:, :, L:] = float("nan")
    w = torch.rand(B, nkv, L + 3, generator=g, device="cuda")
    before = w.double()
    add = torch.zeros_like(before)
    lse = torch.full((B, S, nh), float("-inf"), device="cuda")
    pos, D = past + torch.arange(S, device="cuda"), 0.0
    for b in range(B):
        lo = min(pads[b], L)
        k[b, :, :lo] = float("nan")
        if not accumulate:
            before[b, :, :L] = 0
        if lo == L:
            continue
        qd = q[b * S:(b + 1) * S].double().view(S, nkv, G, HD).permute(1, 2, 0, 3)  # nkv, G, S
        kd = k[b, :, lo:L].double()
        s = torch.matmul(qd, kd[:, None].transpose(2, 3)) * C
        D = max(D, float((torch.matmul(qd.abs(), kd.abs()[:, None].transpose(2, 3)) * C).max()))
        s.masked_fill_(torch.arange(lo, L, device="cuda")[None] > pos[:, None], float("-inf"))
        row = torch.logsumexp(s, dim=3)
        lse[b] = row.permute(2, 0, 1).reshape(S, nh)
        live = row > float("-inf")
        p = torch.where(live[..., None], torch.exp(s - torch.where(live, row, 0.0)[..., None]), 0.0)
        add[b, :, lo:L] = p.sum(dim=(1, 2))
    assert D > 5
    ops.attention_weights(q, lse.view(B * S, nh), k, _i32([past] * B), B, S, w, accumulate=accumulate,
                          kv_start=_i32(pads))
    assert _error() == 0
    _check_weights(w, add, before, D)


@pytest.mark.parametrize("S,nh", [(1, 32), (4, 32), (16, 32), (16, 20), (17, 32)])
def test_prompt_weights_of_many_short_units(cuda_dev, S, nh):
    """64 sequences, four key blocks each: a CTA takes seven units in turn, most
    of one query tile (17 queries of 8 heads: two)."""
    B, past = 64, 2001
    _prompt_weights(B, nh, 4, S, past, [37 * b if b % 3 else 0 for b in range(B)], S % 2 == 0, seed=S)


@pytest.mark.parametrize("B,nh,nkv,S,past,pads", [
    (3, 16, 2, 2000, 500, [0, 700, 2400]),   # chunks of five query tiles, four units a CTA and more
    (40, 32, 4, 70, 1100, [30 * b for b in range(40)]),  # chunks of units, some sequences nearly all padding
    (1, 8, 8, 4000, 0, [1]),
])
def test_prompt_weights_of_many_units(cuda_dev, B, nh, nkv, S, past, pads):
    _prompt_weights(B, nh, nkv, S, past, pads, False, seed=B)


@pytest.mark.parametrize("nh,nkv", [(34, 2), (17, 1), (256, 1)])
def test_unsupported_head_ratios_are_refused(cuda_dev, nh, nkv):
    """More than 16 query heads per KV head: a named error from the wrappers."""
    from nki_moe_7013_b200 import _C, ops

    bf = dict(dtype=torch.bfloat16, device="cuda")
    k, q = torch.zeros(2, nkv, 600, HD, **bf), torch.zeros(2, nh, HD, **bf)
    n, w = _i32([3, 4]), torch.zeros(2, nkv, 600, device="cuda")
    for call in (lambda: ops.attention_prefix_decode(q, k, k, 600, k, k, n, 600),
                 lambda: ops.attention_decode_weights(q, k, k, n, 600, w),
                 lambda: ops.attention_prefix_prefill(q, k, k, 600, k, k, n, 2, 1),
                 lambda: ops.attention_weights(q, torch.zeros(2, nh, device="cuda"), k, n, 2, 1, w)):
        with pytest.raises(_C.QmoeError, match="query heads per KV head"):
            call()
    assert _error() == 0 and not w.any()


# (B, nkv, prefix, max_len): cut own rows, uncut ones, a prefix in parts of the
# warp-level kernel, on the tcgen05 kernel with cut and uncut own rows, rows of
# many parts, one kernel, no own rows
PATHS = [(3, 4, 0, 700), (74, 4, 0, 1100), (3, 4, 600, 90), (20, 4, 3001, 90), (40, 4, 3001, 90), (2, 4, 5000, 9000),
         (3, 4, 70, 90), (3, 4, 600, 0), (20, 4, 3001, 0)]


def _batch(B, nkv, P, max_len):
    g = _gen(P + max_len)
    k, v = _randn(g, B, nkv, max_len + 8, HD), _randn(g, B, nkv, max_len + 8, HD)
    kp, vp = _randn(g, 1, nkv, max(P, 1), HD), _randn(g, 1, nkv, max(P, 1), HD)
    lens = [max(0, max_len - 3 * b) for b in range(B)]
    return k, v, kp, vp, _randn(g, B, 8 * nkv, HD), lens


@pytest.mark.parametrize("path", PATHS)
def test_decode_reports_bad_lengths_and_slots(cuda_dev, path):
    """A length past max_len or below 0, or a slot outside the cache: device
    error 4 whatever form the call takes, and what a sequence without own rows
    gives; the others' outputs and weights as ever."""
    from nki_moe_7013_b200 import ops

    B, nkv, P, max_len = path
    k, v, kp, vp, q, lens = _batch(*path)
    bad = B - 1
    empty = lens[:bad] + [0]

    def call(lens, slots, weights):
        w = torch.full((B, nkv, max_len + 8), 0.5, device="cuda") if weights else None
        out = ops.attention_prefix_decode(q, kp, vp, P, k, v, _i32(lens), max_len, cache_slot=_i32(slots), weights=w)
        return out, w

    for weights in (False, True):
        want, want_w = call(empty, None, weights)
        assert _error() == 0
        for length, slot in ((max_len + 1, bad), (-1, bad), (min(5, max_len), B), (min(5, max_len), -1)):
            out, w = call(lens[:bad] + [length], list(range(bad)) + [slot], weights)
            assert _error() == 4, (length, slot, weights)
            assert torch.equal(out, want)
            assert w is None or torch.equal(w, want_w)


@pytest.mark.parametrize("path", PATHS)
def test_decode_reports_a_slot_given_twice(cuda_dev, path):
    """Weights of two entries of one slot: device error 4 and the first entry's
    weights alone, also where one of the two holds no own rows."""
    from nki_moe_7013_b200 import ops

    B, nkv, P, max_len = path
    k, v, kp, vp, q, lens = _batch(*path)
    for first, second in ((lens[0], lens[1]), (lens[0], 0), (0, lens[1])):
        n = [first, second] + lens[2:]
        w = torch.zeros(B, nkv, max_len + 8, device="cuda")
        slots = list(range(B))
        ops.attention_prefix_decode(q, kp, vp, P, k, v, _i32(n), max_len, cache_slot=_i32(slots), weights=w)
        assert _error() == 0
        twice = torch.zeros_like(w)
        slots[1] = 0
        ops.attention_prefix_decode(q, kp, vp, P, k, v, _i32(n), max_len, cache_slot=_i32(slots), weights=twice)
        assert _error() == 4, (first, second)
        assert torch.equal(twice[0], w[0]) and not twice[1].any() and torch.equal(twice[2:], w[2:])


def test_one_padding_token_behind_a_prefix(cuda_dev):
    """Prompts fed a token at a time, the second sequence's first two tokens
    paddings: zero rows for these, and each sequence as if it were run whole."""
    from helpers import MAX_REL, activations, max_rel_err, to_f32_np
    from nki_moe_7013_b200.attention import Qwen3MoeAttention
    from nki_moe_7013_b200.config import Qwen3MoeConfig

    cfg = Qwen3MoeConfig()
    attn, H = Qwen3MoeAttention(cfg, device=cuda_dev, seed=13), cfg.hidden_size
    P, B, S, pads = 21, 2, 5, [0, 2]
    xp = activations(21, P, H, cuda_dev).view(1, P, H)
    x = activations(22, B * S, H, cuda_dev).view(B, S, H)
    prefix = attn(xp)[1].as_prefix()
    for track in (False, True):
        cache = attn.new_cache(B, S, track=track)
        mask = (torch.arange(S)[None] >= torch.tensor(pads)[:, None]).int()
        got = torch.cat([attn(x[:, i:i + 1], None, cache, attention_mask=mask[:, :i + 1], prefix=prefix)[0]
                         for i in range(S)], dim=1)
        for b in range(B):
            assert not got[b, :pads[b]].any()
            whole, _ = attn(torch.cat([xp, x[b:b + 1, pads[b]:]], dim=1))
            assert max_rel_err(to_f32_np(got[b, pads[b]:]), to_f32_np(whole[0, P:])) <= MAX_REL
        if track:
            assert not cache.weights[1, :, :pads[1]].any()
    assert _error() == 0


def test_another_prefix_of_the_same_length_is_refused(cuda_dev):
    from helpers import activations
    from nki_moe_7013_b200.attention import Qwen3MoeAttention
    from nki_moe_7013_b200.config import Qwen3MoeConfig

    cfg = Qwen3MoeConfig()
    attn, H = Qwen3MoeAttention(cfg, device=cuda_dev, seed=14), cfg.hidden_size
    a, b = (attn(activations(s, 9, H, cuda_dev).view(1, 9, H))[1].as_prefix() for s in (31, 32))
    x = activations(33, 8, H, cuda_dev).view(2, 4, H)
    cache = attn.new_cache(2, 8)
    attn(x, None, cache, prefix=a)
    with pytest.raises(ValueError, match="another prefix"):
        attn(x[:, :1], None, cache, prefix=b)
    assert cache.lengths == [4, 4]
    attn(x[:, :1], None, cache, prefix=a)
    attn(x, None, cache.reset(), prefix=b)
    assert _error() == 0


def test_a_session_steps_behind_the_prefix_of_its_caches(cuda_dev):
    """Prompts prefilled into a session's caches behind another prefix than the
    session's, or behind none: refused before the first step."""
    from nki_moe_7013_b200.config import Qwen3MoeConfig
    from nki_moe_7013_b200.model import DecodeSession, Qwen3MoeModel

    model = Qwen3MoeModel(Qwen3MoeConfig(), num_layers=1, vocab_size=512, device=cuda_dev, seed=15)
    ids = torch.arange(40, device=cuda_dev)
    a, b = model.prefill_prefix(ids[:20]), model.prefill_prefix(ids[20:])
    for mine, other in ((a, b), (a, None), (None, a)):
        for first in ("step", "capture"):
            sess = DecodeSession(model, 2, context=6, max_new=4, prefix=mine, fill_random=False)
            model.forward(ids[:12].view(2, 6), sess.caches, prefix=other)
            with pytest.raises(ValueError, match="another prefix"):
                getattr(sess, first)()
            assert sess.steps_done == 0
        for c in sess.caches:
            c.reset()
        model.forward(ids[:12].view(2, 6), sess.caches, prefix=mine)
        sess.step()
        sess.step()
        DecodeSession(model, 2, context=6, max_new=4, prefix=mine).step()  # random rows follow the session's prefix
    assert _error() == 0


def test_append_refuses_rows_of_other_heads(cuda_dev):
    """Totals and tokens of a cache with fewer KV heads than the tokens have
    would be written past their end."""
    from nki_moe_7013_b200 import ops

    g = _gen(16)
    nh, nkv, T = 8, 4, 3
    qkv, ones, freq = _randn(g, T, (nh + 2 * nkv) * HD), torch.ones(HD, device="cuda"), torch.ones(64, device="cuda")
    for heads, v_heads in ((2, 2), (4, 2)):
        k, v = _randn(g, 1, heads, 8, HD), _randn(g, 1, v_heads, 8, HD)
        tok, w = torch.zeros(1, heads, 8, dtype=torch.int32, device="cuda"), torch.zeros(1, heads, 8, device="cuda")
        with pytest.raises(ValueError, match="KV heads"):
            ops.qk_norm_rope(qkv, _i32([0, 1, 2]), ones, ones, freq, nh, nkv, 1e-6, k, v, row_tokens=tok, row_weights=w)
    with pytest.raises(ValueError, match="one row per token"):
        ops.qk_norm_rope(qkv, _i32([0, 1, 2]), ones, ones, freq, nh, nkv, 1e-6, k, k, cache_rows=_i32([0, 1]))
    assert _error() == 0

"""Shared prefixes and evicting caches in the attention layer, the model and
the decode session: against the same tokens without a prefix, against caches
holding the kept rows alone, and graph replay against eager steps."""
import pytest
import torch

from helpers import MAX_REL, activations, max_rel_err, to_f32_np

pytestmark = pytest.mark.gpu


def _attn(dev, seed=2):
    from nki_moe_7013_b200.attention import Qwen3MoeAttention
    from nki_moe_7013_b200.config import Qwen3MoeConfig

    cfg = Qwen3MoeConfig()
    return Qwen3MoeAttention(cfg, device=dev, seed=seed), cfg.hidden_size


@pytest.mark.parametrize("P", [1, 150])
def test_attention_behind_a_prefix_equals_the_whole_sequence(cuda_dev, P):
    """Prefill, a second prefill and decode steps behind a prefix, some
    sequences left-padded, against each sequence run whole."""
    attn, H = _attn(cuda_dev)
    B, S, pads = 3, 40, [0, 7, 0]
    xp = activations(1, P, H, cuda_dev).view(1, P, H)
    x = activations(2, B * (S + 12), H, cuda_dev).view(B, S + 12, H)
    steps = [(0, S), (S, S + 9), (S + 9, S + 10), (S + 10, S + 11), (S + 11, S + 12)]
    _, pc = attn(xp)
    prefix, cache = pc.as_prefix(), attn.new_cache(B, S + 12)
    mask = torch.ones(B, S, dtype=torch.int32)
    mask[1, :pads[1]] = 0
    got = []
    for i, (a, b) in enumerate(steps):
        pos = torch.arange(a, b)[None] + P - torch.tensor(pads)[:, None]
        out, _ = attn(x[:, a:b], pos, cache, attention_mask=mask if i == 0 else None, prefix=prefix)
        got.append(out)
    got = torch.cat(got, dim=1)
    for b in range(B):
        whole, _ = attn(torch.cat([xp, x[b:b + 1, pads[b]:]], dim=1))
        assert max_rel_err(to_f32_np(got[b, pads[b]:]), to_f32_np(whole[0, P:])) <= MAX_REL
    from nki_moe_7013_b200 import _C

    assert _C.device_error() == 0


def test_a_first_chunk_of_paddings_behind_a_prefix(cuda_dev):
    """Prompts in two chunks, the second sequence's first token in the second
    one, against each sequence run whole."""
    attn, H = _attn(cuda_dev, seed=9)
    P, B, S, cut, pads = 33, 2, 24, 10, [3, 14]
    xp = activations(11, P, H, cuda_dev).view(1, P, H)
    x = activations(12, B * S, H, cuda_dev).view(B, S, H)
    prefix = attn(xp)[1].as_prefix()
    cache = attn.new_cache(B, S)
    mask = (torch.arange(S)[None] >= torch.tensor(pads)[:, None]).int()
    got = torch.cat([attn(x[:, :cut], None, cache, attention_mask=mask[:, :cut], prefix=prefix)[0],
                     attn(x[:, cut:], None, cache, attention_mask=mask, prefix=prefix)[0]], dim=1)
    for b in range(B):
        whole, _ = attn(torch.cat([xp, x[b:b + 1, pads[b]:]], dim=1))
        assert max_rel_err(to_f32_np(got[b, pads[b]:]), to_f32_np(whole[0, P:])) <= MAX_REL


def test_prefix_refusals(cuda_dev):
    attn, H = _attn(cuda_dev)
    x = activations(3, 2 * 6, H, cuda_dev).view(2, 6, H)
    _, pc = attn(x[:1])
    cache = attn.new_cache(2, 20)
    own = attn.new_cache(3, 20)
    attn(x[:1], None, own)
    with pytest.raises(ValueError, match="batch's own"):
        attn(x[:, :1], None, own, prefix=own.as_prefix())
    attn(x, None, cache)
    with pytest.raises(ValueError, match="another prefix"):
        attn(x, None, cache, prefix=pc.as_prefix())
    with pytest.raises(ValueError, match="position_ids"):
        attn(x, torch.arange(6).expand(2, 6), attn.new_cache(2, 20), prefix=pc.as_prefix())
    tracked = attn.new_cache(2, 20, track=True)
    attn(x, None, tracked)
    tracked.evict(4)
    with pytest.raises(ValueError, match="evicted"):
        attn(x, None, tracked, attention_mask=torch.ones(2, 10))


@pytest.mark.parametrize("P,score", [(0, None), (70, None), (70, 16)])
def test_evicted_cache_attends_to_the_kept_rows(cuda_dev, P, score):
    """Prefix, prompts (one left-padded) that score their rows, an eviction,
    more tokens, a second eviction, a decode step: each later output equals
    that of a cache holding the kept rows alone, in token order."""
    from nki_moe_7013_b200 import _C

    attn, H = _attn(cuda_dev, seed=4)
    B, S, keep, recent, pads = 2, 96, 40, 9, [0, 11]
    nkv, G = 4, 8
    prefix = None
    if P:
        prefix = attn(activations(5, P, H, cuda_dev).view(1, P, H))[1].as_prefix()
    cache = attn.new_cache(B, S + 8, track=True, score_queries=score)
    x = activations(6, B * (S + 20), H, cuda_dev).view(B, S + 20, H)
    mask = torch.ones(B, S, dtype=torch.int32)
    mask[1, :pads[1]] = 0
    attn(x[:, :S], None, cache, attention_mask=mask, prefix=prefix)
    torch.cuda.synchronize()
    if not P:
        # every query's probabilities sum to 1 over its own rows
        want = torch.tensor([[G * min(score or S, S - p)] * nkv for p in pads], dtype=torch.float32, device=cuda_dev)
        assert torch.allclose(cache.weights[:, :, :S].sum(dim=2), want, rtol=2.0 ** -12)
    assert not cache.weights[1, :, :pads[1]].any()

    def reference(k0, v0, tok0, at):
        """A cache of the kept rows in token order, entered at the same position."""
        ref = attn.new_cache(B, S + 8, track=True)
        for b in range(B):
            n = cache.lengths[b]
            for g in range(nkv):
                kept = torch.sort(cache.tokens[b, g, :n]).values
                rows = {int(t): r for r, t in enumerate(tok0[b, g].tolist()) if t >= 0}
                idx = torch.tensor([rows[int(t)] for t in kept.tolist()], device=cuda_dev)
                ref.k[b, g, :n], ref.v[b, g, :n], ref.tokens[b, g, :n] = k0[b, g, idx], v0[b, g, idx], kept
            ref.lengths[b], ref.offset[b], ref.dropped[b] = n, at[b] - n, 1
            ref.prefix_len[b] = P
        return ref

    pos = [P + S - (pads[b] if P else 0) for b in range(B)]
    done = S
    for new in (4, 1, 1):
        before = [t.clone() for t in (cache.k, cache.v, cache.tokens)]
        for b in range(B):
            before[2][b, :, :cache.pad[b]] = -1
        old_w = cache.weights.clone()
        cache.evict(keep, recent)
        assert cache.lengths == [keep, keep]
        for b in range(B):
            for g in range(nkv):
                kept = set(cache.tokens[b, g, :keep].tolist())
                assert len(kept) == keep and set(range(pos[b] - recent, pos[b])) <= kept
                # no row left behind outweighs a kept one that is not recent
                tok, w = before[2][b, g], old_w[b, g]
                stay = torch.tensor([int(t) in kept for t in tok.tolist()], device=cuda_dev) & (tok >= 0)
                gone = ~stay & (tok >= 0)
                old = stay & (tok < pos[b] - recent)
                if gone.any() and old.any():
                    assert float(w[gone].max()) <= float(w[old].min())
        ref = reference(*before, pos)
        got, _ = attn(x[:, done:done + new], None, cache, prefix=prefix)
        want, _ = attn(x[:, done:done + new], None, ref, prefix=prefix)
        assert max_rel_err(to_f32_np(got), to_f32_np(want)) <= MAX_REL
        done += new
        pos = [p + new for p in pos]
        assert [cache.lengths[b] + cache.offset[b] for b in range(B)] == pos
    assert _C.device_error() == 0


def _small_model(dev, seed=3):
    from nki_moe_7013_b200.config import Qwen3MoeConfig
    from nki_moe_7013_b200.model import Qwen3MoeModel

    return Qwen3MoeModel(Qwen3MoeConfig(), num_layers=2, vocab_size=2048, device=dev, seed=seed)


def test_session_behind_a_prefix_matches_the_module_path(cuda_dev):
    from nki_moe_7013_b200 import _C
    from nki_moe_7013_b200.model import DecodeSession

    model = _small_model(cuda_dev)
    ids = torch.randint(0, 2048, (100,), device=cuda_dev)
    prefix = model.prefill_prefix(ids)
    B, ctx = 2, 30
    sess = DecodeSession(model, B, context=ctx, max_new=8, seed=5, split_k=False, prefix=prefix)
    caches = model.new_caches(B, ctx + 8)
    for c, s in zip(caches, sess.caches):
        c.k.copy_(s.k)
        c.v.copy_(s.v)
        c.lengths, c.prefix_len, c.offset = [ctx] * B, [100] * B, [100] * B
    tokens = sess.tokens.clone()
    ref, _ = model.forward(tokens.reshape(B, 1), past_key_values=caches, prefix=prefix)
    sess.step()
    assert _C.device_error() == 0
    assert max_rel_err(to_f32_np(sess.logits), to_f32_np(ref.reshape(B, -1))) <= MAX_REL
    assert sess.positions.tolist() == [131, 131] and sess.rows.tolist() == [31, 31]
    with pytest.raises(ValueError, match="layers"):
        model.forward(tokens.reshape(B, 1), prefix=prefix[:1])
    with pytest.raises(ValueError, match="layers"):
        DecodeSession(model, B, context=ctx, max_new=8, prefix=prefix[:1])


@pytest.mark.parametrize("with_prefix", [False, True])
def test_bounded_session_replay_matches_eager_steps(cuda_dev, with_prefix):
    """Two sequences (the deterministic MoE sizes) past the end of their
    caches: captured and eager sessions hold the same tokens, rows and totals
    after several evictions, and every head holds the newest tokens."""
    from nki_moe_7013_b200 import _C
    from nki_moe_7013_b200.model import DecodeSession

    model = _small_model(cuda_dev, seed=6)
    prefix = model.prefill_prefix(torch.randint(0, 2048, (33,), device=cuda_dev)) if with_prefix else None
    P = 33 if with_prefix else 0
    ctx, keep, recent, n = 20, 15, 6, 25
    kw = dict(context=ctx, max_new=5, seed=7, prefix=prefix, keep=keep, recent=recent)
    eager, graphed = DecodeSession(model, 2, **kw), DecodeSession(model, 2, **kw)
    assert torch.equal(eager.tokens, graphed.tokens)
    graphed.capture()  # runs one step
    eager.step()
    for _ in range(n - 1):
        eager.step()
        graphed.step()
    torch.cuda.synchronize()
    assert _C.device_error() == 0
    assert torch.equal(eager.tokens, graphed.tokens) and torch.equal(eager.logits, graphed.logits)
    assert eager.positions.tolist() == [P + ctx + n] * 2
    used = eager.rows_used
    assert used == graphed.rows_used and eager.rows.tolist() == [used] * 2
    assert eager.kv_len.tolist() == [used + 1] * 2 and keep < used <= ctx + 5
    for a, b in zip(eager.caches, graphed.caches):
        assert torch.equal(a.tokens, b.tokens) and torch.equal(a.weights, b.weights)
        assert torch.equal(a.k[:, :, :used], b.k[:, :, :used]) and torch.equal(a.v[:, :, :used], b.v[:, :, :used])
        for row in a.tokens[:, :, :used].reshape(-1, used).tolist():
            assert len(set(row)) == used and set(range(P + ctx + n - recent, P + ctx + n)) <= set(row)
        assert bool((a.tokens[:, :, used:] == -1).all()) and not a.weights[:, :, used:].any()


@pytest.mark.parametrize("keep", [None, 24])
def test_session_after_its_prompts(cuda_dev, keep):
    """Prompts behind a prefix prefilled into a session's caches, then steps,
    against the module path over the same tokens (and, with ``keep``, the same
    evictions)."""
    from nki_moe_7013_b200 import _C
    from nki_moe_7013_b200.model import DecodeSession

    model = _small_model(cuda_dev, seed=10)
    prefix = model.prefill_prefix(torch.randint(0, 2048, (70,), device=cuda_dev))
    B, S = 2, 30
    ids = torch.randint(0, 2048, (B, S), device=cuda_dev)
    sess = DecodeSession(model, B, context=S, max_new=3, prefix=prefix, keep=keep, recent=8 if keep else 0,
                         fill_random=False, split_k=False)
    logits, _ = model.forward(ids, sess.caches, last_only=True, prefix=prefix)
    caches = model.new_caches(B, S + 3, track=keep is not None)
    ref, _ = model.forward(ids, caches, last_only=True, prefix=prefix)
    assert max_rel_err(to_f32_np(logits), to_f32_np(ref)) <= MAX_REL
    sess.tokens.copy_(logits[:, -1].argmax(-1))
    for step in range(3 if keep is None else 8):
        if keep is not None and caches[0].lengths[0] == S + 3:
            for c, s in zip(caches, sess.caches):  # near ties may fall apart: the totals that decide are shared
                c.weights.copy_(s.weights)
                c.evict(keep, recent=8)
        tokens = sess.tokens.clone()
        ref, _ = model.forward(tokens.reshape(B, 1), caches, prefix=prefix)
        sess.step()
        assert max_rel_err(to_f32_np(sess.logits), to_f32_np(ref.reshape(B, -1))) <= MAX_REL, step
    for c, s in zip(caches, sess.caches):
        if keep is not None:
            assert torch.equal(c.tokens, s.tokens)
    assert _C.device_error() == 0


def test_session_refusals(cuda_dev):
    from nki_moe_7013_b200.model import DecodeSession

    model = _small_model(cuda_dev, seed=8)
    for keep, recent in ((25, 0), (10, 11), (10, -1)):
        with pytest.raises(ValueError, match="recent"):
            DecodeSession(model, 1, context=20, max_new=5, keep=keep, recent=recent)

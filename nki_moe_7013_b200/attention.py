"""Attention sub-layer of the Qwen3-MoE decoder layer (secondary target).

``Qwen3MoeAttention.forward(hidden_states, position_ids=None,
past_key_value=None, attention_mask=None) -> (out, present_kv)`` mirrors
NxDI's NeuronQwen3MoEAttention (qwen.py:313-341): fused QKV projection,
per-head q/k RMSNorm (qwen.py:333-335), RoPE theta 1e6 (qwen.py:315-319),
causal GQA over a KV cache, o_proj.  Positions follow the HF convention (the
position of a new token = the number of tokens already cached).

``attention_mask``: causal masking is built in; a 2D key-padding mask
(batch, cached + new tokens; 1 = token, 0 = padding) with LEFT padding only
(each row zeros then ones) is honoured -- the form NxDI / HF batch prefill
uses.  The cache remembers each slot's padding, so later decode steps keep
masking it.  RoPE is applied at the cache row; HF applies it at the
pad-shifted position (cumsum(mask) - 1), and since the rotary score depends
only on the difference of two positions the attention output is the same up
to fp32 rounding.  Padding query rows get a zero attention output.  Any
other mask (holes, right padding, 4D) is refused with a ValueError.

``prefix`` (a ``SharedPrefix``): rows that every sequence of the batch sees
before its own -- a system prompt stored once, in a cache of its own, instead
of in every slot.  New tokens sit at positions ``prefix.length`` + their own
(left padding not counted), and both attention forms read the prefix once for
the batch.

A cache made with ``track=True`` also holds, for every row and KV head, the
attention weight it has received so far and its token's position; its
``evict(keep, recent)`` brings it down to ``keep`` rows per KV head, the most
recent ones and those of the largest weight, and later tokens are appended
behind them at their true positions.

All kernels come from the CUDA library: tcgen05 projections (``ops.linear``),
the fused QK-norm + RoPE + cache append, flash-prefill / split-KV
flash-decode, their forms over a shared prefix, and the eviction.
"""
from __future__ import annotations

import copy
from dataclasses import dataclass
from typing import List, Optional

import torch
from torch import nn

from . import ops
from .config import Qwen3MoeConfig


def rope_inv_freq(head_dim: int, theta: float, device) -> torch.Tensor:
    """fp32 inverse frequencies, computed the way HF / NxDI RotaryEmbedding do."""
    return (1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.int64).float() / head_dim))).to(device)


class KVCache:
    """K and V caches (slots, nkv, max_seq, head_dim) bf16 plus per-slot lengths.

    ``lengths`` is kept on the host (it drives shapes and launch sizes) and
    mirrored on the device for the kernels.

    ``track``: the cache can evict.  It then holds every row's accumulated
    attention weight (``weights``, fp32) and its token's position (``tokens``,
    int32), both (slots, nkv, max_seq); each KV head keeps rows of its own, so
    after an eviction the heads' rows hold different tokens.  Calls with
    several new tokens add the weights of the last ``score_queries`` of them
    (None: of all)."""

    def __init__(self, n_slots: int, nkv: int, max_seq: int, head_dim: int, device="cuda", track: bool = False,
                 score_queries: Optional[int] = None):
        if score_queries is not None and score_queries < 1:
            raise ValueError("score_queries must be at least 1")
        self.k = torch.zeros((n_slots, nkv, max_seq, head_dim), dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)
        self.lengths: List[int] = [0] * n_slots
        self.pad: List[int] = [0] * n_slots      # leading padding rows per slot
        self._clear_positions(n_slots)
        self.max_seq = max_seq
        self.score_queries = score_queries
        self.weights = torch.zeros(self.k.shape[:3], dtype=torch.float32, device=device) if track else None
        self.tokens = (torch.full(self.k.shape[:3], -1, dtype=torch.int32, device=device) if track else None)

    def _clear_positions(self, n_slots: int) -> None:
        self.offset: List[int] = [0] * n_slots      # a new row's position less the row
        self.prefix_len: List[int] = [0] * n_slots  # rows of the shared prefix the slot was filled behind
        self.behind: List[Optional["SharedPrefix"]] = [None] * n_slots  # that prefix (None: none, or not known)
        self.lead: List[int] = [0] * n_slots        # leading paddings the slot was filled with
        self.dropped: List[int] = [0] * n_slots     # rows evicted so far

    def __deepcopy__(self, memo) -> "KVCache":
        # a copy stays behind the same prefix, which is not copied with it
        for p in self.behind:
            if p is not None:
                memo.setdefault(id(p), p)
        c = memo[id(self)] = object.__new__(type(self))
        c.__dict__.update(copy.deepcopy(self.__dict__, memo))
        return c

    @property
    def tracked(self) -> bool:
        return self.weights is not None

    @property
    def n_slots(self) -> int:
        return self.k.shape[0]

    def fill_random(self, length: int, seed: int = 0) -> "KVCache":
        """Config-2 setup: every slot holds `length` tokens of ~N(0,1) bf16."""
        g = torch.Generator(device=self.k.device)
        g.manual_seed(seed)
        self.k[:, :, :length].normal_(generator=g)
        self.v[:, :, :length].normal_(generator=g)
        self.lengths = [length] * self.n_slots
        self.pad = [0] * self.n_slots
        self._clear_positions(self.n_slots)
        if self.tracked:
            self.weights.zero_()
            self.tokens.fill_(-1)
            self.tokens[:, :, :length] = torch.arange(length, dtype=torch.int32, device=self.k.device)
        return self

    def reset(self) -> "KVCache":
        """Empty every slot (the contents are overwritten by the next appends)."""
        self.lengths = [0] * self.n_slots
        self.pad = [0] * self.n_slots
        self._clear_positions(self.n_slots)
        return self

    def _follow(self, prefix_len: int, pads: Optional[List[int]], B: int,
                prefix: Optional["SharedPrefix"] = None) -> None:
        """The host's side of a call that appends to slots 0 .. B-1 behind
        ``prefix_len`` shared rows (those of ``prefix``): refuses what the rows
        already there contradict, and records paddings (``pads``; None: as they
        are), the prefix and the distance of a new row's position from the row."""
        for b in range(B):
            fresh = self.lengths[b] == 0 and self.dropped[b] == 0
            none_yet = self.dropped[b] == 0 and self.lengths[b] <= self.pad[b]
            was = self.behind[b]
            if not fresh and (self.prefix_len[b] != prefix_len or not (
                    none_yet or was is None or prefix is None or was.same_rows(prefix))):
                raise ValueError("the cache was filled behind another prefix (or none)")
            if prefix_len and pads is not None and pads[b] != self.pad[b] and pads[b] < self.lengths[b]:
                raise ValueError("attention_mask: behind a prefix the paddings come with a sequence's first tokens")
        for b in range(B):
            if pads is not None:
                self.pad[b] = self.lead[b] = pads[b]
            if self.dropped[b] == 0 and self.lengths[b] <= self.pad[b]:  # no token yet
                # behind a prefix the distance to it counts, so paddings are left out of the positions
                self.prefix_len[b] = prefix_len
                self.behind[b] = prefix if prefix_len else None
                self.offset[b] = prefix_len - self.pad[b] if prefix_len else 0

    def as_prefix(self, slot: int = 0) -> "SharedPrefix":
        """The rows of one slot as a prefix for other sequences (no copy: the
        slot must not change while the prefix is in use)."""
        if not 0 <= slot < self.n_slots:
            raise ValueError(f"slot {slot} of a cache of {self.n_slots}")
        if self.pad[slot] or self.offset[slot] or self.dropped[slot]:
            raise ValueError("a padded slot, one behind a prefix or one that evicted rows cannot be a prefix")
        return SharedPrefix(self.k, self.v, self.lengths[slot], slot)

    def evict(self, keep: int, recent: int = 0) -> "KVCache":
        """Bring every slot down to min(keep, its tokens) rows per KV head: the
        ``recent`` newest tokens and those of the largest accumulated weight
        (``ops.kv_evict``).  Paddings leave; the rows' order changes."""
        if not self.tracked:
            raise ValueError("only a cache made with track=True can evict")
        if not 0 <= recent <= keep:
            raise ValueError("evict needs 0 <= recent <= keep")
        dev = self.k.device
        kv_len = torch.tensor(self.lengths, dtype=torch.int32).to(dev, non_blocking=True)
        start = torch.tensor(self.pad, dtype=torch.int32).to(dev, non_blocking=True) if any(self.pad) else None
        ops.kv_evict(self.k, self.v, self.weights, self.tokens, kv_len, max(self.lengths), keep, recent=recent,
                     kv_start=start)
        self._evicted(keep)
        return self

    def _evicted(self, keep: int) -> None:
        """The host's side of an eviction: lengths, paddings, and the distance
        of a new row's position from the row."""
        for b, n in enumerate(self.lengths):
            self.lengths[b] = min(keep, n - self.pad[b])
            self.offset[b] += n - self.lengths[b]
            self.dropped[b] += n - self.lengths[b]
            self.pad[b] = 0


@dataclass
class SharedPrefix:
    """Rows 0 .. length-1 of slot ``slot`` of a K / V cache (n, nkv, rows, 128)
    bf16, rotated for positions 0 .. length-1, that every sequence of a batch
    sees before its own rows.  Caches filled behind it hold on to it: their
    later calls take the same prefix, where it was."""

    k: torch.Tensor
    v: torch.Tensor
    length: int
    slot: int = 0

    def same_rows(self, other: "SharedPrefix") -> bool:
        """The same rows of the same memory (contents are not compared)."""
        return (self.length == other.length and self.slot == other.slot and self.k.shape == other.k.shape
                and self.k.data_ptr() == other.k.data_ptr() and self.v.data_ptr() == other.v.data_ptr())


def left_padding(attention_mask: Optional[torch.Tensor], B: int, S: int, L0: List[int]) -> Optional[List[int]]:
    """Leading padding count per sequence of a 2D key-padding mask (B, L0+S),
    1 = token, 0 = padding; None for no mask.  Refuses every other mask."""
    if attention_mask is None:
        return None
    if attention_mask.dim() != 2:
        raise ValueError("attention_mask: only a 2D (batch, cached + new tokens) key-padding mask is "
                         "supported; causal masking is built in")
    m = (attention_mask != 0).to(torch.int32).cpu()
    if m.shape[0] != B:
        raise ValueError(f"attention_mask has {m.shape[0]} rows for a batch of {B}")
    L = m.shape[1]
    if any(l0 + S != L for l0 in L0):
        raise ValueError(f"attention_mask must cover each sequence's cached and new tokens ({L0[0] + S}), "
                         f"got {L}")
    if L > 1 and not bool(torch.all(m[:, 1:] >= m[:, :-1])):
        raise ValueError("attention_mask: only left padding (zeros before ones in every row) is supported")
    return [int(v) for v in (L - m.sum(1)).tolist()]


@dataclass
class AttnWeights:
    wqkv: torch.Tensor     # (nh*hd + 2*nkv*hd, H) bf16: q rows, k rows, v rows
    wo: torch.Tensor       # (H, nh*hd) bf16
    q_norm: torch.Tensor   # (hd,) fp32
    k_norm: torch.Tensor   # (hd,) fp32

    @staticmethod
    def random(cfg: Qwen3MoeConfig, seed: int = 0, device="cuda", std: float = 0.02) -> "AttnWeights":
        from .synth import normal_bf16_device

        H, nh, nkv, hd = cfg.hidden_size, cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        g = torch.Generator(device=device)
        g.manual_seed(seed * 10 + 7)
        return AttnWeights(
            normal_bf16_device(seed * 10 + 5, ((nh + 2 * nkv) * hd, H), std, device),
            normal_bf16_device(seed * 10 + 6, (H, nh * hd), std, device),
            (1.0 + 0.1 * torch.randn(hd, generator=g, device=device)).float(),
            (1.0 + 0.1 * torch.randn(hd, generator=g, device=device)).float())

    @staticmethod
    def from_hf(attn, device="cuda") -> "AttnWeights":
        """From a transformers Qwen3MoeAttention (q/k/v/o_proj, q_norm, k_norm)."""
        bf = dict(device=device, dtype=torch.bfloat16)
        wqkv = torch.cat([attn.q_proj.weight, attn.k_proj.weight, attn.v_proj.weight], 0)
        return AttnWeights(wqkv.detach().to(**bf).contiguous(), attn.o_proj.weight.detach().to(**bf).contiguous(),
                           attn.q_norm.weight.detach().float().to(device).contiguous(),
                           attn.k_norm.weight.detach().float().to(device).contiguous())


class StageTimer:
    """Optional per-stage CUDA events: ``with timer("name"):`` records an
    event pair around the kernels issued inside on the current stream and
    appends (name, start, end) to ``timer.marks``.  A ``None`` timer costs
    nothing (``stage(None, name)``)."""

    def __init__(self):
        self.marks = []

    def __call__(self, name: str):
        return _Stage(self, name)

    def totals_ms(self) -> dict:
        """Summed elapsed time per stage name (synchronise first)."""
        out: dict = {}
        for name, a, b in self.marks:
            out[name] = out.get(name, 0.0) + a.elapsed_time(b)
        return out


class _Stage:
    def __init__(self, timer, name):
        self.timer, self.name = timer, name

    def __enter__(self):
        if self.timer is not None:
            self.a = torch.cuda.Event(enable_timing=True)
            self.b = torch.cuda.Event(enable_timing=True)
            self.a.record()
        return self

    def __exit__(self, *exc):
        if self.timer is not None:
            self.b.record()
            self.timer.marks.append((self.name, self.a, self.b))
        return False


def stage(timer: Optional[StageTimer], name: str) -> _Stage:
    return _Stage(timer, name)


class Qwen3MoeAttention(nn.Module):
    def __init__(self, cfg: Qwen3MoeConfig, weights: Optional[AttnWeights] = None, device="cuda",
                 seed: int = 0):
        super().__init__()
        if cfg.head_dim != 128:
            raise ValueError("the attention kernels are built for head_dim 128")
        self.cfg = cfg
        self.w = weights if weights is not None else AttnWeights.random(cfg, seed, device)
        self.inv_freq = rope_inv_freq(cfg.head_dim, cfg.rope_theta, self.w.wqkv.device)
        self._decode_ws: Optional[torch.Tensor] = None

    def new_cache(self, n_slots: int, max_seq: int, track: bool = False,
                  score_queries: Optional[int] = None) -> KVCache:
        return KVCache(n_slots, self.cfg.num_key_value_heads, max_seq, self.cfg.head_dim, self.w.wqkv.device,
                       track=track, score_queries=score_queries)

    def forward(self, hidden_states: torch.Tensor, position_ids: Optional[torch.Tensor] = None,
                past_key_value: Optional[KVCache] = None, timer: Optional[StageTimer] = None,
                attention_mask: Optional[torch.Tensor] = None, prefix: Optional[SharedPrefix] = None):
        cfg = self.cfg
        B, S, H = hidden_states.shape
        dev = hidden_states.device
        cache = past_key_value if past_key_value is not None else self.new_cache(B, S)
        if cache.n_slots < B:
            raise ValueError("KV cache has fewer slots than the batch")
        L0 = cache.lengths[:B]
        if max(L0) + S > cache.max_seq:
            raise ValueError("KV cache is full")
        x2d = hidden_states.reshape(B * S, H).to(torch.bfloat16).contiguous()
        P = prefix.length if prefix is not None else 0
        if P and prefix.k is cache.k and prefix.slot < B:
            raise ValueError("the prefix's slot is one of the batch's own")
        if attention_mask is not None and any(cache.dropped[:B]):
            raise ValueError("attention_mask: the cache evicted rows (its paddings among them); pass no mask")
        kept = None
        if position_ids is not None:
            kept = {name: list(getattr(cache, name)) for name in ("pad", "lead", "prefix_len", "behind", "offset")}
        cache._follow(P, left_padding(attention_mask, B, S, L0), B, prefix)
        pad_now = cache.pad[:B]
        rows = (torch.tensor(L0, dtype=torch.int32).unsqueeze(1) + torch.arange(S, dtype=torch.int32))
        pos = rows + torch.tensor(cache.offset[:B], dtype=torch.int32).unsqueeze(1)
        # own rows apart from positions: behind a prefix, or in a cache that may evict
        apart = P > 0 or cache.tracked
        if position_ids is not None:
            given = position_ids.reshape(B, S).to(torch.int32).cpu()
            shifted = pos - torch.tensor(cache.lead[:B], dtype=torch.int32).unsqueeze(1)
            if P:
                shifted = pos  # paddings are left out already
            real = rows >= torch.tensor(pad_now, dtype=torch.int32).unsqueeze(1)  # padding tokens may carry any position
            if not (torch.equal(given, pos) or bool(torch.all((given == shifted) | ~real))):
                vars(cache).update(kept)  # a refused call is not remembered
                raise ValueError("position_ids must continue each sequence's cache contiguously (or, with left "
                                 "padding, count from the first real token)")
        positions = pos.reshape(-1).to(dev, non_blocking=True)
        kv_start = (torch.tensor(pad_now, dtype=torch.int32).to(dev, non_blocking=True)
                    if any(pad_now) else None)
        slots = torch.arange(B, dtype=torch.int32).repeat_interleave(S).to(dev, non_blocking=True)
        rows_dev = rows.reshape(-1).to(dev, non_blocking=True) if apart else None
        with stage(timer, "qkv_proj"):
            qkv = ops.linear(x2d, self.w.wqkv)
        with stage(timer, "qk_norm_rope"):
            q = ops.qk_norm_rope(qkv, positions, self.w.q_norm, self.w.k_norm, self.inv_freq,
                                 cfg.num_attention_heads, cfg.num_key_value_heads, cfg.rms_norm_eps,
                                 cache.k, cache.v, cache_slot=slots, cache_rows=rows_dev, row_tokens=cache.tokens,
                                 row_weights=cache.weights)
        kp, vp, pslot = (prefix.k, prefix.v, prefix.slot) if P else (None, None, 0)
        # The decode kernels do not know a query that is itself a padding: it
        # would see the prefix.  The prefill gives it zeros.
        padding = P > 0 and any(p > l for p, l in zip(pad_now, L0))
        if S == 1 and not padding:
            kv_len = torch.tensor([l + 1 for l in L0], dtype=torch.int32).to(dev, non_blocking=True)
            if apart:
                with stage(timer, "attention"):
                    attn = ops.attention_prefix_decode(q, kp, vp, P, cache.k, cache.v, kv_len, max(L0) + 1,
                                                       kv_start=kv_start, prefix_slot=pslot, weights=cache.weights)
            else:
                with stage(timer, "attention"):
                    attn = ops.attention_decode(q, cache.k, cache.v, kv_len, max(L0) + 1,
                                                workspace=self._decode_ws, kv_start=kv_start)
        else:
            q_start = torch.tensor(L0, dtype=torch.int32).to(dev, non_blocking=True)
            with stage(timer, "attention"):
                if apart:
                    attn = ops.attention_prefix_prefill(q, kp, vp, P, cache.k, cache.v, q_start, B, S,
                                                        kv_start=kv_start, prefix_slot=pslot,
                                                        return_lse=cache.tracked)
                    if cache.tracked:
                        attn, lse = attn
                        self._score(q, lse, cache, q_start, B, S, kv_start, max(L0) + S)
                else:
                    attn = ops.attention_prefill(q, cache.k, cache.v, q_start, B, S, kv_start=kv_start)
        for b in range(B):
            cache.lengths[b] += S
        with stage(timer, "o_proj"):
            out = ops.linear(attn, self.w.wo)
        return out.reshape(B, S, H), cache

    @staticmethod
    def _score(q: torch.Tensor, lse: torch.Tensor, cache: KVCache, q_start: torch.Tensor, B: int, S: int,
               kv_start: Optional[torch.Tensor], max_len: int) -> None:
        """Add the attention weights of the call's last queries to the cache's."""
        n = S if cache.score_queries is None else min(S, cache.score_queries)
        if n < S:
            nh, hd = q.shape[1:]
            q = q.view(B, S, nh, hd)[:, S - n:].reshape(B * n, nh, hd)
            lse = lse.view(B, S, nh)[:, S - n:].reshape(B * n, nh)
            q_start = q_start + (S - n)
        ops.attention_weights(q, lse, cache.k, q_start, B, n, cache.weights, kv_start=kv_start, max_len=max_len)

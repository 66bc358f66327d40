"""Cases and plain forms of the shared-prefix and bounded-cache attention operators.

Five operators of a serving decoder (head dim 128, bf16 queries and caches,
grouped query heads), each with its plain form in elementary torch operations:

  prefix_decode    one query per sequence against a prefix that the whole batch
                   shares (stored once) and the sequence's own cache rows
  prefix_prefill   S new queries per sequence against the shared prefix and,
                   causally, the sequence's own rows; also each row's
                   log-sum-exp
  decode_weights   decode attention that also adds every cache row's attention
                   weight (summed over the query heads of its KV head) to a
                   running total
  prompt_weights   the same totals for S queries of a prompt, from the
                   log-sum-exp of their rows
  evict            a cache brought down to `keep` rows per KV head: the most
                   recent ones and those of the largest totals; the kept rows
                   beyond `keep` move into the freed rows below it

`listed()` and `draw(rng)` give cases, `prepare(case, seed)` a program's data,
`run(state)` one pass through an operator, `work(case)` what a pass has to
read, write and compute, `exact(case, seed)` the answer in 64 bits.
"""
import math
import random

import torch

own = False

HD = 128
SCALE = HD ** -0.5


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # two sequences, their first tokens after a short system prompt
        {"name": "prefix_decode_first_tokens", "op": "prefix_decode", "B": 2, "nh": 32, "nkv": 4, "prefix": 129,
         "own": 5, "ragged": True, "pad": False},
        # a chat service: one system prompt and tools text, ragged conversations
        {"name": "prefix_decode_chat", "op": "prefix_decode", "B": 32, "nh": 32, "nkv": 4, "prefix": 2048,
         "own": 700, "ragged": True, "pad": True},
        # many samples over one long document
        {"name": "prefix_decode_document", "op": "prefix_decode", "B": 128, "nh": 32, "nkv": 4, "prefix": 16384,
         "own": 640, "ragged": True, "pad": False},
        # short user turns appended after a system prompt of odd length
        {"name": "prefix_prefill_turns", "op": "prefix_prefill", "B": 8, "nh": 32, "nkv": 4, "prefix": 1001,
         "S": 37, "past": 0, "pad": True},
        # long user documents after a long shared prefix
        {"name": "prefix_prefill_long", "op": "prefix_prefill", "B": 4, "nh": 32, "nkv": 4, "prefix": 4096,
         "S": 2048, "past": 0, "pad": False},
        # one sequence early in its answer
        {"name": "decode_weights_one", "op": "decode_weights", "B": 1, "nh": 32, "nkv": 4, "own": 300,
         "ragged": False, "pad": False, "accumulate": True},
        # the decode batch of the decode benchmark: 8 sequences of 4,096 tokens
        {"name": "decode_weights_batch", "op": "decode_weights", "B": 8, "nh": 32, "nkv": 4, "own": 4096,
         "ragged": True, "pad": False, "accumulate": True},
        # the last 64 tokens of each prompt score its cache before an eviction
        {"name": "prompt_weights_window", "op": "prompt_weights", "B": 8, "nh": 32, "nkv": 4, "S": 64,
         "past": 1984, "pad": True, "accumulate": False},
        # a whole prompt scores its cache
        {"name": "prompt_weights_whole", "op": "prompt_weights", "B": 1, "nh": 32, "nkv": 4, "S": 4096,
         "past": 0, "pad": False, "accumulate": False},
        # a short cache brought to an odd size
        {"name": "evict_short", "op": "evict", "B": 1, "nkv": 4, "rows": 200, "keep": 129, "recent": 17,
         "ragged": False, "pad": False},
        # a serving step's eviction: 8 sequences that grew 128 rows over their budget
        {"name": "evict_step", "op": "evict", "B": 8, "nkv": 4, "rows": 2176, "keep": 2048, "recent": 256,
         "ragged": False, "pad": False},
        # long prompts cut to a budget after their prefill
        {"name": "evict_prompt", "op": "evict", "B": 4, "nkv": 4, "rows": 16384, "keep": 2048, "recent": 64,
         "ragged": True, "pad": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefix_decode", "prefix_prefill", "decode_weights", "prompt_weights", "evict"])
    nkv = rng.choice([1, 2, 4, 4, 4, 8])
    nh = nkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 8, 16])
    nh = min(nh, 32 // nkv * nkv)
    pad = rng.random() < 0.3
    if op == "prefix_decode":
        own_rows = _log(rng, 1, 2000)
        B = _log(rng, 1, max(1, min(128, 4 * 128 * 400 // (own_rows * nkv))))
        return {"op": op, "B": B, "nh": nh, "nkv": nkv, "prefix": _log(rng, 1, 16384), "own": own_rows,
                "ragged": rng.random() < 0.7, "pad": pad}
    if op == "prefix_prefill":
        S = _log(rng, 2, 2048)
        return {"op": op, "B": rng.randint(1, max(1, min(12, 8192 // S))), "nh": nh, "nkv": nkv,
                "prefix": _log(rng, 1, 4096), "S": S, "past": rng.choice([0, 0, rng.randint(1, 300)]) if S < 1700 else 0,
                "pad": pad}
    if op == "decode_weights":
        own_rows = _log(rng, 1, 16384)
        B = _log(rng, 1, max(1, min(64, 4 * 24576 // (own_rows * nkv))))
        return {"op": op, "B": B, "nh": nh, "nkv": nkv, "own": own_rows, "ragged": rng.random() < 0.7,
                "pad": pad, "accumulate": rng.random() < 0.5}
    if op == "prompt_weights":
        S = _log(rng, 1, 2048)
        past = _log(rng, 1, 4096) if rng.random() < 0.6 else 0
        return {"op": op, "B": rng.randint(1, max(1, min(8, 4096 // (S + past)))), "nh": nh, "nkv": nkv, "S": S,
                "past": past, "pad": pad, "accumulate": rng.random() < 0.3}
    rows = _log(rng, 2, 16384)
    keep = rng.randint(1, rows)
    return {"op": op, "B": _log(rng, 1, max(1, min(32, 4 * 49152 // (rows * nkv)))), "nkv": nkv, "rows": rows, "keep": keep,
            "recent": rng.randint(0, keep), "ragged": rng.random() < 0.5, "pad": pad}


# ---------------------------------------------------------------------------
# a program's data
# ---------------------------------------------------------------------------

def _seeded(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 7919 + salt) % (1 << 62))
    return g


def _lengths(case, seed, most):
    """Own rows per sequence: all `most`, or between a third of it and it (the
    longest sequence holds `most`)."""
    B = case["B"]
    if not case.get("ragged"):
        return [most] * B
    r = random.Random(seed * 31 + 5)
    out = [r.randint(max(1, most // 3), most) for _ in range(B)]
    out[r.randrange(B)] = most
    return out


def _pads(case, seed, lens):
    """Leading padding rows of a left-padded batch: up to a quarter of a row."""
    if not case["pad"]:
        return None
    r = random.Random(seed * 37 + 11)
    return [r.randint(0, n // 4) for n in lens]


def _keys(g, n, nkv, rows):
    """Normed and rotated keys: unit variance, the first rows drawn towards one
    direction that queries share (the rows most tokens attend to)."""
    k = torch.randn(n, nkv, rows, HD, generator=g, device="cuda")
    k[:, :, :min(2, rows)] += 1.5
    return k.to(torch.bfloat16)


def _queries(g, n, nh):
    return (torch.randn(n, nh, HD, generator=g, device="cuda") + 0.25).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    op = case["op"]
    B, nkv = case["B"], case["nkv"]
    g = _seeded(seed, 1)
    st = {"op": op, "B": B}
    if op == "evict":
        rows = case["rows"]
        lens = _lengths(case, seed, rows)
        pads = _pads(case, seed, lens)
        max_seq = rows + 3
        st["k"] = torch.randn(B, nkv, max_seq, HD, generator=g, device="cuda").to(torch.bfloat16)
        st["v"] = torch.randn(B, nkv, max_seq, HD, generator=g, device="cuda").to(torch.bfloat16)
        # totals are heavy-tailed, and rows that nothing attended to hold zero
        w = torch.exp(2.0 * torch.randn(B, nkv, max_seq, generator=g, device="cuda") - 4.0)
        w = torch.where(torch.rand(B, nkv, max_seq, generator=g, device="cuda") < 0.1, torch.zeros_like(w), w)
        # every KV head holds its own tokens, in an order of its own after earlier
        # evictions, below the rows appended since
        tok = torch.arange(max_seq, device="cuda").expand(B, nkv, max_seq).clone()
        mixed = max(1, min(min(lens) * 3 // 4, case["keep"]))
        order = torch.rand(B, nkv, mixed, generator=g, device="cuda").argsort(dim=-1)
        tok[:, :, :mixed] = order
        # one buffer for what a pass changes besides the rows: totals, tokens, lengths
        n = B * nkv * max_seq
        saved = torch.empty(2 * n + 2 * B, dtype=torch.int32, device="cuda")
        saved[:n] = w.reshape(-1).view(torch.int32)
        saved[n:2 * n] = tok.reshape(-1).to(torch.int32)
        saved[2 * n:2 * n + B] = _i32(lens)
        saved[2 * n + B:] = _i32(pads) if pads else 0
        live = saved.clone()
        st.update(saved=saved, live=live, weights=live[:n].view(torch.float32).view(B, nkv, max_seq),
                  tokens=live[n:2 * n].view(B, nkv, max_seq), kv_len=live[2 * n:2 * n + B],
                  kv_start=live[2 * n + B:] if pads else None, max_len=rows, keep=case["keep"],
                  recent=case["recent"])
        return st
    nh = case["nh"]
    st["nh"], st["nkv"] = nh, nkv
    if op in ("prefix_decode", "prefix_prefill"):
        P = case["prefix"]
        st["prefix_len"] = P
        st["k_prefix"] = _keys(g, 1, nkv, P + 2)
        st["v_prefix"] = torch.randn(1, nkv, P + 2, HD, generator=g, device="cuda").to(torch.bfloat16)
    if op in ("prefix_decode", "decode_weights"):
        lens = _lengths(case, seed, case["own"])
        max_seq = case["own"] + 8
        st["q"] = _queries(g, B, nh)
        st["kv_len"], st["max_len"] = _i32(lens), case["own"]
    else:
        S, past = case["S"], case["past"]
        st["S"] = S
        lens = [past + S] * B
        max_seq = past + S + 5
        st["q"] = _queries(g, B * S, nh)
        st["q_start"] = _i32([past] * B)
    pads = _pads(case, seed, lens)
    st["kv_start"] = _i32(pads) if pads else None
    st["k"] = _keys(g, B, nkv, max_seq)
    if op != "prompt_weights":
        st["v"] = torch.randn(B, nkv, max_seq, HD, generator=g, device="cuda").to(torch.bfloat16)
    if op in ("decode_weights", "prompt_weights"):
        st["accumulate"] = case["accumulate"]
        st["total"] = torch.rand(B, nkv, max_seq, generator=g, device="cuda")  # what earlier steps added up to
        st["weights"] = st["total"].clone()
    if op == "prompt_weights":
        st["lse"] = _row_lse(st["q"], st["k"], case["S"], case["past"], pads, nkv)  # what the prefill returned
    return st


def _row_lse(q, k, S, past, pads, nkv):
    """Log-sum-exp (B*S, nh) of every query row, -inf for padding rows."""
    nh = q.shape[1]
    G = nh // nkv
    out = torch.empty(q.shape[0], nh, dtype=torch.float32, device="cuda")
    pos = past + torch.arange(S, device="cuda")
    keys = torch.arange(past + S, device="cuda")
    for b in range(q.shape[0] // S):
        for h in range(nkv):
            s = torch.matmul(q[b * S:(b + 1) * S, h * G:(h + 1) * G].float(), k[b, h, :past + S].float().T) * SCALE
            hide = (keys[None] > pos[:, None]) | (keys[None] < (pads[b] if pads else 0))
            s = s.masked_fill(hide[:, None], float("-inf"))
            out[b * S:(b + 1) * S, h * G:(h + 1) * G] = torch.logsumexp(s, dim=-1)
    return out


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from nki_moe_7013_b200 import ops

    op = st["op"]
    if op == "prefix_decode":
        return ops.attention_prefix_decode(st["q"], st["k_prefix"], st["v_prefix"], st["prefix_len"], st["k"], st["v"],
                                           st["kv_len"], st["max_len"], kv_start=st["kv_start"])
    if op == "prefix_prefill":
        out, lse = ops.attention_prefix_prefill(st["q"], st["k_prefix"], st["v_prefix"], st["prefix_len"], st["k"],
                                                st["v"], st["q_start"], st["B"], st["S"], kv_start=st["kv_start"],
                                                return_lse=True)
        return {"out": out, "lse": lse}
    if op == "decode_weights":
        if st["accumulate"]:
            st["weights"].copy_(st["total"])
        out = ops.attention_decode_weights(st["q"], st["k"], st["v"], st["kv_len"], st["max_len"], st["weights"],
                                           accumulate=st["accumulate"], kv_start=st["kv_start"])
        return {"out": out, "weights": st["weights"]}
    if op == "prompt_weights":
        if st["accumulate"]:
            st["weights"].copy_(st["total"])
        ops.attention_weights(st["q"], st["lse"], st["k"], st["q_start"], st["B"], st["S"], st["weights"],
                              accumulate=st["accumulate"], kv_start=st["kv_start"])
        return st["weights"]
    st["live"].copy_(st["saved"])  # totals, tokens and lengths as before the eviction
    ops.kv_evict(st["k"], st["v"], st["weights"], st["tokens"], st["kv_len"], st["max_len"], st["keep"],
                 recent=st["recent"], kv_start=st["kv_start"])
    return {"k": st["k"], "v": st["v"], "weights": st["weights"], "tokens": st["tokens"], "kv_len": st["kv_len"]}


def _run_plain(st):
    op = st["op"]
    if op in ("prefix_decode", "decode_weights"):
        return _plain_decode(st)
    if op == "prefix_prefill":
        return _plain_prefill(st)
    if op == "prompt_weights":
        return _plain_prompt_weights(st)
    return _plain_evict(st)


def _plain_decode(st):
    B, nh, nkv, L = st["B"], st["nh"], st["nkv"], st["max_len"]
    G = nh // nkv
    q = st["q"].float().view(B, nkv, G, HD)
    rows = torch.arange(L, device="cuda")
    hide = rows[None] >= st["kv_len"][:, None]
    if st["kv_start"] is not None:
        hide = hide | (rows[None] < st["kv_start"][:, None])
    k, v = st["k"][:, :, :L].float(), st["v"][:, :, :L].float()
    s = torch.matmul(q, k.transpose(2, 3)) * SCALE
    s = torch.where(hide[:, None, None], float("-inf"), s)
    P = st.get("prefix_len", 0)
    if P:
        qp = q.transpose(0, 1).reshape(nkv, B * G, HD)
        kp, vp = st["k_prefix"][0, :, :P].float(), st["v_prefix"][0, :, :P].float()
        sp = (torch.matmul(qp, kp.transpose(1, 2)) * SCALE).view(nkv, B, G, P).transpose(0, 1)
        s = torch.cat([sp, s], dim=3)
    m = s.amax(dim=3, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    mine = p[..., P:]
    o = torch.matmul(mine, torch.where(hide[:, None, :, None], 0.0, v))
    if P:
        pp = p[..., :P].transpose(0, 1).reshape(nkv, B * G, P)
        o = o + torch.matmul(pp, vp).view(nkv, B, G, HD).transpose(0, 1)
    out = o.reshape(B, nh * HD).to(torch.bfloat16)
    if st["op"] == "prefix_decode":
        return out
    w = st["weights"]
    add = mine.sum(dim=2)
    seen = (rows[None] < st["kv_len"][:, None])[:, None]
    if st["accumulate"]:
        w.copy_(st["total"])
        w[:, :, :L] += torch.where(seen, add, 0.0)
    else:
        w[:, :, :L] = torch.where(seen, add, w[:, :, :L])
    return {"out": out, "weights": w}


def _hidden(st, b, past, S):
    """(S, past + S): own rows that query i of sequence b may not attend to."""
    pos = past + torch.arange(S, device="cuda")
    keys = torch.arange(past + S, device="cuda")
    hide = keys[None] > pos[:, None]
    if st["kv_start"] is not None:
        hide = hide | (keys[None] < st["kv_start"][b])
    return hide


def _plain_prefill(st):
    B, S, nh, nkv, P = st["B"], st["S"], st["nh"], st["nkv"], st["prefix_len"]
    G = nh // nkv
    past = st["k"].shape[2] - 5 - S
    kp, vp = st["k_prefix"][0, :, :P].float(), st["v_prefix"][0, :, :P].float()
    out = torch.empty(B * S, nh * HD, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(B * S, nh, dtype=torch.float32, device="cuda")
    for b in range(B):
        hide = _hidden(st, b, past, S)
        padded = hide.all(dim=1)  # a padding query attends to nothing, the prefix included
        q = st["q"][b * S:(b + 1) * S].float().view(S, nkv, G, HD).permute(1, 2, 0, 3).reshape(nkv, G * S, HD)
        k = torch.cat([kp, st["k"][b, :, :past + S].float()], dim=1)
        v = torch.cat([vp, st["v"][b, :, :past + S].float()], dim=1)
        s = (torch.matmul(q, k.transpose(1, 2)) * SCALE).view(nkv, G, S, P + past + S)
        s[..., P:].masked_fill_(hide, float("-inf"))
        s.masked_fill_(padded[:, None], float("-inf"))
        m = s.amax(dim=3, keepdim=True)
        m = torch.where(m == float("-inf"), 0.0, m)
        p = torch.exp(s.sub_(m))
        total = p.sum(dim=3, keepdim=True)
        o = torch.matmul(p.view(nkv, G * S, -1), v).view(nkv, G, S, HD) / torch.where(total > 0, total, 1.0)
        out[b * S:(b + 1) * S] = o.permute(2, 0, 1, 3).reshape(S, nh * HD).to(torch.bfloat16)
        lse[b * S:(b + 1) * S] = (m + torch.log(total)).view(nh, S).T
    return {"out": out, "lse": lse}


def _plain_prompt_weights(st):
    B, S, nh, nkv = st["B"], st["S"], st["nh"], st["nkv"]
    G = nh // nkv
    past = st["k"].shape[2] - 5 - S
    w = st["weights"]
    if st["accumulate"]:
        w.copy_(st["total"])
    for b in range(B):
        hide = _hidden(st, b, past, S)
        q = st["q"][b * S:(b + 1) * S].float().view(S, nkv, G, HD).permute(1, 2, 0, 3).reshape(nkv, G * S, HD)
        lse = st["lse"][b * S:(b + 1) * S].view(S, nkv, G).permute(1, 2, 0)
        s = (torch.matmul(q, st["k"][b, :, :past + S].float().transpose(1, 2)) * SCALE).view(nkv, G, S, past + S)
        s = s - torch.where(lse == float("-inf"), float("inf"), lse)[..., None]
        s.masked_fill_(hide, float("-inf"))
        add = torch.exp(s).sum(dim=(1, 2))
        if st["accumulate"]:
            w[b, :, :past + S] += add
        else:
            w[b, :, :past + S] = add
    return w


def _plain_evict(st):
    st["live"].copy_(st["saved"])
    k, v, w, tok, kv_len = st["k"], st["v"], st["weights"], st["tokens"], st["kv_len"]
    B, nkv, max_seq = w.shape
    keep, recent = st["keep"], st["recent"]
    start = st["kv_start"] if st["kv_start"] is not None else torch.zeros_like(kv_len)
    rows = torch.arange(max_seq, device="cuda").expand(B, nkv, max_seq)
    live = (rows < kv_len[:, None, None]) & (rows >= start[:, None, None])
    n = (kv_len - start).clamp(max=keep)  # rows kept
    last = torch.where(live, tok, -1).amax(dim=2, keepdim=True)
    rank = torch.where(live & (tok > last - recent), float("inf"), w)
    rank = torch.where(live, rank, float("-inf"))
    order = torch.sort(rank, dim=2, descending=True, stable=True)[1]  # equal totals: the lower row first
    place = torch.empty_like(order).scatter_(2, order, rows)
    kept = place < n[:, None, None]
    below = rows < n[:, None, None]
    holes, moved = below & ~kept, kept & ~below
    # the i-th kept row beyond n goes to the i-th free row below it
    src, dst = moved.nonzero(), holes.nonzero()
    a, c = (src[:, 0], src[:, 1], src[:, 2]), (dst[:, 0], dst[:, 1], dst[:, 2])
    k[c], v[c], w[c], tok[c] = k[a], v[a], w[a], tok[a]
    old = rows < kv_len[:, None, None]
    w.masked_fill_(old & ~below, 0.0)
    tok.masked_fill_(old & ~below, -1)
    kv_len.copy_(n)
    return {"k": k, "v": v, "weights": w, "tokens": tok, "kv_len": kv_len}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op, B, nkv = case["op"], case["B"], case["nkv"]
    row = nkv * HD * 2
    if op == "evict":
        # lengths and paddings of a ragged batch: their average over the seeds
        rows = case["rows"] * (2 / 3 if case["ragged"] else 1) * (7 / 8 if case["pad"] else 1)
        n = min(case["keep"], rows)
        # every total and token is read, the moved rows are read and written (a
        # chosen row lies beyond n with the share of rows that do), and the
        # totals and tokens behind n are written
        moved = max(0.0, (rows - n)) * n / max(rows, 1)
        return {"bytes": int(B * (nkv * 8 * (rows + max(0, rows - n)) + moved * 4 * row)), "flops": 0}
    nh = case["nh"]
    if op == "prompt_weights":
        S, past = case["S"], case["past"]
        L = past + S
        pairs = B * nh * (S * past + S * (S + 1) / 2)
        return {"bytes": int(B * S * nh * (HD * 2 + 4) + B * L * row + B * L * nkv * (8 if case["accumulate"] else 4)),
                "flops": int(2 * HD * pairs)}
    if op == "prefix_prefill":
        S, past, P = case["S"], case["past"], case["prefix"]
        pairs = B * nh * (S * (P + past) + S * (S + 1) / 2)
        return {"bytes": int(2 * B * S * nh * HD * 2 + B * S * nh * 4 + 2 * row * (P + B * (past + S))),
                "flops": int(4 * HD * pairs)}
    rows = case["own"] * (2 / 3 if case["ragged"] and B > 1 else 1) * (7 / 8 if case["pad"] else 1)
    b = 2 * B * nh * HD * 2 + 2 * row * B * rows
    pairs = B * nh * rows
    if op == "prefix_decode":
        b += 2 * row * case["prefix"]
        pairs += B * nh * case["prefix"]
    else:
        b += B * rows * nkv * (8 if case["accumulate"] else 4)
    return {"bytes": int(b), "flops": int(4 * HD * pairs)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "evict":
        return _exact_evict(st)
    B, nh, nkv = case["B"], case["nh"], case["nkv"]
    G = nh // nkv
    starts = st["kv_start"].tolist() if st["kv_start"] is not None else [0] * B
    if op in ("prefix_decode", "decode_weights"):
        out = torch.zeros(B, nh, HD, dtype=torch.float64, device="cuda")
        w = st["total"].double() if op == "decode_weights" else None
        P = st.get("prefix_len", 0)
        lens = st["kv_len"].tolist()
        kp = st["k_prefix"][0, :, :P].double() if P else st["k"][0, :, :0].double()
        vp = st["v_prefix"][0, :, :P].double() if P else st["v"][0, :, :0].double()
        for b in range(B):
            n, a = lens[b], starts[b]
            if w is not None and not case["accumulate"]:
                w[b, :, :n] = 0
            for h in range(nkv):
                k = torch.cat([kp[h], st["k"][b, h, a:n].double()])
                v = torch.cat([vp[h], st["v"][b, h, a:n].double()])
                if k.shape[0] == 0:
                    continue
                p = torch.softmax(st["q"][b, h * G:(h + 1) * G].double() @ k.T / math.sqrt(HD), dim=1)
                out[b, h * G:(h + 1) * G] = p @ v
                if w is not None:
                    w[b, h, a:n] += p[:, P:].sum(dim=0)
        out = out.reshape(B, nh * HD)
        return out if op == "prefix_decode" else {"out": out, "weights": w}
    S, past = case["S"], case["past"]
    if op == "prefix_prefill":
        P = case["prefix"]
        out = torch.zeros(B, S, nh, HD, dtype=torch.float64, device="cuda")
        lse = torch.full((B, S, nh), float("-inf"), dtype=torch.float64, device="cuda")
        for b in range(B):
            first = max(0, starts[b] - past)  # the first query that is no padding
            if first >= S:
                continue
            bias = torch.zeros(S - first, P + past + S - starts[b], dtype=torch.float64, device="cuda")
            at = torch.arange(starts[b], past + S, device="cuda")
            bias[:, P:][at[None] > (past + torch.arange(first, S, device="cuda"))[:, None]] = float("-inf")
            for h in range(nh):
                k = torch.cat([st["k_prefix"][0, h // G, :P], st["k"][b, h // G, starts[b]:past + S]]).double()
                v = torch.cat([st["v_prefix"][0, h // G, :P], st["v"][b, h // G, starts[b]:past + S]]).double()
                s = st["q"][b * S + first:(b + 1) * S, h].double() @ k.T / math.sqrt(HD) + bias
                lse[b, first:, h] = torch.logsumexp(s, dim=1)
                out[b, first:, h] = torch.softmax(s, dim=1) @ v
        return {"out": out.reshape(B * S, nh * HD), "lse": lse.reshape(B * S, nh)}
    w = st["total"].double()
    for b in range(B):
        L = past + S
        if not case["accumulate"]:
            w[b, :, :L] = 0
        first = max(0, starts[b] - past)
        at = torch.arange(starts[b], L, device="cuda")
        seen = at[None] <= (past + torch.arange(first, S, device="cuda"))[:, None]
        for h in range(nh):
            s = st["q"][b * S + first:(b + 1) * S, h].double() @ st["k"][b, h // G, starts[b]:L].double().T
            s = s / math.sqrt(HD) - st["lse"][b * S + first:(b + 1) * S, h].double()[:, None]
            w[b, h // G, starts[b]:L] += torch.where(seen, torch.exp(s), 0.0).sum(dim=0)
    return w


def _exact_evict(st):
    """Row by row on the host, from the definition."""
    k, v = st["k"].clone(), st["v"].clone()
    w, tok = st["weights"].cpu().numpy().copy(), st["tokens"].cpu().numpy().copy()
    lens = st["kv_len"].tolist()
    starts = st["kv_start"].tolist() if st["kv_start"] is not None else [0] * len(lens)
    new = []
    for b in range(w.shape[0]):
        n = min(st["keep"], lens[b] - starts[b])
        new.append(n)
        for h in range(w.shape[1]):
            live = list(range(starts[b], lens[b]))
            newest = max(int(tok[b, h, r]) for r in live) if live else 0
            recent = [r for r in live if tok[b, h, r] > newest - st["recent"]]
            others = [r for r in live if tok[b, h, r] <= newest - st["recent"]]
            others.sort(key=lambda r: (-float(w[b, h, r]), r))
            chosen = set((recent + others)[:n])
            src = [r for r in sorted(chosen) if r >= n]
            dst = [r for r in range(n) if r not in chosen]
            if src:
                k[b, h, dst], v[b, h, dst] = k[b, h, src], v[b, h, src]
                w[b, h, dst], tok[b, h, dst] = w[b, h, src], tok[b, h, src]
            w[b, h, n:lens[b]] = 0
            tok[b, h, n:lens[b]] = -1
    return {"k": k.double(), "v": v.double(), "weights": torch.from_numpy(w).double(),
            "tokens": torch.from_numpy(tok).long(), "kv_len": torch.tensor(new)}

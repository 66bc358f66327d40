"""Attention over a prefix shared by the batch, attention that keeps every
cache row's weight, and eviction by it, against plain implementations in 64
bits.

Tolerances.  The kernels multiply bf16 inputs exactly and add in fp32; the
probabilities enter the second product in bf16 (half a step: 2^-8 relative),
and the output is rounded to bf16 once (2^-8 of itself).  A score is a sum of
128 products: its error is at most 128 * 2^-24 * D, with D the largest
c * sum |q_d k_d| of the call, and (scaling, running maximum, exponential) a
few 2^-24 of it more; 136 * 2^-24 * D covers both.  A probability carries the
error of its own score and of the joined sum, 2 * delta in all, and 2^-18 for
the exponentials and the sums in fp32."""
import pytest
import torch

from helpers import assert_within_one_ulp

pytestmark = pytest.mark.gpu

HD = 128
C = HD ** -0.5


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


class Ref:
    """One query row set over one key set, in 64 bits."""

    def __init__(self, q, k, v, hide=None):
        s = q.double() @ k.double().T * C
        self.D = float((q.double().abs() @ k.double().abs().T * C).max()) if k.shape[0] else 0.0
        if hide is not None:
            s = s.masked_fill(hide, float("-inf"))
        self.lse = torch.logsumexp(s, dim=-1) if k.shape[0] else torch.full(s.shape[:1], float("-inf"), dtype=s.dtype,
                                                                            device=s.device)
        live = self.lse > float("-inf")
        self.p = torch.where(live[:, None], torch.exp(s - torch.where(live, self.lse, 0.0)[:, None]), 0.0)
        if v is not None:
            self.out = self.p @ v.double()
            self.mag = self.p @ v.double().abs()


def _delta(D):
    return 136 * 2.0 ** -24 * D


def _check_out(got, out, mag, D):
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2 * _delta(D) + 2.0 ** -18) * mag * (1 + 2.0 ** -7) + 1e-30
    err = (got.double() - out).abs()
    assert torch.isfinite(got.float()).all()
    worst = float((err / tol).max())
    assert worst <= 1.0, f"output off by {worst:.2f} tolerances"


def _check_weights(got, ref, before, D):
    # one more rounding where the total is added to what was there
    tol = ref * (2 * _delta(D) + 2.0 ** -18) + 2.0 ** -24 * (before.abs() + ref) + 1e-30
    worst = float(((got.double() - before - ref).abs() / tol).max())
    assert worst <= 1.0, f"weights off by {worst:.2f} tolerances"


def _error():
    from nki_moe_7013_b200 import _C

    torch.cuda.synchronize()
    return _C.device_error()


# (B, nh, nkv, prefix, own lengths, paddings, slots, prefix slot)
DECODE = [
    (1, 8, 1, 1, [1], None, None, 0),
    (2, 32, 4, 129, [5, 1], None, None, 1),
    (3, 32, 4, 64, [0, 64, 130], None, [2, 0, 4], 0),          # a sequence with nothing but the prefix
    (3, 32, 4, 0, [0, 77, 300], [0, 77, 13], None, 0),         # no prefix: one row sees nothing, one only padding
    (5, 12, 4, 65, [33, 1, 2, 200, 63], [3, 0, 1, 199, 0], None, 0),
    (9, 64, 4, 1000, [150] * 9, None, None, 0),                # 144 rows, 16 heads per KV head
    (40, 32, 4, 300, list(range(40)), None, None, 2),          # 320 rows
    (33, 10, 2, 131, list(range(33)), None, None, 0),          # 5 heads per KV head
    (70, 2, 2, 127, [3] * 70, None, None, 0),
    (2, 32, 4, 5000, [4096, 700], None, None, 0),              # many parts
    (130, 8, 8, 700, [1] * 130, None, None, 0),                # one head per KV head
    (4, 32, 4, 0, [700, 0, 1300, 129], [0, 0, 700, 128], [3, 1, 0, 2], 0),
    (2, 48, 3, 450, [63, 5], [0, 5], None, 0),
    (40, 16, 4, 0, [20 * i for i in range(40)], None, None, 0),
    (1, 16, 16, 0, [9000], [1], None, 0),
    # enough rows on a long enough prefix for the tcgen05 kernel
    (40, 32, 4, 3001, list(range(40)), None, None, 2),         # 320 rows: two tile pairs
    (33, 10, 2, 12000, [40 * i for i in range(33)], [30 * i for i in range(33)], None, 0),  # tiles of 125 rows
    (9, 64, 4, 6016, [150] * 9, None, [8, 7, 6, 5, 4, 3, 2, 1, 0], 0),
    (12, 8, 1, 33000, [0] * 11 + [1], None, None, 0),          # 96 rows of one KV head: the keys split
    (130, 8, 8, 4000, [1] * 130, None, None, 0),
    (20, 32, 4, 3000, [0] * 20, None, None, 0),                # nothing but the prefix
    (300, 64, 4, 1200, [b % 41 for b in range(300)], None, None, 0),  # row tiles that share a CTA
    (200, 64, 4, 1100, [40 - b % 7 for b in range(200)], None, None, 0),
    # several row tiles that stay on the warp-level kernel
    (8, 32, 4, 700, [400, 3, 77, 0, 128, 129, 399, 1], None, None, 0),
    (7, 20, 4, 900, [333, 0, 64, 65, 300, 2, 1], [30, 0, 64, 1, 0, 2, 0], None, 0),
]


def _decode_inputs(B, nh, nkv, P, lens, pads, slots, pslot, seed):
    g = _gen(seed)
    n_slots = B if slots is None else max(slots) + 1
    max_seq = max(lens) + 9
    k, v = _randn(g, n_slots, nkv, max_seq, HD), _randn(g, n_slots, nkv, max_seq, HD)
    q = _randn(g, B, nh, HD)
    kp, vp = _randn(g, pslot + 1, nkv, P + 3, HD), _randn(g, pslot + 1, nkv, P + 3, HD)
    # what nobody sees holds no numbers
    kp[:, :, P:], vp[:, :, P:] = float("nan"), float("inf")
    kp[:pslot], vp[:pslot] = float("nan"), float("nan")
    seen = torch.zeros(n_slots, max_seq, dtype=torch.bool, device="cuda")
    for b in range(B):
        seen[b if slots is None else slots[b], (pads[b] if pads else 0):lens[b]] = True
    k.masked_fill_(~seen[:, None, :, None], float("nan"))
    v.masked_fill_(~seen[:, None, :, None], float("-inf"))
    return q, kp, vp, k, v


@pytest.mark.parametrize("weights", ["none", "add", "set"])
@pytest.mark.parametrize("case", DECODE)
def test_prefix_decode(cuda_dev, case, weights):
    from nki_moe_7013_b200 import ops

    B, nh, nkv, P, lens, pads, slots, pslot = case
    G = nh // nkv
    q, kp, vp, k, v = _decode_inputs(*case, seed=B * 100 + P)
    n_slots, max_seq = k.shape[0], k.shape[2]
    w = torch.rand(n_slots, nkv, max_seq, generator=_gen(3), device="cuda") if weights != "none" else None
    before = w.double().clone() if w is not None else None
    out = ops.attention_prefix_decode(q, kp, vp, P, k, v, _i32(lens), max(lens), cache_slot=_i32(slots),
                                      kv_start=_i32(pads), prefix_slot=pslot, weights=w,
                                      accumulate=weights == "add")
    assert _error() == 0
    ref = torch.zeros(B, nh, HD, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(ref)
    add = torch.zeros(n_slots, nkv, max_seq, dtype=torch.float64, device="cuda")
    D = 0.0
    for b in range(B):
        sl, lo = (b if slots is None else slots[b]), (pads[b] if pads else 0)
        if w is not None and weights == "set":
            before[sl, :, :lens[b]] = 0
        for g in range(nkv):
            r = Ref(q[b, g * G:(g + 1) * G], torch.cat([kp[pslot, g, :P], k[sl, g, lo:lens[b]]]),
                    torch.cat([vp[pslot, g, :P], v[sl, g, lo:lens[b]]]))
            ref[b, g * G:(g + 1) * G], mag[b, g * G:(g + 1) * G] = r.out, r.mag
            add[sl, g, lo:lens[b]] = r.p[:, P:].sum(dim=0)
            D = max(D, r.D)
    _check_out(out.view(B, nh, HD), ref, mag, D)
    if w is not None:
        _check_weights(w, add, before, D)


def test_prefix_decode_is_attention_decode_without_a_prefix(cuda_dev):
    """The same rows as one cache, and the weights of all heads of a row sum to
    the number of heads."""
    from nki_moe_7013_b200 import ops

    g = _gen(5)
    B, nh, nkv, L = 3, 32, 4, 260
    k, v, q = _randn(g, B, nkv, L, HD), _randn(g, B, nkv, L, HD), _randn(g, B, nh, HD)
    lens = _i32([260, 100, 17])
    w = torch.zeros(B, nkv, L, device="cuda")
    plain = ops.attention_decode(q, k, v, lens, L)
    mine = ops.attention_decode_weights(q, k, v, lens, L, w)
    assert _error() == 0
    # both round the probabilities and the output to bf16: two of each
    mag = v.float().abs().amax(dim=2).repeat_interleave(nh // nkv, dim=1).reshape(B, -1)
    assert bool(((plain.float() - mine.float()).abs() <= 2 * (2.0 ** -8 + 2.0 ** -8) * mag).all())
    assert torch.allclose(w.sum(dim=2), torch.full((B, nkv), 8.0, device="cuda"), rtol=0, atol=8 * 2.0 ** -12)


def test_prefix_in_the_same_cache_and_run_to_run(cuda_dev):
    """A prefix that is a slot of the sequences' own cache; two calls, one of
    them on another stream with a caller's workspace, give the same bits."""
    from nki_moe_7013_b200 import ops

    g = _gen(6)
    B, nh, nkv, P, L = 20, 32, 4, 333, 100
    k, v, q = _randn(g, B + 1, nkv, 400, HD), _randn(g, B + 1, nkv, 400, HD), _randn(g, B, nh, HD)
    slots, lens = _i32(list(range(1, B + 1))), _i32([L] * B)
    w = [torch.zeros(B + 1, nkv, 400, device="cuda") for _ in range(2)]
    a = ops.attention_prefix_decode(q, k, v, P, k, v, lens, L, cache_slot=slots, weights=w[0])
    ws = torch.full((ops.attention_prefix_decode_workspace_size(B, nh, nkv, P, L, True),), 255, dtype=torch.uint8,
                    device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = ops.attention_prefix_decode(q, k, v, P, k, v, lens, L, cache_slot=slots, weights=w[1], workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    assert _error() == 0
    assert torch.equal(a, b) and torch.equal(w[0], w[1])
    r = Ref(q[0, :8], torch.cat([k[0, 0, :P], k[1, 0, :L]]), torch.cat([v[0, 0, :P], v[1, 0, :L]]))
    _check_out(a.view(B, nh, HD)[0, :8], r.out, r.mag, r.D)


def test_decode_bad_lengths_and_slots(cuda_dev):
    """A length past max_len, a slot outside the cache, a slot given twice:
    device error 4; the other sequences are right."""
    from nki_moe_7013_b200 import ops

    g = _gen(7)
    B, nh, nkv, L = 3, 32, 4, 90
    k, v, q = _randn(g, B, nkv, L, HD), _randn(g, B, nkv, L, HD), _randn(g, B, nh, HD)
    good = ops.attention_prefix_decode(q, None, None, 0, k, v, _i32([50, 60, 70]), 80)
    for lens, slots, bad in (([50, 81, 70], None, 1), ([50, -1, 70], None, 1), ([50, 60, 70], [0, 3, 2], 1),
                             ([50, 60, 70], [0, -1, 2], 1)):
        out = ops.attention_prefix_decode(q, None, None, 0, k, v, _i32(lens), 80, cache_slot=_i32(slots))
        assert _error() == 4
        assert not out[bad].any()
        for b in range(B):
            if b != bad:
                assert torch.equal(out[b], good[b])
    w = torch.zeros(B, nkv, L, device="cuda")
    ops.attention_decode_weights(q, k, v, _i32([50, 60, 70]), 80, w, cache_slot=_i32([0, 1, 1]))
    assert _error() == 4
    once = torch.zeros(B, nkv, L, device="cuda")
    ops.attention_decode_weights(q[:2].contiguous(), k, v, _i32([50, 60]), 80, once)
    assert _error() == 0
    assert torch.allclose(w, once, rtol=2.0 ** -12, atol=1e-30)


def test_decode_empty_batch_and_nothing_to_see(cuda_dev):
    from nki_moe_7013_b200 import ops

    g = _gen(8)
    k, q = _randn(g, 2, 4, 8, HD), _randn(g, 2, 32, HD)
    out = ops.attention_prefix_decode(q[:0], None, None, 0, k, k, _i32([]), 8)
    assert out.shape == (0, 32 * HD)
    out = ops.attention_prefix_decode(q, None, None, 0, k, k, _i32([0, 0]), 0)
    assert _error() == 0 and not out.any()


# (B, nh, nkv, prefix, S, past, paddings, slots)
PREFILL = [
    (1, 32, 4, 1, 1, 0, None, None),
    (2, 32, 4, 129, 37, 0, [0, 5], None),
    (1, 8, 1, 128, 300, 0, None, None),
    (3, 12, 4, 0, 129, 0, [0, 128, 129], None),        # a sequence of padding only
    (3, 12, 4, 77, 129, 0, [0, 128, 129], None),
    (2, 6, 2, 1000, 64, 333, [200, 340], [2, 0]),
    (1, 32, 4, 255, 600, 11, None, None),
    (2, 16, 1, 63, 5, 250, None, [1, 0]),
    (2, 32, 4, 300, 700, 20, [5, 400], None),          # queries cut into chunks, padding before the first
    (1, 10, 2, 0, 450, 0, [33], None),
]


@pytest.mark.parametrize("case", PREFILL)
def test_prefix_prefill_and_weights(cuda_dev, case):
    """Output and log-sum-exp of the prefill, and the weights that its queries
    (all, and the last few) put on the sequence's own rows."""
    from nki_moe_7013_b200 import ops

    B, nh, nkv, P, S, past, pads, slots = case
    G = nh // nkv
    g = _gen(B * 10 + S)
    n_slots = B if slots is None else max(slots) + 1
    L, max_seq = past + S, past + S + 7
    k, v = _randn(g, n_slots, nkv, max_seq, HD), _randn(g, n_slots, nkv, max_seq, HD)
    kp, vp = _randn(g, 2, nkv, P + 2, HD), _randn(g, 2, nkv, P + 2, HD)
    q = _randn(g, B * S, nh, HD)
    kp[:, :, P:], vp[:, :, P:] = float("inf"), float("nan")
    kp[0], vp[0] = float("nan"), float("nan")
    k[:, :, L:], v[:, :, L:] = float("nan"), float("nan")
    for b in range(B):
        sl, lo = (b if slots is None else slots[b]), (pads[b] if pads else 0)
        k[sl, :, :lo], v[sl, :, :lo] = float("nan"), float("nan")
    out, lse = ops.attention_prefix_prefill(q, kp, vp, P, k, v, _i32([past] * B), B, S, cache_slot=_i32(slots),
                                            kv_start=_i32(pads), prefix_slot=1, return_lse=True)
    only = ops.attention_prefix_prefill(q, kp, vp, P, k, v, _i32([past] * B), B, S, cache_slot=_i32(slots),
                                        kv_start=_i32(pads), prefix_slot=1)
    assert _error() == 0 and torch.equal(out, only)
    last = max(1, S // 3)
    w = {"set": torch.rand(n_slots, nkv, max_seq, device="cuda"), "add": torch.rand(n_slots, nkv, max_seq, device="cuda"),
         "last": torch.rand(n_slots, nkv, max_seq, device="cuda")}
    before = {n: t.double().clone() for n, t in w.items()}
    ops.attention_weights(q, lse, k, _i32([past] * B), B, S, w["set"], accumulate=False, cache_slot=_i32(slots),
                          kv_start=_i32(pads))
    ops.attention_weights(q, lse, k, _i32([past] * B), B, S, w["add"], cache_slot=_i32(slots), kv_start=_i32(pads),
                          max_len=L)
    q_last = q.view(B, S, nh, HD)[:, S - last:].reshape(B * last, nh, HD).contiguous()
    lse_last = lse.view(B, S, nh)[:, S - last:].reshape(B * last, nh).contiguous()
    ops.attention_weights(q_last, lse_last, k, _i32([L - last] * B), B, last, w["last"], cache_slot=_i32(slots),
                          kv_start=_i32(pads))
    assert _error() == 0
    ref = torch.zeros(B * S, nh, HD, dtype=torch.float64, device="cuda")
    mag, ref_lse = torch.zeros_like(ref), torch.zeros(B * S, nh, dtype=torch.float64, device="cuda")
    add = {n: torch.zeros(n_slots, nkv, max_seq, dtype=torch.float64, device="cuda") for n in w}
    D = 0.0
    for b in range(B):
        sl, lo = (b if slots is None else slots[b]), min(pads[b] if pads else 0, L)
        before["set"][sl, :, :L] = 0
        at = torch.arange(lo, L, device="cuda")
        pos = past + torch.arange(S, device="cuda")
        hide = torch.zeros(S, P + L - lo, dtype=torch.bool, device="cuda")
        hide[:, P:] = at[None] > pos[:, None]
        hide |= (pos < lo)[:, None]
        for h in range(nh):
            r = Ref(q[b * S:(b + 1) * S, h], torch.cat([kp[1, h // G, :P], k[sl, h // G, lo:L]]),
                    torch.cat([vp[1, h // G, :P], v[sl, h // G, lo:L]]), hide)
            ref[b * S:(b + 1) * S, h], mag[b * S:(b + 1) * S, h] = r.out, r.mag
            ref_lse[b * S:(b + 1) * S, h] = r.lse
            D = max(D, r.D)
            for n in ("set", "add"):
                add[n][sl, h // G, lo:L] += r.p[:, P:].sum(dim=0)
            add["last"][sl, h // G, lo:L] += r.p[S - last:, P:].sum(dim=0)
    _check_out(out.view(B * S, nh, HD), ref, mag, D)
    dead = ref_lse == float("-inf")
    assert torch.equal(lse == float("-inf"), dead) and not out.view(B * S, nh, HD)[dead].any()
    # the score's error, the sum's and the logarithm's, and the roundings of numbers of the size of lse
    tol = _delta(D) + 2.0 ** -18 + 4 * 2.0 ** -24 * ref_lse.abs()
    assert bool(((lse.double() - ref_lse).abs() <= tol)[~dead].all())
    for n in w:
        # the given lse is off by up to its tolerance as well
        _check_weights(w[n], add[n], before[n], 1.5 * D + 2.0 ** -19 / (136 * 2.0 ** -24))


def test_prefix_prefill_is_attention_prefill_without_a_prefix(cuda_dev):
    from nki_moe_7013_b200 import ops

    g = _gen(9)
    B, S, nh, nkv = 2, 300, 32, 4
    k, v, q = _randn(g, B, nkv, S, HD), _randn(g, B, nkv, S, HD), _randn(g, B * S, nh, HD)
    start = _i32([0, 0])
    # Both multiply the same bf16 probabilities with the same values, key tile
    # by key tile.  What may differ is the order in which the up to 300
    # probabilities of a row are added, 300 * 2^-24 < 2^-15 of their sum, and
    # the one rounding of out = o / sum to bf16 can then fall to the neighbour:
    # one ulp, at most 2^-7 of the value.
    assert_within_one_ulp(ops.attention_prefill(q, k, v, start, B, S),
                          ops.attention_prefix_prefill(q, None, None, 0, k, v, start, B, S))
    assert _error() == 0


def test_prefill_and_weights_bad_starts_and_slots(cuda_dev):
    from nki_moe_7013_b200 import ops

    g = _gen(10)
    B, S, nh, nkv = 2, 9, 8, 1
    k, q = _randn(g, B, nkv, 40, HD), _randn(g, B * S, nh, HD)
    for start, slots in (([0, 32], None), ([-1, 0], None), ([0, 0], [0, 2])):
        ops.attention_prefix_prefill(q, k, k, 5, k, k, _i32(start), B, S, cache_slot=_i32(slots))
        assert _error() == 4
    lse = torch.zeros(B * S, nh, device="cuda")
    w = torch.zeros(B, nkv, 40, device="cuda")
    for start, slots in (([0, 32], None), ([-1, 0], None), ([0, 0], [2, 0]), ([0, 0], [1, 1])):
        ops.attention_weights(q, lse, k, _i32(start), B, S, w, cache_slot=_i32(slots))
        assert _error() == 4


def _evict_ref(k, v, w, tok, lens, starts, slots, keep, recent):
    """Row by row, on copies on the host."""
    k, v, w, tok = (t.cpu().clone() for t in (k, v, w, tok))
    new = list(lens)
    for b, sl in enumerate(slots):
        lo, n_old = min(starts[b], lens[b]), lens[b]
        n = new[b] = min(keep, n_old - lo)
        for g in range(w.shape[1]):
            live = list(range(lo, n_old))
            newest = max((int(tok[sl, g, r]) for r in live), default=0)

            def rank(r):
                x = float(w[sl, g, r])
                if int(tok[sl, g, r]) > newest - recent:
                    return (0, 0.0, r)
                return (1, 0.0, r) if x != x else (2, -x, r)

            kept = set(sorted(live, key=rank)[:n])
            src, dst = [r for r in sorted(kept) if r >= n], [r for r in range(n) if r not in kept]
            for t in (k, v, w, tok):
                t[sl, g, dst] = t[sl, g, src].clone()
            w[sl, g, n:n_old] = 0
            tok[sl, g, n:n_old] = -1
    return k, v, w, tok, new


# (slots of the call, nkv, lengths, paddings, keep, recent)
EVICT = [
    ([0], 1, [1], None, 1, 0),
    ([0], 4, [200], None, 129, 17),
    ([0, 1], 2, [40, 7], [3, 0], 10, 10),            # only the newest stay; a cache shorter than the budget
    ([2, 0, 1], 4, [300, 0, 64], [0, 0, 64], 33, 1),  # an empty cache, one of padding only
    ([1, 0], 2, [1500, 2000], [0, 700], 1024, 256),
    ([0], 2, [1031], None, 1030, 0),
    ([0], 2, [500], None, 0, 0),                     # nothing stays
    ([0], 1, [50021], None, 20000, 1000),
    ([1, 0], 2, [8200, 5000], [17, 0], 4100, 100),
    ([0], 1, [270001], [3], 100000, 5000),           # more rows than the select kernel holds in shared memory
    ([0, 1], 1, [100, 90], [10, 0], 1000, 5),        # a budget over every length: paddings leave
]


@pytest.mark.parametrize("case", EVICT)
def test_evict(cuda_dev, case):
    from nki_moe_7013_b200 import ops

    slots, nkv, lens, pads, keep, recent = case
    g = _gen(sum(lens) + keep)
    n_slots, max_seq = max(slots) + 1, max(lens) + 5
    k, v = _randn(g, n_slots, nkv, max_seq, HD), _randn(g, n_slots, nkv, max_seq, HD)
    # equal weights (and zeros of both signs), negatives, infinities, NaN
    w = torch.randn(n_slots, nkv, max_seq, generator=g, device="cuda").mul(4).round().div(4)
    odd = torch.rand(n_slots, nkv, max_seq, generator=g, device="cuda")
    w = torch.where(odd < 0.02, float("nan"), torch.where(odd < 0.05, float("inf"), torch.where(odd < 0.08, -0.0, w)))
    tok = torch.rand(n_slots, nkv, max_seq, generator=g, device="cuda").argsort(dim=2).to(torch.int32) + 12
    ref = _evict_ref(k, v, w, tok, lens, pads or [0] * len(lens), slots, keep, recent)
    kv_len, start = _i32(lens), _i32(pads)
    ops.kv_evict(k, v, w, tok, kv_len, max(lens), keep, recent=recent, cache_slot=_i32(slots), kv_start=start)
    assert _error() == 0
    assert kv_len.tolist() == ref[4]
    if start is not None:
        assert start.tolist() == [0] * len(lens)
    for name, got, want in zip(("k", "v", "tokens"), (k, v, tok), (ref[0], ref[1], ref[3])):
        assert torch.equal(got.cpu(), want), name
    assert torch.equal(w.cpu().view(torch.int32), ref[2].view(torch.int32))


def test_evict_bad_entries_stay_as_they_are(cuda_dev):
    """A length past max_len, a slot outside the cache, a slot given twice:
    device error 4, the entry untouched, the others evicted."""
    from nki_moe_7013_b200 import ops

    g = _gen(11)
    for lens, slots, bad in (([30, 41, 30], [0, 1, 2], 1), ([30, 30, 30], [0, 3, 2], 1), ([30, 30, 30], [0, 2, 2], 2)):
        k = _randn(g, 3, 2, 40, HD)
        w = torch.rand(3, 2, 40, generator=g, device="cuda")
        tok = torch.arange(40, dtype=torch.int32, device="cuda").expand(3, 2, 40).contiguous()
        k0, w0 = k.clone(), w.clone()
        kv_len = _i32(lens)
        ops.kv_evict(k, k.clone(), w, tok, kv_len, 40, 10, cache_slot=_i32(slots))
        assert _error() == 4
        assert kv_len.tolist() == [lens[b] if b == bad else 10 for b in range(3)]
        if slots[bad] == 1:
            assert torch.equal(k[1], k0[1]) and torch.equal(w[1], w0[1])


def test_append_rows(cuda_dev):
    """Keys and values go to rows apart from their positions, with the
    positions' rotations; tokens and totals of the rows are set."""
    from nki_moe_7013_b200 import _C, ops
    from nki_moe_7013_b200.attention import rope_inv_freq

    g = _gen(12)
    T, nh, nkv, max_seq = 6, 32, 4, 20
    qkv = _randn(g, T, (nh + 2 * nkv) * HD)
    pos = _i32([100, 7, 3, 0, 19, 5])
    rows, slots = _i32([4, 0, 19, 2, 5, 20]), _i32([0, 0, 0, 1, 1, 1])
    ones = torch.ones(HD, device="cuda")
    freq = rope_inv_freq(HD, 1e6, cuda_dev)
    big = [torch.zeros(2, nkv, 128, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    q0 = ops.qk_norm_rope(qkv, pos, ones, ones, freq, nh, nkv, 1e-6, *big, cache_slot=slots)
    assert _C.device_error() == 0
    kc = [torch.zeros(2, nkv, max_seq, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    tok = torch.full((2, nkv, max_seq), -1, dtype=torch.int32, device="cuda")
    w = torch.full((2, nkv, max_seq), 3.0, device="cuda")
    q = ops.qk_norm_rope(qkv, pos, ones, ones, freq, nh, nkv, 1e-6, *kc, cache_slot=slots, cache_rows=rows,
                         row_tokens=tok, row_weights=w)
    assert _error() == 4  # the last token's row lies outside the cache
    assert torch.equal(q, q0)
    for t in range(T - 1):
        s, r, p = int(slots[t]), int(rows[t]), int(pos[t])
        for a, c in zip(kc, big):
            assert torch.equal(a[s, :, r], c[s, :, p])
        assert bool((tok[s, :, r] == p).all()) and not w[s, :, r].any()
    assert int((tok >= 0).sum()) == 5 * nkv and int((w == 3.0).sum()) == 2 * nkv * max_seq - 5 * nkv


def test_evict_empty_cache(cuda_dev):
    from nki_moe_7013_b200 import ops

    k = _randn(_gen(13), 2, 2, 8, HD)
    w, tok = torch.ones(2, 2, 8, device="cuda"), torch.ones(2, 2, 8, dtype=torch.int32, device="cuda")
    n = _i32([0, 0])
    ops.kv_evict(k, k.clone(), w, tok, n, 0, 4, recent=2)
    ops.kv_evict(k[:0], k[:0], w[:0], tok[:0], _i32([]), 0, 4)
    assert _error() == 0 and n.tolist() == [0, 0] and bool((w == 1).all()) and bool((tok == 1).all())


@pytest.mark.parametrize("P,own", [(3001, 90), (700, 600), (100, 60)])
def test_captured_calls_follow_their_inputs(cuda_dev, P, own):
    """Decode with weights (the tcgen05 prefix, cut sequences, and the single
    kernel), prefill, prompt weights and an eviction in one graph, replayed
    with other inputs, against eager calls; two graphs, each with workspaces of
    its own, in flight on two streams."""
    from nki_moe_7013_b200 import ops

    B, nh, nkv, S, rows = 40, 32, 4, 19, 640
    g = _gen(P)
    kp, vp = _randn(g, 1, nkv, P, HD), _randn(g, 1, nkv, P, HD)

    def state():
        return dict(k=_randn(g, B, nkv, rows, HD), v=_randn(g, B, nkv, rows, HD), q=_randn(g, B, nh, HD),
                    qs=_randn(g, B * S, nh, HD), n=torch.zeros(B, dtype=torch.int32, device="cuda"),
                    start=torch.zeros(B, dtype=torch.int32, device="cuda"),
                    w=torch.zeros(B, nkv, rows, device="cuda"),
                    tok=torch.arange(rows, dtype=torch.int32, device="cuda").expand(B, nkv, rows).contiguous())

    def step(s):
        out = ops.attention_prefix_decode(s["q"], kp, vp, P, s["k"], s["v"], s["n"], own, weights=s["w"])
        pre, lse = ops.attention_prefix_prefill(s["qs"], kp, vp, P, s["k"], s["v"], s["start"], B, S, return_lse=True)
        ops.attention_weights(s["qs"], lse, s["k"], s["start"], B, S, s["w"])
        ops.kv_evict(s["k"], s["v"], s["w"], s["tok"], s["n"], own, 25, recent=3)
        return out, pre, lse

    def fill(s, seed):
        r = _gen(seed)
        for t in ("k", "v", "q", "qs"):
            s[t].copy_(torch.randn(s[t].shape, generator=r, device="cuda"))
        s["w"].zero_()
        s["tok"].copy_(torch.arange(rows, device="cuda").expand(B, nkv, rows))
        s["n"].copy_(torch.randint(1, own + 1, (B,), generator=r, device="cuda"))
        s["start"].copy_(torch.randint(0, rows - S, (B,), generator=r, device="cuda"))

    states, graphs, outs = [state(), state()], [], []
    for s in states:
        fill(s, 1)
        step(s)  # outside the capture first
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    for seed in (2, 3):
        for i, s in enumerate(states):
            fill(s, 10 * seed + i)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i, s in enumerate(states):
            e = state()
            fill(e, 10 * seed + i)
            want = step(e)
            torch.cuda.synchronize()
            for got, ref in zip(outs[i], want):
                assert torch.equal(got, ref)
            for t in ("k", "v", "w", "tok", "n"):
                assert torch.equal(s[t], e[t]), t
    assert _error() == 0


def test_offsets_past_32_bits(cuda_dev):
    """Caches of more than 2^31 elements: the last slot's last rows."""
    from nki_moe_7013_b200 import ops

    g = _gen(14)
    n_slots, nkv, nh, max_seq, L = 3, 8, 16, 700000, 699990
    k = torch.zeros(n_slots, nkv, max_seq, HD, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    lo, S = L - 300, 40
    k[2, :, lo:L], v[2, :, lo:L] = _randn(g, nkv, 300, HD), _randn(g, nkv, 300, HD)
    kk, vv = k[2, :, lo:L].clone(), v[2, :, lo:L].clone()
    q, qs = _randn(g, 1, nh, HD), _randn(g, S, nh, HD)
    w = torch.zeros(n_slots, nkv, max_seq, device="cuda")
    tok = torch.arange(max_seq, dtype=torch.int32, device="cuda").expand(n_slots, nkv, max_seq).contiguous()
    slot, start = _i32([2]), _i32([lo])
    out = ops.attention_decode_weights(q, k, v, _i32([L]), L, w, cache_slot=slot, kv_start=start)
    wide = ops.attention_prefix_decode(q, k, v, L, k, v, _i32([0]), 0, prefix_slot=2)  # a prefix past 2^31
    pre, lse = ops.attention_prefix_prefill(qs, None, None, 0, k, v, _i32([L - S]), 1, S, cache_slot=slot,
                                            kv_start=start, return_lse=True)
    w2 = torch.zeros_like(w)
    ops.attention_weights(qs, lse, k, _i32([L - S]), 1, S, w2, cache_slot=slot, kv_start=start, max_len=L)
    assert _error() == 0
    for gr in range(nkv):
        h = slice(gr * 2, gr * 2 + 2)
        r = Ref(q[0, h], kk[gr], vv[gr])
        _check_out(out.view(nh, HD)[h], r.out, r.mag, r.D)
        _check_weights(w[2, gr, lo:L], r.p.sum(dim=0), torch.zeros(300, dtype=torch.float64, device="cuda"), r.D)
        # the rows before `lo` hold zeros: scores of 0 and no value
        s = torch.cat([torch.exp(q[0, h].double() @ kk[gr].double().T * C), torch.full((2, 1), float(lo), device="cuda",
                                                                                       dtype=torch.float64)], dim=1)
        p = s[:, :300] / s.sum(dim=1, keepdim=True)
        _check_out(wide.view(nh, HD)[h], p @ vv[gr].double(), p @ vv[gr].double().abs(), r.D)
    hide = torch.arange(lo, L, device="cuda")[None] > torch.arange(L - S, L, device="cuda")[:, None]
    for h in range(nh):
        r = Ref(qs[:, h], kk[h // 2], vv[h // 2], hide)
        _check_out(pre.view(S, nh, HD)[:, h], r.out, r.mag, r.D)
    assert abs(float(w2.double().sum()) - S * nh) <= S * nh * 2.0 ** -12
    assert not w2[:2].any() and not w2[2, :, :lo].any() and not w2[2, :, L:].any()
    n = _i32([L])
    ops.kv_evict(k, v, w, tok, n, L, 100, recent=10, cache_slot=slot, kv_start=start)
    assert _error() == 0 and n.tolist() == [100] and start.tolist() == [0]
    assert bool((tok[2, :, :100] >= lo).all()) and bool((tok[2, :, 100:L] == -1).all())
    for gr in range(nkv):
        rows = tok[2, gr, :100].long() - lo
        assert torch.equal(k[2, gr, :100], kk[gr, rows]) and torch.equal(v[2, gr, :100], vv[gr, rows])
        assert set(range(290, 300)) <= set(rows.tolist()) and len(set(rows.tolist())) == 100


def test_wrappers_refuse_what_does_not_fit(cuda_dev):
    """Wrong types, shapes, layouts: refused with a name, before a launch."""
    from nki_moe_7013_b200 import _C, ops

    B, nh, nkv, L = 2, 8, 2, 16
    bf = dict(dtype=torch.bfloat16, device="cuda")
    k, v, q = torch.zeros(B, nkv, L, HD, **bf), torch.zeros(B, nkv, L, HD, **bf), torch.zeros(B, nh, HD, **bf)
    n, w = _i32([3, 4]), torch.zeros(B, nkv, L, device="cuda")
    lse, tok = torch.zeros(B, nh, device="cuda"), torch.zeros(B, nkv, L, dtype=torch.int32, device="cuda")

    def decode(**kw):
        a = dict(q=q, k_prefix=k, v_prefix=v, prefix_len=4, k_cache=k, v_cache=v, kv_len=n, max_len=L)
        a.update(kw)
        return ops.attention_prefix_decode(**a)

    def prefill(**kw):
        a = dict(q=q, k_prefix=k, v_prefix=v, prefix_len=4, k_cache=k, v_cache=v, q_start=n, B=B, S=1)
        a.update(kw)
        return ops.attention_prefix_prefill(**a)

    def weights(**kw):
        a = dict(q=q, lse=lse, k_cache=k, q_start=n, B=B, S=1, weights=w)
        a.update(kw)
        return ops.attention_weights(**a)

    def evict(**kw):
        a = dict(k_cache=k, v_cache=v, weights=w, tokens=tok, kv_len=n.clone(), max_len=L, keep=3)
        a.update(kw)
        return ops.kv_evict(**a)

    for call in (decode, prefill, weights, evict):
        call()
    half = torch.zeros(B, nkv, L, HD, dtype=torch.float16, device="cuda")
    strided = torch.zeros(B, nkv, HD, L, **bf).transpose(2, 3)
    for call, kw, err, name in (
            (decode, dict(q=q.float()), TypeError, "q must"), (decode, dict(q=None), TypeError, "q must"),
            (decode, dict(k_cache=half), TypeError, "k_cache"), (decode, dict(v_cache=strided), ValueError, "v_cache"),
            (decode, dict(q=q[:1].contiguous()), ValueError, "q must"), (decode, dict(kv_len=n.long()), TypeError, "kv_len"),
            (decode, dict(kv_len=n.view(1, 2)), ValueError, "kv_len"), (decode, dict(kv_start=n[:1]), ValueError, "kv_start"),
            (decode, dict(k_prefix=None), ValueError, "prefix"), (decode, dict(v_prefix=k[:1].contiguous()), ValueError, "prefix"),
            (decode, dict(k_prefix=k[:, :1].contiguous(), v_prefix=v[:, :1].contiguous()), ValueError, "prefix"),
            (decode, dict(weights=w[:1].contiguous()), ValueError, "weights"), (decode, dict(weights=w.half()), TypeError, "weights"),
            (decode, dict(workspace=torch.zeros(4, device="cuda")), TypeError, "workspace"),
            (decode, dict(q=torch.zeros(3, nh, HD, **bf), kv_len=_i32([1, 1, 1])), ValueError, "cache_slot"),
            (decode, dict(prefix_len=17), _C.QmoeError, "prefix"), (decode, dict(prefix_slot=2), _C.QmoeError, "prefix"),
            (decode, dict(max_len=17), _C.QmoeError, "sizes"), (decode, dict(scale=0.0), _C.QmoeError, "scale"),
            (decode, dict(q=torch.zeros(B, 7, HD, **bf)), _C.QmoeError, "heads"),
            (prefill, dict(q_start=n.float()), TypeError, "q_start"), (prefill, dict(S=2), ValueError, "q must"),
            (prefill, dict(cache_slot=n[:1]), ValueError, "cache_slot"), (prefill, dict(prefix_len=-1), _C.QmoeError, "prefix"),
            (weights, dict(lse=lse.double()), TypeError, "lse"), (weights, dict(lse=lse[:1].contiguous()), ValueError, "lse"),
            (weights, dict(weights=tok), TypeError, "weights"), (weights, dict(max_len=0), _C.QmoeError, "sizes"),
            (evict, dict(tokens=tok.long()), TypeError, "tokens"), (evict, dict(v_cache=k[:1].contiguous()), ValueError, "cache"),
            (evict, dict(keep=-1), _C.QmoeError, "recent"), (evict, dict(recent=4), _C.QmoeError, "recent"),
            (evict, dict(kv_len=n.tolist()), TypeError, "kv_len")):
        with pytest.raises(err, match=name):
            call(**kw)
    with pytest.raises(TypeError, match="weights"):
        ops.attention_decode_weights(q, k, v, n, L, None)
    with pytest.raises(ValueError, match="together"):
        ops.qk_norm_rope(torch.zeros(1, 12 * HD, **bf), n[:1].contiguous(), torch.ones(HD, device="cuda"),
                         torch.ones(HD, device="cuda"), torch.ones(64, device="cuda"), nh, nkv, 1e-6, k, v,
                         row_tokens=tok)
    assert _error() == 0

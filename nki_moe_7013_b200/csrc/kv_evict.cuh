// Eviction from a KV cache by accumulated attention weight.
//
// Of the live rows [kv_start, kv_len) of each (sequence, KV head),
// n = min(keep, live) stay: first the rows of the `recent` newest tokens, then
// those of the largest weight (equal weights: the lower row first; NaN counts
// as the largest).  Attention does not depend on the order of a cache's rows
// (a key carries its position's rotation), so nothing is shifted: the i-th
// kept row beyond n moves into the i-th free row below n.  Sources lie at or
// beyond n and destinations below it, so the moves need no order among
// themselves, and an eviction of a few rows from a long cache moves only
// these few.
//
// kv_evict_select_kernel (a cluster of one to eight CTAs per (sequence, KV
// head), each holding a run of its rows) finds the n-th largest of the 32-bit
// order keys eight bits at a time, lists the moves and clears the weights and
// tokens of the rows that go; kv_evict_move_kernel copies the kept rows with
// theirs over all SMs and sets the new lengths.
//
// Bound by latency: the selection is a chain of short passes (lengths, the
// newest token, two to four digits, ranks, the lists) of some 1,500 to 5,000
// cycles each, a barrier of the CTA or its cluster after every one, and the
// move waits for it.  8 sequences of 2,176 rows to 2,048 take 15.9 us, 4 of
// up to 16,384 to 2,048 (28 MB moved) 23.7.
#pragma once

#include "attn_shared.cuh"
#include "common.cuh"

namespace qmoe {

constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvMaxCached = 32768;  // order keys a CTA holds in shared memory (128 KB); rows past it are re-read from L2
constexpr int kEvMaxCluster = 8;
constexpr int kEvMoveRows = 32;      // rows per CTA of the move kernel
constexpr int kEvHeld = 4;           // rows of a thread whose weight and token are read once, into registers

struct EvictArgs {
  float* weights;    // (n_slots, nkv, max_seq)
  int32_t* tokens;   // (n_slots, nkv, max_seq)
  int32_t* kv_len;
  int32_t* kv_start;
  const int32_t* cache_slot;
  int32_t* plan;     // [B*nkv][2 + 2 * cap]: moves (-1: refused), n, source rows, destination rows
  int B, nkv, n_slots, max_seq, max_len, keep, recent, cap, cached;
};

// Larger key = kept earlier.
__device__ __forceinline__ uint32_t evict_key(float w, bool is_recent) {
  if (is_recent) return 0xFFFFFFFFu;
  if (isnan(w)) return 0xFFFFFFFEu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 and +0 tie
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sum over the warps before this one, and over all (one value per warp in w).
__device__ __forceinline__ int2 warps_before(const int* w, int warp, int warps, int lane) {
  const int v = lane < warps ? w[lane] : 0;
  return make_int2(__reduce_add_sync(0xFFFFFFFFu, lane < warp ? v : 0), __reduce_add_sync(0xFFFFFFFFu, v));
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
// Barrier of the CTA, or of its whole cluster (shared and global memory).
__device__ __forceinline__ void cluster_sync(int ranks) {
  if (ranks == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
// The word at p in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ int ld_cluster(const int* p, int rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__global__ void __launch_bounds__(kEvThreads) kv_evict_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t ev_keys[];  // of this CTA's first a.cached rows
  __shared__ alignas(16) int hist[2][256];  // read by the whole cluster
  __shared__ int s_newest, s_eq, s_holes, s_moves;
  __shared__ alignas(16) int hsum[256];
  __shared__ int wsum[kEvWarps], wsum2[kEvWarps];
  __shared__ int s_pick, s_rest, s_count;
  griddep_wait();
  griddep_launch_dependents();
  const int rank = int(cluster_rank()), ranks = int(cluster_size());
  const int unit = int(blockIdx.x) / ranks;
  const int b = unit / a.nkv, kvh = unit % a.nkv;
  const int threads = blockDim.x, warps = threads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* plan = a.plan + size_t(unit) * (2 + 2 * size_t(a.cap));
  int32_t* src = plan + 2;
  int32_t* dst = src + a.cap;
  int slot, lo, len;
  const bool ok = own_range(a.kv_len, a.cache_slot, a.kv_start, b, a.max_len, a.n_slots, slot, lo, len);
  if (!ok || slot_seen_before(a.cache_slot, b, lane)) {
    // a bad length or slot, or a slot given twice: nothing of this entry changes
    if (tid == 0) {
      record_device_error(kDevErrBadIndex);
      plan[0] = -1;
    }
    return;
  }
  const int n = min(a.keep, len - lo);
  const bool all = n == len - lo;  // every live row stays
  float* w = a.weights + (size_t(slot) * a.nkv + kvh) * a.max_seq;
  int32_t* tok = a.tokens + (size_t(slot) * a.nkv + kvh) * a.max_seq;
  // this CTA's run of rows, and each warp's run within it: ranks in row order
  // are sums over the CTAs and warps before, plus ballots inside the run
  const int seg = ((len + ranks - 1) / ranks + 31) / 32 * 32;
  const int s0 = min(len, rank * seg), s1 = min(len, s0 + seg);
  const int run = ((s1 - s0 + warps - 1) / warps + 31) / 32 * 32;
  const int r_begin = min(s1, s0 + warp * run), r_end = min(s1, r_begin + run);

  // the newest token; the first rows' weights are read along with their tokens
  float w_held[kEvHeld];
  int t_held[kEvHeld];
  int newest = INT32_MIN;
  if (!all && n > 0) {
#pragma unroll
    for (int i = 0; i < kEvHeld; ++i) {
      const int r = s0 + i * threads + tid;
      const bool live = r >= lo && r < s1;
      w_held[i] = live ? w[r] : 0.f;
      t_held[i] = live && a.recent > 0 ? tok[r] : INT32_MIN;
    }
  }
  if (a.recent > 0 && !all) {
#pragma unroll
    for (int i = 0; i < kEvHeld; ++i) newest = max(newest, t_held[i]);
    for (int r = s0 + kEvHeld * threads + tid; r < s1; r += threads)
      if (r >= lo) newest = max(newest, tok[r]);
    newest = __reduce_max_sync(0xFFFFFFFFu, newest);
    if (lane == 0) wsum[warp] = newest;
    __syncthreads();
    newest = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? wsum[lane] : INT32_MIN);
    if (ranks > 1) {
      if (tid == 0) s_newest = newest;
      cluster_sync(ranks);
      newest = __reduce_max_sync(0xFFFFFFFFu, lane < ranks ? ld_cluster(&s_newest, lane) : INT32_MIN);
    }
  }
  const long long old_most = (long long)newest - a.recent;  // tokens above it are recent
  auto fresh_key = [&](int r) { return evict_key(w[r], a.recent > 0 && (long long)tok[r] > old_most); };
  auto key_at = [&](int r) { return r - s0 < a.cached ? ev_keys[r - s0] : fresh_key(r); };

  // The n-th largest key T, eight bits at a time from the highest: rows above
  // T stay, and `take_eq` of those equal to it.  A warp's equal digits are
  // counted with one addition: the top digit is the exponent, which most rows
  // share.
  uint32_t T = 0;
  int take_eq = INT32_MAX;
  if (!all && n > 0) {
    for (int i = tid; i < 512; i += threads) hist[i >> 8][i & 255] = 0;
    __syncthreads();
    auto count = [&](int r, bool live, uint32_t k) {
      if (live && r - s0 < a.cached) ev_keys[r - s0] = k;
      const uint32_t same = __match_any_sync(0xFFFFFFFFu, live ? k >> 24 : 256u);
      if (live && lane == __ffs(same) - 1) atomicAdd(&hist[0][k >> 24], __popc(same));
    };
#pragma unroll
    for (int i = 0; i < kEvHeld; ++i) {
      const int r = s0 + i * threads + tid;
      if (s0 + i * threads < s1)
        count(r, r >= lo && r < s1, evict_key(w_held[i], a.recent > 0 && (long long)t_held[i] > old_most));
    }
    for (int r0 = s0 + kEvHeld * threads; r0 < s1; r0 += threads) {
      const int r = r0 + tid;
      const bool live = r >= lo && r < s1;
      count(r, live, live ? fresh_key(r) : 0u);
    }
    uint32_t mask = 0xFF000000u;
    int want = n;
    for (int shift = 24, pass = 0;; shift -= 8, ++pass) {
      cluster_sync(ranks);  // the counts of this digit are there
      const int* h = hist[pass & 1];
      if (ranks > 1) {
        for (int i = tid; i < 256; i += threads) {
          int c[kEvMaxCluster], sum = 0;  // all loads in flight
#pragma unroll
          for (int k = 0; k < kEvMaxCluster; ++k) c[k] = k < ranks ? ld_cluster(h + i, k) : 0;
#pragma unroll
          for (int k = 0; k < kEvMaxCluster; ++k) sum += c[k];
          hsum[i] = sum;
        }
        h = hsum;
        __syncthreads();
      }
      if (warp == 0) {
        // lane i holds digits 255-8i .. 248-8i, largest first
        const int4 lo4 = *reinterpret_cast<const int4*>(h + 248 - lane * 8);
        const int4 hi4 = *reinterpret_cast<const int4*>(h + 252 - lane * 8);
        const int c[8] = {hi4.w, hi4.z, hi4.y, hi4.x, lo4.w, lo4.z, lo4.y, lo4.x};
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += c[e];
        int incl = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int t = __shfl_up_sync(0xFFFFFFFFu, incl, off);
          if (lane >= off) incl += t;
        }
        int above = incl - sum;
        if (above < want && want <= incl) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (above < want && want <= above + c[e]) {
              s_pick = 255 - lane * 8 - e;
              s_rest = want - above;
              s_count = c[e];
            }
            above += c[e];
          }
        }
      } else if (warp == 1) {
        // (the cluster read these counts before its last barrier)
        for (int i = lane; i < 256; i += 32) hist[(pass & 1) ^ 1][i] = 0;
      }
      __syncthreads();
      T |= uint32_t(s_pick) << shift;
      want = s_rest;
      if (want == s_count) break;  // every row with these digits stays: T's other digits are 0
      if (shift == 0) {
        take_eq = want;
        break;
      }
      const int next = shift - 8;
      int* hn = hist[(pass & 1) ^ 1];
      for (int r = max(lo, s0) + tid; r < s1; r += threads) {
        const uint32_t k = key_at(r);
        if ((k & mask) == T) atomicAdd(&hn[(k >> next) & 255], 1);
      }
      mask |= 0xFFu << next;
    }
  }
  __syncthreads();  // every thread's keys

  const uint32_t before = (1u << lane) - 1u;
  int eq_before = 0;
  if (take_eq != INT32_MAX) {  // only then do equal rows need their rank
    int eq = 0;
    for (int r0 = r_begin; r0 < r_end; r0 += 32) {
      const int r = r0 + lane;
      eq += __popc(__ballot_sync(0xFFFFFFFFu, r < r_end && r >= lo && key_at(r) == T));
    }
    if (lane == 0) wsum[warp] = eq;
    __syncthreads();
    const int2 e = warps_before(wsum, warp, warps, lane);
    eq_before = e.x;
    if (ranks > 1) {
      if (tid == 0) s_eq = e.y;
      cluster_sync(ranks);
      eq_before += __reduce_add_sync(0xFFFFFFFFu, lane < rank ? ld_cluster(&s_eq, lane) : 0);
    }
    __syncthreads();
  }
  // two passes: count the free rows below n and the kept rows beyond it, then
  // list them; lane i keeps the i-th 32 rows' masks for the second pass
  int holes_before = 0, moves_before = 0, n_moves = 0, e_later = 0;
  uint32_t held_holes = 0, held_moves = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int e = pass == 0 ? eq_before : e_later, holes = holes_before, moves = moves_before;
    for (int r0 = r_begin, it = 0; r0 < r_end; r0 += 32, ++it) {
      const int r = r0 + lane;
      uint32_t hs, ms;
      if (pass == 1 && it < 32) {
        hs = __shfl_sync(0xFFFFFFFFu, held_holes, it);
        ms = __shfl_sync(0xFFFFFFFFu, held_moves, it);
      } else {
        const bool live = r < r_end && r >= lo;
        bool kept = live && all;
        if (!all && n > 0) {
          const uint32_t k = live ? key_at(r) : 0u;
          const bool is_eq = live && k == T;
          kept = live && (k > T || is_eq);
          if (take_eq != INT32_MAX) {
            const uint32_t eqs = __ballot_sync(0xFFFFFFFFu, is_eq);
            kept = kept && (!is_eq || e + __popc(eqs & before) < take_eq);
            e += __popc(eqs);
          }
        }
        hs = __ballot_sync(0xFFFFFFFFu, r < r_end && r < n && !kept);
        ms = __ballot_sync(0xFFFFFFFFu, kept && r >= n);
        if (lane == it) {
          held_holes = hs;
          held_moves = ms;
        }
        if (it == 31 && pass == 0) e_later = e;
      }
      const bool hole = hs >> lane & 1, move = ms >> lane & 1;
      if (pass == 1) {
        if (hole) dst[holes + __popc(hs & before)] = r;
        if (move) {
          src[moves + __popc(ms & before)] = r;
        } else if (r >= n && r < r_end) {  // (a moved row's are cleared once they are copied)
          w[r] = 0.f;
          tok[r] = -1;
        }
      }
      holes += __popc(hs);
      moves += __popc(ms);
    }
    if (pass == 0) {
      if (lane == 0) {
        wsum[warp] = holes;
        wsum2[warp] = moves;
      }
      __syncthreads();
      const int2 h = warps_before(wsum, warp, warps, lane), m = warps_before(wsum2, warp, warps, lane);
      holes_before = h.x;
      moves_before = m.x;
      n_moves = m.y;
      if (ranks > 1) {
        if (tid == 0) {
          s_holes = h.y;
          s_moves = m.y;
        }
        cluster_sync(ranks);
        const int hk = lane < ranks ? ld_cluster(&s_holes, lane) : 0, mk = lane < ranks ? ld_cluster(&s_moves, lane) : 0;
        holes_before += __reduce_add_sync(0xFFFFFFFFu, lane < rank ? hk : 0);
        moves_before += __reduce_add_sync(0xFFFFFFFFu, lane < rank ? mk : 0);
        n_moves = __reduce_add_sync(0xFFFFFFFFu, mk);
      }
      if (rank == 0 && tid == 0) {
        plan[0] = n_moves;
        plan[1] = n;
      }
    }
  }
  cluster_sync(ranks);  // every CTA's words were read
}

// grid (ceil(cap / 32), B * nkv): half a warp copies one 256-byte K row and
// one V row, with the row's weight and token, which are cleared where they were;
// the CTA's 32 rows are all loaded before the first store.
__global__ void __launch_bounds__(256) kv_evict_move_kernel(const EvictArgs a, __nv_bfloat16* k_cache,
                                                            __nv_bfloat16* v_cache) {
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y / a.nkv, kvh = blockIdx.y % a.nkv;
  const int32_t* plan = a.plan + size_t(blockIdx.y) * (2 + 2 * size_t(a.cap));
  const int sub = threadIdx.x >> 4, c = threadIdx.x & 15;
  int from[2], to[2];  // read beside the number of moves; past it they are not used
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int idx = blockIdx.x * kEvMoveRows + i * 16 + sub;
    from[i] = idx < a.cap ? plan[2 + idx] : 0;
    to[i] = idx < a.cap ? plan[2 + a.cap + idx] : 0;
  }
  const int moves = plan[0];
  if (moves < 0) return;
  if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0) {
    a.kv_len[b] = plan[1];
    if (a.kv_start) a.kv_start[b] = 0;
  }
  const int slot = a.cache_slot ? a.cache_slot[b] : b;
  const size_t head = (size_t(slot) * a.nkv + kvh) * a.max_seq;
  // lane 0 of a row also carries its weight, lane 1 its token
  int32_t* words = (c == 0 ? reinterpret_cast<int32_t*>(a.weights) : a.tokens) + head;
  uint4 kr[2], vr[2];
  int word[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (blockIdx.x * kEvMoveRows + i * 16 + sub >= moves) continue;
    kr[i] = reinterpret_cast<const uint4*>(k_cache + (head + from[i]) * kAttnD)[c];
    vr[i] = reinterpret_cast<const uint4*>(v_cache + (head + from[i]) * kAttnD)[c];
    if (c < 2) word[i] = words[from[i]];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (blockIdx.x * kEvMoveRows + i * 16 + sub >= moves) continue;
    reinterpret_cast<uint4*>(k_cache + (head + to[i]) * kAttnD)[c] = kr[i];
    reinterpret_cast<uint4*>(v_cache + (head + to[i]) * kAttnD)[c] = vr[i];
    if (c < 2) {
      words[to[i]] = word[i];
      words[from[i]] = c == 0 ? 0 : -1;  // (0.f is all zero bits)
    }
  }
}

}  // namespace qmoe

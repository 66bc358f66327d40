// Attention weights of a prompt, summed over its queries:
//
//   weights[slot, g, j] (+)= sum_i sum_{h in g} exp(c q_ih . k_j - lse_ih)
//
// over the queries i that see row j (j <= q_start + i, and j >= kv_start), with
// lse the log-sum-exp of the query's whole row, which the prefill returns.  The
// scores are computed a second time; no S x L matrix exists.
//
// S^T = K Q^T on the tensor core (M = 128 keys, N = 128 query rows, fp32 in
// TMEM), so that a thread owns one key and adds up its TMEM lane: no reduction
// across threads.  A query tile is 128 / G positions times the group's G
// heads.  Persistent CTAs, one per SM, draw units in turn: 512 cache rows (four
// K tiles, each with a TMEM accumulator and a group of four summing warps of
// its own) of one (sequence, KV head) against a chunk of the query tiles that
// see them.  Two producer warps, one per query slot, stream the query tiles
// with their lse, and the next unit's K tiles as they become free.  Where the
// queries are cut into several chunks, their sums go to the workspace and
// attn_weights_join_kernel adds them in chunk order: no atomics, run-to-run
// identical.
//
// Four K tiles per query tile: a quarter of the query tiles' traffic through L2
// (550 MB with one, for a 4,096-token prompt: 124 us instead of 111).  Then the
// exponentials bound it: 128 x 128 per tile at 16 a cycle and SM are 1,024
// cycles, against 512 of the products; measured some 1,230 a tile, in 109 us for
// a 4,096-token prompt (0.63 PFLOP/s).  (The approximate exp2 leaves the totals
// within 1e-7 to 6e-7 of 64 bits.)  (A quarter or a half of the exponentials
// as a degree-5 polynomial on the FMA pipe changed nothing or cost 5 %: ten
// multiply-adds take as long as they save.  Three K tiles with a fourth
// accumulator to fill ahead took 142 us.)
#pragma once

#include "attn_shared.cuh"
#include "common.cuh"
#include "flash_prefill.cuh"

namespace qmoe {

constexpr int kAwTiles = 4;       // K tiles of a unit = TMEM accumulators = groups of 4 summing warps
constexpr int kAwKeys = kAwTiles * kFaRows;
constexpr int kAwSlots = 2;       // query tiles in flight = producer warps
constexpr int kAwThreads = (4 * kAwTiles + kAwSlots + 1) * 32;  // and the MMA warp
constexpr int kAwBarriers = 4 * kAwSlots + 4 * kAwTiles + 1;
constexpr int kAwInfo = 8;        // ints per slot
constexpr int kAwSmemBytes = (kAwTiles + kAwSlots) * kFaTileBytes + 1024 + kAwSlots * (kFaRows + kAwInfo) * 4 +
                             kAwBarriers * 8 + 8 + (kAwSlots + kAwTiles) * 4;

struct AttnWeightsArgs {
  const float* lse;
  const int32_t* q_start;
  const int32_t* cache_slot;
  const int32_t* kv_start;
  float* weights;
  float* partial;  // [n_chunks][B*nkv][key_blocks*512], or null: one chunk
  int B, S, nh, nkv, G, n_slots, max_seq, max_len, accumulate;
  int key_blocks, n_chunks, chunk;  // chunk: query tiles
  float scale_log2;
};

// 512 rows of one (sequence, KV head) and the queries that see them.
struct AwBlock {
  int slot, L0, L, kv0, key0, i0, q_tiles;  // q_tiles 0: nothing to do
  bool bad;
};
__device__ __forceinline__ AwBlock aw_block(const AttnWeightsArgs& a, int b, int kb, int lane) {
  AwBlock t;
  t.L0 = a.q_start[b];
  t.slot = a.cache_slot ? a.cache_slot[b] : b;
  t.bad = t.L0 < 0 || t.L0 > a.max_len - a.S || t.slot < 0 || t.slot >= a.n_slots ||
          slot_seen_before(a.cache_slot, b, lane);  // a slot given twice would race
  t.L = t.L0 + a.S;
  t.kv0 = a.kv_start ? max(0, min(a.kv_start[b], t.L)) : 0;
  t.key0 = t.kv0 + kb * kAwKeys;
  t.i0 = max(0, t.key0 - t.L0);
  const int per_q = kFaRows / a.G;
  t.q_tiles = t.bad || t.key0 >= t.L ? 0 : (a.S - t.i0 + per_q - 1) / per_q;
  return t;
}

// tcgen05.wait::ld that the loaded registers pass through, so that no use of
// them can move above it.
__device__ __forceinline__ void tmem_ld_wait_x32(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                 "+f"(v[15])
               :
               : "memory");
  asm volatile(""
               : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}

// Flags of a slot's query tile: the last of its unit, the end of the CTA's
// tiles; from bit kAwSees on the K tiles that any of its queries sees, from
// bit kAwHolds on those that hold rows.
enum : int { kAwLast = 1, kAwEnd = 2, kAwSees = 8, kAwHolds = 16 };

__global__ void __launch_bounds__(kAwThreads, 1)
    attn_weights_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const AttnWeightsArgs a) {
  extern __shared__ uint8_t fa_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(fa_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;                               // [tiles]
  uint8_t* sQ = smem + kAwTiles * kFaTileBytes;     // [slots]
  float* s_neg = reinterpret_cast<float*>(sQ + kAwSlots * kFaTileBytes);  // [slots][128]: -lse, log2 units
  int* s_info = reinterpret_cast<int*>(s_neg + kAwSlots * kFaRows);       // [slots][8]
  uint64_t* bar = reinterpret_cast<uint64_t*>(s_info + kAwSlots * kAwInfo);
  uint64_t* q_full = bar;                  // [slots]: query tile landed
  uint64_t* q_empty = q_full + kAwSlots;   // [slots]: query tile multiplied
  uint64_t* full = q_empty + kAwSlots;     // [slots]: lse and info in place
  uint64_t* done = full + kAwSlots;        // [slots]: lse and info read
  uint64_t* k_full = done + kAwSlots;      // [tiles]: K tile landed
  uint64_t* k_empty = k_full + kAwTiles;   // [tiles]: the unit's products with it are done
  uint64_t* s_full = k_empty + kAwTiles;   // [tiles]: scores in the accumulator
  uint64_t* s_empty = s_full + kAwTiles;   // [tiles]: and read
  uint64_t* drain = s_empty + kAwTiles;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kAwBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* loads = reinterpret_cast<volatile int*>(tmem_slot + 2);  // issued per query slot, per K tile

  constexpr int kProd = 4 * kAwTiles, kMma = kProd + kAwSlots;  // first producer warp, MMA warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_q = kFaRows / a.G;  // query positions per tile
  griddep_wait();
  griddep_launch_dependents();
  // columns of no query (128 is no multiple of G) must hold numbers
  if (a.G * per_q < kFaRows) {
    for (int i = threadIdx.x; i < kAwSlots * kFaTileBytes / 16; i += kAwThreads)
      reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_shared();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAwSlots; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&full[i], 32);  // the lanes of the slot's producer
      mbar_init(&done[i], 4 * kAwTiles);
    }
    for (int i = 0; i < kAwTiles; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    for (int i = 0; i < kAwSlots + kAwTiles; ++i) loads[i] = 0;
    fence_mbarrier_init();
  }
  if (warp == kMma) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= kProd && warp < kMma) {
    // ---------------- producers: slot sl takes query tiles sl, sl + 2, ... of the CTA's units ----------------
    const int sl = warp - kProd;
    const int heads = a.nkv * a.B, per_chunk = a.key_blocks * heads;
    const int n_units = per_chunk * a.n_chunks;
    int col_i[4], col_h[4];  // this lane's columns lane + 32 k: query of the tile, head of the group
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      col_i[k] = (lane + 32 * k) / a.G;
      col_h[k] = (lane + 32 * k) % a.G;
    }
    int u = int(blockIdx.x) - int(gridDim.x);
    int c = 0, kb = 0, kvh = 0, b = 0, t = 0, t0 = 0, t1 = 0;
    int used[kAwTiles] = {}, tiles = 0;  // earlier units of each K tile's place; the unit's K tiles
    AwBlock blk = {};
    int past = 0;
    // `by` query tiles further; false past the last one, `past` tiles behind it
    auto advance = [&](int by) {
      t += by;
      while (t >= t1) {
        const int rest = t - t1;
#pragma unroll
        for (int g = 0; g < kAwTiles; ++g) used[g] += g < tiles;
        tiles = 0;
        do {
          u += gridDim.x;
          if (u >= n_units) {
            past = rest;
            return false;
          }
          // chunks outermost, then the key blocks from the lowest (seen by most
          // queries): the units that exist come in runs, which the CTAs share evenly
          c = u / per_chunk;
          kb = u % per_chunk / heads;
          kvh = u % heads % a.nkv;
          b = u % heads / a.nkv;
          blk = aw_block(a, b, kb, lane);
          if (sl == 0 && blk.bad && lane == 0) record_device_error(kDevErrBadIndex);
          if (sl == 0 && c == 0 && kb == 0 && !a.partial && !a.accumulate && !blk.bad) {
            float* w = a.weights + (size_t(blk.slot) * a.nkv + kvh) * a.max_seq;
            for (int j = lane; j < blk.kv0; j += 32) w[j] = 0.f;
          }
          t0 = c * a.chunk;
          t1 = min(blk.q_tiles, t0 + a.chunk);
        } while (t0 >= t1);
        tiles = min(kAwTiles, (blk.L - blk.key0 + kFaRows - 1) / kFaRows);
        t = t0 + rest;
      }
      return true;
    };
    float nl[4];
    auto load_lse = [&]() {
      const int i_first = blk.i0 + t * per_q;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i_first + col_i[k];
        nl[k] = -INFINITY;  // no query, or one without keys: exp2(s - inf) = 0
        if (col_i[k] < per_q && i < a.S) {
          const float e = a.lse[(size_t(b) * a.S + i) * a.nh + kvh * a.G + col_h[k]];
          if (e != -INFINITY) nl[k] = e * -1.4426950408889634f;
        }
      }
    };
    bool more = advance(sl);
    if (more) load_lse();
    for (int r = 0;; ++r) {  // the slot's r-th query tile
      const int i_first = blk.i0 + t * per_q;
      if (more) {
        if (r > 0 && !fa_wait_warp(&q_empty[sl], (r - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer)) break;
        if (lane == 0) {
          loads[sl] = r + 1;
          mbar_arrive_expect_tx(&q_full[sl], per_q * a.G * kFaD * 2);
          tma_load_3d(sQ + sl * kFaTileBytes, &tm_q, 0, kvh * a.G, b * a.S + i_first, &q_full[sl]);
          tma_load_3d(sQ + sl * kFaTileBytes + kFaHalfBytes, &tm_q, 64, kvh * a.G, b * a.S + i_first, &q_full[sl]);
        }
        if (t == t0) {
          bool ok = true;
#pragma unroll
          for (int g = 0; g < kAwTiles; ++g) {
            if (g >= tiles || !ok) continue;
            // The place's last use must be done.  A parity wait also passes on
            // a barrier two phases behind, and the slots take turns at loading:
            // with units of one query tile the use before the last may still
            // run, so k_empty alone will not do.  First the last use's tile must
            // have landed: it was loaded once the use before was done.  The uses
            // before that have landed, since the q_empty waited for above
            // follows them (below).
            ok = used[g] == 0 ||
                 (fa_wait_warp(&k_full[g], (used[g] - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer) &&
                  fa_wait_warp(&k_empty[g], (used[g] - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer));
            if (ok && lane == 0) {
              const int z = blk.slot * a.nkv + kvh, y = blk.key0 + g * kFaRows;
              loads[kAwSlots + g] = used[g] + 1;
              mbar_arrive_expect_tx(&k_full[g], kFaTileBytes);
              tma_load_3d(sK + g * kFaTileBytes, &tm_k, 0, y, z, &k_full[g]);
              tma_load_3d(sK + g * kFaTileBytes + kFaHalfBytes, &tm_k, 64, y, z, &k_full[g]);
            }
          }
          if (!ok) break;
        }
      }
      if (r > 0 && !fa_wait_warp(&done[sl], (r - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer)) break;
      if (!more) {
        if (past == 0) {  // the CTA's tiles end here
          if (lane == 0) s_info[sl * kAwInfo] = kAwEnd;
          mbar_arrive(&full[sl]);
        }
        break;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s_neg[sl * kFaRows + lane + 32 * k] = nl[k];
      if (lane == 0) {
        int* info = s_info + sl * kAwInfo;
        const int n_q = min(per_q, a.S - i_first);
        // K tiles whose first row the tile's last query sees
        const int seen = max(0, min(tiles, (blk.L0 + i_first + n_q - 1 - blk.key0) / kFaRows + 1));
        info[0] = (t == t1 - 1 ? kAwLast : 0) | ((1 << seen) - 1) << kAwSees | ((1 << tiles) - 1) << kAwHolds;
        info[1] = blk.key0;
        info[2] = blk.L;
        info[3] = blk.L0 + i_first;  // position of the first query
        info[4] = n_q * a.G;         // columns that are queries
        // where the sums go, indexed by the cache row
        *reinterpret_cast<float**>(info + 6) =
            a.partial ? a.partial + ((size_t(c) * heads + b * a.nkv + kvh) * a.key_blocks + kb) * kAwKeys - blk.key0
                      : a.weights + (size_t(blk.slot) * a.nkv + kvh) * a.max_seq;
      }
      mbar_arrive(&full[sl]);
      more = advance(kAwSlots);
      if (more) load_lse();
    }
  } else if (warp == kMma) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      const uint32_t idesc = make_idesc_bf16(kFaRows, kFaRows);
      const uint64_t k_desc = make_sw128_desc(smem_u32(sK)), q_desc = make_sw128_desc(smem_u32(sQ));
      int units[kAwTiles] = {}, uses[kAwTiles] = {};  // of each K tile's place, of each accumulator
      bool ok = true;
      for (int s = 0; ok; ++s) {
        const int sl = s % kAwSlots;
        if (!fa_wait(&full[sl], (s / kAwSlots) & 1, abort_flag, kDevErrWaitTimeoutMma)) break;
        const int flags = s_info[sl * kAwInfo];
        if (flags & kAwEnd) break;
        if (!fa_wait(&q_full[sl], (s / kAwSlots) & 1, abort_flag, kDevErrWaitTimeoutMma)) break;
#pragma unroll
        for (int g = 0; g < kAwTiles; ++g) {
          if (!ok || !((flags >> (kAwSees + g)) & 1)) continue;
          ok = fa_wait(&k_full[g], units[g] & 1, abort_flag, kDevErrWaitTimeoutMma) &&
               (uses[g] == 0 || fa_wait(&s_empty[g], (uses[g] - 1) & 1, abort_flag, kDevErrWaitTimeoutMma));
          if (!ok) continue;
          ++uses[g];
          tc_fence_after();
          umma_bf16_k128(tmem_base + g * kFaRows, k_desc + ((g * kFaTileBytes) >> 4),
                         q_desc + ((sl * kFaTileBytes) >> 4), idesc);
          umma_commit(&s_full[g]);
        }
        // The unit's K tiles are free once these products are done; one that
        // no query of the chunk saw must have landed first.  All this before
        // q_empty, on which a slot takes the unit's K tiles as landed.
        if (flags & kAwLast) {
#pragma unroll
          for (int g = 0; g < kAwTiles; ++g) {
            if (!ok || !((flags >> (kAwHolds + g)) & 1)) continue;
            ok = fa_wait(&k_full[g], units[g] & 1, abort_flag, kDevErrWaitTimeoutMma);
            if (!ok) continue;
            umma_commit(&k_empty[g]);
            ++units[g];
          }
        }
        umma_commit(&q_empty[sl]);
      }
      umma_commit(drain);
      const unsigned long long start = globaltimer_ns();
      while (!mbar_try_wait(drain, 0)) {
        if (globaltimer_ns() - start > kWaitLimitNs) {
          record_device_error(kDevErrWaitTimeoutMma);
          break;
        }
      }
    }
  } else {
    // ---------------- sums: thread r of group g owns row key0 + 128 g + r ----------------
    const int g = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t s_row = tmem_base + (uint32_t((warp & 3) * 32) << 16) + g * kFaRows;
    const f32x2 scale2 = pack2(a.scale_log2, a.scale_log2);
    float total = 0.f;
    int uses = 0;
    for (int s = 0;; ++s) {
      const int sl = s % kAwSlots;
      if (!fa_wait_warp(&full[sl], (s / kAwSlots) & 1, abort_flag, kDevErrWaitTimeoutEpilogue)) break;
      const int* info = s_info + sl * kAwInfo;
      const int flags = info[0];
      if (flags & kAwEnd) break;
      const int key = info[1] + g * kFaRows + r, L = info[2];
      float* dst = *reinterpret_cast<float* const*>(info + 6);
      if ((flags >> (kAwSees + g)) & 1) {
        // columns [c0, c1): the queries of this sequence that see this key
        const int c0 = max(0, key - info[3]) * a.G, c1 = info[4];
        const bool whole = __all_sync(0xFFFFFFFFu, c0 == 0 && c1 == kFaRows);
        const float* neg = s_neg + sl * kFaRows;
        if (!fa_wait_warp(&s_full[g], uses & 1, abort_flag, kDevErrWaitTimeoutEpilogue)) break;
        ++uses;
        tc_fence_after();
        f32x2 sum2[4] = {0, 0, 0, 0};
        float edge[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tmem_ld_x32(s_row + c * 32, v);
          tmem_ld_wait_x32(v);
          if (c == 3) {  // the accumulator is read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[g]);
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const ulonglong2 n4 = *reinterpret_cast<const ulonglong2*>(neg + c * 32 + e);
#pragma unroll
              for (int k = 0; k < 4; k += 2) {
                float x0, x1;
                unpack2(fma2(pack2(v[e + k], v[e + k + 1]), scale2, k ? n4.y : n4.x), x0, x1);
                sum2[((e + k) >> 1) & 3] = add2(sum2[((e + k) >> 1) & 3], pack2(fa_exp2(x0), fa_exp2(x1)));
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int col = c * 32 + e;
              const float p = fa_exp2(fmaf(v[e], a.scale_log2, neg[col]));
              edge[e & 3] += col >= c0 && col < c1 ? p : 0.f;
            }
          }
        }
        float even, odd;
        unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), even, odd);
        total += whole ? even + odd : (edge[0] + edge[1]) + (edge[2] + edge[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[sl]);
      if (flags & kAwLast) {
        if (key < L) dst[key] = a.accumulate && !a.partial ? dst[key] + total : total;
        total = 0.f;
      }
    }
  }

  __syncthreads();
  // every load was waited for by the MMA thread, unless the CTA gave up
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < kAwSlots; ++i)
      if (loads[i]) fa_wait_landed(&q_full[i], (loads[i] - 1) & 1);
    for (int i = 0; i < kAwTiles; ++i)
      if (loads[kAwSlots + i]) fa_wait_landed(&k_full[i], (loads[kAwSlots + i] - 1) & 1);
  }
  if (warp == kMma) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// weights (+)= the chunks' sums, in chunk order; grid (key blocks * 4, B * nkv).
__global__ void __launch_bounds__(kFaRows) attn_weights_join_kernel(const AttnWeightsArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int kb = blockIdx.x / kAwTiles, b = blockIdx.y / a.nkv, kvh = blockIdx.y % a.nkv;
  const AwBlock t = aw_block(a, b, kb, threadIdx.x & 31);
  if (t.bad) return;  // recorded before
  float* w = a.weights + (size_t(t.slot) * a.nkv + kvh) * a.max_seq;
  if (blockIdx.x == 0 && !a.accumulate)
    for (int j = threadIdx.x; j < t.kv0; j += kFaRows) w[j] = 0.f;
  const int r = int(blockIdx.x % kAwTiles) * kFaRows + threadIdx.x, key = t.key0 + r;
  if (key >= t.L) return;
  const size_t step = size_t(a.nkv) * a.B * a.key_blocks * kAwKeys;
  const float* p = a.partial + (size_t(blockIdx.y) * a.key_blocks + kb) * kAwKeys + r;
  const int n = (t.q_tiles + a.chunk - 1) / a.chunk;
  float sum = 0.f;
#pragma unroll 8
  for (int c = 0; c < n; ++c) sum += p[c * step];
  w[key] = (a.accumulate ? w[key] : 0.f) + sum;
}

}  // namespace qmoe

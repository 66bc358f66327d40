// Attention weights of a prompt, summed over its queries:
//
//   weights[slot, g, j] (+)= sum_i sum_{h in g} exp(c q_ih . k_j - lse_ih)
//
// over the queries i that see row j (j <= q_start + i, and j >= kv_start), with
// lse the log-sum-exp of the query's whole row, which the prefill returns.  The
// scores are computed a second time; no S x L matrix exists.
//
// A CTA owns 128 cache rows of one (sequence, KV head) and runs over the
// queries that see them: S^T = K Q^T on the tensor core (M = 128 keys, N = 128
// query rows, fp32 in TMEM), so that a thread owns one key and adds up its
// TMEM lane: no reduction across threads, no atomics, run-to-run identical.
// Queries come as tiles of 128 / G positions times the group's G heads.  Two
// CTAs per SM, two TMEM accumulators and two Q slots each.  Bound by the
// 128 x 128 exponentials per tile (16 a cycle and SM: 1,024 cycles against
// 512 of the products).
#pragma once

#include "attn_shared.cuh"
#include "common.cuh"
#include "flash_prefill.cuh"

namespace qmoe {

constexpr int kAwThreads = 192;   // 4 summing warps, producer, MMA
constexpr int kAwSlots = 2;
constexpr int kAwBarriers = 8;
constexpr int kAwSmemBytes = (1 + kAwSlots) * kFaTileBytes + 1024 + kAwSlots * kFaRows * 4 + kAwBarriers * 8 + 16;

struct AttnWeightsArgs {
  const float* lse;
  const int32_t* q_start;
  const int32_t* cache_slot;
  const int32_t* kv_start;
  float* weights;
  int B, S, nh, nkv, G, n_slots, max_seq, max_len, accumulate;
  float scale_log2;
};

__global__ void __launch_bounds__(kAwThreads, 2)
    attn_weights_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const AttnWeightsArgs a) {
  extern __shared__ uint8_t fa_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(fa_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sQ = smem + kFaTileBytes;
  float* s_lse = reinterpret_cast<float*>(sQ + kAwSlots * kFaTileBytes);  // [slots][128], log2 units
  uint64_t* bar = reinterpret_cast<uint64_t*>(s_lse + kAwSlots * kFaRows);
  uint64_t* k_full = bar;
  uint64_t* full = bar + 1;    // [2]: Q tile landed
  uint64_t* s_full = bar + 3;  // [2]: products done (and the Q slot free)
  uint64_t* done = bar + 5;    // [2]: accumulator read
  uint64_t* drain = bar + 7;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kAwBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_tile = a.nkv * a.B;  // the lowest rows, which most queries see, first
  const int kt = int(blockIdx.x) / per_tile;
  const int kvh = int(blockIdx.x) % per_tile % a.nkv, b = int(blockIdx.x) % per_tile / a.nkv;
  griddep_wait();
  griddep_launch_dependents();
  const int L0 = a.q_start[b];
  const int slot = a.cache_slot ? a.cache_slot[b] : b;
  if (L0 < 0 || L0 > a.max_len - a.S || slot < 0 || slot >= a.n_slots || slot_seen_before(a.cache_slot, b, lane)) {
    if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);  // a slot given twice would race
    return;
  }
  const int L = L0 + a.S;
  const int kv0 = a.kv_start ? max(0, min(a.kv_start[b], L)) : 0;
  float* w = a.weights + (size_t(slot) * a.nkv + kvh) * a.max_seq;
  if (kt == 0 && !a.accumulate)
    for (int j = threadIdx.x; j < kv0; j += kAwThreads) w[j] = 0.f;
  const int key0 = kv0 + kt * kFaRows;
  if (key0 >= L) return;
  const int per_q = kFaRows / a.G;  // query positions per tile
  const int i0 = max(0, key0 - L0);
  const int n_tiles = (a.S - i0 + per_q - 1) / per_q;

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], 32);  // the producer warp: 31 lanes after their lse, one with the expected bytes
      mbar_init(&s_full[i], 1);
      mbar_init(&done[i], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  // columns of no query (128 is no multiple of G) must hold numbers
  for (int i = threadIdx.x; i < kAwSlots * kFaTileBytes / 16; i += kAwThreads)
    if (a.G * per_q < kFaRows) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_shared();
  if (warp == 5) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 4) {
    // ---------------- producer: K once, then Q tiles with their lse ----------------
    if (lane == 0) {
      mbar_arrive_expect_tx(k_full, kFaTileBytes);
      tma_load_3d(sK, &tm_k, 0, key0, slot * a.nkv + kvh, k_full);
      tma_load_3d(sK + kFaHalfBytes, &tm_k, 64, key0, slot * a.nkv + kvh, k_full);
    }
    int issued = 0;
    for (int t = 0; t < n_tiles; ++t, ++issued) {
      const int sl = t & 1;
      // the slot's lse was read and its Q multiplied
      if (t >= kAwSlots && !fa_wait_warp(&done[sl], (t / kAwSlots - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer)) break;
      const int i_first = i0 + t * per_q;
      for (int c = lane; c < kFaRows; c += 32) {
        const int i = i_first + c / a.G;
        float v = INFINITY;  // no query: exp2(s - inf) = 0
        if (c < per_q * a.G && i < a.S) {
          const float e = a.lse[(size_t(b) * a.S + i) * a.nh + kvh * a.G + c % a.G];
          v = e == -INFINITY ? INFINITY : e * 1.4426950408889634f;  // a row without keys: no weight
        }
        s_lse[sl * kFaRows + c] = v;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[sl], per_q * a.G * kFaD * 2);
        tma_load_3d(sQ + sl * kFaTileBytes, &tm_q, 0, kvh * a.G, b * a.S + i_first, &full[sl]);
        tma_load_3d(sQ + sl * kFaTileBytes + kFaHalfBytes, &tm_q, 64, kvh * a.G, b * a.S + i_first, &full[sl]);
      } else {
        mbar_arrive(&full[sl]);
      }
    }
    if (lane == 0) {
      fa_wait_landed(k_full, 0);
      for (int t = max(0, issued - kAwSlots); t < issued; ++t) fa_wait_landed(&full[t & 1], (t / kAwSlots) & 1);
    }
  } else if (warp == 5) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t idesc = make_idesc_bf16(kFaRows, kFaRows);
      const uint32_t k_addr = smem_u32(sK), q_addr = smem_u32(sQ);
      bool ok = fa_wait(k_full, 0, abort_flag, kDevErrWaitTimeoutMma);
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int sl = t & 1;
        if (!fa_wait(&full[sl], (t / kAwSlots) & 1, abort_flag, kDevErrWaitTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kFaD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kFaHalfBytes + (kk & 3) * 32;
          umma_bf16(tmem_base + sl * kFaRows, make_sw128_desc(k_addr + off),
                    make_sw128_desc(q_addr + sl * kFaTileBytes + off), idesc, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[sl]);
      }
      if (!ok) *abort_flag = 1;
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
    // ---------------- sums: thread r owns key key0 + r ----------------
    const int r = warp * 32 + lane;
    const int key = key0 + r;
    const uint32_t s_row = tmem_base + (uint32_t(warp * 32) << 16);
    float total = 0.f;
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int sl = t & 1;
      // s_full follows full: the lse of this slot is in place
      if (!fa_wait_warp(&full[sl], (t / kAwSlots) & 1, abort_flag, kDevErrWaitTimeoutEpilogue) ||
          !fa_wait_warp(&s_full[sl], (t / kAwSlots) & 1, abort_flag, kDevErrWaitTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float sv[kFaRows];
#pragma unroll
      for (int c = 0; c < kFaRows / 32; ++c) tmem_ld_x32(s_row + sl * kFaRows + c * 32, sv + c * 32);
      tmem_ld_wait();
      const float4* le = reinterpret_cast<const float4*>(s_lse + sl * kFaRows);
      const int i_first = i0 + t * per_q;
      float p8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      // a tile that every key of this CTA sees whole
      if (L0 + i_first >= key0 + kFaRows - 1 && i_first + per_q <= a.S && per_q * a.G == kFaRows) {
#pragma unroll
        for (int c = 0; c < kFaRows / 4; ++c) {
          const float4 e = le[c];
          const int j = (c & 1) * 4;
          p8[j] += fa_exp2(sv[4 * c] * a.scale_log2 - e.x);
          p8[j + 1] += fa_exp2(sv[4 * c + 1] * a.scale_log2 - e.y);
          p8[j + 2] += fa_exp2(sv[4 * c + 2] * a.scale_log2 - e.z);
          p8[j + 3] += fa_exp2(sv[4 * c + 3] * a.scale_log2 - e.w);
        }
      } else {
        // columns [c0, c1): the queries of this sequence that see this key
        const int c0 = max(0, key - L0 - i_first) * a.G;
        const int c1 = min(per_q, a.S - i_first) * a.G;
#pragma unroll
        for (int c = 0; c < kFaRows; ++c) {
          const float p = fa_exp2(sv[c] * a.scale_log2 - s_lse[sl * kFaRows + c]);
          p8[c & 7] += c >= c0 && c < c1 ? p : 0.f;
        }
      }
      total += ((p8[0] + p8[1]) + (p8[2] + p8[3])) + ((p8[4] + p8[5]) + (p8[6] + p8[7]));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[sl]);
    }
    if (ok && key < L) w[key] = a.accumulate ? w[key] + total : total;
  }

  __syncthreads();
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

}  // namespace qmoe

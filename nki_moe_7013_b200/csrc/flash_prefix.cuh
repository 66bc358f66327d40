// Attention over a prefix shared by the whole batch, on the 5th-generation
// tensor cores; head_dim 128, bf16 in, fp32 scores / softmax / sums.
//
// flash_prefix_kernel<false> (prefill): S new queries per sequence; query i of
// sequence b attends to the prefix rows 0 .. P-1 and to its own cache rows
// kv_start[b] .. q_start[b] + i.  One CTA takes 256 queries of one (sequence,
// head).  The prefix is stored once: its K and V tiles come from L2 for every
// CTA after the first, and the kernel is bound by the tensor cores and the
// softmax beside them.
//
// flash_prefix_kernel<true> (the prefix part of a decode step): the rows are
// the B * G (sequence, head) rows of one KV head, so a prefix tile is read
// once for up to 256 of them; the keys are cut into parts whose running
// maximum, sum and unnormalised output go to shared_decode_combine_kernel.
//
// One CTA = two tiles of 128 rows (A, B) sharing every K / V tile of 128 keys;
// 320 threads: warps 0-3 softmax of tile A, warps 4-7 of tile B (a thread owns
// a row = a TMEM lane), warp 8 the TMA producer (Q once, then K_0, V_0, K_1,
// ... through three 32 KB slots), warp 9 issues the MMAs in the order
//   S_A(0) S_B(0) | PV_A(0) S_A(1) PV_B(0) S_B(1) | ...
// so one tile's products run while the other tile's softmax does.  S and O
// stay in TMEM (512 columns); P goes to shared memory in bf16.  A row's O is
// rescaled only when its maximum grew by more than 2^8.
//
// Key tiles begin at row 0 of the prefix and at kv_start of the own rows, so
// rows that nobody sees lie only behind a range's end: the prefix's tensor map
// ends at P (zeros behind it), and the own rows' last V tile is zeroed past
// the last query by the producer.  Every wait is bounded, as in
// flash_prefill_kernel.
#pragma once

#include "attn_shared.cuh"
#include "common.cuh"
#include "flash_prefill.cuh"

namespace qmoe {

struct FlashPrefixArgs {
  const int32_t* q_start;
  const int32_t* cache_slot;
  const int32_t* kv_start;
  __nv_bfloat16* out;  // prefill
  float* lse;          // prefill: (B*S, nh) natural log, or null
  float* part_o;       // decode parts, as shared_decode_kernel's
  float* part_ml;
  int S, nh, nkv, max_seq, n_slots, B, n_pairs;
  int P, prefix_z, G, nparts, tiles_per_part;
  float scale_log2;
};

template <bool kPartial>
__global__ void __launch_bounds__(kFaThreads, 1)
    flash_prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_kp,
                        const __grid_constant__ CUtensorMap tm_vp, const FlashPrefixArgs a) {
  extern __shared__ uint8_t fa_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(fa_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sPool = smem + 2 * kFaTileBytes;
  uint8_t* sP = sPool + kFaPool * kFaTileBytes;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kFaTiles * kFaTileBytes);
  uint64_t* q_full = bar + 0;
  uint64_t* full = bar + 1;     // [kFaPool]
  uint64_t* empty = bar + 4;    // [kFaPool]
  uint64_t* s_full = bar + 7;   // [2] per row tile
  uint64_t* p_full = bar + 9;   // [2]
  uint64_t* o_full = bar + 11;  // [2]
  uint64_t* v_tail = bar + 13;
  uint64_t* drain = bar + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kFaBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  griddep_wait();
  if (kPartial) griddep_launch_dependents();

  // prefill: 128 queries of one head per tile; decode: as many whole groups of G heads as fit
  const int rows_per_tile = kPartial ? kFaRows / a.G * a.G : kFaRows;
  int kvh, h = 0, b = 0, q0 = 0, part = 0, pair = 0, slot = 0, L0 = 0, kv0 = 0;
  int t0 = 0, n_pre, n_own = 0, n_keys = 0, nq_a = 0, nq_b = 0;
  const int p_tiles = (a.P + kFaRows - 1) / kFaRows;
  if constexpr (kPartial) {
    pair = blockIdx.x % a.n_pairs;
    const int rest = blockIdx.x / a.n_pairs;
    kvh = rest % a.nkv;
    part = rest / a.nkv;
    t0 = part * a.tiles_per_part;
    n_pre = max(0, min(p_tiles, t0 + a.tiles_per_part) - t0);
    if (n_pre == 0) {  // an empty part: l = 0
      for (int i = threadIdx.x; i < 2 * rows_per_tile; i += blockDim.x) {
        const int row = pair * 2 * rows_per_tile + i;
        if (row < a.B * a.G)
          *reinterpret_cast<float2*>(a.part_ml + ((size_t(row / a.G) * a.nh + kvh * a.G + row % a.G) * a.nparts + part) * 2) =
              make_float2(-INFINITY, 0.f);
      }
      return;
    }
  } else {
    // heaviest tile pairs (the latest queries: most keys) first over all heads
    const int per_pair = a.nh * a.B;
    pair = a.n_pairs - 1 - int(blockIdx.x) / per_pair;
    const int rest = int(blockIdx.x) % per_pair;
    h = rest % a.nh;
    b = rest / a.nh;
    q0 = pair * 2 * kFaRows;
    kvh = h / (a.nh / a.nkv);
    L0 = a.q_start[b];
    slot = a.cache_slot ? a.cache_slot[b] : b;
    if (L0 < 0 || L0 > a.max_seq - a.S || slot < 0 || slot >= a.n_slots) {  // block-uniform
      if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);
      return;
    }
    nq_a = min(kFaRows, a.S - q0);
    nq_b = max(0, min(kFaRows, a.S - q0 - kFaRows));
    n_keys = L0 + q0 + nq_a + nq_b;  // own rows visible to the last query
    kv0 = a.kv_start ? max(0, min(a.kv_start[b], L0 + a.S)) : 0;
    if (kv0 >= n_keys) {  // every query is a padding position: zeros
      const size_t out_ld = size_t(a.nh) * kFaD;
      __nv_bfloat16* o = a.out + (size_t(b) * a.S + q0) * out_ld + size_t(h) * kFaD;
      for (int i = threadIdx.x; i < (nq_a + nq_b) * (kFaD / 8); i += blockDim.x)
        reinterpret_cast<uint4*>(o + size_t(i / (kFaD / 8)) * out_ld)[i % (kFaD / 8)] = make_uint4(0, 0, 0, 0);
      if (a.lse)
        for (int i = threadIdx.x; i < nq_a + nq_b; i += blockDim.x)
          a.lse[(size_t(b) * a.S + q0 + i) * a.nh + h] = -INFINITY;
      return;
    }
    n_pre = p_tiles;
    n_own = (n_keys - kv0 + kFaRows - 1) / kFaRows;
  }
  const int n_tiles = n_pre + n_own;
  const bool tail = n_own > 0 && (n_keys - kv0) % kFaRows != 0;  // the last tile has rows past n_keys

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kFaPool; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 4);
      mbar_init(&o_full[g], 1);
    }
    mbar_init(v_tail, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 8) {
    // ---------------- TMA producer ----------------
    int issued[kFaPool] = {0, 0, 0};
    bool ok = true;
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, 2 * rows_per_tile * kFaD * 2);
      for (int g = 0; g < 2; ++g) {
        const int y = kPartial ? kvh * a.G : h;
        const int z = kPartial ? (pair * 2 + g) * (kFaRows / a.G) : b * a.S + q0 + g * kFaRows;
        tma_load_3d(sQ + g * kFaTileBytes, &tm_q, 0, y, z, q_full);
        tma_load_3d(sQ + g * kFaTileBytes + kFaHalfBytes, &tm_q, 64, y, z, q_full);
      }
      for (int n = 0; n < 2 * n_tiles; ++n) {  // K_i = item 2i, V_i = item 2i + 1
        const int sl = n % kFaPool, u = n / kFaPool;
        if (n >= kFaPool && !fa_wait(&empty[sl], (u - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer)) {
          ok = false;
          break;
        }
        const int i = n >> 1;
        const bool pre = i < n_pre;
        const int key0 = pre ? (t0 + i) * kFaRows : kv0 + (i - n_pre) * kFaRows;
        const int z = pre ? a.prefix_z + kvh : slot * a.nkv + kvh;
        const CUtensorMap* tm = pre ? ((n & 1) ? &tm_vp : &tm_kp) : ((n & 1) ? &tm_v : &tm_k);
        uint8_t* dst = sPool + sl * kFaTileBytes;
        mbar_arrive_expect_tx(&full[sl], kFaTileBytes);
        tma_load_3d(dst, tm, 0, key0, z, &full[sl]);
        tma_load_3d(dst + kFaHalfBytes, tm, 64, key0, z, &full[sl]);
        ++issued[sl];
      }
    }
    ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;
    if (ok && tail) {
      // zero the last V tile's rows past the last visible key
      const int n = 2 * n_tiles - 1;
      const int sl = n % kFaPool;
      if (fa_wait_warp(&full[sl], (n / kFaPool) & 1, abort_flag, kDevErrWaitTimeoutProducer)) {
        const int first = (n_keys - kv0) % kFaRows;
        uint8_t* vt = sPool + sl * kFaTileBytes;
        for (int i = first * 8 + lane; i < kFaRows * 8; i += 32) {  // 16-byte chunks of whole rows
          const int r = i >> 3, c = i & 7;
          *reinterpret_cast<uint4*>(vt + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(vt + kFaHalfBytes + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_tail);
      }
    }
    if (lane == 0) {
      // loads still in flight land before the CTA can exit
      fa_wait_landed(q_full, 0);
      for (int sl = 0; sl < kFaPool; ++sl)
        if (issued[sl]) fa_wait_landed(&full[sl], (issued[sl] - 1) & 1);
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      const uint32_t idesc_s = make_idesc_bf16(kFaRows, kFaRows);
      const uint32_t idesc_o = make_idesc_bf16(kFaRows, kFaD) | (1u << 16);  // B (V) MN-major
      const uint64_t q_desc = make_sw128_desc(smem_u32(sQ)), p_desc = make_sw128_desc(smem_u32(sP));
      const uint64_t k_desc = make_sw128_desc(smem_u32(sPool));
      const uint64_t v_desc = make_sw128_desc_mn(smem_u32(sPool), kFaHalfBytes, 1024);
      constexpr uint32_t kTile = kFaTileBytes >> 4;
      auto item_full = [&](int n) {
        return fa_wait(&full[n % kFaPool], (n / kFaPool) & 1, abort_flag, kDevErrWaitTimeoutMma);
      };
      auto issue_s = [&](int g, int i) {  // S_g = Q_g K_i^T
        umma_bf16_k128(tmem_base + g * kFaRows, q_desc + g * kTile, k_desc + ((2 * i) % kFaPool) * kTile, idesc_s);
        umma_commit(&s_full[g]);
      };
      auto issue_pv = [&](int g, int i) {  // O_g (+)= P_g V_i
        const uint64_t vd = v_desc + ((2 * i + 1) % kFaPool) * kTile, pd = p_desc + g * kTile;
        const uint32_t d = tmem_base + 2 * kFaRows + g * kFaD;
#pragma unroll
        for (int kk = 0; kk < kFaRows / 16; ++kk)  // 16 keys per MMA
          umma_bf16(d, pd + (((kk >> 2) * kFaHalfBytes + (kk & 3) * 32) >> 4), vd + ((kk * 16 * 128) >> 4), idesc_o,
                    (i > 0 || kk > 0) ? 1u : 0u);
      };
      bool ok = fa_wait(q_full, 0, abort_flag, kDevErrWaitTimeoutMma) && item_full(0);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        issue_s(1, 0);
        umma_commit(&empty[0]);  // K_0 read by both
      }
      for (int i = 0; ok && i < n_tiles; ++i) {
        const int nv = 2 * i + 1, nk = 2 * i + 2;
        const bool last = i == n_tiles - 1;
        // PV_A(i), then S_A(i+1)
        if (!fa_wait(&p_full[0], i & 1, abort_flag, kDevErrWaitTimeoutMma) || !item_full(nv) ||
            (tail && last && !fa_wait(v_tail, 0, abort_flag, kDevErrWaitTimeoutMma))) {
          ok = false;
          break;
        }
        tc_fence_after();
        issue_pv(0, i);
        if (last) umma_commit(&o_full[0]);
        if (!last) {
          if (!item_full(nk)) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_s(0, i + 1);
        }
        // PV_B(i), then S_B(i+1)
        if (!fa_wait(&p_full[1], i & 1, abort_flag, kDevErrWaitTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        issue_pv(1, i);
        umma_commit(&empty[nv % kFaPool]);  // V_i read by both
        if (last) umma_commit(&o_full[1]);
        if (!last) {
          issue_s(1, i + 1);
          umma_commit(&empty[nk % kFaPool]);  // K_{i+1} read by both
        }
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
    // ---------------- softmax: warps 0-3 tile A, warps 4-7 tile B ----------------
    const int g = warp >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const int qpos = L0 + q0 + g * kFaRows + r;  // prefill: the query's own row
    const bool dead = !kPartial && qpos < kv0;   // a padding query sees nothing
    const uint32_t t_lane = uint32_t(quad * 32) << 16;
    const uint32_t s_col = tmem_base + t_lane + g * kFaRows;
    const uint32_t o_col = tmem_base + t_lane + 2 * kFaRows + g * kFaD;
    const uint32_t p_row = smem_u32(sP + g * kFaTileBytes) + r * 128;
    const int sw = r & 7;
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      if (!fa_wait_warp(&s_full[g], i & 1, abort_flag, kDevErrWaitTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // this row sees the tile's first `vis` keys
      int vis = i < n_pre ? a.P - (t0 + i) * kFaRows : qpos - (kv0 + (i - n_pre) * kFaRows) + 1;
      if (dead) vis = 0;
      float sv[kFaRows];
#pragma unroll
      for (int c = 0; c < kFaRows / 32; ++c) tmem_ld_x32(s_col + c * 32, sv + c * 32);
      tmem_ld_wait();
      if (__any_sync(0xFFFFFFFFu, vis < kFaRows)) {
#pragma unroll
        for (int e = 0; e < kFaRows; ++e)
          if (e >= vis) sv[e] = -INFINITY;
      }
      // row max as 8 independent chains
      float mx8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) mx8[j] = sv[j];
#pragma unroll
      for (int e = 8; e < kFaRows; ++e) mx8[e & 7] = fmaxf(mx8[e & 7], sv[e]);
      const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                             fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
      const float m_new = fmaxf(m_used, mx * a.scale_log2);
      float alpha = 1.f;
      if (m_new > m_used + kFaRescaleLog2) {
        alpha = m_used == -INFINITY ? 0.f : exp2f(m_used - m_new);
        m_used = m_new;
      }
      const float mb = m_used == -INFINITY ? 0.f : m_used;
      // P = exp2(S*scale - m) as bf16 into the swizzled P tile
      float ls8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kFaRows / 16; ++c) {
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = fa_exp2(sv[c * 16 + e] * a.scale_log2 - mb);
          const float p1 = fa_exp2(sv[c * 16 + e + 1] * a.scale_log2 - mb);
          ls8[e >> 1] += p0 + p1;
          pk[e >> 1] = pack_bf16x2(p0, p1);
        }
        const uint32_t base = p_row + (c >> 2) * kFaHalfBytes;
        const int ch = (c & 3) * 2;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + ((ch ^ sw) << 4)), "r"(pk[0]),
                     "r"(pk[1]), "r"(pk[2]), "r"(pk[3])
                     : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + (((ch + 1) ^ sw) << 4)), "r"(pk[4]),
                     "r"(pk[5]), "r"(pk[6]), "r"(pk[7])
                     : "memory");
      }
      const float lsum = ((ls8[0] + ls8[1]) + (ls8[2] + ls8[3])) + ((ls8[4] + ls8[5]) + (ls8[6] + ls8[7]));
      l = l * alpha + lsum;
      // a grown row max: rescale this group's O rows (PV of the earlier tiles
      // is complete -- it was issued before S of this tile)
      if (i > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.f)) {
#pragma unroll
        for (int c = 0; c < kFaD / 32; ++c) {
          float ov[32];
          tmem_ld_x32(o_col + c * 32, ov);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] *= alpha;
          tmem_st_x32(o_col + c * 32, ov);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[g]);
    }
    if (ok && fa_wait_warp(&o_full[g], 0, abort_flag, kDevErrWaitTimeoutEpilogue)) {
      tc_fence_after();
      if constexpr (kPartial) {
        const int row = (pair * 2 + g) * rows_per_tile + r;
        const bool mine = r < rows_per_tile && row < a.B * a.G;
        const size_t pidx = (size_t(row / a.G) * a.nh + kvh * a.G + row % a.G) * a.nparts + part;
        if (mine) *reinterpret_cast<float2*>(a.part_ml + pidx * 2) = make_float2(m_used, l);
        float4* dst = reinterpret_cast<float4*>(a.part_o + pidx * kFaD);
#pragma unroll
        for (int c = 0; c < kFaD / 32; ++c) {
          float ov[32];
          tmem_ld_x32(o_col + c * 32, ov);
          tmem_ld_wait();
          if (mine) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              dst[c * 8 + q] = make_float4(ov[q * 4], ov[q * 4 + 1], ov[q * 4 + 2], ov[q * 4 + 3]);
          }
        }
      } else {
        const bool mine = r < (g ? nq_b : nq_a);
        const size_t row = size_t(b) * a.S + q0 + g * kFaRows + r;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (mine && a.lse)
          a.lse[row * a.nh + h] = l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.6931471805599453f;
        uint4* dst = reinterpret_cast<uint4*>(a.out + row * (size_t(a.nh) * kFaD) + size_t(h) * kFaD);
#pragma unroll
        for (int c = 0; c < kFaD / 32; ++c) {
          float ov[32];
          tmem_ld_x32(o_col + c * 32, ov);
          tmem_ld_wait();
          if (mine) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              dst[c * 4 + q] = make_uint4(pack_bf16x2(ov[q * 8] * inv, ov[q * 8 + 1] * inv),
                                          pack_bf16x2(ov[q * 8 + 2] * inv, ov[q * 8 + 3] * inv),
                                          pack_bf16x2(ov[q * 8 + 4] * inv, ov[q * 8 + 5] * inv),
                                          pack_bf16x2(ov[q * 8 + 6] * inv, ov[q * 8 + 7] * inv));
          }
        }
      }
      tc_fence_before();
    }
  }

  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace qmoe

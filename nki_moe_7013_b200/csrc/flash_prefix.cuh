// Attention over a prefix shared by the whole batch, on the 5th-generation
// tensor cores; head_dim 128, bf16 in, fp32 scores / softmax / sums.
//
// Prefill (kPartial false): S new queries per sequence; query i of sequence b
// attends to the prefix rows 0 .. P-1 and to its own cache rows kv_start[b] ..
// q_start[b] + i.  The rows of a tile are 128 / G positions times the G query
// heads of one KV head, so a K / V tile serves the whole group, short prompts
// fill their tiles (37 queries of 8 heads are 296 rows) and the causal
// diagonal crosses few of them.
//
// The prefix part of a decode step (kPartial true): the rows are the B * G
// (sequence, head) rows of one KV head, so the prefix is read once for 128 of
// them (with kSplit) or 256; the keys are cut into parts whose running maximum,
// sum and unnormalised output go to shared_decode_combine_kernel.  128
// sequences on 16,384 rows: 22 steps on 96 SMs, 42 us, the tensor pipe 52 %
// busy, the own rows' kernel on the other SMs beside it.
//
// One CTA = two softmax groups A and B; 320 threads: warps 0-3 and 4-7 softmax
// (a thread owns a row = a TMEM lane), warp 8 the TMA producer (Q once, then K
// and V tiles of 128 keys through 32 KB slots), warp 9 issues the MMAs so that
// one group's products run while the other group's softmax does:
//   S_A(0) S_B(0) | PV_A(0) S_A(1) | PV_B(0) S_B(1) | PV_A(1) S_A(2) | ...
// Without kSplit A and B are two row tiles sharing every K / V tile; with it
// they are the even and the odd key tiles of one row tile, joined at the end
// (each thread reads both groups' O of its TMEM lane): half the steps, for twice
// the CTAs, where the row tiles are too few to fill the SMs, or half the parts
// of a decode step.  S and O stay in TMEM (512 columns); P goes to
// shared memory in bf16, as the tensor core takes it beside a bf16 V (half a
// step, 2^-8 of each probability; their sum is taken before, in fp32).  A row's
// O is rescaled only when its maximum grew by
// more than 2^8.
//
// Bound by the softmax beside the tensor core: 4 sequences of 2,048 queries
// behind 4,096 rows take 0.64 ms when repeated (1.07 PFLOP/s, 0.64 of the
// measured bf16 burst and 0.77 of the sustained rate; the card is at its power
// limit, at 1,732 MHz), 0.61 to 0.63 in short bursts and up to 0.69 after other
// work; in bursts 0.52 ms without the exponentials, 0.61 without the second
// product.  The head-packed row tiles took 8 short prompts of 37 queries behind
// 1,001 rows from 53 to 17 us.
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

constexpr int kFpBarriers = 18;
constexpr int kFpSmemBytes = kFaTiles * kFaTileBytes + 1024 + kFpBarriers * 8 + 16;

// Two columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st_x2(uint32_t taddr, float a, float b) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(taddr), "r"(__float_as_uint(a)),
               "r"(__float_as_uint(b))
               : "memory");
}
__device__ __forceinline__ void tmem_ld_x2(uint32_t taddr, float& a, float& b) {
  uint32_t x, y;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x), "+r"(y) : : "memory");
  a = __uint_as_float(x);
  b = __uint_as_float(y);
}

struct FlashPrefixArgs {
  const int32_t* q_start;
  const int32_t* cache_slot;
  const int32_t* kv_start;
  __nv_bfloat16* out;  // prefill
  float* lse;          // prefill: (B*S, nh) natural log, or null
  float* part_o;       // decode parts, as shared_decode_kernel's
  float* part_ml;
  int S, nh, nkv, max_seq, n_slots, B, n_blocks;  // n_blocks: row blocks (one or two tiles) of a CTA column
  int P, prefix_z, G, nparts, tiles_per_part;
  float scale_log2;
};

template <bool kPartial, bool kSplit>
__global__ void __launch_bounds__(kFaThreads, 1)
    flash_prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_kp,
                        const __grid_constant__ CUtensorMap tm_vp, const FlashPrefixArgs a) {
  constexpr int kQTiles = kSplit ? 1 : 2;
  constexpr int kPool = kFaTiles - 2 - kQTiles;  // K / V slots: 4 or 3
  extern __shared__ uint8_t fa_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(fa_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sPool = smem + kQTiles * kFaTileBytes;
  uint8_t* sP = sPool + kPool * kFaTileBytes;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kFaTiles * kFaTileBytes);
  uint64_t* q_full = bar + 0;
  uint64_t* full = bar + 1;     // [kPool]
  uint64_t* empty = bar + 5;    // [kPool]
  uint64_t* s_full = bar + 9;   // [2] per group
  uint64_t* p_full = bar + 11;  // [2]
  uint64_t* o_full = bar + 13;  // [2]
  uint64_t* v_tail = bar + 15;
  uint64_t* drain = bar + 16;
  uint64_t* ml_ready = bar + 17;  // kSplit: both groups' maxima and sums
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kFpBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kp);
    prefetch_tmap(&tm_vp);
  }
  griddep_wait();
  if (kPartial) griddep_launch_dependents();

  const int per_q = kFaRows / a.G;       // positions (prefill) or sequences (decode) per row tile
  const int tile_rows = per_q * a.G;
  int kvh, b = 0, q0 = 0, part = 0, slot = 0, L0 = 0, kv0 = 0;
  int t0 = 0, n_pre, n_own = 0, n_keys = 0;
  const int p_tiles = (a.P + kFaRows - 1) / kFaRows;
  if constexpr (kPartial) {
    q0 = int(blockIdx.x) % a.n_blocks * kQTiles * per_q;  // first sequence
    const int rest = blockIdx.x / a.n_blocks;
    kvh = rest % a.nkv;
    part = rest / a.nkv;
    t0 = part * a.tiles_per_part;
    n_pre = min(p_tiles, t0 + a.tiles_per_part) - t0;  // at least 1
  } else {
    // heaviest blocks (the latest queries: most keys) first over all heads
    const int heads = a.nkv * a.B;
    q0 = (a.n_blocks - 1 - int(blockIdx.x) / heads) * kQTiles * per_q;
    kvh = int(blockIdx.x) % heads % a.nkv;
    b = int(blockIdx.x) % heads / a.nkv;
    L0 = a.q_start[b];
    slot = a.cache_slot ? a.cache_slot[b] : b;
    if (L0 < 0 || L0 > a.max_seq - a.S || slot < 0 || slot >= a.n_slots) {  // block-uniform
      if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);
      return;
    }
    const int nq = min(a.S - q0, kQTiles * per_q);
    n_keys = L0 + q0 + nq;  // own rows visible to the last query
    kv0 = a.kv_start ? max(0, min(a.kv_start[b], L0 + a.S)) : 0;
    if (kv0 >= n_keys) {  // every query is a padding position: zeros
      for (int i = threadIdx.x; i < nq * a.G * (kFaD / 8); i += blockDim.x) {
        const int row = i / (kFaD / 8);
        const size_t at = (size_t(b) * a.S + q0 + row / a.G) * a.nh + kvh * a.G + row % a.G;
        reinterpret_cast<uint4*>(a.out + at * kFaD)[i % (kFaD / 8)] = make_uint4(0, 0, 0, 0);
        if (a.lse && i % (kFaD / 8) == 0) a.lse[at] = -INFINITY;
      }
      return;
    }
    n_pre = p_tiles;
    n_own = (n_keys - kv0 + kFaRows - 1) / kFaRows;
  }
  const int n_tiles = n_pre + n_own;
  const bool tail = n_own > 0 && (n_keys - kv0) % kFaRows != 0;  // the last tile has rows past n_keys
  // Slot items in the order of their use.  Two row tiles: K_0 V_0 K_1 V_1 ...;
  // split: K_0 K_1 V_0 K_2 V_1 K_3 ... (K_n_tiles, the one before the last
  // item, does not exist).
  auto k_item = [](int j) { return kSplit ? (j == 0 ? 0 : 2 * j - 1) : 2 * j; };
  auto v_item = [](int j) { return kSplit ? 2 * j + 2 : 2 * j + 1; };
  const int n_items = v_item(n_tiles - 1) + 1;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kPool; ++i) {
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
    mbar_init(ml_ready, 8);
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
    int issued[kPool] = {};
    bool ok = true;
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, kQTiles * tile_rows * kFaD * 2);
      for (int g = 0; g < kQTiles; ++g) {
        const int y = kvh * a.G, z = b * a.S + q0 + g * per_q;
        tma_load_3d(sQ + g * kFaTileBytes, &tm_q, 0, y, z, q_full);
        tma_load_3d(sQ + g * kFaTileBytes + kFaHalfBytes, &tm_q, 64, y, z, q_full);
      }
      for (int n = 0; n < n_items; ++n) {
        const bool is_v = kSplit ? n > 0 && n % 2 == 0 : n % 2 == 1;
        const int j = kSplit ? (is_v ? n / 2 - 1 : (n + 1) / 2) : n / 2;
        if (j >= n_tiles) continue;
        const int sl = n % kPool, u = n / kPool;
        if (n >= kPool && !fa_wait(&empty[sl], (u - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer)) {
          ok = false;
          break;
        }
        const bool pre = j < n_pre;
        const int key0 = pre ? (t0 + j) * kFaRows : kv0 + (j - n_pre) * kFaRows;
        const int z = pre ? a.prefix_z + kvh : slot * a.nkv + kvh;
        const CUtensorMap* tm = pre ? (is_v ? &tm_vp : &tm_kp) : (is_v ? &tm_v : &tm_k);
        uint8_t* dst = sPool + sl * kFaTileBytes;
        mbar_arrive_expect_tx(&full[sl], kFaTileBytes);
        tma_load_3d(dst, tm, 0, key0, z, &full[sl]);
        tma_load_3d(dst + kFaHalfBytes, tm, 64, key0, z, &full[sl]);
#pragma unroll
        for (int s = 0; s < kPool; ++s) issued[s] += s == sl;
      }
    }
    ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;
    if (ok && tail) {
      // zero the last V tile's rows past the last visible key
      const int n = n_items - 1;
      const int sl = n % kPool;
      if (fa_wait_warp(&full[sl], (n / kPool) & 1, abort_flag, kDevErrWaitTimeoutProducer)) {
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
#pragma unroll
      for (int sl = 0; sl < kPool; ++sl)
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
        return fa_wait(&full[n % kPool], (n / kPool) & 1, abort_flag, kDevErrWaitTimeoutMma);
      };
      auto issue_s = [&](int g, int j) {  // S_g = Q_g K_j^T
        umma_bf16_k128(tmem_base + g * kFaRows, q_desc + (kSplit ? 0 : g) * kTile, k_desc + k_item(j) % kPool * kTile,
                       idesc_s);
        umma_commit(&s_full[g]);
      };
      auto issue_pv = [&](int g, int j, bool add) {  // O_g (+)= P_g V_j
        const uint64_t vd = v_desc + v_item(j) % kPool * kTile, pd = p_desc + g * kTile;
        const uint32_t d = tmem_base + 2 * kFaRows + g * kFaD;
#pragma unroll
        for (int kk = 0; kk < kFaRows / 16; ++kk)  // 16 keys per MMA
          umma_bf16(d, pd + (((kk >> 2) * kFaHalfBytes + (kk & 3) * 32) >> 4), vd + ((kk * 16 * 128) >> 4), idesc_o,
                    add || kk > 0 ? 1u : 0u);
      };
      bool ok = fa_wait(q_full, 0, abort_flag, kDevErrWaitTimeoutMma) && item_full(0);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        if (!kSplit) issue_s(1, 0);
        umma_commit(&empty[0]);
        if (kSplit && n_tiles > 1) {
          ok = item_full(1);
          if (ok) {
            tc_fence_after();
            issue_s(1, 1);
            umma_commit(&empty[1]);
          }
        }
      }
      constexpr int kStep = kSplit ? 2 : 1;  // a group's tiles: g, g + 2, ... or all
      for (int i = 0; ok && i * kStep < n_tiles; ++i) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int j = kSplit ? 2 * i + g : i;
          if (!ok || j >= n_tiles) continue;
          const bool more = j + kStep < n_tiles;
          const int nv = v_item(j), nk = k_item(j + kStep);
          ok = fa_wait(&p_full[g], i & 1, abort_flag, kDevErrWaitTimeoutMma) && item_full(nv) &&
               (!(tail && j == n_tiles - 1) || fa_wait(v_tail, 0, abort_flag, kDevErrWaitTimeoutMma));
          if (!ok) continue;
          tc_fence_after();
          issue_pv(g, j, i > 0);
          if (kSplit || g == 1) umma_commit(&empty[nv % kPool]);  // V_j read (by both)
          if (!more) {
            umma_commit(&o_full[g]);
            continue;
          }
          ok = item_full(nk);
          if (!ok) continue;
          tc_fence_after();
          issue_s(g, j + kStep);
          if (kSplit || g == 1) umma_commit(&empty[nk % kPool]);
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
    // ---------------- softmax: warps 0-3 group A, warps 4-7 group B ----------------
    const int g = warp >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const int row_q = q0 + (kSplit ? 0 : g * per_q) + r / a.G;  // the row's query (prefill) or sequence
    const int row_h = kvh * a.G + r % a.G;
    const int qpos = L0 + row_q;
    const bool dead = !kPartial && qpos < kv0;  // a padding query sees nothing
    const uint32_t t_lane = uint32_t(quad * 32) << 16;
    const uint32_t s_col = tmem_base + t_lane + g * kFaRows;
    const uint32_t o_col = tmem_base + t_lane + 2 * kFaRows + g * kFaD;
    const uint32_t p_row = smem_u32(sP + g * kFaTileBytes) + r * 128;
    const int sw = r & 7;
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; (kSplit ? 2 * i + g : i) < n_tiles; ++i) {
      const int j = kSplit ? 2 * i + g : i;
      if (!fa_wait_warp(&s_full[g], i & 1, abort_flag, kDevErrWaitTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // this row sees the tile's first `vis` keys
      int vis = j < n_pre ? a.P - (t0 + j) * kFaRows : qpos - (kv0 + (j - n_pre) * kFaRows) + 1;
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
      for (int e = 0; e < 8; ++e) mx8[e] = sv[e];
#pragma unroll
      for (int e = 8; e < kFaRows - 8; e += 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) mx8[k] = max3(mx8[k], sv[e + k], sv[e + 8 + k]);
#pragma unroll
      for (int k = 0; k < 8; ++k) mx8[k] = fmaxf(mx8[k], sv[kFaRows - 8 + k]);
      const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                             fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
      const float m_new = fmaxf(m_used, mx * a.scale_log2);
      float alpha = 1.f;
      if (m_new > m_used + kFaRescaleLog2) {
        alpha = m_used == -INFINITY ? 0.f : exp2f(m_used - m_new);
        m_used = m_new;
      }
      const float mb = m_used == -INFINITY ? 0.f : m_used;
      // P = exp2(S*scale - m) as bf16 into the swizzled P tile, its sum in fp32.
      // The softmax is bound by its instructions (without the exponentials a
      // step takes 17 % less, with a fifth of them as polynomials 3 % more), so
      // the arithmetic runs two values an instruction: 2 % of the long prefill.
      const f32x2 scale2 = pack2(a.scale_log2, a.scale_log2), minus_m = pack2(-mb, -mb);
      f32x2 sum2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kFaRows / 16; ++c) {
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float x0, x1;
          unpack2(fma2(pack2(sv[c * 16 + e], sv[c * 16 + e + 1]), scale2, minus_m), x0, x1);
          const float p0 = fa_exp2(x0), p1 = fa_exp2(x1);
          sum2[(e >> 1) & 3] = add2(sum2[(e >> 1) & 3], pack2(p0, p1));
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
      float even, odd;
      unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), even, odd);
      l = l * alpha + (even + odd);
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
    // Epilogue.  Split: both groups rescale to the larger maximum, exchanging
    // (m, l) through the group's own, now idle score columns; group g writes
    // dims 64 g .. 64 g + 63 of O_A + O_B.
    float m_row = m_used, l_row = l, f[2] = {1.f, 1.f};
    const bool two = !kSplit || n_tiles > 1;  // group B had a tile
    if constexpr (kSplit) {
      tmem_st_x2(s_col, m_used, l);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ml_ready);
      ok = ok && fa_wait_warp(ml_ready, 0, abort_flag, kDevErrWaitTimeoutEpilogue) &&
           fa_wait_warp(&o_full[0], 0, abort_flag, kDevErrWaitTimeoutEpilogue) &&
           (!two || fa_wait_warp(&o_full[1], 0, abort_flag, kDevErrWaitTimeoutEpilogue));
      if (ok) {
        tc_fence_after();
        float mo, lo;
        tmem_ld_x2(tmem_base + t_lane + (g ^ 1) * kFaRows, mo, lo);
        m_row = fmaxf(m_used, mo);
        const float base = m_row == -INFINITY ? 0.f : m_row;
        f[g] = exp2f(m_used - base);
        f[g ^ 1] = exp2f(mo - base);
        l_row = l * f[g] + lo * f[g ^ 1];
      }
    } else {
      ok = ok && fa_wait_warp(&o_full[g], 0, abort_flag, kDevErrWaitTimeoutEpilogue);
      tc_fence_after();
    }
    if (ok) {
      const bool mine = r < tile_rows && row_q < (kPartial ? a.B : a.S);
      const size_t row = (kPartial ? size_t(row_q) : size_t(b) * a.S + row_q) * a.nh + row_h;
      const float inv = kPartial ? 1.f : l_row == 0.f ? 0.f : 1.f / l_row;
      if (mine && (!kSplit || g == 0)) {
        if (kPartial)
          *reinterpret_cast<float2*>(a.part_ml + (row * a.nparts + part) * 2) = make_float2(m_row, l_row);
        else if (a.lse)
          a.lse[row] = l_row == 0.f ? -INFINITY : (m_row + log2f(l_row)) * 0.6931471805599453f;
      }
      const uint32_t o_a = tmem_base + t_lane + 2 * kFaRows;
#pragma unroll
      for (int i = 0; i < (kSplit ? 2 : 4); ++i) {
        const int c = kSplit ? 2 * g + i : i;
        float ov[32];
        if constexpr (kSplit) {
          float ob[32];
          tmem_ld_x32(o_a + c * 32, ov);
          if (two) tmem_ld_x32(o_a + kFaD + c * 32, ob);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = ov[e] * f[0] + (two ? ob[e] * f[1] : 0.f);
        } else {
          tmem_ld_x32(o_col + c * 32, ov);
          tmem_ld_wait();
        }
        if constexpr (kPartial) {
          // through this warp's 4 KB of the group's P tile, so that a store
          // covers whole 128-byte lines of four rows
          const uint32_t stage = smem_u32(sP + g * kFaTileBytes) + quad * 4096;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((q ^ (lane & 7)) << 4)),
                         "f"(ov[q * 4]), "f"(ov[q * 4 + 1]), "f"(ov[q * 4 + 2]), "f"(ov[q * 4 + 3])
                         : "memory");
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int rr = q * 4 + (lane >> 3), ch = lane & 7;  // row of the warp, 16-byte chunk
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(stage + rr * 128 + ((ch ^ (rr & 7)) << 4)));
            const int tr = quad * 32 + rr, rq = q0 + (kSplit ? 0 : g * per_q) + tr / a.G;
            if (tr < tile_rows && rq < a.B) {
              const size_t at = size_t(rq) * a.nh + kvh * a.G + tr % a.G;
              *(reinterpret_cast<float4*>(a.part_o + (at * a.nparts + part) * kFaD) + c * 8 + ch) = v;
            }
          }
          __syncwarp();
        } else if (mine) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + row * kFaD) + c * 4;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            dst[q] = make_uint4(pack_bf16x2(ov[q * 8] * inv, ov[q * 8 + 1] * inv),
                                pack_bf16x2(ov[q * 8 + 2] * inv, ov[q * 8 + 3] * inv),
                                pack_bf16x2(ov[q * 8 + 4] * inv, ov[q * 8 + 5] * inv),
                                pack_bf16x2(ov[q * 8 + 6] * inv, ov[q * 8 + 7] * inv));
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

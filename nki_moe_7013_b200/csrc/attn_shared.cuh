// Decode attention over a prefix that the whole batch shares, and decode
// attention that keeps every cache row's accumulated attention weight.
// head_dim 128, bf16 in, fp32 scores, softmax and sums; 1 to 16 query heads
// per KV head.
//
//   out_bh = softmax(c q_bh [Kp; K_b]^T) [Vp; V_b]
//   weights[slot, g, j] (+)= sum over the heads h of group g of p_bh[j]
//
// over the prefix rows 0 .. P-1 (one slot of a prefix cache, the same for all
// sequences) and the sequence's own rows kv_start[b] .. kv_len[b]-1.  Either
// part may be empty; a row with neither gets zeros and no weight.
//
// The keys are cut into parts; a part yields a row's running maximum m (in
// log2 units), its sum l of exp2(s - m) and its unnormalised output, which
// shared_decode_combine_kernel joins:  M = max m,  out = sum_i 2^(m_i - M) o_i
// / sum_i 2^(m_i - M) l_i.  The joined M and l also turn the scores of the
// own rows, kept in fp32 by the first kernel, into attention weights.  Own
// rows are cut by the batch's total, so that every part of a ragged batch holds
// about as many rows -- while the sequences are too few to fill the SMs; more of
// them are one part each, however uneven.  Short calls run as one CTA per
// (sequence, KV head) over prefix and own rows, without a second kernel (5.2 us
// instead of 6.7 for two sequences of 5 rows behind 129).
//
// Bound by HBM: 8 sequences of 1,400 to 4,096 rows (45 MB) stream at the copy
// rate once the pipeline runs; 3.5 us before it (lengths, the cut, the first
// tile's latency), 1.3 us of merging the warps and the joining kernel remain on
// top: 21 us a call with weights, against 7 us of bytes.
//
// Scores, running maxima, sums and outputs are fp32.  Probabilities enter the
// second product as bf16, the type that its other operand, V, has on the tensor
// core; their sum l is taken before that rounding (at most 2^-8 of each, of
// either sign, so most of it averages out over the keys).  exp2 is the
// approximate instruction where a key costs one; the joins use exp2f.  Against
// 64 bits the outputs are off by 0.0017 to 0.0022 of their norm, of which their
// own rounding to bf16 is 0.0017.
#pragma once

#include "attention.cuh"
#include "common.cuh"
#include "flash_prefill.cuh"

namespace qmoe {

constexpr int kSdKeys = 64;                           // keys per stage
constexpr int kSdHalfBytes = kSdKeys * 128;           // 64 keys x 64 dims
constexpr int kSdTileBytes = 2 * kSdHalfBytes;        // one K or V tile: 16 KB
constexpr int kSdStageBytes = 2 * kSdTileBytes;       // K and V
constexpr int kSdStages = 3;
constexpr int kSdThreads = 160;                       // 4 MMA warps, 1 producer warp
constexpr int kSdRedStride = kAttnD + 4;
constexpr int kSdSmemBytes = kSdStages * kSdStageBytes + 1024 + 128;
constexpr int kSdMaxGroup = 16;                       // rows of one MMA tile
constexpr int kSdCombineRows = 256;                   // cache rows per weight block
static_assert(4 * 16 * kSdRedStride * 4 <= kSdStages * kSdStageBytes, "the warps are merged in the stages' memory");

struct SharedDecodeArgs {
  const __nv_bfloat16* q;
  const int32_t* kv_len;
  const int32_t* cache_slot;
  const int32_t* kv_start;
  float* pre_o;     // prefix parts [B*nh][psplits][128]
  float* pre_ml;    // [B*nh][psplits][2]
  float* own_o;     // own parts [own_cap][nh][128]
  float* own_ml;    // [own_cap][nh][2]
  int2* plan;       // [B] a sequence's first own part and their number
  float* scores;    // [B*nkv][score_rows][G] log2-scaled scores of the own rows, or null
  float* weights;   // (n_slots, nkv, max_seq) or null
  __nv_bfloat16* out;
  int B, nh, nkv, G, max_seq, max_len, n_slots, accumulate;
  int P, prefix_z, psplits, pchunk, row_tiles, n_prefix_units;
  int own_slots;    // parts per KV head that the own rows are cut into (at least one per sequence); 0: one per sequence
  int n_own_units, score_rows, n_out_blocks, row_blocks;
  int direct;       // one unit per (sequence, KV head), nothing to join
  int wide;         // many parts: a block joins one row, not a warp
  int overlaps;     // the kernel before it (the tcgen05 prefix part) may still run
  float scale_log2;
};

// The sequence's own visible rows [lo, hi): false (device error 4) when its
// length or slot lies outside the cache.
__device__ __forceinline__ bool own_range(const int32_t* kv_len, const int32_t* cache_slot, const int32_t* kv_start,
                                          int b, int max_len, int n_slots, int& slot, int& lo, int& hi) {
  slot = cache_slot ? cache_slot[b] : b;
  hi = kv_len[b];
  const bool ok = hi >= 0 && hi <= max_len && slot >= 0 && slot < n_slots;
  if (!ok) {
    slot = 0;
    hi = 0;
  }
  lo = kv_start ? max(0, min(kv_start[b], hi)) : 0;
  return ok;
}

__device__ __forceinline__ int own_rows(const SharedDecodeArgs& a, int b) {
  if (b >= a.B) return 0;
  int slot, lo, hi;
  own_range(a.kv_len, a.cache_slot, a.kv_start, b, a.max_len, a.n_slots, slot, lo, hi);
  return hi - lo;
}
// How the own rows of a batch are cut, found by every warp for itself: `chunk`
// rows per part, the sequence that part `part` belongs to (B when there is no
// such part), and the sequence's first part and their number.
struct OwnParts {
  int b, chunk, first, count;
};
__device__ __forceinline__ OwnParts own_parts(const SharedDecodeArgs& a, int part, int lane) {
  const int first_rows = own_rows(a, lane);  // of the first 32 sequences: read once
  long long total = first_rows;
  for (int i = lane + 32; i < a.B; i += 32) total += own_rows(a, i);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
  OwnParts p;
  const uint32_t rows = uint32_t(min(total, 0x7FFFFFFFll));  // (more are cut as if they were 2^31)
  const int even = int(min((rows + a.own_slots - 1) / uint32_t(a.own_slots), uint32_t(a.max_len)));
  p.chunk = max(2 * kSdKeys, (even + kSdKeys - 1) / kSdKeys * kSdKeys);
  if (total > 0x7FFFFFFFll) p.chunk = max(p.chunk, (a.max_len + kSdKeys - 1) / kSdKeys * kSdKeys);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int n = ((b0 == 0 ? first_rows : own_rows(a, b0 + lane)) + p.chunk - 1) / p.chunk;
    int incl = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, incl, off);
      if (lane >= off) incl += t;
    }
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + incl > part);
    if (hit) {
      const int src = __ffs(hit) - 1;
      p.b = b0 + src;
      p.first = before + __shfl_sync(0xFFFFFFFFu, incl - n, src);
      p.count = __shfl_sync(0xFFFFFFFFu, n, src);
      return p;
    }
    before += __shfl_sync(0xFFFFFFFFu, incl, 31);
  }
  p.b = a.B;
  p.first = p.count = 0;
  return p;
}

// Is slot of entry b also the slot of an earlier entry?  (One warp.)
__device__ __forceinline__ bool slot_seen_before(const int32_t* cache_slot, int b, int lane) {
  if (!cache_slot) return false;
  const int mine = cache_slot[b];
  bool hit = false;
  for (int i = lane; i < b; i += 32) hit |= cache_slot[i] == mine;
  return __any_sync(0xFFFFFFFFu, hit);
}

// One lane of a converged warp, for a role that issues MMAs: measured, a
// tcgen05.mma takes 16 cycles to issue under it, and 120, whatever its size,
// under lane == 0.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// D (+)= A B^T over K = 128: eight MMAs on two swizzled 32 KB tiles, the
// descriptors' offsets known at compile time.
template <bool kAdd = false>
__device__ __forceinline__ void umma_bf16_k128(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < kFaD / 16; ++kk) {
    const uint32_t off = ((kk >> 2) * kFaHalfBytes + (kk & 3) * 32) >> 4;
    umma_bf16(d, adesc + off, bdesc + off, idesc, kAdd || kk > 0 ? 1u : 0u);
  }
}

// Packed fp32 arithmetic of sm_100: two values in one register pair.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One 16-byte chunk of a 128-byte-swizzled 64-column half tile.
__device__ __forceinline__ uint32_t sw128_addr(uint32_t tile, int row, int chunk) {
  return tile + uint32_t(chunk >> 3) * kSdHalfBytes + uint32_t(row) * 128u + (uint32_t((chunk ^ row) & 7) << 4);
}
__device__ __forceinline__ void ldsm_x4_at(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans_at(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// One CTA = one part: 16 query rows of one KV head over a range of keys, read
// once.  Rows are the heads of one sequence (own rows) or 16 consecutive
// (sequence, head) rows of the batch (prefix).  A producer thread streams
// 64-key K and V tiles by TMA through three 32 KB stages; four warps take 16
// keys each (m16n8k16), each with its own running softmax, and are merged in
// shared memory at the end.  HBM-bound: 2 CTAs per SM hold 192 KB in flight.
// Ranges begin at their first visible row, so only a range's last tile holds
// foreign rows: their scores are masked and their V fragments zeroed, and a
// non-finite value there reaches nothing.
__global__ void __launch_bounds__(kSdThreads)
    shared_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                         const __grid_constant__ CUtensorMap tm_kp, const __grid_constant__ CUtensorMap tm_vp,
                         const SharedDecodeArgs a) {
  extern __shared__ uint8_t sd_smem_raw[];
  __shared__ float2 s_ml[kSdMaxGroup];  // direct: a row's maximum and 1 / l
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sd_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kSdStages * kSdStageBytes);
  uint64_t* empty = full + kSdStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kSdStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSdStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (threadIdx.x == 128) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kp);
    prefetch_tmap(&tm_vp);
  }
  // The prefix part's kernel reads nothing of this one's and let it start only
  // after everything before had completed: the two run side by side.
  if (!a.overlaps) griddep_wait();
  griddep_launch_dependents();
  // the unit: rows row0 .. row0+n_rows-1 of (sequence, head in group) order over
  // prefix rows [p0, p1) and own rows [k0, k1)
  const int u = blockIdx.x;
  const bool is_prefix = u < a.n_prefix_units;
  int kvh, part = 0, row0, n_rows, p0 = 0, p1 = 0, k0 = 0, k1 = 0, own_b = 0, slot = 0, lo = 0;
  bool live = true;
  if (is_prefix) {
    const int rt = u % a.row_tiles, rest = u / a.row_tiles;
    kvh = rest % a.nkv;
    part = rest / a.nkv;
    row0 = rt * 16;
    n_rows = min(16, a.B * a.G - row0);
    p0 = part * a.pchunk;
    p1 = min(a.P, p0 + a.pchunk);
  } else {
    const int v = u - a.n_prefix_units;
    kvh = v % a.nkv;
    part = v / a.nkv;
    const bool whole = a.own_slots == 0;  // a sequence is one part (and with `direct` the only one)
    OwnParts parts = {part, 0, part, 1};
    if (!whole) parts = own_parts(a, part, lane);
    own_b = parts.b;
    live = own_b < a.B;  // there may be fewer parts than units
    if (live) {
      int hi;
      if (!own_range(a.kv_len, a.cache_slot, a.kv_start, own_b, a.max_len, a.n_slots, slot, lo, hi) &&
          threadIdx.x == 0)
        record_device_error(kDevErrBadIndex);
      k0 = whole ? lo : lo + (part - parts.first) * parts.chunk;
      k1 = whole ? hi : min(hi, k0 + parts.chunk);
      if (a.direct)
        p1 = a.P;
      else if (kvh == 0 && part == parts.first && threadIdx.x == 0)
        a.plan[own_b] = make_int2(parts.first, k1 > k0 ? parts.count : 0);
    }
    row0 = own_b * a.G;
    n_rows = a.G;
  }
  const int n_pre = (p1 - p0 + kSdKeys - 1) / kSdKeys;
  const int n_tiles = live ? n_pre + (k1 - k0 + kSdKeys - 1) / kSdKeys : 0;
  __syncthreads();

  if (warp == 4) {
    if (lane == 0 && n_tiles > 0) {
      int issued = 0;
      for (int j = 0; j < n_tiles; ++j, ++issued) {
        const int st = j % kSdStages;
        if (j >= kSdStages &&
            !mbar_wait_bounded(&empty[st], (j / kSdStages - 1) & 1, abort_flag, kDevErrWaitTimeoutProducer))
          break;
        uint8_t* kt = smem + st * kSdStageBytes;
        const bool pre = j < n_pre;
        const CUtensorMap* mk = pre ? &tm_kp : &tm_k;
        const CUtensorMap* mv = pre ? &tm_vp : &tm_v;
        const int y = pre ? p0 + j * kSdKeys : k0 + (j - n_pre) * kSdKeys;
        const int z = pre ? a.prefix_z + kvh : slot * a.nkv + kvh;
        mbar_arrive_expect_tx(&full[st], kSdStageBytes);
        tma_load_3d(kt, mk, 0, y, z, &full[st]);
        tma_load_3d(kt + kSdHalfBytes, mk, 64, y, z, &full[st]);
        tma_load_3d(kt + kSdTileBytes, mv, 0, y, z, &full[st]);
        tma_load_3d(kt + kSdTileBytes + kSdHalfBytes, mv, 64, y, z, &full[st]);
      }
      // copies in flight land before the CTA can exit
      for (int j = max(0, issued - kSdStages); j < issued; ++j)
        fa_wait_landed(&full[j % kSdStages], (j / kSdStages) & 1);
    }
  }
  const int g = lane >> 2, tq = lane & 3;
  float o[16][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  bool ok = true;
  if (warp < 4 && n_tiles > 0) {
    // query fragments straight from global memory; rows past n_rows are zero
    uint32_t qa[8][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = g + 8 * h;
      const int r = row0 + i;
      const __nv_bfloat16* qrow = a.q + (size_t(r / a.G) * a.nh + kvh * a.G + r % a.G) * kAttnD;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        qa[kk][h] = i < n_rows ? *reinterpret_cast<const uint32_t*>(qrow + kk * 16 + 2 * tq) : 0u;
        qa[kk][2 + h] = i < n_rows ? *reinterpret_cast<const uint32_t*>(qrow + kk * 16 + 8 + 2 * tq) : 0u;
      }
    }
#pragma unroll
    for (int dn = 0; dn < 16; ++dn)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dn][i] = 0.f;
    float* sc_out = a.scores ? a.scores + size_t(own_b * a.nkv + kvh) * a.score_rows * a.G : nullptr;
    const int mi = lane >> 3, r8 = lane & 7;
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j % kSdStages;
      if (!fa_wait_warp(&full[st], (j / kSdStages) & 1, abort_flag, kDevErrWaitTimeoutEpilogue)) {
        ok = false;
        break;
      }
      const bool pre = j < n_pre;
      const int end = pre ? p1 : k1;
      const int key0 = (pre ? p0 + j * kSdKeys : k0 + (j - n_pre) * kSdKeys) + warp * 16;
      if (key0 < end) {
        const uint32_t kt = smem_u32(smem + st * kSdStageBytes), vt = kt + kSdTileBytes;
        // four independent chains of MMAs (a chain of eight waits on itself)
        float s[2][4], s1[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][i] = s1[nt][i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; kk += 2)
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            uint32_t b[4];
            ldsm_x4_at(b, sw128_addr(kt, warp * 16 + nt * 8 + r8, kk * 2 + mi));
            mma_bf16_16816(s[nt], qa[kk], b[0], b[1]);
            mma_bf16_16816(s1[nt], qa[kk + 1], b[2], b[3]);
          }
        const bool tail = key0 + 16 > end;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[nt][i] = (s[nt][i] + s1[nt][i]) * a.scale_log2;
            if (tail && key0 + nt * 8 + 2 * tq + (i & 1) >= end) s[nt][i] = -INFINITY;
          }
        if (sc_out && !pre) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + nt * 8 + 2 * tq + (i & 1), row = g + 8 * (i >> 1);
              if (key < end && row < n_rows) sc_out[size_t(key) * a.G + row] = s[nt][i];
            }
        }
        // The running maximum moves only when a score exceeds it by more than
        // 2^8: the exponentials stay below 2^8, and most tiles need no
        // exchange between lanes and no rescaling.  Rows 8..15 are idle with
        // up to 8 rows.
        float mx[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) mx[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        if (__any_sync(0xFFFFFFFFu, mx[0] > m[0] + kFaRescaleLog2 || (n_rows > 8 && mx[1] > m[1] + kFaRescaleLog2))) {
          float alpha[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], 2));
            const float m_new = fmaxf(m[h], mx[h]);
            alpha[h] = fa_exp2(m[h] - (m_new == -INFINITY ? 0.f : m_new));  // m[h] == -inf -> 0
            m[h] = m_new;
            l[h] *= alpha[h];
          }
#pragma unroll
          for (int dn = 0; dn < 16; ++dn)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[dn][i] *= alpha[i >> 1];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && n_rows <= 8) {
            s[0][2] = s[0][3] = s[1][2] = s[1][3] = 0.f;
            continue;
          }
          const float base = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[nt][2 * h + e] = fa_exp2(s[nt][2 * h + e] - base);
          l[h] += (s[0][2 * h] + s[0][2 * h + 1]) + (s[1][2 * h] + s[1][2 * h + 1]);
        }
        // P in bf16 (in [0, 2^8], relative rounding 2^-8), as the tensor core takes it beside a bf16 V
        uint32_t pa[4];
        pa[0] = pack_bf16x2(s[0][0], s[0][1]);
        pa[1] = pack_bf16x2(s[0][2], s[0][3]);
        pa[2] = pack_bf16x2(s[1][0], s[1][1]);
        pa[3] = pack_bf16x2(s[1][2], s[1][3]);
        uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;  // V rows of this lane's keys
        if (tail) {
          const int ka = key0 + 2 * tq;
          keep0 = (ka < end ? 0xFFFFu : 0u) | (ka + 1 < end ? 0xFFFF0000u : 0u);
          keep1 = (ka + 8 < end ? 0xFFFFu : 0u) | (ka + 9 < end ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int dn = 0; dn < 16; dn += 2) {
          uint32_t bb[4];
          ldsm_x4_trans_at(bb, sw128_addr(vt, warp * 16 + (mi & 1) * 8 + r8, dn + (mi >> 1)));
          mma_bf16_16816(o[dn], pa, bb[0] & keep0, bb[1] & keep1);
          mma_bf16_16816(o[dn + 1], pa, bb[2] & keep0, bb[3] & keep1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
      l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
    }
  }
  // every load has landed and been read: the stages hold the warps' results now
  const bool all_ok = __syncthreads_and(ok) != 0;
  if (all_ok && live) {
    float* red = reinterpret_cast<float*>(smem);
    if (warp < 4 && n_tiles > 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* wr = red + (warp * 16 + g + 8 * h) * kSdRedStride;
#pragma unroll
        for (int dn = 0; dn < 16; ++dn)
          *reinterpret_cast<float2*>(wr + dn * 8 + 2 * tq) = make_float2(o[dn][2 * h], o[dn][2 * h + 1]);
        if (tq == 0) *reinterpret_cast<float2*>(wr + kAttnD) = make_float2(m[h], l[h]);
      }
    }
    __syncthreads();
    // eight threads per row, 16 dims each
    const int i = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * 16;
    if (warp < 4 && i < n_rows) {
      const int r = row0 + i;
      const int bh = r / a.G * a.nh + kvh * a.G + r % a.G;
      float M = -INFINITY, L = 0.f;
      float acc[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = 0.f;
      if (n_tiles > 0) {
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, red[(w * 16 + i) * kSdRedStride + kAttnD]);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float* rw = red + (w * 16 + i) * kSdRedStride;
          const float sc = exp2f(rw[kAttnD] - base);
          L += rw[kAttnD + 1] * sc;
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(rw + d0 + e);
            acc[e] += v.x * sc;
            acc[e + 1] += v.y * sc;
            acc[e + 2] += v.z * sc;
            acc[e + 3] += v.w * sc;
          }
        }
      }
      if (a.direct) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        uint4* po = reinterpret_cast<uint4*>(a.out + size_t(bh) * kAttnD + d0);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          po[e] = make_uint4(pack_bf16x2(acc[8 * e] * inv, acc[8 * e + 1] * inv),
                             pack_bf16x2(acc[8 * e + 2] * inv, acc[8 * e + 3] * inv),
                             pack_bf16x2(acc[8 * e + 4] * inv, acc[8 * e + 5] * inv),
                             pack_bf16x2(acc[8 * e + 6] * inv, acc[8 * e + 7] * inv));
        if (d0 == 0) s_ml[i] = make_float2(M == -INFINITY ? 0.f : M, inv);
      } else {
        const size_t pidx = is_prefix ? size_t(bh) * a.psplits + part : size_t(part) * a.nh + kvh * a.G + i;
        float4* po = reinterpret_cast<float4*>((is_prefix ? a.pre_o : a.own_o) + pidx * kAttnD + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) po[e] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
        if (d0 == 0) *reinterpret_cast<float2*>((is_prefix ? a.pre_ml : a.own_ml) + pidx * 2) = make_float2(M, L);
      }
    }
    if (a.direct && a.weights) {
      const bool dup = slot_seen_before(a.cache_slot, own_b, lane);  // two entries of one slot would race
      __syncthreads();  // the scores and s_ml are there
      if (dup) {
        if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);
      } else {
        float* w = a.weights + (size_t(slot) * a.nkv + kvh) * a.max_seq;
        const float* sc = a.scores + size_t(own_b * a.nkv + kvh) * a.score_rows * a.G;
        for (int row = (a.accumulate ? lo : 0) + threadIdx.x; row < k1; row += kSdThreads) {
          float x = 0.f;
          if (row >= lo)
            for (int h = 0; h < a.G; ++h) x += exp2f(sc[size_t(row) * a.G + h] - s_ml[h].x) * s_ml[h].y;
          w[row] = a.accumulate ? w[row] + x : x;
        }
      }
    }
  }
  // the grid completes after the kernel before it, for the one that joins both
  if (a.overlaps && blockIdx.x == gridDim.x - 1) griddep_wait();
}

// A row's parts: the prefix's, then its own.
struct RowParts {
  const float* pre_ml;
  const float* pre_o;
  const float* own_ml;  // of the sequence's first part
  const float* own_o;
  int n_pre, n, nh;
  __device__ __forceinline__ float2 ml(int i) const {
    return *reinterpret_cast<const float2*>(i < n_pre ? pre_ml + i * 2 : own_ml + size_t(i - n_pre) * nh * 2);
  }
  __device__ __forceinline__ float4 o(int i, int lane) const {
    return *reinterpret_cast<const float4*>((i < n_pre ? pre_o + size_t(i) * kAttnD
                                                       : own_o + size_t(i - n_pre) * nh * kAttnD) +
                                            lane * 4);
  }
};
__device__ __forceinline__ RowParts row_parts(const SharedDecodeArgs& a, int own_count, int own_first, int b, int h) {
  const size_t bh = size_t(b) * a.nh + h, first = size_t(own_first) * a.nh + h;
  return {a.pre_ml + bh * a.psplits * 2, a.pre_o + bh * a.psplits * kAttnD, a.own_ml + first * 2,
          a.own_o + first * kAttnD,      a.psplits, a.psplits + own_count,  a.nh};
}
// A sequence's first own part and their number; one without own rows has no
// part that wrote its plan.  `ok` as of own_range.
__device__ __forceinline__ int2 own_plan(const SharedDecodeArgs& a, int b, bool& ok) {
  int slot, lo, hi;
  const int2 p = a.plan[b];
  ok = own_range(a.kv_len, a.cache_slot, a.kv_start, b, a.max_len, a.n_slots, slot, lo, hi);
  return hi > lo ? p : make_int2(0, 0);
}

// M and 1/l of one row from its parts, in every lane of the warp.
__device__ __forceinline__ void join_ml(const RowParts& p, int lane, float& M, float& inv_l) {
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < p.n) ml = p.ml(lane);
  float mm = ml.x;
  for (int s = lane + 32; s < p.n; s += 32) mm = fmaxf(mm, p.ml(s).x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, off));
  M = mm == -INFINITY ? 0.f : mm;
  float L = ml.y == 0.f ? 0.f : ml.y * exp2f(ml.x - M);
  for (int s = lane + 32; s < p.n; s += 32) {
    const float2 v = p.ml(s);
    if (v.y != 0.f) L += v.y * exp2f(v.x - M);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, off);
  inv_l = L == 0.f ? 0.f : 1.f / L;
}

// Blocks [0, n_out_blocks): one warp per (sequence, head), or with many parts
// one block, joins the parts of its output row in a fixed order (run-to-run
// identical).  The blocks after them: 256 own rows of one (sequence, KV head)
// each, one thread per row, weights (+)= sum over the group's heads of
// exp2(s - M) / l.
__global__ void __launch_bounds__(256) shared_decode_combine_kernel(const SharedDecodeArgs a) {
  __shared__ float sM[kSdMaxGroup], sInv[kSdMaxGroup];
  __shared__ float4 s_acc[8][32];
  __shared__ int s_dup;
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (int(blockIdx.x) < a.n_out_blocks) {
    const int gw = a.wide ? blockIdx.x : blockIdx.x * 8 + warp;
    if (gw >= a.B * a.nh) return;
    const int b = gw / a.nh;
    bool ok;
    const int2 own = own_plan(a, b, ok);
    // (where own rows are cut, a sequence whose length or slot lies outside the
    // cache has no part that could report it)
    if (!ok && gw % a.nh == 0 && lane == 0 && (!a.wide || warp == 0)) record_device_error(kDevErrBadIndex);
    const RowParts p = row_parts(a, own.y, own.x, b, gw % a.nh);
    float M, inv;
    join_ml(p, lane, M, inv);
    const int first = a.wide ? warp : 0, step = a.wide ? 8 : 1;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = first; s0 < p.n; s0 += 8 * step) {
      float4 v[8];
      float sc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int s = s0 + j * step;
        sc[j] = 0.f;
        v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < p.n) {
          const float2 ml = p.ml(s);
          v[j] = p.o(s, lane);
          if (ml.y != 0.f) sc[j] = exp2f(ml.x - M);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (sc[j] == 0.f) continue;  // an empty part has no output; one so small adds nothing
        acc[0] += v[j].x * sc[j];
        acc[1] += v[j].y * sc[j];
        acc[2] += v[j].z * sc[j];
        acc[3] += v[j].w * sc[j];
      }
    }
    if (a.wide) {
      s_acc[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      __syncthreads();
      if (warp > 0) return;
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        const float4 v = s_acc[i][lane];
        acc[0] += v.x;
        acc[1] += v.y;
        acc[2] += v.z;
        acc[3] += v.w;
      }
    }
    uint2 w;
    w.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(a.out + size_t(gw) * kAttnD + lane * 4) = w;
    return;
  }
  const int v = blockIdx.x - a.n_out_blocks;
  const int rb = v % a.row_blocks, rest = v / a.row_blocks;
  const int kvh = rest % a.nkv, b = rest / a.nkv;
  int slot, lo, hi;
  if (!own_range(a.kv_len, a.cache_slot, a.kv_start, b, a.max_len, a.n_slots, slot, lo, hi)) return;  // (reported above)
  const int first = rb * kSdCombineRows;
  if (first >= hi && rb > 0) return;  // (the first block also looks for a slot given twice)
  const int row = first + threadIdx.x;
  // the row's scores and total, in flight while the maxima are joined
  const float* sp = a.scores + (size_t(b * a.nkv + kvh) * a.score_rows + row) * a.G;
  float* dst = a.weights + (size_t(slot) * a.nkv + kvh) * a.max_seq + row;
  float sc[kSdMaxGroup];
#pragma unroll
  for (int h = 0; h < kSdMaxGroup; ++h) sc[h] = h < a.G && row >= lo && row < hi ? sp[h] : -INFINITY;
  const float total = a.accumulate && row < hi ? *dst : 0.f;
  bool ok;
  const int2 own = own_plan(a, b, ok);
  for (int h = warp; h < a.G; h += 8) {
    float M, inv;
    join_ml(row_parts(a, own.y, own.x, b, kvh * a.G + h), lane, M, inv);
    if (lane == 0) {
      sM[h] = M;
      sInv[h] = inv;
    }
  }
  if (warp == 0) {
    // two entries of one slot would race: the first one's weights are added
    const bool dup = slot_seen_before(a.cache_slot, b, lane);
    if (lane == 0) {
      s_dup = dup;
      if (dup) record_device_error(kDevErrBadIndex);
    }
  }
  __syncthreads();
  if (s_dup || row >= hi) return;
  float w = 0.f;
#pragma unroll
  for (int h = 0; h < kSdMaxGroup; ++h)
    if (h < a.G && row >= lo) w += exp2f(sc[h] - sM[h]) * sInv[h];
  *dst = total + w;
}

}  // namespace qmoe

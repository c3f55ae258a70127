// Attention of new tokens over the paged 8-bit cache: the kernel for few rows, and the choice
// between it and the one for many (cache_attention_many.cu).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   k_j = ks_j kc_j, v_j = vs_j vc_j (s8 codes)
//
// with j over the cached tokens that token i sees: all of them, or (causal) those at positions up
// to its own.  A row that sees nothing is 0.
//
// The weights w_j = p_j vs_j carry the value scales.  Codes are exact in fp16, and a weight is split into
// two fp16 terms, w = hi + lo with 11 bits each, after scaling by a power of two that bounds the
// weights; two products with fp32 sums then give 22 bits where one would give 11.  That power is taken
// per row from the keys the row sees, w_j among them and not vs_j alone: a token that is hidden from a row, or
// has next to no weight in it, takes no bits from the others however large its values are.  The softmax is
// the one-pass form: a reference maximum and a sum in fp32, sums rescaled when a score exceeds the
// reference by more than kLazy (in log2 units), which is rare after the first keys.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cache_attention.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "ptx.cuh"

namespace tfccb200 {

namespace {

// ---- few rows: memory-bound ----------------------------------------------------------------------
//
// Up to 8 (or 16) rows of a kv head against its whole cache: every code is used for a handful
// of products, so what counts is streaming the cache and spending few instructions on a code.  A warp
// works alone: it brings 16 keys and their values at a time through its own ring of cp.async stages (no
// CTA barrier in the loop) and multiplies with mma.sync, whose fragments are read straight from
// the rows as they lie because the order of k is free: a lane's 16 bytes of a key row serve as its k slots of
// successive steps.
//   Scores: q is a 31-bit integer per element (scaled by a power of two per row) in four balanced
//   8-bit digits, and the codes are multiplied as they are, m16n8k32 in integers: exact sums and no conversion of
//   K at all.  Elements down to 2^-6 of the row's largest are held exactly, smaller ones to 2^-30 of it: with
//   three digits (2^-22) a head with one large channel lost what the others say.  With 8 rows
//   two digits fill the 16 rows of one product.
//   Output: V becomes fp16 (1.5 instructions a code), weights as above; with 8 rows the 16 rows of
//   m16n8k16 hold their hi and lo terms side by side.
// Eight warps take the eight 16-key groups of a 128-key block and are added at the item's end.
// Two sequences of 65536 keys, 64 / 8 heads of 128: 68 us, 4.1 TB/s, 0.62 of the measured copy rate; 32 ragged
// ones, 32 / 8 heads: 72 us; 24 ragged ones with 3 or 4 new tokens (16 rows): 111 us, 104 with three digits.
// Inside the loop a CTA pair reads 44 GB/s per SM, the copy rate; what is left is 4 us until the
// first loads, CTAs that finish 10 us apart, 4 us per item of a short sequence, and the merge.  (Scores from fp16 terms of q instead of digits 83 us; three CTAs per SM with 80 registers
// 126 us, because of spills.)
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;

template <int DIM, int ROWS>
struct FewLayout {
  static constexpr int kStages = DIM == 128 ? 3 : 6;
  static constexpr int kCodeBytes = 16 * DIM;               // codes of 16 keys (or values)
  static constexpr int kStageBytes = 2 * kCodeBytes + 128;  // + their scales
  static constexpr int kRingBytes = kStages * kStageBytes;  // per warp
  static constexpr int kFragBytes = (DIM / 32) * 32 * (ROWS == 8 ? 2 : 4) * 16;  // digits of q
  static constexpr int kSmall = kFragBytes + kFewWarps * kRingBytes;
  static constexpr int kSmem = kSmall + kFewWarps * 3 * ROWS * 4;
  static_assert(ROWS * DIM * 4 <= kRingBytes, "a warp's sums reuse its ring");
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// Four integers below 2^30 -> four words of their balanced base-256 digits, lowest first.
__device__ __forceinline__ void digits4(const int (&v)[4], uint32_t (&d)[4]) {
  uint32_t x[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int r = v[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int low = static_cast<int8_t>(r);
      x[i][k] = low & 0xff;
      r = (r - low) >> 8;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) d[k] = x[0][k] | (x[1][k] << 8) | (x[2][k] << 16) | (x[3][k] << 24);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint4 a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}

// Where 16-byte chunk `c` of code row `r` of a stage lies.  K rows are read by four lanes per row,
// V rows by lanes that share a chunk over four rows of one parity; both orders then touch eight different
// chunks of a 128-byte line in every quarter of a warp's access.
template <int DIM>
__device__ __forceinline__ unsigned key_chunk(unsigned r, unsigned c) {
  if constexpr (DIM == 128) return r * 128 + ((c ^ ((r & 1u) << 2)) << 4);
  else return r * 64 + (c << 4);
}
template <int DIM>
__device__ __forceinline__ unsigned value_chunk(unsigned r, unsigned c) {
  if constexpr (DIM == 128) return r * 128 + ((c ^ (r & 6u)) << 4);
  else return (r >> 1) * 128 + (((((r & 1u) << 2) + c) ^ (r & 6u)) << 4);
}

// The unit of a row's weights: the value scale `vref`, a power of two, is held as kWeightTop = 2^10, so that weights
// reach at most 2^10 2^kLazy, inside fp16's range, and have 22 bits down to 2^-13 of the top.  vref is the largest
// scale that the row has met, but at most kValueRange times its largest weight so far (p_j vs_j, with p_j = 1 at
// the reference maximum): a weight's absolute error is then at most 2^-25 2^-10 vref <= 2^-26 of the largest weight.
constexpr float kWeightTop = 1024.f;
constexpr float kLazy = 5.f;
constexpr float kValueRange = 512.f;
constexpr float kValueFloor = 7.8886091e-31f;  // 2^-100

template <int DIM, int ROWS>
__global__ void __launch_bounds__(kFewThreads, 2) cache_attention_few_kernel(const __grid_constant__ CacheAttention a) {
  using L = FewLayout<DIM, ROWS>;
  constexpr int kSteps = DIM / 32;   // k-steps of a score
  constexpr int kVecs = DIM / 16;    // quads of a row that a lane holds
  constexpr int kTiles = DIM / 8;    // 8-wide column tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ ScheduleShared sched;
  pdl_release();
  pdl_wait();
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
  uint4* frag = reinterpret_cast<uint4*>(smem);
  uint8_t* ring = smem + L::kFragBytes + warp * L::kRingBytes;
  const uint32_t ring_addr = ptx::smem_u32(ring);
  float* red_m = reinterpret_cast<float*>(smem + L::kSmall);  // [warp][row]
  float* red_l = red_m + kFewWarps * ROWS;
  float* red_v = red_l + kFewWarps * ROWS;

  ThreadSequence mine;
  const unsigned long long units = all_units<ROWS, kFewThreads>(a, &sched, &mine);
  const unsigned busy = busy_ctas(units, a.grid);
  const bool mine_any = blockIdx.x < busy;
  const unsigned long long u0 = mine_any ? range_begin(units, busy, blockIdx.x) : 0;
  const unsigned long long u1 = mine_any ? range_begin(units, busy, blockIdx.x + 1) : 0;
  if (u0 == u1) {
    if (a.scratch && tid == 0) write_note<ROWS>(a, blockIdx.x, busy, units, u1, nullptr);
    return;
  }
  find_unit<ROWS, kFewThreads>(a, u0, mine, &sched);

  bool noted = false;
  for (ItemWalk<ROWS> item(a, u1 - u0, &sched); !item.done(); item.next()) {
    if (a.scratch && item.taken == item.left) {  // the range's last
      if (tid == 0) write_note<ROWS>(a, blockIdx.x, busy, units, u1, &item);
      noted = true;
    }
    const unsigned rows = static_cast<unsigned>(item.seq.count) * a.group;
    const int length = item.seq.length, past = length - item.seq.count;
    const unsigned head = item.head;
    const int b = item.b;

    // ---- the warp's loads: 16 keys of block `blk` into stage `st` ----
    // `slot`: place of key lane % 16 of the group in the scale arrays, ~0u for none.  It is looked up
    // a step ahead, so that the page table's latency is not in the way.
    auto look_up = [&](unsigned blk) {
      const unsigned pos = blk * kBlockKeys + warp * 16 + (lane & 15u);
      if (blk >= item.hi || static_cast<int>(pos) >= length) return ~0u;
      const int page = page_of(a.c, b, pos);
      return page < 0 ? ~0u : static_cast<unsigned>(cache_slot(a.c, page, head, pos));
    };
    auto load = [&](unsigned slot, int st) {
      const uint32_t dst = ring_addr + st * L::kStageBytes;
      {  // scales: lanes 0-15 of the keys, 16-31 of the values
        const uint32_t d = dst + 2 * L::kCodeBytes + lane * 4;
        if (slot != ~0u) {
          cp_async_4(d, (lane < 16 ? a.c.key_scales : a.c.value_scales) + slot);
        } else {  // a page that does not exist shows as NaN (a place behind the end is masked anyway)
          *reinterpret_cast<uint32_t*>(ring + (d - ring_addr)) = 0x7fffffffu;
        }
      }
      constexpr int kChunks = DIM / 16;  // 16-byte chunks of a row
      constexpr int kPer = 16 * kChunks / 32;
      if (a.c.page_shift >= 4) {
        // the 16 places follow one another in one page: two addresses, the rest are constant steps
        const unsigned r0 = lane / kChunks, c = lane % kChunks;
        const unsigned sl = __shfl_sync(0xffffffffu, slot, 0);  // (a group is loaded when its first key exists)
        const unsigned n = __popc(__ballot_sync(0xffffffffu, slot != ~0u) & 0xffffu);
        const size_t at = static_cast<size_t>(n ? sl + r0 : 0u) * DIM + c * 16;
        const int8_t* const k = a.c.keys + at;
        const int8_t* const v = a.c.values + at;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const unsigned r = i * (32 / kChunks) + r0;
          const bool in = r < n;
          cp_async_16(dst + key_chunk<DIM>(r, c), in ? k + i * (32 / kChunks) * DIM : a.c.keys, in);
          cp_async_16(dst + L::kCodeBytes + value_chunk<DIM>(r, c), in ? v + i * (32 / kChunks) * DIM : a.c.values, in);
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const unsigned r = (i * 32 + lane) / kChunks, c = lane % kChunks;
        const unsigned sl = __shfl_sync(0xffffffffu, slot, r);
        const size_t at = (sl != ~0u ? static_cast<size_t>(sl) : 0) * DIM + c * 16;
        cp_async_16(dst + key_chunk<DIM>(r, c), a.c.keys + at, sl != ~0u);
        cp_async_16(dst + L::kCodeBytes + value_chunk<DIM>(r, c), a.c.values + at, sl != ~0u);
      }
    };
    auto has_keys = [&](unsigned blk) {  // warp-uniform
      return blk < item.hi && static_cast<int>(blk * kBlockKeys + warp * 16) < length;
    };
    unsigned next_slot;
    {
      unsigned slot[L::kStages];
#pragma unroll
      for (int s = 0; s < L::kStages; ++s) slot[s] = look_up(item.lo + s);
#pragma unroll
      for (int s = 0; s < L::kStages - 1; ++s) {
        if (has_keys(item.lo + s)) load(slot[s], s);
        cp_async_commit();
      }
      next_slot = slot[L::kStages - 1];
    }

    // ---- digits of the rows of q, scaled by a power of two per row ----
    // Lane (g, t) holds row g's (and, 16 rows, row g + 8's) values d = 64 [i >= 4] + 16 t + 4 (i & 3) + 0..3
    // for i = 0 .. DIM / 16 - 1, and i = 2 s, 2 s + 1 are its k slots of step s.
    float row_scale[ROWS / 8];
    int sees[ROWS / 8];
#pragma unroll
    for (int h = 0; h < ROWS / 8; ++h) {
      const unsigned r = item.tile * ROWS + g + 8 * h;
      const unsigned tok = r / a.group;
      const bool live = r < rows;
      sees[h] = !live ? 0 : (a.causal ? past + static_cast<int>(tok) + 1 : length);
      const float* src = a.q + a.ldq * (static_cast<size_t>(item.seq.first) + (live ? tok : 0)) +
                         (static_cast<size_t>(head) * a.group + (live ? r % a.group : 0)) * DIM;
      float4 f[kVecs];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        f[i] = live ? *reinterpret_cast<const float4*>(src + (i >> 2) * 64 + 16 * t + 4 * (i & 3))
                    : make_float4(0.f, 0.f, 0.f, 0.f);
        f[i].x *= a.scale; f[i].y *= a.scale; f[i].z *= a.scale; f[i].w *= a.scale;
        m = max(m, max(max(__float_as_uint(f[i].x) & 0x7fffffffu, __float_as_uint(f[i].y) & 0x7fffffffu),
                       max(__float_as_uint(f[i].z) & 0x7fffffffu, __float_as_uint(f[i].w) & 0x7fffffffu)));
      }
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // 2^(29 - exponent): the row's largest value lands in [2^29, 2^30), inside four balanced digits.  Zero and
      // tiny rows (below 2^-97) take the bound of the range; a row with an infinity or a NaN is NaN.
      const int ex = static_cast<int>(m >> 23) - 127;
      const int sh = ex == 128 ? 0 : 29 - max(ex, -97);
      const float up = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
      row_scale[h] = ex == 128 ? __uint_as_float(0x7fffffffu) : __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s % kFewWarps != static_cast<int>(warp) % kSteps) continue;
        uint32_t d[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 x = f[2 * s + e];
          const int v[4] = {__float2int_rn(x.x * up), __float2int_rn(x.y * up), __float2int_rn(x.z * up), __float2int_rn(x.w * up)};
          digits4(v, d[e]);
        }
        if constexpr (ROWS == 8) {
          frag[s * 32 + lane] = make_uint4(d[0][3], d[0][2], d[1][3], d[1][2]);
          frag[(kSteps + s) * 32 + lane] = make_uint4(d[0][1], d[0][0], d[1][1], d[1][0]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t* w = reinterpret_cast<uint32_t*>(frag + (k * kSteps + s) * 32 + lane);
            w[h] = d[0][k];
            w[2 + h] = d[1][k];
          }
        }
      }
    }
    __syncthreads();

    float o[kTiles][ROWS / 4];  // [tile i][2 h + c]: column kTiles (2 t + c) + i of row g + 8 h
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < ROWS / 4; ++j) o[i][j] = 0.f;
    float top[ROWS / 8], sum[ROWS / 8], vup[ROWS / 8];  // vup = kWeightTop / vref
#pragma unroll
    for (int h = 0; h < ROWS / 8; ++h) top[h] = -INFINITY, sum[h] = 0.f, vup[h] = kWeightTop / kValueFloor;

    int st = 0;
    // keys below this are seen by every row of the item
    const int all_see = a.causal ? past + static_cast<int>(item.tile * ROWS / a.group) + 1 : length;
    // One group of 16 keys; kMask: with keys that not every row sees (compiled apart).
    auto group16 = [&](unsigned blk, auto mask) {
      constexpr bool kMask = decltype(mask)::value;
      cp_async_wait<L::kStages - 2>();
      __syncwarp();
      const uint8_t* stage = ring + st * L::kStageBytes;
      {
        const unsigned ahead = blk + L::kStages - 1;
        if (has_keys(ahead)) load(next_slot, st == 0 ? L::kStages - 1 : st - 1);
        cp_async_commit();
        next_slot = look_up(ahead + 1);
      }
      if (++st == L::kStages) st = 0;

      // scores of keys 0-7 and 8-15 of the group: [2 j + e] of a lane (g, t) are keys 2 t + e (+ 8 j)
      float x[ROWS / 8][4];
      {
        constexpr int kProducts = ROWS == 8 ? 2 : 4;
        int c[kProducts][2][4];
#pragma unroll
        for (int k = 0; k < kProducts; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) c[k][0][i] = c[k][1][i] = 0;
#pragma unroll
        for (int q = 0; q < DIM / 64; ++q) {
          const uint4 ka = *reinterpret_cast<const uint4*>(stage + key_chunk<DIM>(g, q * 4 + t));
          const uint4 kb = *reinterpret_cast<const uint4*>(stage + key_chunk<DIM>(g + 8, q * 4 + t));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int s = 2 * q + e;
            const uint32_t a0 = e ? ka.z : ka.x, a1 = e ? ka.w : ka.y, b0 = e ? kb.z : kb.x, b1 = e ? kb.w : kb.y;
#pragma unroll
            for (int k = 0; k < kProducts; ++k) {
              const uint4 f = frag[(k * kSteps + s) * 32 + lane];
              mma_s8(c[k][0], f, a0, a1);
              mma_s8(c[k][1], f, b0, b1);
            }
          }
        }
        // (highest digit * 2^8 + next) * 2^16 + (third * 2^8 + lowest): the brackets stay below 2^30
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (ROWS == 8) {
              x[0][2 * j + e] = fmaf(static_cast<float>(c[0][j][e] * 256 + c[0][j][2 + e]), 65536.f,
                                     static_cast<float>(c[1][j][e] * 256 + c[1][j][2 + e]));
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                x[h][2 * j + e] = fmaf(static_cast<float>(c[3][j][2 * h + e] * 256 + c[2][j][2 * h + e]), 65536.f,
                                       static_cast<float>(c[1][j][2 * h + e] * 256 + c[0][j][2 * h + e]));
            }
          }
      }
      const float* ks = reinterpret_cast<const float*>(stage + 2 * L::kCodeBytes);
      const float2 ka = *reinterpret_cast<const float2*>(ks + 2 * t), kb = *reinterpret_cast<const float2*>(ks + 2 * t + 8);
      const float2 va = *reinterpret_cast<const float2*>(ks + 16 + 2 * t), vb = *reinterpret_cast<const float2*>(ks + 24 + 2 * t);
      const int key0 = static_cast<int>(blk * kBlockKeys + warp * 16 + 2 * t);
      const float kscale[4] = {ka.x, ka.y, kb.x, kb.y};
      const float vscale[4] = {va.x, va.y, vb.x, vb.y};
      auto seen = [&](int h, int j) { return !kMask || key0 + (j & 1) + (j >> 1) * 8 < sees[h]; };
      float vs[ROWS / 8][4];  // value scales in the row's unit, 0 where it does not see the key
      auto scale_values = [&](int h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) vs[h][j] = seen(h, j) ? vscale[j] * vup[h] : 0.f;
      };
      bool grows = false;
#pragma unroll
      for (int h = 0; h < ROWS / 8; ++h) {
        const float limit = top[h] + kLazy;  // -inf before the first key
        scale_values(h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[h][j] *= kscale[j] * row_scale[h];
          if constexpr (kMask) x[h][j] = seen(h, j) ? x[h][j] : -INFINITY;
          grows |= x[h][j] > limit;
          grows |= fabsf(vs[h][j]) > kWeightTop;
        }
      }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int h = 0; h < ROWS / 8; ++h) {
          float m = fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const float next = m > top[h] + kLazy ? m : top[h];
          const float ref = next == -INFINITY ? 0.f : next;
          const float f = exp2_fast(top[h] - ref);
          const float vref = kWeightTop / vup[h];
          float v = vref, w = f * (vref * (1.f / kValueRange));  // (the largest weight so far is no smaller)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y = seen(h, j) ? fabsf(vscale[j]) : 0.f;
            v = fmaxf(v, y);
            w = fmaxf(w, exp2_fast(x[h][j] - ref) * y);
          }
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 2));
          // powers of two: v upwards, the bound on it downwards
          v = __uint_as_float(min((__float_as_uint(v) + 0x7fffffu) & 0x7f800000u, 0x7f000000u));
          v = fmaxf(fminf(v, __uint_as_float(__float_as_uint(w * kValueRange) & 0x7f800000u)), kValueFloor);
          const float up = kWeightTop / v;
          // (f = 0: nothing so far counts, and up / vup may be infinite)
          const float fv = f == 0.f ? 0.f : f * (up / vup[h]);
          sum[h] *= f;
          top[h] = next;
          vup[h] = up;
          scale_values(h);
#pragma unroll
          for (int j = 0; j < 4; ++j)  // (a finite scale of a weight that underflows stays finite: 0 * inf)
            if (fabsf(vscale[j]) < INFINITY) vs[h][j] = fminf(fmaxf(vs[h][j], -3.4e38f), 3.4e38f);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            o[i][2 * h] *= fv;
            o[i][2 * h + 1] *= fv;
          }
        }
      }
      uint32_t hi[ROWS / 8][2], lo[ROWS / 8][2];
#pragma unroll
      for (int h = 0; h < ROWS / 8; ++h) {
        const float base = top[h] == -INFINITY ? 0.f : top[h];
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2_fast(x[h][j] - base);
          sum[h] += p;
          w[j] = p * vs[h][j];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          hi[h][i] = pack_half2(w[2 * i], w[2 * i + 1]);
          lo[h][i] = pack_rest(w[2 * i], w[2 * i + 1], hi[h][i]);
        }
      }
      uint4 pa, pb;
      if constexpr (ROWS == 8) {
        pa = make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1]);
      } else {
        pa = make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
        pb = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
      }
      // sums: lane (g, t) reads values 2t, 2t+1, 2t+8, 2t+9 at its DIM / 8 columns from DIM / 8 * g
      const uint8_t* vals = stage + L::kCodeBytes;
      constexpr int kWords = DIM / 32;
      uint32_t v[4][kWords];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned r = 2 * t + (j & 1) + (j >> 1) * 8;
        if constexpr (DIM == 128) {
          const uint4 q = *reinterpret_cast<const uint4*>(vals + value_chunk<DIM>(r, g));
          v[j][0] = q.x; v[j][1] = q.y; v[j][2] = q.z; v[j][3] = q.w;
        } else {
          const uint2 q = *reinterpret_cast<const uint2*>(vals + value_chunk<DIM>(r, g >> 1) + (g & 1u) * 8);
          v[j][0] = q.x; v[j][1] = q.y;
        }
      }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const uint32_t r0 = v[0][w] ^ 0x80808080u, r1 = v[1][w] ^ 0x80808080u;
        const uint32_t r2 = v[2][w] ^ 0x80808080u, r3 = v[3][w] ^ 0x80808080u;
        const uint32_t a01 = __byte_perm(r0, r1, 0x5140), a23 = __byte_perm(r0, r1, 0x7362);
        const uint32_t b01 = __byte_perm(r2, r3, 0x5140), b23 = __byte_perm(r2, r3, 0x7362);
        const uint32_t x0[4] = {codes_low(a01), codes_high(a01), codes_low(a23), codes_high(a23)};
        const uint32_t x1[4] = {codes_low(b01), codes_high(b01), codes_low(b23), codes_high(b23)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // from zero, and added in fp32: the instruction's own accumulation narrows without rounding
          // to nearest, which over thousands of keys doubled the error (6e-7 to 1.2e-6 at 65536)
          float d[4];
          mma_f16_zero(d, pa, x0[i], x1[i]);
          if constexpr (ROWS == 8) {
            o[w * 4 + i][0] += d[0] + d[2];
            o[w * 4 + i][1] += d[1] + d[3];
          } else {
            mma_f16(d, pb, x0[i], x1[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[w * 4 + i][j] += d[j];
          }
        }
      }
      __syncwarp();  // the stage may be overwritten
    };
    for (unsigned blk = item.lo; blk < item.hi; ++blk) {
      if (!has_keys(blk)) break;  // nor do later blocks have any for this warp
      if (static_cast<int>(blk * kBlockKeys + warp * 16 + 16) > all_see) group16(blk, std::true_type());
      else group16(blk, std::false_type());
    }
    cp_async_wait<0>();

    // ---- the warps' sums meet: maxima and weight sums in shared memory, sums in the rings ----
#pragma unroll
    for (int h = 0; h < ROWS / 8; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      if (t == 0) {
        red_m[warp * ROWS + g + 8 * h] = top[h];
        red_l[warp * ROWS + g + 8 * h] = sum[h];
        red_v[warp * ROWS + g + 8 * h] = 1.f / vup[h];
      }
    }
    __syncwarp();
    {
      float* dst = reinterpret_cast<float*>(ring);
      // lane (g, t): columns (DIM / 8) (2t + c) + i of the row, c = 0, 1
#pragma unroll
      for (int h = 0; h < ROWS / 8; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < kTiles; i += 4) {
            float4 y;
            float* yy = &y.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) yy[k] = o[i + k][2 * h + c];
            *reinterpret_cast<float4*>(dst + (g + 8 * h) * DIM + kTiles * (2 * t + c) + i) = y;
          }
    }
    __syncthreads();
    const bool whole = item.whole();
    float* out_piece = whole ? nullptr : piece<ROWS, DIM>(a, blockIdx.x, item.lo == 0);
    for (unsigned e = tid * 4; e < ROWS * DIM; e += kFewThreads * 4) {
      const unsigned r = e / DIM, d = e % DIM, row = item.tile * ROWS + r;
      if (row >= rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, red_m[w * ROWS + r]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float f = exp2_fast(red_m[w * ROWS + r] - base);
        l += f * red_l[w * ROWS + r];
        const float fv = f * red_v[w * ROWS + r];
        const float4 y = *reinterpret_cast<const float4*>(smem + L::kFragBytes + w * L::kRingBytes + (r * DIM + d) * 4);
        acc.x += fv * y.x; acc.y += fv * y.y; acc.z += fv * y.z; acc.w += fv * y.w;
      }
      if (whole) {
        const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;  // nothing seen: 0
        const unsigned tok = row / a.group;
        float* dst = a.out + a.ldo * (static_cast<size_t>(item.seq.first) + tok) +
                     (static_cast<size_t>(head) * a.group + row % a.group) * DIM + d;
        *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      } else {
        if (d == 0) {
          out_piece[r] = m;
          out_piece[ROWS + r] = l;
        }
        *reinterpret_cast<float4*>(out_piece + 2 * ROWS + e) = acc;
      }
    }
    __syncthreads();  // rings, fragments and maxima are free for the next item
  }
  if (a.scratch && !noted && tid == 0) write_note<ROWS>(a, blockIdx.x, busy, units, u1, nullptr);
}

// ---- host ----------------------------------------------------------------------------------------

constexpr unsigned kFewCtasPerSm = 2;

// Largest number of units a launch of these bounds can have.
unsigned long long few_units_bound(const CacheAttentionArgs& a) {
  return static_cast<unsigned long long>(a.cache.batch) * a.cache.kv_heads *
         ((a.max_length + kBlockKeys - 1) / kBlockKeys + kLeadUnits);
}

template <int DIM, int ROWS>
int launch_few(const CacheAttentionArgs& args, CacheAttention a, int sm_count) {
  using L = FewLayout<DIM, ROWS>;
  static std::atomic<unsigned long long> configured{0};
  int st = opt_in_smem(cache_attention_few_kernel<DIM, ROWS>, L::kSmem, configured);
  if (st != TFCCB200_OK) return st;
  // With one block per item nothing is cut as long as every item can have a CTA of its own or
  // shares one whole; the bound on the lengths tells.
  const unsigned long long bound = few_units_bound(args);
  a.grid = static_cast<unsigned>(bound < kFewCtasPerSm * sm_count ? bound : kFewCtasPerSm * sm_count);
  const bool cut = args.max_length > kBlockKeys;
  cudaError_t e = launch_after_previous(cache_attention_few_kernel<DIM, ROWS>, dim3(a.grid), dim3(kFewThreads),
                                        L::kSmem, args.cache.stream, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  if (cut && a.grid > 1) {
    e = launch_after_previous(cache_attention_merge_kernel<DIM, ROWS>, dim3(a.grid), dim3(256), 0,
                              args.cache.stream, a);
    if (e != cudaSuccess) return static_cast<int>(e);
    count_launch();
  }
  return TFCCB200_OK;
}

int few_rows_of(const CacheAttentionArgs& a) {  // 8 or 16: rows the few-rows kernel has to hold
  return static_cast<unsigned long long>(a.max_new) * (a.heads / a.cache.kv_heads) <= 8 ? 8 : 16;
}

}  // namespace

size_t cache_attention_workspace(const CacheAttentionArgs& a) {
  cudaError_t ce;
  const DeviceInfo* di = current_device_info(&ce);
  const size_t sms = di ? di->sm_count : 148;
  if (a.max_length <= kBlockKeys) return 0;  // one block per item: nothing is cut
  const size_t row = (a.cache.dim + 2) * sizeof(float);
  const size_t few = kNotesBytes + 2 * kFewCtasPerSm * sms * few_rows_of(a) * row;
  const bool many = static_cast<unsigned long long>(a.max_new) * (a.heads / a.cache.kv_heads) > kFewRows;
  // the two kernels run one after the other and share it
  return many ? std::max(few, kNotesBytes + 2 * sms * kManyRows * row) : few;
}

int cache_attention(const CacheAttentionArgs& args) {
  cudaError_t ce;
  const DeviceInfo* di = current_device_info(&ce);
  if (!di) return static_cast<int>(ce);
  if (di->cc_major != 10) return TFCCB200_EUNSUPPORTED;
  CacheAttention a = {};
  a.c = cache_params(args.cache);
  a.q = args.q; a.out = args.out; a.ldq = args.ldq; a.ldo = args.ldo;
  a.heads = args.heads; a.group = args.heads / args.cache.kv_heads;
  a.c.max_new = args.max_new;
  a.c.max_length = args.max_length;
  a.causal = args.causal;
  a.scale = args.scale * 1.4426950408889634f;
  a.scratch = args.max_length > kBlockKeys ? static_cast<float*>(args.workspace) : nullptr;
  const bool wide = args.cache.dim == 128;
  int st = TFCCB200_OK;
  // Whether a sequence has few rows or many is device data.  Where max_new says that there may be both
  // kinds, both kernels are launched, unless all blocks together are so few (7 per SM, the bound over all
  // sequences) that the second kernel and its merge cost more than the many-rows kernel loses on the others.  Measured
  // with 4 to 32 sequences of 1 to 24 new tokens, and with one chunk among single tokens: up to 7 blocks per SM
  // 10 to 37 us in one kernel and 22 to 62 in two; they meet at 20 to 40 blocks per SM at dim 64 and at 50 or more at
  // dim 128, so that the rule errs on the side of two kernels.
  const bool only_few = static_cast<unsigned long long>(args.max_new) * a.group <= kFewRows;
  const bool only_many = a.group > kFewRows || (!only_few && few_units_bound(args) * 14 <= 100ull * di->sm_count);
  if (!only_many) {
    a.min_rows = 1;
    a.max_rows = kFewRows;
    if (few_rows_of(args) == 8)
      st = wide ? launch_few<128, 8>(args, a, di->sm_count) : launch_few<64, 8>(args, a, di->sm_count);
    else
      st = wide ? launch_few<128, 16>(args, a, di->sm_count) : launch_few<64, 16>(args, a, di->sm_count);
    if (st != TFCCB200_OK) return st;
  }
  if (!only_few) {
    a.min_rows = only_many ? 1 : kFewRows + 1;
    a.max_rows = 0xffffffffu;
    st = cache_attention_many(args, a, di->sm_count);
  }
  return st;
}

}  // namespace tfccb200

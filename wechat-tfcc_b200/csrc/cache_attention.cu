// Attention of new tokens over the paged 8-bit cache: the kernel for few rows, and the choice
// between it and the one for many (cache_attention_many.cu).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   k_j = ks_j kc_j, v_j = vs_j vc_j (s8 codes)
//
// with j over the cached tokens that token i sees: all of them, or (causal) those at positions up
// to its own.  A row that sees nothing is 0.
//
// Arithmetic (both kernels).  A code is exact in fp16, so nothing is lost by handing K and V to
// the tensor cores as fp16.  The fp32 operands are split into two fp16 terms, x = hi + lo with 11
// bits each: q per row after scaling by a power of two, and the weights w_j = p_j vs_j, which carry
// the value scales, after scaling by a power of two that bounds them.  Two products with fp32 sums
// instead of one then give 22 bits, and the key scales are applied to the scores in fp32.  The softmax is
// the one-pass form: running maximum and sum in fp32, sums rescaled when the maximum grows.
#include <cuda_runtime.h>

#include <algorithm>

#include "cache_attention.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "ptx.cuh"

namespace tfccb200 {

namespace {

// ---- few rows: memory-bound ----------------------------------------------------------------------
//
// Up to 8 (or 16) rows of a kv head against its whole cache: every code is used for a handful
// of products, so what counts is streaming the cache.  A warp works alone: it brings 16 keys and their values
// at a time through its own ring of cp.async stages (no CTA barrier in the loop) and multiplies with
// mma.sync m16n8k16, whose operand fragments can be read straight from the rows as they lie
// because the order of k is free: a lane's 16 bytes of a key row serve as its k slots of
// successive steps.  With 8 rows the 16 rows of the instruction hold their hi and lo terms side by side.
// Eight warps take the eight 16-key groups of a 128-key block and are added at the item's end.
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;

template <int DIM, int ROWS>
struct FewLayout {
  static constexpr int kStages = DIM == 128 ? 3 : 6;
  static constexpr int kCodeBytes = 16 * DIM;               // codes of 16 keys (or values)
  static constexpr int kStageBytes = 2 * kCodeBytes + 128;  // + their scales
  static constexpr int kRingBytes = kStages * kStageBytes;  // per warp
  static constexpr int kFragBytes = (ROWS / 8) * (DIM / 16) * 32 * 16;
  static constexpr int kSmall = kFragBytes + kFewWarps * kRingBytes;
  static constexpr int kSmem = kSmall + (kFewWarps * 2 * ROWS + kFewWarps) * 4;
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

__device__ __forceinline__ void mma_f16(float (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
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

constexpr float kWeightTop = 16384.f;        // weights are scaled to at most 2^14: fp16 keeps 22 bits of
                                             // them down to 2^-17 of the largest
constexpr float kValueFloor = 7.8886091e-31f;  // 2^-100

template <int DIM, int ROWS>
__global__ void __launch_bounds__(kFewThreads, 2) cache_attention_few_kernel(const __grid_constant__ CacheAttention a) {
  using L = FewLayout<DIM, ROWS>;
  constexpr int kSteps = DIM / 16;   // k-steps of a score
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
  float* red_v = red_l + kFewWarps * ROWS;  // [warp]

  unsigned long long mine;
  const unsigned long long units = all_units<ROWS, kFewThreads>(a, &sched, &mine);
  const unsigned long long u0 = range_begin(units, a.grid, blockIdx.x);
  const unsigned long long u1 = range_begin(units, a.grid, blockIdx.x + 1);
  if (u0 == u1) return;
  find_unit<ROWS, kFewThreads>(a, u0, mine, &sched);

  for (ItemWalk<ROWS> item(a, u1 - u0, &sched); !item.done(); item.next()) {
    const unsigned rows = static_cast<unsigned>(item.seq.count) * a.group;
    const int length = item.seq.length, past = length - item.seq.count;
    const unsigned head = item.head;
    const int b = item.b;

    // ---- the warp's loads: 16 keys of block `blk` into stage `st` ----
    auto load = [&](unsigned blk, int st) {
      const int key0 = static_cast<int>(blk * kBlockKeys + warp * 16);
      const int pos = key0 + static_cast<int>(lane & 15u);
      const bool live = pos < length;
      const int page = live ? page_of(a.c, b, pos) : -1;
      const uint32_t dst = ring_addr + st * L::kStageBytes;
      {  // scales: lanes 0-15 of the keys, 16-31 of the values
        const uint32_t d = dst + 2 * L::kCodeBytes + lane * 4;
        if (page >= 0) {
          const size_t at = cache_slot(a.c, page, head, pos);
          cp_async_4(d, (lane < 16 ? a.c.key_scales : a.c.value_scales) + at);
        } else {  // a page that does not exist shows as NaN (a place behind the end is masked anyway)
          *reinterpret_cast<uint32_t*>(ring + (d - ring_addr)) = 0x7fffffffu;
        }
      }
      constexpr int kChunks = DIM / 16;  // 16-byte chunks of a row
      constexpr int kPer = 16 * kChunks / 32;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const unsigned r = (i * 32 + lane) / kChunks, c = lane % kChunks;
        const int pg = __shfl_sync(0xffffffffu, page, r);
        const size_t at = (pg >= 0 ? cache_slot(a.c, pg, head, key0 + r) : 0) * DIM + c * 16;
        cp_async_16(dst + key_chunk<DIM>(r, c), a.c.keys + at, pg >= 0);
        cp_async_16(dst + L::kCodeBytes + value_chunk<DIM>(r, c), a.c.values + at, pg >= 0);
      }
    };
    auto has_keys = [&](unsigned blk) {  // warp-uniform
      return blk < item.hi && static_cast<int>(blk * kBlockKeys + warp * 16) < length;
    };
#pragma unroll
    for (int s = 0; s < L::kStages - 1; ++s) {
      if (has_keys(item.lo + s)) load(item.lo + s, s);
      cp_async_commit();
    }

    // ---- query fragments: hi and lo terms of the rows, scaled by a power of two per row ----
    // Lane (g, t) holds row g's (and, 16 rows, row g + 8's) values d = 64 [step >= 4] + 16 t +
    // 4 (step & 3) + 0..3 as the k slots 2t, 2t+1, 2t+8, 2t+9 of k-step `step`.
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
      float4 f[kSteps];
      uint32_t m = 0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        f[s] = live ? *reinterpret_cast<const float4*>(src + (s >> 2) * 64 + 16 * t + 4 * (s & 3))
                    : make_float4(0.f, 0.f, 0.f, 0.f);
        f[s].x *= a.scale; f[s].y *= a.scale; f[s].z *= a.scale; f[s].w *= a.scale;
        m = max(m, max(max(__float_as_uint(f[s].x) & 0x7fffffffu, __float_as_uint(f[s].y) & 0x7fffffffu),
                       max(__float_as_uint(f[s].z) & 0x7fffffffu, __float_as_uint(f[s].w) & 0x7fffffffu)));
      }
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // 2^(10 - exponent): the row's largest value lands in [2^10, 2^11).  Zero and tiny rows (below
      // 2^-100) take the bound of the range, a non-finite row 1 (it becomes NaN in any case).
      const int ex = static_cast<int>(m >> 23) - 127;
      const int sh = ex == 128 ? 0 : 10 - max(ex, -100);
      const float up = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
      row_scale[h] = __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s % kFewWarps != static_cast<int>(warp) % kSteps) continue;
        const float x = f[s].x * up, y = f[s].y * up, z = f[s].z * up, w = f[s].w * up;
        const uint32_t h0 = pack_half2(x, y), h1 = pack_half2(z, w);
        const uint32_t l0 = pack_rest(x, y, h0), l1 = pack_rest(z, w, h1);
        if constexpr (ROWS == 8) {
          frag[s * 32 + lane] = make_uint4(h0, l0, h1, l1);
        } else {
          uint32_t* hi = reinterpret_cast<uint32_t*>(frag + s * 32 + lane);
          uint32_t* lo = reinterpret_cast<uint32_t*>(frag + (kSteps + s) * 32 + lane);
          hi[h] = h0; hi[2 + h] = h1;
          lo[h] = l0; lo[2 + h] = l1;
        }
      }
    }
    __syncthreads();

    float o[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float top[ROWS / 8], sum[ROWS / 8], vref = kValueFloor;
#pragma unroll
    for (int h = 0; h < ROWS / 8; ++h) top[h] = -INFINITY, sum[h] = 0.f;

    int st = 0;
    for (unsigned blk = item.lo; blk < item.hi; ++blk) {
      if (!has_keys(blk)) break;  // nor do later blocks have any for this warp
      cp_async_wait<L::kStages - 2>();
      __syncwarp();
      const uint8_t* stage = ring + st * L::kStageBytes;
      {
        const unsigned ahead = blk + L::kStages - 1;
        if (has_keys(ahead)) load(ahead, st == 0 ? L::kStages - 1 : st - 1);
        cp_async_commit();
      }
      if (++st == L::kStages) st = 0;

      // scores of keys 0-7 and 8-15 of the group
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < DIM / 64; ++c) {
        const uint4 ka = *reinterpret_cast<const uint4*>(stage + key_chunk<DIM>(g, c * 4 + t));
        const uint4 kb = *reinterpret_cast<const uint4*>(stage + key_chunk<DIM>(g + 8, c * 4 + t));
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t ua = wa[w] ^ 0x80808080u, ub = wb[w] ^ 0x80808080u;
          const uint32_t a0 = codes_low(ua), a1 = codes_high(ua), b0 = codes_low(ub), b1 = codes_high(ub);
          const uint4 q = frag[(c * 4 + w) * 32 + lane];
          mma_f16(s0, q, a0, a1);
          mma_f16(s1, q, b0, b1);
          if constexpr (ROWS == 16) {
            const uint4 ql = frag[(kSteps + c * 4 + w) * 32 + lane];
            mma_f16(s0, ql, a0, a1);
            mma_f16(s1, ql, b0, b1);
          }
        }
      }
      // lane (g, t): keys 2t, 2t+1, 2t+8, 2t+9 of rows g (and g + 8)
      const float* ks = reinterpret_cast<const float*>(stage + 2 * L::kCodeBytes);
      const float2 ka = *reinterpret_cast<const float2*>(ks + 2 * t), kb = *reinterpret_cast<const float2*>(ks + 2 * t + 8);
      const float2 va = *reinterpret_cast<const float2*>(ks + 16 + 2 * t), vb = *reinterpret_cast<const float2*>(ks + 24 + 2 * t);
      const int key0 = static_cast<int>(blk * kBlockKeys + warp * 16 + 2 * t);
      const float kscale[4] = {ka.x, ka.y, kb.x, kb.y}, vscale[4] = {va.x, va.y, vb.x, vb.y};
      float x[ROWS / 8][4];
      if constexpr (ROWS == 8) {
        x[0][0] = s0[0] + s0[2]; x[0][1] = s0[1] + s0[3]; x[0][2] = s1[0] + s1[2]; x[0][3] = s1[1] + s1[3];
      } else {
        x[0][0] = s0[0]; x[0][1] = s0[1]; x[0][2] = s1[0]; x[0][3] = s1[1];
        x[1][0] = s0[2]; x[1][1] = s0[3]; x[1][2] = s1[2]; x[1][3] = s1[3];
      }
      bool grows = false;
      float next_top[ROWS / 8];
#pragma unroll
      for (int h = 0; h < ROWS / 8; ++h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + (j & 1) + (j >> 1) * 8;
          x[h][j] = key < sees[h] ? x[h][j] * (kscale[j] * row_scale[h]) : -INFINITY;
        }
        float m = fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        next_top[h] = fmaxf(top[h], m);
        grows |= next_top[h] > top[h];
      }
      // largest value scale of the group, rounded up to a power of two
      float vmax = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + (j & 1) + (j >> 1) * 8;
        if (key < length) vmax = fmaxf(vmax, fabsf(vscale[j]));
      }
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
      grows |= vmax > vref;
      if (__any_sync(0xffffffffu, grows)) {
        float vnext = vref;
        if (vmax > vref) vnext = __uint_as_float(min((__float_as_uint(vmax) + 0x7fffffu) & 0x7f800000u, 0x7f000000u));
        const float vf = vref / vnext;
        vref = vnext;
#pragma unroll
        for (int h = 0; h < ROWS / 8; ++h) {
          const float f = exp2_fast(top[h] - (next_top[h] == -INFINITY ? 0.f : next_top[h]));
          sum[h] *= f;
          top[h] = next_top[h];
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            o[i][2 * h] *= f * vf;
            o[i][2 * h + 1] *= f * vf;
            if constexpr (ROWS == 8) {
              o[i][2] *= f * vf;
              o[i][3] *= f * vf;
            }
          }
        }
      }
      const float vup = kWeightTop / vref;
      uint32_t hi[ROWS / 8][2], lo[ROWS / 8][2];
#pragma unroll
      for (int h = 0; h < ROWS / 8; ++h) {
        const float base = top[h] == -INFINITY ? 0.f : top[h];
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + (j & 1) + (j >> 1) * 8;
          const float p = exp2_fast(x[h][j] - base);
          sum[h] += p;
          w[j] = key < sees[h] ? p * (vscale[j] * vup) : 0.f;  // (0 * NaN behind the end would be NaN)
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
          mma_f16(o[w * 4 + i], pa, x0[i], x1[i]);
          if constexpr (ROWS == 16) mma_f16(o[w * 4 + i], pb, x0[i], x1[i]);
        }
      }
      __syncwarp();  // the stage may be overwritten
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
      }
    }
    if (lane == 0) red_v[warp] = vref;
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
            for (int k = 0; k < 4; ++k) yy[k] = ROWS == 8 ? o[i + k][c] + o[i + k][2 + c] : o[i + k][2 * h + c];
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
        const float fv = f * (red_v[w] * (1.f / kWeightTop));
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
}

// ---- host ----------------------------------------------------------------------------------------

constexpr unsigned kFewCtasPerSm = 2;

// Largest number of units a launch of these bounds can have.
unsigned long long few_units_bound(const CacheAttentionArgs& a) {
  return static_cast<unsigned long long>(a.cache.batch) * a.cache.kv_heads *
         ((a.max_length + kBlockKeys - 1) / kBlockKeys);
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
    e = launch_after_previous(cache_attention_merge_kernel<DIM, ROWS>, dim3(a.grid - 1), dim3(256), 0,
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
  const size_t few = 2 * kFewCtasPerSm * sms * few_rows_of(a) * row;
  const bool many = static_cast<unsigned long long>(a.max_new) * (a.heads / a.cache.kv_heads) > kFewRows;
  // the two kernels run one after the other and share it
  return many ? std::max(few, 2 * sms * kManyRows * row) : few;
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
  if (args.max_new < a.c.max_new) a.c.max_new = args.max_new;
  if (args.max_length < a.c.max_length) a.c.max_length = args.max_length;
  a.causal = args.causal;
  a.scale = args.scale * 1.4426950408889634f;
  a.scratch = static_cast<float*>(args.workspace);
  const bool wide = args.cache.dim == 128;
  int st = TFCCB200_OK;
  if (a.group <= kFewRows) {
    a.min_rows = 1;
    a.max_rows = kFewRows;
    if (few_rows_of(args) == 8)
      st = wide ? launch_few<128, 8>(args, a, di->sm_count) : launch_few<64, 8>(args, a, di->sm_count);
    else
      st = wide ? launch_few<128, 16>(args, a, di->sm_count) : launch_few<64, 16>(args, a, di->sm_count);
    if (st != TFCCB200_OK) return st;
  }
  if (static_cast<unsigned long long>(args.max_new) * a.group > kFewRows) {
    a.min_rows = kFewRows + 1;
    a.max_rows = 0xffffffffu;
    st = cache_attention_many(args, a, di->sm_count);
  }
  return st;
}

}  // namespace tfccb200

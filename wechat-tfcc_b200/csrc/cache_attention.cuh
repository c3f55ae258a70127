// What the two attention kernels over the paged 8-bit cache share beside the schedule: fp16 terms of fp32
// values, codes as fp16, and the kernel that joins the pieces of cut items.
#pragma once

#include <atomic>

#include "cache_schedule.cuh"
#include "pdl.cuh"

namespace tfccb200 {

constexpr int kManyRows = 128;  // rows of an item of the many-rows kernel

// Two floats as packed fp16 (first in the low half), and what the rounding left over.
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float half_low(uint32_t h) {
  float f;
  asm("{.reg .f16 l, u; mov.b32 {l, u}, %1; cvt.f32.f16 %0, l;}" : "=f"(f) : "r"(h));
  return f;
}
__device__ __forceinline__ float half_high(uint32_t h) {
  float f;
  asm("{.reg .f16 l, u; mov.b32 {l, u}, %1; cvt.f32.f16 %0, u;}" : "=f"(f) : "r"(h));
  return f;
}
// Pairs of floats in the packed fp32 instructions of this architecture (one issue slot for two).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 r = unpair(fma2(pair(half_low(hi), half_high(hi)), pair(-1.f, -1.f), pair(a, b)));
  return pack_half2(r.x, r.y);
}

// Codes (biased to unsigned by an exclusive or with 0x80) to fp16: the byte becomes the low mantissa
// bits of 1024 + u, from which 1152 is taken.
__device__ __forceinline__ uint32_t unbias(uint32_t h) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ uint32_t codes_low(uint32_t u) { return unbias(__byte_perm(u, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t codes_high(uint32_t u) { return unbias(__byte_perm(u, 0x64646464u, 0x4342)); }

// ---- the pieces of cut items ---------------------------------------------------------------------
//
// One CTA (or several, blockIdx.y sharing out the elements) per range of the attention kernel that began an item
// without ending it: the item's pieces are added in key order.
template <int DIM, int ROWS>
static __global__ void __launch_bounds__(256) cache_attention_merge_kernel(const __grid_constant__ CacheAttention a) {
  pdl_release();
  pdl_wait();
  const unsigned c = blockIdx.x;
  const PieceNote note = *piece_note(a, c);
  const unsigned more = note.ranges;  // pieces after the first
  if (more == 0) return;
  constexpr size_t kPitch = 2 * piece_floats<ROWS, DIM>();  // from one range's slot to the next one's
  const float* const p1 = piece<ROWS, DIM>(a, c, true);     // the piece that begins with the item
  const float* const p0 = piece<ROWS, DIM>(a, c, false) + kPitch;
  for (unsigned e = (blockIdx.y * 256 + threadIdx.x) * 4; e < ROWS * DIM; e += gridDim.y * 1024) {
    const unsigned r = e / DIM, d = e % DIM, row = note.tile * ROWS + r;
    if (row >= note.rows) continue;
    const float m1 = p1[r];
    float m = m1;
#pragma unroll 8
    for (unsigned k = 0; k < more; ++k) m = fmaxf(m, p0[k * kPitch + r]);
    const float base = m == -INFINITY ? 0.f : m;
    float f = exp2_fast(m1 - base);
    float l = f * p1[ROWS + r];
    const float4 y1 = *reinterpret_cast<const float4*>(p1 + 2 * ROWS + e);
    float4 acc = make_float4(f * y1.x, f * y1.y, f * y1.z, f * y1.w);
#pragma unroll 8
    for (unsigned k = 0; k < more; ++k) {
      const float* p = p0 + k * kPitch;
      const float4 y = *reinterpret_cast<const float4*>(p + 2 * ROWS + e);
      f = exp2_fast(p[r] - base);
      l = fmaf(f, p[ROWS + r], l);
      acc.x = fmaf(f, y.x, acc.x); acc.y = fmaf(f, y.y, acc.y);
      acc.z = fmaf(f, y.z, acc.z); acc.w = fmaf(f, y.w, acc.w);
    }
    const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
    const unsigned tok = row / a.group;
    float* dst = a.out + a.ldo * (static_cast<size_t>(note.first) + tok) +
                 (static_cast<size_t>(note.head) * a.group + row % a.group) * DIM + d;
    *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
}

template <class K>
inline int opt_in_smem(K kernel, int bytes, std::atomic<unsigned long long>& configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured.fetch_or(bit, std::memory_order_release);
  }
  return TFCCB200_OK;
}

// Sequences with more than kFewRows rows per kv head (cache_attention_many.cu).
int cache_attention_many(const CacheAttentionArgs& args, CacheAttention a, int sm_count);

}  // namespace tfccb200

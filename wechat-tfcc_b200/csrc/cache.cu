// The paged 8-bit cache: quantizing new keys and values as they are written, and reading tokens
// back as floats.
//
// Both are one pass over memory: a token's kv head is dim floats in and dim + 4 bytes out (or the
// reverse).  Four lanes' worth of 16-byte words make 64 floats, so a vector of 64 takes half a
// warp and one of 128 a whole warp, and its maximum stays in registers and shuffles.  A warp takes
// one row (the sequence and page are looked up once for it) and walks the row's 2 * kv_heads
// vectors, four per step with all their loads requested before the first is used; append asks for its first
// values before it looks up where they go.  Bound by memory once there are rows enough: 16384 tokens of 8 x 128
// read back in 30 us (5.5 TB/s), written in 41 us (4.1 TB/s; 51 us with the look-up first): append asks for a
// warp's next four vectors when the present ones have been quantized, into the same registers, and has no load in
// flight meanwhile.
#include <cuda_runtime.h>

#include "cache.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "token_quant.cuh"

namespace tfccb200 {

namespace {

constexpr int kThreads = 256;

struct CacheRows {  // the float side: row r of k at k + r * ldk, kv_heads * dim values
  float* k;
  float* v;
  unsigned long long ldk, ldv;
};

template <int DIM>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const CacheParams p, const CacheRows x) {
  constexpr int kLanes = DIM / 4;  // lanes of one vector
  constexpr int kPer = 32 / kLanes;  // vectors a warp takes side by side
  pdl_release();
  pdl_wait();
  check_all_sequences(p);
  const unsigned lane = threadIdx.x & 31u, sub = lane / kLanes, l = lane % kLanes;
  const unsigned row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const unsigned vectors = 2 * p.kv_heads;
  constexpr int kUnroll = 4;
  float4 f[kUnroll];
  auto load = [&](unsigned v0) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned i = v0 + u * kPer + sub, head = i >> 1;
      f[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < vectors) {
        const float* src = (i & 1u) ? x.v + x.ldv * row : x.k + x.ldk * row;
        f[u] = __ldcs(reinterpret_cast<const float4*>(src + head * DIM) + l);
      }
    }
  };
  // the values do not depend on where they go: their loads run while the place is looked up
  unsigned v0 = blockIdx.y * kUnroll * kPer;
  load(v0);
  const int b = sequence_of_row(p, row);
  if (b < 0) return;
  const DeviceSequence seq = load_sequence(p, b);
  if (!seq.ok) return;
  const int pos = seq.length - seq.count + (static_cast<int>(row) - seq.first);
  if (pos < 0) return;
  const int page = page_of(p, b, pos);
  if (page < 0) return;
  while (true) {
    uint32_t c[kUnroll];
    float scale[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t m = max_abs_bits(0u, f[u]);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const TokenQuant q(m);
      c[u] = q.codes4(f[u]);
      scale[u] = q.scale;
    }
    const unsigned at0 = v0;
    v0 += gridDim.y * kUnroll * kPer;
    if (v0 < vectors) load(v0);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned i = at0 + u * kPer + sub, head = i >> 1;
      if (i < vectors) {
        const size_t at = cache_slot(p, page, head, pos);
        reinterpret_cast<uint32_t*>(((i & 1u) ? p.values : p.keys) + at * DIM)[l] = c[u];
        if (l == 0) ((i & 1u) ? p.value_scales : p.key_scales)[at] = scale[u];
      }
    }
    if (v0 >= vectors) break;
  }
}

template <int DIM>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const CacheParams p, const CacheRows x) {
  constexpr int kLanes = DIM / 4;
  constexpr int kPer = 32 / kLanes;
  pdl_release();
  pdl_wait();
  check_all_sequences(p);
  const unsigned lane = threadIdx.x & 31u, sub = lane / kLanes, l = lane % kLanes;
  const unsigned row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int b = sequence_of_row(p, row);
  if (b < 0) return;
  const DeviceSequence seq = load_sequence(p, b);
  if (!seq.ok) return;
  const int pos = seq.length - seq.count + (static_cast<int>(row) - seq.first);
  const int page = pos < 0 ? -1 : page_of(p, b, pos);
  const unsigned vectors = 2 * p.kv_heads;
  constexpr int kUnroll = 4;
  for (unsigned v0 = blockIdx.y * kUnroll * kPer; v0 < vectors; v0 += gridDim.y * kUnroll * kPer) {
    uint32_t c[kUnroll];
    float s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned i = v0 + u * kPer + sub, head = i >> 1;
      c[u] = 0u;
      s[u] = 0.f;
      if (i < vectors && page >= 0) {
        const size_t at = cache_slot(p, page, head, pos);
        c[u] = __ldcs(reinterpret_cast<const uint32_t*>(((i & 1u) ? p.values : p.keys) + at * DIM) + l);
        s[u] = ((i & 1u) ? p.value_scales : p.key_scales)[at];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned i = v0 + u * kPer + sub, head = i >> 1;
      if (i < vectors) {
        float4 f;
        f.x = static_cast<float>(static_cast<int8_t>(c[u])) * s[u];
        f.y = static_cast<float>(static_cast<int8_t>(c[u] >> 8)) * s[u];
        f.z = static_cast<float>(static_cast<int8_t>(c[u] >> 16)) * s[u];
        f.w = static_cast<float>(static_cast<int8_t>(c[u] >> 24)) * s[u];
        float* dst = (i & 1u) ? x.v + x.ldv * row : x.k + x.ldk * row;
        __stcs(reinterpret_cast<float4*>(dst + head * DIM) + l, f);
      }
    }
  }
}

CacheParams params_of(const CacheArgs& a) {
  CacheParams p = {};
  p.keys = a.keys; p.key_scales = a.key_scales;
  p.values = a.values; p.value_scales = a.value_scales;
  p.pages = a.pages; p.kv_heads = a.kv_heads; p.dim = a.dim;
  while ((1u << p.page_shift) < a.page_size) ++p.page_shift;
  p.starts = a.starts; p.lengths = a.lengths; p.table = a.table;
  p.batch = a.batch; p.table_width = a.table_width; p.rows = a.rows;
  p.max_new = a.rows;
  p.max_length = a.table_width * a.page_size;
  p.status = a.status;
  return p;
}

template <class K>
int launch_rows(const CacheArgs& a, K kernel, const CacheRows& x) {
  cudaError_t ce;
  const DeviceInfo* di = current_device_info(&ce);
  if (!di) return static_cast<int>(ce);
  const unsigned blocks = (a.rows + kThreads / 32 - 1) / (kThreads / 32);
  // Few rows: their vectors are spread over blockIdx.y as well, so that more SMs take part.
  const unsigned steps = (2 * a.kv_heads * a.dim / 128 + 3) / 4;
  unsigned y = blocks < 2u * di->sm_count ? steps : 1u;
  cudaError_t e = launch_after_previous(kernel, dim3(blocks, y), dim3(kThreads), 0, a.stream, params_of(a), x);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  return TFCCB200_OK;
}

}  // namespace

CacheParams cache_params(const CacheArgs& a) { return params_of(a); }

int cache_append(const CacheArgs& a, const float* k, unsigned long long ldk, const float* v,
                 unsigned long long ldv) {
  const CacheRows x{const_cast<float*>(k), const_cast<float*>(v), ldk, ldv};
  return a.dim == 128 ? launch_rows(a, cache_append_kernel<128>, x) : launch_rows(a, cache_append_kernel<64>, x);
}

int cache_read(const CacheArgs& a, float* k, unsigned long long ldk, float* v, unsigned long long ldv) {
  const CacheRows x{k, v, ldk, ldv};
  return a.dim == 128 ? launch_rows(a, cache_read_kernel<128>, x) : launch_rows(a, cache_read_kernel<64>, x);
}

}  // namespace tfccb200

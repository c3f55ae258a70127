// The 8-bit linear layer's CUDA-core kernels: quantizing activations with one scale per token,
// and the product for operands the tensor-core path cannot take.
#include <cuda_runtime.h>

#include "act.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "token_quant.cuh"

namespace tfccb200 {

namespace {

// One pass over x: THREADS threads share a row, each holding up to kHold 16-byte words of it in
// registers between the maximum and the codes, so that the row is read from memory once; a row
// longer than 4 * kHold * THREADS values is read a second time (from L2) for its tail.
// The exact rounding costs about 15 instructions a value, which 5 bytes of traffic leave time for.
template <int THREADS>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS)
quantize_tokens_kernel(const float* __restrict__ src, unsigned long long ld_src, unsigned rows, unsigned cols,
                       int8_t* __restrict__ codes, unsigned long long ld_codes, float* __restrict__ scales,
                       bool vec) {
  constexpr int kHold = 4;
  constexpr int kBlock = THREADS < 128 ? 128 : THREADS;
  __shared__ uint32_t sh[kBlock / 32];
  pdl_release();
  pdl_wait();
  const unsigned t = threadIdx.x % THREADS;
  const unsigned long long row = static_cast<unsigned long long>(blockIdx.x) * (kBlock / THREADS) + threadIdx.x / THREADS;
  const bool live = row < rows;
  const float* p = src + (live ? row : 0) * ld_src;
  int8_t* out = codes + (live ? row : 0) * ld_codes;
  float4 held[kHold];
  uint32_t m = 0;
  const unsigned words = vec ? cols / 4 : 0;
  if (live) {
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      const unsigned i = t + u * THREADS;
      held[u] = i < words ? __ldcs(reinterpret_cast<const float4*>(p) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kHold; ++u) m = max_abs_bits(m, held[u]);
    for (unsigned i = t + kHold * THREADS; i < words; i += THREADS)
      m = max_abs_bits(m, reinterpret_cast<const float4*>(p)[i]);
    for (unsigned i = words * 4 + t; i < cols; i += THREADS) m = max(m, abs_bits(p[i]));
  }
  if constexpr (THREADS >= 32) {
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (THREADS > 32) {
      if ((threadIdx.x & 31u) == 0) sh[threadIdx.x >> 5] = m;
      __syncthreads();
      const unsigned w0 = threadIdx.x / THREADS * (THREADS / 32);
      m = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) m = max(m, sh[w0 + w]);
    }
  }
  if (!live) return;
  const TokenQuant q(m);
  if (t == 0) scales[row] = q.scale;
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const unsigned i = t + u * THREADS;
    if (i < words) reinterpret_cast<uint32_t*>(out)[i] = q.codes4(held[u]);
  }
  for (unsigned i = t + kHold * THREADS; i < words; i += THREADS)
    reinterpret_cast<uint32_t*>(out)[i] = q.codes4(reinterpret_cast<const float4*>(p)[i]);
  for (unsigned i = words * 4 + t; i < cols; i += THREADS) out[i] = static_cast<int8_t>(q.code(p[i]));
}

// Any pitch, any alignment: 64 x 64 results per CTA, 4 x 4 per thread, int32 sums.
__global__ void __launch_bounds__(256) s8_gemm_simt_kernel(const S8GemmArgs a) {
  constexpr int T = 64, KB = 32;
  __shared__ int8_t sa[KB][T + 4], sb[KB][T + 4];
  pdl_release();
  pdl_wait();
  const unsigned m0 = blockIdx.y * T, n0 = blockIdx.x * T;
  const unsigned tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (unsigned k0 = 0; k0 < a.K; k0 += KB) {
    for (unsigned i = threadIdx.x; i < KB * T; i += 256) {
      const unsigned ka = i % KB, ma = i / KB, kb = i / T, nb = i % T;
      sa[ka][ma] = (k0 + ka < a.K && m0 + ma < a.M) ? a.A[(m0 + ma) * a.lda + k0 + ka] : int8_t(0);
      sb[kb][nb] = (k0 + kb < a.K && n0 + nb < a.N) ? a.B[(k0 + kb) * a.ldb + n0 + nb] : int8_t(0);
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < KB; ++k) {
      int x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = sa[k][ty * 4 + i], y[i] = sb[k][tx * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += x[i] * y[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned m = m0 + ty * 4 + i;
    if (m >= a.M) continue;
    const float s = a.a_scales[m];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned n = n0 + tx * 4 + j;
      if (n >= a.N) continue;
      float y = static_cast<float>(acc[i][j]) * s * a.b_scales[n];
      if (a.bias) y += a.bias[n];
      a.C[static_cast<size_t>(m) * a.N + n] = apply_activation(y, a.activation);
    }
  }
}

}  // namespace

int quantize_tokens(cudaStream_t stream, const float* src, unsigned long long ld_src, unsigned rows, unsigned cols,
                    int8_t* codes, unsigned long long ld_codes, float* scales) {
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 && ld_src % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(codes) & 3u) == 0 && ld_codes % 4 == 0;
  cudaError_t e;
  if (cols <= 512)
    e = launch_after_previous(quantize_tokens_kernel<32>, dim3((rows + 3) / 4), dim3(128), 0, stream, src, ld_src,
                              rows, cols, codes, ld_codes, scales, vec);
  else if (cols <= 2048)
    e = launch_after_previous(quantize_tokens_kernel<128>, dim3(rows), dim3(128), 0, stream, src, ld_src, rows, cols,
                              codes, ld_codes, scales, vec);
  else
    e = launch_after_previous(quantize_tokens_kernel<512>, dim3(rows), dim3(512), 0, stream, src, ld_src, rows, cols,
                              codes, ld_codes, scales, vec);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  return TFCCB200_OK;
}

int simt_s8_gemm(const S8GemmArgs& a) {
  const dim3 grid((a.N + 63) / 64, (a.M + 63) / 64);
  if (grid.y > 65535u) return TFCCB200_EUNSUPPORTED;
  cudaError_t e = launch_after_previous(s8_gemm_simt_kernel, grid, dim3(256), 0, a.stream, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  return TFCCB200_OK;
}

}  // namespace tfccb200

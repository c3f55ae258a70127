// The 8-bit linear layer's CUDA-core kernels: quantizing activations with one scale per token,
// and the product for operands the tensor-core path cannot take.
#include <cuda_runtime.h>

#include "act.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "ptx.cuh"
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

// ---- few tokens: memory-bound on the weights ------------------------------------------------------
//
// Up to 16 tokens against W [K, N]: a CTA takes 128 columns and a share of K, its eight warps deal the
// share out in steps of 32 rows.  A lane reads 16 bytes of each of 8 rows straight into
// registers (whole 128-byte lines per row over the warp, two steps in flight); a byte transposition
// turns four rows into mma.sync m16n8k32 operands, whose columns may come in any order: lane group g
// holds columns 16 g .. 16 g + 15, column j of each for the j-th product.  With the tokens as rows the
// products cost 16 instructions per 4 KB of weights.  The int32 sums of the warps meet in shared memory and
// those of a K split in the shared memory of a thread-block cluster; integer sums are exact in any order.
// The tcgen05 kernel pads 16 tokens to 128 rows and leaves its epilogue to one warp per tile
// (16x4096x16384 with GELU: 43 us).
constexpr int kFewThreads = 256;
constexpr int kFewCols = 128;
constexpr int kFewPitch = kFewCols + 12;  // ints per token in shared memory: rows start 12 banks apart

struct FewStep {
  uint4 w[8];     // rows 4 t + i and (from 4 on) 16 + 4 t + i of the step, 16 columns
  uint32_t a[4];  // codes of tokens g and g + 8 in the product's operand order
};

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four words of four rows -> four words of four columns.
__device__ __forceinline__ void transpose4(const uint32_t (&r)[4], uint32_t (&c)[4]) {
  const uint32_t x0 = __byte_perm(r[0], r[1], 0x5140), x1 = __byte_perm(r[0], r[1], 0x7362);
  const uint32_t y0 = __byte_perm(r[2], r[3], 0x5140), y1 = __byte_perm(r[2], r[3], 0x7362);
  c[0] = __byte_perm(x0, y0, 0x5410);
  c[1] = __byte_perm(x0, y0, 0x7632);
  c[2] = __byte_perm(x1, y1, 0x5410);
  c[3] = __byte_perm(x1, y1, 0x7632);
}

__global__ void __launch_bounds__(kFewThreads, 1) s8_few_kernel(const __grid_constant__ S8GemmArgs a, unsigned splits) {
  __shared__ int sums[16 * kFewPitch];
  pdl_release();
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
  const unsigned rank = blockIdx.x % splits;
  const unsigned col0 = blockIdx.x / splits * kFewCols;
  const unsigned steps = (a.K + 31) / 32, per = (steps + splits - 1) / splits;
  const unsigned first = rank * per, last = min(steps, first + per);  // this CTA's steps
  for (unsigned i = tid; i < 16 * kFewPitch; i += kFewThreads) sums[i] = 0;
  pdl_wait();

  const unsigned col = col0 + 16 * g;
  const int8_t* const wp = a.B + col;
  const int cols = static_cast<int>(a.N) - static_cast<int>(col);  // of the lane's 16 columns, those that exist
  auto load = [&](unsigned step, FewStep& f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned k = step * 32 + (i >> 2) * 16 + 4 * t + (i & 3);
      f.w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (k < a.K && cols > 0) {
        const int8_t* p = wp + k * a.ldb;
        if (cols >= 16) {
          asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(f.w[i].x), "=r"(f.w[i].y), "=r"(f.w[i].z), "=r"(f.w[i].w)
                       : "l"(p));
        } else {  // the ragged end: only what exists is touched
          uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (4 * q + 4 <= cols) {
              v[q] = __ldg(reinterpret_cast<const uint32_t*>(p) + q);
            } else {
#pragma unroll
              for (int e = 0; e < 3; ++e)
                if (4 * q + e < cols) v[q] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(p + 4 * q + e))) << (8 * e);
            }
          }
          f.w[i] = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned m = g + (i & 1) * 8, k = step * 32 + (i >> 1) * 16 + 4 * t;
      const int8_t* p = a.A + m * a.lda + k;
      f.a[i] = 0u;
      if (m < a.M) {
        if (k + 4 <= a.K) {
          f.a[i] = __ldg(reinterpret_cast<const uint32_t*>(p));
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (k + e < a.K) f.a[i] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(p + e))) << (8 * e);
        }
      }
    }
  };
  int acc[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0;
  auto use = [&](const FewStep& f) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t r0[4] = {(&f.w[0].x)[q], (&f.w[1].x)[q], (&f.w[2].x)[q], (&f.w[3].x)[q]};
      const uint32_t r1[4] = {(&f.w[4].x)[q], (&f.w[5].x)[q], (&f.w[6].x)[q], (&f.w[7].x)[q]};
      uint32_t c0[4], c1[4];
      transpose4(r0, c0);
      transpose4(r1, c1);
#pragma unroll
      for (int e = 0; e < 4; ++e) mma_s8(acc[4 * q + e], f.a, c0[e], c1[e]);
    }
  };
  {
    FewStep f0, f1;
    unsigned s = first + warp;
    if (s < last) load(s, f0);
    for (; s < last; s += 16) {
      if (s + 8 < last) load(s + 8, f1);
      use(f0);
      if (s + 16 < last) load(s + 16, f0);
      if (s + 8 < last) use(f1);
    }
  }
  __syncthreads();
  // column 16 n + j of the tile lies at place 8 j + n
  if (first + warp < last) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) atomicAdd(&sums[(g + (i >> 1) * 8) * kFewPitch + 8 * j + 2 * t + (i & 1)], acc[j][i]);
  }
  __syncthreads();
  if (splits > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  // every CTA of the cluster finishes its share of the tokens' columns
  const unsigned share = kFewCols / splits;  // a power of two
  const unsigned rows = min(a.M, 16u);
  const uint32_t base = ptx::smem_u32(sums);
  for (unsigned e = tid; e < rows * share; e += kFewThreads) {
    const unsigned m = e / share, c = rank * share + e % share, n = col0 + c;
    const unsigned at = m * kFewPitch + 8 * (c & 15u) + (c >> 4);
    int v = sums[at];
    for (unsigned r = 1; r < splits; ++r) {
      int o;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(o) : "r"(ptx::mapa(base + 4 * at, (rank + r) % splits)) : "memory");
      v += o;
    }
    if (n < a.N) {
      float y = static_cast<float>(v) * __ldg(a.a_scales + m);
      y = fmaf(y, __ldg(a.b_scales + n), a.bias ? __ldg(a.bias + n) : 0.f);
      a.C[static_cast<size_t>(m) * a.N + n] = apply_activation(y, a.activation);
    }
  }
  if (splits > 1) {  // nobody leaves while its sums may be read
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
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

bool few_s8_gemm_supported(const S8GemmArgs& a) {
  return a.M <= 16 && a.lda % 16 == 0 && a.ldb % 16 == 0 && (reinterpret_cast<uintptr_t>(a.A) & 15u) == 0 &&
         (reinterpret_cast<uintptr_t>(a.B) & 15u) == 0;
}

int few_s8_gemm(const S8GemmArgs& a) {
  cudaError_t ce;
  const DeviceInfo* di = current_device_info(&ce);
  if (!di) return static_cast<int>(ce);
  const unsigned tiles = (a.N + kFewCols - 1) / kFewCols, steps = (a.K + 31) / 32;
  // One CTA per SM: K is split while the CTAs still fit and every warp keeps a step of its own.
  unsigned splits = 1;
  while (splits < 8 && tiles * splits * 2 <= static_cast<unsigned>(di->sm_count) && steps >= splits * 2 * 8) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * splits);
  cfg.blockDim = dim3(kFewThreads);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, s8_few_kernel, a, splits);
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

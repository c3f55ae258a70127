// The 8-bit linear layer's CUDA-core kernels: quantizing activations with one scale per token,
// and the product for operands the tensor-core path cannot take.
#include <cuda_runtime.h>

#include <atomic>

#include "act.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "ptx.cuh"
#include "token_quant.cuh"

namespace tfccb200 {

namespace {

// One pass over x: THREADS threads share a row, each holding up to kHold 16-byte words of it (or, rows
// that do not start on 16 bytes, 4 * kHold single values) in registers between the maximum and the codes, so
// that the row is read from memory once; what is left of a row longer than 4 * kHold * THREADS values
// is read a second time, from L2.  A thread count per row is chosen by the row's length so that up to 4096
// values are held and several rows share an SM: 4096 x 4096 takes 14 us (5.9 TB/s of the 5 bytes a value) with
// 256 threads a row and 27 with 512; 8192 x 8192 64 us (5.2 TB/s).  Few rows are bound by latency (1.5 us).
template <int THREADS, bool kVec>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS)
quantize_tokens_kernel(const float* src, unsigned long long ld_src, unsigned rows, unsigned cols,
                       int8_t* codes, unsigned long long ld_codes, float* scales) {
  constexpr int kHold = 4;
  constexpr int kBlock = THREADS < 128 ? 128 : THREADS;
  __shared__ uint32_t sh[kBlock / 32];
  // In this order: once the next kernel may start, everything before this one is complete, and the
  // product that follows can begin with its weights (S8GemmArgs::early_weights).
  pdl_wait();
  pdl_release();
  const unsigned t = threadIdx.x % THREADS;
  const unsigned long long row = static_cast<unsigned long long>(blockIdx.x) * (kBlock / THREADS) + threadIdx.x / THREADS;
  const bool live = row < rows;
  const float* p = src + (live ? row : 0) * ld_src;
  int8_t* out = codes + (live ? row : 0) * ld_codes;
  // unit i of the row: 4 values (kVec) or 1
  const unsigned units = !live ? 0 : (kVec ? cols / 4 : cols);
  constexpr int kUnits = kVec ? kHold : 4 * kHold;
  float4 held[kHold];
  uint32_t m = 0;
  if constexpr (kVec) {
#pragma unroll
    for (int u = 0; u < kHold; ++u)
      held[u] = t + u * THREADS < units ? __ldcs(reinterpret_cast<const float4*>(p) + t + u * THREADS)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) (&held[u / 4].x)[u % 4] = t + u * THREADS < units ? __ldcs(p + t + u * THREADS) : 0.f;
  }
#pragma unroll
  for (int u = 0; u < kHold; ++u) m = max_abs_bits(m, held[u]);
  for (unsigned i = t + kUnits * THREADS; i < units; i += THREADS) {
    if constexpr (kVec) m = max_abs_bits(m, reinterpret_cast<const float4*>(p)[i]);
    else m = max(m, abs_bits(p[i]));
  }
  if (kVec && live && cols / 4 * 4 + t < cols) m = max(m, abs_bits(p[cols / 4 * 4 + t]));
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
  if constexpr (kVec) {
#pragma unroll
    for (int u = 0; u < kHold; ++u)
      if (t + u * THREADS < units) reinterpret_cast<uint32_t*>(out)[t + u * THREADS] = q.codes4(held[u]);
    for (unsigned i = t + kUnits * THREADS; i < units; i += THREADS)
      reinterpret_cast<uint32_t*>(out)[i] = q.codes4(reinterpret_cast<const float4*>(p)[i]);
    if (cols / 4 * 4 + t < cols) out[cols / 4 * 4 + t] = static_cast<int8_t>(q.code(p[cols / 4 * 4 + t]));
  } else {
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      const uint32_t c = q.codes4(held[u]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t + (4 * u + e) * THREADS < units) out[t + (4 * u + e) * THREADS] = static_cast<int8_t>(c >> (8 * e));
    }
    for (unsigned i = t + kUnits * THREADS; i < units; i += THREADS) out[i] = static_cast<int8_t>(q.code(p[i]));
  }
}

// ---- few tokens: memory-bound on the weights ------------------------------------------------------
//
// Up to 16 tokens against W [K, N]: a CTA takes 128 columns and a share of K, its eight warps deal the
// share out in steps of 32 rows.  Each warp brings its steps (32 x 128 weights, 16 x 32 codes)
// through a cp.async ring of its own, five stages deep: about 180 KB in flight per SM, which the
// latency of memory asks for, without holding registers.  A lane reads 16 bytes of each of 8 rows; a byte
// transposition turns four rows into mma.sync m16n8k32 operands, whose columns may come in any
// order: lane group g holds columns 16 g .. 16 g + 15, column j of each for the j-th product.  With
// the tokens as rows the products cost 16 instructions per 4 KB of weights.  The int32 sums of the warps
// meet in shared memory and those of a K split in the shared memory of a thread-block cluster;
// integer sums are exact in any order.  16x4096x16384 with GELU, weights from memory: 16.4 us, 4.1 TB/s.  The
// tcgen05 kernel, which pads 16 tokens to 128 rows and leaves its epilogue to one warp per tile, takes 22.8; over
// 4096 -> 11008, 4096 -> 16384 and 5120 -> 20480 it takes 21 to 37 us for 16 tokens and this one 15 to 34, which is why
// this one goes up to the 16 rows of its product.  (Two steps held in registers instead of the ring: 21 us for
// the first case; six stages no faster.)  What it leaves: whole 128-column tiles, and K split by powers of two only
// while all CTAs fit, keep 128 of 148 SMs busy at N = 16384 (K in one piece) and 86 at 11008; at 20480 there are
// 160 CTAs, two waves.
constexpr int kFewThreads = 256;
constexpr int kFewCols = 128;
constexpr int kFewPitch = kFewCols + 12;  // ints per token in shared memory: rows start 12 banks apart
constexpr int kFewStages = 5;
constexpr int kFewStageBytes = 32 * kFewCols + 16 * 32;
constexpr int kFewSmem = 8 * kFewStages * kFewStageBytes + 16 * kFewPitch * 4;

// 16 bytes of which the first `live` exist (the rest arrives as zeros).
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live) : "memory");
}

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

__global__ void __launch_bounds__(kFewThreads, 1)
s8_few_kernel(const __grid_constant__ S8GemmArgs a, unsigned splits) {
  extern __shared__ __align__(128) uint8_t few_smem[];
  int* const sums = reinterpret_cast<int*>(few_smem + 8 * kFewStages * kFewStageBytes);
  pdl_release();
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
  const unsigned rank = blockIdx.x % splits;
  const unsigned col0 = blockIdx.x / splits * kFewCols;
  const unsigned steps = (a.K + 31) / 32, per = (steps + splits - 1) / splits;
  const unsigned first = min(steps, rank * per), last = min(steps, first + per);  // this CTA's steps
  const uint8_t* const ring = few_smem + warp * kFewStages * kFewStageBytes;
  const uint32_t ring_addr = ptx::smem_u32(ring);

  // 16-byte chunk c of row r of a step lies at chunk c ^ (r / 4 % 4 * 2): the four rows and two chunks
  // that a quarter of a warp reads together then differ in their banks.
  auto load_weights = [&](unsigned step, unsigned st) {
    const unsigned c = lane & 7u, col = col0 + c * 16;
    const int live = min(16, max(0, static_cast<int>(a.N) - static_cast<int>(col)));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned r = i * 4 + (lane >> 3), k = step * 32 + r;
      const bool in = k < a.K && live > 0;
      cp_async_16(ring_addr + st * kFewStageBytes + r * kFewCols + ((c ^ ((r >> 1) & 6u)) << 4),
                  in ? a.B + k * a.ldb + col : a.B, in ? live : 0);
    }
  };
  auto load_codes = [&](unsigned step, unsigned st) {
    const unsigned m = lane >> 1, k = step * 32 + (lane & 1u) * 16;
    const int live = m < a.M ? min(16, max(0, static_cast<int>(a.K) - static_cast<int>(k))) : 0;
    cp_async_16(ring_addr + st * kFewStageBytes + 32 * kFewCols + lane * 16, live > 0 ? a.A + m * a.lda + k : a.A, live);
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // What comes before the wait for the kernel ahead may only read what that kernel does not write
  // and what was complete when that kernel began: see S8GemmArgs::early_weights.
  if (a.early_weights)
    for (unsigned s = 0; s < kFewStages - 1; ++s)
      if (first + warp + 8 * s < last) load_weights(first + warp + 8 * s, s);
  for (unsigned i = tid; i < 16 * kFewPitch; i += kFewThreads) sums[i] = 0;
  pdl_wait();
  for (unsigned s = 0; s < kFewStages - 1; ++s) {
    if (first + warp + 8 * s < last) {
      if (!a.early_weights) load_weights(first + warp + 8 * s, s);
      load_codes(first + warp + 8 * s, s);
    }
    commit();
  }

  int acc[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0;
  unsigned st = 0;
  for (unsigned s = first + warp; s < last; s += 8) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
    __syncwarp();
    const uint8_t* const stage = ring + st * kFewStageBytes;
    {
      const unsigned ahead = s + 8 * (kFewStages - 1), into = st == 0 ? kFewStages - 1 : st - 1;
      if (ahead < last) {
        load_weights(ahead, into);
        load_codes(ahead, into);
      }
      commit();
    }
    if (++st == kFewStages) st = 0;
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // tokens g, g + 8, k = 4 t and 16 + 4 t
      f[i] = *reinterpret_cast<const uint32_t*>(stage + 32 * kFewCols + (g + (i & 1) * 8) * 32 + (i >> 1) * 16 + 4 * t);
    uint4 w[8];  // rows 4 t + i and (from 4 on) 16 + 4 t + i
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned r = (i >> 2) * 16 + 4 * t + (i & 3);
      w[i] = *reinterpret_cast<const uint4*>(stage + r * kFewCols + ((g ^ ((r >> 1) & 6u)) << 4));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t r0[4] = {(&w[0].x)[q], (&w[1].x)[q], (&w[2].x)[q], (&w[3].x)[q]};
      const uint32_t r1[4] = {(&w[4].x)[q], (&w[5].x)[q], (&w[6].x)[q], (&w[7].x)[q]};
      uint32_t c0[4], c1[4];
      transpose4(r0, c0);
      transpose4(r1, c1);
#pragma unroll
      for (int e = 0; e < 4; ++e) mma_s8(acc[4 * q + e], f, c0[e], c1[e]);
    }
    __syncwarp();  // the stage may be overwritten
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
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
      float y = static_cast<float>(v) * a.a_scales[m];
      y = fmaf(y, a.b_scales[n], a.bias ? a.bias[n] : 0.f);
      a.C[static_cast<size_t>(m) * a.N + n] = apply_activation(y, a.activation);
    }
  }
  if (splits > 1) {  // nobody leaves while its sums may be read
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
}

// Any pitch, any alignment: 64 x 64 results per CTA, 4 x 4 per thread, int32 sums.  Tiles along one grid dimension, so
// that neither M nor N meets the bound of the others.
__global__ void __launch_bounds__(256) s8_gemm_simt_kernel(const S8GemmArgs a) {
  constexpr int T = 64, KB = 32;
  __shared__ int8_t sa[KB][T + 4], sb[KB][T + 4];
  pdl_release();
  pdl_wait();
  const unsigned across = (a.N - 1) / T + 1;
  const unsigned m0 = blockIdx.x / across * T, n0 = blockIdx.x % across * T;
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
  auto run = [&](auto kernel, unsigned rows_per_block, unsigned threads) {
    return launch_after_previous(kernel, dim3((rows + rows_per_block - 1) / rows_per_block), dim3(threads), 0, stream,
                                 src, ld_src, rows, cols, codes, ld_codes, scales);
  };
  cudaError_t e;
  if (cols <= 512) e = vec ? run(quantize_tokens_kernel<32, true>, 4, 128) : run(quantize_tokens_kernel<32, false>, 4, 128);
  else if (cols <= 2048) e = vec ? run(quantize_tokens_kernel<128, true>, 1, 128) : run(quantize_tokens_kernel<128, false>, 1, 128);
  else if (cols <= 4096) e = vec ? run(quantize_tokens_kernel<256, true>, 1, 256) : run(quantize_tokens_kernel<256, false>, 1, 256);
  else e = vec ? run(quantize_tokens_kernel<512, true>, 1, 512) : run(quantize_tokens_kernel<512, false>, 1, 512);
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
  static std::atomic<unsigned long long> configured{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(s8_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured.fetch_or(bit, std::memory_order_release);
  }
  // One CTA per SM: K is split while the CTAs still fit and every warp keeps a step of its own.
  unsigned splits = 1;
  while (splits < 8 && tiles * splits * 2 <= static_cast<unsigned>(di->sm_count) && steps >= splits * 2 * 8) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * splits);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = kFewSmem;
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
  e = cudaLaunchKernelEx(&cfg, s8_few_kernel, a, splits);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  return TFCCB200_OK;
}

int simt_s8_gemm(const S8GemmArgs& a) {
  // (M * N fits 32 bits, M and N 31: fewer than 2^27 tiles)
  const dim3 grid(((a.N - 1) / 64 + 1) * ((a.M - 1) / 64 + 1));
  cudaError_t e = launch_after_previous(s8_gemm_simt_kernel, grid, dim3(256), 0, a.stream, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  return TFCCB200_OK;
}

}  // namespace tfccb200

// Attention of new tokens over the paged 8-bit cache.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   k_j = ks_j kc_j, v_j = vs_j vc_j (s8 codes)
//
// with j over the cached tokens that token i sees: all of them, or (causal) those at positions up
// to its own.  A row that sees nothing is 0.
#include <cuda_runtime.h>

#include "cache.cuh"
#include "internal.h"
#include "pdl.cuh"

namespace tfccb200 {

namespace {

struct CacheAttention {
  CacheParams c;
  const float* q;
  float* out;
  unsigned long long ldq, ldo;
  unsigned heads, group;  // group = heads / kv_heads
  int causal;
  float scale;  // times log2(e)
};

// One (row, head) per CTA, keys dealt to its warps one by one, a running maximum and sum per warp.
template <int DIM>
__global__ void __launch_bounds__(128) cache_attention_simple_kernel(const CacheAttention a) {
  constexpr int kPer = DIM / 32;
  __shared__ float sh_m[4], sh_l[4], sh_o[4][DIM];
  pdl_release();
  pdl_wait();
  check_all_sequences(a.c);
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const unsigned row = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int b = sequence_of_row(a.c, row);
  if (b < 0) return;
  const DeviceSequence seq = load_sequence(a.c, b);
  if (!seq.ok) return;
  int sees = seq.length;
  if (a.causal) sees = seq.length - seq.count + (static_cast<int>(row) - seq.first) + 1;
  const float* q = a.q + a.ldq * row + head * DIM + lane * kPer;
  float qr[kPer], o[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) qr[i] = q[i] * a.scale, o[i] = 0.f;
  for (int j = warp; j < sees; j += 4) {
    const int page = page_of(a.c, b, j);
    float s = 0.f, vs = __uint_as_float(0x7fffffffu), v[kPer];
    if (page >= 0) {
      const size_t at = cache_slot(a.c, page, head / a.group, j);
#pragma unroll
      for (int i = 0; i < kPer; ++i) s += qr[i] * static_cast<float>(a.c.keys[at * DIM + lane * kPer + i]);
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = static_cast<float>(a.c.values[at * DIM + lane * kPer + i]);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= a.c.key_scales[at];
      vs = a.c.value_scales[at];
    } else {
      s = vs;
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = 0.f;
    }
    const float m2 = fmaxf(m, s), al = m == -INFINITY ? 0.f : exp2f(m - m2), pr = exp2f(s - m2);
    l = l * al + pr;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * al + pr * vs * v[i];
    m = m2;
  }
  if (lane == 0) sh_m[warp] = m, sh_l[warp] = l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sh_o[warp][lane * kPer + i] = o[i];
  __syncthreads();
  if (threadIdx.x < DIM) {
    const float top = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
    float sum = 0.f, acc = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = sh_l[w] == 0.f ? 0.f : exp2f(sh_m[w] - top);
      sum += f * sh_l[w];
      acc += f * sh_o[w][threadIdx.x];
    }
    a.out[a.ldo * row + head * DIM + threadIdx.x] = sees <= 0 ? 0.f : acc / sum;
  }
}

}  // namespace

size_t cache_attention_workspace(const CacheAttentionArgs&) { return 0; }

int cache_attention(const CacheAttentionArgs& a) {
  cudaError_t ce;
  const DeviceInfo* di = current_device_info(&ce);
  if (!di) return static_cast<int>(ce);
  CacheAttention p = {};
  p.c = cache_params(a.cache);
  p.q = a.q; p.out = a.out; p.ldq = a.ldq; p.ldo = a.ldo;
  p.heads = a.heads; p.group = a.heads / a.cache.kv_heads;
  p.c.max_new = a.max_new < p.c.max_new ? a.max_new : p.c.max_new;
  p.c.max_length = a.max_length < p.c.max_length ? a.max_length : p.c.max_length;
  p.causal = a.causal;
  p.scale = a.scale * 1.4426950408889634f;
  const dim3 grid(a.cache.rows * a.heads);
  cudaError_t e = a.cache.dim == 128
      ? launch_after_previous(cache_attention_simple_kernel<128>, grid, dim3(128), 0, a.cache.stream, p)
      : launch_after_previous(cache_attention_simple_kernel<64>, grid, dim3(128), 0, a.cache.stream, p);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  return TFCCB200_OK;
}

}  // namespace tfccb200

// Attention over the paged 8-bit cache for many rows per kv head: chunks of prompts, tcgen05.
//
// An item is 256 query rows of one kv head (two halves of 128, the rows of one MMA) against a run
// of 128-key blocks.  Arithmetic as in cache_attention.cu: K, V exact in fp16, Q and the weights as two
// fp16 terms each, so per block and half
//   S = Q_hi K^T + Q_lo K^T          A and B from shared memory, 128 x 128 fp32 in tensor memory
//   P = exp2(S ks - m) vs            by one thread per row; hi and lo terms go back over S
//   O_block = P_hi V + P_lo V        A from tensor memory, V as it lies (MN-major)
//   O = O alpha + O_block            fp32 registers
// The tensor core's accumulator narrows without rounding to nearest, which would bias O over
// thousands of keys; summed from zero per block and added to registers it does not, and a block's own power
// of two for the value scales comes along for nothing.
//
// Roles (512 threads, registers shifted with setmaxnreg):
//   warp 0      issues the MMAs: PV of one half, then S of its next block, so that the other half's
//               softmax runs while the tensor core is busy
//   warp 1      loads the blocks' scales
//   warp 2      walks the schedule and hands the items to the others
//   warps 4-7   turn codes into fp16 operand tiles (global -> registers -> shared memory): the tiles
//               of K and V share a ring, one row's 64 values per 128-byte swizzled line
//   warps 8-11  softmax, sums and output of half 0; warps 12-15 of half 1
// Bound by the tensor core: 8 dim flops per (row, key) pair instead of the 4 counted, and its
// operand reads from shared memory; the softmax's instructions come next.
//
// Every wait is bounded: on expiry a status bit is raised and all roles run to their end.
#include <cuda_runtime.h>

#include "cache_attention.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "ptx.cuh"

namespace tfccb200 {

namespace {

constexpr int kThreads = 512;
constexpr int kTileBytes = 128 * 128;  // 128 rows x 64 fp16, 128-byte swizzle
constexpr int kRegsControl = 56, kRegsConvert = 88, kRegsSoftmax = 184;
static_assert(kRegsControl + kRegsConvert + 2 * kRegsSoftmax == 512, "shares of 128 registers per thread at launch");

constexpr float kWeightTop = 1024.f;  // weights reach at most 2^10 times 2^kLazy, inside fp16's range
constexpr float kLazy = 5.f;          // the maximum moves only when it grows by more (log2 units)
constexpr float kValueFloor = 7.8886091e-31f;  // 2^-100

struct Item {  // what the roles need to know of an item; hi == 0 ends the walk
  int first, count, length, b;
  unsigned head, tile, lo, hi;
  unsigned whole, rows;
  unsigned pad[2];
};

template <int DIM>
struct ManyLayout {
  static constexpr int kHalves = DIM / 64;               // 64-wide tiles of a row
  static constexpr int kOperand = kHalves * kTileBytes;  // 128 rows of Q_hi, Q_lo, K or V
  static constexpr int kRing = DIM == 128 ? 3 : 6;
  static constexpr int kQ = 0;                           // [half][hi, lo]
  static constexpr int kKv = 4 * kOperand;
  static constexpr int kScales = kKv + kRing * kOperand;  // 2 x {ks[128], vr[128]}
  static constexpr int kItems = kScales + 2 * 1024;
  static constexpr int kBars = kItems + 2 * static_cast<int>(sizeof(Item));
  static constexpr int kMisc = kBars + 8 * 32;            // tensor memory address, abort flag, value factors
  static constexpr int kSched = kMisc + 16;
  static constexpr int kSmem = kSched + static_cast<int>(sizeof(ScheduleShared));
  static_assert(kSmem <= 232448, "shared memory");
};

struct Waiter {
  volatile uint32_t* abort_flag;
  int* status;
  unsigned long long timeout_ns;
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity, int bit) const {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    uint64_t start = 0;
    uint32_t spins = 0;
    while (true) {
      if (ptx::mbar_try_wait(bar, parity)) return true;
      if ((++spins & 0xFF) == 0) {
        if (*abort_flag) return false;
        const uint64_t now = ptx::globaltimer_ns();
        if (start == 0) {
          start = now;
        } else if (now - start > timeout_ns) {
          *abort_flag = 1;
          raise_status(status, bit);
          return false;
        }
      }
    }
  }
};

template <int DIM>
__global__ void __launch_bounds__(kThreads, 1)
cache_attention_many_kernel(const __grid_constant__ CacheAttention a, unsigned long long timeout_ns) {
  using L = ManyLayout<DIM>;
  constexpr int kSteps = DIM / 16;  // k-steps of S
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_release();
  const uint32_t base = ptx::smem_u32(smem);
  if (base & 1023u) {  // (the swizzled tiles start the window, which does begin on 1024 bytes)
    if (threadIdx.x == 0) raise_status(a.c.status, TFCCB200_DEV_TIMEOUT_MMA);
    return;
  }
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  auto bar = [&](int i) { return base + L::kBars + 8u * i; };
  const uint32_t q_full = bar(0), s_full = bar(2), p_full = bar(4), o_full = bar(6);  // one per half
  const uint32_t sc_full = bar(8), sc_empty = bar(10), it_full = bar(12), it_empty = bar(14);  // two stages
  const uint32_t kv_full = bar(16), kv_empty = bar(16 + L::kRing);
  static_assert(16 + 2 * L::kRing <= 32, "barriers");
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem + L::kMisc);
  volatile uint32_t* abort_flag = misc + 1;
  volatile float* value_back = reinterpret_cast<volatile float*>(misc + 2);  // per scale stage
  const Item* items = reinterpret_cast<const Item*>(smem + L::kItems);
  ScheduleShared* sched = reinterpret_cast<ScheduleShared*>(smem + L::kSched);
  const Waiter wait{abort_flag, a.c.status, timeout_ns};

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(q_full + 8 * i, 4);
      ptx::mbar_init(s_full + 8 * i, 1);
      ptx::mbar_init(p_full + 8 * i, 4);
      ptx::mbar_init(o_full + 8 * i, 1);
      ptx::mbar_init(sc_full + 8 * i, 1);
      ptx::mbar_init(sc_empty + 8 * i, 8);
      ptx::mbar_init(it_full + 8 * i, 1);
      ptx::mbar_init(it_empty + 8 * i, 14);  // warps 0, 1, 4-15
    }
    for (int i = 0; i < L::kRing; ++i) {
      ptx::mbar_init(kv_full + 8 * i, 4);
      ptx::mbar_init(kv_empty + 8 * i, 1);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc<1>(base + L::kMisc, 512);  // S of both halves, O of both halves
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = misc[0];
  pdl_wait();

  unsigned long long mine;
  const unsigned long long units = all_units<kManyRows, kThreads>(a, sched, &mine);
  const unsigned long long u0 = range_begin(units, a.grid, blockIdx.x);
  const unsigned long long u1 = range_begin(units, a.grid, blockIdx.x + 1);
  if (u0 < u1) find_unit<kManyRows, kThreads>(a, u0, mine, sched);

  // Hands every item to `body`; the stage is released when body has returned (and has therefore
  // read what it needs).
  auto for_items = [&](auto&& body) {
    for (unsigned n = 0;; ++n) {
      const unsigned s = n & 1u;
      if (!wait(it_full + 8 * s, (n >> 1) & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return;
      const Item it = items[s];
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(it_empty + 8 * s);
      if (it.hi == 0) return;
      if (!body(it)) return;
    }
  };
  auto second_half = [](const Item& it) { return it.rows > it.tile * kManyRows + 128; };

  if (warp < 4) {
    ptx::setmaxnreg_dec<kRegsControl>();
    if (warp == 0) {
      // ======================= MMA issuer =======================
      uint32_t kv_n = 0;             // ring buffers consumed
      uint32_t nq0 = 0, nq1 = 0, np0 = 0, np1 = 0;  // phases per half
      constexpr uint32_t idesc_s = ptx::make_idesc(1u, 0u, 0u, 0u, 0u, 128u, 128u);
      constexpr uint32_t idesc_o = ptx::make_idesc(1u, 0u, 0u, 0u, 1u, 128u, static_cast<uint32_t>(DIM));
      for_items([&](const Item& it) {
        const int halves = second_half(it) ? 2 : 1;
        const unsigned blocks = it.hi - it.lo;
        auto kv_wait = [&](uint32_t n) {
          return wait(kv_full + 8 * (n % L::kRing), (n / L::kRing) & 1u, TFCCB200_DEV_TIMEOUT_MMA);
        };
        auto tile = [&](uint32_t n) { return base + L::kKv + (n % L::kRing) * L::kOperand; };
        auto score = [&](int h, uint32_t n) {
          if (lane == 0) {
            const uint32_t k = tile(n);
#pragma unroll
            for (int part = 1; part >= 0; --part) {  // the small terms first
              const uint32_t q = base + L::kQ + (2 * h + part) * L::kOperand;
#pragma unroll
              for (int s = 0; s < kSteps; ++s) {
                const uint32_t off = (s >> 2) * kTileBytes + (s & 3) * 32;
                ptx::umma<ptx::MmaKind::BF16, 1>(tmem + h * 128, ptx::smem_desc(q + off, 16, 1024, ptx::kLayoutSw128),
                                                 ptx::smem_desc(k + off, 16, 1024, ptx::kLayoutSw128), idesc_s,
                                                 (part == 1 && s == 0) ? 0u : 1u);
              }
            }
            ptx::umma_commit<1>(s_full + 8 * h, 0);
          }
          __syncwarp();
        };
        auto weigh = [&](int h, uint32_t n) {
          if (lane == 0) {
            const uint32_t v = tile(n);
#pragma unroll
            for (int part = 1; part >= 0; --part)
#pragma unroll
              for (int s = 0; s < 8; ++s)
                ptx::umma_f16_ts(tmem + 256 + h * 128, tmem + h * 128 + (s >> 1) * 32 + (s & 1) * 8 + part * 16,
                                 ptx::smem_desc(v + s * 2048, kTileBytes, 1024, ptx::kLayoutSw128), idesc_o,
                                 (part == 1 && s == 0) ? 0u : 1u);
            ptx::umma_commit<1>(o_full + 8 * h, 0);
          }
          __syncwarp();
        };
        auto release = [&](uint32_t n) {
          if (lane == 0) ptx::umma_commit<1>(kv_empty + 8 * (n % L::kRing), 0);
          __syncwarp();
        };
        if (!wait(q_full, nq0++ & 1u, TFCCB200_DEV_TIMEOUT_MMA)) return false;
        if (!kv_wait(kv_n)) return false;
        ptx::tc_fence_after_sync();
        score(0, kv_n);
        if (halves == 2) {
          if (!wait(q_full + 8, nq1++ & 1u, TFCCB200_DEV_TIMEOUT_MMA)) return false;
          ptx::tc_fence_after_sync();
          score(1, kv_n);
        }
        release(kv_n);
        for (unsigned j = 0; j < blocks; ++j) {
          const uint32_t v = kv_n + 1, k = kv_n + 2;
          const bool more = j + 1 < blocks;
          for (int h = 0; h < halves; ++h) {
            if (!wait(p_full + 8 * h, (h ? np1++ : np0++) & 1u, TFCCB200_DEV_TIMEOUT_MMA)) return false;
            if (h == 0 && !kv_wait(v)) return false;
            ptx::tc_fence_after_sync();
            weigh(h, v);
            if (h == halves - 1) release(v);
            // S of the half's next block goes over the weights that the products just issued read:
            // one thread's MMAs run in the order of issue
            if (more) {
              if (h == 0 && !kv_wait(k)) return false;
              ptx::tc_fence_after_sync();
              score(h, k);
              if (h == halves - 1) release(k);
            }
          }
          kv_n += more ? 2 : 1;
        }
        kv_n += 1;
        return true;
      });
    } else if (warp == 1) {
      // ======================= scales =======================
      uint32_t n = 0;
      for_items([&](const Item& it) {
        for (unsigned blk = it.lo; blk < it.hi; ++blk, ++n) {
          const uint32_t s = n & 1u;
          float ks[4], vs[4];
          uint32_t top = __float_as_uint(kValueFloor);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = static_cast<int>(blk * kBlockKeys + i * 32 + lane);
            ks[i] = vs[i] = 0.f;
            if (pos < it.length) {
              const int page = page_of(a.c, it.b, pos);
              if (page >= 0) {
                const size_t at = cache_slot(a.c, page, it.head, pos);
                ks[i] = __ldg(a.c.key_scales + at);
                vs[i] = __ldg(a.c.value_scales + at);
              } else {  // a page that does not exist shows as NaN
                ks[i] = vs[i] = __uint_as_float(0x7fffffffu);
              }
            }
            const uint32_t bits = __float_as_uint(vs[i]) & 0x7fffffffu;
            if (bits < 0x7f800000u) top = max(top, bits);
          }
          top = __reduce_max_sync(0xffffffffu, top);
          top = min((top + 0x7fffffu) & 0x7f800000u, 0x7f000000u);  // up to a power of two
          const float up = kWeightTop / __uint_as_float(top);
          if (!wait(sc_empty + 8 * s, ((n >> 1) & 1u) ^ 1u, TFCCB200_DEV_TIMEOUT_CONVERT)) return false;
          float* dst = reinterpret_cast<float*>(smem + L::kScales + s * 1024);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dst[i * 32 + lane] = ks[i];
            dst[128 + i * 32 + lane] = vs[i] * up;
          }
          if (lane == 0) value_back[s] = __uint_as_float(top) * (1.f / kWeightTop);
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sc_full + 8 * s);
        }
        return true;
      });
    } else if (warp == 2) {
      // ======================= walker =======================
      unsigned n = 0;
      auto put = [&](const Item& it) {
        const unsigned s = n & 1u;
        if (!wait(it_empty + 8 * s, ((n >> 1) & 1u) ^ 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        if (lane == 0) {
          *reinterpret_cast<Item*>(smem + L::kItems + s * sizeof(Item)) = it;
          ptx::mbar_arrive(it_full + 8 * s);
        }
        __syncwarp();
        ++n;
        return true;
      };
      bool live = true;
      for (ItemWalk<kManyRows> w(a, u1 - u0, sched); live && !w.done(); w.next()) {
        Item it;
        it.first = w.seq.first; it.count = w.seq.count; it.length = w.seq.length; it.b = w.b;
        it.head = w.head; it.tile = w.tile; it.lo = w.lo; it.hi = w.hi;
        it.whole = w.whole() ? 1u : 0u;
        it.rows = static_cast<unsigned>(w.seq.count) * a.group;
        live = put(it);
      }
      Item end = {};
      if (live) put(end);
    }
  } else if (warp < 8) {
    // ======================= converters =======================
    ptx::setmaxnreg_dec<kRegsConvert>();
    constexpr int kLoads = 4 * L::kHalves;  // 16-byte chunks per thread and tile
    const unsigned cw = warp - 4, r8 = lane & 7u, c4 = lane >> 3;
    uint32_t n = 0;
    uint4 ahead[kLoads];
    int page = -1;  // of key 32 cw + lane of the block at hand
    for_items([&](const Item& it) {
      const unsigned tiles = 2 * (it.hi - it.lo);
      // tile i of the item: keys (even) or values (odd) of block lo + i / 2
      auto load = [&](unsigned i) {
        const unsigned key0 = (it.lo + (i >> 1)) * kBlockKeys + cw * 32;
        if ((i & 1u) == 0) {
          const unsigned pos = key0 + lane;
          page = static_cast<int>(pos) < it.length ? page_of(a.c, it.b, pos) : -1;
        }
        const int8_t* src = (i & 1u) ? a.c.values : a.c.keys;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const unsigned r = g * 8 + r8;
          const int pg = __shfl_sync(0xffffffffu, page, r);
          const uint4* p = reinterpret_cast<const uint4*>(src + (pg >= 0 ? cache_slot(a.c, pg, it.head, key0 + r) : 0) * DIM);
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            ahead[g * L::kHalves + h] = pg >= 0 ? __ldg(p + h * 4 + c4) : make_uint4(0u, 0u, 0u, 0u);
        }
      };
      load(0);
      for (unsigned i = 0; i < tiles; ++i, ++n) {
        const unsigned s = n % L::kRing;
        if (!wait(kv_empty + 8 * s, ((n / L::kRing) & 1u) ^ 1u, TFCCB200_DEV_TIMEOUT_CONVERT)) return false;
        uint8_t* dst = smem + L::kKv + s * L::kOperand;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const unsigned r = cw * 32 + g * 8 + r8;
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h) {
            const uint4 c = ahead[g * L::kHalves + h];
            const uint32_t x = c.x ^ 0x80808080u, y = c.y ^ 0x80808080u, z = c.z ^ 0x80808080u, w = c.w ^ 0x80808080u;
            uint8_t* row = dst + h * kTileBytes + r * 128;
            *reinterpret_cast<uint4*>(row + (((2 * c4) ^ r8) << 4)) =
                make_uint4(codes_low(x), codes_high(x), codes_low(y), codes_high(y));
            *reinterpret_cast<uint4*>(row + (((2 * c4 + 1) ^ r8) << 4)) =
                make_uint4(codes_low(z), codes_high(z), codes_low(w), codes_high(w));
          }
        }
        if (i + 1 < tiles) load(i + 1);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(kv_full + 8 * s);
      }
      return true;
    });
  } else {
    // ======================= softmax, sums, output =======================
    ptx::setmaxnreg_inc<kRegsSoftmax>();
    const int h = static_cast<int>(warp >> 2) - 2;
    const unsigned r = (warp & 3u) * 32 + lane;  // row of the half = lane of tensor memory
    const uint32_t lane_addr = tmem + (((warp & 3u) * 32) << 16);
    const uint32_t t_s = lane_addr + h * 128, t_o = lane_addr + 256 + h * 128;
    uint32_t ns = 0, nb = 0;  // blocks of this half, blocks of the CTA
    for_items([&](const Item& it) {
      const unsigned blocks = it.hi - it.lo;
      if (h == 1 && !second_half(it)) {  // nothing to do, but the scale stages count on every warp
        for (unsigned j = 0; j < blocks; ++j, ++nb) {
          if (!wait(sc_full + 8 * (nb & 1u), (nb >> 1) & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sc_empty + 8 * (nb & 1u));
        }
        return true;
      }
      const unsigned row = it.tile * kManyRows + h * 128 + r;
      const bool live = row < it.rows;
      const unsigned tok = live ? row / a.group : 0, hd = it.head * a.group + (live ? row % a.group : 0);
      const int past = it.length - it.count;
      const int sees = !live ? 0 : (a.causal ? past + static_cast<int>(tok) + 1 : it.length);
      // keys below this are seen by every row of the half
      const int all_see = a.causal ? past + static_cast<int>((it.tile * kManyRows + h * 128) / a.group) + 1 : it.length;

      // ---- the row of Q as two fp16 terms, scaled by a power of two ----
      float row_scale;
      {
        const float4* q = reinterpret_cast<const float4*>(
            a.q + a.ldq * (static_cast<size_t>(it.first) + tok) + static_cast<size_t>(hd) * DIM);
        uint32_t m = 0;
        if (live) {
#pragma unroll 8
          for (int i = 0; i < DIM / 4; ++i) {
            const float4 f = __ldg(q + i);
            m = max(m, max(max(__float_as_uint(f.x * a.scale) & 0x7fffffffu, __float_as_uint(f.y * a.scale) & 0x7fffffffu),
                           max(__float_as_uint(f.z * a.scale) & 0x7fffffffu, __float_as_uint(f.w * a.scale) & 0x7fffffffu)));
          }
        }
        // 2^(10 - exponent): the largest value lands in [2^10, 2^11); tiny rows take the bound of the
        // range, a non-finite row 1 (it becomes NaN in any case)
        const int ex = static_cast<int>(m >> 23) - 127;
        const int sh = ex == 128 ? 0 : 10 - max(ex, -100);
        const float up = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
        row_scale = __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
        uint8_t* hi = smem + L::kQ + 2 * h * L::kOperand + r * 128;
        uint8_t* lo = hi + L::kOperand;
#pragma unroll 4
        for (int u = 0; u < DIM / 8; ++u) {  // 16-byte units of the operand row
          float4 f = make_float4(0.f, 0.f, 0.f, 0.f), e = f;
          if (live) f = __ldg(q + 2 * u), e = __ldg(q + 2 * u + 1);
          // scaled in two steps, as the maximum was taken
          const float x[8] = {f.x * a.scale * up, f.y * a.scale * up, f.z * a.scale * up, f.w * a.scale * up,
                              e.x * a.scale * up, e.y * a.scale * up, e.z * a.scale * up, e.w * a.scale * up};
          const unsigned off = (u >> 3) * kTileBytes + (((u & 7u) ^ (r & 7u)) << 4);
          uint4 hh, ll;
          hh.x = pack_half2(x[0], x[1]); hh.y = pack_half2(x[2], x[3]); hh.z = pack_half2(x[4], x[5]); hh.w = pack_half2(x[6], x[7]);
          ll.x = pack_rest(x[0], x[1], hh.x); ll.y = pack_rest(x[2], x[3], hh.y);
          ll.z = pack_rest(x[4], x[5], hh.z); ll.w = pack_rest(x[6], x[7], hh.w);
          *reinterpret_cast<uint4*>(hi + off) = hh;
          *reinterpret_cast<uint4*>(lo + off) = ll;
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(q_full + 8 * h);
      }

      float o[DIM];
#pragma unroll
      for (int i = 0; i < DIM; ++i) o[i] = 0.f;
      float m = -INFINITY, l = 0.f, back = 0.f;
      // adds the finished block's products (accumulated in tensor memory from zero) to o
      auto drain = [&](uint32_t n) {
        if (!wait(o_full + 8 * h, n & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < DIM / 32; ++c) {
          uint32_t x[32];
          ptx::tmem_ld_32x32(t_o + c * 32, x);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[c * 32 + i] = fmaf(__uint_as_float(x[i]), back, o[c * 32 + i]);
        }
        return true;
      };
      for (unsigned j = 0; j < blocks; ++j, ++ns, ++nb) {
        if (!wait(s_full + 8 * h, ns & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        ptx::tc_fence_after_sync();
        if (j && !drain(ns - 1)) return false;
        const unsigned s = nb & 1u;
        if (!wait(sc_full + 8 * s, (nb >> 1) & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        const float4* ks = reinterpret_cast<const float4*>(smem + L::kScales + s * 1024);
        const float4* vr = ks + 32;
        back = value_back[s];
        const int key0 = static_cast<int>((it.lo + j) * kBlockKeys);
        const bool masked = key0 + static_cast<int>(kBlockKeys) > all_see;  // uniform in the half
        // -- largest score of the row --
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t x[32];
          ptx::tmem_ld_32x32(t_s + c * 32, x);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 k = ks[c * 8 + i / 4];
            const float y[4] = {__uint_as_float(x[i]) * k.x, __uint_as_float(x[i + 1]) * k.y,
                                __uint_as_float(x[i + 2]) * k.z, __uint_as_float(x[i + 3]) * k.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!masked || key0 + c * 32 + i + e < sees) top = fmaxf(top, y[e]);
          }
        }
        top *= row_scale;
        const bool grows = top > m + kLazy;  // (true for the first finite one: m is -inf)
        if (__any_sync(0xffffffffu, grows)) {
          const float next = grows ? top : m;
          const float f = exp2_fast(m - (next == -INFINITY ? 0.f : next));
          m = next;
          l *= f;
#pragma unroll
          for (int i = 0; i < DIM; ++i) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        // -- weights, as two terms over the scores they come from --
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t x[32];
          ptx::tmem_ld_32x32(t_s + c * 32, x);
          ptx::tmem_ld_wait();
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 k = ks[c * 8 + i / 4], v = vr[c * 8 + i / 4];
            float p[4] = {exp2_fast(fmaf(__uint_as_float(x[i]) * k.x, row_scale, -ref)),
                          exp2_fast(fmaf(__uint_as_float(x[i + 1]) * k.y, row_scale, -ref)),
                          exp2_fast(fmaf(__uint_as_float(x[i + 2]) * k.z, row_scale, -ref)),
                          exp2_fast(fmaf(__uint_as_float(x[i + 3]) * k.w, row_scale, -ref))};
            float y[4] = {p[0] * v.x, p[1] * v.y, p[2] * v.z, p[3] * v.w};
            if (masked) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (key0 + c * 32 + i + e >= sees) p[e] = y[e] = 0.f;
            }
            l += (p[0] + p[1]) + (p[2] + p[3]);
            w[i / 2] = pack_half2(y[0], y[1]);
            w[i / 2 + 1] = pack_half2(y[2], y[3]);
            w[16 + i / 2] = pack_rest(y[0], y[1], w[i / 2]);
            w[16 + i / 2 + 1] = pack_rest(y[2], y[3], w[i / 2 + 1]);
          }
          ptx::tmem_st_32x32(t_s + c * 32, w);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(sc_empty + 8 * s);
          ptx::mbar_arrive(p_full + 8 * h);
        }
      }
      if (!drain(ns - 1)) return false;
      if (!live) return true;
      if (it.whole) {
        const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;  // nothing seen: 0
        float4* dst = reinterpret_cast<float4*>(a.out + a.ldo * (static_cast<size_t>(it.first) + tok) +
                                                static_cast<size_t>(hd) * DIM);
#pragma unroll
        for (int i = 0; i < DIM; i += 4)
          dst[i / 4] = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
      } else {
        float* p = piece<kManyRows, DIM>(a, blockIdx.x, it.lo == 0);
        const unsigned pr = h * 128 + r;
        p[pr] = m;
        p[kManyRows + pr] = l;
        float4* dst = reinterpret_cast<float4*>(p + 2 * kManyRows + pr * DIM);
#pragma unroll
        for (int i = 0; i < DIM; i += 4) dst[i / 4] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
      return true;
    });
  }

  // ---- teardown ----
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {  // a wait was abandoned: give MMAs in flight a bounded moment
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  if (warp == 0) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<1>(tmem, 512);
  }
}

template <int DIM>
int launch_many(const CacheAttentionArgs& args, CacheAttention a, int sm_count) {
  using L = ManyLayout<DIM>;
  static std::atomic<unsigned long long> configured{0};
  const int st = opt_in_smem(cache_attention_many_kernel<DIM>, L::kSmem, configured);
  if (st != TFCCB200_OK) return st;
  // units that a launch of these bounds can have at most: tiles of all rows (one more per sequence
  // for its ragged end) times the blocks of the longest
  const unsigned long long rows = static_cast<unsigned long long>(args.cache.rows) * a.group;
  const unsigned long long bound = (rows / kManyRows + args.cache.batch) * args.cache.kv_heads *
                                   ((args.max_length + kBlockKeys - 1) / kBlockKeys);
  a.grid = static_cast<unsigned>(bound < static_cast<unsigned long long>(sm_count) ? bound : sm_count);
  cudaError_t e = launch_after_previous(cache_attention_many_kernel<DIM>, dim3(a.grid), dim3(kThreads), L::kSmem,
                                        args.cache.stream, a, kDefaultTimeoutNs);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  if (args.max_length > kBlockKeys && a.grid > 1) {
    e = launch_after_previous(cache_attention_merge_kernel<DIM, kManyRows>, dim3(a.grid - 1, 4), dim3(256), 0,
                              args.cache.stream, a);
    if (e != cudaSuccess) return static_cast<int>(e);
    count_launch();
  }
  return TFCCB200_OK;
}

}  // namespace

int cache_attention_many(const CacheAttentionArgs& args, CacheAttention a, int sm_count) {
  return args.cache.dim == 128 ? launch_many<128>(args, a, sm_count) : launch_many<64>(args, a, sm_count);
}

}  // namespace tfccb200

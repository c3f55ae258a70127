// Attention over the paged 8-bit cache for many rows per kv head: chunks of prompts, tcgen05.
//
// An item is 128 query rows of one kv head (the rows of one MMA) against a run of 128-key blocks.
// K and V are exact in fp16, and the fp32 operands are split into two fp16 terms each, x = hi + lo with 11 bits:
// q per row after scaling by a power of two, and the weights w_j = p_j vs_j as in
// cache_attention.cu.  Per block
//   S = Q_hi K^T + Q_lo K^T          A from tensor memory, K from shared memory, fp32 sums
//   P = exp2(S ks - r) vs            r: the row's largest score in the block; hi and lo terms go back over S
//   O_block = P_hi V + P_lo V        A from tensor memory, V as it lies (MN-major)
//   O = O alpha + 2^(r - m) O_block  fp32 registers, m the row's running maximum
// The tensor core's accumulator narrows without rounding to nearest, which would bias O over
// thousands of keys; summed from zero per block and added to registers it does not, and a block's
// own power of two for the value scales comes along for nothing.
//
// Tensor memory (512 columns): Q_hi, Q_lo | S of even blocks | S of odd blocks | O_block.  With two S
// buffers the tensor core computes the next block's scores while the weights of this one are made.
//
// Roles (512 threads, registers shifted with setmaxnreg):
//   warp 0      issues the MMAs: S of block j + 1, then the products with V of block j
//   warp 1      loads the blocks' scales
//   warp 2      walks the schedule and hands the items to the others
//   warps 4-7   turn codes into fp16 operand tiles (global -> registers -> shared memory): the tiles
//               of K and V share a ring, one row's 64 values per 128-byte swizzled line
//   warps 8-15  softmax, sums and output of 16 rows each.  Tensor memory is read and written in the
//               layout of matrix fragments, two rows and every fourth pair of keys per thread: 64 scores
//               and 64 sums fit the registers, a row's maximum and sum are two shuffles, and a
//               thread reads the scales of 32 keys instead of 128
// Bound by the tensor core: 8 dim flops per row and key instead of the 4 counted, at the rate the card
// sustains on dense data.  4096 new tokens on 4096 cached ones, 32 / 8 heads of 128: 843 us, 489 TFLOP/s
// counted, 978 executed (0.60 of the measured burst rate of bf16 products, 0.70 of the sustained one).  What was
// measured on the way there (the same case): a thread per row with all of its 128 sums, two
// tiles per CTA 1137; two threads per row 1193; this layout 955; products issued with precomputed
// descriptors 932; items weighted in the schedule 870; scales in the order of their reading 838.
// Ordinary loads in place of read-only ones, pages looked up four at a time: 840.  References per block
// and the path for value scales that spread wide: 833 to 843 (with that path in the registers of the main one 850 to
// 885).
// Slower: sixteen softmax warps 1088, products summed over four blocks in tensor memory 972, codes
// through a ring of bulk copies 880, code loads two tiles ahead 930,
// the next tile's loads between this one's stores 995.
//
// Every wait is bounded: on expiry a status bit is raised and all roles run to their end.
#include <cuda_runtime.h>

#include <type_traits>

#include "cache_attention.cuh"
#include "internal.h"
#include "pdl.cuh"
#include "ptx.cuh"

namespace tfccb200 {

namespace {

constexpr int kThreads = 512;
constexpr int kTileBytes = 128 * 128;  // 128 rows x 64 fp16, 128-byte swizzle
constexpr int kRegsControl = 48, kRegsConvert = 96, kRegsSoftmax = 184;
static_assert(kRegsControl + kRegsConvert + 2 * kRegsSoftmax == 512, "shares of 128 registers per thread at launch");

// The unit of a block's weights: its largest value scale, rounded up to a power of two E, is held as kWeightTop
// = 2^14, and a row's exponentials are taken relative to its own largest score in the block, so that
// weights reach at most 2^14.  As long as the block's scales lie within 2^kValueRange of E, the row's largest weight
// is no less than 2^(14 - kValueRange), and fp16's absolute error of 2^-25 is 2^-30 of it.  Where they spread
// wider, in keys that the row may not even see, the unit is a row's own largest weight instead (wide_block).
constexpr float kWeightTop = 16384.f;
constexpr int kValueRange = 9;
constexpr uint32_t kWideTop = 0x71800000u;     // 2^100
constexpr float kWideUnit = 1.0995116e12f;     // 2^40
constexpr float kLazy = 5.f;          // the maximum moves only when it grows by more (log2 units)
constexpr float kValueFloor = 7.8886091e-31f;  // 2^-100

struct Item {  // what the roles need to know of an item; hi == 0 ends the walk
  int first, count, length, b;
  unsigned head, tile, lo, hi;
  unsigned whole, rows;
  unsigned pad[2];
};

// A block's 128 key (or value) scales in shared memory, in the order the softmax reads them: the 32 of the
// keys 8 i + 2 t, + 1 of thread t of a quad together, and the quad's four groups on different banks.
constexpr int kScalePitch = 36;
__device__ __forceinline__ unsigned scale_place(unsigned key) {
  return ((key >> 1) & 3u) * kScalePitch + (key >> 3) * 2 + (key & 1u);
}

template <int DIM>
struct ManyLayout {
  static constexpr int kHalves = DIM / 64;               // 64-wide tiles of a row
  static constexpr int kOperand = kHalves * kTileBytes;  // 128 rows of K or V
  static constexpr int kRing = DIM == 128 ? 6 : 8;
  static constexpr int kScales = kRing * kOperand;       // 2 x {ks[128], vr[128]}
  static constexpr int kScaleBytes = 2 * 4 * kScalePitch * 4;
  static constexpr int kItems = kScales + 2 * kScaleBytes;
  static constexpr int kBars = kItems + 2 * static_cast<int>(sizeof(Item));
  static constexpr int kNumBars = 30;
  static constexpr int kMisc = kBars + 8 * kNumBars;           // tensor memory address, abort flag, value factors
  static constexpr int kSched = kMisc + 16;
  static constexpr int kSmem = kSched + static_cast<int>(sizeof(ScheduleShared));
  static constexpr int kTmemQ = 0, kTmemS = 128, kTmemO = 384;  // columns
  static_assert(kSmem <= 232448, "shared memory");
};

// 2^(x - m), 0 for x = -inf whatever m is.
__device__ __forceinline__ float relative_to(float x, float m) { return x == -INFINITY ? 0.f : exp2_fast(x - m); }
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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
  const uint32_t q_full = bar(0), p_full = bar(1), o_full = bar(2);
  const uint32_t s_full = bar(4), sc_full = bar(6), sc_empty = bar(8), it_full = bar(10), it_empty = bar(12);  // two each
  const uint32_t kv_full = bar(14), kv_empty = bar(14 + L::kRing);
  static_assert(14 + 2 * L::kRing <= L::kNumBars, "barriers");
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem + L::kMisc);
  volatile uint32_t* abort_flag = misc + 1;
  volatile float* value_back = reinterpret_cast<volatile float*>(misc + 2);  // per scale stage: value of the scales' unit, negative where they spread wide
  const Item* items = reinterpret_cast<const Item*>(smem + L::kItems);
  ScheduleShared* sched = reinterpret_cast<ScheduleShared*>(smem + L::kSched);
  const Waiter wait{abort_flag, a.c.status, timeout_ns};

  if (tid == 0) {
    ptx::mbar_init(q_full, 8);
    ptx::mbar_init(p_full, 8);
    ptx::mbar_init(o_full, 1);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(s_full + 8 * i, 1);
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
    ptx::tmem_alloc<1>(base + L::kMisc, 512);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = misc[0];
  pdl_wait();

  ThreadSequence mine;
  const unsigned long long units = all_units<kManyRows, kThreads>(a, sched, &mine);
  const unsigned busy = busy_ctas(units, a.grid);
  const bool mine_any = blockIdx.x < busy;
  const unsigned long long u0 = mine_any ? range_begin(units, busy, blockIdx.x) : 0;
  const unsigned long long u1 = mine_any ? range_begin(units, busy, blockIdx.x + 1) : 0;
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

  if (warp < 4) {
    ptx::setmaxnreg_dec<kRegsControl>();
    if (warp == 0) {
      // ======================= MMA issuer =======================
      uint32_t kv_n = 0;  // ring buffers used by earlier items
      uint32_t nb = 0;    // blocks of earlier items
      uint32_t ni = 0;    // items
      constexpr uint32_t idesc_s = ptx::make_idesc(1u, 0u, 0u, 0u, 0u, 128u, 128u);
      constexpr uint32_t idesc_o = ptx::make_idesc(1u, 0u, 0u, 0u, 1u, 128u, static_cast<uint32_t>(DIM));
      for_items([&](const Item& it) {
        const unsigned blocks = it.hi - it.lo;
        auto kv_wait = [&](uint32_t n) {
          return wait(kv_full + 8 * (n % L::kRing), (n / L::kRing) & 1u, TFCCB200_DEV_TIMEOUT_MMA);
        };
        auto tile = [&](uint32_t n) { return base + (n % L::kRing) * L::kOperand; };
        // S of the item's block j, from ring buffer kv_n + 2 j
        auto score = [&](unsigned j) {
          const uint32_t n = kv_n + 2 * j, s2 = (nb + j) & 1u;
          if (!kv_wait(n)) return false;
          ptx::tc_fence_after_sync();
          __syncwarp();
          if (ptx::elect_one()) {
            const uint64_t desc = ptx::smem_desc(tile(n), 16, 1024, ptx::kLayoutSw128);
            const uint32_t lo = static_cast<uint32_t>(desc), hi = static_cast<uint32_t>(desc >> 32);
            const uint32_t d = tmem + L::kTmemS + s2 * 128, q = tmem + L::kTmemQ;
            ptx::umma_f16_ts<false>(d, q + DIM / 2, lo, hi, idesc_s);  // the small terms first
#pragma unroll
            for (int s = 1; s < kSteps; ++s)
              ptx::umma_f16_ts<true>(d, q + DIM / 2 + s * 8, lo + ((s >> 2) * kTileBytes + (s & 3) * 32) / 16, hi, idesc_s);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
              ptx::umma_f16_ts<true>(d, q + s * 8, lo + ((s >> 2) * kTileBytes + (s & 3) * 32) / 16, hi, idesc_s);
            ptx::umma_commit<1>(s_full + 8 * s2, 0);
            ptx::umma_commit<1>(kv_empty + 8 * (n % L::kRing), 0);
          }
          __syncwarp();
          return true;
        };
        if (!wait(q_full, ni++ & 1u, TFCCB200_DEV_TIMEOUT_MMA)) return false;
        if (!score(0)) return false;
        for (unsigned j = 0; j < blocks; ++j) {
          // The next block's S goes over the weights of the block before this one, whose products
          // were issued earlier: one thread's MMAs run in the order of issue.
          if (j + 1 < blocks && !score(j + 1)) return false;
          const uint32_t n = kv_n + 2 * j + 1, s2 = (nb + j) & 1u;
          if (!kv_wait(n) || !wait(p_full, (nb + j) & 1u, TFCCB200_DEV_TIMEOUT_MMA)) return false;
          ptx::tc_fence_after_sync();
          __syncwarp();
          if (ptx::elect_one()) {
            const uint64_t desc = ptx::smem_desc(tile(n), kTileBytes, 1024, ptx::kLayoutSw128);
            const uint32_t lo = static_cast<uint32_t>(desc), hi = static_cast<uint32_t>(desc >> 32);
            const uint32_t d = tmem + L::kTmemO, p = tmem + L::kTmemS + s2 * 128;
            ptx::umma_f16_ts<false>(d, p + 8, lo, hi, idesc_o);
#pragma unroll
            for (int s = 1; s < 8; ++s) ptx::umma_f16_ts<true>(d, p + s * 16 + 8, lo + s * (2048 / 16), hi, idesc_o);
#pragma unroll
            for (int s = 0; s < 8; ++s) ptx::umma_f16_ts<true>(d, p + s * 16, lo + s * (2048 / 16), hi, idesc_o);
            ptx::umma_commit<1>(o_full, 0);
            ptx::umma_commit<1>(kv_empty + 8 * (n % L::kRing), 0);
          }
          __syncwarp();
        }
        kv_n += 2 * blocks;
        nb += blocks;
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
          // (pages first, then all scales, reports last: a report between two loads would order them)
          int page[4];
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = static_cast<int>(blk * kBlockKeys + i * 32 + lane);
            page[i] = pos < it.length ? page_entry(a.c, it.b, pos) : 0;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = static_cast<int>(blk * kBlockKeys + i * 32 + lane);
            const bool real = page_exists(a.c, page[i]);
            bad |= !real;
            ks[i] = vs[i] = real ? 0.f : __uint_as_float(0x7fffffffu);  // a page that does not exist shows as NaN
            if (pos < it.length && real) {
              const size_t at = cache_slot(a.c, page[i], it.head, pos);
              ks[i] = a.c.key_scales[at];
              vs[i] = a.c.value_scales[at];
            }
          }
          if (bad) raise_status(a.c.status, TFCCB200_DEV_BAD_PAGE);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bits = __float_as_uint(vs[i]) & 0x7fffffffu;
            if (bits < 0x7f800000u) top = max(top, bits);
          }
          top = __reduce_max_sync(0xffffffffu, top);
          top = min((top + 0x7fffffu) & 0x7f800000u, 0x7f000000u);  // up to a power of two
          bool wide = false;  // a key's scale lies 2^kValueRange below (0 does, whose key may have all the weight)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            wide |= static_cast<int>(blk * kBlockKeys + i * 32 + lane) < it.length &&
                    (__float_as_uint(vs[i]) & 0x7fffffffu) < top - (static_cast<uint32_t>(kValueRange) << 23);
          wide = __any_sync(0xffffffffu, wide);
          // wide: scales as they are, or brought down so that exponentials relative to a weight have the range for it
          const float unit = !wide ? __uint_as_float(top) * (1.f / kWeightTop) : top > kWideTop ? kWideUnit : 1.f;
          const float up = 1.f / unit;
          if (!wait(sc_empty + 8 * s, ((n >> 1) & 1u) ^ 1u, TFCCB200_DEV_TIMEOUT_CONVERT)) return false;
          float* dst = reinterpret_cast<float*>(smem + L::kScales + s * L::kScaleBytes);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned at = scale_place(i * 32 + lane);
            dst[at] = ks[i];
            dst[4 * kScalePitch + at] = vs[i] * up;
          }
          if (lane == 0) value_back[s] = wide ? -unit : unit;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sc_full + 8 * s);
        }
        return true;
      });
    } else if (warp == 2) {
      // ======================= walker =======================
      unsigned n = 0;
      // An item's place is free when the softmax takes it up, which may be a whole item later: the limit
      // grows with the range (20 us a block, several times what one takes).
      const Waiter wait_item{abort_flag, a.c.status, timeout_ns + 20000ull * (u1 - u0)};
      auto put = [&](const Item& it) {
        const unsigned s = n & 1u;
        if (!wait_item(it_empty + 8 * s, ((n >> 1) & 1u) ^ 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        if (lane == 0) {
          *reinterpret_cast<Item*>(smem + L::kItems + s * sizeof(Item)) = it;
          ptx::mbar_arrive(it_full + 8 * s);
        }
        __syncwarp();
        ++n;
        return true;
      };
      bool live = true, noted = false;
      for (ItemWalk<kManyRows> w(a, u1 - u0, sched); live && !w.done(); w.next()) {
        if (a.scratch && w.taken == w.left) {  // the range's last
          if (lane == 0) write_note<kManyRows>(a, blockIdx.x, busy, units, u1, &w);
          noted = true;
        }
        Item it;
        it.first = w.seq.first; it.count = w.seq.count; it.length = w.seq.length; it.b = w.b;
        it.head = w.head; it.tile = w.tile; it.lo = w.lo; it.hi = w.hi;
        it.whole = w.whole() ? 1u : 0u;
        it.rows = static_cast<unsigned>(w.seq.count) * a.group;
        live = put(it);
      }
      if (a.scratch && !noted && lane == 0) write_note<kManyRows>(a, blockIdx.x, busy, units, u1, nullptr);
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
            ahead[g * L::kHalves + h] = pg >= 0 ? p[h * 4 + c4] : make_uint4(0u, 0u, 0u, 0u);
        }
      };
      load(0);
      for (unsigned i = 0; i < tiles; ++i, ++n) {
        const unsigned s = n % L::kRing;
        if (!wait(kv_empty + 8 * s, ((n / L::kRing) & 1u) ^ 1u, TFCCB200_DEV_TIMEOUT_CONVERT)) return false;
        uint8_t* dst = smem + s * L::kOperand;
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
    const unsigned g = lane >> 2, t = lane & 3u;
    const unsigned lane0 = (warp & 3u) * 32 + ((warp >> 2) - 2) * 16;  // the warp's first row = lane of tensor memory
    const uint32_t rows_addr = tmem + (lane0 << 16);
    uint32_t nb = 0;  // blocks so far
    for_items([&](const Item& it) {
      const unsigned blocks = it.hi - it.lo;
      const int past = it.length - it.count;
      // keys below this are seen by every row of the item
      const int all_see = a.causal ? past + static_cast<int>(it.tile * kManyRows / a.group) + 1 : it.length;
      float rs[2];  // of the thread's rows lane0 + g + 8 k: scale of the scores, visible keys
      int sees[2];

      // ---- Q as two fp16 terms, scaled by a power of two per row ----
      {
        float f[2][DIM / 4];  // columns 8 i + 2 t, + 1
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const unsigned row = it.tile * kManyRows + lane0 + g + 8 * k;
          const bool live = row < it.rows;
          const unsigned tok = live ? row / a.group : 0, hd = it.head * a.group + (live ? row % a.group : 0);
          sees[k] = !live ? 0 : (a.causal ? past + static_cast<int>(tok) + 1 : it.length);
          const float2* q = reinterpret_cast<const float2*>(
              a.q + a.ldq * (static_cast<size_t>(it.first) + tok) + static_cast<size_t>(hd) * DIM) + t;
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i) {
            const float2 x = live ? q[4 * i] : make_float2(0.f, 0.f);
            f[k][2 * i] = x.x * a.scale;
            f[k][2 * i + 1] = x.y * a.scale;
          }
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < DIM / 4; ++i) m = max(m, __float_as_uint(f[k][i]) & 0x7fffffffu);
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
          // 2^(10 - exponent): the largest value lands in [2^10, 2^11); tiny rows take the bound of the
          // range, a non-finite row 1 (it becomes NaN in any case)
          const int ex = static_cast<int>(m >> 23) - 127;
          const int sh = ex == 128 ? 0 : 10 - max(ex, -100);
          const float up = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
          rs[k] = __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
#pragma unroll
          for (int i = 0; i < DIM / 4; ++i) f[k][i] *= up;
        }
#pragma unroll
        for (int c = 0; c < DIM / 64; ++c) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float x = f[k][16 * c + 2 * i], y = f[k][16 * c + 2 * i + 1];
              hi[2 * i + k] = pack_half2(x, y);
              lo[2 * i + k] = pack_rest(x, y, hi[2 * i + k]);
            }
          ptx::tmem_st_16x32(rows_addr + L::kTmemQ + c * 32, hi);
          ptx::tmem_st_16x32(rows_addr + L::kTmemQ + DIM / 2 + c * 32, lo);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(q_full);
      }

      float o[DIM / 2];  // [4 i + 2 k + e]: column 8 i + 2 t + e of row k
#pragma unroll
      for (int i = 0; i < DIM / 2; ++i) o[i] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      float back[2] = {0.f, 0.f};  // what the products of the block to be drained are worth
      // adds the products of the block before (accumulated in tensor memory from zero) to o
      auto drain = [&](uint32_t n) {
        if (!wait(o_full, n & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < DIM / 64; ++c) {
          uint32_t x[32];
          ptx::tmem_ld_16x64(rows_addr + L::kTmemO + c * 64, x);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float b = back[(i >> 1) & 1];
            const float2 y = unpair(fma2(pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), pair(b, b),
                                         pair(o[c * 32 + i], o[c * 32 + i + 1])));
            o[c * 32 + i] = y.x;
            o[c * 32 + i + 1] = y.y;
          }
        }
        return true;
      };
      // One block; kMask: with keys that not every row sees (compiled apart: the comparisons would
      // take more issue slots than the exponentials).
      auto block = [&](unsigned j, auto mask) {
        constexpr bool kMask = decltype(mask)::value;
        const unsigned s = nb & 1u;
        const uint32_t t_s = rows_addr + L::kTmemS + s * 128;
        // scales of this thread's keys 8 i + 2 t, + 1 for two i at a time, then of their values
        const ulonglong2* ks_at = reinterpret_cast<const ulonglong2*>(smem + L::kScales + s * L::kScaleBytes) + t * (kScalePitch / 4);
        const ulonglong2* vs_at = ks_at + kScalePitch;
        if (!wait(s_full + 8 * s, (nb >> 1) & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        ptx::tc_fence_after_sync();
        const int first = static_cast<int>((it.lo + j) * kBlockKeys + 2 * t);  // the thread's first key
        // -- scores times key scales, [4 i + 2 k + e]: key first + 8 i + e of row k --
        float y[64];
        float top[2] = {-INFINITY, -INFINITY};
        ptx::tmem_ld_16x64(t_s, reinterpret_cast<uint32_t(&)[32]>(y[0]));
        ptx::tmem_ld_16x64(t_s + 64, reinterpret_cast<uint32_t(&)[32]>(y[32]));
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t ks = (i & 1) ? ks_at[i / 2].y : ks_at[i / 2].x;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float* e = &y[4 * i + 2 * k];
            float2 u = unpair(mul2(pair(e[0], e[1]), ks));
            if constexpr (kMask) {
              u.x = first + 8 * i < sees[k] ? u.x : -INFINITY;
              u.y = first + 8 * i + 1 < sees[k] ? u.y : -INFINITY;
            }
            e[0] = u.x;
            e[1] = u.y;
            top[k] = fmaxf(top[k], fmaxf(u.x, u.y));
          }
        }
        const uint64_t rs2[2] = {pair(rs[0], rs[0]), pair(rs[1], rs[1])};
        bool grows = false;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
          top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2)) * rs[k];
          grows |= top[k] > m[k] + kLazy;  // (true for the first finite one: m is -inf)
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float next = top[k] > m[k] + kLazy ? top[k] : m[k];
            const float f = relative_to(m[k], next);
            m[k] = next;
            l[k] *= f;
            back[k] *= f;
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) {
              o[4 * i + 2 * k] *= f;
              o[4 * i + 2 * k + 1] *= f;
            }
          }
        }
        // -- weights, as two terms over the scores they come from: 16 scores become 8 columns of hi
        // and 8 of lo terms --
        const float r0 = top[0] == -INFINITY ? 0.f : -top[0], r1 = top[1] == -INFINITY ? 0.f : -top[1];
        const uint64_t ref2[2] = {pair(r0, r0), pair(r1, r1)};
        uint64_t l2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {  // 32 keys at a time
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = 4 * ch + i;
            const uint64_t vs = (c & 1) ? vs_at[c / 2].y : vs_at[c / 2].x;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float2 e = unpair(fma2(pair(y[4 * c + 2 * k], y[4 * c + 2 * k + 1]), rs2[k], ref2[k]));
              const uint64_t p = pair(exp2_fast(e.x), exp2_fast(e.y));
              l2[k] = add2(l2[k], p);
              float2 u = unpair(mul2(p, vs));
              if constexpr (kMask) {  // (0 * NaN)
                u.x = first + 8 * c < sees[k] ? u.x : 0.f;
                u.y = first + 8 * c + 1 < sees[k] ? u.y : 0.f;
              }
              // keys 8 c + 2 t, + 1: column 4 (c % 2) + t of the group c / 2 of 16 columns; lo 8 further
              const uint32_t hi = pack_half2(u.x, u.y);
              w[2 * (4 * (i >> 1) + (i & 1)) + k] = hi;
              w[2 * (4 * (i >> 1) + 2 + (i & 1)) + k] = pack_rest(u.x, u.y, hi);
            }
          }
          ptx::tmem_st_16x32(t_s + ch * 32, w);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 f = unpair(l2[k]);
          top[k] = relative_to(top[k], m[k]);
          l[k] = fmaf(f.x + f.y, top[k], l[k]);
        }
        if (j && !drain(nb - 1)) return false;
#pragma unroll
        for (int k = 0; k < 2; ++k) back[k] = value_back[s] * top[k];
        ptx::tmem_st_wait();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(sc_empty + 8 * s);
          ptx::mbar_arrive(p_full);
        }
        return true;
      };
      // One block whose value scales spread wide.  A row's reference is the one that puts its largest weight at
      // 2^13 (but no less than 2^-90 of its largest exponential, for the sum of these).  The scores are
      // read from tensor memory twice, 64 at a time: kept, they would cost the loop above registers.
      auto wide_block = [&](unsigned j) {
        const unsigned s = nb & 1u;
        const uint32_t t_s = rows_addr + L::kTmemS + s * 128;
        const float2* const ks_at = reinterpret_cast<const float2*>(smem + L::kScales + s * L::kScaleBytes) + t * (kScalePitch / 2);
        const float2* const vs_at = ks_at + 2 * kScalePitch;
        if (!wait(s_full + 8 * s, (nb >> 1) & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        ptx::tc_fence_after_sync();
        const int first = static_cast<int>((it.lo + j) * kBlockKeys + 2 * t);
        float ref[2] = {-INFINITY, -INFINITY}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        // scores 64 h .. of the block, -inf where a row does not see the key
        auto scores = [&](int h, uint32_t (&x)[32]) {
          __syncwarp();  // accesses to tensor memory want the warp whole
          ptx::tmem_ld_16x64(t_s + 64 * h, x);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 ks = ks_at[8 * h + i];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t* const e = &x[4 * i + 2 * k];
              const int key = first + 64 * h + 8 * i;
              e[0] = __float_as_uint(key < sees[k] ? __uint_as_float(e[0]) * ks.x * rs[k] : -INFINITY);
              e[1] = __float_as_uint(key + 1 < sees[k] ? __uint_as_float(e[1]) * ks.y * rs[k] : -INFINITY);
            }
          }
        };
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t x[32];
          scores(h, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 vs = vs_at[8 * h + i];
            const float lx = fabsf(vs.x) < INFINITY ? log2_fast(fabsf(vs.x)) : -INFINITY;
            const float ly = fabsf(vs.y) < INFINITY ? log2_fast(fabsf(vs.y)) : -INFINITY;
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // (the maxima pass over NaN)
              const float u = __uint_as_float(x[4 * i + 2 * k]), v = __uint_as_float(x[4 * i + 2 * k + 1]);
              top[k] = fmaxf(top[k], fmaxf(u, v));
              ref[k] = fmaxf(ref[k], fmaxf(u + lx, v + ly));
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int o2 = 1; o2 < 4; o2 <<= 1) {
            top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o2));
            ref[k] = fmaxf(ref[k], __shfl_xor_sync(0xffffffffu, ref[k], o2));
          }
          ref[k] = fmaxf(ref[k] - 13.f, top[k] - 90.f);
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + kLazy || top[1] > m[1] + kLazy)) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float next = top[k] > m[k] + kLazy ? top[k] : m[k];
            const float f = relative_to(m[k], next);
            m[k] = next;
            l[k] *= f;
            back[k] *= f;
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) {
              o[4 * i + 2 * k] *= f;
              o[4 * i + 2 * k + 1] *= f;
            }
          }
        }
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t x[32];
          scores(h, x);
#pragma unroll
          for (int ch = 0; ch < 2; ++ch) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = 4 * ch + i, key = first + 64 * h + 8 * c;
              const float2 vs = vs_at[8 * h + c];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float r = ref[k] == -INFINITY ? 0.f : ref[k];
                const float px = exp2_fast(__uint_as_float(x[4 * c + 2 * k]) - r), py = exp2_fast(__uint_as_float(x[4 * c + 2 * k + 1]) - r);
                sum[k] += px + py;
                const float ux = key < sees[k] ? px * vs.x : 0.f, uy = key + 1 < sees[k] ? py * vs.y : 0.f;
                const uint32_t hi = pack_half2(ux, uy);
                w[2 * (4 * (i >> 1) + (i & 1)) + k] = hi;
                w[2 * (4 * (i >> 1) + 2 + (i & 1)) + k] = pack_rest(ux, uy, hi);
              }
            }
            ptx::tmem_st_16x32(t_s + 64 * h + ch * 32, w);
          }
          ptx::tmem_st_wait();
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          ref[k] = relative_to(ref[k], m[k]);
          l[k] = fmaf(sum[k], ref[k], l[k]);
        }
        if (j && !drain(nb - 1)) return false;
        back[0] = -value_back[s] * ref[0];
        back[1] = -value_back[s] * ref[1];
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(sc_empty + 8 * s);
          ptx::mbar_arrive(p_full);
        }
        return true;
      };
      for (unsigned j = 0; j < blocks; ++j, ++nb) {
        if (!wait(sc_full + 8 * (nb & 1u), (nb >> 1) & 1u, TFCCB200_DEV_TIMEOUT_EPILOGUE)) return false;
        if (value_back[nb & 1u] < 0.f) {
          if (!wide_block(j)) return false;
          continue;
        }
        const bool masked = static_cast<int>((it.lo + j + 1) * kBlockKeys) > all_see;  // the same in all rows
        if (!(masked ? block(j, std::true_type()) : block(j, std::false_type()))) return false;
      }
      if (!drain(nb - 1)) return false;

      float* const part = it.whole ? nullptr : piece<kManyRows, DIM>(a, blockIdx.x, it.lo == 0);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
        const unsigned r = lane0 + g + 8 * k, row = it.tile * kManyRows + r;
        if (row < it.rows) {
          float inv = 1.f;
          float* dst;
          if (part) {
            if (t == 0) {
              part[r] = m[k];
              part[kManyRows + r] = l[k];
            }
            dst = part + 2 * kManyRows + r * DIM + 2 * t;
          } else {
            inv = m[k] == -INFINITY && l[k] == 0.f ? 0.f : 1.f / l[k];  // nothing seen: 0
            dst = a.out + a.ldo * (static_cast<size_t>(it.first) + row / a.group) +
                  (static_cast<size_t>(it.head) * a.group + row % a.group) * DIM + 2 * t;
          }
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i)
            *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[4 * i + 2 * k] * inv, o[4 * i + 2 * k + 1] * inv);
        }
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
                                   ((args.max_length + kBlockKeys - 1) / kBlockKeys + kLeadUnits);
  a.grid = static_cast<unsigned>(bound < static_cast<unsigned long long>(sm_count) ? bound : sm_count);
  cudaError_t e = launch_after_previous(cache_attention_many_kernel<DIM>, dim3(a.grid), dim3(kThreads), L::kSmem,
                                        args.cache.stream, a, kDefaultTimeoutNs);
  if (e != cudaSuccess) return static_cast<int>(e);
  count_launch();
  if (args.max_length > kBlockKeys && a.grid > 1) {
    e = launch_after_previous(cache_attention_merge_kernel<DIM, kManyRows>, dim3(a.grid, 4), dim3(256), 0,
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

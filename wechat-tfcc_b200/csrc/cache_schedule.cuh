// How the attention kernels share out their work.
//
// An item is a tile of kRows query rows of one kv head of one sequence (row r of a sequence's head
// is new token r / group, query head r % group of the head's group), and its units are the blocks
// of kBlockKeys cached tokens that the tile's last row sees.  Lengths are device data and differ, so no
// grid the host could choose would be even: instead the units of all items are laid end to
// end (sequence, head, tile, block), each item led by kLeadUnits that stand for what beginning and
// ending an item costs, and every CTA takes an equal range.  (Without the lead a CTA that
// drew eight short sequences took 85 us where the others took 60.)  A range may begin and end inside an
// item.  Items that lie whole in one range are finished there; the pieces of a
// cut one go to scratch as unnormalised sums with their maximum, and the merge kernel adds
// them in key order.  Cuts depend on lengths and grid alone, so results repeat bit by bit.
#pragma once

#include "cache.cuh"

namespace tfccb200 {

constexpr unsigned kBlockKeys = 128;
constexpr unsigned kLeadUnits = 2;
// Sequences with up to this many rows per kv head go to the few-rows kernel.
constexpr unsigned kFewRows = 16;

struct CacheAttention {
  CacheParams c;
  const float* q;
  float* out;
  unsigned long long ldq, ldo;
  unsigned heads, group;  // group = heads / kv_heads
  unsigned min_rows, max_rows;  // rows per kv head of the sequences this launch takes
  unsigned grid;          // CTAs that share the units
  int causal;
  float scale;            // times log2(e)
  float* scratch;         // pieces, see piece_*; nullptr when no item can be cut
};

// Blocks of one tile; one at least, so that a row that sees nothing is still written.
template <int kRows>
__device__ __forceinline__ unsigned tile_blocks(const CacheAttention& a, const DeviceSequence& s, unsigned tile) {
  int end = s.length;
  if (a.causal) {
    const unsigned last = min(static_cast<unsigned>(s.count) * a.group, (tile + 1) * kRows) - 1;
    end = s.length - s.count + static_cast<int>(last / a.group) + 1;
  }
  return end <= 0 ? 1u : (static_cast<unsigned>(end) + kBlockKeys - 1) / kBlockKeys;
}

template <int kRows>
__device__ __forceinline__ unsigned sequence_tiles(const CacheAttention& a, const DeviceSequence& s) {
  const unsigned long long rows = static_cast<unsigned long long>(s.count) * a.group;
  if (rows == 0 || rows < a.min_rows || rows > a.max_rows) return 0;
  return static_cast<unsigned>((rows + kRows - 1) / kRows);
}

// Units of one kv head of a sequence.
template <int kRows>
__device__ __forceinline__ unsigned head_units(const CacheAttention& a, const DeviceSequence& s) {
  const unsigned tiles = sequence_tiles<kRows>(a, s);
  unsigned n = tiles * kLeadUnits;
  for (unsigned t = 0; t < tiles; ++t) n += tile_blocks<kRows>(a, s, t);
  return n;
}

struct ScheduleShared {
  unsigned long long sums[32];
  unsigned long long rem;  // find_unit: place within the sequence,
  int b;                   // the sequence,
  unsigned per_head;       // its units per kv head
  DeviceSequence seq;
};

// Sum of v over the block (to every thread).
template <int kThreads>
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, ScheduleShared* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) sh->sums[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long t = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) t += sh->sums[w];
  return t;
}

// Units of all sequences.  `mine` keeps those of sequence threadIdx.x for find_unit.
struct ThreadSequence {  // of sequence threadIdx.x (+ the block's size times the round)
  DeviceSequence seq;
  unsigned per_head;
  template <int kRows>
  __device__ __forceinline__ void load(const CacheAttention& a, unsigned b) {
    per_head = 0;
    if (b < a.c.batch) {
      seq = load_sequence(a.c, b);
      per_head = head_units<kRows>(a, seq);
    }
  }
};
template <int kRows, int kThreads>
__device__ __forceinline__ unsigned long long all_units(const CacheAttention& a, ScheduleShared* sh,
                                                        ThreadSequence* mine) {
  unsigned long long n = 0;
  mine->template load<kRows>(a, threadIdx.x);
  n = mine->per_head;
  for (unsigned b = threadIdx.x + kThreads; b < a.c.batch; b += kThreads) {
    ThreadSequence t;
    t.template load<kRows>(a, b);
    n += t.per_head;
  }
  return block_sum<kThreads>(n, sh) * a.c.kv_heads;
}

// The sequence that unit u (< all units) belongs to and u's place within it -> *sh.
template <int kRows, int kThreads>
__device__ __forceinline__ void find_unit(const CacheAttention& a, unsigned long long u, ThreadSequence mine,
                                          ScheduleShared* sh) {
  unsigned long long before = 0;  // units of the sequences of earlier rounds
  // (stays so only if the lengths change while the kernel reads them, which the caller must not let happen
  // and which must not send a walk beyond the arrays)
  if (threadIdx.x == 0) sh->b = -1;
  for (unsigned b0 = 0; b0 < a.c.batch; b0 += kThreads) {
    if (b0) mine.template load<kRows>(a, b0 + threadIdx.x);
    const unsigned long long own = static_cast<unsigned long long>(mine.per_head) * a.c.kv_heads;
    unsigned long long v = own;  // inclusive scan over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, v, o);
      if ((threadIdx.x & 31u) >= static_cast<unsigned>(o)) v += t;
    }
    __syncthreads();
    if ((threadIdx.x & 31u) == 31u) sh->sums[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long total = 0;
    unsigned long long base = before;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < static_cast<int>(threadIdx.x >> 5)) base += sh->sums[w];
      total += sh->sums[w];
    }
    if (own && base + v - own <= u && u < base + v) {
      sh->b = static_cast<int>(b0 + threadIdx.x);
      sh->rem = u - (base + v - own);
      sh->per_head = mine.per_head;
      sh->seq = mine.seq;
    }
    before += total;
    if (before > u) break;
  }
  __syncthreads();
}

// CTAs that get a range: as many as there are units at most, so that no range is empty.
__device__ __forceinline__ unsigned busy_ctas(unsigned long long units, unsigned grid) {
  return units < grid ? static_cast<unsigned>(units) : grid;
}
__device__ __forceinline__ unsigned long long range_begin(unsigned long long units, unsigned busy, unsigned cta) {
  return units / busy * cta + units % busy * cta / busy;
}

// Walks the items of a range of units; those of which the range holds no block are passed over.
template <int kRows>
struct ItemWalk {
  const CacheAttention& a;
  unsigned long long left;  // units still to come, this item's included
  unsigned long long rem;   // the range's first unit of this item within the sequence
  int b;
  DeviceSequence seq;
  unsigned per_head, head, tile, blocks;  // `blocks`: all of the item's
  unsigned lo, hi;                        // this range's blocks of it
  unsigned taken;                         // this range's units of it

  __device__ ItemWalk(const CacheAttention& a_, unsigned long long units, const ScheduleShared* sh)
      : a(a_), left(units), rem(0), b(0), per_head(0), head(0), tile(0), blocks(0), lo(0), hi(0), taken(0) {
    if (left == 0) return;
    b = sh->b;
    if (b < 0) {
      left = 0;
      return;
    }
    rem = sh->rem;
    seq = sh->seq;
    per_head = sh->per_head;
    place();
    if (lo == hi) next();
  }
  __device__ void place() {
    head = static_cast<unsigned>(rem / per_head);
    unsigned at = static_cast<unsigned>(rem % per_head);
    tile = 0;
    while (true) {
      blocks = tile_blocks<kRows>(a, seq, tile);
      if (at < blocks + kLeadUnits) break;
      at -= blocks + kLeadUnits;
      ++tile;
    }
    const unsigned end = static_cast<unsigned>(min(static_cast<unsigned long long>(blocks + kLeadUnits), at + left));
    taken = end - at;
    lo = at < kLeadUnits ? 0 : at - kLeadUnits;
    hi = end < kLeadUnits ? 0 : end - kLeadUnits;
  }
  __device__ bool done() const { return left == 0; }
  __device__ bool whole() const { return lo == 0 && hi == blocks; }
  __device__ void next() {
    do {
      left -= taken;
      rem += taken;
      if (left == 0) return;
      while (rem >= static_cast<unsigned long long>(per_head) * a.c.kv_heads) {
        rem = 0;
        do {
          // units are left, so a sequence that has some follows (unless lengths change under the kernel)
          if (static_cast<unsigned>(++b) >= a.c.batch) {
            left = 0;
            return;
          }
          seq = load_sequence(a.c, b);
          per_head = head_units<kRows>(a, seq);
        } while (per_head == 0);
      }
      place();
    } while (lo == hi);
  }
};

// The pieces of cut items: a CTA has at most one that begins inside an item (slot 0) and one that
// begins with it (slot 1).  A piece: kRows maxima (log2 units), kRows weight sums, kRows * DIM sums.
// In front of the pieces lies a note per CTA that tells the merge kernel what it began, so that the
// schedule is not worked out again.
struct PieceNote {
  unsigned ranges;  // CTAs whose ranges hold the rest of the item that this one began; 0: none
  unsigned head, tile, rows;
  int first;        // the sequence's first row
  unsigned pad[3];
};
constexpr size_t kNotesBytes = 32768;  // for up to 1024 CTAs
static_assert(sizeof(PieceNote) == 32, "notes");
template <int kRows, int DIM>
__host__ __device__ constexpr size_t piece_floats() { return static_cast<size_t>(kRows) * (DIM + 2); }
template <int kRows, int DIM>
__device__ __forceinline__ float* piece(const CacheAttention& a, unsigned cta, bool begins) {
  return a.scratch + kNotesBytes / 4 + (2ull * cta + (begins ? 1u : 0u)) * piece_floats<kRows, DIM>();
}
__device__ __forceinline__ PieceNote* piece_note(const CacheAttention& a, unsigned cta) {
  return reinterpret_cast<PieceNote*>(a.scratch) + cta;
}
// By one thread of every CTA of the grid: the note of a CTA whose range [u0, u1) ends inside an item that it
// began (`item` the range's last; nullptr: there is none).
template <int kRows>
__device__ __forceinline__ void write_note(const CacheAttention& a, unsigned cta, unsigned busy,
                                           unsigned long long units, unsigned long long u1, const ItemWalk<kRows>* item) {
  PieceNote n = {};
  if (item && item->lo == 0 && item->hi < item->blocks) {
    const unsigned long long end = u1 + (item->blocks - item->hi);  // the item's last unit + 1
    unsigned last = static_cast<unsigned>(min(static_cast<unsigned long long>(busy - 1), (end - 1) * busy / units));
    while (range_begin(units, busy, last) > end - 1) --last;
    while (last + 1 < busy && range_begin(units, busy, last + 1) <= end - 1) ++last;
    n.ranges = last - cta;
    n.head = item->head;
    n.tile = item->tile;
    n.rows = static_cast<unsigned>(item->seq.count) * a.group;
    n.first = item->seq.first;
  }
  *piece_note(a, cta) = n;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace tfccb200

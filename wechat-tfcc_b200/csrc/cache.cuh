// What the kernels of the paged 8-bit cache share: where a token of a sequence lies.
//
// Pool:      codes  [pages, kv_heads, page_size, dim] int8, scales [pages, kv_heads, page_size]
//            fp32, one pair for keys and one for values.
// Sequences: rows starts[b] .. starts[b+1] of a packed [rows, ...] tensor are the new tokens of
//            sequence b, lengths[b] the tokens it has in the cache with the new ones, and
//            position p of it lies in page table[b][p / page_size], slot p % page_size.
// All three arrays are device data that the host never sees, so every kernel checks what it reads
// before it uses it as an index: see DeviceSequence and page_of.  All of it, and what the kernels read of
// the cache, is read with ordinary loads: a kernel may be resident before the one that writes them is done,
// and loads through the read-only path are only defined for data constant over a kernel's life.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "internal.h"

namespace tfccb200 {

struct CacheParams {
  int8_t* keys;
  float* key_scales;
  int8_t* values;
  float* value_scales;
  unsigned pages, page_shift, kv_heads, dim;
  const int32_t* starts;
  const int32_t* lengths;
  const int32_t* table;
  unsigned batch, table_width, rows;
  unsigned max_new, max_length;  // of any one sequence
  int* status;
};

__device__ __forceinline__ void raise_status(int* status, int bit) {
  if (status) atomicOr(status, bit);
}

// One sequence's extents; `ok` false (and the status bit raised) where they contradict the sizes
// the host gave: rows outside the packed tensor, more tokens than the table has pages for or than the
// caller stated.
struct DeviceSequence {
  int first, count, length;  // first row, new tokens, cached tokens
  bool ok;
};
__device__ __forceinline__ DeviceSequence load_sequence(const CacheParams& p, unsigned b) {
  DeviceSequence s;
  s.first = p.starts[b];
  const int end = p.starts[b + 1];
  s.length = p.lengths[b];
  s.ok = s.first >= 0 && end >= s.first && static_cast<unsigned>(end) <= p.rows &&
         static_cast<unsigned>(end - s.first) <= p.max_new && s.length >= 0 &&
         static_cast<unsigned>(s.length) <= p.max_length;
  s.count = s.ok ? end - s.first : 0;
  if (!s.ok) raise_status(p.status, TFCCB200_DEV_BAD_SEQUENCE);
  return s;
}

// A kernel that goes by rows meets only the sequences that own some; its first CTA looks at all, so
// that every contradiction is reported.
__device__ __forceinline__ void check_all_sequences(const CacheParams& p) {
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (unsigned b = threadIdx.x; b < p.batch; b += blockDim.x) load_sequence(p, b);
}

// Page of position `pos` (< length <= table_width * page_size) of sequence b, as it stands in the table, and
// whether there is such a page.
__device__ __forceinline__ int page_entry(const CacheParams& p, unsigned b, unsigned pos) {
  return p.table[static_cast<size_t>(b) * p.table_width + (pos >> p.page_shift)];
}
__device__ __forceinline__ bool page_exists(const CacheParams& p, int page) {
  return page >= 0 && static_cast<unsigned>(page) < p.pages;
}
// The same at once: -1 (and a report) where there is none.
__device__ __forceinline__ int page_of(const CacheParams& p, unsigned b, unsigned pos) {
  const int page = page_entry(p, b, pos);
  if (!page_exists(p, page)) {
    raise_status(p.status, TFCCB200_DEV_BAD_PAGE);
    return -1;
  }
  return page;
}

// Index of (page, head, slot) in the scale arrays; times dim in the code arrays.
__device__ __forceinline__ size_t cache_slot(const CacheParams& p, int page, unsigned head, unsigned pos) {
  const unsigned mask = (1u << p.page_shift) - 1u;
  return ((static_cast<size_t>(page) * p.kv_heads + head) << p.page_shift) + (pos & mask);
}

// The sequence a packed row belongs to, found by the whole warp: the number of sequences that end
// at or before it.  Sequences are few, so the ends are counted (independent loads, one round of
// latency for up to 32 sequences) instead of searched by halving (a chain of loads).
// -1: behind the last sequence, or ends that are out of order.
__device__ __forceinline__ int sequence_of_row(const CacheParams& p, unsigned row) {
  unsigned n = 0;
  for (unsigned i = threadIdx.x & 31u; i < p.batch; i += 32)
    n += static_cast<long long>(p.starts[i + 1]) <= static_cast<long long>(row) ? 1u : 0u;
  n = __reduce_add_sync(0xffffffffu, n);
  if (n >= p.batch) return -1;
  const int first = p.starts[n], end = p.starts[n + 1];
  return static_cast<long long>(first) <= static_cast<long long>(row) &&
                 static_cast<long long>(row) < static_cast<long long>(end)
             ? static_cast<int>(n)
             : -1;
}

}  // namespace tfccb200

// Shared pieces of the paged key/value cache's kernels (paged_append.cu, paged_rows.cu,
// paged_chunk.cu): the device view of a cache and a batch, 16-bit conversions, and the split
// of a call's work over its CTAs.
//
// The split.  A call is a list of items (a tile of query rows of one sequence and one key/value
// head), each with a number of equal units of keys that only the device knows (the lengths are
// device arrays).  All units of all items are laid end to end and every CTA takes an equal,
// contiguous slice of them, so ragged batches load the SMs evenly whatever the lengths.  A CTA
// that holds the whole of an item writes its output; otherwise it leaves a partial result
// (running maximum, sum, unnormalised output, all float32) in the workspace, and the last CTA
// of the item to arrive adds the partials up in slice order -- the order does not depend on
// who arrives last, so results do not change from run to run.
#pragma once

#include "common.cuh"
#include "kernels.cuh"
#include "ptx.cuh"

namespace tdsa {

struct PagedView {
  const uint16_t* keys;
  const uint16_t* values;
  int64_t page_stride, row_stride, head_stride;  // elements
  int pages, page_shift, kv_heads;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* starts;
  const int32_t* lengths;
  int batch, max_pages, tokens;
};

struct SeqSpan {
  int q0;   // first row of the sequence's new tokens
  int n;    // new tokens
  int len;  // positions with them
};

// The batch arrays come from the device, so every value is clamped to what its buffer holds.
__device__ __forceinline__ SeqSpan load_span(const PagedView& p, int b) {
  SeqSpan s;
  const int a = __ldg(p.starts + b), e = __ldg(p.starts + b + 1), l = __ldg(p.lengths + b);
  s.q0 = min(max(a, 0), p.tokens);
  s.n = min(max(e, s.q0), p.tokens) - s.q0;
  s.len = min(max(l, 0), p.max_pages << p.page_shift);  // the host bounds this product
  return s;
}

// Element offset of position j's row of head 0, or -1 when its page is not one of the cache's.
__device__ __forceinline__ int64_t paged_row(const PagedView& p, int entry, int j) {
  if (entry < 0 || entry >= p.pages) return -1;
  return static_cast<int64_t>(entry) * p.page_stride +
         static_cast<int64_t>(j & ((1 << p.page_shift) - 1)) * p.row_stride;
}

template <bool kBF16>
__device__ __forceinline__ float2 unpack16(uint32_t p) {
  if (kBF16) return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&p));
}

// lo in the low half, both rounded to nearest even
template <bool kBF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (kBF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Whether one of the two 16-bit values is infinite or NaN.
template <bool kBF16>
__device__ __forceinline__ bool nonfinite16(uint32_t p) {
  constexpr uint32_t e = kBF16 ? 0x7F80u : 0x7C00u;
  return (p & e) == e || ((p >> 16) & e) == e;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Slice of CTA c of `ctas` (at most `units`) over `units`, and the CTA whose slice holds unit u.
__device__ __forceinline__ int64_t slice_begin(int64_t units, int ctas, int c) {
  return units * c / ctas;
}
__device__ __forceinline__ int slice_owner(int64_t units, int ctas, int64_t u) {
  return static_cast<int>(((u + 1) * ctas - 1) / units);
}

// Workspace of a split call: one arrival counter per CTA (an item that is split is known by
// the CTA it starts in; zero between calls), then two partial results per CTA (slot 0: the
// item the CTA's slice begins inside of, slot 1: the item it ends inside of).
constexpr int kPagedCounters = 1024;
struct PagedPartials {
  uint32_t* counters;
  float2* ml;   // [slot][rows]: running maximum (log2 units), sum
  float* o;     // [slot][rows][dim]
};

inline size_t paged_partial_bytes(int ctas, int rows, int dim) {
  return kPagedCounters * 4 + static_cast<size_t>(ctas) * 2 * rows * (8 + 4 * dim);
}

inline PagedPartials paged_partials(void* ws, int ctas, int rows) {
  PagedPartials p;
  p.counters = static_cast<uint32_t*>(ws);
  p.ml = reinterpret_cast<float2*>(p.counters + kPagedCounters);
  p.o = reinterpret_cast<float*>(p.ml + static_cast<size_t>(ctas) * 2 * rows);
  return p;
}

struct PagedQuery {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  uint16_t* out;
  int64_t o_ts, o_hs;
  float* lse;        // [tokens][heads] or null
  int heads, group;  // query heads, query heads per key/value head
  float scale_log2;  // scale * log2(e)
  int window;        // keys a token sees up to its own position; 0: all
  // selected attention: [tokens][topk] positions of idx_bytes each
  const void* idx;
  int64_t idx_stride;
  int idx_bytes, topk;
};

}  // namespace tdsa

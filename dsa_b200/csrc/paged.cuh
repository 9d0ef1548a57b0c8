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
  int* status;
};

struct SeqSpan {
  int q0;   // first row of the sequence's new tokens
  int n;    // new tokens
  int len;  // positions with them, as far as the page table reaches
  int pos;  // position of the first new token, by the length as it stands
};

// The batch arrays come from the device, so every value is clamped to what its buffer holds; a
// length that is none, or past the page table's end, is reported.
__device__ __forceinline__ void load_rows(const PagedView& p, int b, int& q0, int& n) {
  const int a = __ldg(p.starts + b), e = __ldg(p.starts + b + 1);
  q0 = min(max(a, 0), p.tokens);
  n = min(max(e, q0), p.tokens) - q0;
}
__device__ __forceinline__ SeqSpan load_span(const PagedView& p, int b) {
  SeqSpan s;
  const int l = __ldg(p.lengths + b);
  load_rows(p, b, s.q0, s.n);
  s.len = min(max(l, 0), p.max_pages << p.page_shift);  // the host bounds this product
  s.pos = max(l, 0) - s.n;
  if (s.len != l) atomicOr(p.status, TDSA_STATUS_RANGE);
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

// The same of several pairs: bits of 0x80008000 in the or of nonfinite_bits(p).  An exponent of
// ones carries into the sign's place, which the mask has cleared, and no further.
template <bool kBF16>
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t p) {
  return kBF16 ? (p & 0x7F807F80u) + 0x00800080u : (p & 0x7C007C00u) + 0x04000400u;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two float32 in a register pair, and a * b + c of both in one issue slot.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// A weight is held as 2^((s - t) scale + kBias), s the score and t the score of the row's maximum
// as it stood when t was last moved, which happens when it has grown by kGrow log2 units, so no
// weight is above 2^(kBias + kGrow).  (The difference comes before the product: t scale alone, once
// its rounding is worth a power of two, would make a largest weight infinite or nothing.)
// bfloat16 has float32's exponents, so no weight needs to be above 1, and with none above it a
// value near the type's largest does not overflow a product.  float16 would lose every weight below
// 2^-25 of the largest, which a long row has many of: up to 2^15 of float16's 2^16, weights above
// 2^-25 of the row's largest keep 11 bits, and a smaller one is off by no more than 2^-36 of it.
template <bool kBF16>
struct WeightRange {
  static constexpr float kGrow = kBF16 ? 8.f : 4.f, kBias = kBF16 ? -8.f : 11.f;
};

// Slice of CTA c of `ctas` (at most `units`) over `units`, and the CTA whose slice holds unit u:
// the first units % ctas slices have one unit more.  32-bit divisions where they do.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if ((a | b) >> 31) return a / b;
  return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}
__device__ __forceinline__ int64_t slice_begin(int64_t units, int ctas, int c) {
  const int64_t base = quotient(units, ctas);
  return base * c + min(static_cast<int64_t>(c), units - base * ctas);
}
__device__ __forceinline__ int slice_owner(int64_t units, int ctas, int64_t u) {
  const int64_t base = quotient(units, ctas), more = units - base * ctas;
  if (u < more * (base + 1)) return static_cast<int>(quotient(u, base + 1));
  return static_cast<int>(more + quotient(u - more * (base + 1), base));
}

// Workspace of a split call: one arrival counter per CTA (an item that is split is known by
// the CTA it starts in; zero between calls), then two partial results per CTA (slot 0: the
// item the CTA's slice begins inside of, slot 1: the item it ends inside of).
constexpr int kPagedCounters = TDSA_PAGED_COUNTER_BYTES / 4;
struct PagedPartials {
  uint32_t* counters;
  float2* ml;   // [slot][rows]: running maximum (few rows: t; chunks: t scale - kBias), sum
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

// One more part of a split item has arrived, whose stores (the whole block's, behind a barrier)
// are visible to whoever sees the count; true for the last of n, which then sees all the others'
// and leaves the counter at zero.
__device__ __forceinline__ bool paged_arrive(uint32_t* counter, uint32_t n) {
  uint32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
               : "=r"(old)
               : "l"(counter)
               : "memory");
  if (old == n - 1) *counter = 0u;
  return old == n - 1;
}

struct PagedQuery {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  uint16_t* out;
  int64_t o_ts, o_hs;
  float* lse;        // [tokens][heads] or null
  int heads, group;  // query heads, query heads per key/value head
  uint32_t group_magic;  // floor(2^32 / group) + 1 (0 for a group of 1): see row_token
  float scale_log2;  // scale * log2(e)
  int window;        // keys a token sees up to its own position; 0: all
  // selected attention: [tokens][topk] positions of idx_bytes each
  const void* idx;
  int64_t idx_stride;
  int idx_bytes, topk;
};

// r / group for r below 2^16 (groups up to 2^10): r (magic group - 2^32) < 2^32 / group holds, so
// the high half of r * magic is the quotient.
__device__ __forceinline__ int row_token(const PagedQuery& q, int r) {
  return q.group_magic ? static_cast<int>(__umulhi(static_cast<uint32_t>(r), q.group_magic)) : r;
}

// One item: rows [r0, r0 + rows) of the (token, head) rows of a sequence and key/value head.
struct PagedItem {
  int seq, head;      // sequence, key/value head
  int tok0;           // batch row of the sequence's (or the only) token 0
  int r0, rows;       // row range (row r: token tok0 + r / group, head h * group + r % group)
  int pos0;           // position of token 0
  int k0, k1;         // keys any row sees
  int u0, u1;         // units [u0, u1) of kUnit keys covering them (at least one)
};

template <int kRows, int kUnit>
__device__ __forceinline__ void paged_range_item(const PagedQuery& q, const SeqSpan& s, int rt,
                                                 PagedItem& it) {
  const int g = q.group;
  it.tok0 = s.q0;
  it.r0 = rt * kRows;
  it.rows = min(kRows, s.n * g - it.r0);
  it.pos0 = s.pos;
  const int first = it.pos0 + it.r0 / g;
  const int last = it.pos0 + (it.r0 + it.rows - 1) / g;
  it.k1 = min(max(0, last + 1), s.len);
  it.k0 = q.window > 0 ? max(0, first - (q.window - 1)) : 0;
  it.k0 = min(it.k0, it.k1);
  it.u0 = it.k0 / kUnit;
  it.u1 = max(it.u0 + 1, (it.k1 + kUnit - 1) / kUnit);
}

// Where CTA `cta` of at most `ctas` begins in the call's list of units (sequence, row tile,
// head, unit), found by all kThreads threads of the block from the sequences' unit counts.
struct PagedSlice {
  int64_t units, begin, end;
  int ctas;  // CTAs that have work: no more than there are units
  int seq, row_tile, head, off;
};

// Sum over the block's threads before this one, and over all of them.
template <int kThreads>
__device__ __forceinline__ int64_t block_scan(int64_t mine, int64_t* s_scan, int64_t& all) {
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_scan[w];
    all += s_scan[w];
  }
  __syncthreads();
  return before;
}

// Row tiles are numbered over the whole batch and shared out evenly, so that one long sequence
// costs no more than many short ones.  s_scan: kThreads / 32 values; s_first: kThreads values.
//
// CTAs.  An item of n units in p parts takes about n / p times the time of a unit and p times the
// time to add a part, which are alike (3600 and 3400 cycles), so p = sqrt(n) is the best split of
// few long items, four parts at least; more CTAs than that are left out.  (8 items of 128 rows
// and 64 units: 39 us with this bound, 60 without.)
template <int kThreads, int kRows, int kUnit>
__device__ __forceinline__ PagedSlice paged_find_slice(const PagedView& p, const PagedQuery& q,
                                                       int ctas, int cta, int64_t* s_scan,
                                                       int* s_first, int* s_found) {
  const int tid = threadIdx.x;
  const int chunk = (p.batch + kThreads - 1) / kThreads;
  auto tiles_of = [&](const SeqSpan& s) { return (s.n * q.group + kRows - 1) / kRows; };
  int64_t mine = 0, all_tiles;
  for (int b = tid * chunk; b < min(p.batch, (tid + 1) * chunk); ++b)
    mine += tiles_of(load_span(p, b));
  const int64_t first = block_scan<kThreads>(mine, s_scan, all_tiles);
  s_first[tid] = static_cast<int>(first);  // tiles: fewer than the call's rows, 2^30
  __syncthreads();

  // this thread's tiles [t0, t1): the sequence and the row tile of the first
  const int tiles = static_cast<int>(all_tiles);
  const int per = (tiles + kThreads - 1) / kThreads;
  const int t0 = min(tiles, tid * per), t1 = min(tiles, t0 + per);
  int b = 0, rt = 0;
  SeqSpan s = {};
  auto seek = [&]() {
    int lo = 0, hi = kThreads - 1;  // the last chunk that begins at or before t0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= t0) lo = mid;
      else hi = mid - 1;
    }
    b = lo * chunk;
    rt = t0 - s_first[lo];
    for (;; ++b) {
      s = load_span(p, b);
      const int n = tiles_of(s);
      if (rt < n) return;
      rt -= n;
    }
  };
  // calls f(units of the tile) for this thread's tiles until it returns false
  auto each = [&](auto&& f) {
    for (int t = t0; t < t1; ++t) {
      PagedItem x;
      paged_range_item<kRows, kUnit>(q, s, rt, x);
      if (!f(x.u1 - x.u0)) return;
      if (++rt == tiles_of(s) && t + 1 < t1) {
        rt = 0;
        do {
          s = load_span(p, ++b);
        } while (s.n == 0);
      }
    }
  };
  if (t0 < t1) seek();
  const int b_first = b, rt_first = rt;
  const SeqSpan s_first_span = s;
  int64_t sum = 0, all;
  each([&](int n) {
    sum += n;
    return true;
  });
  const int64_t before = block_scan<kThreads>(sum, s_scan, all);
  PagedSlice r;
  r.units = all * p.kv_heads;
  const float items = static_cast<float>(all_tiles) * p.kv_heads;
  const float most = fmaxf(4.f * items, sqrtf(static_cast<float>(r.units) * items));
  r.ctas = static_cast<int>(min(static_cast<int64_t>(ctas), r.units));
  if (most < r.ctas) r.ctas = max(1, static_cast<int>(most));
  r.begin = r.end = 0;
  r.seq = r.row_tile = r.head = r.off = 0;
  if (cta >= r.ctas) return r;
  r.begin = slice_begin(r.units, r.ctas, cta);
  r.end = slice_begin(r.units, r.ctas, cta + 1);
  int64_t at = before * p.kv_heads;
  if (r.begin >= at && r.begin < at + sum * p.kv_heads) {
    b = b_first;  // the slice begins in this thread's tiles
    rt = rt_first;
    s = s_first_span;
    each([&](int n) {
      const int64_t w = static_cast<int64_t>(n) * p.kv_heads;
      if (r.begin >= at + w) {
        at += w;
        return true;
      }
      const int64_t rest = r.begin - at;
      s_found[0] = b;
      s_found[1] = rt;
      const int64_t head = quotient(rest, n);
      s_found[2] = static_cast<int>(head);
      s_found[3] = static_cast<int>(rest - head * n);
      return false;
    });
  }
  __syncthreads();
  r.seq = s_found[0];
  r.row_tile = s_found[1];
  r.head = s_found[2];
  r.off = s_found[3];
  return r;
}

// The same for calls whose sequences have a row tile or two each (the decode step): a thread
// counts its sequences' units itself, which saves a pass over the block.
template <int kThreads, int kRows, int kUnit>
__device__ __forceinline__ PagedSlice paged_find_slice_few(const PagedView& p,
                                                           const PagedQuery& q, int ctas,
                                                           int cta, int64_t* s_scan,
                                                           int* s_found) {
  const int tid = threadIdx.x;
  const int chunk = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(p.batch, tid * chunk), b1 = min(p.batch, b0 + chunk);
  // calls f(sequence, row tile, units) until it returns false
  auto each = [&](auto&& f) {
    for (int b = b0; b < b1; ++b) {
      const SeqSpan s = load_span(p, b);
      PagedItem x;
      for (int t = 0; t * kRows < s.n * q.group; ++t) {
        paged_range_item<kRows, kUnit>(q, s, t, x);
        if (!f(b, t, x.u1 - x.u0)) return;
      }
    }
  };
  int64_t mine = 0, all;
  each([&](int, int, int n) {
    mine += n;
    return true;
  });
  int64_t at = block_scan<kThreads>(mine, s_scan, all) * p.kv_heads;
  PagedSlice r;
  r.units = all * p.kv_heads;
  r.ctas = static_cast<int>(min(static_cast<int64_t>(ctas), r.units));
  r.begin = r.end = 0;
  r.seq = r.row_tile = r.head = r.off = 0;
  if (cta >= r.ctas) return r;
  r.begin = slice_begin(r.units, r.ctas, cta);
  r.end = slice_begin(r.units, r.ctas, cta + 1);
  if (r.begin >= at && r.begin < at + mine * p.kv_heads) {
    each([&](int b, int t, int n) {
      const int64_t w = static_cast<int64_t>(n) * p.kv_heads;
      if (r.begin >= at + w) {
        at += w;
        return true;
      }
      const int64_t rest = r.begin - at, head = quotient(rest, n);
      s_found[0] = b;
      s_found[1] = t;
      s_found[2] = static_cast<int>(head);
      s_found[3] = static_cast<int>(rest - head * n);
      return false;
    });
  }
  __syncthreads();
  r.seq = s_found[0];
  r.row_tile = s_found[1];
  r.head = s_found[2];
  r.off = s_found[3];
  return r;
}

// The item after `it` in the list (there is one).
template <int kRows, int kUnit>
__device__ __forceinline__ void paged_next_item(const PagedView& p, const PagedQuery& q,
                                                SeqSpan& span, int& row_tile, PagedItem& it) {
  if (++it.head < p.kv_heads) return;
  it.head = 0;
  if (static_cast<int64_t>(++row_tile) * kRows >= static_cast<int64_t>(span.n) * q.group) {
    row_tile = 0;
    do {
      span = load_span(p, ++it.seq);
    } while (span.n == 0 && it.seq + 1 < p.batch);
  }
  paged_range_item<kRows, kUnit>(q, span, row_tile, it);
}

}  // namespace tdsa

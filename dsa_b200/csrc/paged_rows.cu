// Attention of few query rows over a paged key/value cache: the decode step (one or a few new
// tokens per sequence) and the attention over the positions a top-k selected.
//
//   out[t,h] = sum_j softmax_j(scale q[t,h].K[j]) V[j],  lse[t,h] = log sum_j exp(scale q.K[j])
//
// over the keys j that token t sees.  The rows of an item are the query heads that share one
// key/value head (times the sequence's new tokens), 16 MT of them, so every key and value is
// read from the cache once.
//
// HBM bound: a key and its value are 4 D bytes for 4 D rows multiply-adds.  32 ragged sequences
// (979 MB) take 168 us, 5.8 TB/s of the 6.55 that a copy reaches, and up to 6 % less on other
// cards; 2048 selected positions for 64 sequences (537 MB in pieces of 256 bytes) 96 us, 5.6
// TB/s; one sequence of 32768 positions (134 MB) 36 us, 9 of them before the first tile is there
// and after the last, and the slowest SM a third later than the fastest.  17 to 32 rows (16
// sequences of 8192, 537 MB) take 125 us at 128 features, 4.3 TB/s, and 80 at 64 (half the bytes),
// 3.4 TB/s: the instructions of two row tiles a key tile do not hide behind the loads.
//
// Layout.  A CTA is four or eight warps.  Each warp runs its own stream of 16-key tiles (a unit is
// a tile per warp) with its own ring of tiles in shared memory, filled by 16-byte asynchronous
// copies -- a row of the cache is gathered by address, so pages and selected positions cost the
// same -- and its own running maximum, sum and output in registers; warps meet only at the end of
// an item's segment.  No block-wide barrier is in the key loop.  S = Q K^T and O += P V are
// warp-level 16x8x16 matrix instructions with float32 accumulators: with 1 to 32 rows they keep
// the tensor pipe busy for a quarter of the time the keys take to arrive, and their operands and
// results stay in registers, which a tile of fewer rows than the 64 to 128 of a tcgen05
// instruction could not.
//
// Scores, maxima, sums and O are float32.  P enters the second product as a 16-bit value and a
// second one that holds what its rounding left (2^-16 relative in bf16; in f16 2^-22, or 2^-36 of
// the row's largest weight where that is more): twice the products, which are not what bounds this
// kernel -- 161 us against 160 with one term at 128 features, 149 against 142 at 64 -- for errors
// 0.7 times as large.
//
// Values of keys that no row of the item sees (past the length, or of a page that is not one)
// are zero-filled on arrival.  In a tile that some rows see and others do not, a value that is
// not finite would turn the zero weight of the others into NaN; such a tile's product is formed
// element by element.
#include <algorithm>

#include "paged.cuh"

namespace tdsa {

namespace {

constexpr int kPrNarrow = 4, kPrWide = 8;       // warps of a CTA (see launch_rows_d)
constexpr int kPrTile = 16;                     // keys per warp and tile

struct RowsArgs {
  PagedView p;
  PagedQuery q;
  PagedPartials part;
  int* status;
};

template <int D, int MT, bool kSel, int kWarps, bool kSolo = false>
struct RowsCfg {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTileBytes = kPrTile * kRowBytes;       // K or V tile
  static constexpr int kStageBytes = 2 * kTileBytes;
  // CTAs per SM, and tiles of a warp's ring (96 KB of ring per SM and more): selected keys of 64
  // features gain from more warps (683 tokens x 2 heads x 512: 38 us with 4 CTAs, 44 with 2), runs
  // of pages do not (11 sequences x 16 heads x 16461: 150 us against 141).
  static constexpr int kSmWarps = D == 64 && MT == 1 && kSel ? 16 : 8;
  static constexpr int kCtas = kSmWarps / kWarps;
  static constexpr int kStages = D == 128 || kSmWarps == 16 ? 3 : 6;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kRows = 16 * MT;
  static constexpr int kMergeO = kRows * D * 4;                // a warp's output, float32
  static constexpr int kRing = kWarps * kWarpBytes;
  static constexpr int kMl = kWarps * kRows * 8;
  // Queries are in registers where they fit beside the output.  32 rows of 128 features do not,
  // and a team reads them from shared memory for every tile (16 sequences of 8192, 4 tokens x 8
  // heads per group: 125 us, 168 with registers, of which 370 bytes spill).
  static constexpr bool kQShared = MT == 2 && D == 128 && !kSolo;
  static constexpr int kQ = (kRing + kMl + 256 + kWarps * kStages * 4 + 127) / 128 * 128;
  static constexpr int kSmem =
      kQShared ? kQ + kRows * kRowBytes : kRing + kMl + 256 + kWarps * kStages * 4;
  static_assert(kMergeO <= kWarpBytes, "a warp's output fits its ring");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool kBF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if (kBF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0 source bytes: the 16 bytes are zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// kSolo (selected attention): a warp takes items of its own instead of a quarter of the CTA's, so
// that nothing waits for the other warps where items are short and many.
template <bool kBF16, int D, int MT, bool kSel, bool kSolo, int kPrWarps>
__global__ void __launch_bounds__(kPrWarps * 32, RowsCfg<D, MT, kSel, kPrWarps, kSolo>::kCtas)
    paged_rows_kernel(const RowsArgs a) {
  using C = RowsCfg<D, MT, kSel, kPrWarps, kSolo>;
  constexpr int kPrThreads = kPrWarps * 32;
  constexpr int kPrUnit = kPrWarps * kPrTile;      // keys per unit of work
  static_assert(kSel || !kSolo, "");
  constexpr int kTeam = kSolo ? 1 : kPrWarps;      // warps that share an item
  constexpr int kUnitTiles = kPrWarps / kTeam;     // tiles of a unit per warp
  constexpr int kRows = C::kRows, kStages = C::kStages;
  constexpr float kGrow = WeightRange<kBF16>::kGrow, kBias = WeightRange<kBF16>::kBias;
  constexpr int kKs = D / 16;   // 16-wide steps of the head dimension
  constexpr int kNt = D / 8;    // 8-wide output tiles
  constexpr int kLanesPerRow = D / 8;
  constexpr int kRowsPerCopy = 32 / kLanesPerRow;
  extern __shared__ __align__(128) uint8_t smem[];
  // [warp of the team][row]
  float2* s_ml =
      reinterpret_cast<float2*>(smem + C::kRing) + (kSolo ? (threadIdx.x >> 5) * kRows : 0);
  int* s_meta = reinterpret_cast<int*>(smem + C::kRing + C::kMl);
  int64_t* s_scan = reinterpret_cast<int64_t*>(s_meta + 8);   // [warp] totals
  // [warp][stage]: bit r is set when row r of the stage's tile holds a key of the cache
  uint32_t* s_valid = reinterpret_cast<uint32_t*>(smem + C::kRing + C::kMl + 256) +
                      (threadIdx.x >> 5) * kStages;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quad = lane >> 2, ql = lane & 3;
  const int g = a.q.group, hkv = a.p.kv_heads;
  // the team, of so many; as many as there are units get work
  int ctas = gridDim.x * (kPrWarps / kTeam);
  const int cta = kSolo ? blockIdx.x * kPrWarps + warp : blockIdx.x;
  const int share = kSolo ? 0 : warp;         // of the team's warps
  const int member = kSolo ? lane : tid;      // of the team's threads
  auto team_sync = [&]() {
    if (kSolo) __syncwarp();
    else __syncthreads();
  };
  pdl_wait();
  pdl_launch_dependents();

  // ---------------------------------------------------------------- this CTA's slice
  int64_t units;       // of the whole call
  int64_t u_begin, u_end;
  PagedItem it;
  int rt = 0;          // row tile of the current item
  int off;             // unit of the item the slice begins at
  SeqSpan span;
  const int sel_units = kSel ? max(1, (a.q.topk + kPrUnit - 1) / kPrUnit) : 1;
  const int sel_rts = kSel ? (g + kRows - 1) / kRows : 1;
  // selected attention: items are (token, row tile, head); a token's sequence comes from the starts
  auto sel_token = [&](int t) {
    int c = 0;
    for (int b = lane; b < a.p.batch; b += 32) c += __ldg(a.p.starts + b + 1) <= t;
    c = __reduce_add_sync(0xffffffffu, c);
    it.seq = min(c, a.p.batch - 1);
    span = load_span(a.p, it.seq);
    it.tok0 = t;
    // a row before the first sequence or past the last one: nothing is read or written
    it.k1 = c >= a.p.batch || t < span.q0 ? 0 : a.q.topk;
    it.pos0 = it.k0 = it.u0 = 0;
    it.u1 = sel_units;
  };
  auto sel_rows = [&]() {
    it.r0 = rt * kRows;
    it.rows = it.k1 ? min(kRows, g - it.r0) : 0;
  };
  if (kSel) {
    units = static_cast<int64_t>(a.p.tokens) * sel_rts * hkv * sel_units;
    ctas = static_cast<int>(min(static_cast<int64_t>(ctas), units));
    if (cta >= ctas) return;
    u_begin = slice_begin(units, ctas, cta);
    u_end = slice_begin(units, ctas, cta + 1);
    const int64_t item = quotient(u_begin, sel_units);
    off = static_cast<int>(u_begin - item * sel_units);
    const int64_t tr = quotient(item, hkv);  // token and row tile
    const int t = static_cast<int>(quotient(tr, sel_rts));
    it.head = static_cast<int>(item - tr * hkv);
    rt = static_cast<int>(tr - static_cast<int64_t>(t) * sel_rts);
    sel_token(t);
    sel_rows();
  } else {
    const PagedSlice sl = paged_find_slice_few<kPrThreads, kRows, kPrUnit>(a.p, a.q, ctas,
                                                                           cta, s_scan, s_meta);
    units = sl.units;
    ctas = sl.ctas;
    if (cta >= ctas) return;
    u_begin = sl.begin;
    u_end = sl.end;
    it.seq = sl.seq;
    it.head = sl.head;
    rt = sl.row_tile;
    off = sl.off;
    span = load_span(a.p, it.seq);
    paged_range_item<kRows, kPrUnit>(a.q, span, rt, it);
  }

  uint8_t* ring = smem + warp * C::kWarpBytes;
  const uint32_t ring_u = smem_u32(ring);
  const uint32_t lm_k = ((lane >> 4) << 3) + (lane & 7);        // key row of a K ldmatrix lane
  const uint32_t lm_kc = (lane >> 3) & 1;                       // its 16-byte chunk (0/1)
  const uint32_t lm_v = (((lane >> 3) & 1) << 3) + (lane & 7);  // the same for V (transposed)
  const uint32_t lm_vc = lane >> 4;
  bool bad = false;  // a position or page outside the cache was named

  // The second term of P is p + second * (p rounded): what the rounding left, or the first once
  // more when a segment is formed again because its output was not finite (see there).
  float second = -1.f;
  for (int64_t u = u_begin; u < u_end;) {
    const int n_units = it.u1 - it.u0;
    const int seg = static_cast<int>(min(static_cast<int64_t>(n_units - off), u_end - u));
    const int unit0 = it.u0 + off;  // first unit of this segment

    // keys row ra / rb of m-tile m sees: [lo, hi)
    int lo[MT][2], hi[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = it.r0 + m * 16 + quad + 8 * e;
        const int p = it.pos0 + r / g;
        hi[m][e] = kSel ? it.k1 : min(p + 1, it.k1);
        lo[m][e] = kSel ? 0 : (a.q.window > 0 ? max(0, p - (a.q.window - 1)) : 0);
      }
    // keys that every row sees: tiles inside need no mask
    int all_lo = it.k0, all_hi = it.k1;
    if (!kSel) {
      all_hi = min(all_hi, it.pos0 + it.r0 / g + 1);
      if (a.q.window > 0)
        all_lo = max(all_lo, it.pos0 + (it.r0 + it.rows - 1) / g - (a.q.window - 1));
    }

    // ------------------------------------------------------------ key addresses
    // Pair pr of the warp's tiles (tiles 2 pr and 2 pr + 1, 32 keys): lane l holds the key of
    // row l.  raw: its position; then its page; then its offset, each loaded a pair ahead.
    const int32_t* table = a.p.table + it.seq * a.p.table_stride;
    const int cap = a.p.max_pages << a.p.page_shift;
    const int64_t head_off = it.head * a.p.head_stride;
    const int n_tiles = seg * kUnitTiles;
    auto tile_base = [&](int i) {  // first key of the warp's tile i
      return kSolo ? unit0 * kPrUnit + i * kPrTile : (unit0 + i) * kPrUnit + warp * kPrTile;
    };
    auto key_slot = [&](int pr) {  // index of lane l's key in the item's key list
      return tile_base(2 * pr + (lane >> 4)) + (lane & 15);
    };
    auto load_raw = [&](int pr) -> int {
      const int s = key_slot(pr);
      if (2 * pr + (lane >> 4) >= n_tiles) return -1;
      if (!kSel) return s >= it.k0 && s < it.k1 ? s : -1;
      if (s >= it.k1) return -1;
      const int64_t at = static_cast<int64_t>(it.tok0) * a.q.idx_stride + s;
      if (a.q.idx_bytes == 4) return __ldg(static_cast<const int32_t*>(a.q.idx) + at);
      const int64_t v = __ldg(static_cast<const long long*>(a.q.idx) + at);
      return v < 0 ? -1 : static_cast<int>(min(v, static_cast<int64_t>(0x7FFFFFFF)));
    };
    auto load_entry = [&](int raw) -> int {
      if (raw < 0) return -1;
      if (raw >= cap || (kSel && raw >= span.len)) return -2;
      return __ldg(table + (raw >> a.p.page_shift));
    };
    auto to_row = [&](int raw, int entry) -> int64_t {
      if (raw < 0) return -1;
      const int64_t r = paged_row(a.p, entry, raw);
      if (r < 0) bad = true;
      return r;
    };
    int64_t row_now, row_next;
    int raw2, entry2, raw3;  // of the pairs after row_next's
    {
      const int raw0 = load_raw(0), raw1 = load_raw(1);
      raw2 = load_raw(2);
      raw3 = load_raw(3);
      const int e0 = load_entry(raw0), e1 = load_entry(raw1);
      entry2 = load_entry(raw2);
      row_now = to_row(raw0, e0);
      row_next = to_row(raw1, e1);
    }
    int load_pair = 0;  // the pair of row_now
    uint32_t valid_now = __ballot_sync(0xffffffffu, row_now >= 0);

    // issue the copies of tile i of the segment (one group, empty past the end)
    auto issue = [&](int i) {
      if (i < n_tiles) {
        const int pr = i >> 1;
        if (pr != load_pair) {
          load_pair = pr;
          row_now = row_next;
          row_next = to_row(raw2, entry2);
          raw2 = raw3;
          entry2 = load_entry(raw2);
          raw3 = load_raw(pr + 3);
          valid_now = __ballot_sync(0xffffffffu, row_now >= 0);
        }
        if (lane == 0) s_valid[i % kStages] = (valid_now >> ((i & 1) * 16)) & 0xFFFFu;
        const uint32_t st = ring_u + (i % kStages) * C::kStageBytes;
        const int chunk = lane % kLanesPerRow;
#pragma unroll
        for (int c = 0; c < kPrTile / kRowsPerCopy; ++c) {
          const int r = c * kRowsPerCopy + lane / kLanesPerRow;
          const int64_t row = __shfl_sync(0xffffffffu, row_now, (i & 1) * 16 + r);
          const bool ok = row >= 0;
          const int64_t at = (ok ? row : 0) + head_off + chunk * 8;
          const uint32_t dst = st + r * C::kRowBytes + ((chunk ^ (r & 7)) << 4);
          cp_async16_fill(dst, a.p.keys + at, ok);
          cp_async16_fill(dst + C::kTileBytes, a.p.values + at, ok);
        }
      }
      cp_async_commit();
    };

#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // ------------------------------------------------------------ query fragments
    uint32_t qf[C::kQShared ? 1 : MT][C::kQShared ? 1 : kKs][4];
    const uint32_t s_q = smem_u32(smem + C::kQ);
    if (C::kQShared) {
      if (second != 0.f) {  // a warp that goes over its segment again finds them there
        for (int x = tid; x < kRows * kLanesPerRow; x += kPrThreads) {
          const int r = x / kLanesPerRow, c = x % kLanesPerRow;
          const int rr = it.r0 + r, tk = kSel ? 0 : rr / g;
          const uint16_t* from = a.q.q + static_cast<int64_t>(it.tok0 + tk) * a.q.q_ts +
                                 (it.head * g + rr - tk * g) * a.q.q_hs + c * 8;
          *reinterpret_cast<uint4*>(smem + C::kQ + r * C::kRowBytes + ((c ^ (r & 7)) << 4)) =
              r < it.rows ? *reinterpret_cast<const uint4*>(from) : make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();
      }
    } else {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int ra = it.r0 + m * 16 + quad, rb = ra + 8;
        const int lim = it.r0 + it.rows;
        const int ta = kSel ? 0 : ra / g, tb = kSel ? 0 : rb / g;
        const uint16_t* pa = a.q.q + static_cast<int64_t>(it.tok0 + ta) * a.q.q_ts +
                             (it.head * g + ra - ta * g) * a.q.q_hs + ql * 2;
        const uint16_t* pb = a.q.q + static_cast<int64_t>(it.tok0 + tb) * a.q.q_ts +
                             (it.head * g + rb - tb * g) * a.q.q_hs + ql * 2;
#pragma unroll
        for (int k = 0; k < kKs; ++k) {
          qf[m][k][0] = ra < lim ? *reinterpret_cast<const uint32_t*>(pa + k * 16) : 0u;
          qf[m][k][1] = rb < lim ? *reinterpret_cast<const uint32_t*>(pb + k * 16) : 0u;
          qf[m][k][2] = ra < lim ? *reinterpret_cast<const uint32_t*>(pa + k * 16 + 8) : 0u;
          qf[m][k][3] = rb < lim ? *reinterpret_cast<const uint32_t*>(pb + k * 16 + 8) : 0u;
        }
      }
    }
    // ------------------------------------------------------------ the key loop
    float o[MT][kNt][4];
    float mx[MT][2], sum[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int n = 0; n < kNt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][n][e] = 0.f;
      mx[m][0] = mx[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
    }
    for (int i = 0; i < n_tiles; ++i) {
      issue(i + kStages - 1);
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t st = ring_u + (i % kStages) * C::kStageBytes;
      const uint32_t vmask = s_valid[i % kStages];
      const int base = tile_base(i);
      float s[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < kKs; ++k) {
        uint32_t b[4];
        ldsm4(b, st + lm_k * C::kRowBytes + (((2 * k + lm_kc) ^ (lm_k & 7)) << 4));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t qs[4];
          if (C::kQShared)
            ldsm4(qs, s_q + (m * 16 + lm_v) * C::kRowBytes + (((2 * k + lm_vc) ^ (lm_v & 7)) << 4));
          const uint32_t(&qa)[4] = C::kQShared ? qs : qf[C::kQShared ? 0 : m][C::kQShared ? 0 : k];
          mma16816<kBF16>(s[m][0], qa, b[0], b[1]);
          mma16816<kBF16>(s[m][1], qa, b[2], b[3]);
        }
      }
      const bool whole = vmask == 0xFFFFu && base >= all_lo && base + kPrTile <= all_hi;
      if (!whole) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int c = n * 8 + ql * 2 + (e & 1);
              const bool see = ((vmask >> c) & 1u) && base + c >= lo[m][e >> 1] &&
                               base + c < hi[m][e >> 1];
              if (!see) s[m][n][e] = -INFINITY;
            }
      }
      // running maximum mx (a score): it moves only when a row's has grown by a factor of 2^8 or
      // 2^4 of weight (see WeightRange), so most tiles rescale nothing
      bool grow = false;
      float top[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = fmaxf(fmaxf(s[m][0][2 * e], s[m][0][2 * e + 1]),
                          fmaxf(s[m][1][2 * e], s[m][1][2 * e + 1]));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
          top[m][e] = t;
          grow |= (t - mx[m][e]) * a.q.scale_log2 > kGrow;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float now = fmaxf(mx[m][e], top[m][e]);
            const float f =
                now == mx[m][e] ? 1.f : exp2_approx((mx[m][e] - now) * a.q.scale_log2);
            mx[m][e] = now;
            sum[m][e] *= f;
#pragma unroll
            for (int n = 0; n < kNt; ++n) {
              o[m][n][2 * e] *= f;
              o[m][n][2 * e + 1] *= f;
            }
          }
      }
      uint32_t pf[MT][4], pl[MT][4];  // P rounded, and what the rounding left
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ref = mx[m][e] == -INFINITY ? 0.f : mx[m][e];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float p = exp2_approx(fmaf(s[m][n][2 * e + x] - ref, a.q.scale_log2, kBias));
              s[m][n][2 * e + x] = p;
              sum[m][e] += p;
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float u = s[m][x >> 1][2 * (x & 1)], w = s[m][x >> 1][2 * (x & 1) + 1];
          pf[m][x] = pack16<kBF16>(u, w);
          const float2 r = unpack16<kBF16>(pf[m][x]);
          pl[m][x] = pack16<kBF16>(fmaf(second, r.x, u), fmaf(second, r.y, w));
        }
      }
      const uint32_t sv = st + C::kTileBytes;
      bool slow = false;
      if (!kSel && !whole) {
        // does a value that only some rows see break the product with zero weights?
        for (int c = lane; c < kPrTile * kLanesPerRow; c += 32) {
          uint32_t x[4];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                       : "r"(sv + c * 16)
                       : "memory");
          slow |= nonfinite16<kBF16>(x[0]) || nonfinite16<kBF16>(x[1]) ||
                  nonfinite16<kBF16>(x[2]) || nonfinite16<kBF16>(x[3]);
        }
        slow = __any_sync(0xffffffffu, slow);
      }
      if (!slow) {
#pragma unroll
        for (int c = 0; c < kKs; ++c) {
          uint32_t b[4];
          ldsm4t(b, sv + lm_v * C::kRowBytes + (((2 * c + lm_vc) ^ (lm_v & 7)) << 4));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816<kBF16>(o[m][2 * c], pf[m], b[0], b[1]);
            mma16816<kBF16>(o[m][2 * c + 1], pf[m], b[2], b[3]);
            mma16816<kBF16>(o[m][2 * c], pl[m], b[0], b[1]);
            mma16816<kBF16>(o[m][2 * c + 1], pl[m], b[2], b[3]);
          }
        }
      } else {
        // element by element, only the keys a row sees, with the weight of both terms
        const float w_all = 2.f + second;
#pragma unroll
        for (int n2 = 0; n2 < 2; ++n2)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            for (int src = 0; src < 4; ++src) {
              const int c = n2 * 8 + src * 2 + x;
              const bool there = (vmask >> c) & 1u;
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const float pa = w_all * __shfl_sync(0xffffffffu, s[m][n2][x], (lane & ~3) | src);
                const float pb =
                    w_all * __shfl_sync(0xffffffffu, s[m][n2][2 + x], (lane & ~3) | src);
                const bool va = there && base + c >= lo[m][0] && base + c < hi[m][0];
                const bool vb = there && base + c >= lo[m][1] && base + c < hi[m][1];
#pragma unroll
                for (int n = 0; n < kNt; ++n) {
                  uint32_t w;
                  asm volatile("ld.shared.u32 %0, [%1];"
                               : "=r"(w)
                               : "r"(sv + c * C::kRowBytes + ((n ^ (c & 7)) << 4) + ql * 4)
                               : "memory");
                  const float2 v = unpack16<kBF16>(w);
                  if (va) {
                    o[m][n][0] = fmaf(pa, v.x, o[m][n][0]);
                    o[m][n][1] = fmaf(pa, v.y, o[m][n][1]);
                  }
                  if (vb) {
                    o[m][n][2] = fmaf(pb, v.x, o[m][n][2]);
                    o[m][n][3] = fmaf(pb, v.y, o[m][n][3]);
                  }
                }
              }
            }
      }
      __syncwarp();  // every lane is done with the stage before the next copies into it
    }
    cp_async_wait<0>();
    __syncwarp();
    // An infinite value times what the rounding left, which is zero or negative as often as not,
    // is NaN where the average is infinite.  Twice the first term is right, and is halved here.  A
    // warp goes back alone: the second time nothing up to here waits for other warps.  Segments
    // whose output is finite pay 1 to 2 % for the look at it where items are short, and nothing
    // that shows where they are long.
    if (second == 0.f) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < kNt; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][n][e] *= 0.5f;
    } else {
      uint64_t zero[2] = {0ull, 0ull};  // stays that when all are finite
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (m * 16 + 8 * e < it.rows) {
#pragma unroll
            for (int n = 0; n < kNt; ++n)
              zero[n & 1] = fma2(pair(o[m][n][2 * e], o[m][n][2 * e + 1]), 0ull, zero[n & 1]);
          }
      const float2 z0 = unpair(zero[0]), z1 = unpair(zero[1]);
      if (__any_sync(0xffffffffu, z0.x + z0.y + z1.x + z1.y != 0.f)) {
        second = 0.f;
        continue;
      }
    }
    second = -1.f;

    // ------------------------------------------------------------ the warps' results meet
    float* wo = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = sum[m][e];
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        const int r = m * 16 + quad + 8 * e;
        if (ql == 0) s_ml[share * kRows + r] = make_float2(mx[m][e], t);
        if (r < it.rows) {
#pragma unroll
          for (int n = 0; n < kNt; ++n)
            *reinterpret_cast<float2*>(wo + r * D + n * 8 + ql * 2) =
                make_float2(o[m][n][2 * e], o[m][n][2 * e + 1]);
        }
      }
    team_sync();
    const bool entire = seg == n_units;
    const int64_t item_u0 = u - off;  // the item's first unit in the call's list
    const int c_first = entire ? cta : slice_owner(units, ctas, item_u0);
    const int c_last = entire ? cta : slice_owner(units, ctas, item_u0 + n_units - 1);
    const int slot = 2 * cta + (cta == c_first ? 1 : 0);
    constexpr int kV = D / 4;              // float4 columns
    constexpr int kG = kTeam * 32 / kV;    // row groups
    const int col = member % kV, rg = member / kV;
    // adds up the team's results in shared memory and writes rows of the output, or a partial
    auto combine = [&](bool to_out) {
      for (int r = rg; r < it.rows; r += kG) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kTeam; ++w) m = fmaxf(m, s_ml[w * kRows + r].x);
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kTeam; ++w) {
          const float2 ml = s_ml[w * kRows + r];
          const float f = exp2_approx((ml.x - ref) * a.q.scale_log2);
          const uint8_t* from = kSolo ? ring : smem + w * C::kWarpBytes;
          const float4 x = *reinterpret_cast<const float4*>(
              reinterpret_cast<const float*>(from) + r * D + col * 4);
          if (ml.x != -INFINITY) {
            l += ml.y * f;
            v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
          } else {
            l += ml.y;  // zero, or NaN when a score was NaN
          }
        }
        if (to_out) {
          const int row = it.r0 + r, tk = kSel ? 0 : row / g;
          const int64_t t = it.tok0 + tk;
          const int h = it.head * g + row - tk * g;
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays NaN
          uint2 w;
          w.x = pack16<kBF16>(v.x * inv, v.y * inv);
          w.y = pack16<kBF16>(v.z * inv, v.w * inv);
          if (l == 0.f) w = make_uint2(0u, 0u);
          *reinterpret_cast<uint2*>(a.q.out + t * a.q.o_ts + h * a.q.o_hs + col * 4) = w;
          if (a.q.lse && col == 0)
            a.q.lse[t * a.q.heads + h] =
                l == 0.f ? -INFINITY
                         : (fmaf(m, a.q.scale_log2, -kBias) + log2f(l)) * 0.6931471805599453f;
        } else {
          if (col == 0) a.part.ml[static_cast<int64_t>(slot) * kRows + r] = make_float2(m, l);
          *reinterpret_cast<float4*>(a.part.o + (static_cast<int64_t>(slot) * kRows + r) * D +
                                     col * 4) = v;
        }
      }
    };
    combine(entire);
    if (!entire) {
      team_sync();
      bool last = false;
      if (member == 0)
        last = paged_arrive(a.part.counters + c_first, static_cast<uint32_t>(c_last - c_first + 1));
      if (kSolo) {
        last = __shfl_sync(0xffffffffu, last, 0);
      } else {
        if (member == 0) s_meta[4] = last;
        __syncthreads();
        last = s_meta[4] != 0;
      }
      if (last) {
        // The last to arrive adds the partials of teams c_first .. c_last up, four rows at a
        // time: a warp takes every kTeam-th partial where there are many, else every kTeam-th
        // group of rows; then the warps' sums meet as the segment's did.
        const int parts = c_last - c_first + 1;
        const bool by_part = parts >= 2 * kTeam;
        auto slot_of = [&](int p) { return 2 * static_cast<int64_t>(c_first + p) + (p == 0); };
        const int first = by_part ? share : 0, step = by_part ? kTeam : 1;
        const int count = (parts - first + step - 1) / step;
        for (int r = lane; r < kRows; r += 32) s_ml[share * kRows + r] = make_float2(-INFINITY, 0.f);
        __syncwarp();
        for (int r0 = by_part ? 0 : share * 4; r0 < it.rows; r0 += by_part ? 4 : 4 * kTeam) {
          float m[4], l[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) m[x] = -INFINITY, l[x] = 0.f;
          float4 v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int j0 = 0; j0 < count; j0 += 32) {
            const int p = first + (j0 + lane) * step;
            const bool in = j0 + lane < count;
            float2 ml[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              ml[x] = in && r0 + x < it.rows ? __ldcg(&a.part.ml[slot_of(p) * kRows + r0 + x])
                                             : make_float2(-INFINITY, 0.f);
            float f[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float now = ml[x].x;
#pragma unroll
              for (int o2 = 16; o2 > 0; o2 >>= 1)
                now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o2));
              now = fmaxf(now, m[x]);
              const float ref = now == -INFINITY ? 0.f : now;
              const float keep = exp2_approx((m[x] - ref) * a.q.scale_log2);
              f[x] = exp2_approx((ml[x].x - ref) * a.q.scale_log2);
              l[x] = l[x] * keep + ml[x].y * f[x];  // this lane's partials
              v[x].x *= keep, v[x].y *= keep, v[x].z *= keep, v[x].w *= keep;
              m[x] = now;
            }
            const int n = min(32, count - j0);
            const int lc = lane % kV;
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
              const int64_t sl_j = slot_of(first + (j0 + j) * step) * kRows;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float fx = __shfl_sync(0xffffffffu, f[x], j);
                if (r0 + x < it.rows) {
                  const float4 w = __ldcg(
                      reinterpret_cast<const float4*>(a.part.o + (sl_j + r0 + x) * D) + lc);
                  v[x].x += w.x * fx, v[x].y += w.y * fx;
                  v[x].z += w.z * fx, v[x].w += w.w * fx;
                }
              }
            }
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float t = l[x];
#pragma unroll
            for (int o2 = 16; o2 > 0; o2 >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o2);
            if (r0 + x < it.rows) {
              if (lane == 0) s_ml[share * kRows + r0 + x] = make_float2(m[x], t);
              if (lane < kV)
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(ring) + (r0 + x) * D +
                                           lane * 4) = v[x];
            }
          }
        }
        team_sync();
        combine(true);
      }
    }

    // ------------------------------------------------------------ the next item
    u += seg;
    if (u >= u_end) break;
    team_sync();  // the ring and s_ml are free again
    off = 0;
    if (kSel) {
      if (++it.head == hkv) {
        it.head = 0;
        if (++rt == sel_rts) {
          rt = 0;
          sel_token(it.tok0 + 1);
        }
        sel_rows();
      }
    } else {
      paged_next_item<kRows, kPrUnit>(a.p, a.q, span, rt, it);
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(a.status, TDSA_STATUS_RANGE);
}

template <bool kBF16, int D, int MT, bool kSel, bool kSolo, int kWarps>
int launch_rows_t(RowsArgs a, void* ws, cudaStream_t stream) {
  using C = RowsCfg<D, MT, kSel, kWarps, kSolo>;
  const int ctas = C::kCtas * device_sm_count(current_device());
  a.part = paged_partials(ws, ctas * (kSolo ? kWarps : 1), C::kRows);
  auto kern = paged_rows_kernel<kBF16, D, MT, kSel, kSolo, kWarps>;
  TDSA_CUDA_CHECK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmem));
  TDSA_CUDA_CHECK(launch_pdl(kern, dim3(static_cast<unsigned>(ctas)), dim3(kWarps * 32), C::kSmem,
                             stream, a));
  TDSA_CUDA_CHECK(cudaGetLastError());
  return TDSA_OK;
}

// Three layouts by the number of items a call can have (`most`).  With fewer than SMs, every item
// is split, and CTAs of eight warps leave half the parts to join of CTAs of four (2048 selected
// positions for one sequence: 10.9 us against 13.7); with more, smaller CTAs fill each other's
// pauses between items (32 ragged sequences x 8 heads: 160 us against 171).  Selected attention
// with an item for every warp leaves the teams out: 6225 tokens x 8 heads x 22 positions take 146
// us against 253; with 512 positions both take 36 us.
template <bool kBF16, int D, int MT>
int launch_rows_d(const RowsArgs& a, int rows, void* ws, cudaStream_t stream) {
  const int sms = device_sm_count(current_device());
  const int64_t tiles = (rows + 16 * MT - 1) / (16 * MT);
  const int64_t most = (a.q.idx ? a.p.tokens : a.p.batch) * tiles * a.p.kv_heads;
  if (!a.q.idx) {
    if (most <= sms) return launch_rows_t<kBF16, D, MT, false, false, kPrWide>(a, ws, stream);
    return launch_rows_t<kBF16, D, MT, false, false, kPrNarrow>(a, ws, stream);
  }
  if (most <= sms) return launch_rows_t<kBF16, D, MT, true, false, kPrWide>(a, ws, stream);
  if (most >= static_cast<int64_t>(RowsCfg<D, MT, true, kPrNarrow>::kSmWarps) * sms)
    return launch_rows_t<kBF16, D, MT, true, true, kPrNarrow>(a, ws, stream);
  return launch_rows_t<kBF16, D, MT, true, false, kPrNarrow>(a, ws, stream);
}

}  // namespace

size_t paged_rows_workspace_bytes(int dim) {
  // the most of any variant: teams of one warp, and their rows
  const int sms = device_sm_count(current_device());
  const int warps = dim == 128 ? RowsCfg<128, 1, true, kPrNarrow>::kSmWarps
                               : RowsCfg<64, 1, true, kPrNarrow>::kSmWarps;
  const int wide_rows = dim == 128 ? RowsCfg<128, 2, true, kPrNarrow>::kSmWarps
                                   : RowsCfg<64, 2, true, kPrNarrow>::kSmWarps;
  return std::max(paged_partial_bytes(warps * sms, 16, dim),
                  paged_partial_bytes(wide_rows * sms, 32, dim));
}

int launch_paged_rows(const PagedView& p, const PagedQuery& q, int dtype, int dim, int rows,
                      void* ws, int* status, cudaStream_t stream) {
  RowsArgs a;
  a.p = p;
  a.q = q;
  a.status = status;
  const bool narrow = rows <= 16;
  if (dtype == TDSA_BF16) {
    if (dim == 128)
      return narrow ? launch_rows_d<true, 128, 1>(a, rows, ws, stream)
                    : launch_rows_d<true, 128, 2>(a, rows, ws, stream);
    return narrow ? launch_rows_d<true, 64, 1>(a, rows, ws, stream)
                  : launch_rows_d<true, 64, 2>(a, rows, ws, stream);
  }
  if (dim == 128)
    return narrow ? launch_rows_d<false, 128, 1>(a, rows, ws, stream)
                  : launch_rows_d<false, 128, 2>(a, rows, ws, stream);
  return narrow ? launch_rows_d<false, 64, 1>(a, rows, ws, stream)
                : launch_rows_d<false, 64, 2>(a, rows, ws, stream);
}

}  // namespace tdsa

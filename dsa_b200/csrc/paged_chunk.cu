// Attention of a chunk of new tokens over a paged key/value cache on the tensor cores.
//
//   out[t,h] = sum_j softmax_j(scale q[t,h].K[j]) V[j] over the keys j that token t sees.
//
// An item is 256 query rows -- the (token, head) rows that share one key/value head -- in two
// tiles of 128, and walks its keys in units of 128, each in two parts of 64.  One CTA per SM;
// roles:
//   warps 0-3, 4-7: one tile each, one row per thread (softmax, output);
//   warp 8: the CTA's list of items, page lookups and TMA copies of K and V units into a ring
//     in shared memory (a unit is fetched once for both tiles);
//   warps 9, 10: one tile's tcgen05 products each, S = Q K^T (both from shared memory) and
//     O += P V (P from TMEM).
// TMEM holds two S buffers (64 columns) and O (D columns) per tile; P, 16-bit, takes the place
// of S once its thread has read the row.  S of part n + 2 is issued behind O += P V of part n,
// so a row finds the scores of its next part ready when it is done with one, and the time from
// P to the next S (products, and 500 cycles of their start and completion) is hidden behind a
// part's exponentials.  With one 128-wide S buffer per tile that time was not hidden: 3980
// cycles a unit against 2048 of products.
//
// The products that one thread issues complete in order, so the completion of S(n + 1) also
// says that O += P V of part n - 1 is done: the thread that owns a row waits for it before it
// rescales its row of O in place, which it does only when the row's maximum has grown by a
// factor of more than 2^8 of weight (2^4 in f16; rare after the first units).
//
// What bounds it.  A unit of both tiles is 2048 cycles of tensor work (2560 with S in parts of 64,
// whose operands shared memory delivers in 48 cycles instead of 32) and 3600 cycles of the rows'
// warps (3800 with clocks read in between): 64 scores of a row and part are read, compared and
// exponentiated in 1710 cycles with two warps on an SM quarter, 940 of them the exponentials, where
// the special-function pipe, the fma pipe (a third of the exponentials) and the latency of either
// add up.  Sixteen warps of rows with half a part each, and turns between the two tiles'
// exponentials, both measured the same.  4096 tokens over 16384 positions (32 heads in groups of
// 4, 128 features, 962 GFLOP): 0.87 ms alone, 1.11 PFLOP/s against the 1.67 of a library product;
// 1.00 ms, 0.96 PFLOP/s, in a loop that holds the card at its power limit, where the library
// product reaches 1.39.
//
// Scores, maxima, sums and O are float32.  P is rounded to the cache's type for the second
// product (2^-8 relative in bf16, 2^-11 in f16 or 2^-36 of the row's largest weight where that is
// more: the rounding that the output gets too; a second term for what it leaves would be half as
// much tensor work again); the sum adds the unrounded P.
#include <algorithm>

#include "paged.cuh"

namespace tdsa {

namespace {

constexpr int kPcThreads = 352;
constexpr int kPcTile = 128;           // rows of a tile
constexpr int kPcRows = 2 * kPcTile;   // rows of an item
constexpr int kPcUnit = 128;           // keys of a unit
constexpr int kPcPart = 64;            // keys of a part of a unit
constexpr int kPcHalf = kPcUnit * 128; // bytes of a 64-wide half of a unit (or of a Q tile)

struct ChunkArgs {
  PagedView p;
  PagedQuery q;
  PagedPartials part;
  int page_box;  // rows of a page's copy: min(page_size, 128)
  int* status;
};

template <int D>
struct ChunkCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kHalves * kPcHalf;  // K, V unit or Q tile
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kRing = kStages * kTileBytes;
  static constexpr int kQ = 2 * kTileBytes;
  static constexpr int kBar = 1024;
  static constexpr int kSmem = kRing + kQ + kBar + 1024;
  static constexpr int kOCol = 256;  // TMEM: S of tile t at 128 t, O of tile t at 256 + D t
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr)
               : "memory");
  return r;
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r));
  return r;
}

// The products are issued by the whole warp under the predicate of one lane: their operands
// stay in uniform registers, where a branch on the lane would move each of them there first
// (a group of eight took 720 to 910 cycles to issue that way, longer than it takes to run).
// D[tmem] (+)= A[smem desc] * B[smem desc]^T, kind::f16.
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc], A's 16-bit values packed two to a column.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void umma_commit_on(uint64_t* bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::
          "r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}

// Operand whose rows (keys) are the reduction: 64-wide halves kPcHalf apart (LBO), groups of
// 8 keys 1024 bytes apart (SBO), 128-byte swizzle.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) |
         (static_cast<uint64_t>(kPcHalf >> 4) << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}

// Two sums at once.
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Largest of three (two) values, NaN when one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max2_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// O += P V of one part for one row, element by element over its keys [j0, j1) that the row
// sees: P from TMEM (s_addr), V from its swizzled rows in shared memory.  first: O starts at 0.
template <bool kBF16, int D>
__device__ __noinline__ void add_visible(uint32_t s_addr, uint32_t o_addr, const uint8_t* sv,
                                         int j0, int j1, bool first) {
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    __syncwarp();
    if (!first) {
      tmem_ld32(o_addr + c * 32, o);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int x = 0; x < 32; ++x) o[x] = 0u;
    }
    for (int jp = 0; jp < kPcPart / 2; ++jp) {
      __syncwarp();
      const uint32_t w = tmem_ld1(s_addr + jp);
      tmem_wait_ld();
      const float2 pw = unpack16<kBF16>(w);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 2 * jp + e;
        if (j < j0 || j >= j1) continue;
        const float pj = e ? pw.y : pw.x;
        const uint8_t* vr = sv + (c >> 1) * kPcHalf + j * 128;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint4 v =
              *reinterpret_cast<const uint4*>(vr + ((((c & 1) * 4 + x) ^ (j & 7)) << 4));
          const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 f = unpack16<kBF16>(vv[y]);
            const int at = x * 8 + y * 2;
            o[at] = __float_as_uint(fmaf(pj, f.x, __uint_as_float(o[at])));
            o[at + 1] = __float_as_uint(fmaf(pj, f.y, __uint_as_float(o[at + 1])));
          }
        }
      }
    }
    __syncwarp();
    tmem_st32(o_addr + c * 32, o);
    tmem_wait_st();
  }
}

// A warp's wait: every lane gets the same answer, so a wait that runs out ends the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity,
                                          volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// 2^x of two values on the fma pipe, for x well below 2^22. x = n + f with n the nearest integer
// (read off the low bits of x + 1.5 2^23) and |f| <= 1/2, 2^f by the degree-4 polynomial of least
// largest relative error (2.6e-6, found by Remez exchange), n added to the exponent. x below -127 is
// taken as -127, whose sum of exponents is negative: the larger of it and 0 as integers makes the
// weight of a key that a row does not see exactly 0, as the special-function pipe does, and between
// -127 and -126 the result is some number below 2^-126. (A weight that stayed at 2^-126 would let
// a value near the type's largest through.)
__device__ __forceinline__ float2 exp2_poly2(uint64_t x2) {
  const float2 v = unpair(x2);
  const uint64_t x = pair(fmaxf(v.x, -127.f), fmaxf(v.y, -127.f));
  const uint64_t magic = pair(12582912.f, 12582912.f);
  const uint64_t r = add2(x, magic);
  const uint64_t n = add2(r, pair(-12582912.f, -12582912.f));
  const uint64_t f = fma2(n, pair(-1.f, -1.f), x);
  uint64_t p = fma2(pair(0x1.3997d6p-7f, 0x1.3997d6p-7f), f, pair(0x1.ca1440p-5f, 0x1.ca1440p-5f));
  p = fma2(p, f, pair(0x1.ec06dap-3f, 0x1.ec06dap-3f));
  p = fma2(p, f, pair(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
  p = fma2(p, f, pair(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  const float2 pv = unpair(p), rv = unpair(r);
  return make_float2(__int_as_float(max(__float_as_int(pv.x) + (__float_as_int(rv.x) << 23), 0)),
                     __int_as_float(max(__float_as_int(pv.y) + (__float_as_int(rv.y) << 23), 0)));
}

// The keys of a part (from `base` on) that a row sees of [lo, hi), a bit each; gone: bit x is set
// when keys 16 x .. 16 x + 15 are of no page.
__device__ __forceinline__ uint64_t seen_keys(int lo, int hi, int base, uint32_t gone) {
  const int from = max(0, lo - base), to = min(kPcPart, hi - base);
  const uint64_t below_to = to >= 64 ? ~0ull : (to <= 0 ? 0ull : (1ull << to) - 1);
  const uint64_t below_from = from >= 64 ? ~0ull : (1ull << from) - 1;
  uint64_t seen = below_to & ~below_from;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if ((gone >> x) & 1u) seen &= ~(0xFFFFull << (16 * x));
  return seen;
}

// A part's weights of one row, the maximum taken off the scores before the product (see
// WeightRange): S from TMEM, P to TMEM, their sum returned.  Not inlined: the code in the loop over
// parts cost every call 2 to 4 %.
template <bool kBF16>
__device__ __noinline__ float far_weights(uint32_t s_addr, int lo, int hi, uint32_t gone, float mx,
                                          float scale) {
  const uint64_t seen = seen_keys(lo, hi, 0, gone);
  const float t = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  for (int c = 0; c < 2; ++c) {
    uint32_t s[32], p[16];
    __syncwarp();
    tmem_ld32(s_addr + c * 32, s);
    tmem_wait_ld();
    const uint32_t w = static_cast<uint32_t>(seen >> (32 * c));
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float e[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float d = __uint_as_float(s[2 * j + x]) - t;
        e[x] = (w >> (2 * j + x)) & 1u
                   ? exp2_approx(fmaf(d, scale, WeightRange<kBF16>::kBias))
                   : 0.f;
        sum += e[x];
      }
      p[j] = pack16<kBF16>(e[0], e[1]);
    }
    tmem_st16(s_addr + c * 16, p);
  }
  return sum;
}

// A segment of an item, published by the copy warp to the others.
struct ChunkSegment {
  int unit0, units;    // first unit and number of units (0: the CTA's list ends)
  int item_units, rows;
  int64_t item_u0;     // the item's first unit in the call's list
  // row r of the item: rl = sub + r; token tok + rl / group at position pos + rl / group, query
  // head head0 + rl % group
  int head0, tok, pos, sub;
  int k0, k1;          // keys any row sees
};

template <bool kBF16, int D>
__global__ void __launch_bounds__(kPcThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const ChunkArgs a) {
  using C = ChunkCfg<D>;
  constexpr float kBias = WeightRange<kBF16>::kBias;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem + C::kRing;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_q + C::kQ);
  uint64_t* empty = full + C::kStages;
  uint64_t* qfull = empty + C::kStages;  // [tile]
  uint64_t* sfull = qfull + 2;           // [tile][buffer] S(n) and O += P V (n - 2) are complete
  uint64_t* pfull = sfull + 4;           // [tile][buffer] P(n) is in TMEM, O rescaled or read out
  uint64_t* met = pfull + 4;             // [tile] the tile's four warps meet
  uint64_t* gfull = met + 2;             // [2] a segment is published
  uint64_t* gempty = gfull + 2;          // [2] everyone is done with it
  uint64_t* done = gempty + 2;           // [tile]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // [tile][buffer]: the threads formed this part's O += P V themselves
  volatile int* skip = abort_flag + 1;
  volatile int* s_odd = abort_flag + 5;             // [tile][3] votes of the tile's warps
  int* s_last = const_cast<int*>(abort_flag) + 11;  // [tile]
  int* s_found = s_last + 2;             // [4]
  // [unit mod 16]: bit b is set when keys 16 b .. 16 b + 15 of the unit lie in a page that is
  // not the cache's (the ring holds fewer than 16 units)
  volatile uint32_t* absent = reinterpret_cast<volatile uint32_t*>(s_found + 4);
  int64_t* s_scan = reinterpret_cast<int64_t*>(
      (reinterpret_cast<uintptr_t>(s_found + 20) + 15) & ~uintptr_t(15));  // [12]
  ChunkSegment* s_seg = reinterpret_cast<ChunkSegment*>(s_scan + 12);      // [2]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&qfull[t], 4);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sfull[2 * t + b], 1);
        mbar_init(&pfull[2 * t + b], 4);
        skip[2 * t + b] = 0;
      }
      for (int v = 0; v < 3; ++v) s_odd[3 * t + v] = 0;
      mbar_init(&gfull[t], 1);
      mbar_init(&gempty[t], 10);
      mbar_init(&done[t], 1);
      mbar_init(&met[t], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  if (warp == 9) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();
  pdl_launch_dependents();

  const PagedSlice sl = paged_find_slice<kPcThreads, kPcRows, kPcUnit>(
      a.p, a.q, gridDim.x, blockIdx.x, s_scan, reinterpret_cast<int*>(smem), s_found);
  fence_proxy_async_smem();  // the ring was its scratch: copies may write there after this
  __syncthreads();

  if (warp == 8) {
    // ------------------------------------------------------------ the list, copies of K and V
    const int box = a.page_box, boxes = kPcUnit / box;
    uint32_t n_loads = 0, n_seg = 0;
    bool bad = false, ok = true;
    PagedItem it = {};
    SeqSpan span = {};
    int rt = sl.row_tile, off = sl.off;
    int64_t u = sl.begin;
    if (u < sl.end) {
      it.seq = sl.seq;
      it.head = sl.head;
      span = load_span(a.p, it.seq);
      paged_range_item<kPcRows, kPcUnit>(a.q, span, rt, it);
    }
    while (ok) {
      const bool end = u >= sl.end;
      const int n = end ? 0 : it.u1 - it.u0;
      const int seg = end ? 0 : static_cast<int>(min(static_cast<int64_t>(n - off), sl.end - u));
      const uint32_t gs = n_seg & 1u;
      if (!warp_wait(&gempty[gs], ((n_seg >> 1) & 1u) ^ 1u, abort_flag)) break;
      if (lane == 0) {
        ChunkSegment g;
        g.unit0 = it.u0 + off;
        g.units = seg;
        g.item_units = n;
        g.item_u0 = u - off;
        g.rows = it.rows;
        const int t0 = it.r0 / a.q.group;
        g.head0 = it.head * a.q.group;
        g.tok = it.tok0 + t0;
        g.pos = it.pos0 + t0;
        g.sub = it.r0 - t0 * a.q.group;
        g.k0 = it.k0, g.k1 = it.k1;
        s_seg[gs] = g;
        mbar_arrive(&gfull[gs]);
      }
      __syncwarp();
      ++n_seg;
      if (end) break;
      const int unit0 = it.u0 + off;
      const int32_t* table = a.p.table + it.seq * a.p.table_stride;
      // lane l looks up the page of the unit's l-th box; positions no row sees are not looked
      // up, and like pages that are not the cache's they are read past its end, as zeros
      auto entry_of = [&](int i) {
        const int pos = (unit0 + i) * kPcUnit + lane * box;
        if (i >= seg || lane >= boxes || pos >= it.k1 || pos + box <= it.k0) return a.p.pages;
        return __ldg(table + (pos >> a.p.page_shift));
      };
      int entry = entry_of(0);
      for (int i = 0; i < seg && ok; ++i) {
        const int pos = (unit0 + i) * kPcUnit + lane * box;
        int page = entry;
        if (page < 0 || page > a.p.pages) page = a.p.pages;
        const bool none = page == a.p.pages && lane < boxes && pos < it.k1 && pos + box > it.k0;
        const uint32_t gone = __ballot_sync(
            0xffffffffu, __shfl_sync(0xffffffffu, none, (lane * 16 / box) & 31) && lane < 8);
        bad |= gone != 0u;
        if (lane == 0) absent[(n_loads >> 1) & 15] = gone;
        entry = entry_of(i + 1);
        const int at = (unit0 + i) * kPcUnit & ((1 << a.p.page_shift) - 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t s = n_loads % C::kStages, ph = (n_loads / C::kStages) & 1u;
          if (!warp_wait(&empty[s], ph ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[s], C::kTileBytes);
          __syncwarp();
          uint8_t* dst = smem + s * C::kTileBytes;
          const int from = __shfl_sync(0xffffffffu, page, (lane / C::kHalves) & 31);
          const int b = lane / C::kHalves, h = lane % C::kHalves;
          if (b < boxes)
            tma_load_4d(dst + h * kPcHalf + b * box * 128, kv ? &vmap : &kmap, &full[s], h * 64,
                        boxes > 1 ? 0 : at, it.head, from);
          ++n_loads;
        }
      }
      u += seg;
      if (u < sl.end) {
        off = 0;
        paged_next_item<kPcRows, kPcUnit>(a.p, a.q, span, rt, it);
      }
    }
    __syncwarp();
    if (bad && lane == 0) atomicOr(a.status, TDSA_STATUS_RANGE);
    // every issued copy lands before the CTA can exit
    volatile int no_abort = 0;
    for (uint32_t s = 0; s < C::kStages && s < n_loads; ++s) {
      const uint32_t n = (n_loads - s + C::kStages - 1) / C::kStages;
      mbar_wait(&full[s], (n - 1) & 1u, &no_abort);
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ rows: softmax and output
    const int t = warp >> 2;                      // tile
    const int row = (warp & 3) * 32 + lane;       // of the tile; also the TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>(warp & 3) << 21;
    const uint32_t s_addr = tmem + lane_base + t * 128;
    const uint32_t o_addr = tmem + lane_base + C::kOCol + t * D;
    const float scale = a.q.scale_log2, grow = WeightRange<kBF16>::kGrow / scale;
    // one bit per buffer: the parity of its next S, and whether its last product was the threads'
    uint32_t s_ph = 0, was_alone = 0;
    uint32_t n_unit = 0;  // units of the CTA's list before the segment
    // the tile's warps meet (a bounded wait); false when the CTA aborts
    uint32_t met_n = 0;
    int vote = 0;
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&met[t]);
      return warp_wait(&met[t], met_n++ & 1u, abort_flag);
    };
    for (uint32_t n_seg = 0;; ++n_seg) {
      const ChunkSegment* sg = &s_seg[n_seg & 1u];
      if (!warp_wait(&gfull[n_seg & 1u], (n_seg >> 1) & 1u, abort_flag)) break;
      const int units = sg->units;
      if (units == 0) break;
      if (t == 1 && sg->rows <= kPcTile) {
        n_unit += units;
        __syncwarp();
        if (lane == 0) mbar_arrive(&gempty[n_seg & 1u]);
        continue;
      }
      const int g = a.q.group;
      const int w_row0 = t * kPcTile + (warp & 3) * 32;    // the warp's first row
      const int w_rows = min(32, sg->rows - w_row0);       // its rows (none: <= 0)
      const bool valid = lane < w_rows;
      // the address of 16 bytes of row r of the warp's, chunk c: whole rows side by side
      constexpr int kLanes = D / 8;
      const int my_c = lane % kLanes;
      auto row_at = [&](auto* p, int64_t ts, int64_t hs, int r) {
        const int rl = sg->sub + w_row0 + r, tk = row_token(a.q, rl);
        return p + static_cast<int64_t>(sg->tok + tk) * ts + (sg->head0 + rl - tk * g) * hs +
               my_c * 8;
      };
      // the warp's rows of the query tile (later of the output): chunk c of row r
      uint8_t* const s_rows = s_q + t * C::kTileBytes + (warp & 3) * 32 * 128;
      auto staged = [&](int r, int c) {
        return reinterpret_cast<uint4*>(s_rows + (c >> 3) * kPcHalf + r * 128 +
                                        (((c & 7) ^ (r & 7)) << 4));
      };
      int lo, hi, all_lo, all_hi;  // keys this row sees; keys every row of the tile sees
      {
        // every load is under way before the first is stored
        constexpr int kStep = 32 / kLanes;
        uint4 x[kLanes];
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
          const int r = lane / kLanes + i * kStep;
          x[i] = r < w_rows
                     ? *reinterpret_cast<const uint4*>(row_at(a.q.q, a.q.q_ts, a.q.q_hs, r))
                     : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < kLanes; ++i) *staged(lane / kLanes + i * kStep, my_c) = x[i];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfull[t]);
        const int w = a.q.window;
        const int pos = sg->pos + row_token(a.q, sg->sub + w_row0 + lane);
        const int first = sg->pos + row_token(a.q, sg->sub + t * kPcTile);
        const int last =
            sg->pos + row_token(a.q, sg->sub + min(sg->rows, (t + 1) * kPcTile) - 1);
        hi = valid ? min(pos + 1, sg->k1) : sg->k1;
        lo = valid && w > 0 ? max(0, pos - (w - 1)) : 0;
        all_hi = min(sg->k1, first + 1);
        all_lo = w > 0 ? max(sg->k0, last - (w - 1)) : sg->k0;
      }
      float mx = -INFINITY, sum = 0.f;  // the running maximum, a score
      // A weight is 2^(s scale + add), the difference from the maximum formed by one fma.  Where
      // the rounding of mx scale would show, past 2^20 units in any row of the warp, far_weights
      // forms them; every part then counts as past the limit, so that others pay nothing for it.
      float add = 0.f;
      float limit = -INFINITY;  // a score above it moves the maximum
      int base = sg->unit0 * kPcUnit;
      bool ok = true;
      for (int i = 0; i < units && ok; ++i) {
#pragma unroll 1
        for (int b = 0; b < 2; ++b, base += kPcPart) {
          ok = warp_wait(&sfull[2 * t + b], (s_ph >> b) & 1u, abort_flag);
          if (!ok) break;
          s_ph ^= 1u << b;
          tc_fence_after();
          const uint32_t sb = s_addr + b * kPcPart;
          uint32_t s[2][32];
          tmem_ld32(sb, s[0]);
          tmem_ld32(sb + 32, s[1]);
          // written before the unit's copies were, so it is there when S is
          const uint32_t gone = (absent[(n_unit + i) & 15] >> (4 * b)) & 15u;
          const bool masked = base < all_lo || base + kPcPart > all_hi || gone;
          if (((was_alone >> b) & 1u) && !masked) {  // the tensor core's again
            if (row == 0) skip[2 * t + b] = 0;
            was_alone &= ~(1u << b);
          }
          tmem_wait_ld();
          if (masked) {
            const uint64_t seen = seen_keys(lo, hi, base, gone);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t w = static_cast<uint32_t>(seen >> (32 * c));
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((w >> j) & 1u)) s[c][j] = 0xFF800000u;  // -infinity
            }
          }
          float tops[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t* x = s[c >> 1] + (c & 1) * 16;
            tops[c] =
                max3_nan(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
#pragma unroll
            for (int j = 3; j < 15; j += 2)
              tops[c] = max3_nan(tops[c], __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
            tops[c] = max2_nan(tops[c], __uint_as_float(x[15]));
          }
          const float top = max2_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3]);
          if (__any_sync(0xffffffffu, top > limit)) {
            const float now = fmaxf(mx, top);
            const float f = now == mx ? 1.f : exp2_approx((mx - now) * scale);
            mx = now;
            const float ref = fmaf(mx, scale, -kBias);
            add = mx == -INFINITY ? 0.f : -ref;
            limit = mx + grow;
            sum *= f;
            if (i > 0 || b > 0) {
              // O += P V of the part before is complete with the S after this one
              ok = warp_wait(&sfull[2 * t + (b ^ 1)], (s_ph >> (b ^ 1)) & 1u, abort_flag);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(o_addr + c * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                tmem_st16(o_addr + c * 16, o);
              }
            }
            if (__any_sync(0xffffffffu, fabsf(add) > 0x1p20f)) {
              sum += far_weights<kBF16>(sb, lo - base, hi - base, gone, mx, scale);
              limit = -INFINITY;
              goto weighed;
            }
          }
          {
            // A score that is NaN or +infinity makes the whole row NaN: the polynomial below would
            // drop it, so it is carried into every weight of the part.
            const float neg = top < INFINITY ? add : __int_as_float(0x7FFFFFFF);
            const uint64_t scale2 = pair(scale, scale), neg2 = pair(neg, neg);
            uint64_t part[2] = {0ull, 0ull};
            // a third of the pairs take the polynomial
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t p[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const uint64_t x2 =
                    fma2(pair(__uint_as_float(s[c][2 * j]), __uint_as_float(s[c][2 * j + 1])),
                         scale2, neg2);
                float2 e;
                if (j % 3 == 1) {
                  e = exp2_poly2(x2);
                } else {
                  const float2 x = unpair(x2);
                  e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                }
                part[j & 1] = add2(part[j & 1], pair(e.x, e.y));
                p[j] = pack16<kBF16>(e.x, e.y);
              }
              tmem_st16(sb + c * 16, p);
            }
            {
              const float2 x = unpair(add2(part[0], part[1]));
              sum += x.x + x.y;
            }
          }
        weighed:
          tmem_wait_st();
          if (masked) {
            // A value that only some rows see and that is not finite: zero weights times it
            // would be NaN for the others, so the threads then form this part's product
            // themselves.
            const uint32_t vi = 2 * (n_unit + i) + 1;  // K, V, K, V, ... fill the ring
            const uint32_t st = vi % C::kStages;
            ok = warp_wait(&full[st], (vi / C::kStages) & 1u, abort_flag);
            if (!ok) break;
            const uint8_t* sv = smem + st * C::kTileBytes + b * kPcPart * 128;
            const int key0 = sg->k0 - base, key1 = sg->k1 - base;
            uint32_t odd = 0u;
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {  // 16 bytes at a time, side by side
              const int c = (x & 3) * kPcTile + row;
              const uint4 w = *reinterpret_cast<const uint4*>(sv + (x >> 2) * kPcHalf + c * 16);
              const uint32_t bits = nonfinite_bits<kBF16>(w.x) | nonfinite_bits<kBF16>(w.y) |
                                    nonfinite_bits<kBF16>(w.z) | nonfinite_bits<kBF16>(w.w);
              if ((c >> 3) >= key0 && (c >> 3) < key1) odd |= bits;
            }
            // three ballots in turn: the next one was last read before the meeting before this
            if (__any_sync(0xffffffffu, odd & 0x80008000u) && lane == 0) s_odd[3 * t + vote] = 1;
            if (row == 0) s_odd[3 * t + (vote == 2 ? 0 : vote + 1)] = 0;
            ok = meet();
            if (!ok) break;
            const bool alone = s_odd[3 * t + vote] != 0;
            vote = vote == 2 ? 0 : vote + 1;
            if (alone) {
              ok = warp_wait(&sfull[2 * t + (b ^ 1)], (s_ph >> (b ^ 1)) & 1u, abort_flag);
              if (!ok) break;
              tc_fence_after();
              add_visible<kBF16, D>(sb, o_addr, sv, max(0, lo - base), min(kPcPart, hi - base),
                                    i == 0 && b == 0);
            }
            if (row == 0) skip[2 * t + b] = alone ? 1 : 0;
            was_alone = (was_alone & ~(1u << b)) | (static_cast<uint32_t>(alone) << b);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pfull[2 * t + b]);
        }
      }
      n_unit += units;

      // ---------------------------------------------------------- output
      for (int b = 0; b < 2; ++b)
        if (ok) ok = warp_wait(&sfull[2 * t + b], (s_ph >> b) & 1u, abort_flag);
      s_ph ^= 3u;
      if (!ok) break;
      tc_fence_after();
      const int r_item = t * kPcTile + row;  // row of the item
      int c_first = 0, c_last = 0;  // CTAs that hold parts of the item
      bool write = true;
      if (units != sg->item_units) {
        c_first = slice_owner(sl.units, sl.ctas, sg->item_u0);
        c_last = slice_owner(sl.units, sl.ctas, sg->item_u0 + sg->item_units - 1);
        // a part of the item: float32, the rows of a column quad side by side
        const int cta = blockIdx.x;
        const int64_t slot = 2 * cta + (cta == c_first ? 1 : 0);
        a.part.ml[slot * kPcRows + r_item] = make_float2(fmaf(mx, scale, -kBias), sum);
        float4* dst = reinterpret_cast<float4*>(a.part.o + slot * kPcRows * D) + r_item;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 8; ++x)
            dst[(c * 8 + x) * kPcRows] =
                make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                            __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
        }
        if (!meet()) break;
        if (row == 0)
          s_last[t] = paged_arrive(a.part.counters + 2 * c_first + t,
                                   static_cast<uint32_t>(c_last - c_first + 1));
        if (!meet()) break;
        write = s_last[t] != 0;
      }
      if (write) {
        float m = fmaf(mx, scale, -kBias), l = sum;
        const bool split = units != sg->item_units;
        auto slot_of = [&](int c) { return (2 * static_cast<int64_t>(c) + (c == c_first)) * kPcRows; };
        if (split) {  // the last to arrive adds the parts up, in the CTAs' order
          m = -INFINITY;
          l = 0.f;
#pragma unroll 4
          for (int c = c_first; c <= c_last; ++c)
            m = fmaxf(m, __ldcg(&a.part.ml[slot_of(c) + r_item]).x);
        }
        const float mr = m == -INFINITY ? 0.f : m;
        if (split) {
#pragma unroll 4
          for (int c = c_first; c <= c_last; ++c) {
            const float2 ml = __ldcg(&a.part.ml[slot_of(c) + r_item]);
            l += ml.y * exp2_approx(ml.x - mr);
          }
        }
        // a row that sees no key has no maximum; one whose scores are all NaN has a NaN sum
        const bool none = m == -INFINITY && l == l;
        const float inv = 1.f / l;
        // 16-bit rows by way of the warp's own rows of the queries, which nothing reads any
        // more, then whole rows side by side to memory
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          if (split) {
#pragma unroll
            for (int x = 0; x < 32; ++x) v[x] = 0.f;
            for (int k = c_first; k <= c_last; ++k) {
              const int64_t sl_k = slot_of(k);
              const float f = exp2_approx(__ldcg(&a.part.ml[sl_k + r_item]).x - mr);
              const float4* o = reinterpret_cast<const float4*>(a.part.o + sl_k * D) + r_item;
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float4 w = __ldcg(o + (c * 8 + x) * kPcRows);
                v[4 * x] += w.x * f, v[4 * x + 1] += w.y * f;
                v[4 * x + 2] += w.z * f, v[4 * x + 3] += w.w * f;
              }
            }
          } else {
            uint32_t o[32];
            tmem_ld32(o_addr + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(o[x]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w[y] = none ? 0u : pack16<kBF16>(v[x * 8 + 2 * y] * inv, v[x * 8 + 2 * y + 1] * inv);
            *staged(lane, c * 4 + x) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        {
          constexpr int kStep = 32 / kLanes;
          uint4 x[kLanes];
#pragma unroll
          for (int i = 0; i < kLanes; ++i) x[i] = *staged(lane / kLanes + i * kStep, my_c);
#pragma unroll
          for (int i = 0; i < kLanes; ++i) {
            const int r = lane / kLanes + i * kStep;
            if (r < w_rows)
              *reinterpret_cast<uint4*>(row_at(a.q.out, a.q.o_ts, a.q.o_hs, r)) = x[i];
          }
        }
        __syncwarp();
        if (valid && a.q.lse) {
          const int rl = sg->sub + r_item, tk = row_token(a.q, rl);
          a.q.lse[static_cast<int64_t>(sg->tok + tk) * a.q.heads + sg->head0 + rl - tk * g] =
              none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&gempty[n_seg & 1u]);
    }
  } else {
    // ------------------------------------------------------------ tensor products of a tile
    const int t = warp - 9;
    constexpr uint32_t idesc_s = umma_idesc_f16(kBF16, kPcTile, kPcPart);
    constexpr uint32_t idesc_o = umma_idesc_f16(kBF16, kPcTile, D) | (1u << 16);
    const uint32_t one = elect_one();
    const uint32_t qa = smem_u32(s_q) + t * C::kTileBytes, ring_base = smem_u32(smem);
    uint32_t stage = 0, stage_ph = 0;  // the ring's next stage
    uint32_t q_ph = 0, p_ph = 0;
    auto take = [&](uint32_t& s) -> bool {
      s = stage;
      if (!warp_wait(&full[s], stage_ph, abort_flag)) return false;
      if (++stage == C::kStages) stage = 0, stage_ph ^= 1u;
      return true;
    };
    auto issue_s = [&](uint32_t s, int b) {  // keys 64 b .. of the unit, into buffer b
      const uint32_t ka = ring_base + s * C::kTileBytes + b * kPcPart * 128;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        umma_ss(tmem + t * 128 + b * kPcPart,
                sw128_kmajor_desc(qa + (k >> 2) * kPcHalf + (k & 3) * 32),
                sw128_kmajor_desc(ka + (k >> 2) * kPcHalf + (k & 3) * 32), idesc_s,
                k > 0 ? 1u : 0u, one);
    };
    bool ok = true;
    for (uint32_t n_seg = 0; ok; ++n_seg) {
      const uint32_t gs = n_seg & 1u;
      if (!warp_wait(&gfull[gs], (n_seg >> 1) & 1u, abort_flag)) break;
      const int units = s_seg[gs].units;
      const int base0 = s_seg[gs].unit0 * kPcUnit;
      const int k0 = s_seg[gs].k0, k1 = s_seg[gs].k1;
      const bool mine = t == 0 || s_seg[gs].rows > kPcTile;
      __syncwarp();
      if (lane == 0) mbar_arrive(&gempty[gs]);
      if (units == 0) break;
      uint32_t ks = 0, vs = 0;
      if (!mine) {  // the item has one tile: only hand the stages on
        for (int i = 0; i < 2 * units && ok; ++i) {
          ok = take(ks);
          if (ok && lane == 0) mbar_arrive(&empty[ks]);
          __syncwarp();
        }
        continue;
      }
      ok = take(ks) && warp_wait(&qfull[t], q_ph, abort_flag);
      q_ph ^= 1u;
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        issue_s(ks, b);
        umma_commit_on(&sfull[2 * t + b], one);
      }
      umma_commit_on(&empty[ks], one);
      for (int i = 0; i < units; ++i) {
        ok = take(vs);
        if (!ok) break;
        // rows of V that no row of the item sees may hold anything: zero weights times
        // infinities or NaN would be NaN, so they become zeros (both tiles' warps write them)
        const int base = base0 + i * kPcUnit;
        if (base < k0 || base + kPcUnit > k1) {
          for (int x = lane; x < C::kHalves * kPcUnit * 8; x += 32) {
            const int r = (x >> 3) & (kPcUnit - 1);
            if (base + r < k0 || base + r >= k1)
              *reinterpret_cast<uint4*>(smem + vs * C::kTileBytes + x * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        const bool more = i + 1 < units;
        if (more) ok = take(ks);
        if (!ok) break;
        const uint32_t va = ring_base + vs * C::kTileBytes;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (ok) ok = warp_wait(&pfull[2 * t + b], p_ph, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t on = skip[2 * t + b] ? 0u : one;
#pragma unroll
          for (int k = 0; k < kPcPart / 16; ++k)
            umma_ts(tmem + C::kOCol + t * D, tmem + t * 128 + b * kPcPart + k * 8,
                    sw128_mnmajor_desc(va + (4 * b + k) * 2048), idesc_o,
                    (i > 0 || b > 0 || k > 0) ? 1u : 0u, on);
          if (more) issue_s(ks, b);
          // past the last part too: its second commit says that O is complete
          umma_commit_on(&sfull[2 * t + b], one);
        }
        if (!ok) break;
        p_ph ^= 1u;
        umma_commit_on(&empty[vs], one);
        if (more) umma_commit_on(&empty[ks], one);
      }
    }
    __syncwarp();
    umma_commit_on(&done[t], one);
    volatile int no_abort = 0;
    mbar_wait(&done[t], 0, &no_abort);
  }

  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(a.status, TDSA_ERR_TIMEOUT);
}

template <bool kBF16, int D>
int launch_chunk_t(const ChunkArgs& a, const CUtensorMap& kmap, const CUtensorMap& vmap, int ctas,
                   cudaStream_t stream) {
  auto kern = paged_chunk_kernel<kBF16, D>;
  TDSA_CUDA_CHECK(
      ensure_dynamic_smem(reinterpret_cast<const void*>(kern), ChunkCfg<D>::kSmem));
  TDSA_CUDA_CHECK(launch_pdl(kern, dim3(static_cast<unsigned>(ctas)), dim3(kPcThreads),
                             ChunkCfg<D>::kSmem, stream, kmap, vmap, a));
  TDSA_CUDA_CHECK(cudaGetLastError());
  return TDSA_OK;
}

}  // namespace

size_t paged_chunk_workspace_bytes(int dim) {
  return paged_partial_bytes(device_sm_count(current_device()), kPcRows, dim);
}

int launch_paged_chunk(const PagedView& p, const PagedQuery& q, int dtype, int dim, void* ws,
                       int* status, cudaStream_t stream) {
  ChunkArgs a;
  a.p = p;
  a.q = q;
  a.status = status;
  const int ctas = device_sm_count(current_device());
  a.part = paged_partials(ws, ctas, kPcRows);
  const int page = 1 << p.page_shift;
  a.page_box = std::min(page, kPcUnit);
  CUtensorMap maps[2];
  // [pages][kv_heads][page_size][dim]; strides of axes of extent 1 are never used
  const uint64_t rs = static_cast<uint64_t>(p.row_stride) * 2;
  const uint64_t hs = p.kv_heads > 1 ? static_cast<uint64_t>(p.head_stride) * 2 : rs;
  const uint64_t ps = p.pages > 1 ? static_cast<uint64_t>(p.page_stride) * 2 : rs * page;
  const uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(page),
                            static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(p.pages)};
  const uint64_t strides[3] = {rs, hs, ps};
  const uint32_t box[4] = {64, static_cast<uint32_t>(a.page_box), 1, 1};
  const CUtensorMapDataType dt = dtype == TDSA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  for (int i = 0; i < 2; ++i) {
    const int rc = encode_tmap(&maps[i], dt, 4, i ? p.values : p.keys, dims, strides, box,
                               CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  if (dtype == TDSA_BF16)
    return dim == 128 ? launch_chunk_t<true, 128>(a, maps[0], maps[1], ctas, stream)
                      : launch_chunk_t<true, 64>(a, maps[0], maps[1], ctas, stream);
  return dim == 128 ? launch_chunk_t<false, 128>(a, maps[0], maps[1], ctas, stream)
                    : launch_chunk_t<false, 64>(a, maps[0], maps[1], ctas, stream);
}

}  // namespace tdsa

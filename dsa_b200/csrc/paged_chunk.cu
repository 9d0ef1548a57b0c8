// Attention of a chunk of new tokens over a paged key/value cache on the tensor cores.
//
//   out[t,h] = sum_j softmax_j(scale q[t,h].K[j]) V[j] over the keys j that token t sees.
//
// An item is 256 query rows -- the (token, head) rows that share one key/value head -- in two
// tiles of 128, and walks its keys in units of 128.  One CTA per SM; roles:
//   warps 0-3, 4-7: one tile each, one row per thread (softmax, output);
//   warp 8: page lookups and TMA copies of K and V units into a ring in shared memory;
//   warp 9: tcgen05 products, S = Q K^T (both from shared memory) and O += P V (P from TMEM).
// TMEM holds S (128 columns) and O (D columns) of both tiles; P, 16-bit, takes the place of S
// once its thread has read the row.  The two tiles alternate: while one tile's rows take their
// exponentials, the tensor core runs the other tile's products, and a unit of K and V is
// fetched once for both.
//
// S is only issued for unit i + 1 after O += P V of unit i, and tensor products of one CTA
// complete in the order of their issue, so the completion of S(i + 1) also says that O is at
// rest: the thread that owns a row then rescales it in place when the row's maximum has grown
// by a factor of more than 2^8 (rare after the first units), with no extra hand-shake.
//
// Scores, maxima, sums and O are float32.  P is rounded to the cache's type for the second
// product (2^-8 relative in bf16, 2^-11 in f16, the rounding that the output gets too); the sum
// adds the unrounded P.
#include <algorithm>

#include "paged.cuh"

namespace tdsa {

namespace {

constexpr int kPcThreads = 384;        // warps 10 and 11 only fill the third warpgroup
// Registers per thread: 168 at launch (65536 / 384); the third warpgroup gives 96 of its own to
// the two that hold rows.  2 * 216 + 72 = 3 * 168.
constexpr int kPcRegsRows = 216, kPcRegsRest = 72;
static_assert(2 * kPcRegsRows + kPcRegsRest <= 3 * 168, "registers of the launch");
constexpr int kPcTile = 128;           // rows of a tile
constexpr int kPcRows = 2 * kPcTile;   // rows of an item
constexpr int kPcUnit = 128;           // keys of a unit
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

// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16, A's 16-bit values packed two to a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
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

// Barrier of the 128 threads of tile t (named barrier 1 + t).
__device__ __forceinline__ void tile_sync(int t) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
}
__device__ __forceinline__ bool tile_any(int t, bool v) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(1 + t), "r"(static_cast<int>(v))
      : "memory");
  return r != 0;
}

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Two float32 at once (one issue slot): a * b + c, a + b.
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// O += P V of one unit for one row, element by element over the keys [j0, j1) that the row
// sees: P from TMEM (s_addr), V from its swizzled unit in shared memory.  first: O starts at 0.
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
    for (int jp = 0; jp < kPcUnit / 2; ++jp) {
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

template <bool kBF16, int D>
__global__ void __launch_bounds__(kPcThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const ChunkArgs a) {
  using C = ChunkCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem + C::kRing;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_q + C::kQ);
  uint64_t* empty = full + C::kStages;
  uint64_t* qfull = empty + C::kStages;  // [tile]
  uint64_t* sfull = qfull + 2;           // [tile] S is complete (and O at rest)
  uint64_t* pfull = sfull + 2;           // [tile] P is in TMEM, O rescaled or read out
  uint64_t* ofull = pfull + 2;           // [tile] the segment's last product is complete
  uint64_t* done = ofull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile int* skip = abort_flag + 1;   // [tile] this unit's product was formed by the threads
  int* s_last = const_cast<int*>(abort_flag) + 3;  // [tile]
  int* s_found = s_last + 2;             // [4]
  // [unit mod 16]: bit b is set when keys 16 b .. 16 b + 15 of the unit lie in a page that is
  // not the cache's (the ring holds fewer than 16 units)
  volatile uint32_t* absent = reinterpret_cast<volatile uint32_t*>(s_found + 4);
  int64_t* s_scan = reinterpret_cast<int64_t*>(
      (reinterpret_cast<uintptr_t>(s_found + 20) + 7) & ~uintptr_t(7));  // [10]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&qfull[t], 4);
      mbar_init(&sfull[t], 1);
      mbar_init(&pfull[t], 4);
      mbar_init(&ofull[t], 1);
      skip[t] = 0;
    }
    mbar_init(done, 1);
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
      a.p, a.q, gridDim.x, blockIdx.x, s_scan, s_found);
  const int cta = blockIdx.x;
  PagedItem it;
  SeqSpan span;
  int rt = sl.row_tile, off = sl.off;
  if (sl.begin < sl.end) {
    it.seq = sl.seq;
    it.head = sl.head;
    span = load_span(a.p, it.seq);
    paged_range_item<kPcRows, kPcUnit>(a.q, span, rt, it);
  }
  // every role walks the same segments: calls f(unit0, units in the segment, units in the
  // item, the item's first unit in the list) for each until it returns false
  auto walk = [&](auto&& f) {
    int64_t u = sl.begin;
    while (u < sl.end) {
      const int n = it.u1 - it.u0;
      const int seg = static_cast<int>(min(static_cast<int64_t>(n - off), sl.end - u));
      if (!f(it.u0 + off, seg, n, u - off)) return;
      u += seg;
      if (u >= sl.end) return;
      off = 0;
      paged_next_item<kPcRows, kPcUnit>(a.p, a.q, span, rt, it);
    }
  };

  if (warp >= 8) regs_dec<kPcRegsRest>();
  if (warp == 8) {
    // ------------------------------------------------------------ copies of K and V
    const int box = a.page_box, boxes = kPcUnit / box;
    uint32_t n_loads = 0;
    bool bad = false;
    walk([&](int unit0, int seg, int, int64_t) {
      const int32_t* table = a.p.table + it.seq * a.p.table_stride;
      // lane l looks up the page of the unit's l-th box; positions no row sees are not looked
      // up, and like pages that are not the cache's they are read past its end, as zeros
      auto entry_of = [&](int i) {
        const int pos = (unit0 + i) * kPcUnit + lane * box;
        if (i >= seg || lane >= boxes || pos >= it.k1 || pos + box <= it.k0) return a.p.pages;
        return __ldg(table + (pos >> a.p.page_shift));
      };
      int entry = entry_of(0);
      for (int i = 0; i < seg; ++i) {
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
          if (!warp_wait(&empty[s], ph ^ 1u, abort_flag)) return false;
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
      return true;
    });
    __syncwarp();
    if (bad && lane == 0) atomicOr(a.status, TDSA_STATUS_RANGE);
    // every issued copy lands before the CTA can exit
    volatile int no_abort = 0;
    for (uint32_t s = 0; s < C::kStages && s < n_loads; ++s) {
      const uint32_t n = (n_loads - s + C::kStages - 1) / C::kStages;
      mbar_wait(&full[s], (n - 1) & 1u, &no_abort);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ tensor products
    constexpr uint32_t idesc_s = umma_idesc_f16(kBF16, kPcTile, kPcUnit);
    constexpr uint32_t idesc_o = umma_idesc_f16(kBF16, kPcTile, D) | (1u << 16);
    uint32_t n_take = 0, q_n[2] = {0, 0}, p_n[2] = {0, 0};
    auto take = [&]() -> int {  // the ring's next stage, -1 when the CTA aborts
      const uint32_t s = n_take % C::kStages, ph = (n_take / C::kStages) & 1u;
      if (!warp_wait(&full[s], ph, abort_flag)) return -1;
      ++n_take;
      return static_cast<int>(s);
    };
    auto issue_s = [&](int t, int stage) {
      if (lane == 0) {
        const uint32_t qa = smem_u32(s_q + t * C::kTileBytes);
        const uint32_t ka = smem_u32(smem + stage * C::kTileBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(tmem + t * 128, sw128_kmajor_desc(qa + (k >> 2) * kPcHalf + (k & 3) * 32),
                   sw128_kmajor_desc(ka + (k >> 2) * kPcHalf + (k & 3) * 32), idesc_s,
                   k > 0 ? 1u : 0u);
        umma_commit(&sfull[t]);
      }
      __syncwarp();
    };
    walk([&](int unit0, int seg, int, int64_t) {
      const int tiles = it.rows > kPcTile ? 2 : 1;
      int ks = take();
      if (ks < 0) return false;
      for (int t = 0; t < tiles; ++t) {
        if (!warp_wait(&qfull[t], q_n[t]++ & 1u, abort_flag)) return false;
        tc_fence_after();
        issue_s(t, ks);
      }
      if (lane == 0) umma_commit(&empty[ks]);
      __syncwarp();
      for (int i = 0; i < seg; ++i) {
        const int vs = take();
        if (vs < 0) return false;
        // rows of V that no row of the item sees may hold anything: zero weights times
        // infinities or NaN would be NaN, so they become zeros
        const int base = (unit0 + i) * kPcUnit;
        if (base < it.k0 || base + kPcUnit > it.k1) {
          for (int x = lane; x < C::kHalves * kPcUnit * 8; x += 32) {
            const int r = (x >> 3) & (kPcUnit - 1);
            if (base + r < it.k0 || base + r >= it.k1)
              *reinterpret_cast<uint4*>(smem + vs * C::kTileBytes + x * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        const bool more = i + 1 < seg;
        if (more) {
          ks = take();
          if (ks < 0) return false;
        }
        for (int t = 0; t < tiles; ++t) {
          if (!warp_wait(&pfull[t], p_n[t]++ & 1u, abort_flag)) return false;
          tc_fence_after();
          if (lane == 0 && !skip[t]) {
            const uint32_t va = smem_u32(smem + vs * C::kTileBytes);
#pragma unroll
            for (int k = 0; k < kPcUnit / 16; ++k)
              umma_f16_ts(tmem + C::kOCol + t * D, tmem + t * 128 + k * 8,
                          sw128_mnmajor_desc(va + k * 2048), idesc_o, (i > 0 || k > 0) ? 1u : 0u);
          }
          __syncwarp();
          if (more) {
            issue_s(t, ks);
          } else {
            if (lane == 0) umma_commit(&ofull[t]);
            __syncwarp();
          }
        }
        if (lane == 0) {
          umma_commit(&empty[vs]);
          if (more) umma_commit(&empty[ks]);
        }
        __syncwarp();
      }
      return true;
    });
    __syncwarp();
    if (lane == 0) umma_commit(done);
    __syncwarp();
    volatile int no_abort = 0;
    mbar_wait(done, 0, &no_abort);
  } else if (warp < 8) {
    // ------------------------------------------------------------ rows: softmax and output
    regs_inc<kPcRegsRows>();
    const int t = warp >> 2;                      // tile
    const int row = (warp & 3) * 32 + lane;       // of the tile; also the TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>(warp & 3) << 21;
    const uint32_t s_addr = tmem + lane_base + t * 128;
    const uint32_t o_addr = tmem + lane_base + C::kOCol + t * D;
    const int g = a.q.group;
    uint32_t s_n = 0, o_n = 0;
    uint32_t n_v = 1;  // ring index of the current unit's V (K, V, K, V, ...)
    walk([&](int unit0, int seg, int n_units, int64_t item_u0) {
      const uint32_t v0 = n_v;
      n_v += 2 * seg;
      if (t == 1 && it.rows <= kPcTile) return true;
      const int r_item = t * kPcTile + row;  // row of the item
      const bool valid = r_item < it.rows;
      const int r = it.r0 + r_item;
      const int tok = it.tok0 + r / g, qh = it.head * g + r % g;
      {
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q.q + static_cast<int64_t>(valid ? tok : 0) * a.q.q_ts + (valid ? qh : 0) * a.q.q_hs);
        uint8_t* dst = s_q + t * C::kTileBytes + row * 128;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = valid ? src[c] : make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(dst + (c >> 3) * kPcHalf + (((c & 7) ^ (row & 7)) << 4)) = x;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfull[t]);
      }
      // keys this row sees, and keys every row of the tile sees
      const int pos = it.pos0 + r / g;
      const int hi = valid ? min(pos + 1, it.k1) : it.k1;
      const int lo = valid && a.q.window > 0 ? max(0, pos - (a.q.window - 1)) : 0;
      const int last_row = min(it.rows, (t + 1) * kPcTile) - 1;
      const int all_hi = min(it.k1, it.pos0 + (it.r0 + t * kPcTile) / g + 1);
      const int all_lo =
          a.q.window > 0
              ? max(it.k0, it.pos0 + (it.r0 + last_row) / g - (a.q.window - 1))
              : it.k0;
      float ref = -INFINITY, sum = 0.f;
      for (int i = 0; i < seg; ++i) {
        const int base = (unit0 + i) * kPcUnit;
        if (!warp_wait(&sfull[t], s_n++ & 1u, abort_flag)) return false;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, s[c]);
        tmem_wait_ld();
        const bool masked = base < all_lo || base + kPcUnit > all_hi;
        if (masked) {
#pragma unroll
          for (int j = 0; j < 128; ++j)
            if (base + j < lo || base + j >= hi) s[j >> 5][j & 31] = 0xFF800000u;  // -infinity
        }
        const uint32_t gone = absent[((v0 >> 1) + i) & 15];
        if (gone) {
#pragma unroll
          for (int j = 0; j < 128; ++j)
            if ((gone >> (j >> 4)) & 1u) s[j >> 5][j & 31] = 0xFF800000u;
        }
        float tops[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tops[c] = __uint_as_float(s[c][0]);
#pragma unroll
          for (int j = 1; j < 31; j += 2)
            tops[c] = max3(tops[c], __uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1]));
          tops[c] = fmaxf(tops[c], __uint_as_float(s[c][31]));
        }
        const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]) * a.q.scale_log2;
        const bool grow = top > ref + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float now = fmaxf(ref, top);
          const float f = now == ref ? 1.f : exp2_approx(ref - now);
          ref = now;
          sum *= f;
          if (i > 0) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_addr + c * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(o_addr + c * 16, o);
            }
          }
        }
        const float neg = ref == -INFINITY ? 0.f : -ref;
        const uint64_t scale2 = pair(a.q.scale_log2, a.q.scale_log2), neg2 = pair(neg, neg);
        uint64_t part[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 x = unpair(fma2(
                pair(__uint_as_float(s[c][2 * j]), __uint_as_float(s[c][2 * j + 1])), scale2, neg2));
            const float e0 = exp2_approx(x.x), e1 = exp2_approx(x.y);
            part[j & 1] = add2(part[j & 1], pair(e0, e1));
            p[j] = pack16<kBF16>(e0, e1);
          }
          tmem_st16(s_addr + c * 16, p);
        }
        {
          const float2 x = unpair(add2(part[0], part[1]));
          sum += x.x + x.y;
        }
        tmem_wait_st();
        bool alone = false;
        if (masked) {
          // a value that only some rows see and that is not finite: zero weights times it
          // would be NaN for the others, so the threads form this unit's product themselves
          const uint32_t vi = v0 + 2 * i;
          const uint32_t st = vi % C::kStages;
          if (!warp_wait(&full[st], (vi / C::kStages) & 1u, abort_flag)) return false;
          const uint8_t* sv = smem + st * C::kTileBytes;
          bool odd = false;
          if (base + row >= it.k0 && base + row < it.k1) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
              const uint4 x = *reinterpret_cast<const uint4*>(sv + (c >> 3) * kPcHalf + row * 128 +
                                                              (c & 7) * 16);
              odd |= nonfinite16<kBF16>(x.x) || nonfinite16<kBF16>(x.y) ||
                     nonfinite16<kBF16>(x.z) || nonfinite16<kBF16>(x.w);
            }
          }
          alone = tile_any(t, odd);
          if (alone)
            add_visible<kBF16, D>(s_addr, o_addr, sv, max(0, lo - base), min(kPcUnit, hi - base),
                                  i == 0);
        }
        if (row == 0) skip[t] = alone ? 1 : 0;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[t]);
      }

      // ---------------------------------------------------------- output
      if (!warp_wait(&ofull[t], o_n++ & 1u, abort_flag)) return false;
      tc_fence_after();
      const bool entire = seg == n_units;
      if (entire) {
        const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays NaN
        uint4* dst = reinterpret_cast<uint4*>(a.q.out + static_cast<int64_t>(tok) * a.q.o_ts +
                                              qh * a.q.o_hs);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
          if (valid) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t w[4];
#pragma unroll
              for (int y = 0; y < 4; ++y)
                w[y] = sum == 0.f ? 0u
                                  : pack16<kBF16>(__uint_as_float(o[x * 8 + 2 * y]) * inv,
                                                  __uint_as_float(o[x * 8 + 2 * y + 1]) * inv);
              dst[c * 4 + x] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        tc_fence_before();
        if (valid && a.q.lse)
          a.q.lse[static_cast<int64_t>(tok) * a.q.heads + qh] =
              sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
        return true;
      }
      const int c_first = slice_owner(sl.units, sl.ctas, item_u0);
      const int c_last = slice_owner(sl.units, sl.ctas, item_u0 + n_units - 1);
      {
        const int64_t slot = 2 * cta + (cta == c_first ? 1 : 0);
        const int64_t at = slot * kPcRows + r_item;
        a.part.ml[at] = make_float2(ref, sum);
        float4* dst = reinterpret_cast<float4*>(a.part.o + at * D);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 8; ++x)
            dst[c * 8 + x] =
                make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                            __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
        }
        tc_fence_before();
      }
      tile_sync(t);
      if (row == 0) {
        __threadfence();
        uint32_t* counter = a.part.counters + 2 * c_first + t;
        const uint32_t n = static_cast<uint32_t>(c_last - c_first + 1);
        const uint32_t old = atomicAdd(counter, 1u);
        if (old == n - 1) *counter = 0u;
        s_last[t] = old == n - 1;
        __threadfence();
      }
      tile_sync(t);
      if (s_last[t]) {
        // the last to arrive: partials of CTAs c_first .. c_last in that order, a warp per row
        constexpr int kV = D / 32;  // floats of a row per lane
        const int rows = min(it.rows - t * kPcTile, kPcTile);
        for (int x = warp & 3; x < rows; x += 4) {
          const int ri = t * kPcTile + x;
          float m = -INFINITY;
          for (int c = c_first; c <= c_last; ++c)
            m = fmaxf(m, __ldcg(&a.part.ml[(2 * static_cast<int64_t>(c) + (c == c_first)) *
                                               kPcRows + ri]).x);
          const float mr = m == -INFINITY ? 0.f : m;
          float l = 0.f, v[kV];
#pragma unroll
          for (int y = 0; y < kV; ++y) v[y] = 0.f;
#pragma unroll 2
          for (int c = c_first; c <= c_last; ++c) {
            const int64_t at = (2 * static_cast<int64_t>(c) + (c == c_first)) * kPcRows + ri;
            const float2 ml = __ldcg(&a.part.ml[at]);
            const float f = exp2_approx(ml.x - mr);
            l += ml.y * f;
#pragma unroll
            for (int y = 0; y < kV / 2; ++y) {
              const float2 w = __ldcg(
                  reinterpret_cast<const float2*>(a.part.o + at * D) + y * 32 + lane);
              v[2 * y] += w.x * f;
              v[2 * y + 1] += w.y * f;
            }
          }
          const int rg = it.r0 + ri;
          const int64_t to = it.tok0 + rg / g;
          const int h = it.head * g + rg % g;
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
          for (int y = 0; y < kV / 2; ++y)
            *(reinterpret_cast<uint32_t*>(a.q.out + to * a.q.o_ts + h * a.q.o_hs) + y * 32 + lane) =
                l == 0.f ? 0u : pack16<kBF16>(v[2 * y] * inv, v[2 * y + 1] * inv);
          if (a.q.lse && lane == 0)
            a.q.lse[to * a.q.heads + h] =
                l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        }
      }
      return true;
    });
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

// Append of new tokens to a paged key/value cache, with the rotation of keys and queries.
//
//   K[slot(p)][h] = R_p k[t][h],  V[slot(p)][h] = v[t][h],  q_out[t][h] = R_p q[t][h]
//
// for token t at position p of its sequence, slot(p) = (table[p / page_size], p % page_size).
// R_p turns the pairs of the leading rope_dim features by the angles p * inv_freq[j].
//
// The angle is formed and reduced by 2 pi in float64 (a float32 product is off by up to 2^-24 p
// radians, 0.002 at p = 32768), the hardware sine and cosine take the reduced angle, and the
// products are float32 with one rounding at the end.
#include <algorithm>

#include "paged.cuh"

namespace tdsa {

namespace {

// Threads of a CTA and the rows a lane loads ahead: long calls take fewer threads with more loads
// under way each (8698 tokens of 48 heads: 38 us with 128, 42 with 256), short ones more threads
// (64 tokens: 4.0 us with 128, 3.1 with 256).
constexpr int kPaShort = 256, kPaLong = 128;
constexpr int kPaHeldRows = 768;  // threads times rows ahead

struct AppendArgs {
  PagedView p;
  uint16_t* keys;
  uint16_t* values;
  const uint16_t *k, *v, *q;
  uint16_t* q_out;
  int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, qo_ts, qo_hs;
  int q_heads;
  const float* inv_freq;
  const int64_t* positions;
  int rope_dim, pairs;
  int* status;
};

// A CTA takes one token.  A lane keeps one 16-byte vector of the row for all the rows it handles --
// K's, Q's, then V's heads, 32 / (D / 8) of them per warp and step -- so its angles sit in
// registers and a row costs a load, the products and a store; the partner of a feature in the
// other half comes from the lane that holds it.  The first kPaHeld rows per lane are loaded before
// anything is known about the token, so the loads from HBM run while its sequence, its page and
// its angles are found (three dependent reads).
//
// HBM bound: 8698 tokens of 32 + 8 + 8 heads of 128 (214 MB) take 39 us, 5.5 TB/s, against the 33 us
// that a copy of as many bytes takes; a few tokens take the time of the three reads, 3.1 us.
template <bool kBF16, int D, int kPaThreads>
__global__ void __launch_bounds__(kPaThreads, kPaThreads == kPaShort ? 5 : 9)
    paged_append_kernel(const AppendArgs a) {
  constexpr int kPaHeld = kPaHeldRows / kPaThreads;
  __shared__ float2 cs[64];
  __shared__ int64_t s_row;
  __shared__ int s_pos, s_page;             // s_page < 0: no slot
  constexpr int kVecs = D / 8;              // lanes of a row
  constexpr int kStep = kPaThreads / kVecs; // rows a step of the CTA takes
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t t = blockIdx.x;
  const int half = a.rope_dim >> 1, hv = half >> 3;
  const int v = tid % kVecs, r0 = tid / kVecs;
  const int hkv = a.p.kv_heads, rows = 2 * hkv + a.q_heads;
  auto source = [&](int r) {
    const uint16_t* p = r < hkv ? a.k + t * a.k_ts + r * a.k_hs
                                : (r < hkv + a.q_heads ? a.q + t * a.q_ts + (r - hkv) * a.q_hs
                                                       : a.v + t * a.v_ts +
                                                             (r - hkv - a.q_heads) * a.v_hs);
    return reinterpret_cast<const uint4*>(p + v * 8);
  };
  uint4 x[kPaHeld];
#pragma unroll
  for (int n = 0; n < kPaHeld; ++n)
    if (r0 + n * kStep < rows) x[n] = *source(r0 + n * kStep);

  // the token's sequence: the one whose rows hold it
  bool found = false;
  for (int b = tid; b < a.p.batch; b += kPaThreads) {
    int q0, n;
    load_rows(a.p, b, q0, n);
    const int len = __ldg(a.p.lengths + b);
    if (t >= q0 && t < q0 + n) {
      const int64_t pos = static_cast<int64_t>(len) - n + (t - q0);
      const bool in = pos >= 0 && (pos >> a.p.page_shift) < a.p.max_pages;
      s_pos = static_cast<int>(max(int64_t(-0x7FFFFFFF), pos));  // at most len - 1
      s_page = in ? __ldg(a.p.table + b * a.p.table_stride + (pos >> a.p.page_shift)) : -1;
      found = true;
    }
  }
  if (!__syncthreads_or(found)) return;  // a row of no sequence
  if (tid < half) {
    const int64_t turn = a.positions ? a.positions[t] : s_pos;
    const double z = static_cast<double>(turn) * static_cast<double>(a.inv_freq[tid]);
    const double m = rint(z * 0.15915494309189535);
    const float r = static_cast<float>(fma(-m, 6.283185307179586, z));
    cs[tid] = make_float2(__cosf(r), __sinf(r));
  }
  if (tid == kPaThreads - 1) {
    s_row = paged_row(a.p, s_page, s_pos);
    if (s_row < 0) atomicOr(a.status, TDSA_STATUS_RANGE);
  }
  __syncthreads();

  const bool mine = a.pairs ? v * 8 < a.rope_dim : v < 2 * hv;  // this vector is turned
  const bool upper = v >= hv;                                   // (halves) of the second half
  const int partner = a.pairs || !mine ? lane : (upper ? lane - hv : lane + hv);
  const int64_t row = s_row;
  float2 c[8];  // feature e of the vector becomes x c.x + partner c.y
  if (mine) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = cs[a.pairs ? v * 4 + e / 2 : (upper ? v - hv : v) * 8 + e];
      if (a.pairs ? !(e & 1) : !upper) c[e].y = -c[e].y;
    }
  }
  auto finish = [&](int r, uint4 u) {
    uint16_t* dst = r < hkv ? a.keys + row + r * a.p.head_stride
                            : (r < hkv + a.q_heads
                                   ? a.q_out + t * a.qo_ts + (r - hkv) * a.qo_hs
                                   : a.values + row + (r - hkv - a.q_heads) * a.p.head_stride);
    const bool there = row >= 0 || (r >= hkv && r < hkv + a.q_heads);
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (a.rope_dim) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t other = __shfl_sync(0xffffffffu, w[e], partner);
        if (mine && r < hkv + a.q_heads) {
          const float2 f = unpack16<kBF16>(w[e]);
          float2 o = unpack16<kBF16>(other);
          if (a.pairs) o = make_float2(o.y, o.x);
          w[e] = pack16<kBF16>(fmaf(f.x, c[2 * e].x, o.x * c[2 * e].y),
                               fmaf(f.y, c[2 * e + 1].x, o.y * c[2 * e + 1].y));
        }
      }
    }
    if (there && r < rows)
      *reinterpret_cast<uint4*>(dst + v * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  };
#pragma unroll
  for (int n = 0; n < kPaHeld; ++n)
    if (n * kStep < rows) finish(r0 + n * kStep, x[n]);
  for (int r = kPaHeld * kStep; r < rows; r += kStep) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (r0 + r < rows) u = *source(r0 + r);
    finish(r0 + r, u);
  }
}

template <int kThreads>
auto append_kernel(bool bf16, int dim) {
  return dim == 128 ? (bf16 ? paged_append_kernel<true, 128, kThreads>
                            : paged_append_kernel<false, 128, kThreads>)
                    : (bf16 ? paged_append_kernel<true, 64, kThreads>
                            : paged_append_kernel<false, 64, kThreads>);
}

}  // namespace

int launch_paged_append(const PagedView& p, void* keys, void* values, int dtype, int dim,
                        const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts,
                        int64_t v_hs, const void* q, int64_t q_ts, int64_t q_hs, int q_heads,
                        void* q_out, int64_t qo_ts, int64_t qo_hs, const float* inv_freq,
                        int rope_dim, int pairs, const int64_t* positions, int* status,
                        cudaStream_t stream) {
  AppendArgs a;
  a.p = p;
  a.keys = static_cast<uint16_t*>(keys);
  a.values = static_cast<uint16_t*>(values);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q = static_cast<const uint16_t*>(q);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_ts = k_ts, a.k_hs = k_hs, a.v_ts = v_ts, a.v_hs = v_hs;
  a.q_ts = q_ts, a.q_hs = q_hs, a.qo_ts = qo_ts, a.qo_hs = qo_hs;
  a.q_heads = q_heads;
  a.inv_freq = inv_freq;
  a.positions = positions;
  a.rope_dim = rope_dim;
  a.pairs = pairs;
  a.status = status;
  const bool bf16 = dtype == TDSA_BF16;
  // short: every CTA of the call can be resident at once
  const bool brief = p.tokens <= 5 * device_sm_count(current_device());
  auto kern = brief ? append_kernel<kPaShort>(bf16, dim) : append_kernel<kPaLong>(bf16, dim);
  TDSA_CUDA_CHECK(launch_pdl(kern, dim3(static_cast<unsigned>(p.tokens)),
                             dim3(brief ? kPaShort : kPaLong), 0, stream, a));
  TDSA_CUDA_CHECK(cudaGetLastError());
  return TDSA_OK;
}

}  // namespace tdsa

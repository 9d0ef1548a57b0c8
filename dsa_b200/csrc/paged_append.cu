// Append of new tokens to a paged key/value cache, with the rotation of keys and queries.
//
//   K[slot(p)][h] = R_p k[t][h],  V[slot(p)][h] = v[t][h],  q_out[t][h] = R_p q[t][h]
//
// for token t at position p of its sequence, slot(p) = (table[p / page_size], p % page_size).
// R_p turns the pairs of the leading rope_dim features by the angles p * inv_freq[j].
//
// The angle is formed and reduced by 2 pi in float64 (a float32 product is off by up to 2^-24 p
// radians, 0.002 at p = 32768), the hardware sine and cosine take the reduced angle, and the
// products are float32 with one rounding at the end.  The angles of a token are computed once,
// by one thread each, into shared memory and used by all its heads.
#include <algorithm>

#include "paged.cuh"

namespace tdsa {

namespace {

constexpr int kPaThreads = 256;

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

// 8 features (16 bytes) of one row: out = R x for the pairs in it
template <bool kBF16>
__device__ __forceinline__ uint4 turn_pairs(uint4 x, const float2* cs) {
  uint32_t r[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack16<kBF16>(r[i]), c = cs[i];
    r[i] = pack16<kBF16>(v.x * c.x - v.y * c.y, v.y * c.x + v.x * c.y);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <bool kBF16>
__device__ __forceinline__ void turn_halves(uint4& a, uint4& b, const float2* cs) {
  uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = unpack16<kBF16>(x[i]), w = unpack16<kBF16>(y[i]);
    const float2 c0 = cs[2 * i], c1 = cs[2 * i + 1];
    x[i] = pack16<kBF16>(u.x * c0.x - w.x * c0.y, u.y * c1.x - w.y * c1.y);
    y[i] = pack16<kBF16>(w.x * c0.x + u.x * c0.y, w.y * c1.x + u.y * c1.y);
  }
  a = make_uint4(x[0], x[1], x[2], x[3]);
  b = make_uint4(y[0], y[1], y[2], y[3]);
}

template <bool kBF16, int D>
__global__ void __launch_bounds__(kPaThreads) paged_append_kernel(const AppendArgs a) {
  __shared__ float2 cs[64];
  constexpr int kVecs = D / 8;
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, tid = threadIdx.x;
  const int half = a.rope_dim >> 1, hv = half >> 3;
  // the token's sequence: the number of sequences that end at or before it
  int seq = 0;
  for (int b0 = 0; b0 < a.p.batch; b0 += kPaThreads) {
    const int b = b0 + tid;
    seq += __syncthreads_count(b < a.p.batch && __ldg(a.p.starts + b + 1) <= t);
  }
  if (seq >= a.p.batch) return;  // a row past the last sequence
  const SeqSpan s = load_span(a.p, seq);
  const int pos = s.len - s.n + (t - s.q0);
  const bool in = pos >= 0 && t >= s.q0 && t < s.q0 + s.n;
  const int64_t turn = a.positions ? a.positions[t] : pos;
  if (tid < half) {
    const double x = static_cast<double>(turn) * static_cast<double>(a.inv_freq[tid]);
    const double m = rint(x * 0.15915494309189535);
    const float r = static_cast<float>(fma(-m, 6.283185307179586, x));
    cs[tid] = make_float2(__cosf(r), __sinf(r));
  }
  int64_t row = -1;
  if (in) {
    const int entry = __ldg(a.p.table + seq * a.p.table_stride + (pos >> a.p.page_shift));
    row = paged_row(a.p, entry, pos);
  }
  if (row < 0 && tid == 0) atomicOr(a.status, TDSA_STATUS_RANGE);
  __syncthreads();

  // Work of the token: per head, the vectors of the row; with halves, a thread takes a vector
  // of the first half and its partner, so only vectors [0, hv) and [2 hv, kVecs) lead.
  const int lead = a.pairs ? kVecs : kVecs - hv;
  const int total = (a.p.kv_heads + (a.q ? a.q_heads : 0)) * lead;
  for (int i = tid; i < total; i += kPaThreads) {
    const int h = i / lead, l = i - h * lead;
    const bool key = h < a.p.kv_heads;
    const uint16_t* src = key ? a.k + t * a.k_ts + h * a.k_hs
                              : a.q + t * a.q_ts + (h - a.p.kv_heads) * a.q_hs;
    uint16_t* dst = key ? (row < 0 ? nullptr : a.keys + row + h * a.p.head_stride)
                        : a.q_out + t * a.qo_ts + (h - a.p.kv_heads) * a.qo_hs;
    if (!dst) continue;
    if (a.pairs) {
      uint4 x = *reinterpret_cast<const uint4*>(src + l * 8);
      if (l * 8 < a.rope_dim) x = turn_pairs<kBF16>(x, cs + l * 4);
      *reinterpret_cast<uint4*>(dst + l * 8) = x;
    } else if (l < hv) {
      uint4 x = *reinterpret_cast<const uint4*>(src + l * 8);
      uint4 y = *reinterpret_cast<const uint4*>(src + half + l * 8);
      turn_halves<kBF16>(x, y, cs + l * 8);
      *reinterpret_cast<uint4*>(dst + l * 8) = x;
      *reinterpret_cast<uint4*>(dst + half + l * 8) = y;
    } else {
      const int v = l + hv;
      *reinterpret_cast<uint4*>(dst + v * 8) = *reinterpret_cast<const uint4*>(src + v * 8);
    }
  }
  if (row < 0) return;
  for (int i = tid; i < a.p.kv_heads * kVecs; i += kPaThreads) {
    const int h = i / kVecs, l = i - h * kVecs;
    *reinterpret_cast<uint4*>(a.values + row + h * a.p.head_stride + l * 8) =
        *reinterpret_cast<const uint4*>(a.v + t * a.v_ts + h * a.v_hs + l * 8);
  }
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
  auto kern = dim == 128 ? (bf16 ? paged_append_kernel<true, 128> : paged_append_kernel<false, 128>)
                         : (bf16 ? paged_append_kernel<true, 64> : paged_append_kernel<false, 64>);
  TDSA_CUDA_CHECK(
      launch_pdl(kern, dim3(static_cast<unsigned>(p.tokens)), dim3(kPaThreads), 0, stream, a));
  TDSA_CUDA_CHECK(cudaGetLastError());
  return TDSA_OK;
}

}  // namespace tdsa

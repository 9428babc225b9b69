// New tokens enter a paged key/value cache: norms of queries and keys per head, the position rotation, and
// the write of keys and values into their pages, in one pass over the projections.
//
//   x' = x rsqrt(mean(x^2) + eps) w                      (q and k, when weights are given)
//   (a, b) -> (a cos - b sin, b cos + a sin)             pairs (i, i + rot/2), or (2i, 2i+1) interleaved
//   slot len - n + i of request r <- k', v ;  attention weight there <- 0 ;  q' -> q_out
//
// Bound by memory: every row is read once and written once.  Sixteen lanes hold one head's row, eight
// elements each as two chunks of four, so the sum of squares is four shuffles.  Which columns a lane holds is chosen so
// that both elements of a rotated pair are in one lane: neighbouring chunks for interleaved pairs, chunks half a row
// apart for pairs (i, i + d/2); only a rotation of part of the columns in halves exchanges through shared
// memory.  A lane's columns are the same for every head of a token, so its angles and norm weights are loaded once.
//
// Measured: prompts of 6868 tokens, 32 + 8 + 8 heads of 128, norm and rotation: 40..42 us, 4.1..4.3 TB/s (issue is busy 47 %
// of the time at 22 warps an SM: the rest is the latency of a CTA's chain of look-ups, loads and stores); 64 tokens: 4 us.
#include "om_paged.cuh"

namespace cb2 {
namespace {

constexpr int kThreads = 256, kGroups = kThreads / 16;
constexpr int kAhead = 4;     // rows of q a group has in flight

struct AppendArgs {
  const void *q, *k, *v;
  long long q_token, q_head, k_token, k_head, v_token, v_head;
  void* q_out;
  void *k_pages, *v_pages;
  long long k_page_stride, v_page_stride;
  float* weights;
  const int* positions;
  const void *q_weight, *k_weight;
  const float *cos, *sin;
  int table_rows, rot, interleaved;
  float eps;
  int Hq, Hkv, d, tokens_per_cta;
};

// How the columns of a row are paired by the rotation.
enum { kNone, kInterleaved, kHalves, kExchange };

// Eight elements of a row: columns [o0, o0 + 4) and [o1, o1 + 4).
template <class T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint2 a, b;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int o0, int o1) {
    a = *reinterpret_cast<const uint2*>(p + o0);
    b = *reinterpret_cast<const uint2*>(p + o1);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p, int o0, int o1) const {
    *reinterpret_cast<uint2*>(p + o0) = a;
    *reinterpret_cast<uint2*>(p + o1) = b;
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16lo_to_f32(w[i]);
      x[2 * i + 1] = bf16hi_to_f32(w[i]);
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[8]) {
    a = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    b = make_uint2(pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct Raw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, int o0, int o1) {
    a = *reinterpret_cast<const float4*>(p + o0);
    b = *reinterpret_cast<const float4*>(p + o1);
  }
  __device__ __forceinline__ void store(float* p, int o0, int o1) const {
    *reinterpret_cast<float4*>(p + o0) = a;
    *reinterpret_cast<float4*>(p + o1) = b;
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  __device__ __forceinline__ void pack(const float (&x)[8]) {
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(x[4], x[5], x[6], x[7]);
  }
};

struct TokenPlace {
  int page, slot;     // page < 0: the token has no place (behind the last sequence, or a bad index)
  int position;
  int live;
};

// Norm and rotation of the eight elements that a lane holds; `mine`: this row's place in shared memory (kExchange).
template <int MODE>
__device__ __forceinline__ void turn(float (&x)[8], bool norm, const float (&w)[8], float inv_d, float eps, const float (&cs)[8],
                                     const float (&sn)[8], unsigned half_mask, float* mine, int gl, int rot) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int off = 8; off; off >>= 1) ss += __shfl_xor_sync(half_mask, ss, off);
    const float inv = rsqrtf(ss * inv_d + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv * w[i];
  }
  if (MODE == kInterleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (gl * 8 + i >= rot) break;          // columns behind the rotation stay what they are (0 x Inf is NaN)
      const float a = x[i], b = x[i + 1];
      x[i] = fmaf(-b, sn[i >> 1], a * cs[i >> 1]);
      x[i + 1] = fmaf(a, sn[i >> 1], b * cs[i >> 1]);
    }
  } else if (MODE == kHalves) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[i], b = x[i + 4];
      x[i] = fmaf(-b, sn[i], a * cs[i]);
      x[i + 4] = fmaf(a, sn[i], b * cs[i]);
    }
  } else if (MODE == kExchange) {
    const int half = rot / 2;
    __syncwarp(half_mask);
    *reinterpret_cast<float4*>(mine + gl * 8) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(mine + gl * 8 + 4) = make_float4(x[4], x[5], x[6], x[7]);
    __syncwarp(half_mask);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = gl * 8 + i;
      if (e < rot) x[i] = fmaf(mine[e < half ? e + half : e - half], sn[i], x[i] * cs[i]);
    }
  }
}

template <class T, int MODE>
__global__ void __launch_bounds__(kThreads)
paged_append_kernel(const AppendArgs a, const PagedBatch batch) {
  __shared__ TokenPlace place[kGroups];
  __shared__ __align__(16) float rows[MODE == kExchange ? kGroups : 1][128];
  const int tid = threadIdx.x, group = tid / 16, gl = tid % 16;
  const int t_first = blockIdx.x * a.tokens_per_cta;
  const int t_count = min(a.tokens_per_cta, batch.n_tokens - t_first);
  if (tid < kGroups) place[tid].live = 0;
  __syncthreads();
  // the request of each token: every thread looks at one request, whose token range may meet this CTA's
  for (int r = tid; r < batch.R; r += kThreads) {
    const int c0 = __ldg(batch.cu + r), c1 = __ldg(batch.cu + r + 1);
    // (offsets out of order, or behind the batch, may meet no CTA's tokens)
    if (blockIdx.x == 0 && (c0 < 0 || c1 < c0 || c1 > batch.n_tokens)) paged_flag(batch);
    if (c1 <= t_first || c0 >= t_first + t_count) continue;
    const PagedReq q = paged_request(batch, r);
    for (int t = max(q.t0, t_first); t < min(q.t0 + q.n, t_first + t_count); ++t) {
      TokenPlace p;
      const int j = q.len - q.n + (t - q.t0);
      p.page = -1;
      p.slot = 0;
      if (j >= 0) {
        const int id = __ldg(batch.table + (long long)r * batch.max_pages + (j >> batch.page_log2));
        if (unsigned(id) < unsigned(batch.n_pages)) {
          p.page = id;
          p.slot = j & ((1 << batch.page_log2) - 1);
        }
      }
      if (p.page < 0) paged_flag(batch);
      p.position = 0;
      if (a.rot) {
        const int pos = __ldg(a.positions + t);
        p.position = min(max(pos, 0), a.table_rows - 1);
        if (p.position != pos) paged_flag(batch);
      }
      p.live = 1;
      place[t - t_first] = p;
    }
  }
  __syncthreads();

  const int per_token = kGroups / a.tokens_per_cta;      // groups that share a token's heads
  const int ti = group / per_token;
  const unsigned half_mask = 0xffffu << (tid & 16);
  const TokenPlace here = place[ti];
  if (ti >= t_count || !here.live) return;
  const int t = t_first + ti, d = a.d, half = a.rot / 2;
  const bool in = gl * 8 < d;
  const int ps = 1 << batch.page_log2;

  const int o0 = MODE == kHalves ? gl * 4 : gl * 8, o1 = MODE == kHalves ? half + gl * 4 : gl * 8 + 4;
  // what the group reads first is on its way before the angles are looked up
  const int sub = group % per_token;
  const T* qp = static_cast<const T*>(a.q) + t * a.q_token;
  const T* kp = static_cast<const T*>(a.k) + t * a.k_token;
  const T* vp = static_cast<const T*>(a.v) + t * a.v_token;
  Raw<T> rq[kAhead], rk, rv;
  auto fetch_q = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (in && h0 + u * per_token < a.Hq) rq[u].load(qp + (h0 + u * per_token) * a.q_head, o0, o1);
  };
  fetch_q(sub);
  if (in && sub < a.Hkv) {
    rk.load(kp + sub * a.k_head, o0, o1);
    rv.load(vp + sub * a.v_head, o0, o1);
  }
  float cs[8], sn[8], w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f, w[i] = 0.f;
  const float* ct = a.cos + (long long)here.position * half;
  const float* st = a.sin + (long long)here.position * half;
  if (MODE == kInterleaved || MODE == kHalves) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = gl * 4 + i;
      if (f < half) cs[i] = __ldg(ct + f), sn[i] = __ldg(st + f);
    }
  } else if (MODE == kExchange) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = gl * 8 + i;
      if (e < a.rot) {
        const float s = __ldg(st + (e < half ? e : e - half));
        cs[i] = __ldg(ct + (e < half ? e : e - half));
        sn[i] = e < half ? -s : s;          // x' = x cos + partner * sn
      }
    }
  }
  const float inv_d = 1.f / float(d);
  float* mine = rows[MODE == kExchange ? group : 0];
  auto weight = [&](const void* p) {
    Raw<T> r;
    if (in && p) {
      r.load(static_cast<const T*>(p), o0, o1);
      r.unpack(w);
    }
  };
  weight(a.q_weight);
  T* qo = static_cast<T*>(a.q_out) + (long long)t * a.Hq * d;
  for (int h0 = sub; h0 < a.Hq; h0 += kAhead * per_token) {
    if (h0 != sub) fetch_q(h0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * per_token;
      if (h >= a.Hq) break;
      float x[8] = {};
      if (in) rq[u].unpack(x);
      turn<MODE>(x, a.q_weight != nullptr, w, inv_d, a.eps, cs, sn, half_mask, mine, gl, a.rot);
      rq[u].pack(x);
      if (in) rq[u].store(qo + h * d, o0, o1);
    }
  }
  if (here.page < 0) return;
  weight(a.k_weight);
  T* ko = static_cast<T*>(a.k_pages) + here.page * a.k_page_stride + here.slot * d;
  T* vo = static_cast<T*>(a.v_pages) + here.page * a.v_page_stride + here.slot * d;
  for (int h = sub; h < a.Hkv; h += per_token) {
    if (in && h != sub) {
      rk.load(kp + h * a.k_head, o0, o1);
      rv.load(vp + h * a.v_head, o0, o1);
    }
    const int at = h * ps * d;          // Hkv * page_size * d is a page: below 2^31
    if (in) rv.store(vo + at, o0, o1);
    float x[8] = {};
    if (in) rk.unpack(x);
    turn<MODE>(x, a.k_weight != nullptr, w, inv_d, a.eps, cs, sn, half_mask, mine, gl, a.rot);
    rk.pack(x);
    if (in) rk.store(ko + at, o0, o1);
    if (a.weights && gl == 0) a.weights[((long long)here.page * a.Hkv + h) * ps + here.slot] = 0.f;
  }
}

template <class T>
int launch(int mode, unsigned grid, const AppendArgs& a, const PagedBatch& batch, cudaStream_t st) {
  switch (mode) {
    case kNone: paged_append_kernel<T, kNone><<<grid, kThreads, 0, st>>>(a, batch); break;
    case kInterleaved: paged_append_kernel<T, kInterleaved><<<grid, kThreads, 0, st>>>(a, batch); break;
    case kHalves: paged_append_kernel<T, kHalves><<<grid, kThreads, 0, st>>>(a, batch); break;
    default: paged_append_kernel<T, kExchange><<<grid, kThreads, 0, st>>>(a, batch);
  }
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

}  // namespace
}  // namespace cb2

extern "C" int cb2_paged_append(const void* q, long long q_token_stride, long long q_head_stride, const void* k,
                                long long k_token_stride, long long k_head_stride, const void* v, long long v_token_stride,
                                long long v_head_stride, void* q_out, void* k_pages, void* v_pages,
                                long long k_page_stride, long long v_page_stride, float* weights, const int* block_table,
                                const int* seq_lens, const int* cu_q, const int* positions, const void* q_weight,
                                const void* k_weight, float eps, const float* cos, const float* sin, int table_rows,
                                int rotary, int interleaved, int n_tokens, int R, int Hq, int Hkv, int d, int page_size,
                                int n_pages, int max_pages, int dtype, int* dev_status, void* stream) {
  using namespace cb2;
  if (!k_pages || !v_pages || !block_table || !seq_lens || !cu_q) return CB2_NULL_PTR;
  if (n_tokens < 0 || R < 1 || Hq < 0 || Hkv < 1 || d < 8 || d > 128 || d % 8 || n_pages < 1 || max_pages < 1) return CB2_BAD_SHAPE;
  if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1)) || int64_t(max_pages) * page_size > (1 << 30)) return CB2_BAD_SHAPE;
  if (rotary < 0 || rotary > d || rotary % 2 || (rotary && table_rows < 1) || !(eps >= 0.f)) return CB2_BAD_SHAPE;
  const long long page = (long long)Hkv * page_size * d;
  if (page >= (1ll << 31) || k_page_stride < page || v_page_stride < page || q_token_stride < 0 || q_head_stride < 0 || k_token_stride < 0 ||
      k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
    return CB2_BAD_SHAPE;
  if (dtype != CB2_BF16 && dtype != CB2_F32) return CB2_UNSUPPORTED_DTYPE;
  if (n_tokens == 0) return CB2_OK;
  if (!k || !v || (Hq && (!q || !q_out)) || (rotary && (!cos || !sin || !positions))) return CB2_NULL_PTR;
  const int vec = dtype == CB2_BF16 ? 8 : 4;
  if ((Hq && (!aligned16(q) || !aligned16(q_out))) || !aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(q_weight) || !aligned16(k_weight) || (Hq && (q_token_stride % vec || q_head_stride % vec)) ||
      k_token_stride % vec || k_head_stride % vec || v_token_stride % vec || v_head_stride % vec || k_page_stride % vec ||
      v_page_stride % vec)
    return CB2_BAD_ALIGN;
  if (Hq) {
    // a row of q is read before its own place in q_out is written: in place is fine, any other overlap is not
    const int esz = dtype == CB2_BF16 ? 2 : 4;
    const long long bytes = (long long)n_tokens * Hq * d * esz;
    const bool in_place = q == q_out && (n_tokens == 1 || q_token_stride == (long long)Hq * d) && (Hq == 1 || q_head_stride == d);
    if ((!in_place && paged_rows_meet(q, n_tokens, q_token_stride, Hq, q_head_stride, d, esz, q_out, bytes)) ||
        paged_rows_meet(k, n_tokens, k_token_stride, Hkv, k_head_stride, d, esz, q_out, bytes) ||
        paged_rows_meet(v, n_tokens, v_token_stride, Hkv, v_head_stride, d, esz, q_out, bytes))
      return CB2_BAD_SHAPE;
  }
  int page_log2 = 0;
  while ((1 << page_log2) < page_size) ++page_log2;
  const PagedBatch batch{block_table, seq_lens, cu_q, R, max_pages, n_pages, page_log2, n_tokens, n_tokens, max_pages * page_size, dev_status};
  AppendArgs a{q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, q_out,
               k_pages, v_pages, k_page_stride, v_page_stride, weights, positions, q_weight, k_weight, cos, sin, table_rows,
               rotary, interleaved, eps, Hq, Hkv, d, 1};
  // Few tokens: sixteen groups share one token's heads (latency).  Many: four groups keep a token, so that its
  // angles are loaded once for a quarter of its heads.
  while (a.tokens_per_cta < 4 && n_tokens / (2 * a.tokens_per_cta) >= 2 * kNumSMs) a.tokens_per_cta *= 2;
  const unsigned grid = unsigned((n_tokens + a.tokens_per_cta - 1) / a.tokens_per_cta);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int mode = !rotary ? kNone : interleaved ? kInterleaved : rotary == d ? kHalves : kExchange;
  return dtype == CB2_BF16 ? launch<__nv_bfloat16>(mode, grid, a, batch, st) : launch<float>(mode, grid, a, batch, st);
}

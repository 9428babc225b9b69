// New tokens enter a paged key/value cache: norms of queries and keys per head, the position rotation, and
// the write of keys and values into their pages, in one pass over the projections.
//
//   x' = x rsqrt(mean(x^2) + eps) w                      (q and k, when weights are given)
//   (a, b) -> (a cos - b sin, b cos + a sin)             pairs (i, i + rot/2), or (2i, 2i+1) interleaved
//   slot len - n + i of request r <- k', v ;  attention weight there <- 0 ;  q' -> q_out
//
// Bound by memory: every row is read once and written once.  Sixteen lanes hold one head's row, eight
// elements each, so the sum of squares is four shuffles; the lanes' columns are the same for every head of
// a token, so its cos / sin and the norm weights are loaded once and stay in registers across the heads.
#include "om_paged.cuh"

namespace cb2 {
namespace {

constexpr int kThreads = 256, kGroups = kThreads / 16;
constexpr int kAhead = 4;     // rows a group has in flight

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

template <class T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = u; }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16lo_to_f32(w[i]);
      x[2 * i + 1] = bf16hi_to_f32(w[i]);
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[8]) {
    u = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct Raw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
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

template <class T>
__global__ void __launch_bounds__(kThreads)
paged_append_kernel(const AppendArgs a, const PagedBatch batch) {
  __shared__ TokenPlace place[kGroups];
  __shared__ __align__(16) float rows[kGroups][128];
  const int tid = threadIdx.x, group = tid / 16, gl = tid % 16;
  const int t_first = blockIdx.x * a.tokens_per_cta;
  const int t_count = min(a.tokens_per_cta, batch.n_tokens - t_first);
  if (tid < kGroups) place[tid].live = 0;
  __syncthreads();
  // the request of each token: every thread looks at one request, whose token range may meet this CTA's
  for (int r = tid; r < batch.R; r += kThreads) {
    const int c0 = __ldg(batch.cu + r), c1 = __ldg(batch.cu + r + 1);
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

  float cs[8], sn[8];
  Raw<T> wq, wk;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = gl * 8 + i;
    cs[i] = 1.f, sn[i] = 0.f;
    if (e < a.rot) {
      const int f = a.interleaved ? e >> 1 : (e < half ? e : e - half);
      const bool first = a.interleaved ? !(e & 1) : e < half;
      cs[i] = __ldg(a.cos + (long long)here.position * half + f);
      const float s = __ldg(a.sin + (long long)here.position * half + f);
      sn[i] = first ? -s : s;          // y = x cos + partner * sn
    }
  }
  if (in && a.q_weight) wq.load(static_cast<const T*>(a.q_weight) + gl * 8);
  if (in && a.k_weight) wk.load(static_cast<const T*>(a.k_weight) + gl * 8);
  const int n_rows = a.Hq + 2 * a.Hkv;
  for (int row0 = group % per_token; row0 < n_rows; row0 += kAhead * per_token) {
    Raw<T> raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int row = row0 + u * per_token;
      if (in && row < n_rows) {
        const bool is_q = row < a.Hq, is_v = row >= a.Hq + a.Hkv;
        const T* src = is_q ? static_cast<const T*>(a.q) + t * a.q_token + row * a.q_head
                       : is_v ? static_cast<const T*>(a.v) + t * a.v_token + (row - a.Hq - a.Hkv) * a.v_head
                              : static_cast<const T*>(a.k) + t * a.k_token + (row - a.Hq) * a.k_head;
        raw[u].load(src + gl * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int row = row0 + u * per_token;
      if (row >= n_rows) break;
      const bool is_q = row < a.Hq, is_v = row >= a.Hq + a.Hkv;
      const int h = is_q ? row : (is_v ? row - a.Hq - a.Hkv : row - a.Hq);
      if (!is_v) {
        float x[8] = {};
        if (in) raw[u].unpack(x);
        if (is_q ? a.q_weight != nullptr : a.k_weight != nullptr) {
          float ss = 0.f, weight[8] = {};
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
          for (int off = 8; off; off >>= 1) ss += __shfl_xor_sync(half_mask, ss, off);
          const float inv = rsqrtf(ss / float(d) + a.eps);
          if (in) (is_q ? wq : wk).unpack(weight);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= inv * weight[i];
        }
        if (a.rot) {
          float y[8];
          if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
          } else {
            // the partner lies rot/2 columns away, in another lane: through shared memory
            float* mine = rows[group];
            __syncwarp(half_mask);
            *reinterpret_cast<float4*>(mine + gl * 8) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(mine + gl * 8 + 4) = make_float4(x[4], x[5], x[6], x[7]);
            __syncwarp(half_mask);
            if ((half & 7) == 0) {       // a lane's eight columns have their partners in one lane
              const int e = gl * 8 < half ? gl * 8 + half : (gl * 8 < a.rot ? gl * 8 - half : 0);
              const float4 lo = *reinterpret_cast<const float4*>(mine + e), hi = *reinterpret_cast<const float4*>(mine + e + 4);
              y[0] = lo.x, y[1] = lo.y, y[2] = lo.z, y[3] = lo.w, y[4] = hi.x, y[5] = hi.y, y[6] = hi.z, y[7] = hi.w;
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int e = gl * 8 + i;
                y[i] = e < a.rot ? mine[e < half ? e + half : e - half] : 0.f;
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (gl * 8 + i < a.rot) x[i] = fmaf(y[i], sn[i], x[i] * cs[i]);
        }
        raw[u].pack(x);
      }
      if (!in) continue;
      if (is_q) {
        raw[u].store(static_cast<T*>(a.q_out) + ((long long)t * a.Hq + h) * d + gl * 8);
      } else if (here.page >= 0) {
        T* pool = static_cast<T*>(is_v ? a.v_pages : a.k_pages);
        const long long at = here.page * (is_v ? a.v_page_stride : a.k_page_stride) + (long long)(h * ps + here.slot) * d;
        raw[u].store(pool + at + gl * 8);
        if (is_v && a.weights && gl == 0) a.weights[((long long)here.page * a.Hkv + h) * ps + here.slot] = 0.f;
      }
    }
  }
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
  if (k_page_stride < page || v_page_stride < page || q_token_stride < 0 || q_head_stride < 0 || k_token_stride < 0 ||
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
  if (dtype == CB2_BF16)
    paged_append_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a, batch);
  else
    paged_append_kernel<float><<<grid, kThreads, 0, st>>>(a, batch);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

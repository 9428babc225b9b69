// Attention over a paged key/value cache (see om_paged.cuh): entry point, the kernel for any type on the
// FMA pipes, the join of partial carriers, and the accumulation of attention weight.
//
//   o[t, head] = sum_j softmax_j(scale q.k_j) v_j over the slots j <= len - n + i that row i of the n new
//   tokens of a request sees (all of its len slots without the causal mask); a row that sees nothing is 0.
//   weight[key] += sum over the rows that see it and the heads of its group of the softmax probability.
#include "om_paged.cuh"

namespace cb2 {
namespace {

constexpr int kRT = 16, kKB = 64, kThreads = 128;
using Cost = PagedCost<kRT, kKB, 1>;

template <class T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(bf16lo_to_f32(u.x), bf16hi_to_f32(u.x), bf16lo_to_f32(u.y), bf16hi_to_f32(u.y));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

// Rows [row0, row0 + kRT) of (request, kv head) as fp32 in shared memory, zeros past the last.
template <class T>
__device__ __forceinline__ void load_rows(float* Qs, int ld, const PagedRows& rows, const PagedReq& q, int h, int row0, int d) {
  const T* base = static_cast<const T*>(rows.q);
  for (int e = threadIdx.x; e < kRT * (d / 4); e += kThreads) {
    const int r = e / (d / 4), c = (e % (d / 4)) * 4, row = row0 + r;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < q.n * rows.G) {
      const int tok = row / rows.G, g = row % rows.G;
      v = load4(base + (q.t0 + tok) * rows.q_token + (h * rows.G + g) * rows.q_head + c);
    }
    *reinterpret_cast<float4*>(Qs + r * ld + c) = v;
  }
}

// Keys (or values) [k0, k0 + kKB) of (request r, kv head h), zeros past len: what an unwritten slot
// holds must not reach the products (0 x NaN).
template <class T>
__device__ __forceinline__ void load_keys(float* Ks, int ld, const void* pool, long long page_stride, const PagedBatch& b,
                                          int r, int h, int len, int k0, int d) {
  const T* base = static_cast<const T*>(pool);
  const int ps = 1 << b.page_log2;
  for (int e = threadIdx.x; e < kKB * (d / 4); e += kThreads) {
    const int row = e / (d / 4), c = (e % (d / 4)) * 4, j = k0 + row;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (j < len) {
      const int page = paged_page(b, r, j >> b.page_log2);
      v = load4(base + page * page_stride + (long long)(h * ps + (j & (ps - 1))) * d + c);
    }
    *reinterpret_cast<float4*>(Ks + row * ld + c) = v;
  }
}

// Scores of rows 2 ty, 2 ty + 1 against keys tx + 16 k of the block.
__device__ __forceinline__ void scores_2x4(const float* Qs, const float* Ks, int ld, int d, int ty, int tx, float (&s)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) s[i][k] = 0.f;
  for (int c = 0; c < d; c += 4) {
    float4 q[2], kk[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) q[i] = *reinterpret_cast<const float4*>(Qs + (2 * ty + i) * ld + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) kk[k] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * k) * ld + c);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        s[i][k] = fmaf(q[i].x, kk[k].x, fmaf(q[i].y, kk[k].y, fmaf(q[i].z, kk[k].z, fmaf(q[i].w, kk[k].w, s[i][k]))));
  }
}

// Last slot that a packed row sees (-1: none).
__device__ __forceinline__ int last_slot(const PagedReq& q, int row, int G, int causal) {
  if (row >= q.n * G) return -1;
  return causal ? min(q.len - q.n + row / G, q.len - 1) : q.len - 1;
}

template <class T>
__global__ void __launch_bounds__(kThreads)
paged_fma_kernel(const PagedRows rows, const PagedPools pools, const PagedBatch batch, const Cost cost, T* __restrict__ o,
                 float* __restrict__ lse2, PagedScratch scratch) {
  extern __shared__ __align__(16) float sm[];
  __shared__ PagedFindSmem find;
  const int d = pools.d, ld = d + 4, tid = threadIdx.x;
  float* Qs = sm;
  float* Ks = Qs + kRT * ld;
  float* Vs = Ks + kKB * ld;
  float* Ps = Vs + kKB * d;            // [kRT][kKB + 4]
  float* alphas = Ps + kRT * (kKB + 4);
  constexpr int kLdP = kKB + 4;
  const int cta = blockIdx.x, n_cta = gridDim.x;
  const PagedShare share = paged_find_share<kThreads>(batch, cost, cta, n_cta, &find);
  if (tid == 0) scratch.joins[cta].r = -1;
  const int ty = tid / 16, tx = tid % 16, lane = tid % 32, wq = tid / 32;
  for (PagedWalk<Cost> w(batch, cost, share); w.valid(); w.next()) {
    w.clip();
    const int row0 = w.tile * kRT;
    __syncthreads();
    load_rows<T>(Qs, ld, rows, w.q, w.h, row0, d);
    int lim[2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) lim[i] = last_slot(w.q, row0 + 2 * ty + i, rows.G, cost.causal);
    float acc[4][4] = {};
    for (int kb = w.b0; kb < w.b1; ++kb) {
      const int k0 = kb * kKB;
      __syncthreads();
      load_keys<T>(Ks, ld, pools.k, pools.k_page_stride, batch, w.r, w.h, w.q.len, k0, d);
      load_keys<T>(Vs, d, pools.v, pools.v_page_stride, batch, w.r, w.h, w.q.len, k0, d);
      __syncthreads();
      float s[2][4];
      scores_2x4(Qs, Ks, ld, d, ty, tx, s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          s[i][k] = k0 + tx + 16 * k <= lim[i] ? s[i][k] * rows.scale_log2e : -INFINITY;
          mx = fmaxf(mx, s[i][k]);
        }
#pragma unroll
        for (int off = 8; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_new = fmaxf(m[i], mx);
        const float ref = m_new == -INFINITY ? 0.f : m_new;   // nothing visible yet: every p is 0
        const float alpha = ex2_approx(m[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = ex2_approx(s[i][k] - ref);
          sum += p;
          Ps[(2 * ty + i) * kLdP + tx + 16 * k] = p;
        }
#pragma unroll
        for (int off = 8; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l[i] = l[i] * alpha + sum;
        m[i] = m_new;
        if (tx == 0) alphas[2 * ty + i] = alpha;
      }
      __syncthreads();
      if (4 * lane < d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float al = alphas[4 * wq + i];
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][c] *= al;
        }
        for (int j = 0; j < kKB; j += 4) {
          float4 v[4], p[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(Vs + (j + k) * d + 4 * lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(Ps + (4 * wq + i) * kLdP + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float pp[4] = {p[i].x, p[i].y, p[i].z, p[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              acc[i][0] = fmaf(pp[k], v[k].x, acc[i][0]);
              acc[i][1] = fmaf(pp[k], v[k].y, acc[i][1]);
              acc[i][2] = fmaf(pp[k], v[k].z, acc[i][2]);
              acc[i][3] = fmaf(pp[k], v[k].w, acc[i][3]);
            }
          }
        }
      }
    }
    const bool whole = w.b0 == 0 && w.b1 == w.nb;
    float* ml = Ps;      // m and l of the rows, for the threads that hold the sums
    __syncthreads();
    if (tx == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ml[2 * ty + i] = m[i];
        ml[kRT + 2 * ty + i] = l[i];
      }
    }
    __syncthreads();
    if (whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = 4 * wq + i, row = row0 + rr;
        if (row >= w.q.n * rows.G) continue;
        const float lr = ml[kRT + rr], inv = lr > 0.f ? 1.f / lr : 0.f;
        const long long at = (long long)(w.q.t0 + row / rows.G) * (rows.G * rows.Hkv) + w.h * rows.G + row % rows.G;
        if (4 * lane < d) store4(o + at * d + 4 * lane, make_float4(acc[i][0] * inv, acc[i][1] * inv, acc[i][2] * inv, acc[i][3] * inv));
        if (lse2 && lane == 0) lse2[at] = lr > 0.f ? ml[rr] + log2f(lr) : INFINITY;
      }
    } else {
      if (tid == 0 && w.b0 == 0) paged_write_join(w, share.total, cta, share.n_share, scratch.joins);
      float* slot = scratch.parts + paged_slot_floats(kRT, d) * (2 * cta + (w.b0 == 0));
      if (tid < kRT) {
        slot[tid] = ml[tid];
        slot[kRT + tid] = ml[kRT + tid];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * lane < d)
          *reinterpret_cast<float4*>(slot + 2 * kRT + (4 * wq + i) * d + 4 * lane) =
              make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    }
  }
}

// Joins the partial carriers of a unit, (m, l, a) + (m', l', a') with both scaled to the larger m, over the
// shares c .. last, none of them empty.  Block (c, y) takes rows [RB y, RB y + RB) of the unit that starts in share c.
// A warp holds one row at a time, a lane four columns; with few rows several warps share a row's shares (every
// `stride`-th one) and meet in shared memory, always in the same order.
constexpr int kJoinWarps = 16;

struct Carrier {
  float m, l;
  float4 a;
  __device__ __forceinline__ void add(float m1, float l1, const float4& v) {
    const float m_new = fmaxf(m, m1), ref = m_new == -INFINITY ? 0.f : m_new;
    const float f0 = ex2_approx(m - ref), f1 = ex2_approx(m1 - ref);
    m = m_new;
    l = l * f0 + l1 * f1;
    a = make_float4(a.x * f0 + v.x * f1, a.y * f0 + v.y * f1, a.z * f0 + v.z * f1, a.w * f0 + v.w * f1);
  }
};

template <class T>
__global__ void __launch_bounds__(kJoinWarps * 32)
paged_combine_kernel(const PagedScratch scratch, T* __restrict__ o, float* __restrict__ lse2, const PagedBatch batch, int G, int Hkv,
                     int d) {
  static_assert(kRT == kJoinWarps, "a warp a row");
  __shared__ float sh_m[kJoinWarps], sh_l[kJoinWarps];
  __shared__ __align__(16) float sh_a[kJoinWarps][128];
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PagedJoin j = scratch.joins[c];
  if (j.r < 0) return;
  const PagedReq q = paged_request(batch, j.r);
  const int row_first = j.tile * kRT, n_rows = min(kRT, q.n * G - row_first);
  int stride = 1;                                        // warps a row
  while (stride * 2 * n_rows <= kJoinWarps) stride *= 2;
  const int rr = warp / stride, part = warp % stride, col = 4 * lane;
  const size_t slot = paged_slot_floats(kRT, d);
  Carrier x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  if (rr < n_rows) {
    const float* base = scratch.parts + rr;
#pragma unroll 4
    for (int s = c + part; s <= j.last; s += stride) {
      const float* p = base + slot * (2 * s + (s == c));
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < d) v = *reinterpret_cast<const float4*>(p - rr + 2 * kRT + rr * d + col);
      x.add(p[0], p[kRT], v);
    }
  }
  if (stride > 1) {
    *reinterpret_cast<float4*>(&sh_a[warp][col]) = x.a;
    if (lane == 0) {
      sh_m[warp] = x.m;
      sh_l[warp] = x.l;
    }
    __syncthreads();
    if (part != 0) return;
    for (int w = warp + 1; w < warp + stride; ++w) x.add(sh_m[w], sh_l[w], *reinterpret_cast<const float4*>(&sh_a[w][col]));
  }
  if (rr >= n_rows) return;
  const int row = row_first + rr;
  const float inv = x.l > 0.f ? 1.f / x.l : 0.f;
  const long long at = (long long)(q.t0 + row / G) * (G * Hkv) + j.h * G + row % G;
  if (col < d) store4(o + at * d + col, make_float4(x.a.x * inv, x.a.y * inv, x.a.z * inv, x.a.w * inv));
  if (lse2 && lane == 0) lse2[at] = x.l > 0.f ? x.m + log2f(x.l) : INFINITY;
}

// The same for tiles of 128 rows, a stored [d / 4][128][4]: block (c, y) takes 32 of the rows, a lane one row, a warp
// every eighth group of four columns; the result is turned in shared memory into whole rows.
constexpr int kTileRows = 128, kTileWarps = 8;

__global__ void __launch_bounds__(kTileWarps * 32)
paged_combine_tiles_kernel(const PagedScratch scratch, __nv_bfloat16* __restrict__ o, float* __restrict__ lse2, const PagedBatch batch,
                           int G, int Hkv, int d) {
  __shared__ __align__(16) __nv_bfloat16 sh[32][128 + 8];
  __shared__ long long sh_at[32];
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PagedJoin j = scratch.joins[c];
  if (j.r < 0) return;
  const PagedReq q = paged_request(batch, j.r);
  const int in_tile = blockIdx.y * 32 + lane, row = j.tile * kTileRows + in_tile;
  const int n_rows = min(32, q.n * G - j.tile * kTileRows - int(blockIdx.y) * 32);
  if (n_rows <= 0) return;
  const size_t slot = paged_slot_floats(kTileRows, d);
  constexpr int kGroups = 128 / 4 / kTileWarps;
  Carrier x[kGroups];
#pragma unroll
  for (int k = 0; k < kGroups; ++k) x[k] = Carrier{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  if (lane < n_rows) {
    for (int s = c; s <= j.last; ++s) {
      const float* p = scratch.parts + slot * (2 * s + (s == c)) + in_tile;
      float4 v[kGroups];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const int c4 = warp + k * kTileWarps;
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c4 * 4 < d) v[k] = *reinterpret_cast<const float4*>(p - in_tile + 2 * kTileRows + (c4 * kTileRows + in_tile) * 4);
      }
      const float m1 = p[0], l1 = p[kTileRows];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) x[k].add(m1, l1, v[k]);
    }
    const float inv = x[0].l > 0.f ? 1.f / x[0].l : 0.f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
      store4(&sh[lane][(warp + k * kTileWarps) * 4], make_float4(x[k].a.x * inv, x[k].a.y * inv, x[k].a.z * inv, x[k].a.w * inv));
    if (warp == 0) {
      const long long at = (long long)(q.t0 + row / G) * (G * Hkv) + j.h * G + row % G;
      sh_at[lane] = at;
      if (lse2) lse2[at] = x[0].l > 0.f ? x[0].m + log2f(x[0].l) : INFINITY;
    }
  }
  __syncthreads();
  const int col = (threadIdx.x & 15) * 8;
  for (int rr = threadIdx.x >> 4; rr < n_rows; rr += kTileWarps * 2)
    if (col < d) *reinterpret_cast<uint4*>(o + sh_at[rr] * d + col) = *reinterpret_cast<const uint4*>(&sh[rr][col]);
}

// weight[key] += sum over rows of 2^(score - lse): a share of (request, kv head, key block) units per CTA,
// every key of a block summed by one CTA over all rows in order.
template <class T>
__global__ void __launch_bounds__(kThreads)
paged_weights_fma_kernel(PagedRows rows, PagedPools pools, PagedBatch batch, Cost cost,
                         const float* __restrict__ lse2, float* __restrict__ weights) {
  extern __shared__ __align__(16) float sm[];
  const int d = pools.d, ld = d + 4, tid = threadIdx.x;
  float* Qs = sm;
  float* Ks = Qs + kRT * ld;
  float* part = Ks + kKB * ld;         // [8][kKB]
  const int ps = 1 << batch.page_log2;
  const int ty = tid / 16, tx = tid % 16;
  const int kb = blockIdx.x, h = blockIdx.y;
  for (int r = blockIdx.z; r < batch.R; r += gridDim.z) {
    const PagedReq q = paged_request(batch, r);
    if (!cost.takes(q) || kb * kKB >= q.len) continue;
    const int k0 = kb * kKB;
    __syncthreads();
    load_keys<T>(Ks, ld, pools.k, pools.k_page_stride, batch, r, h, q.len, k0, d);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int row0 = 0; row0 < q.n * rows.G; row0 += kRT) {
      if (last_slot(q, min(row0 + kRT, q.n * rows.G) - 1, rows.G, cost.causal) < k0) continue;
      __syncthreads();
      load_rows<T>(Qs, ld, rows, q, h, row0, d);
      __syncthreads();
      float s[2][4];
      scores_2x4(Qs, Ks, ld, d, ty, tx, s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + 2 * ty + i, lim = last_slot(q, row, rows.G, cost.causal);
        if (lim < 0) continue;
        const long long at = (long long)(q.t0 + row / rows.G) * (rows.G * rows.Hkv) + h * rows.G + row % rows.G;
        const float z = lse2[at];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k0 + tx + 16 * k <= lim) sum[k] += ex2_approx(fmaf(s[i][k], rows.scale_log2e, -z));
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) part[ty * kKB + tx + 16 * k] = sum[k];
    __syncthreads();
    if (tid < kKB && k0 + tid < q.len) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += part[i * kKB + tid];
      const int j = k0 + tid, page = paged_page(batch, r, j >> batch.page_log2);
      weights[((long long)page * rows.Hkv + h) * ps + (j & (ps - 1))] += s;
    }
  }
}

// CTAs of the FMA kernel: three per SM hold its shared memory for d = 128.
constexpr int kFmaCtas = kNumSMs * 3;

size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

// Which kernels a bf16 call takes.  A request of at most `few` packed rows is bound by reading its keys and
// goes to the streaming kernel, whose products hold 8 or 16 rows; the others go to the tensor-core tiles.
struct Plan {
  int few;                     // 0: no streaming kernel
  bool chunks;
  size_t lse, scores, parts, total;
};

// Attention weight of few rows is summed from scores that the streaming kernel leaves in scratch (4 bytes per
// row and key, against 2 d bytes for reading the keys again), up to this size.
constexpr size_t kMostScores = size_t(256) << 20;

Plan plan(int n_tokens, int R, int Hq, int Hkv, int d, int max_q, int max_k, bool weights, int dtype) {
  Plan p{};
  const int G = Hq / Hkv;
  p.lse = weights ? up16(size_t(n_tokens) * Hq * 4) : 0;
  if (dtype == CB2_F32) {
    p.parts = paged_scratch_bytes(kFmaCtas, kRT, d);
  } else {
    const int64_t rows = int64_t(max_q) * G;
    if (rows <= 16) {
      p.few = rows <= 8 ? 8 : 16;
    } else {
      p.chunks = true;
      p.few = R == 1 || G > 16 ? 0 : (G <= 8 ? 8 : 16);       // the single tokens of a mixed batch
    }
    p.parts = p.chunks ? paged_tc_scratch_bytes(d) : 0;
    if (p.few && paged_few_scratch_bytes(d) > p.parts) p.parts = paged_few_scratch_bytes(d);   // one after the other
    if (weights && p.few) {
      const size_t s = size_t(R) * Hkv * p.few * max_k * 4;
      p.scores = s <= kMostScores ? up16(s) : 0;
    }
  }
  if (weights && dtype == CB2_BF16 && paged_weights_tc_scratch_bytes() > p.parts) p.parts = paged_weights_tc_scratch_bytes();
  p.parts = up16(p.parts);
  p.total = p.lse + p.scores + p.parts;
  return p;
}

template <class T>
int join(int n_cta, const PagedScratch& ws, T* o, float* lse2, const PagedBatch& batch, const PagedRows& rows, int d, cudaStream_t st) {
  paged_combine_kernel<T><<<n_cta, kJoinWarps * 32, 0, st>>>(ws, o, lse2, batch, rows.G, rows.Hkv, d);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

int join_tiles(int n_cta, const PagedScratch& ws, __nv_bfloat16* o, float* lse2, const PagedBatch& batch, const PagedRows& rows, int d,
               cudaStream_t st) {
  paged_combine_tiles_kernel<<<dim3(n_cta, kTileRows / 32), kTileWarps * 32, 0, st>>>(ws, o, lse2, batch, rows.G, rows.Hkv, d);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

template <class T>
int fma_weights(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, const Cost& cost,
                const float* lse2, float* weights, cudaStream_t st) {
  const int ld = pools.d + 4, smem = (kRT * ld + kKB * ld + 8 * kKB) * 4;
  if (cudaFuncSetAttribute(paged_weights_fma_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return CB2_LAUNCH_FAIL;
  const dim3 grid((batch.max_k + kKB - 1) / kKB, rows.Hkv, batch.R < 256 ? batch.R : 256);
  paged_weights_fma_kernel<T><<<grid, kThreads, smem, st>>>(rows, pools, batch, cost, lse2, weights);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

int run_f32(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, float* o, float* weights,
            char* scratch, const Plan& p, cudaStream_t st) {
  const Cost cost{rows.G, rows.Hkv, causal, kPagedAll, 0, 2};
  float* lse2 = weights ? reinterpret_cast<float*>(scratch) : nullptr;
  const PagedScratch ws = paged_scratch(scratch + p.lse, kFmaCtas);
  const int d = pools.d, ld = d + 4;
  const int smem = (kRT * ld + kKB * ld + kKB * d + kRT * (kKB + 4) + kRT) * 4;
  if (cudaFuncSetAttribute(paged_fma_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return CB2_LAUNCH_FAIL;
  paged_fma_kernel<float><<<kFmaCtas, kThreads, smem, st>>>(rows, pools, batch, cost, o, lse2, ws);
  CB2_LAUNCH_CHECK();
  int rc = join(kFmaCtas, ws, o, lse2, batch, rows, d, st);
  if (rc == CB2_OK && weights) rc = fma_weights<float>(rows, pools, batch, cost, lse2, weights, st);
  return rc;
}

int run_bf16(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, __nv_bfloat16* o, float* weights,
             char* scratch, const Plan& p, cudaStream_t st) {
  float* lse2 = weights ? reinterpret_cast<float*>(scratch) : nullptr;
  float* scores = p.scores ? reinterpret_cast<float*>(scratch + p.lse) : nullptr;
  char* parts = scratch + p.lse + p.scores;
  PagedScratch ws;
  int n_cta, rc = CB2_OK;
  if (p.chunks) {
    rc = paged_tc_run(rows, pools, batch, causal, p.few, o, lse2, parts, &ws, &n_cta, st);
    if (rc == CB2_OK) rc = join_tiles(n_cta, ws, o, lse2, batch, rows, pools.d, st);
    if (rc == CB2_OK && weights) rc = paged_weights_tc_run(rows, pools, batch, causal, kPagedChunk, p.few, lse2, weights, parts, st);
  }
  if (rc == CB2_OK && p.few) {
    rc = paged_few_run(rows, pools, batch, causal, p.few, o, lse2, scores, parts, &ws, &n_cta, st);
    if (rc == CB2_OK) rc = join(n_cta, ws, o, lse2, batch, rows, pools.d, st);
    if (rc == CB2_OK && scores) rc = paged_few_weights_run(rows, batch, causal, p.few, scores, lse2, weights, st);
    if (rc == CB2_OK && weights && !scores)
      rc = paged_weights_tc_run(rows, pools, batch, causal, kPagedFew, p.few, lse2, weights, parts, st);
  }
  return rc;
}

bool sizes_ok(int n_tokens, int R, int Hq, int Hkv, int d, int max_q, int max_k) {
  if (n_tokens < 0 || R < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || Hkv > 65535 || d < 8 || d > 128 || d % 8 || max_q < 0 || max_k < 1) return false;
  // the cost line counts in 32 bits inside a request
  return (int64_t(n_tokens) + max_k + 256) * (Hq / Hkv) < (int64_t(1) << 30);
}

}  // namespace
}  // namespace cb2

extern "C" size_t cb2_om_paged_scratch_bytes(int n_tokens, int R, int Hq, int Hkv, int d, int max_q, int max_k, int weights,
                                             int dtype) {
  using namespace cb2;
  if (!sizes_ok(n_tokens, R, Hq, Hkv, d, max_q, max_k) || n_tokens == 0) return 0;
  if (dtype != CB2_F32 && dtype != CB2_BF16) return 0;
  return plan(n_tokens, R, Hq, Hkv, d, max_q, max_k, weights != 0, dtype).total;
}

extern "C" int cb2_om_paged_fwd(const void* q, long long q_token_stride, long long q_head_stride, const void* k_pages,
                                const void* v_pages, long long k_page_stride, long long v_page_stride, void* o,
                                float* weights, const int* block_table, const int* seq_lens, const int* cu_q, int n_tokens,
                                int R, int Hq, int Hkv, int d, int page_size, int n_pages, int max_pages, int max_q,
                                int max_k, float scale, int causal, int dtype, void* scratch, size_t scratch_bytes,
                                int* dev_status, void* stream) {
  using namespace cb2;
  if (!k_pages || !v_pages || !block_table || !seq_lens || !cu_q) return CB2_NULL_PTR;
  if (!sizes_ok(n_tokens, R, Hq, Hkv, d, max_q, max_k)) return CB2_BAD_SHAPE;
  if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1)) || n_pages < 1 || max_pages < 1) return CB2_BAD_SHAPE;
  if (int64_t(max_pages) * page_size < max_k || !(scale > 0.f) || scale > 3e38f) return CB2_BAD_SHAPE;
  const long long page = (long long)Hkv * page_size * d;
  if (k_page_stride < page || v_page_stride < page || q_token_stride < 0 || q_head_stride < 0) return CB2_BAD_SHAPE;
  if ((n_tokens > 1 && q_token_stride == 0) || (Hq > 1 && q_head_stride == 0)) return CB2_BAD_SHAPE;
  if (dtype != CB2_BF16 && dtype != CB2_F32) return CB2_UNSUPPORTED_DTYPE;
  if (n_tokens == 0) return CB2_OK;
  if (!q || !o || !scratch) return CB2_NULL_PTR;
  const int vec = dtype == CB2_BF16 ? 8 : 4;      // elements in 16 bytes
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o) || !aligned16(scratch) ||
      q_token_stride % vec || q_head_stride % vec || k_page_stride % vec || v_page_stride % vec)
    return CB2_BAD_ALIGN;
  const Plan p = plan(n_tokens, R, Hq, Hkv, d, max_q, max_k, weights != nullptr, dtype);
  if (scratch_bytes < p.total) return CB2_SCRATCH_TOO_SMALL;
  int page_log2 = 0;
  while ((1 << page_log2) < page_size) ++page_log2;
  const PagedBatch batch{block_table, seq_lens, cu_q, R, max_pages, n_pages, page_log2, n_tokens, max_q, max_k, dev_status};
  const PagedPools pools{k_pages, v_pages, k_page_stride, v_page_stride, Hkv, d};
  const PagedRows rows{q, q_token_stride, q_head_stride, Hq / Hkv, Hkv, scale * 1.4426950408889634f};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(scratch);
  if (dtype == CB2_BF16) return run_bf16(rows, pools, batch, causal != 0, static_cast<__nv_bfloat16*>(o), weights, ws, p, st);
  return run_f32(rows, pools, batch, causal != 0, static_cast<float*>(o), weights, ws, p, st);
}

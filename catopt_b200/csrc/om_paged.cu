// Attention over a paged key/value cache (see om_paged.cuh): the entry point, which kernels a call takes, and the
// join of partial carriers.
//
//   o[t, head] = sum_j softmax_j(scale q.k_j) v_j over the slots j <= len - n + i that row i of the n new
//   tokens of a request sees (all of its len slots without the causal mask); a row that sees nothing is 0.
//   weight[key] += sum over the rows that see it and the heads of its group of the softmax probability.
#include "om_paged.cuh"

namespace cb2 {
namespace {

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

// Joins the partial carriers of a unit, (m, l, a) + (m', l', a') with both scaled to the larger m, over the
// shares c .. last, none of them empty.  Block (c, y) takes rows [16 y, 16 y + 16) of the unit that starts in share c.
// A warp holds one row, a lane four columns; with few rows several warps share a row's shares (every
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
paged_combine_kernel(int rt, const PagedScratch scratch, T* __restrict__ o, float* __restrict__ lse2, int G, int Hkv, int d) {
  __shared__ float sh_m[kJoinWarps], sh_l[kJoinWarps];
  __shared__ __align__(16) float sh_a[kJoinWarps][128];
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  let_next();
  after_previous();
  const PagedJoin j = scratch.joins[c];
  if (j.r < 0) return;
  const int in_tile = blockIdx.y * kJoinWarps, row_first = j.tile * rt + in_tile, n_rows = min(kJoinWarps, j.n * G - row_first);
  if (n_rows <= 0) return;
  int stride = 1;                                        // warps a row
  while (stride * 2 * n_rows <= kJoinWarps) stride *= 2;
  const int rr = warp / stride, part = warp % stride, col = 4 * lane;
  const size_t slot = paged_slot_floats(rt, d);
  Carrier x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  if (rr < n_rows) {
    const float* base = scratch.parts + in_tile + rr;
#pragma unroll 8
    for (int s = c + part; s <= j.last; s += stride) {
      const float* p = base + slot * (2 * s + (s == c));
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < d) v = *reinterpret_cast<const float4*>(p - in_tile - rr + 2 * rt + (in_tile + rr) * d + col);
      x.add(p[0], p[rt], v);
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
  const float inv = x.l == 0.f ? 0.f : 1.f / x.l;      // a NaN sum stays one
  const long long at = (long long)(j.t0 + row / G) * (G * Hkv) + j.h * G + row % G;
  if (col < d) store4(o + at * d + col, make_float4(x.a.x * inv, x.a.y * inv, x.a.z * inv, x.a.w * inv));
  if (lse2 && lane == 0) lse2[at] = x.l == 0.f ? INFINITY : x.m + log2f(x.l);
}

// The same for tiles of 128 rows, a stored [d / 4][128][4]: block (c, y) takes 32 of the rows, a lane one row, a warp
// every eighth group of four columns; the result is turned in shared memory into whole rows.
constexpr int kTileRows = 128, kTileWarps = 8;

__global__ void __launch_bounds__(kTileWarps * 32)
paged_combine_tiles_kernel(const PagedScratch scratch, __nv_bfloat16* __restrict__ o, float* __restrict__ lse2, int G, int Hkv, int d) {
  __shared__ __align__(16) __nv_bfloat16 sh[32][128 + 8];
  __shared__ long long sh_at[32];
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  let_next();
  after_previous();
  const PagedJoin j = scratch.joins[c];
  if (j.r < 0) return;
  const int in_tile = blockIdx.y * 32 + lane, row = j.tile * kTileRows + in_tile;
  const int n_rows = min(32, j.n * G - j.tile * kTileRows - int(blockIdx.y) * 32);
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
    const float inv = x[0].l == 0.f ? 0.f : 1.f / x[0].l;
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
      store4(&sh[lane][(warp + k * kTileWarps) * 4], make_float4(x[k].a.x * inv, x[k].a.y * inv, x[k].a.z * inv, x[k].a.w * inv));
    if (warp == 0) {
      const long long at = (long long)(j.t0 + row / G) * (G * Hkv) + j.h * G + row % G;
      sh_at[lane] = at;
      if (lse2) lse2[at] = x[0].l == 0.f ? INFINITY : x[0].m + log2f(x[0].l);
    }
  }
  __syncthreads();
  const int col = (threadIdx.x & 15) * 8;
  for (int rr = threadIdx.x >> 4; rr < n_rows; rr += kTileWarps * 2)
    if (col < d) *reinterpret_cast<uint4*>(o + sh_at[rr] * d + col) = *reinterpret_cast<const uint4*>(&sh[rr][col]);
}

constexpr float kLog2e = 1.4426950408889634f;
size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

// Which kernels a call takes.  Requests of at most `few` packed rows are bound by reading their keys: a batch of
// nothing else goes to the streaming kernel (bf16: products with 8 or 16 rows; fp32: tiles of 8 or 16 rows).  A batch
// with chunks goes to the wide tiles as a whole in bf16: their line takes single tokens at the pace of memory, too, and
// the two launches more of the streaming kernel never paid (31 single tokens on up to 16384 keys beside a chunk of 64:
// 237 us with one kernel, 255 with both; 21 on up to 2048 beside three chunks: 45 and 62).  In fp32 a row that is not
// there costs as much as one that is, so there the few rows of a mixed batch have the narrow tiles, unless the batch is
// sure to be small.  Measured with a chunk of 64 beside 1, 3, 7, 15 or 31 single tokens on up to 128, 512, 2048 or 8192
// keys, 32 heads on 8 (d 128), 8 on 2 and 4 on 4 (d 64): with up to 4 blocks an SM one kernel is the faster, by up to 21 us
// (but for one case, 66 us and 64 with both); from 14 on both are, or are within 3 % (16 blocks an SM: 148 us with one, 112 with
// both; 223: 1706 and 1076); around 8 it goes either way (95 and 79; 43 and 51).
struct Plan {
  int few;                     // 0: no streaming kernel
  bool chunks;
  size_t lse, scores, parts, total;
};

// Attention weight of few rows is summed from scores that the streaming kernel leaves in scratch (4 bytes per
// row and key, against d elements for reading the keys again), up to this size.
constexpr size_t kMostScores = size_t(256) << 20;

Plan plan(int n_tokens, int R, int Hq, int Hkv, int d, int max_q, int max_k, bool weights, int dtype) {
  Plan p{};
  const int G = Hq / Hkv;
  const int64_t rows = int64_t(max_q) * G;
  if (rows <= 16) {
    p.few = rows <= 8 ? 8 : 16;
  } else {
    p.chunks = true;
    const int64_t blocks = int64_t(R) * Hkv * (1 + (max_k + 63) / 64);
    if (dtype == CB2_F32 && R > 1 && G <= 16 && blocks > 8 * kNumSMs) p.few = G <= 8 ? 8 : 16;
  }
  p.lse = weights ? up16(size_t(n_tokens) * Hq * 4) : 0;
  if (weights && p.few) {
    const size_t s = size_t(R) * Hkv * p.few * paged_score_stride(max_k) * 4;
    p.scores = s <= kMostScores ? up16(s) : 0;
  }
  auto at_least = [&p](size_t n) { p.parts = n > p.parts ? n : p.parts; };      // the kernels use it one after the other
  if (dtype == CB2_BF16) {
    if (p.chunks) at_least(paged_tc_scratch_bytes(d));
    if (p.few) at_least(paged_few_scratch_bytes(d));
    if (weights) at_least(paged_weights_tc_scratch_bytes());
  } else {
    if (p.chunks) at_least(paged_fma_scratch_bytes(64, d));
    if (p.few) at_least(paged_fma_scratch_bytes(p.few, d));
  }
  p.parts = up16(p.parts);
  p.total = p.lse + p.scores + p.parts;
  return p;
}

template <class T>
int join(int rt, int n_cta, const PagedScratch& ws, T* o, float* lse2, const PagedRows& rows, int d, cudaStream_t st) {
  return launch_next(paged_combine_kernel<T>, dim3(n_cta, (rt + kJoinWarps - 1) / kJoinWarps), kJoinWarps * 32, st, rt, ws, o, lse2, rows.G,
                     rows.Hkv, d);
}

int join_tiles(int n_cta, const PagedScratch& ws, __nv_bfloat16* o, float* lse2, const PagedRows& rows, int d, cudaStream_t st) {
  return launch_next(paged_combine_tiles_kernel, dim3(n_cta, kTileRows / 32), kTileWarps * 32, st, ws, o, lse2, rows.G, rows.Hkv, d);
}

int run_f32(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, float* o, float* weights,
            char* scratch, const Plan& p, cudaStream_t st) {
  float* lse2 = weights ? reinterpret_cast<float*>(scratch) : nullptr;
  float* scores = p.scores ? reinterpret_cast<float*>(scratch + p.lse) : nullptr;
  char* parts = scratch + p.lse + p.scores;
  PagedScratch ws;
  int n_cta, rc = CB2_OK;
  if (p.chunks) {
    rc = paged_fma_run(64, rows, pools, batch, causal, kPagedChunk, p.few, o, lse2, nullptr, parts, &ws, &n_cta, st);
    if (rc == CB2_OK) rc = join(64, n_cta, ws, o, lse2, rows, pools.d, st);
    if (rc == CB2_OK && weights) rc = paged_weights_fma_run(rows, pools, batch, causal, kPagedChunk, p.few, lse2, weights, st);
  }
  if (rc == CB2_OK && p.few) {
    rc = paged_fma_run(p.few, rows, pools, batch, causal, kPagedFew, p.few, o, lse2, scores, parts, &ws, &n_cta, st);
    if (rc == CB2_OK) rc = join(p.few, n_cta, ws, o, lse2, rows, pools.d, st);
    if (rc == CB2_OK && scores) rc = paged_few_weights_run(rows, batch, causal, p.few, scores, lse2, weights, st);
    if (rc == CB2_OK && weights && !scores) rc = paged_weights_fma_run(rows, pools, batch, causal, kPagedFew, p.few, lse2, weights, st);
  }
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
    if (rc == CB2_OK) rc = join_tiles(n_cta, ws, o, lse2, rows, pools.d, st);
    if (rc == CB2_OK && weights) rc = paged_weights_tc_run(rows, pools, batch, causal, kPagedChunk, p.few, lse2, weights, parts, st);
  }
  if (rc == CB2_OK && p.few) {
    rc = paged_few_run(rows, pools, batch, causal, p.few, o, lse2, scores, parts, &ws, &n_cta, st);
    if (rc == CB2_OK) rc = join(16, n_cta, ws, o, lse2, rows, pools.d, st);
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
  if (int64_t(max_pages) * page_size < max_k || !(scale > 0.f) || !(scale * kLog2e < INFINITY)) return CB2_BAD_SHAPE;
  const long long page = (long long)Hkv * page_size * d;
  if (k_page_stride < page || v_page_stride < page || q_token_stride < 0 || q_head_stride < 0) return CB2_BAD_SHAPE;
  if ((n_tokens > 1 && q_token_stride == 0) || (Hq > 1 && q_head_stride == 0)) return CB2_BAD_SHAPE;
  if (dtype != CB2_BF16 && dtype != CB2_F32) return CB2_UNSUPPORTED_DTYPE;
  if (n_tokens == 0) return CB2_OK;
  if (!q || !o || !scratch) return CB2_NULL_PTR;
  const int vec = dtype == CB2_BF16 ? 8 : 4;      // elements in 16 bytes
  if (!aligned16(q) || !aligned16(weights) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o) || !aligned16(scratch) ||
      q_token_stride % vec || q_head_stride % vec || k_page_stride % vec || v_page_stride % vec)
    return CB2_BAD_ALIGN;
  const Plan p = plan(n_tokens, R, Hq, Hkv, d, max_q, max_k, weights != nullptr, dtype);
  if (scratch_bytes < p.total) return CB2_SCRATCH_TOO_SMALL;
  // rows of q are read after others of o have been written
  const int esz = dtype == CB2_BF16 ? 2 : 4;
  if (paged_rows_meet(q, n_tokens, q_token_stride, Hq, q_head_stride, d, esz, o, (long long)n_tokens * Hq * d * esz)) return CB2_BAD_SHAPE;
  int page_log2 = 0;
  while ((1 << page_log2) < page_size) ++page_log2;
  const PagedBatch batch{block_table, seq_lens, cu_q, R, max_pages, n_pages, page_log2, n_tokens, max_q, max_k, dev_status};
  const PagedPools pools{k_pages, v_pages, k_page_stride, v_page_stride, Hkv, d};
  const PagedRows rows{q, q_token_stride, q_head_stride, Hq / Hkv, Hkv, scale * kLog2e};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(scratch);
  if (dtype == CB2_BF16) return run_bf16(rows, pools, batch, causal != 0, static_cast<__nv_bfloat16*>(o), weights, ws, p, st);
  return run_f32(rows, pools, batch, causal != 0, static_cast<float*>(o), weights, ws, p, st);
}

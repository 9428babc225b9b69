// Attention over a paged key/value cache in fp32, on the FMA pipes, over the work line of om_paged.cuh.
//
// Row tiles: 8 or 16 packed rows for requests of few rows (single tokens: rows that are not there cost as much as
// others), 64 for chunks, where every key block that is read serves 64 rows (with 16, reading keys from L2 at the FMA
// pipes' pace would take 9 TB/s).
// A CTA keeps its rows in shared memory and walks 64-key blocks in two stages: the block after next is looked up in the
// page table, the next one is on its way by asynchronous copies, the present one is worked on: scores as SR x KP patches of
// registers, row statistics by shuffles among the KX lanes that share rows, P through shared memory, O as RP x 4 patches.
//
// Measured, 32 heads on 8, d 128: 1024 tokens on 4096 keys 2.0 ms, 30 TFLOP/s (of about 72 on the FMA pipes; shared-memory
// reads feed 16 products a 16-byte load); 16 single tokens on up to 8192 keys 0.38 ms, 1.6 TB/s, bound by the eight rows that
// are worked out for four.
#include "om_paged.cuh"

namespace cb2 {
namespace {

constexpr int kKB = 64;

template <int RT_>
struct Tile {
  static constexpr int RT = RT_, kThreads = RT <= 16 ? 128 : 256;
  static constexpr int KX = RT == 8 ? 32 : 16, KP = kKB / KX;     // lanes that share rows, keys a lane
  static constexpr int SR = RT * KX / kThreads;              // score rows a thread
  static constexpr int kLdP = kKB + 4;
  using Cost = PagedCost<RT, kKB, 1>;
  static int smem_bytes(int d) {
    return (RT * (d + 4) + 2 * (kKB * (d + 4) + kKB * d) + RT * kLdP + 2 * RT) * 4;
  }
  // CTAs that run side by side: shared memory decides
  static int ctas(int d) { return kNumSMs * (227 * 1024 / (smem_bytes(d) + 2048)); }
};

// Copies rows of 16-byte chunks into shared memory, zeros where a row is not there (`any`: an address to name then).
template <int THREADS, class At>
__device__ __forceinline__ void copy_rows(float* dst, int ld, int rows, int d, const void* any, At at) {
  const int nv = d / 4;
  for (int e = threadIdx.x; e < rows * nv; e += THREADS) {
    const int r = e / nv, c = (e - r * nv) * 4;
    const float* src = at(r);
    cp_async16_or_zero(smem_u32(dst + r * ld + c), src ? src + c : any, src != nullptr);
  }
}

// Last slot that a packed row sees (-1: none).
__device__ __forceinline__ int last_slot(const PagedReq& q, int row, int G, int causal) {
  if (row >= q.n * G) return -1;
  return causal ? min(q.len - q.n + row / G, q.len - 1) : q.len - 1;
}

// Scores of rows SR ty .. SR ty + SR - 1 against keys tx + KX k, k < KP, of a block.
template <int SR, int KX, int KP>
__device__ __forceinline__ void scores(const float* Qs, const float* Ks, int ld, int d, int ty, int tx, float (&s)[SR][KP]) {
#pragma unroll
  for (int i = 0; i < SR; ++i)
#pragma unroll
    for (int k = 0; k < KP; ++k) s[i][k] = 0.f;
#pragma unroll 2
  for (int c = 0; c < d; c += 4) {
    float4 q[SR], kk[KP];
#pragma unroll
    for (int i = 0; i < SR; ++i) q[i] = *reinterpret_cast<const float4*>(Qs + (SR * ty + i) * ld + c);
#pragma unroll
    for (int k = 0; k < KP; ++k) kk[k] = *reinterpret_cast<const float4*>(Ks + (tx + KX * k) * ld + c);
#pragma unroll
    for (int i = 0; i < SR; ++i)
#pragma unroll
      for (int k = 0; k < KP; ++k)
        s[i][k] = fmaf(q[i].x, kk[k].x, fmaf(q[i].y, kk[k].y, fmaf(q[i].z, kk[k].z, fmaf(q[i].w, kk[k].w, s[i][k]))));
  }
}

template <int RT, int CG>
__global__ void __launch_bounds__(Tile<RT>::kThreads)
paged_fma_kernel(const PagedRows rows, const PagedPools pools, const PagedBatch batch, const typename Tile<RT>::Cost cost,
                 float* __restrict__ o, float* __restrict__ lse2, float* __restrict__ kept_scores, const PagedScratch scratch) {
  using TT = Tile<RT>;
  using Cost = typename TT::Cost;
  constexpr int kThreads = TT::kThreads, SR = TT::SR, KX = TT::KX, KP = TT::KP, kLdP = TT::kLdP;
  constexpr int RP = RT * CG / kThreads;                     // rows a thread sums O for, by 4 columns
  extern __shared__ __align__(16) float sm[];
  __shared__ PagedFindSmem find;
  __shared__ int pages[2][kKB / 8];
  const int d = pools.d, ld = d + 4, tid = threadIdx.x, G = rows.G;
  float* Qs = sm;
  float* Ks = Qs + RT * ld;                                  // [2][kKB][ld]
  float* Vs = Ks + 2 * kKB * ld;                             // [2][kKB][d]
  float* Ps = Vs + 2 * kKB * d;                              // [RT][kLdP]
  float* stat = Ps + RT * kLdP;                              // rescaling of a block, then m and l
  const int cta = blockIdx.x, n_cta = gridDim.x;
  let_next();
  const PagedShare share = paged_find_share<kThreads>(batch, cost, cta, n_cta, &find);
  if (tid == 0) scratch.joins[cta].r = -1;
  const int ty = tid / KX, tx = tid % KX, cg = tid % CG, rg = tid / CG;
  const int ps = 1 << batch.page_log2;
  const float* qb = static_cast<const float*>(rows.q);
  for (PagedWalk<Cost> w(batch, cost, share); w.valid(); w.next()) {
    w.clip();
    const int row0 = w.tile * RT, n_rows = w.q.n * G, len = w.q.len;
    // pages of a block, one entry for every 8 keys; -1 behind the length
    auto look_up = [&](int kb) {
      if (tid < kKB / 8 && kb < w.b1) {
        const int j = kb * kKB + tid * 8;
        pages[kb & 1][tid] = j < len ? paged_page(batch, w.r, j >> batch.page_log2) : -1;
      }
    };
    auto fetch = [&](int kb) {
      if (kb < w.b1) {
        const int k0 = kb * kKB, st = kb & 1;
        auto key = [&](const void* pool, long long stride, int r) -> const float* {
          const int j = k0 + r;
          if (j >= len) return nullptr;          // what an unwritten slot holds must not reach the products (0 x NaN)
          return static_cast<const float*>(pool) + pages[st][r >> 3] * stride + (long long)(w.h * ps + (j & (ps - 1))) * d;
        };
        copy_rows<kThreads>(Ks + st * kKB * ld, ld, kKB, d, pools.k, [&](int r) { return key(pools.k, pools.k_page_stride, r); });
        copy_rows<kThreads>(Vs + st * kKB * d, d, kKB, d, pools.v, [&](int r) { return key(pools.v, pools.v_page_stride, r); });
      }
      cp_async_commit();
    };
    __syncthreads();
    copy_rows<kThreads>(Qs, ld, RT, d, qb, [&](int r) -> const float* {
      const int row = row0 + r;
      return row < n_rows ? qb + (w.q.t0 + row / G) * rows.q_token + (w.h * G + row % G) * rows.q_head : nullptr;
    });
    look_up(w.b0);
    __syncthreads();
    fetch(w.b0);
    look_up(w.b0 + 1);
    int lim[SR];
    float m[SR], l[SR], acc[RP][4];
#pragma unroll
    for (int i = 0; i < SR; ++i) {
      lim[i] = last_slot(w.q, row0 + SR * ty + i, G, cost.causal);
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < RP; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
    for (int kb = w.b0; kb < w.b1; ++kb) {
      const int k0 = kb * kKB, st = kb & 1;
      cp_async_wait_all();
      __syncthreads();               // this block is there, its other stage and the next block's pages, too
      fetch(kb + 1);
      float s[SR][KP];
      scores<SR, KX, KP>(Qs, Ks + st * kKB * ld, ld, d, ty, tx, s);
#pragma unroll
      for (int i = 0; i < SR; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < KP; ++k) {
          s[i][k] = k0 + tx + KX * k <= lim[i] ? s[i][k] * rows.scale_log2e : -INFINITY;
          mx = fmaxf(mx, s[i][k]);
        }
        if (kept_scores && row0 + SR * ty + i < n_rows) {
          float* to = kept_scores + (((long long)w.r * rows.Hkv + w.h) * cost.few + row0 + SR * ty + i) * paged_score_stride(batch.max_k) + k0 + tx;
#pragma unroll
          for (int k = 0; k < KP; ++k)
            if (k0 + tx + KX * k < len) to[KX * k] = s[i][k];
        }
#pragma unroll
        for (int off = KX / 2; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_new = fmaxf(m[i], mx);
        const float ref = m_new == -INFINITY ? 0.f : m_new;   // nothing visible yet: every p is 0
        const float alpha = ex2_approx(m[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < KP; ++k) {
          const float p = ex2_approx(s[i][k] - ref);
          sum += p;
          Ps[(SR * ty + i) * kLdP + tx + KX * k] = p;
        }
#pragma unroll
        for (int off = KX / 2; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l[i] = l[i] * alpha + sum;
        m[i] = m_new;
        if (tx == 0) stat[SR * ty + i] = alpha;
      }
      __syncthreads();
      look_up(kb + 2);               // (the copies of block kb + 1, which reads the other entry, have been issued)
      if (4 * cg < d) {
        const float* V = Vs + st * kKB * d + 4 * cg;
        const float* P = Ps + RP * rg * kLdP;
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          const float al = stat[RP * rg + i];
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][c] *= al;
        }
#pragma unroll 2
        for (int j = 0; j < kKB; j += 4) {
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(V + (j + k) * d);
#pragma unroll
          for (int i = 0; i < RP; ++i) {
            const float4 p = *reinterpret_cast<const float4*>(P + i * kLdP + j);
            const float pp[4] = {p.x, p.y, p.z, p.w};
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
    cp_async_wait_all();
    __syncthreads();
    if (tx == 0) {
#pragma unroll
      for (int i = 0; i < SR; ++i) {
        stat[SR * ty + i] = m[i];
        stat[RT + SR * ty + i] = l[i];
      }
    }
    __syncthreads();
    const bool whole = w.b0 == 0 && w.b1 == w.nb;
    if (!whole && w.b0 == 0 && tid == 0) paged_write_join(w, share.total, cta, share.n_share, scratch.joins);
    float* slot = scratch.parts + paged_slot_floats(RT, d) * (2 * cta + (w.b0 == 0));
    if (!whole && tid < RT) {
      slot[tid] = stat[tid];
      slot[RT + tid] = stat[RT + tid];
    }
#pragma unroll
    for (int i = 0; i < RP; ++i) {
      const int rr = RP * rg + i, row = row0 + rr;
      if (row >= n_rows) continue;
      const float lr = stat[RT + rr], inv = whole ? (lr == 0.f ? 0.f : 1.f / lr) : 1.f;      // a NaN sum stays one
      const long long at = (long long)(w.q.t0 + row / G) * (G * rows.Hkv) + w.h * G + row % G;
      float* dst = whole ? o + at * d : slot + 2 * RT + rr * d;
      if (4 * cg < d)
        *reinterpret_cast<float4*>(dst + 4 * cg) = make_float4(acc[i][0] * inv, acc[i][1] * inv, acc[i][2] * inv, acc[i][3] * inv);
      if (whole && lse2 && cg == 0) lse2[at] = lr == 0.f ? INFINITY : stat[rr] + log2f(lr);
    }
  }
}

// weight[key] += sum over rows of 2^(score - lse): a CTA owns 64 keys of a (request, kv head) and goes over the
// rows in tiles of 64, every key summed in one order.
constexpr int kWRows = 64, kWThreads = 256;

__global__ void __launch_bounds__(kWThreads)
paged_weights_fma_kernel(const PagedRows rows, const PagedPools pools, const PagedBatch batch, const Tile<64>::Cost cost,
                         const float* __restrict__ lse2, float* __restrict__ weights) {
  extern __shared__ __align__(16) float sm[];
  __shared__ int pages[kKB / 8];
  constexpr int SR = 4;
  const int d = pools.d, ld = d + 4, tid = threadIdx.x, G = rows.G;
  float* Ks = sm;                          // [kKB][ld]
  float* Qs = Ks + kKB * ld;               // [2][kWRows][ld]
  float* part = Qs + 2 * kWRows * ld;      // [16][kKB]
  const int ps = 1 << batch.page_log2, ty = tid / 16, tx = tid % 16;
  const int k0 = blockIdx.x * kKB, h = blockIdx.y;
  const float* qb = static_cast<const float*>(rows.q);
  for (int r = blockIdx.z; r < batch.R; r += gridDim.z) {
    const PagedReq q = paged_request(batch, r);
    if (!cost.takes(q) || k0 >= q.len) continue;
    const int n_rows = q.n * G;
    // first row tile that sees the block
    const int first = cost.causal ? max(k0 - (q.len - q.n), 0) * G / kWRows * kWRows : 0;
    auto fetch = [&](int row0) {
      if (row0 < n_rows)
        copy_rows<kWThreads>(Qs + (row0 / kWRows & 1) * kWRows * ld, ld, kWRows, d, qb, [&](int i) -> const float* {
          const int row = row0 + i;
          return row < n_rows ? qb + (q.t0 + row / G) * rows.q_token + (h * G + row % G) * rows.q_head : nullptr;
        });
      cp_async_commit();
    };
    __syncthreads();
    if (tid < kKB / 8) pages[tid] = k0 + tid * 8 < q.len ? paged_page(batch, r, (k0 + tid * 8) >> batch.page_log2) : -1;
    __syncthreads();
    copy_rows<kWThreads>(Ks, ld, kKB, d, pools.k, [&](int i) -> const float* {
      const int j = k0 + i;
      if (j >= q.len) return nullptr;
      return static_cast<const float*>(pools.k) + pages[i >> 3] * pools.k_page_stride + (long long)(h * ps + (j & (ps - 1))) * d;
    });
    fetch(first);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int row0 = first; row0 < n_rows; row0 += kWRows) {
      cp_async_wait_all();
      __syncthreads();
      fetch(row0 + kWRows);
      float s[SR][4];
      scores<SR, 16, 4>(Qs + (row0 / kWRows & 1) * kWRows * ld, Ks, ld, d, ty, tx, s);
#pragma unroll
      for (int i = 0; i < SR; ++i) {
        const int row = row0 + SR * ty + i, lim = last_slot(q, row, G, cost.causal);
        if (lim < 0) continue;
        const float z = lse2[(long long)(q.t0 + row / G) * (G * rows.Hkv) + h * G + row % G];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k0 + tx + 16 * k <= lim) sum[k] += ex2_approx(fmaf(s[i][k], rows.scale_log2e, -z));
      }
    }
    cp_async_wait_all();
#pragma unroll
    for (int k = 0; k < 4; ++k) part[ty * kKB + tx + 16 * k] = sum[k];
    __syncthreads();
    if (tid < kKB && k0 + tid < q.len) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += part[i * kKB + tid];
      const int j = k0 + tid, page = pages[tid >> 3];
      weights[((long long)page * rows.Hkv + h) * ps + (j & (ps - 1))] += s;
    }
  }
}

template <int RT, int CG>
int launch(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, const typename Tile<RT>::Cost& cost, float* o,
           float* lse2, float* kept_scores, const PagedScratch& ws, cudaStream_t st) {
  const int smem = Tile<RT>::smem_bytes(pools.d);
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(paged_fma_kernel<RT, CG>), Tile<RT>::smem_bytes(CG * 4), done)) return CB2_LAUNCH_FAIL;
  paged_fma_kernel<RT, CG><<<Tile<RT>::ctas(pools.d), Tile<RT>::kThreads, smem, st>>>(rows, pools, batch, cost, o, lse2, kept_scores, ws);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

template <int RT>
int run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few, float* o, float* lse2,
        float* kept_scores, void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st) {
  *n_cta = Tile<RT>::ctas(pools.d);
  *parts = paged_scratch(scratch, *n_cta);
  const typename Tile<RT>::Cost cost{rows.G, rows.Hkv, causal, which, few, 2};
  return pools.d <= 64 ? launch<RT, 16>(rows, pools, batch, cost, o, lse2, kept_scores, *parts, st)
                       : launch<RT, 32>(rows, pools, batch, cost, o, lse2, kept_scores, *parts, st);
}

}  // namespace

size_t paged_fma_scratch_bytes(int rt, int d) {
  return rt == 8    ? paged_scratch_bytes(Tile<8>::ctas(d), 8, d)
         : rt == 16 ? paged_scratch_bytes(Tile<16>::ctas(d), 16, d)
                    : paged_scratch_bytes(Tile<64>::ctas(d), 64, d);
}

int paged_fma_run(int rt, const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few, float* o,
                  float* lse2, float* kept_scores, void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st) {
  return rt == 8    ? run<8>(rows, pools, batch, causal, which, few, o, lse2, kept_scores, scratch, parts, n_cta, st)
         : rt == 16 ? run<16>(rows, pools, batch, causal, which, few, o, lse2, kept_scores, scratch, parts, n_cta, st)
                    : run<64>(rows, pools, batch, causal, which, few, o, lse2, kept_scores, scratch, parts, n_cta, st);
}

int paged_weights_fma_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few,
                          const float* lse2, float* weights, cudaStream_t st) {
  const int ld = pools.d + 4, smem = (kKB * ld + 2 * kWRows * ld + 16 * kKB) * 4;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(paged_weights_fma_kernel), (kKB * 132 + 2 * kWRows * 132 + 16 * kKB) * 4, done))
    return CB2_LAUNCH_FAIL;
  const Tile<64>::Cost cost{rows.G, rows.Hkv, causal, which, few, 1};
  const dim3 grid((batch.max_k + kKB - 1) / kKB, rows.Hkv, batch.R < 256 ? batch.R : 256);
  paged_weights_fma_kernel<<<grid, kWThreads, smem, st>>>(rows, pools, batch, cost, lse2, weights);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

}  // namespace cb2

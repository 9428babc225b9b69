// Attention over a paged key/value cache for requests with at most 16 packed rows (single tokens, a few
// speculated ones), bf16: bound by the one pass over K and V.
//
// Keys are the long side of both products, so they take the M side of m16n8k16: S^T[16 keys, 8 rows] = K Q^T
// and O^T[16 columns, 8 rows] += V^T P^T; a group of four to eight query heads fills the N side, where the
// other orientation would leave half of the rows empty.  K comes by ldmatrix, V^T by its transposing form, and P
// turns from accumulator into operand by one 8x8 register transpose a half.  A probability is split into two
// bf16 halves, p = hi + lo up to 2^-16 of it, and V^T multiplied by both, since one half alone would lose more than the
// rounding of o (error against 64 bits 2.1e-3 in place of 1.7e-3; 32 single tokens on up to 16384 keys: 197 us a call
// with one half, 199 with two).  hi is p cut off, and lo at least 2^-24 of p, so that neither half of a positive p is
// zero or negative: an infinite value that a row sees comes out as it is.  The pace is set by memory: per 16 keys of
// d = 128 a warp issues about 115 instructions for 8 KB.
//
// Warps are independent: each streams every fourth 16-key tile of the CTA's piece through its own ring of
// asynchronous copies (two CTAs of four warps per SM keep 128 KB in flight) and keeps its own (m, l, O); they
// meet once per piece, in shared memory.  m follows the maximum lazily (by 2^8), decided by one vote per tile.
//
// Measured: 32 single tokens on 2048 .. 16384 keys, 32 heads on 8, d 128: 199 us, 6.2 TB/s, 95 % of the copy rate.  One
// stream of 65536 keys: 49 us, 5.5 TB/s; the rest is its CTAs' start and the join of 37 carriers a head.
#include "om_paged.cuh"

namespace cb2 {
namespace {

constexpr int kRT = 16, kKB = 64, kTileKeys = 16;
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kCtas = 2 * kNumSMs;

using Cost = PagedCost<kRT, kKB, 1>;

template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// KS = 16-column steps that hold d (4 or 8), NB = groups of 8 packed rows (1 or 2).
template <int KS>
struct Ring {
  static constexpr int kRow = KS * 32;                       // bytes of one key in shared memory
  static constexpr int kHalf = kTileKeys * kRow;             // K tile; the V tile follows
  static constexpr int kStages = KS == 8 ? 3 : 6;            // 24 KB a warp either way
  static constexpr int kWarpBytes = kStages * 2 * kHalf;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kLdO = KS * 16 + 4;                   // pitch of the merged rows (floats)
};

template <int KS, int NB>
__global__ void __launch_bounds__(kThreads, 2)
paged_few_kernel(const PagedRows rows, const PagedPools pools, const PagedBatch batch, const Cost cost, __nv_bfloat16* __restrict__ o,
                 float* __restrict__ lse2, float* __restrict__ scores, const PagedScratch scratch) {
  using R = Ring<KS>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ PagedFindSmem find;
  __shared__ float sh_m[kWarps][kRT], sh_l[kWarps][kRT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, n_cta = gridDim.x, d = pools.d, G = rows.G;
  let_next();
  const PagedShare share = paged_find_share<kThreads>(batch, cost, cta, n_cta, &find);
  if (tid == 0) scratch.joins[cta].r = -1;
  unsigned char* ring = smem + warp * R::kWarpBytes;
  const uint32_t ring_addr = smem_u32(ring);
  const int ps_log2 = batch.page_log2, ps = 1 << ps_log2;
  const int ksteps = (d + 15) >> 4;
  constexpr int kChunks = KS * 2, kRowsPerCopy = 32 / kChunks, kCopies = kTileKeys / kRowsPerCopy;
  const int cp_chunk = lane % kChunks, cp_row = lane / kChunks;
  const bool cp_col = cp_chunk * 8 < d;
  constexpr float kLazy = 8.f, kLeast = 0x1p-24f;

  for (PagedWalk<Cost> w(batch, cost, share); w.valid(); w.next()) {
    w.clip();
    const int n_rows = w.q.n * G, len = w.q.len;
    const int key0 = w.b0 * kKB + warp * kTileKeys, key_end = min(w.b1 * kKB, len);
    const int n_tiles = key_end > key0 ? (key_end - key0 + kWarps * kTileKeys - 1) / (kWarps * kTileKeys) : 0;

    // Q^T as the N-side operand: row g of a group, columns 2t, 2t+1 and 2t+8, 2t+9 of each step
    uint32_t qf[NB][KS][2];
    const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(rows.q);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int row = b * 8 + g;
      const bool there = row < n_rows;
      const __nv_bfloat16* src = qb + (w.q.t0 + (there ? row / G : 0)) * rows.q_token + (w.h * G + (there ? row % G : 0)) * rows.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = ks * 16 + e * 8 + t * 2;
          qf[b][ks][e] = there && col < d ? *reinterpret_cast<const uint32_t*>(src + col) : 0u;
        }
    }
    // last slot that rows 2t, 2t+1 of a group see, and the least of all rows
    int lim[NB][2];
    const int base = len - w.q.n;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = b * 8 + 2 * t + e;
        lim[b][e] = row >= n_rows ? -1 : (cost.causal ? min(base + row / G, len - 1) : len - 1);
      }
    const int first_last = cost.causal ? min(base, len - 1) : len - 1;

    const long long head = (long long)w.h * ps * d;
    const __nv_bfloat16* kp = static_cast<const __nv_bfloat16*>(pools.k) + head;
    const __nv_bfloat16* vp = static_cast<const __nv_bfloat16*>(pools.v) + head;
    // pages of the two halves of a tile (pages hold 8 keys or more), looked up one tile ahead
    int page_a = 0, page_b = 0;
    auto look_up = [&](int i) {
      const int k0 = key0 + i * kWarps * kTileKeys;
      if (i < n_tiles) {
        page_a = paged_page(batch, w.r, k0 >> ps_log2);
        page_b = k0 + 8 < len && ps_log2 == 3 ? paged_page(batch, w.r, (k0 + 8) >> ps_log2) : page_a;
      }
    };
    auto issue = [&](int i) {
      if (i < n_tiles) {
        const int k0 = key0 + i * kWarps * kTileKeys;
        const uint32_t dst = ring_addr + (i % R::kStages) * (2 * R::kHalf);
        const long long ka = page_a * pools.k_page_stride, kb = page_b * pools.k_page_stride;
        const long long va = page_a * pools.v_page_stride, vb = page_b * pools.v_page_stride;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          const int row = c * kRowsPerCopy + cp_row, j = k0 + row;
          const bool there = j < len && cp_col;
          const int at = there ? (j & (ps - 1)) * d + cp_chunk * 8 : 0;
          const uint32_t to = dst + row * R::kRow + ((cp_chunk ^ (row & 7)) << 4);
          cp_async16_or_zero(to, kp + (c < kCopies / 2 ? ka : kb) + at, there);
          cp_async16_or_zero(to + R::kHalf, vp + (c < kCopies / 2 ? va : vb) + at, there);
        }
      }
      cp_async_commit();
      look_up(i + 1);
    };

    float m[NB][2], l[NB][2], acc[KS][NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b][0] = m[b][1] = -INFINITY;
      l[b][0] = l[b][1] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[ks][b][e] = 0.f;
    }
    look_up(0);
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) issue(i);
    for (int i = 0; i < n_tiles; ++i) {
      cp_async_wait_group<R::kStages - 2>();
      __syncwarp();
      issue(i + R::kStages - 1);
      const uint32_t k_tile = ring_addr + (i % R::kStages) * (2 * R::kHalf), v_tile = k_tile + R::kHalf;
      const int k0 = key0 + i * kWarps * kTileKeys;
      float s[NB][4];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[b][e] = 0.f;
      {
        const int row = (lane & 7) + ((lane >> 3) & 1) * 8, half = lane >> 4;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (ks < ksteps) {
            uint32_t a[4];
            ldsm4(k_tile + row * R::kRow + (((2 * ks + half) ^ (row & 7)) << 4), a);
#pragma unroll
            for (int b = 0; b < NB; ++b) mma16816(s[b], a, qf[b][ks]);
          }
        }
      }
      // scaled scores in log2 units; element e: key g + 8 (e / 2), row 2t + e % 2
      const bool cut = k0 + kTileKeys - 1 > first_last;
      bool grow = false;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[b][e] *= rows.scale_log2e;
          if (cut && k0 + g + 8 * (e >> 1) > lim[b][e & 1]) s[b][e] = -INFINITY;
          grow |= s[b][e] > m[b][e & 1] + kLazy;
        }
      if (scores) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = b * 8 + 2 * t + (e & 1), j = k0 + g + 8 * (e >> 1);
            if (row < n_rows && j < len)
              scores[(((long long)w.r * rows.Hkv + w.h) * cost.few + row) * paged_score_stride(batch.max_k) + j] = s[b][e];
          }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[b][e], s[b][e + 2]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float m_new = fmaxf(m[b][e], mx);
            const float alpha = m_new == -INFINITY ? 1.f : ex2_approx(m[b][e] - m_new);
            m[b][e] = m_new;
            l[b][e] *= alpha;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              acc[ks][b][e] *= alpha;
              acc[ks][b][e + 2] *= alpha;
            }
          }
      }
      uint32_t pf[NB][2], pl[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ref = m[b][e & 1] == -INFINITY ? 0.f : m[b][e & 1];
          p[e] = ex2_approx(s[b][e] - ref);
          l[b][e & 1] += p[e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p0 = p[2 * e], p1 = p[2 * e + 1];
          const uint32_t hi = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
          pf[b][e] = transpose8x8(hi);
          pl[b][e] = transpose8x8(pack_bf16x2(fmaxf(p0 - bf16lo_to_f32(hi), p0 * kLeast), fmaxf(p1 - bf16hi_to_f32(hi), p1 * kLeast)));
        }
      }
      {
        const int row = (lane & 7) + (lane >> 4) * 8, half = (lane >> 3) & 1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (ks < ksteps) {
            uint32_t a[4];
            ldsm4_t(v_tile + row * R::kRow + (((2 * ks + half) ^ (row & 7)) << 4), a);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              mma16816(acc[ks][b], a, pf[b]);
              mma16816(acc[ks][b], a, pl[b]);
            }
          }
        }
      }
    }
    cp_async_wait_all();
    __syncwarp();

    // the four warps' carriers meet
    float* part = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float ls = l[b][e];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
        const int row = b * 8 + 2 * t + e;
        if (g == 0) {
          sh_m[warp][row] = m[b][e];
          sh_l[warp][row] = ls;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          part[row * R::kLdO + ks * 16 + g] = acc[ks][b][e];
          part[row * R::kLdO + ks * 16 + g + 8] = acc[ks][b][e + 2];
        }
      }
    __syncthreads();
    const bool whole = w.b0 == 0 && w.b1 == w.nb;
    if (!whole && w.b0 == 0 && tid == 0) paged_write_join(w, share.total, cta, share.n_share, scratch.joins);
    float* slot = scratch.parts + paged_slot_floats(kRT, d) * (2 * cta + (w.b0 == 0));
    for (int row = 0; row < n_rows; ++row) {
      float mm = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) mm = fmaxf(mm, sh_m[x][row]);
      const float ref = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, a = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float f = ex2_approx(sh_m[x][row] - ref);
        ll += sh_l[x][row] * f;
        if (tid < d) a += reinterpret_cast<const float*>(smem + x * R::kWarpBytes)[row * R::kLdO + tid] * f;
      }
      if (whole) {
        const long long at = (long long)(w.q.t0 + row / G) * (G * rows.Hkv) + w.h * G + row % G;
        if (tid < d) o[at * d + tid] = __float2bfloat16_rn(ll == 0.f ? 0.f : a / ll)      /* a NaN sum stays one */;
        if (lse2 && tid == 0) lse2[at] = ll == 0.f ? INFINITY : mm + log2f(ll);
      } else {
        if (tid < d) slot[2 * kRT + row * d + tid] = a;
        if (tid == 0) {
          slot[row] = mm;
          slot[kRT + row] = ll;
        }
      }
    }
    __syncthreads();
  }
}

// weight[key] += sum over the packed rows of 2^(score - lse), from the scores that the kernel above left: a
// thread four neighbouring keys (they lie in one page), the same line cut into more shares, so that all loads are in
// flight at once.
constexpr int kWeightThreads = 256, kWeightCtas = 4 * kNumSMs;

__global__ void __launch_bounds__(kWeightThreads)
paged_few_weights_kernel(const PagedBatch batch, const Cost cost, const float* scores, const float* lse2, float* weights) {
  __shared__ PagedFindSmem find;
  __shared__ float sh_lse[kRT];
  const PagedShare share = paged_find_share<kWeightThreads>(batch, cost, blockIdx.x, gridDim.x, &find);
  const int G = cost.G, ps = 1 << batch.page_log2, tid = threadIdx.x;
  const long long stride = paged_score_stride(batch.max_k);
  let_next();
  after_previous();          // (the share comes from index tensors alone)
  for (PagedWalk<Cost> w(batch, cost, share); w.valid(); w.next()) {
    w.clip();
    const float* sc = scores + ((long long)w.r * cost.Hkv + w.h) * cost.few * stride;
    const int n_rows = w.q.n * G, end = min(w.b1 * kKB, w.q.len);
    __syncthreads();
    if (tid < n_rows) sh_lse[tid] = lse2[(long long)(w.q.t0 + tid / G) * (G * cost.Hkv) + w.h * G + tid % G];
    __syncthreads();
    for (int j = w.b0 * kKB + 4 * tid; j < end; j += 4 * kWeightThreads) {
      const int page = paged_page(batch, w.r, j >> batch.page_log2);
      float* at = weights + ((long long)page * cost.Hkv + w.h) * ps + (j & (ps - 1));
      const float4 was = *reinterpret_cast<const float4*>(at);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int row = 0; row < n_rows; ++row) {
        const float4 x = *reinterpret_cast<const float4*>(sc + row * stride + j);
        const float z = sh_lse[row];
        sum[0] += ex2_approx(x.x - z);
        sum[1] += ex2_approx(x.y - z);
        sum[2] += ex2_approx(x.z - z);
        sum[3] += ex2_approx(x.w - z);
      }
      if (j + 4 <= end) {
        *reinterpret_cast<float4*>(at) = make_float4(was.x + sum[0], was.y + sum[1], was.z + sum[2], was.w + sum[3]);
      } else {               // slots behind the length, and scores there, are nobody's
        at[0] = was.x + sum[0];
        if (j + 1 < end) at[1] = was.y + sum[1];
        if (j + 2 < end) at[2] = was.z + sum[2];
      }
    }
  }
}

template <int KS, int NB>
int launch(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, const Cost& cost, __nv_bfloat16* o, float* lse2,
           float* scores, const PagedScratch& ws, cudaStream_t st) {
  constexpr int smem = Ring<KS>::kSmem;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(paged_few_kernel<KS, NB>), smem, done)) return CB2_LAUNCH_FAIL;
  paged_few_kernel<KS, NB><<<kCtas, kThreads, smem, st>>>(rows, pools, batch, cost, o, lse2, scores, ws);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

}  // namespace

size_t paged_few_scratch_bytes(int d) { return paged_scratch_bytes(kCtas, kRT, d); }

int paged_few_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int few, void* o, float* lse2,
                  float* scores, void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st) {
  *parts = paged_scratch(scratch, kCtas);
  *n_cta = kCtas;
  // 256 keys a share at least: four tiles a warp, less than that is mostly start and join
  const Cost cost{rows.G, rows.Hkv, causal, kPagedFew, few, 4};
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(o);
  if (pools.d <= 64)
    return few <= 8 ? launch<4, 1>(rows, pools, batch, cost, out, lse2, scores, *parts, st)
                    : launch<4, 2>(rows, pools, batch, cost, out, lse2, scores, *parts, st);
  return few <= 8 ? launch<8, 1>(rows, pools, batch, cost, out, lse2, scores, *parts, st)
                  : launch<8, 2>(rows, pools, batch, cost, out, lse2, scores, *parts, st);
}

int paged_few_weights_run(const PagedRows& rows, const PagedBatch& batch, int causal, int few, const float* scores, const float* lse2,
                          float* weights, cudaStream_t st) {
  const Cost cost{rows.G, rows.Hkv, causal, kPagedFew, few, 2};
  return launch_next(paged_few_weights_kernel, dim3(kWeightCtas), kWeightThreads, st, batch, cost, scores, lse2, weights);
}

}  // namespace cb2

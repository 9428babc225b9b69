// Attention weight of cached keys on the tensor cores (bf16): weight[key] += sum over the packed rows that see it
// of 2^(scale q.k - lse), after the attention kernels have left lse (log2 units) in scratch.
//
// The scores are taken a second time, turned over: S^T = K Q^T with 128 keys on the M side, so that a thread owns
// a key (TMEM lane) and sums its probabilities over the columns without meeting another thread; the scores
// themselves, 4 bytes for every pair, never leave the chip.  One product and one exponential a pair: half of what
// the attention costs.  Unit of the work line = (request, kv head, 128-key block), cost = the 64-row tiles that
// see it; a unit cut between shares leaves 128 partial sums a share, added in share order.
//
// Roles: warp 0 = the key block (pages by TMA), warp 1 = MMA issue and TMEM owner, warps 2..5 = sums, warps 6, 7 = rows
// of a tile (16-byte asynchronous copies), their -lse and the last slot each sees.  A ring of three stages holds
// row tile, -lse and S together; two CTAs share an SM.  Every wait is bounded.
#include "om_paged.cuh"
#include "umma.cuh"

namespace cb2 {
int paged_pool_map(CUtensorMap* out, const void* base, int d, int page_size, int Hkv, int n_pages, long long page_stride);   // om_paged_tc.cu

namespace {

constexpr int kKeys = 128, kRows = 64, kStages = 3;
constexpr int kThreads = 256;
constexpr int kCtas = 2 * kNumSMs;
constexpr uint32_t kSub = 64 * 128;                       // 64 rows x 64 columns of a row tile
constexpr uint32_t kRowTile = 2 * kSub;
constexpr uint32_t kOffK = 0, kOffQ = umma::kTileBytes;
constexpr uint32_t kOffBars = kOffQ + kStages * kRowTile;
constexpr int kNumBars = 3 * kStages + 2;
constexpr uint32_t kTmemCols = 256;

// The line of key blocks: block i of a request is seen by its rows from token i * 128 - base on.
struct KeyCost {
  static constexpr int kOv = 2;
  int G, Hkv, causal, which, few, min_blocks;
  __device__ __forceinline__ bool takes(const PagedReq& q) const {
    if (q.n == 0 || q.len == 0) return false;
    return which == kPagedAll || (which == kPagedFew) == (q.n * G <= few);
  }
  __device__ __forceinline__ int row_tiles(const PagedReq& q) const { return (q.n * G + kRows - 1) / kRows; }
  __device__ __forceinline__ int first_row_tile(const PagedReq& q, int i) const {
    return causal ? int(unsigned(max(i * kKeys - (q.len - q.n), 0)) * G / kRows) : 0;
  }
  __device__ __forceinline__ int tiles(const PagedReq& q) const { return (q.len + kKeys - 1) / kKeys; }
  __device__ __forceinline__ int blocks(const PagedReq& q, int i) const { return row_tiles(q) - first_row_tile(q, i); }
  __device__ __forceinline__ long long before(const PagedReq& q, int k) const {
    long long s = (long long)k * (row_tiles(q) + kOv);
    const int base = q.len - q.n, i1 = base < 0 ? 0 : base / kKeys + 1;       // first block that not all rows see
    if (causal && k > i1) s -= stair_sum(k - i1, kRows, unsigned(kKeys) * G, unsigned(i1 * kKeys - base) * G);
    return s;
  }
  __device__ __forceinline__ long long of_request(const PagedReq& q) const { return takes(q) ? before(q, tiles(q)) * Hkv : 0; }
};

struct Piece {
  int r, h, k0, t0, n, len, tile0, tiles, whole, first;     // row tiles [tile0, tile0 + tiles)
};

constexpr int kBatch = 16;

struct Smem {
  uint32_t tmem;
  int abort, count, loads_k, n_share;
  long long total;
  PagedWalkState walk;
  Piece pieces[kBatch];
  PagedFindSmem find;
  float neg_lse[kStages][kRows];
  int last[kStages][kRows];
  long long row_at[2][32];
};
constexpr uint32_t kOffMisc = (kOffBars + kNumBars * 8 + 15) & ~15u;
constexpr uint32_t kSmemBytes = kOffMisc + uint32_t(sizeof(Smem)) + 1024;
static_assert(2 * kSmemBytes <= 226 * 1024, "two CTAs per SM");

__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int ks) {
  return umma::smem_desc(tile + (ks >> 2) * kSub + (ks & 3) * 32u, 16u, 1024u);
}

__global__ void __launch_bounds__(kThreads, 2)
paged_weights_tc_kernel(const __grid_constant__ CUtensorMap map_k, const PagedRows rows, const int d, const PagedBatch batch,
                        const KeyCost cost, const float* __restrict__ lse2, float* __restrict__ weights, PagedJoin* __restrict__ joins,
                        float* __restrict__ parts) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint64_t *q_full = bars, *s_ready = bars + kStages, *s_empty = bars + 2 * kStages, *k_full = bars + 3 * kStages, *k_empty = k_full + 1;
  Smem* sh = reinterpret_cast<Smem*>(smem + kOffMisc);
  volatile int* s_abort = &sh->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, n_cta = gridDim.x;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&q_full[i], 64);
      mbar_init(&s_ready[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    sh->abort = sh->loads_k = 0;
    joins[cta].r = -1;
    mbar_fence_init();
  }
  if (warp == 1) {
    __syncwarp();
    umma::tmem_alloc(&sh->tmem, kTmemCols);
  }
  {
    const PagedShare share = paged_find_share<kThreads>(batch, cost, cta, n_cta, &sh->find);
    if (warp == 0) {
      const PagedWalk<KeyCost> walk(batch, cost, share);
      if (lane == 0) {
        sh->walk = walk;
        sh->total = share.total;
        sh->n_share = share.n_share;
      }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = sh->tmem;
  const uint32_t k_addr = smem_u32(smem + kOffK), q_addr = smem_u32(smem + kOffQ);
  const int halves = (d + 63) >> 6, G = rows.G, ps_log2 = batch.page_log2, ps = 1 << ps_log2;
  uint32_t n_tile = 0, n_piece = 0;
  auto stage_of = [](uint32_t n) { return n % kStages; };
  auto phase_of = [](uint32_t n) { return (n / kStages) & 1u; };

  for (;;) {
    if (warp == 0) {
      PagedWalk<KeyCost> walk(batch, cost, sh->walk);
      __syncwarp();
      int count = 0;
      for (; count < kBatch && walk.valid(); ++count, walk.next()) {
        walk.clip();
        if (lane == 0) {
          const bool whole = walk.b0 == 0 && walk.b1 == walk.nb;
          sh->pieces[count] = Piece{walk.r, walk.h, walk.tile * kKeys, walk.q.t0, walk.q.n, walk.q.len,
                                    cost.first_row_tile(walk.q, walk.tile) + walk.b0, walk.b1 - walk.b0, whole, walk.b0 == 0};
          if (walk.b0 == 0 && !whole) paged_write_join(walk, sh->total, cta, sh->n_share, joins);
        }
      }
      if (lane == 0) {
        sh->count = count;
        sh->walk = walk;
      }
    }
    __syncthreads();
    const int count = sh->count;

    if (warp == 0) {
      const int box_log2 = min(ps_log2, 6), boxes = kKeys >> box_log2;
      for (int p = 0; p < count; ++p, ++n_piece) {
        const Piece pc = sh->pieces[p];
        const int k0 = pc.k0 + (lane << box_log2);
        const bool mine = lane < boxes && k0 < pc.len;
        const int page = mine ? paged_page(batch, pc.r, k0 >> ps_log2) : 0;
        const unsigned have = __ballot_sync(0xffffffffu, mine);
        const uint32_t box_bytes = 128u << box_log2;
        const bool ok = n_piece == 0 || mbar_wait_abortable(k_empty, (n_piece - 1) & 1, s_abort, kDefaultWaitNs, __LINE__);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(k_full, __popc(have) * halves * box_bytes);
          ++sh->loads_k;
        }
        __syncwarp();
        if (mine)
          for (int hf = 0; hf < halves; ++hf)
            umma::tma_load_4d(smem + kOffK + hf * umma::kSubTileBytes + lane * box_bytes, &map_k, hf * 64, ps_log2 > 6 ? k0 & (ps - 1) : 0,
                           pc.h, page, k_full);
      }
    } else if (warp == 1) {
      const int ksteps = (d + 15) >> 4;
      constexpr uint32_t idesc = umma::instr_desc_bf16(kKeys, kRows, false, false);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, mbar_wait_abortable(bar, parity, s_abort, kDefaultWaitNs, site));
      };
      for (int p = 0; p < count; ++p, ++n_piece) {
        const int tiles = sh->pieces[p].tiles;
        bool ok = wait(k_full, n_piece & 1, __LINE__);
        for (int i = 0; ok && i < tiles; ++i, ++n_tile) {
          const uint32_t st = stage_of(n_tile);
          ok = wait(&q_full[st], phase_of(n_tile), __LINE__);      // the rows' writers have waited for S to be free
          if (!ok) break;
          umma::fence_after_sync();
          if (lane == 0) {
            const uint32_t tile = q_addr + st * kRowTile;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              if (ks < ksteps)
                umma::mma_bf16(tmem + st * kRows, umma::desc_kmajor(k_addr, ks), desc_rows(tile, ks), idesc, ks > 0);
            umma::mma_commit(&s_ready[st]);
            if (i == tiles - 1) umma::mma_commit(k_empty);
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    } else if (warp < 6) {
      const int q4 = warp & 3, key = q4 * 32 + lane;
      const uint32_t lane_base = tmem + (uint32_t(q4 * 32) << 16);
      const uint64_t scale2 = umma::f2_pack(rows.scale_log2e, rows.scale_log2e);
      for (int p = 0; p < count; ++p) {
        const Piece* pc = &sh->pieces[p];
        const int tiles = pc->tiles, j = pc->k0 + key, base = pc->len - pc->n;
        float sum = 0.f;
        bool ok = true;
        for (int i = 0; i < tiles; ++i, ++n_tile) {
          const uint32_t st = stage_of(n_tile);
          // (the second wait, long over, makes the row warps' -lse and last slots visible)
          ok = mbar_wait_abortable(&s_ready[st], phase_of(n_tile), s_abort, kDefaultWaitNs, __LINE__) &&
               mbar_wait_abortable(&q_full[st], phase_of(n_tile), s_abort, kDefaultWaitNs, __LINE__);
          if (!__all_sync(0xffffffffu, ok)) break;
          umma::fence_after_sync();
          uint32_t sv[2][32];
#pragma unroll
          for (int cb = 0; cb < 2; ++cb) umma::tmem_ld32(lane_base + st * kRows + cb * 32, sv[cb]);
          umma::tmem_wait_ld();
          umma::tmem_loaded(sv[0]);
          umma::tmem_loaded(sv[1]);
          // rows that do not see the whole key block: hidden per element
          if (cost.causal && base + (pc->tile0 + i) * kRows / G < pc->k0 + kKeys - 1) {
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (sh->last[st][cb * 32 + c] < j) sv[cb][c] = 0xff800000u;
          }
          uint64_t s2[2] = {0ull, 0ull};
#pragma unroll
          for (int cb = 0; cb < 2; ++cb)
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 z = *reinterpret_cast<const float4*>(&sh->neg_lse[st][cb * 32 + c]);
              float x0, x1, x2, x3;
              umma::f2_unpack(umma::f2_fma(umma::f2_pack(__uint_as_float(sv[cb][c]), __uint_as_float(sv[cb][c + 1])), scale2,
                                           umma::f2_pack(z.x, z.y)), x0, x1);
              umma::f2_unpack(umma::f2_fma(umma::f2_pack(__uint_as_float(sv[cb][c + 2]), __uint_as_float(sv[cb][c + 3])), scale2,
                                           umma::f2_pack(z.z, z.w)), x2, x3);
              s2[0] = umma::f2_add(s2[0], umma::f2_pack(ex2_approx(x0), ex2_approx(x1)));
              s2[1] = umma::f2_add(s2[1], umma::f2_pack(ex2_approx(x2), ex2_approx(x3)));
            }
          float a, b;
          umma::f2_unpack(umma::f2_add(s2[0], s2[1]), a, b);
          sum += a + b;
          umma::fence_before_sync();
          mbar_arrive(&s_empty[st]);
        }
        if (!__all_sync(0xffffffffu, ok)) break;
        if (!pc->whole) {
          parts[(2 * cta + pc->first) * kKeys + key] = sum;
        } else if (j < pc->len) {
          const int page = paged_page(batch, pc->r, j >> ps_log2);
          weights[((long long)page * rows.Hkv + pc->h) * ps + (j & (ps - 1))] += sum;
        }
      }
    } else {
      // rows of the tiles, 32 a warp: a lane works out one row's place, then 8 or 16 neighbouring lanes copy its chunks
      const int lw = warp - 6, lt = lw * 32 + lane;
      const int chunks = halves * 8, c = lane & (chunks - 1), sub = lane / chunks, step = 32 / chunks;
      const uint32_t dst = q_addr + lw * 32 * 128u + (c >> 3) * kSub;
      const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(rows.q);
      uint32_t issued = n_tile;          // tiles whose copies have been issued; n_tile: handed to the MMA warp
      for (int p = 0; p < count; ++p) {
        const Piece pc = sh->pieces[p];
        bool ok = true;
        for (int i = 0; i < pc.tiles; ++i, ++issued) {
          const uint32_t st = stage_of(issued);
          if (issued >= kStages) ok = mbar_wait_abortable(&s_empty[st], phase_of(issued - kStages), s_abort, kDefaultWaitNs, __LINE__);
          if (!__all_sync(0xffffffffu, ok)) break;
          const int row = (pc.tile0 + i) * kRows + lt;
          const bool there = row < pc.n * G;
          const int tok = there ? row / G : 0, g = there ? row - tok * G : 0;
          const float z = there ? __ldg(lse2 + (long long)(pc.t0 + tok) * (G * rows.Hkv) + pc.h * G + g) : INFINITY;
          sh->neg_lse[st][lt] = -z;
          sh->last[st][lt] = cost.causal ? min(pc.len - pc.n + tok, pc.len - 1) : pc.len - 1;
          sh->row_at[lw][lane] = there ? (pc.t0 + tok) * rows.q_token + (pc.h * G + g) * rows.q_head : -1;
          __syncwarp();
#pragma unroll 4
          for (int r = sub; r < 32; r += step) {
            const long long at = sh->row_at[lw][r];
            const bool have = at >= 0 && c * 8 < d;
            cp_async16_or_zero(dst + st * kRowTile + r * 128u + (((c & 7) ^ (r & 7)) << 4), qb + (have ? at + c * 8 : 0), have);
          }
          cp_async_commit();
          // the tile before this one has landed
          if (issued > n_tile) {
            cp_async_wait_one();
            fence_proxy_async_smem();
            mbar_arrive(&q_full[stage_of(n_tile)]);
            ++n_tile;
          }
          __syncwarp();            // row_at is read
        }
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      if (issued > n_tile) {
        cp_async_wait_all();
        fence_proxy_async_smem();
        mbar_arrive(&q_full[stage_of(n_tile)]);
        ++n_tile;
      }
    }
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (count < kBatch || *s_abort) break;
  }
  if (*s_abort) {
    if (tid == 0) {
      if (sh->loads_k) mbar_wait_bounded(k_full, (sh->loads_k - 1) & 1);      // a load in flight lands before the memory goes
      if (batch.status) atomicExch(batch.status, CB2_WAIT_TIMEOUT | (*s_abort << 8));
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    umma::tmem_dealloc(tmem, kTmemCols);
  }
}

// Adds up the partial sums of key blocks that were cut between shares, in share order.
__global__ void __launch_bounds__(kKeys)
paged_weights_join_kernel(const PagedBatch batch, int Hkv, const PagedJoin* __restrict__ joins, const float* __restrict__ parts,
                          float* __restrict__ weights) {
  const int c = blockIdx.x, key = threadIdx.x;
  const PagedJoin jn = joins[c];
  if (jn.r < 0) return;
  const int len = min(max(__ldg(batch.lens + jn.r), 0), batch.max_k), j = jn.tile * kKeys + key, ps = 1 << batch.page_log2;
  if (j >= len) return;
  float sum = 0.f;
#pragma unroll 4
  for (int s = c; s <= jn.last; ++s) sum += parts[(2 * s + (s == c)) * kKeys + key];
  const int page = paged_page(batch, jn.r, j >> batch.page_log2);
  weights[((long long)page * Hkv + jn.h) * ps + (j & (ps - 1))] += sum;
}

}  // namespace

size_t paged_weights_tc_scratch_bytes() { return size_t(kCtas) * (sizeof(PagedJoin) + 2 * kKeys * 4); }

int paged_weights_tc_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few,
                         const float* lse2, float* weights, void* scratch, cudaStream_t st) {
  CUtensorMap mk;
  const int rc = paged_pool_map(&mk, pools.k, pools.d, 1 << batch.page_log2, pools.Hkv, batch.n_pages, pools.k_page_stride);
  if (rc != CB2_OK) return rc;
  if (cudaFuncSetAttribute(paged_weights_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes)) != cudaSuccess)
    return CB2_LAUNCH_FAIL;
  const KeyCost cost{rows.G, rows.Hkv, causal, which, few, 4};
  PagedJoin* joins = static_cast<PagedJoin*>(scratch);
  float* parts = reinterpret_cast<float*>(joins + kCtas);
  paged_weights_tc_kernel<<<kCtas, kThreads, kSmemBytes, st>>>(mk, rows, pools.d, batch, cost, lse2, weights, joins, parts);
  CB2_LAUNCH_CHECK();
  paged_weights_join_kernel<<<kCtas, kKeys, 0, st>>>(batch, rows.Hkv, joins, parts, weights);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

}  // namespace cb2

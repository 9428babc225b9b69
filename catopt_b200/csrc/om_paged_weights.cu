// Attention weight of cached keys on the tensor cores (bf16): weight[key] += sum over the packed rows that see it
// of 2^(scale q.k - lse), after the attention kernels have left lse (log2 units) in scratch.
//
// The scores are taken a second time, turned over: S^T = K Q^T with 128 keys on the M side, so that a thread owns
// a key (TMEM lane) and sums its probabilities over the columns without meeting another thread; the scores
// themselves, 4 bytes for every pair, never leave the chip.  One product and one exponential a pair: half of what
// the attention costs.  Unit of the work line = (request, kv head, 128-key block), cost = the 64-row tiles that
// see it; a unit cut between shares leaves 128 partial sums a share, added in share order.
//
// A row tile is T = 64 / G whole tokens of a group (64 heads of one token when G > 64), so that one TMA box of q brings
// it; columns past T G stay zero and count as hidden.  Roles: warp 0 = the key block (pages by TMA), warp 1 = MMA issue and TMEM owner,
// warps 2..5 = sums, warp 6 = row tiles, their -lse and the last slot each row sees (copying the rows by 16-byte
// asynchronous copies took 2.8 k cycles a tile and set the pace).  A ring of four stages holds row tile, -lse and S
// together; two CTAs share an SM.  Every wait is bounded.
//
// Measured: chunks of 1024 and 828 tokens on 4096 and 2727 keys, 32 heads on 8, d 128: 85 us (the attention before it:
// 110 us); the exponential unit is busy about 60 % of the time.  Fetching -lse one tile ahead cost 8 us (the row warp sets the
// pace), a division in every tile of the sums 3 us.  Two threads a key (eight sum warps), scores in two halves: slower.
#include "om_paged.cuh"
#include "umma.cuh"

namespace cb2 {
int paged_pool_map(CUtensorMap* out, const void* base, int d, int page_size, int Hkv, int n_pages, long long page_stride);   // om_paged_tc.cu

namespace {

constexpr int kKeys = 128, kRows = 64, kStages = 4;
constexpr int kThreads = 224;
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
  int T, per_token;         // tokens a row tile, row tiles a token: one of them is 1
  __device__ __forceinline__ bool takes(const PagedReq& q) const {
    if (q.n == 0 || q.len == 0) return false;
    return (which == kPagedFew) == (q.n * G <= few);
  }
  __device__ __forceinline__ int row_tiles(const PagedReq& q) const { return (q.n + T - 1) / T * per_token; }
  __device__ __forceinline__ int first_row_tile(const PagedReq& q, int i) const {
    return causal ? max(i * kKeys - (q.len - q.n), 0) / T * per_token : 0;
  }
  __device__ __forceinline__ int tiles(const PagedReq& q) const { return (q.len + kKeys - 1) / kKeys; }
  __device__ __forceinline__ int blocks(const PagedReq& q, int i) const { return row_tiles(q) - first_row_tile(q, i); }
  __device__ __forceinline__ long long before(const PagedReq& q, int k) const {
    long long s = (long long)k * (row_tiles(q) + kOv);
    const int base = q.len - q.n, i1 = base < 0 ? 0 : base / kKeys + 1;       // first block that not all rows see
    if (causal && k > i1) s -= stair_sum(k - i1, T, kKeys, unsigned(i1 * kKeys - base)) * per_token;
    return s;
  }
  __device__ __forceinline__ long long per_head(const PagedReq& q) const { return takes(q) ? before(q, tiles(q)) : 0; }
};

struct Piece {
  int r, h, k0, t0, n, len, tile0, tiles, whole, first;     // row tiles [tile0, tile0 + tiles)
};

constexpr int kBatch = 16;

struct Smem {
  uint32_t tmem;
  int abort, count, loads_k, loads_q, n_share;
  long long total;
  PagedWalkState walk;
  Piece pieces[kBatch];
  PagedFindSmem find;
  alignas(16) float neg_lse[kStages][kRows];      // read four at a time
  int last[kStages][kRows];
};
constexpr uint32_t kOffMisc = (kOffBars + kNumBars * 8 + 15) & ~15u;
constexpr uint32_t kSmemBytes = kOffMisc + uint32_t(sizeof(Smem)) + 1024;
static_assert(alignof(Smem) == 16 && kOffMisc % 16 == 0, "alignment of neg_lse");
static_assert(2 * kSmemBytes <= 226 * 1024, "two CTAs per SM");

__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int ks) {
  return umma::smem_desc(tile + (ks >> 2) * kSub + (ks & 3) * 32u, 16u, 1024u);
}

__global__ void __launch_bounds__(kThreads, 2)
paged_weights_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, const PagedRows rows, const int d, const PagedBatch batch,
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

  let_next();
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&q_full[i], 33);           // the TMA box and the 32 lanes that write -lse
      mbar_init(&s_ready[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    sh->abort = sh->loads_k = sh->loads_q = 0;
    joins[cta].r = -1;
    mbar_fence_init();
  }
  if (warp == 1) {
    __syncwarp();
    umma::tmem_alloc(&sh->tmem, kTmemCols);
  }
  // columns that no box writes count as rows of zeros
  for (uint32_t e = tid; e < kStages * kRowTile / 16; e += kThreads)
    *reinterpret_cast<uint4*>(smem + kOffQ + e * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
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
      // the whole warp computes the operands (shuffled: uniform), one lane issues
      const bool lead = lane == 0;
      auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
      const int ksteps = int(uniform((d + 15) >> 4));
      const uint32_t s_cols = uniform(tmem), ka = uniform(k_addr), qa = uniform(q_addr);
      constexpr uint32_t idesc = umma::instr_desc_bf16(kKeys, kRows, false, false);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, mbar_wait_abortable(bar, parity, s_abort, kDefaultWaitNs, site));
      };
      for (int p = 0; p < count; ++p, ++n_piece) {
        const int tiles = int(uniform(sh->pieces[p].tiles));
        bool ok = wait(k_full, n_piece & 1, __LINE__);
        for (int i = 0; ok && i < tiles; ++i, ++n_tile) {
          const uint32_t st = uniform(stage_of(n_tile)), tile = qa + st * kRowTile;
          ok = wait(&q_full[st], phase_of(n_tile), __LINE__);      // the rows' writers have waited for S to be free
          if (!ok) break;
          umma::fence_after_sync();
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            if (ks < ksteps)
              umma::mma_bf16_by(lead, s_cols + st * kRows, umma::desc_kmajor(ka, ks), desc_rows(tile, ks), idesc, ks > 0);
          umma::mma_commit_by(lead, &s_ready[st]);
          if (i == tiles - 1) umma::mma_commit_by(lead, k_empty);
        }
        if (!ok) break;
      }
    } else if (warp < 6) {
      const int q4 = warp & 3, key = q4 * 32 + lane;
      const uint32_t lane_base = tmem + (uint32_t(q4 * 32) << 16);
      const uint64_t scale2 = umma::f2_pack(rows.scale_log2e, rows.scale_log2e);
      const int used = G < kRows ? cost.T * G : kRows;        // columns of a tile that are rows
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
          // rows that do not see the whole key block, or are not of this request: hidden per element
          const int tok0 = (cost.per_token == 1 ? pc->tile0 + i : (pc->tile0 + i) / cost.per_token) * cost.T;
          if ((cost.causal && base + tok0 < pc->k0 + kKeys - 1) || tok0 + cost.T > pc->n || cost.per_token > 1) {
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (sh->last[st][cb * 32 + c] < j) sv[cb][c] = 0xff800000u;
          }
          // columns past T G hold rows of zeros, whose product with a key of infinities is NaN: no score either.  (They
          // lie in the second half: 33 columns at least are used.)
          if (used < kRows) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (32 + c >= used) sv[1][c] = 0xff800000u;
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
      // columns lane and lane + 32 of a tile: token and head inside it
      const int hb = min(G, kRows), per = cost.per_token;
      const int tok_of[2] = {lane / hb, (lane + 32) / hb}, g_of[2] = {lane % hb, (lane + 32) % hb};
      // a tile of the list: T tokens from tok0 on (one, if per > 1: heads from g0 on)
      struct Cursor {
        int p, left, tok0, g0;
      };
      auto start = [&](Cursor& c) {
        if (c.p >= count) return;
        const int tile = sh->pieces[c.p].tile0, tb = per == 1 ? tile : tile / per;
        c.left = sh->pieces[c.p].tiles;
        c.tok0 = tb * cost.T;
        c.g0 = (tile - tb * per) * kRows;
      };
      auto advance = [&](Cursor& c) {
        if (--c.left == 0) {
          ++c.p;
          start(c);
        } else if (per == 1 || (c.g0 += kRows) == per * kRows) {
          c.g0 = 0;
          c.tok0 += cost.T;
        }
      };
      struct Columns {
        float z[2];
        int last[2];
      };
      Cursor seen{0, 0, 0, 0};
      auto look_up = [&](Columns& x) {
        if (seen.p >= count) return;
        const Piece* pc = &sh->pieces[seen.p];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = seen.tok0 + tok_of[e], g = seen.g0 + g_of[e];
          const bool there = tok_of[e] < cost.T && tok < pc->n && g < G;
          x.z[e] = there ? __ldg(lse2 + (long long)(pc->t0 + tok) * (G * rows.Hkv) + pc->h * G + g) : INFINITY;
          x.last[e] = there ? (cost.causal ? min(pc->len - pc->n + tok, pc->len - 1) : pc->len - 1) : -1;
        }
        advance(seen);
      };
      Cursor now{0, 0, 0, 0};
      auto step = [&](Columns& x) {
        const uint32_t st = stage_of(n_tile);
        const bool ok = n_tile < kStages || mbar_wait_abortable(&s_empty[st], phase_of(n_tile - kStages), s_abort, kDefaultWaitNs, __LINE__);
        if (!__all_sync(0xffffffffu, ok)) return false;
        if (lane == 0) {
          const Piece* pc = &sh->pieces[now.p];
          mbar_arrive_expect_tx(&q_full[st], halves * hb * cost.T * 128);
          ++sh->loads_q;
          for (int hf = 0; hf < halves; ++hf)
            umma::tma_load_3d(smem + kOffQ + st * kRowTile + hf * kSub, &map_q, hf * 64, pc->h * G + now.g0, pc->t0 + now.tok0, &q_full[st]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sh->neg_lse[st][lane + 32 * e] = -x.z[e];
          sh->last[st][lane + 32 * e] = x.last[e];
        }
        mbar_arrive(&q_full[st]);
        advance(now);
        ++n_tile;
        look_up(x);
        return now.p < count;
      };
      // -lse is fetched two tiles ahead (one warp feeds the tiles: its pace is theirs)
      Columns a, b;
      start(seen);
      start(now);
      look_up(a);
      look_up(b);
      if (count > 0)
        while (step(a) && step(b)) {
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
      // loads in flight land before the shared memory goes (bounded waits, too)
      if (sh->loads_k) mbar_wait_bounded(k_full, (sh->loads_k - 1) & 1);
      for (int n = max(sh->loads_q - kStages, 0); n < sh->loads_q; ++n) mbar_wait_bounded(&q_full[stage_of(n)], phase_of(n));
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
paged_weights_join_kernel(const PagedBatch batch, int Hkv, const PagedJoin* joins, const float* parts, float* weights) {
  const int c = blockIdx.x, key = threadIdx.x;
  after_previous();
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
  CUtensorMap mk, mq;
  int rc = paged_pool_map(&mk, pools.k, pools.d, 1 << batch.page_log2, pools.Hkv, batch.n_pages, pools.k_page_stride);
  // q as {d, Hq, n_tokens}: a box holds T tokens of a group
  const int Hq = rows.G * rows.Hkv, T = rows.G < kRows ? kRows / rows.G : 1;
  const long long head = Hq > 1 ? rows.q_head : pools.d, token = batch.n_tokens > 1 ? rows.q_token : (long long)Hq * pools.d;
  if (rc == CB2_OK) rc = umma::make_map_3d_strided(&mq, rows.q, pools.d, Hq, batch.n_tokens, head, token, 64, rows.G < kRows ? rows.G : kRows, T);
  if (rc != CB2_OK) return rc;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(paged_weights_tc_kernel), kSmemBytes, done)) return CB2_LAUNCH_FAIL;
  const KeyCost cost{rows.G, rows.Hkv, causal, which, few, 4, T, rows.G > kRows ? (rows.G + kRows - 1) / kRows : 1};
  PagedJoin* joins = static_cast<PagedJoin*>(scratch);
  float* parts = reinterpret_cast<float*>(joins + kCtas);
  paged_weights_tc_kernel<<<kCtas, kThreads, kSmemBytes, st>>>(mk, mq, rows, pools.d, batch, cost, lse2, weights, joins, parts);
  CB2_LAUNCH_CHECK();
  return launch_next(paged_weights_join_kernel, dim3(kCtas), kKeys, st, batch, rows.Hkv, static_cast<const PagedJoin*>(joins),
                     static_cast<const float*>(parts), weights);
}

}  // namespace cb2

// Attention over a paged key/value cache on the tensor cores (bf16), for requests with many packed rows
// (chunks of prompts): the work line of om_paged.cuh with tiles of 128 packed rows and 64-key blocks.
//
// Two CTAs share an SM (half of the tensor memory and of the shared memory each); a CTA walks its share of the line:
//   MMA1  S = Q K_j^T -> TMEM, two blocks ahead of the softmax (two S buffers of 64 columns);
//   softmax   P = 2^(S scale - m) as bf16 over S, l and the running m in registers (thread = row = TMEM lane);
//   MMA2  O += P V_j, P read from TMEM.
// With S ready before it is asked for, the softmax warps never wait for the tensor core, which finds the next
// block's P after every product: one exponential per score (16 a clock and SM) and the products (1024 clocks per
// 128 x 128 scores either way) overlap.  The reference point m follows the maximum lazily (when it moved by
// more than 2^8), so O is rarely rescaled, and only then does the softmax wait for the product before.
// P is rounded once, to bf16, as the dense chunks' kernel of this library does (error against 64 bits 2.3e-3, of which the
// rounding of o alone is 1.7e-3).  A second half of it (p = hi + lo, half as many products again) takes two chunks of 2048 on
// 8192 keys from 414 to 518 us a call, chunks of 1024 with weights from 207 to 237, a mixed batch of 24 from 39 to 43.
// Only a block that some row of the tile may not see whole is masked, per element.  Of the last block of a
// request the value rows behind its length are zeroed in shared memory, since 0 x NaN is NaN.
//
// Roles: warps 0 and 6 = loads of K and of V (pages by TMA: one box per page and 64 columns, each lane its own page; one
// warp for both set the pace where a block is many pages: 24 requests on pages of 16, 46 -> 41 us with two), warp 1 = MMA
// issue and TMEM owner, warps 2..5 = softmax and the query rows (16-byte asynchronous copies, since a tile may start
// inside a token's group; a piece's rows are fetched during the last softmax of the piece before).  The
// pieces of a share are listed in shared memory in batches, so that the softmax threads spend no registers on
// the walk.  Every wait is bounded.
//
// Measured: two chunks of 2048 tokens on 8192 keys in all, 32 heads on 8, d 128, with the join, at 1965 MHz: 352..367 us
// replayed in a graph (1.0 PFLOP/s), 414..420 us a call when the inputs change from call to call; a piece costs about four
// blocks' time to start and end, which the line counts.  What bounds a long piece is shared memory: a 64-column product reads
// Q again for every 64 keys (48 KB a block), P V reads 16 KB, the loads write 32 KB; two CTAs move 192 KB in about 1680
// clocks of a long piece, 115 of 128 bytes a clock.  Tried and slower: 128-key blocks with one S buffer (487 us), two row tiles that share key and value blocks in one CTA of an SM (595 us), part of the
// exponentials as polynomials on the FMA pipes (+7 %), eight softmax warps (+7 %).
#include "om_paged.cuh"
#include "umma.cuh"

namespace cb2 {
namespace {

constexpr int kRT = 128, kKB = 64;
constexpr int kThreads = 224;
// Rows in, scores of the first blocks, results out: as long as four blocks.
using Cost = PagedCost<kRT, kKB, 4>;
constexpr int kBatch = 32;                // pieces listed at a time
constexpr uint32_t kQTile = umma::kTileBytes;            // 128 x 128 bf16
constexpr uint32_t kSub = 64 * 128;                      // 64 keys x 64 columns
constexpr uint32_t kKvTile = 2 * kSub;
constexpr uint32_t kOffQ = 0, kOffK = kQTile, kOffV = kOffK + 2 * kKvTile;
constexpr uint32_t kOffStage = kOffV + 2 * kKvTile;      // a warp's 32 rows x 32 columns of output
constexpr uint32_t kStagePitch = 80, kStageBytes = 32 * kStagePitch;
constexpr uint32_t kOffBars = kOffStage + 4 * kStageBytes;
constexpr int kNumBars = 15;
constexpr uint32_t kColS = 0, kColO = 128, kTmemCols = 256;

// Byte offset of the 16-byte chunk of columns [col, col + 8) of a key row in a 64-key tile.
__device__ __forceinline__ uint32_t kv_chunk_offset(uint32_t row, uint32_t col) {
  return (col >> 6) * kSub + row * 128u + ((((col & 63u) >> 3) ^ (row & 7u)) << 4);
}
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int ks) {      // K-major, 16 columns a step
  return umma::smem_desc(tile + (ks >> 2) * kSub + (ks & 3) * 32u, 16u, 1024u);
}
__device__ __forceinline__ uint64_t desc_v(uint32_t tile, int ks) {      // MN-major, 16 keys a step
  return umma::smem_desc(tile + ks * 2048u, kSub, 1024u);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// arguments of a wait: where to see that another role gave up, the budget, and the line to report
#define CB2_SITE s_abort, kDefaultWaitNs, __LINE__

struct Piece {
  int r, h, row0, t0, n, len, b0, b1;
  int whole;      // the unit's blocks all lie in this share
};

struct Smem {
  uint32_t tmem;
  int abort;
  int count;      // pieces listed; more follow if count == kBatch
  int loads_k, loads_v;     // issued so far
  PagedWalkState walk;
  long long total;
  int n_share;
  Piece pieces[kBatch];
  PagedFindSmem find;
};
constexpr uint32_t kOffMisc = kOffBars + kNumBars * 8;
constexpr uint32_t kSmemBytes = kOffMisc + uint32_t(sizeof(Smem)) + 1024;
static_assert(2 * kSmemBytes <= 227 * 1024, "two CTAs per SM");

struct TcArgs {
  const __nv_bfloat16* q;
  long long q_token, q_head;
  __nv_bfloat16* o;
  float* lse2;
  float scale_log2e;
  int G, Hkv, d;
};

__global__ void __launch_bounds__(kThreads, 2)
paged_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TcArgs a,
                const PagedBatch batch, const Cost cost, const PagedScratch scratch) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;      // two slots each
  uint64_t *s_ready = bars + 8, *p_ready = bars + 10, *o_done = bars + 12, *q_full = bars + 14;
  Smem* sh = reinterpret_cast<Smem*>(smem + kOffMisc);
  volatile int* s_abort = &sh->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, n_cta = gridDim.x;

  let_next();
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_ready[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(q_full, 128);
    sh->abort = sh->loads_k = sh->loads_v = 0;
    scratch.joins[cta].r = -1;
    mbar_fence_init();
  }
  if (warp == 1) {
    __syncwarp();
    umma::tmem_alloc(&sh->tmem, kTmemCols);
  }
  if (tid == 32) {
    umma::tma_prefetch_desc(&map_k);
    umma::tma_prefetch_desc(&map_v);
  }
  {
    const PagedShare share = paged_find_share<kThreads>(batch, cost, cta, n_cta, &sh->find);
    if (warp == 0) {
      const PagedWalk<Cost> walk(batch, cost, share);
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
  const uint32_t q_addr = smem_u32(smem + kOffQ), k_addr = smem_u32(smem + kOffK), v_addr = smem_u32(smem + kOffV);
  const int d = a.d, halves = (d + 63) >> 6;

  uint32_t n_blk = 0, n_piece = 0;        // blocks and pieces this role has gone through: the barriers' phases
  for (;;) {
    if (warp == 0) {
      PagedWalk<Cost> walk(batch, cost, sh->walk);
      __syncwarp();
      int count = 0;
      for (; count < kBatch && walk.valid(); ++count, walk.next()) {
        walk.clip();
        if (lane == 0) {
          const bool whole = walk.b0 == 0 && walk.b1 == walk.nb;
          sh->pieces[count] = Piece{walk.r, walk.h, walk.tile * kRT, walk.q.t0, walk.q.n, walk.q.len, walk.b0, walk.b1, whole};
          if (walk.b0 == 0 && !whole) paged_write_join(walk, sh->total, cta, sh->n_share, scratch.joins);
        }
      }
      if (lane == 0) {
        sh->count = count;
        sh->walk = walk;
      }
    }
    __syncthreads();
    const int count = sh->count;

    if (warp == 0 || warp == 6) {
      const bool is_v = warp == 6;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      const CUtensorMap* map = is_v ? &map_v : &map_k;
      unsigned char* ring = smem + (is_v ? kOffV : kOffK);
      const int ps_log2 = batch.page_log2, box_log2 = min(ps_log2, 6), boxes = kKB >> box_log2;
      const uint32_t box_bytes = 128u << box_log2;
      bool fine = true;
      for (int p = 0; fine && p < count; ++p) {
        const Piece pc = sh->pieces[p];
        // this lane's page of a block, looked up a block ahead
        auto look_up = [&](int b) {
          const int k = b * kKB + (lane << box_log2);
          return lane < boxes && b < pc.b1 && k < pc.len ? paged_page(batch, pc.r, k >> ps_log2) : -1;
        };
        int next = look_up(pc.b0);
        for (int b = pc.b0; b < pc.b1; ++b, ++n_blk) {
          const int slot = n_blk & 1, page = next;
          next = look_up(b + 1);
          const bool mine = page >= 0;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * halves * box_bytes;
          const int y = ps_log2 > 6 ? (b * kKB) & ((1 << ps_log2) - 1) : 0;       // inside a page longer than a block
          const bool ok = n_blk < 2 || mbar_wait_abortable(&empty[slot], ((n_blk >> 1) - 1) & 1, CB2_SITE);
          fine = __all_sync(0xffffffffu, ok);
          if (!fine) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[slot], bytes);
            ++*(is_v ? &sh->loads_v : &sh->loads_k);
          }
          __syncwarp();
          if (mine) {
            unsigned char* dst = ring + slot * kKvTile + lane * box_bytes;
            for (int hf = 0; hf < halves; ++hf) umma::tma_load_4d(dst + hf * kSub, map, hf * 64, y, pc.h, page, &full[slot]);
          }
        }
      }
    } else if (warp == 1) {
      // the whole warp walks, waits and computes the operands (shuffled, which tells the compiler that they are uniform:
      // 391 -> 375 us at the size above), one lane issues
      const bool lead = lane == 0;
      auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
      const int ksteps = int(uniform((d + 15) >> 4));
      const uint32_t d_cols = uniform(tmem), qa = uniform(q_addr), ka = uniform(k_addr), va = uniform(v_addr);
      constexpr uint32_t idesc_kk = umma::instr_desc_bf16(128, kKB, false, false);
      const uint32_t idesc_kn = umma::instr_desc_bf16(128, uint32_t(d + 15) & ~15u, false, true);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, mbar_wait_abortable(bar, parity, s_abort, kDefaultWaitNs, site));
      };
      for (int p = 0; p < count; ++p, ++n_piece) {
        const int blocks = int(uniform(sh->pieces[p].b1 - sh->pieces[p].b0));
        bool ok = wait(q_full, n_piece & 1, __LINE__);
        // scores run two blocks ahead; the tensor pipe runs in issue order, so those of block j + 2 may overwrite P of
        // block j right behind the product that reads it
        for (int j = -2; ok && j < blocks; ++j) {
          const uint32_t n = uniform(n_blk + j), slot = n & 1;        // (block j + 2 has the same slot)
          const uint32_t s_cols = d_cols + kColS + slot * kKB, k_tile = ka + slot * kKvTile, v_tile = va + slot * kKvTile;
          if (j >= 0) {
            ok = wait(&p_ready[slot], (n >> 1) & 1, __LINE__) && wait(&v_full[slot], (n >> 1) & 1, __LINE__);
            if (!ok) break;
            umma::fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < kKB / 16; ++ks)
              umma::mma_bf16_ts_by(lead, d_cols + kColO, s_cols + ks * 8, desc_v(v_tile, ks), idesc_kn, j > 0 || ks > 0);
            umma::mma_commit_by(lead, &o_done[slot]);
            umma::mma_commit_by(lead, &v_empty[slot]);
          }
          if (j + 2 < blocks) {
            ok = wait(&k_full[slot], ((n + 2) >> 1) & 1, __LINE__);
            if (!ok) break;
            umma::fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              if (ks < ksteps)
                umma::mma_bf16_by(lead, s_cols, umma::desc_kmajor(qa, ks), desc_k(k_tile, ks), idesc_kk, ks > 0);
            umma::mma_commit_by(lead, &s_ready[slot]);
            umma::mma_commit_by(lead, &k_empty[slot]);
          }
        }
        if (!ok) break;
        n_blk += blocks;
      }
    } else {
      // lanes q4 * 32 of tensor memory hold the tile's rows from `first_row` on; every second CTA begins in the other half,
      // so that the few rows of short tiles fall to different quarters of the SM
      const int q4 = warp & 3, first_row = ((q4 + (cta * 2 < n_cta ? 0 : 2)) & 3) * 32, rr = first_row + lane;
      const uint32_t lane_base = tmem + (uint32_t(q4 * 32) << 16);
      constexpr float kLazy = 8.f;
      const int ncb = (d + 31) >> 5;
      const float scale = a.scale_log2e;
      // The 32 packed rows of this warp, into the query tile: a lane works out the place of one row, 8 or 16
      // neighbouring lanes copy its chunks (a copy instruction then touches two or four rows, not 32).
      auto load_rows = [&](const Piece* pc) {
        if (pc->row0 + first_row >= pc->n * a.G) return;
        const int row = pc->row0 + rr;
        const bool there = row < pc->n * a.G;
        const int tok = there ? row / a.G : 0, g = there ? row - tok * a.G : 0;
        const long long at = (pc->t0 + tok) * a.q_token + (pc->h * a.G + g) * a.q_head;
        const unsigned have = __ballot_sync(0xffffffffu, there);
        const int chunks = halves * 8, c = lane & (chunks - 1), sub = lane / chunks, step = 32 / chunks;
        const bool col = c * 8 < d;
        const uint32_t dst = q_addr + q4 * 32 * 128u + (c >> 3) * umma::kSubTileBytes;
        // not unrolled: at a kernel's start every instruction line is a miss
#pragma unroll 1
        for (int from = sub; from < 32; from += step) {
          const long long off = __shfl_sync(0xffffffffu, at, from);
          const bool ok = ((have >> from) & 1) && col;
          cp_async16_or_zero(dst + from * 128u + (((c & 7) ^ (from & 7)) << 4), a.q + off + (ok ? c * 8 : 0), ok);
        }
        cp_async_commit();
      };
      auto rows_there = [&] {
        cp_async_wait_all();
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      };
      if (count > 0) {
        load_rows(&sh->pieces[0]);
        rows_there();
      }
      for (int p = 0; p < count; ++p) {
        const Piece* pc = &sh->pieces[p];
        const int blocks = pc->b1 - pc->b0, b0 = pc->b0, len = pc->len;
        const int rows = pc->n * a.G - pc->row0;                 // of this tile, kRT at most count
        // last slot this row sees, and the least of the tile's rows
        const int base = len - pc->n;
        // a warp without rows only keeps step: what the products make of its lanes is never read (12 chunks of 17 tokens,
        // d 96: 22.7 -> 21.9 us)
        const bool busy = first_row < rows;
        const int last = cost.causal ? min(base + (pc->row0 + rr) / a.G, len - 1) : len - 1;
        const int first_last = cost.causal ? min(base + pc->row0 / a.G, len - 1) : len - 1;
        float m_ref = -INFINITY, l_run = 0.f;
        bool ok = true;
        for (int j = 0; j < blocks; ++j) {
          const uint32_t n = n_blk + j, slot = n & 1;
          const uint32_t s_cols = lane_base + kColS + slot * kKB;
          ok = mbar_wait_abortable(&s_ready[slot], (n >> 1) & 1, CB2_SITE);
          if (!__all_sync(0xffffffffu, ok)) break;
          umma::fence_after_sync();
          const int k0 = (b0 + j) * kKB;
          // the last scores of this piece are out, so the next piece's rows may take its place
          const bool next_rows = j == blocks - 1 && p + 1 < count;
          if (next_rows) load_rows(pc + 1);
          float alpha = 1.f;
          if (busy) {
            uint32_t sv[2][32];
#pragma unroll
            for (int cb = 0; cb < 2; ++cb) umma::tmem_ld32(s_cols + cb * 32, sv[cb]);
            umma::tmem_wait_ld();
            umma::tmem_loaded(sv[0]);
            umma::tmem_loaded(sv[1]);
            if (k0 + kKB - 1 > first_last) {
              const int lim = last - k0;
#pragma unroll
              for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  if (cb * 32 + c > lim) sv[cb][c] = 0xff800000u;
            }
            float mx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(sv[0][i]), __uint_as_float(sv[1][i]));
#pragma unroll
            for (int c = 4; c < 32; ++c) mx[c & 3] = max3(mx[c & 3], __uint_as_float(sv[0][c]), __uint_as_float(sv[1][c]));
            const float m_blk = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * scale;
            if (m_blk > m_ref + kLazy || m_ref == -INFINITY) {
              const float m_new = fmaxf(m_ref, m_blk);
              alpha = (m_new == -INFINITY) ? 1.f : ex2_approx(m_ref - m_new);
              m_ref = m_new;
            }
            const float neg_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
            const uint64_t scale2 = umma::f2_pack(scale, scale), neg2 = umma::f2_pack(neg_m, neg_m);
            uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
            for (int cb = 0; cb < 2; ++cb) {
              uint32_t w[16];
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                const uint64_t x = umma::f2_fma(umma::f2_pack(__uint_as_float(sv[cb][c]), __uint_as_float(sv[cb][c + 1])), scale2, neg2);
                float x0, x1;
                umma::f2_unpack(x, x0, x1);
                const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                sum2[(c >> 1) & 1] = umma::f2_add(sum2[(c >> 1) & 1], umma::f2_pack(p0, p1));
                w[c >> 1] = pack_bf16x2(p0, p1);
              }
              umma::tmem_st16(s_cols + cb * 16, w);
            }
            float s0, s1;
            umma::f2_unpack(umma::f2_add(sum2[0], sum2[1]), s0, s1);
            l_run = fmaf(l_run, alpha, s0 + s1);
            umma::tmem_wait_st();
          }
          if (k0 + kKB > len) {
            // the request's last block: value rows that nobody has written
            ok = mbar_wait_abortable(&v_full[slot], (n >> 1) & 1, CB2_SITE);
            if (!__all_sync(0xffffffffu, ok)) break;
            const int row = rr & (kKB - 1);
            if (k0 + row >= len && (rr >> 6) < halves)
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(smem + kOffV + slot * kKvTile + kv_chunk_offset(row, (rr >> 6) * 64 + c * 8)) =
                    make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
          // O <- O alpha once the product before has landed.  This wait is often skipped, so the products
          // alternate between two barriers: of one barrier's phases, all but the awaited one are then known to be over
          if (busy && j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            ok = mbar_wait_abortable(&o_done[slot ^ 1], ((n - 1) >> 1) & 1, CB2_SITE);
            if (!__all_sync(0xffffffffu, ok)) break;
            umma::fence_after_sync();
            uint32_t ov[32];
            for (int cb = 0; cb < ncb; ++cb) {
              umma::tmem_ld32(lane_base + kColO + cb * 32, ov);
              umma::tmem_wait_ld();
              umma::tmem_loaded(ov);
#pragma unroll
              for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
              umma::tmem_st32(lane_base + kColO + cb * 32, ov);
            }
            umma::tmem_wait_st();
          }
          umma::fence_before_sync();
          mbar_arrive(&p_ready[slot]);
          if (next_rows) rows_there();
        }
        if (!__all_sync(0xffffffffu, ok)) break;
        n_blk += blocks;
        if (!busy) continue;
        ok = mbar_wait_abortable(&o_done[(n_blk - 1) & 1], ((n_blk - 1) >> 1) & 1, CB2_SITE);
        if (!__all_sync(0xffffffffu, ok)) break;
        umma::fence_after_sync();
        const bool live = rr < rows, whole = pc->whole;
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;      // a NaN sum stays one
        const int row = pc->row0 + rr;
        const long long at = (long long)(pc->t0 + row / a.G) * (a.G * a.Hkv) + pc->h * a.G + row % a.G;
        float* slot = scratch.parts + paged_slot_floats(kRT, d) * (2 * cta + (b0 == 0));
        unsigned char* stage = smem + kOffStage + q4 * kStageBytes;
        for (int cb = 0; cb < ncb; ++cb) {
          uint32_t sv[32];
          umma::tmem_ld32(lane_base + kColO + cb * 32, sv);
          umma::tmem_wait_ld();
          umma::tmem_loaded(sv);
          if (whole) {
            // 32 columns of 32 rows, turned in shared memory so that a store covers 64 bytes of 8 rows
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = pack_bf16x2(__uint_as_float(sv[c * 8 + 2 * i]) * inv, __uint_as_float(sv[c * 8 + 2 * i + 1]) * inv);
              *reinterpret_cast<uint4*>(stage + lane * kStagePitch + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            const int col = cb * 32 + (lane & 3) * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r8 = i * 8 + (lane >> 2);
              const uint4 v = *reinterpret_cast<const uint4*>(stage + r8 * kStagePitch + (lane & 3) * 16);
              const long long to = __shfl_sync(0xffffffffu, at, r8);
              if (first_row + r8 < rows && col < d) *reinterpret_cast<uint4*>(a.o + to * d + col) = v;
            }
            __syncwarp();
          } else if (live) {
            float* dst = slot + 2 * kRT + (cb * 8 * kRT + rr) * 4;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              if (cb * 32 + c * 4 < d)
                *reinterpret_cast<uint4*>(dst + c * kRT * 4) = make_uint4(sv[4 * c], sv[4 * c + 1], sv[4 * c + 2], sv[4 * c + 3]);
          }
          __syncwarp();
        }
        if (live && whole && a.lse2) a.lse2[at] = l_run == 0.f ? INFINITY : m_ref + log2f(l_run);
        if (live && !whole) {
          slot[rr] = m_ref;
          slot[kRT + rr] = l_run;
        }
      }
    }
    // the batch's pieces may be listed anew once every role is through with them
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (count < kBatch || *s_abort) break;
  }
  if (*s_abort) {
    // loads in flight land before the shared memory goes (a bounded wait, too)
    if (tid == 0) {
      for (int n = max(sh->loads_k - 2, 0); n < sh->loads_k; ++n) mbar_wait_bounded(&k_full[n & 1], (n >> 1) & 1);
      for (int n = max(sh->loads_v - 2, 0); n < sh->loads_v; ++n) mbar_wait_bounded(&v_full[n & 1], (n >> 1) & 1);
      if (batch.status) atomicExch(batch.status, CB2_WAIT_TIMEOUT | (*s_abort << 8));     // which wait: its source line
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    umma::tmem_dealloc(tmem, kTmemCols);
  }
}

constexpr int kCtas = 2 * kNumSMs;

}  // namespace

// Pools as a 4-D tensor {d, page_size, Hkv, n_pages}; box = 64 columns of a page, 64 rows at most.
int paged_pool_map(CUtensorMap* out, const void* base, int d, int page_size, int Hkv, int n_pages, long long page_stride) {
  const umma::EncodeTiledFn fn = umma::encode_tiled();
  if (!fn) return CB2_LAUNCH_FAIL;
  const cuuint64_t dims[4] = {cuuint64_t(d), cuuint64_t(page_size), cuuint64_t(Hkv), cuuint64_t(n_pages)};
  const cuuint64_t strides[3] = {cuuint64_t(d) * 2, cuuint64_t(page_size) * d * 2, cuuint64_t(page_stride) * 2};
  const cuuint32_t box[4] = {64, cuuint32_t(page_size < 64 ? page_size : 64), 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CB2_OK : CB2_LAUNCH_FAIL;
}

size_t paged_tc_scratch_bytes(int d) { return paged_scratch_bytes(kCtas, kRT, d); }

// Requests of more than `few` packed rows; partial carriers are left in `scratch` (kRT rows a slot, kCtas shares).
int paged_tc_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int few, void* o, float* lse2,
                 void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st) {
  CUtensorMap mk, mv;
  int rc = paged_pool_map(&mk, pools.k, pools.d, 1 << batch.page_log2, pools.Hkv, batch.n_pages, pools.k_page_stride);
  if (rc == CB2_OK) rc = paged_pool_map(&mv, pools.v, pools.d, 1 << batch.page_log2, pools.Hkv, batch.n_pages, pools.v_page_stride);
  if (rc != CB2_OK) return rc;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(paged_tc_kernel), kSmemBytes, done)) return CB2_LAUNCH_FAIL;
  *parts = paged_scratch(scratch, kCtas);
  *n_cta = kCtas;
  const TcArgs a{static_cast<const __nv_bfloat16*>(rows.q), rows.q_token, rows.q_head, static_cast<__nv_bfloat16*>(o), lse2,
                 rows.scale_log2e, rows.G, rows.Hkv, pools.d};
  const Cost cost{rows.G, rows.Hkv, causal, kPagedChunk, few, 4};
  paged_tc_kernel<<<kCtas, kThreads, kSmemBytes, st>>>(mk, mv, a, batch, cost, *parts);
  CB2_LAUNCH_CHECK();
  return CB2_OK;
}

}  // namespace cb2

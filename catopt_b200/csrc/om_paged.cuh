// Attention of a ragged batch of new tokens over a paged key/value cache: what its kernels share.
//
// Pools   k_pages, v_pages: [n_pages, Hkv, page_size, d] (a page of one kv head is contiguous; the
//         distance between pages is free), page_size a power of two.  Request r owns the pages
//         table[r][0..]; key slot j of it sits in page table[r][j / page_size], row j % page_size.
// Rows    The G = Hq / Hkv query heads of a kv head share its keys, so the rows of a unit of work are
//         the packed pairs (token, head of the group): row = token * G + g, n_r * G rows per
//         (request, kv head), cut into tiles of RT rows.
// Work    One unit = (request, kv head, row tile); its cost is the number of KB-key blocks some row of
//         the tile can see.  All blocks of all units form one line, which is cut into equal shares, one
//         per CTA: ragged lengths, causal tiles and single long requests balance by themselves, from
//         lengths that only the device knows (a captured graph stays right when they change).  A unit
//         that lies in one share is finished there; one that crosses shares leaves a partial carrier
//         (m, l, a) per share, which paged_combine_kernel joins in share order (no atomics: the same
//         inputs give the same bits).
#pragma once
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "paged_clamp.cuh"

namespace cb2 {

// Lets a kernel use `bytes` of dynamic shared memory, asked for once per device (`done`: one bit each): a decode step is
// short enough for the question to show.
inline bool allow_smem(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// A kernel that reads what the kernel before it leaves is launched while that one still runs (programmatic dependent
// launch): it waits with after_previous() at its top, and the one before has called let_next() at its own.  Of a chain, every
// kernel waits in all of its blocks, so what the last one sees is complete.  What the one before writes is read through
// ordinary pointers: a load that is declared constant (const __restrict__, __ldg) may be moved ahead of the wait.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... Args>
inline int launch_next(void (*kernel)(Args...), dim3 grid, unsigned threads, cudaStream_t st, std::common_type_t<Args>... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? CB2_OK : CB2_LAUNCH_FAIL;
}

// The index tensors of a ragged batch.  Values out of range are clamped where they are read and
// reported as CB2_BAD_INDEX, so that no index tensor can lead to an access out of bounds.
struct PagedBatch {
  const int* table;   // [R, max_pages]
  const int* lens;    // [R] cached keys, the new tokens included
  const int* cu;      // [R+1] first row of each request in q
  int R, max_pages, n_pages, page_log2, n_tokens, max_q, max_k;
  int* status;
};

struct PagedPools {
  const void* k;
  const void* v;
  long long k_page_stride, v_page_stride;   // elements
  int Hkv, d;
};

struct PagedRows {
  const void* q;
  long long q_token, q_head;   // strides in elements
  int G, Hkv;
  float scale_log2e;
};

__device__ __forceinline__ void paged_flag(const PagedBatch& b) {
  if (b.status) atomicExch(b.status, CB2_BAD_INDEX);
}

__device__ __forceinline__ PagedReq paged_request(const PagedBatch& b, int r) {
  PagedReq q;
  if (!paged_clamp(__ldg(b.cu + r), __ldg(b.cu + r + 1), __ldg(b.lens + r), b.n_tokens, b.max_q, b.max_k, &q)) paged_flag(b);
  return q;
}

// Pool page of table entry i of request r; page 0 (always there) for an id out of range.
__device__ __forceinline__ int paged_page(const PagedBatch& b, int r, int i) {
  const int p = __ldg(b.table + (long long)r * b.max_pages + i);
  if (unsigned(p) < unsigned(b.n_pages)) return p;
  paged_flag(b);
  return 0;
}

// sum of floor((a i + b) / m) over i < n, for 0 <= a, b and a n + b < 2^31: the lattice points under
// a line, counted by exchanging the axes as in Euclid's algorithm.
__device__ inline long long lattice_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  long long sum = 0;
  bool add = true;    // the exchanged problem counts the complement
  while (n > 0) {
    long long part = 0;
    if (a >= m) {
      part += (long long)(a / m) * ((long long)n * (n - 1) / 2);
      a %= m;
    }
    if (b >= m) {
      part += (long long)(b / m) * n;
      b %= m;
    }
    sum += add ? part : -part;
    // with a, b < m: sum_i floor((a i + b)/m) = n h - #{(i, y): 0 < y <= h, a i + b < m y}, h = the
    // largest term; the y-th row holds ceil((m y - b)/a) = floor((m y - b + a - 1)/a) of these points
    const unsigned h = a == 0 ? 0 : (a * (n - 1) + b) / m;
    if (h == 0) break;
    sum += add ? (long long)n * h : -(long long)n * h;
    add = !add;
    // rows y = 1..h  ->  i' = y - 1: floor((m i' + m - b + a - 1) / a)
    const unsigned nb = m - b + a - 1, na = m, nm = a;
    n = h;
    a = na;
    b = nb;
    m = nm;
  }
  return sum;
}

// The same for the steps that a tile count of a power of two gives, without Euclid's divisions.
//   m = a k:  floor((a i + b) / m) = floor((i + c) / k), c = floor(b / a): a difference of two sums of floor(j / k);
//   a = m k:  floor((a i + b) / m) = k i + floor(b / m).
__device__ __forceinline__ long long stair_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  if (m >= a && m % a == 0) {
    const unsigned k = m / a, c = b / a;
    auto upto = [k](unsigned x) {
      const unsigned q = x / k, r = x - q * k;
      return (long long)k * ((long long)q * (q - 1) / 2) + (long long)q * r;     // q = 0 gives 0
    };
    return upto(n + c) - upto(c);
  }
  if (a % m == 0) return (long long)(a / m) * ((long long)n * (n - 1) / 2) + (long long)n * (b / m);
  return lattice_sum(n, m, a, b);
}

// The requests that a kernel takes: those with at most `few` packed rows, or the others.
enum { kPagedFew, kPagedChunk };

// OV: what starting and ending a unit costs, in blocks; a unit takes OV + blocks of the line.
template <int RT, int KB, int OV>
struct PagedCost {
  static constexpr int kOv = OV;
  int G, Hkv, causal, which, few;
  int min_blocks;          // a share holds at least so many: fewer CTAs work on a short line
  __device__ __forceinline__ bool takes(const PagedReq& q) const {
    if (q.n == 0) return false;
    return (which == kPagedFew) == (q.n * G <= few);
  }
  __device__ __forceinline__ int tiles(const PagedReq& q) const { return (q.n * G + RT - 1) / RT; }
  __device__ __forceinline__ int all_blocks(const PagedReq& q) const { return max(1, (q.len + KB - 1) / KB); }
  // blocks that tile i visits: up to the last token of the tile
  __device__ __forceinline__ int blocks(const PagedReq& q, int i) const {
    const int base = q.len - q.n;
    if (!causal || base < 0 || i == tiles(q) - 1) return all_blocks(q);
    return int((unsigned(i) * RT + RT - 1 + unsigned(G) * (base + KB)) / (unsigned(G) * KB));
  }
  // length of the first `k` tiles of one kv head
  __device__ __forceinline__ long long before(const PagedReq& q, int k) const {
    const int base = q.len - q.n, nt = tiles(q);
    if (!causal || base < 0) return (long long)k * (all_blocks(q) + OV);
    const int m = min(k, nt - 1);
    long long s = stair_sum(m, unsigned(G) * KB, RT, RT - 1 + unsigned(G) * (base + KB));
    if (k == nt) s += all_blocks(q);
    return s + (long long)k * OV;
  }
  // length of one kv head of a request
  __device__ __forceinline__ long long per_head(const PagedReq& q) const { return takes(q) ? before(q, tiles(q)) : 0; }
};

struct PagedFindSmem {
  long long warp_sum[32];
  long long per_head, off;
  PagedReq q;
  int r;
};

// Start of this CTA's share [lo, hi) of the line: request and offset in it.  All T threads call it.
struct PagedShare {
  long long total, lo, hi;
  int n_share;      // shares that are not empty: [0, n_share)
  int r;            // request that holds lo
  PagedReq q;
  long long per_head;
  long long off;    // lo - start of that request
};

__device__ __forceinline__ long long paged_cut(long long total, int c, int n) {
  if (total < (1 << 20) && n <= 4096) return unsigned(total) * unsigned(c) / unsigned(n);     // without a 64-bit division
  return total * c / n;
}

template <int T, class Cost>
__device__ PagedShare paged_find_share(const PagedBatch& b, const Cost& cost, int cta, int n_cta, PagedFindSmem* s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  PagedShare out;
  const int passes = (b.R + T - 1) / T;
  PagedReq q{0, 0, 0};
  long long per_head = 0, mine = 0;        // of the request this thread looked at last
  // inclusive prefix of the costs of requests [pass * T, pass * T + T), on top of `carry`
  auto scan = [&](int pass, long long carry, long long& block_total) -> long long {
    const int r = pass * T + tid;
    if (r < b.R) q = paged_request(b, r);
    per_head = r < b.R ? cost.per_head(q) : 0;
    mine = per_head * cost.Hkv;
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s->warp_sum[warp] = x;
    __syncthreads();
    long long pre = carry;
    for (int w = 0; w < warp; ++w) pre += s->warp_sum[w];
    block_total = 0;
    for (int w = 0; w < T / 32; ++w) block_total += s->warp_sum[w];
    if (passes > 1) __syncthreads();       // before the sums of the next pass
    return x + pre;
  };
  if (tid == 0) {
    s->r = 0;
    s->off = 0;
    s->per_head = 0;
    s->q = PagedReq{0, 0, 0};
  }
  long long block_total, incl = 0, total = 0;
  for (int p = 0; p < passes; ++p) {
    incl = scan(p, total, block_total);
    total += block_total;
  }
  out.total = total;
  out.n_share = total >= (long long)n_cta * cost.min_blocks ? n_cta : max(1, int(unsigned(total) / unsigned(cost.min_blocks)));
  out.lo = out.hi = total;
  if (cta < out.n_share) {
    out.lo = paged_cut(total, cta, out.n_share);
    out.hi = paged_cut(total, cta + 1, out.n_share);
  }
  long long carry = 0;
  for (int p = 0; p < passes; ++p) {
    if (passes > 1) {
      incl = scan(p, carry, block_total);
      carry += block_total;
    }
    if (mine > 0 && out.lo >= incl - mine && out.lo < incl) {
      s->r = p * T + tid;
      s->off = out.lo - (incl - mine);
      s->per_head = per_head;
      s->q = q;
    }
  }
  __syncthreads();
  out.r = s->r;
  out.off = s->off;
  out.per_head = s->per_head;
  out.q = s->q;
  return out;
}

// Walks the pieces of a share: piece = blocks [b0, b1) of the nb blocks of unit (r, h, tile).
// Every thread of a warp keeps the same walk; the state may rest in shared memory between uses.
struct PagedWalkState {
  long long cur, hi;
  PagedReq q;
  int r, h, tile, nb, b0, b1;
};

template <class Cost>
struct PagedWalk : PagedWalkState {
  const PagedBatch& batch;
  const Cost& cost;

  __device__ PagedWalk(const PagedBatch& b, const Cost& c, const PagedWalkState& s) : PagedWalkState(s), batch(b), cost(c) {}
  __device__ PagedWalk(const PagedBatch& b, const Cost& c, const PagedShare& s) : batch(b), cost(c) {
    cur = s.lo;
    hi = s.hi;
    r = s.r;
    h = tile = nb = b0 = b1 = 0;
    q = s.q;
    if (cur >= hi) return;
    h = s.off < (1ll << 32) && s.per_head < (1ll << 32) ? int(unsigned(s.off) / unsigned(s.per_head)) : int(s.off / s.per_head);
    const long long rest = s.off - h * s.per_head;
    // last tile whose start is <= rest: 32 candidates a round, one per lane
    int lo = 0, n = cost.tiles(q);
    const int lane = threadIdx.x & 31;
    while (n > 1) {
      const int step = (n + 31) / 32;
      const bool le = lane * step < n && cost.before(q, lo + lane * step) <= rest;
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, le));
      n = min(step, n - k * step);
      lo += k * step;
    }
    tile = lo;
    nb = cost.blocks(q, tile);
    b0 = int(rest - cost.before(q, tile)) - Cost::kOv;
    enter();
  }
  __device__ bool valid() const { return cur < hi; }
  __device__ void clip() { b1 = int(min((long long)nb, b0 + (hi - cur))); }
  // past the unit's overhead, to its first block (a share may end before)
  __device__ void enter() {
    if (b0 < 0) {
      cur -= b0;
      b0 = 0;
    }
  }
  __device__ void next() {
    cur += b1 - b0;
    b0 = -Cost::kOv;
    if (cur >= hi) return;
    if (++tile == cost.tiles(q)) {
      tile = 0;
      if (++h == cost.Hkv) {
        h = 0;
        do {
          ++r;
          q = paged_request(batch, r);
        } while (!cost.takes(q));
      }
    }
    nb = cost.blocks(q, tile);
    enter();
  }
};

// A unit that starts in share c and goes on in the next ones: written by CTA c for the combine kernel.
struct PagedJoin {
  int r, h, tile, last;     // r < 0: none; last = share that holds the unit's last block
  int t0, n, pad[2];        // the request's rows
};
// Partial carriers: share c owns slot 2c (a piece that does not start its unit) and 2c + 1 (a piece
// that starts a unit and does not finish it).  Slot: m[RT], l[RT], a, fp32, m in log2 units; a is [RT][d], or
// [d / 4][RT][4] for tiles of 128 rows, whose writers hold a row a thread.
__host__ __device__ __forceinline__ size_t paged_slot_floats(int rt, int d) { return size_t(rt) * (d + 2); }

// 16-byte asynchronous copy that writes zeros when `there` is false.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void paged_write_join(const PagedWalkState& w, long long total, int cta, int n_share, PagedJoin* joins) {
  // called for a piece with b0 == 0 and b1 < nb: the unit's last block sits at cur + nb - 1 of the line
  PagedJoin j;
  j.r = w.r;
  j.h = w.h;
  j.tile = w.tile;
  j.t0 = w.q.t0;
  j.n = w.q.n;
  j.pad[0] = j.pad[1] = 0;
  const long long x = (w.cur + w.nb) * n_share - 1;
  j.last = x < (1ll << 32) ? int(unsigned(x) / unsigned(total)) : int(x / total);
  joins[cta] = j;
}

// Kept scores of a request, kv head and packed row: so many floats apart, a multiple of four.
__host__ __device__ __forceinline__ long long paged_score_stride(int max_k) { return (max_k + 3ll) & ~3ll; }

// Scratch of one attention kernel of n_cta shares: the joins, the partial carriers.
struct PagedScratch {
  PagedJoin* joins;
  float* parts;
};
__host__ __device__ inline size_t paged_scratch_bytes(int n_cta, int rt, int d) {
  return size_t(n_cta) * sizeof(PagedJoin) + size_t(n_cta) * 2 * paged_slot_floats(rt, d) * 4;
}
inline PagedScratch paged_scratch(void* base, int n_cta) {
  PagedScratch s;
  s.joins = static_cast<PagedJoin*>(base);
  s.parts = reinterpret_cast<float*>(static_cast<char*>(base) + size_t(n_cta) * sizeof(PagedJoin));
  return s;
}

// om_paged_tc.cu: requests of more than `few` packed rows (bf16), on the tensor cores.  What it leaves for
// the join: tiles of 128 rows, *n_cta shares.
size_t paged_tc_scratch_bytes(int d);
int paged_tc_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int few, void* o,
                 float* lse2, void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st);

// om_paged_few.cu: requests of at most `few` (8 or 16) packed rows (bf16), one pass over K and V.  scores (may be
// NULL): [R, Hkv, few, max_k] floats for paged_few_weights_run.
size_t paged_few_scratch_bytes(int d);
int paged_few_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int few, void* o,
                  float* lse2, float* scores, void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st);
int paged_few_weights_run(const PagedRows& rows, const PagedBatch& batch, int causal, int few, const float* scores,
                          const float* lse2, float* weights, cudaStream_t st);

// om_paged_weights.cu: attention weight of the requests of class `which` (bf16), from their lse.
size_t paged_weights_tc_scratch_bytes();
int paged_weights_tc_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few,
                         const float* lse2, float* weights, void* scratch, cudaStream_t st);

// om_paged_fma.cu: fp32.  Row tiles of rt = 8, 16 or 64; scores as for the streaming kernel.
size_t paged_fma_scratch_bytes(int rt, int d);
int paged_fma_run(int rt, const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few,
                  float* o, float* lse2, float* kept_scores, void* scratch, PagedScratch* parts, int* n_cta, cudaStream_t st);
int paged_weights_fma_run(const PagedRows& rows, const PagedPools& pools, const PagedBatch& batch, int causal, int which, int few,
                          const float* lse2, float* weights, cudaStream_t st);

}  // namespace cb2

// Eviction from a paged key/value cache by accumulated attention weight.
//
// A request longer than the budget keeps, for every kv head by itself, its first and last slots and, of the
// slots between, those of the largest weight (ties to the lowest slot; NaN counts as the smallest), in slot
// order; they are copied to the pages of another table, keys, values and weights alike.  A shorter request is
// copied whole.  The old pages stay as they are, so shared prefixes are no hazard and the copy needs no order.
//
// Two launches.  paged_select_kernel: one CTA per (request, kv head) finds the budget-th weight by radix
// selection (11, 11 and 10 bits) on the weights' order-preserving bit patterns and writes the kept slots in ascending order.
// paged_move_kernel: copies rows, bound by memory (kept rows read once and written once).
//
// Measured: 16 streams of up to 8192 keys, 8 kv heads of 128, cut to 4096: selection 16 us (the weights come from memory
// once; the three passes and the write of the kept slots are a chain of barriers in one CTA, issue 20 % busy), copy 73 us
// (6.2 TB/s of rows read and written), 91 us together.
#include "om_paged.cuh"

namespace cb2 {
namespace {

constexpr int kSelThreads = 1024, kMoveThreads = 256, kMoveRows = 64;
constexpr int kMostHeld = 48 * 1024;       // keys that fit shared memory beside the histogram
constexpr int kBins = 2048;

// Unsigned key of the same order as the float: NaN lowest, -0 and +0 the same.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictArgs {
  const float* weights;
  int Hkv, budget, first, last;
  int* kept;        // [R, Hkv, budget]
  int* new_lens;    // [R]
  int held;         // keys of a request that shared memory holds
};

struct WeightReader {
  const PagedBatch& b;
  const float* w;
  int r, h, Hkv;
  __device__ __forceinline__ uint32_t operator()(int j) const {
    const int page = paged_page(b, r, j >> b.page_log2), ps = 1 << b.page_log2;
    return weight_key(w[((long long)page * Hkv + h) * ps + (j & (ps - 1))]);
  }
  // slots j .. j + 3, j a multiple of four
  __device__ __forceinline__ void four(int j, uint32_t (&k)[4]) const {
    const int page = paged_page(b, r, j >> b.page_log2), ps = 1 << b.page_log2;
    const float4 x = *reinterpret_cast<const float4*>(w + ((long long)page * Hkv + h) * ps + (j & (ps - 1)));
    k[0] = weight_key(x.x);
    k[1] = weight_key(x.y);
    k[2] = weight_key(x.z);
    k[3] = weight_key(x.w);
  }
};

// Positions among the true flags of a block, thread order: exclusive rank and total.
__device__ __forceinline__ int block_rank(bool flag, int* warp_count, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned b = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) warp_count[warp] = __popc(b);
  __syncthreads();
  const int c = warp_count[lane];                       // kSelThreads / 32 = 32 warps
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0);
  total = __reduce_add_sync(0xffffffffu, c);
  return before + __popc(b & ((1u << lane) - 1));
}
static_assert(kSelThreads == 1024, "block_rank reads one count a lane");

__global__ void __launch_bounds__(kSelThreads)
paged_select_kernel(const EvictArgs a, const PagedBatch batch) {
  extern __shared__ __align__(16) uint32_t sh_keys[];                 // [held]
  __shared__ int hist[kBins];
  __shared__ int warp_count[2][2][32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  let_next();
  const int l0 = __ldg(batch.lens + r), len = min(max(l0, 0), batch.max_k);
  if (len != l0) paged_flag(batch);
  int* kept = a.kept + ((long long)r * a.Hkv + h) * a.budget;
  if (h == 0 && tid == 0) a.new_lens[r] = min(len, a.budget);
  if (len <= a.budget) {
    for (int i = tid; i < a.budget; i += kSelThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const WeightReader key{batch, a.weights, r, h, a.Hkv};
  const int lo = a.first, hi = len - a.last;             // first + last <= budget < len
  const int want = a.budget - a.first - a.last;          // of [lo, hi)
  const int held = min(a.held, len);
#pragma unroll 2
  for (int j = 4 * tid; j < held; j += 4 * kSelThreads) {      // four neighbouring slots lie in one page
    uint32_t k[4];
    key.four(j, k);
    *reinterpret_cast<uint4*>(sh_keys + j) = make_uint4(k[0], k[1], k[2], k[3]);
  }
  auto key_at = [&](int j) { return j < held ? sh_keys[j] : key(j); };
  if (tid == 0) {
    s_prefix = 0;
    s_need = want;
  }
  // the want-th largest key of [lo, hi), 11, 11 and 10 bits at a time
  for (int pass = 0; want > 0 && pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t mask = pass == 0 ? 0u : ~0u << (shift + bits), bin_mask = (1u << bits) - 1;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    const int need = s_need;
    for (int j0 = lo; j0 < hi; j0 += kSelThreads) {
      const int j = j0 + tid;
      const uint32_t k = j < hi ? key_at(j) : 0u;
      const bool in = j < hi && (k & mask) == prefix;
      const uint32_t bin = (k >> shift) & bin_mask;
      // many keys may be the same (0, say): the lanes that agree with the first one add together
      const unsigned all = __ballot_sync(0xffffffffu, in);
      const uint32_t first = __shfl_sync(0xffffffffu, bin, all ? __ffs(all) - 1 : 0);
      const unsigned same = __ballot_sync(0xffffffffu, in && bin == first);
      if (in && bin != first) atomicAdd(&hist[bin], 1);
      if (same && lane == __ffs(same) - 1) atomicAdd(&hist[first], __popc(same));
    }
    __syncthreads();
    // from the top: the 64 bins in which the need runs out (a warp each), then the bin
    const int top = kBins - 1 - warp * 64;
    const int c0 = hist[top - lane], c1 = hist[top - 32 - lane];
    const int mine = __reduce_add_sync(0xffffffffu, c0 + c1);
    if (lane == 0) warp_count[0][0][warp] = mine;
    __syncthreads();
    const int other = warp_count[0][0][lane];
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? other : 0);
    if (before < need && before + mine >= need) {          // one warp
      int incl0 = c0, incl1 = c1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y0 = __shfl_up_sync(0xffffffffu, incl0, o), y1 = __shfl_up_sync(0xffffffffu, incl1, o);
        if (lane >= o) {
          incl0 += y0;
          incl1 += y1;
        }
      }
      incl0 += before;
      incl1 += __shfl_sync(0xffffffffu, incl0, 31);
      if (incl0 - c0 < need && incl0 >= need) {
        s_prefix = prefix | (uint32_t(top - lane) << shift);
        s_need = need - (incl0 - c0);
      }
      if (incl1 - c1 < need && incl1 >= need) {
        s_prefix = prefix | (uint32_t(top - 32 - lane) << shift);
        s_need = need - (incl1 - c1);
      }
    }
    __syncthreads();
  }
  const uint32_t cut = s_prefix;
  const int ties = want > 0 ? s_need : 0;  // how many keys equal to the cut are kept, the lowest slots first
  int base_keep = 0, base_tie = 0, phase = 0;
  for (int j0 = 0; j0 < len; j0 += kSelThreads, phase ^= 1) {
    const int j = j0 + tid;
    bool keep = false, tie = false;
    if (j < len) {
      if (j < lo || j >= hi) {
        keep = true;
      } else if (want > 0) {
        const uint32_t k = key_at(j);
        keep = k > cut;
        tie = k == cut;
      }
    }
    int n_tie, n_keep;
    const int tie_rank = base_tie + block_rank(tie, warp_count[phase][0], n_tie);
    keep |= tie && tie_rank < ties;
    const int rank = base_keep + block_rank(keep, warp_count[phase][1], n_keep);
    if (keep) kept[rank] = j;
    base_keep += n_keep;
    base_tie += n_tie;
  }
}

struct MoveArgs {
  char *k, *v;
  long long k_page_bytes, v_page_bytes;
  float* weights;
  const int* kept;
  const int* to_table;
  int to_pages, Hkv, budget, row_bytes;
};

__global__ void __launch_bounds__(kMoveThreads)
paged_move_kernel(const MoveArgs a, const PagedBatch batch) {
  __shared__ long long src[kMoveRows], dst[kMoveRows];    // (page * 2^32 + slot), -1: nothing
  const int r = blockIdx.z, h = blockIdx.y, i0 = blockIdx.x * kMoveRows, tid = threadIdx.x;
  const int ps = 1 << batch.page_log2;
  after_previous();
  if (tid < kMoveRows) {
    const int i = i0 + tid;
    long long s = -1, t = -1;
    if (i < a.budget) {
      const int j = a.kept[((long long)r * a.Hkv + h) * a.budget + i];
      if (j >= 0) {
        const int from = __ldg(batch.table + (long long)r * batch.max_pages + (j >> batch.page_log2));
        const int to = __ldg(a.to_table + (long long)r * a.to_pages + (i >> batch.page_log2));
        if (unsigned(from) < unsigned(batch.n_pages) && unsigned(to) < unsigned(batch.n_pages)) {
          s = ((long long)from << 32) | (j & (ps - 1));
          t = ((long long)to << 32) | (i & (ps - 1));
        } else {
          paged_flag(batch);
        }
      }
    }
    src[tid] = s;
    dst[tid] = t;
    if (s >= 0)
      a.weights[((t >> 32) * a.Hkv + h) * ps + int(t & 0xffffffff)] = a.weights[((s >> 32) * a.Hkv + h) * ps + int(s & 0xffffffff)];
  }
  __syncthreads();
  const int nv = a.row_bytes / 16;
  const int total = kMoveRows * nv;
  for (int e = tid; e < total; e += kMoveThreads) {
    const int row = e / nv, c = (e % nv) * 16;
    const long long s = src[row], t = dst[row];
    if (s < 0) continue;
    const long long so = (long long)(h * ps + int(s & 0xffffffff)) * a.row_bytes + c;
    const long long to = (long long)(h * ps + int(t & 0xffffffff)) * a.row_bytes + c;
    const uint4 kk = *reinterpret_cast<const uint4*>(a.k + (s >> 32) * a.k_page_bytes + so);
    const uint4 vv = *reinterpret_cast<const uint4*>(a.v + (s >> 32) * a.v_page_bytes + so);
    *reinterpret_cast<uint4*>(a.k + (t >> 32) * a.k_page_bytes + to) = kk;
    *reinterpret_cast<uint4*>(a.v + (t >> 32) * a.v_page_bytes + to) = vv;
  }
}

}  // namespace
}  // namespace cb2

extern "C" int cb2_paged_evict(void* k_pages, void* v_pages, long long k_page_stride, long long v_page_stride, float* weights,
                               const int* block_table, const int* seq_lens, const int* new_table, int* kept, int* new_lens,
                               int R, int Hkv, int d, int page_size, int n_pages, int max_pages, int new_pages, int max_k,
                               int budget, int keep_first, int keep_last, int dtype, int* dev_status, void* stream) {
  using namespace cb2;
  if (!k_pages || !v_pages || !weights || !block_table || !seq_lens || !new_table || !kept || !new_lens) return CB2_NULL_PTR;
  if (R < 1 || R > 65535 || Hkv < 1 || Hkv > 65535 || d < 8 || d > 128 || d % 8 || n_pages < 1 || max_pages < 1 || new_pages < 1)
    return CB2_BAD_SHAPE;
  if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1)) || max_k < 1 || max_k > (1 << 30) ||
      int64_t(max_pages) * page_size < max_k)
    return CB2_BAD_SHAPE;
  // (the kernels step over the budget in 32 bits)
  if (budget < 1 || budget > (1 << 30) || keep_first < 0 || keep_last < 0 || int64_t(keep_first) + keep_last > budget || int64_t(new_pages) * page_size < budget)
    return CB2_BAD_SHAPE;
  const long long page = (long long)Hkv * page_size * d;
  if (k_page_stride < page || v_page_stride < page) return CB2_BAD_SHAPE;
  if (dtype != CB2_BF16 && dtype != CB2_F32) return CB2_UNSUPPORTED_DTYPE;
  const int esz = dtype == CB2_BF16 ? 2 : 4;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(weights) || k_page_stride * esz % 16 || v_page_stride * esz % 16) return CB2_BAD_ALIGN;
  int page_log2 = 0;
  while ((1 << page_log2) < page_size) ++page_log2;
  const PagedBatch batch{block_table, seq_lens, nullptr, R, max_pages, n_pages, page_log2, 0, 0, max_k, dev_status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const EvictArgs e{weights, Hkv, budget, keep_first, keep_last, kept, new_lens, max_k < kMostHeld ? max_k : kMostHeld};
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(paged_select_kernel), kMostHeld * 4, done)) return CB2_LAUNCH_FAIL;
  paged_select_kernel<<<dim3(Hkv, R), kSelThreads, size_t((e.held + 3) & ~3) * 4, st>>>(e, batch);
  CB2_LAUNCH_CHECK();
  const MoveArgs m{static_cast<char*>(k_pages), static_cast<char*>(v_pages), k_page_stride * esz, v_page_stride * esz, weights,
                   kept, new_table, new_pages, Hkv, budget, d * esz};
  return launch_next(paged_move_kernel, dim3((budget + kMoveRows - 1) / kMoveRows, Hkv, R), kMoveThreads, st, m, batch);
}

// What a ragged batch's index tensors say about a request, clamped so that no value in them, the extremes of int
// included, leads out of bounds.  Plain arithmetic: a host compiler takes it, too.
#pragma once

#ifdef __CUDACC__
#define CB2_ANYWHERE __host__ __device__ __forceinline__
#else
#define CB2_ANYWHERE inline
#endif

namespace cb2 {

struct PagedReq {
  int t0, n, len;     // first row in q, new tokens, cached keys
};

CB2_ANYWHERE int paged_clamped(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Rows [c0, c1) of n_tokens, at most max_q of them, and len cached keys, at most max_k; false if a value was out of range.
CB2_ANYWHERE bool paged_clamp(int c0, int c1, int len, int n_tokens, int max_q, int max_k, PagedReq* q) {
  q->t0 = paged_clamped(c0, 0, n_tokens);
  const int end = paged_clamped(c1, q->t0, n_tokens);      // before the difference, which may pass 32 bits
  q->n = end - q->t0 < max_q ? end - q->t0 : max_q;
  q->len = paged_clamped(len, 0, max_k);
  return q->t0 == c0 && q->t0 + q->n == c1 && q->len == len;
}

}  // namespace cb2

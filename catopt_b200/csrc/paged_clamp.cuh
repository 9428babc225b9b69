// What a ragged batch's index tensors say about a request, clamped so that no value in them, the extremes of int
// included, leads out of bounds; and whether an output lies on an operand.  Plain arithmetic: a host compiler takes it, too.
#pragma once

#include <cstdint>

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

// Whether the `bytes` from `to` on meet rows [n, heads, d] of `size` bytes an element with these strides (elements).  Exact
// along the longer stride; what lies between the rows of the shorter one counts as met.
inline bool paged_rows_meet(const void* at, long long n, long long token, long long heads, long long head, int d, int size, const void* to,
                            long long bytes) {
  if (n < 1 || heads < 1 || bytes < 1) return false;
  if (n > 1 && heads > 1 && head > token) {
    const long long a = n, b = token;
    n = heads, token = head, heads = a, head = b;
  }
  if (token == 0) n = 1;
  const long long step = n > 1 ? token * size : 1, run = ((heads - 1) * head + d) * size;
  const long long off = (long long)(reinterpret_cast<uintptr_t>(to) - reinterpret_cast<uintptr_t>(at));
  const long long first = off - run < 0 ? 0 : (off - run) / step + 1;      // the first run that ends behind `to`
  return first < n && first * step < off + bytes;
}

}  // namespace cb2

// Which of a draft plan's bits a tree sets: one rule for the host, which plans chains, and for ft_draft_tree's kernel.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define FT_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FT_HOST_DEVICE inline
#endif

// A stretch of a K/V tile that tokens of one request see differently from tree to tree (ft_extend_plan.cu).
struct DraftSpan {
  int32_t bits;      // place of the first token's words in the extra table
  int32_t tokens;
  int32_t token0;    // the first token's number among the request's drafted ones
  int32_t bit0, bit1;
  int32_t pos0;      // position of bit0 less the request's cached tokens: below 0 are cached ones, the rest are drafted
  int32_t zero0, zero1;  // to eight ints, which are read as two times four
};

// Token k of the span, word by word from the last: emit(word, mask of the span's bits in it, those that the token sees).
// parent: -1 at a root, -2 of a padding token, which sees the cached tokens alone; depth: of each token.  A token of depth e sees
// position x (less the cached tokens) if e - window < x, where a window is, and x is cached or stands for an ancestor or itself.
// Ancestors come before their descendants, so one climb from the token to its root meets the words' bits in order.
template <typename Emit>
FT_HOST_DEVICE void draft_span_words(const DraftSpan& s, int k, int window, const int16_t* parent, const int16_t* depth, Emit emit) {
  const int i = s.token0 + k, mine = depth[i];
  int at = parent[i] == -2 ? -1 : i, at_depth = mine;
  for (int w = (s.bit1 - 1) >> 5; w >= s.bit0 >> 5; --w) {
    const int b0 = s.bit0 > 32 * w ? s.bit0 : 32 * w, b1 = s.bit1 < 32 * w + 32 ? s.bit1 : 32 * w + 32;
    const uint32_t mask = (b1 - 32 * w == 32 ? 0xffffffffu : (1u << (b1 - 32 * w)) - 1u) & ~((1u << (b0 - 32 * w)) - 1u);
    const int x0 = s.pos0 + (b0 - s.bit0), x1 = s.pos0 + (b1 - s.bit0);
    uint32_t bits = 0;
    const int first = window > 0 && mine - window + 1 > x0 ? mine - window + 1 : x0, last = x1 < 0 ? x1 : 0;
    if (first < last) {
      const int from = b0 - 32 * w + (first - x0), n = last - first;
      bits |= (n == 32 ? 0xffffffffu : (1u << n) - 1u) << from;
    }
    while (x1 > 0 && at >= x0 && at >= 0) {
      if (at < x1 && (window == 0 || mine - at_depth < window)) bits |= 1u << (b0 - 32 * w + (at - x0));
      at = parent[at];
      --at_depth;
    }
    emit(w, mask, bits);
  }
}

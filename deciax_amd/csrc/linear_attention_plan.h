// How linear attention cuts a sequence into segments, as plain constexpr functions: the kernels, the launches and the
// workspace have to agree for every length, and tests/test_linear_attention_plan.py checks on the CPU that they do.
#pragma once

namespace la {

// Up to STEP tokens (STEP_F32 in fp32) a sequence goes token by token, 1 to 2.4 us each, where a chunk takes the same for
// 1 token and 64. Measured at heads of 128 by 128: 32 of them 7.7 and 8.6 us at 5 and 6 tokens against 9.8 in a chunk, 24
// sequences 26.3 and 27.9 against 28.2; in fp32, 24 sequences of 8 tokens 31 against 57.
//
// Beyond, in chunks. A segment's end state needs its start state only at the end, so segments of a long sequence run side
// by side: their own part first, then the join, then their outputs, which is the work of the states twice. One segment up
// to ONE tokens: with 640, 12 sequences of 700 take 148 us instead of 88, and one of them 39 instead of 47. No shorter
// segments than LEAST: of 256, 320 and 384, one sequence of 2111 tokens (heads of 256 by 256) takes 79, 79 and 86 us, one
// of 1024 (128 by 128) 42, 41 and 50, 12 of 517 to 16384 tokens 675, 661 and 654, 30 of 300 to 3000 558, 522 and 503.
// Up to 16 of them: 8192 tokens take 127 us (148 with 8, 149 with 32), 65536 806 (1030, 860). With keys of 256 dimensions
// a CU holds one workgroup and not two, and 8 fill it: 8192 tokens 194 us (222 with 16), 30000 635 (676).
// All of it goes by a sequence's own length, never by the batch it is in.
constexpr int STEP = 6, STEP_F32 = 8, ONE = 768, LEAST = 320, MOST_SEGMENTS = 16;

struct Segments {
  int tokens, count;  // a segment's tokens, a multiple of 64
};

// The most segments of any sequence of keys of k_dim dimensions.
constexpr int limit(int k_dim) { return k_dim == 256 ? MOST_SEGMENTS / 2 : MOST_SEGMENTS; }

// The most segments of any length up to max_len.
constexpr int most_segments(int max_len, int limit) {
  if (max_len <= ONE) return 1;
  const int n = (int)(((long)max_len + LEAST - 1) / LEAST);
  return n < limit ? n : limit;
}

constexpr Segments segments(int len, int limit) {
  if (len <= ONE) return {ONE, 1};
  const int most = most_segments(len, limit), tokens = (int)((((long)len + most - 1) / most + 63) & ~63L);
  return {tokens, (int)(((long)len + tokens - 1) / tokens)};
}

}  // namespace la

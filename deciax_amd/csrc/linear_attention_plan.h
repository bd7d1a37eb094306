// How linear attention cuts a sequence into segments, as plain constexpr functions: the kernels, the launches and the
// workspace have to agree for every length, and tests/test_linear_attention_plan.py checks on the CPU that they do.
#pragma once

namespace la {

// Up to STEP tokens (STEP_F32 in fp32) a sequence goes token by token, 1 to 2.4 us each, where a chunk takes the same for
// 1 token and 64. Measured at 32 heads of 128 by 128: 5 and 6 tokens 7.6 and 8.5 us against 8.0 and 8.1 in a chunk, 24
// sequences of them 26.9 and 28.4 against 28.7 and 27.8; in fp32, 8 tokens 9.8 against 9.5, 24 sequences 31 against 54.
//
// Beyond, in chunks. A segment's end state needs its start state only at the end, so segments of a long sequence run side
// by side: their own part first, then the join, then their outputs, which is the work of the states twice. One segment up
// to ONE tokens: with 640, 12 sequences of 700 take 149 us instead of 88, and one of them 39 instead of 46. No shorter
// segments than LEAST: of 256, 320 and 384, one sequence of 2111 tokens (heads of 256 by 256) takes 79, 80 and 87 us, one
// of 1024 (128 by 128) 40, 40 and 49, 12 of 517 to 16384 tokens 669, 669 and 655, 30 of 300 to 3000 567, 530 and 502.
// Up to 16 of them: 8192 tokens take 121 us (147 with 8, 148 with 32), 65536 827 (1074, 853). With keys of 256 dimensions
// a CU holds one workgroup and not two, and 8 fill it: 8192 tokens 194 us (221 with 16), 30000 658 (685).
//
// fp32 has the same cut, a compromise of the same kind. ONE: a sequence of 700 tokens takes 99 us, 60 in segments of 192 or
// more, but 12 of them 300 and 465. LEAST, of 192, 320 and 512: one sequence of 2111 tokens 136, 144 and 158 us (4 heads of 64
// by 64: 41, 57 and 74), 12 of 500 to 5000 1077, 1037 and 983. The most segments, of 8, 16 and 32: 8192 tokens 408, 418
// and 464 us, 4 heads of 64 by 64 156, 86 and 62, 6 sequences of 4000 to 9000 at 8 heads of 64 by 64 214, 155 and 146; at
// keys of 256, of 4, 8 and 16, 812, 758 and 782.
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

// How linear attention cuts a sequence into segments, as plain constexpr functions: the kernels, the launches and the
// workspace have to agree for every length, and tests/test_linear_attention_plan.py checks on the CPU that they do.
#pragma once

namespace la {

// Up to STEP tokens a sequence goes token by token (its state's bytes are what it costs), beyond in chunks of its
// segments. A segment's end state needs its start state only at the end, so segments run side by side: their own part
// first, then the join, then their outputs.
constexpr int STEP = 16, ONE = 512, LEAST = 384, MOST_SEGMENTS = 16;

struct Segments {
  int tokens, count;  // a segment's tokens, a multiple of 64
};

constexpr Segments segments(int len) {
  if (len <= ONE) return {ONE, 1};
  const int even = (int)(((long)len + MOST_SEGMENTS - 1) / MOST_SEGMENTS), whole = (even + 63) & ~63;
  const int tokens = whole > LEAST ? whole : LEAST;
  return {tokens, (int)(((long)len + tokens - 1) / tokens)};
}

// The most segments of any length up to max_len: not that of max_len itself.
constexpr int most_segments(int max_len) {
  if (max_len <= ONE) return 1;
  const int n = (int)(((long)max_len + LEAST - 1) / LEAST);
  return n < MOST_SEGMENTS ? n : MOST_SEGMENTS;
}

}  // namespace la

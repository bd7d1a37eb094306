// How attention over the 4-bit cache splits a sequence's keys, and the sizes that the host lays out for it, as plain
// constexpr functions: the kernels, the launches and the workspace have to agree for every size, and
// tests/test_kv4_plan.py checks on the CPU that they do.
#pragma once

namespace kv4 {

// A sequence's keys [lo, ctx) in `count` spans of `keys`.
struct Spans {
  int lo, keys, count;
};

// Keys of a span at least; spans of a sequence, and rows of all its spans together, at most (a row's part of a span is
// written and read in 8 D bytes, where 512 keys have 544 D). With spans of 256 keys one sequence of 2111 takes 13.6 us
// instead of 16.2, but 16 of 8000 72 instead of 61 and 64 of 4000 146 instead of 127.
constexpr int SPAN = 512, MAX_SPANS = 32, SPLIT_ROWS = 4096;
// Rows from here on have one span: no parts, and nothing to join.
constexpr int MOST_SPLIT_ROWS = SPLIT_ROWS / 2;

constexpr int most_spans(int rows) {
  const int most = SPLIT_ROWS / (rows > 0 ? rows : 1);
  return most < 1 ? 1 : most > MAX_SPANS ? MAX_SPANS : most;
}

constexpr Spans spans(int ctx, int n, int rows, int window) {
  int lo = window > 0 && ctx - n - window + 1 > 0 ? ctx - n - window + 1 : 0;
  lo &= ~63;
  const int len = ctx - lo, most = most_spans(rows);
  if (len == 0) return {lo, SPAN, 1};
  const int wanted = len / SPAN < most ? (len + SPAN - 1) / SPAN : most;
  // all of len over the spans wanted, one included, in whole turns of kv4_attn_kernel's waves
  const int keys = ((len + wanted - 1) / wanted + 127) & ~127;
  return {lo, keys, 1 + (len - 1) / keys};
}

// Rows of a KV head up to which their scores are kept for the accumulated weights (4 bytes a row and slot of workspace),
// instead of computed again. 24 sequences over 3000 slots, 8 heads of 256, attention with weights: 2 rows 48 and 80 us, 16
// rows 70 and 91; 28 rows would gain 133 -> 114 for 112 bytes a slot, near the 136 of the key itself.
constexpr int SCORE_ROWS = 16;

// Sizes that depend on the largest lengths alone: rows and partial rows per (sequence, kv head), splits; rows and slots
// of kept scores. A shorter sequence may have more splits than a longer one, and fewer rows more parts.
struct Plan {
  int part_rows, max_rows, max_splits, score_rows, score_slots;
};

constexpr Plan attn_plan(int max_seq_len, int max_ctx, int group, int window) {
  Plan p{};
  p.max_rows = max_seq_len * group;
  // a window's span starts at a multiple of 64 below it and ends with the newest tokens
  const long seen = window > 0 ? (long)window + 64 + max_seq_len : max_ctx;
  const long len = seen < max_ctx ? seen : max_ctx, most = (len + SPAN - 1) / SPAN;
  p.max_splits = most < 1 ? 1 : most > MAX_SPANS ? MAX_SPANS : (int)most;
  const long rows = (long)p.max_splits * p.max_rows;
  p.part_rows = p.max_splits == 1 ? 0 : (int)(rows < SPLIT_ROWS ? rows : SPLIT_ROWS);
  p.score_rows = p.max_rows < SCORE_ROWS ? p.max_rows : SCORE_ROWS;
  p.score_slots = (max_ctx + 63) & ~63;  // whole steps
  return p;
}

}  // namespace kv4

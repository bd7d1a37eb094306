// Writing rows into the 4-bit cache, reading them back, and eviction by accumulated attention weight.
#include "kv4.h"

namespace {

using namespace kv4;

constexpr int THREADS = 256;

template <typename T>
DX_DEVICE void load8(const T *p, float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = lo_bf(w[i]);
      x[2 * i + 1] = hi_bf(w[i]);
    }
  } else {
    const floatx4 a = *reinterpret_cast<const floatx4 *>(p), b = *reinterpret_cast<const floatx4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  }
}

// Eight values a thread: four neighbouring lanes share a block, and its largest value crosses them in two exchanges.
DX_DEVICE void store_block(const float (&x)[8], uint8_t *codes, uint8_t *scales, long at) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1, 64));
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2, 64));
  const uint32_t byte = scale_byte(amax);
  if (at < 0) return;
  *reinterpret_cast<uint32_t *>(codes + at / 2) = byte == 255 ? 0u : encode8(x, scale_of(byte));
  if (at % 32 == 0) scales[at / 32] = (uint8_t)byte;
}

// An item is eight values of k and the same eight of v. Items go by blocks of BLOCK tokens, by head, by token: a head's
// rows of neighbouring slots, its scales and positions, are then written together (token by token a line of 128 bytes of
// scales was written 8 bytes at a time by 16 workgroups). A thread takes ITER items, all loads of one kind before the next,
// since each waits for the one before: lengths, page, rows.
// Bound: memory. 12 states, 50545 tokens of 8 heads of 256, bf16: written in 128 us (524 MB, 4.1 TB/s, where a copy reaches
// 5.0), read back in 83 us (6.3 TB/s: what was just written). 48 tokens: 3.7 and 3.2 us, a launch and four loads in turn.
struct Item {
  int slot, col;
  long row, at;  // the packed row (-1: none), the place in the cache (-1: none)
};

// False for a workgroup behind its sequence's last row.
template <int ITER, int BLOCK>
DX_DEVICE bool find_items(const Kv4Cache &c, const Kv4Batch &q, Item (&item)[ITER]) {
  const int b = blockIdx.y;
  const Sequence s = sequence(q, b, c.shift);
  const int32_t *table = q.table + (long)b * q.table_width;
  const uint32_t head_items = c.d / 8, row_items = c.hkv * head_items;
  if (blockIdx.x * ITER * THREADS >= (s.n + BLOCK - 1) / BLOCK * (BLOCK * row_items)) return false;
  int page[ITER];
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const uint32_t i = (blockIdx.x * ITER + k) * THREADS + threadIdx.x;
    const uint32_t block = i / (BLOCK * row_items), r = i - block * (BLOCK * row_items);
    const uint32_t g = r / (BLOCK * head_items), x = r - g * (BLOCK * head_items);
    const int t = (int)(block * BLOCK + x / head_items);
    item[k].col = (int)(g * c.d + x % head_items * 8);
    item[k].slot = s.ctx - s.n + t;
    item[k].row = s.start + t;
    if (t >= s.n || item[k].row < 0 || item[k].row >= q.rows) item[k].row = -1;
    const bool placed = item[k].row >= 0 && item[k].slot >= 0;
    page[k] = placed ? table[item[k].slot >> c.shift] : -1;
  }
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int g = item[k].col / c.d, d = item[k].col % c.d;
    const long row = (((long)page[k] * c.hkv + g) << c.shift) + (item[k].slot & ((1 << c.shift) - 1));
    item[k].at = page[k] >= 0 && page[k] < c.pages ? row * c.d + d : -1;
  }
  return true;
}

template <typename T, int ITER, int BLOCK>
__global__ void __launch_bounds__(THREADS)
append_kernel(Kv4Cache c, Kv4Batch q, const T *__restrict__ k, const T *__restrict__ v,
              const int32_t *__restrict__ positions, long k_stride, long v_stride) {
  Item item[ITER];
  if (!find_items<ITER, BLOCK>(c, q, item)) return;
  float xk[ITER][8], xv[ITER][8];
  int pos[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const long row = max(item[i].row, 0L);  // rows are there: a call without any is not launched
    const int col = item[i].row >= 0 ? item[i].col : 0;
    load8(k + row * k_stride + col, xk[i]);
    load8(v + row * v_stride + col, xv[i]);
    pos[i] = positions[row];
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    if (item[i].at >= 0 && item[i].at % c.d == 0) c.pos[item[i].at / c.d] = pos[i];
    store_block(xk[i], c.k, c.ks, item[i].at);
    store_block(xv[i], c.v, c.vs, item[i].at);
  }
}

template <int ITER, int BLOCK>
__global__ void __launch_bounds__(THREADS)
read_kernel(Kv4Cache c, Kv4Batch q, uint16_t *__restrict__ k, uint16_t *__restrict__ v, long k_stride, long v_stride) {
  Item item[ITER];
  if (!find_items<ITER, BLOCK>(c, q, item)) return;
  uint32_t wk[ITER], wv[ITER], sk[ITER], sv[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const long at = max(item[i].at, 0L);
    wk[i] = *reinterpret_cast<const uint32_t *>(c.k + at / 2);
    wv[i] = *reinterpret_cast<const uint32_t *>(c.v + at / 2);
    sk[i] = c.ks[at / 32];
    sv[i] = c.vs[at / 32];
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    if (item[i].row < 0) continue;
    const bool there = item[i].at >= 0;
    const u32x4 none = {0, 0, 0, 0};
    *reinterpret_cast<u32x4 *>(k + item[i].row * k_stride + item[i].col) = there ? decode8(wk[i], scale_of(sk[i])) : none;
    *reinterpret_cast<u32x4 *>(v + item[i].row * v_stride + item[i].col) = there ? decode8(wv[i], scale_of(sv[i])) : none;
  }
}

// ------------------------------------------------------------------------------------------ eviction

constexpr int SEL_THREADS = 1024, SEL_WAVES = SEL_THREADS / 64;

// A weight as a whole number that orders as it does: -0 equals 0, and a NaN is above all numbers.
constexpr uint32_t PROTECTED = 0xffffffffu;
DX_DEVICE uint32_t order(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return PROTECTED - 1;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The slots one (sequence, kv head) keeps, ascending, into list[0, kept). One workgroup; thread t holds slots
// i 1024 + t. The kept-th largest key is found bit by bit from the top: a round counts the keys at or above a
// candidate with one compare an item and the wave's population counts, no memory but one number a wave. ITEMS = 0
// reads the weights again every round, for spans beyond the registers. A slot without a page has the key of no slot.
// Bound: the 32 rounds, one after the other, of one workgroup: 11 us for 2900 slots, 30 us for up to 16384.
template <int ITEMS>
__global__ void __launch_bounds__(SEL_THREADS)
select_kernel(const float *__restrict__ weights, long w_seq, long w_head, const int32_t *__restrict__ table, int width,
              int pages, int shift, const int32_t *__restrict__ ctx_len, int max_ctx, int keep, int recent,
              int32_t *__restrict__ list, int32_t *__restrict__ out_len) {
  __shared__ int counts[2][SEL_WAVES];
  __shared__ uint32_t spread[ITEMS ? ITEMS : 16][SEL_WAVES];
  const int g = blockIdx.x, b = blockIdx.y, hkv = gridDim.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ctx = min(max(ctx_len[b], 0), max_ctx);
  int32_t *mine = list + ((long)b * hkv + g) * keep;
  const float *w = weights + b * w_seq + g * w_head;
  const int32_t *page_of = table + (long)b * width;
  auto no_page = [&](int page) { return page < 0 || page >= pages; };
  int gone = 0;  // whether some slot has no page
  const int guard = ctx - recent;  // slots from here on are kept
  const int rounds = (ctx + SEL_THREADS - 1) / SEL_THREADS;
  auto fetch = [&](int i) -> uint32_t {  // 0: no slot; order() of a number is never 0
    const int slot = i * SEL_THREADS + tid, at = min(slot, ctx - 1);
    const uint32_t x = max(order(w[at]), 1u);  // no branch: a thread's loads are on their way at once
    return slot >= ctx ? 0u : slot >= guard ? PROTECTED : x;
  };
  auto fetch_there = [&](int i) -> uint32_t {
    const uint32_t x = fetch(i);
    return no_page(page_of[min(i * SEL_THREADS + tid, ctx - 1) >> shift]) ? 0u : x;
  };
  uint32_t key[ITEMS ? ITEMS : 1];
  if (ctx == 0) {
    if (g == 0 && tid == 0) out_len[b] = 0;
    return;
  }
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) key[i] = fetch(i);
  }
  for (int p = tid; p << shift < ctx; p += SEL_THREADS) gone |= no_page(page_of[p]);
  gone = __syncthreads_or(gone);
  if (!gone && ctx <= keep) {
    if (g == 0 && tid == 0) out_len[b] = ctx;
    for (int i = tid; i < ctx; i += SEL_THREADS) mine[i] = i;
    return;
  }
  // waves' numbers to every wave; `turn` alternates, so one barrier a sum is enough
  auto total = [&](int c, int turn) {
    if (lane == 0) counts[turn][wave] = c;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int j = 0; j < SEL_WAVES; ++j) sum += counts[turn][j];
    return sum;
  };
  int present = ctx;
  if (gone) {
    int c = 0;
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int at = min(i * SEL_THREADS + tid, ctx - 1);
        key[i] = no_page(page_of[at >> shift]) ? 0u : key[i];
        c += __popcll(__ballot(key[i] != 0));
      }
    } else {
      for (int i = 0; i < rounds; ++i) c += __popcll(__ballot(fetch_there(i) != 0));
    }
    present = total(c, 0);
  }
  auto count = [&](uint32_t least) {  // a wave's keys from `least` on
    int c = 0;
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) c += __popcll(__ballot(key[i] >= least));
    } else if (gone) {
      for (int i = 0; i < rounds; ++i) c += __popcll(__ballot(fetch_there(i) >= least));
    } else {
      for (int i = 0; i < rounds; ++i) c += __popcll(__ballot(fetch(i) >= least));
    }
    return c;
  };
  const int kept = min(present, keep);
  if (g == 0 && tid == 0) out_len[b] = kept;
  uint32_t least = 0;  // the kept-th largest key, or that of no slot where all are kept
  bool found = present == kept;
  int above = found ? kept : 0;
  for (int bit = 31; bit >= 0 && !found; --bit) {
    const uint32_t cand = least | (1u << bit);
    const int c = total(count(cand), bit & 1);
    if (c >= kept) least = cand;
    if (c == kept) {  // these are they
      least = cand - 1;
      above = kept;
      found = true;
    }
  }
  // least + 1 is a number: as many keys as are kept and no more are PROTECTED, and with so many the search has ended
  if (!found) above = total(count(least + 1), 1);
  const int ties = kept - above;  // of the keys that equal `least`, the first in slot order
  // Ranks: every wave its counts of both kinds for each 1024 slots, ITEMS (or 16) of those at a time, then sums over the
  // waves before it and the slots before those. A wave of 64 neighbouring slots takes two ballots.
  constexpr int SPREAD = ITEMS ? ITEMS : 16;
  int tied = 0, done = 0;
  const uint64_t lower = (1ull << lane) - 1;
  for (int i0 = 0; i0 < rounds; i0 += SPREAD) {
    uint32_t k[SPREAD];
#pragma unroll
    for (int i = 0; i < SPREAD; ++i) {
      if constexpr (ITEMS > 0) k[i] = key[i];
      else k[i] = gone ? fetch_there(i0 + i) : fetch(i0 + i);
      const uint64_t eq = __ballot(k[i] == least && k[i] != 0), gt = __ballot(k[i] > least);
      if (lane == 0) spread[i][wave] = (uint32_t)__popcll(gt) << 16 | (uint32_t)__popcll(eq);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SPREAD; ++i) {
      uint32_t sum = spread[i][lane & (SEL_WAVES - 1)];
#pragma unroll
      for (int off = 1; off < SEL_WAVES; off *= 2) {
        const uint32_t under = __shfl_up(sum, off, SEL_WAVES);
        sum += (lane & (SEL_WAVES - 1)) >= off ? under : 0;
      }
      const uint32_t all = __builtin_amdgcn_readlane(sum, SEL_WAVES - 1);
      const uint32_t under = wave > 0 ? __builtin_amdgcn_readlane(sum, wave - 1) : 0;
      const bool is_eq = k[i] == least && k[i] != 0, is_gt = k[i] > least;
      const uint64_t eq = __ballot(is_eq), gt = __ballot(is_gt);
      const int eq_rank = tied + (int)(under & 0xffff) + __popcll(eq & lower);
      // ranks among the kept: greater ones before, and the tied ones before that are within the quota
      const int rank = done + (int)(under >> 16) + __popcll(gt & lower) + min(eq_rank, ties);
      if (is_gt || (is_eq && eq_rank < ties)) mine[rank] = (i0 + i) * SEL_THREADS + tid;
      tied += (int)(all & 0xffff);
      done += (int)(all >> 16);
    }
    __syncthreads();
  }
}

// Kept rows to their new pages: 16 bytes of codes a thread, the row's scales, position and weight by one of its threads
// each. Every step (slot, pages, rows) waits for the one before, so a thread takes four rows' steps together.
// 12 sequences cut to 4096 slots, 8 heads of 256: 47 to 62 us for 210 MB, rows of 128 bytes from anywhere.
template <int D>
__global__ void __launch_bounds__(THREADS)
move_kernel(Kv4Cache c, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ out_table,
            int out_width, const int32_t *__restrict__ out_len, int keep, const int32_t *__restrict__ list,
            const float *__restrict__ weights, long w_seq, long w_head, float *__restrict__ out_weights, long o_seq,
            long o_head) {
  constexpr int CHUNKS = D / 32, LANES = 2 * CHUNKS;  // 16-byte chunks of K's row, then of V's
  constexpr int ROWS = THREADS / LANES, ITER = 4;
  const int g = blockIdx.y, b = blockIdx.z;
  const int kept = out_len[b];
  const int32_t *from = table + (long)b * width, *to = out_table + (long)b * out_width;
  const int32_t *mine = list + ((long)b * c.hkv + g) * keep;
  const int l = threadIdx.x % LANES, chunk = l % CHUNKS;
  const bool is_k = l < CHUNKS;
  uint8_t *codes = is_k ? c.k : c.v, *scales = is_k ? c.ks : c.vs;
  if (blockIdx.x * ITER * ROWS >= keep) return;
  int j[ITER], slot[ITER];
  long src[ITER], dst[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    j[i] = (blockIdx.x * ITER + i) * ROWS + threadIdx.x / LANES;
    slot[i] = mine[max(min(j[i], kept - 1), 0)];
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const bool there = j[i] < kept;
    src[i] = there ? row_of(c, from, g, slot[i]) : -1;
    dst[i] = there ? row_of(c, to, g, j[i]) : -1;
  }
  u32x4 x[ITER];
  uint64_t sc[ITER];
  int pos[ITER];
  float w[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const long at = max(src[i], 0L);
    x[i] = *reinterpret_cast<const u32x4 *>(codes + at * (D / 2) + chunk * 16);
    if constexpr (D == 256) sc[i] = *reinterpret_cast<const uint64_t *>(scales + at * CHUNKS);
    else if constexpr (D == 128) sc[i] = *reinterpret_cast<const uint32_t *>(scales + at * CHUNKS);
    else sc[i] = *reinterpret_cast<const uint16_t *>(scales + at * CHUNKS);
    pos[i] = c.pos[at];
    w[i] = j[i] < kept ? weights[b * w_seq + g * w_head + slot[i]] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    if (l == 0 && j[i] < keep) out_weights[b * o_seq + g * o_head + j[i]] = w[i];
    if (src[i] < 0 || dst[i] < 0) continue;
    *reinterpret_cast<u32x4 *>(codes + dst[i] * (D / 2) + chunk * 16) = x[i];
    if (chunk == 0) {
      if constexpr (D == 256) *reinterpret_cast<uint64_t *>(scales + dst[i] * CHUNKS) = sc[i];
      else if constexpr (D == 128) *reinterpret_cast<uint32_t *>(scales + dst[i] * CHUNKS) = (uint32_t)sc[i];
      else *reinterpret_cast<uint16_t *>(scales + dst[i] * CHUNKS) = (uint16_t)sc[i];
    }
    if (l == CHUNKS) c.pos[dst[i]] = pos[i];
  }
}

}  // namespace

// One item a thread up to 2^19 items (twice what the card holds at once), two and blocks of 16 tokens beyond. Append and
// read of 8 heads of 256, us: 48 sequences of a token 7.2 and 7.8, 4 of 300 10.4 and 11.0, 2 of 1000 14.1 and 14.4; 4 of
// 1000 22.1 and 21.4, 12 of 517 to 16384 261 and 222 (four items 225, two without blocks 229).
static bool few_items(const Kv4Cache &c, const Kv4Batch &q) {
  return (long)q.num_seqs * q.max_seq_len * (c.hkv * c.d / 8) <= 1L << 19;
}
static dim3 item_grid(const Kv4Cache &c, const Kv4Batch &q, int iter, int tokens) {
  const long items = (long)(q.max_seq_len + tokens - 1) / tokens * tokens * (c.hkv * c.d / 8), block = (long)iter * THREADS;
  return dim3((unsigned)((items + block - 1) / block), q.num_seqs);
}

template <typename T>
static void append(const Kv4Cache &c, const Kv4Batch &q, const void *k, const void *v, const int32_t *positions,
                   long k_stride, long v_stride, hipStream_t s) {
  const T *kt = static_cast<const T *>(k), *vt = static_cast<const T *>(v);
  if (few_items(c, q))
    append_kernel<T, 1, 1><<<item_grid(c, q, 1, 1), dim3(THREADS), 0, s>>>(c, q, kt, vt, positions, k_stride, v_stride);
  else
    append_kernel<T, 2, 16><<<item_grid(c, q, 2, 16), dim3(THREADS), 0, s>>>(c, q, kt, vt, positions, k_stride, v_stride);
}

hipError_t dx_kv4_append_launch(const Kv4Cache &c, const Kv4Batch &q, const void *k, const void *v,
                                const int32_t *positions, long k_stride, long v_stride, bool f32, hipStream_t s) {
  if (f32) append<float>(c, q, k, v, positions, k_stride, v_stride, s);
  else append<uint16_t>(c, q, k, v, positions, k_stride, v_stride, s);
  return hipGetLastError();
}

hipError_t dx_kv4_read_launch(const Kv4Cache &c, const Kv4Batch &q, uint16_t *k, uint16_t *v, long k_stride,
                              long v_stride, hipStream_t s) {
  if (few_items(c, q))
    read_kernel<1, 1><<<item_grid(c, q, 1, 1), dim3(THREADS), 0, s>>>(c, q, k, v, k_stride, v_stride);
  else
    read_kernel<2, 16><<<item_grid(c, q, 2, 16), dim3(THREADS), 0, s>>>(c, q, k, v, k_stride, v_stride);
  return hipGetLastError();
}

hipError_t dx_kv4_evict_launch(const Kv4Cache &c, const int32_t *table, int width, const int32_t *out_table,
                               int out_width, const int32_t *ctx_len, int num_seqs, int max_ctx, int keep, int recent,
                               const float *weights, long w_seq, long w_head, float *out_weights, long o_seq,
                               long o_head, int32_t *out_len, int32_t *list, hipStream_t s) {
  const dim3 grid(c.hkv, num_seqs), block(SEL_THREADS);
  const int rounds = (max_ctx + SEL_THREADS - 1) / SEL_THREADS;
// By the slots that a thread holds. us of an eviction to 1000, in a graph: 2900 slots 15.3 with 4 a thread and 23.4 with
// 16, 14000 27 with 16 and 74 with 64, 60000 88 with 64 and 326 when read again every round.
#define SELECT(N) \
  select_kernel<N><<<grid, block, 0, s>>>(weights, w_seq, w_head, table, width, c.pages, c.shift, ctx_len, max_ctx,      \
                                          keep, recent, list, out_len)
  if (rounds <= 4) SELECT(4);
  else if (rounds <= 16) SELECT(16);
  else if (rounds <= 64) SELECT(64);
  else SELECT(0);
#undef SELECT
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
#define MOVE(D)                                                                                                     \
  move_kernel<D><<<dim3((keep + 4 * (THREADS * 16 / (D)) - 1) / (4 * (THREADS * 16 / (D))), c.hkv, num_seqs),       \
                   dim3(THREADS), 0, s>>>(c, table, width, out_table, out_width, out_len, keep, list,               \
                                          weights, w_seq, w_head, out_weights, o_seq, o_head)
  if (c.d == 64) MOVE(64);
  else if (c.d == 128) MOVE(128);
  else MOVE(256);
#undef MOVE
  return hipGetLastError();
}

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

// Eight values of k and the same eight of v a thread. Rows of one sequence are consecutive items.
template <typename T>
__global__ void __launch_bounds__(THREADS)
append_kernel(Kv4Cache c, Kv4Batch q, const T *__restrict__ k, const T *__restrict__ v,
              const int32_t *__restrict__ positions, long k_stride, long v_stride, int per_block) {
  const int b = blockIdx.y;
  const Sequence s = sequence(q, b, c.shift);
  const int32_t *table = q.table + (long)b * q.table_width;
  const uint32_t row_items = c.hkv * c.d / 8, items = s.n * row_items;  // below 2^31 for the longest sequence
  const uint32_t i0 = blockIdx.x * per_block;
  for (uint32_t i = i0 + threadIdx.x; i < min(i0 + per_block, items); i += THREADS) {
    const int t = (int)(i / row_items), col = (int)(i % row_items) * 8;
    const long row = s.start + t;
    const int slot = s.ctx - s.n + t, g = col / c.d, d = col % c.d;
    float xk[8] = {}, xv[8] = {};
    long at = -1;
    if (slot >= 0 && row >= 0 && row < q.rows) {
      load8(k + row * k_stride + col, xk);
      load8(v + row * v_stride + col, xv);
      const long r = row_of(c, table, g, slot);
      if (r >= 0) {
        at = r * c.d + d;
        if (d == 0) c.pos[r] = positions[row];
      }
    }
    store_block(xk, c.k, c.ks, at);
    store_block(xv, c.v, c.vs, at);
  }
}

__global__ void __launch_bounds__(THREADS)
read_kernel(Kv4Cache c, Kv4Batch q, uint16_t *__restrict__ k, uint16_t *__restrict__ v, long k_stride, long v_stride,
            int per_block) {
  const int b = blockIdx.y;
  const Sequence s = sequence(q, b, c.shift);
  const int32_t *table = q.table + (long)b * q.table_width;
  const uint32_t row_items = c.hkv * c.d / 8, items = s.n * row_items;  // below 2^31 for the longest sequence
  const uint32_t i0 = blockIdx.x * per_block;
  for (uint32_t i = i0 + threadIdx.x; i < min(i0 + per_block, items); i += THREADS) {
    const int t = (int)(i / row_items), col = (int)(i % row_items) * 8;
    const long row = s.start + t;
    const int slot = s.ctx - s.n + t, g = col / c.d, d = col % c.d;
    if (row < 0 || row >= q.rows) continue;
    u32x4 wk = {0, 0, 0, 0}, wv = {0, 0, 0, 0};
    const long r = slot >= 0 ? row_of(c, table, g, slot) : -1;
    if (r >= 0) {
      const long at = r * c.d + d;
      wk = decode8(*reinterpret_cast<const uint32_t *>(c.k + at / 2), scale_of(c.ks[at / 32]));
      wv = decode8(*reinterpret_cast<const uint32_t *>(c.v + at / 2), scale_of(c.vs[at / 32]));
    }
    *reinterpret_cast<u32x4 *>(k + row * k_stride + col) = wk;
    *reinterpret_cast<u32x4 *>(v + row * v_stride + col) = wv;
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
// reads the weights again every round, for spans beyond the registers.
template <int ITEMS>
__global__ void __launch_bounds__(SEL_THREADS)
select_kernel(const float *__restrict__ weights, long w_seq, long w_head, const int32_t *__restrict__ ctx_len,
              int max_ctx, int keep, int recent, int32_t *__restrict__ list, int32_t *__restrict__ out_len) {
  __shared__ int counts[2][SEL_WAVES];
  __shared__ int before[2][SEL_WAVES];
  const int g = blockIdx.x, b = blockIdx.y, hkv = gridDim.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ctx = min(max(ctx_len[b], 0), max_ctx), kept = min(ctx, keep);
  if (g == 0 && tid == 0) out_len[b] = kept;
  int32_t *mine = list + ((long)b * hkv + g) * keep;
  if (kept == ctx) {
    for (int i = tid; i < kept; i += SEL_THREADS) mine[i] = i;
    return;
  }
  const float *w = weights + b * w_seq + g * w_head;
  const int guard = ctx - recent;  // slots from here on are kept
  const int rounds = (ctx + SEL_THREADS - 1) / SEL_THREADS;
  auto fetch = [&](int i) -> uint32_t {  // 0: no slot; order() of a number is never 0
    const int slot = i * SEL_THREADS + tid;
    return slot >= ctx ? 0u : slot >= guard ? PROTECTED : max(order(w[slot]), 1u);
  };
  uint32_t key[ITEMS ? ITEMS : 1];
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) key[i] = fetch(i);
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
  uint32_t least = 0;  // the kept-th largest key
  int above = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = least | (1u << bit);
    int c = 0;
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) c += __popcll(__ballot(key[i] >= cand));
    } else {
      for (int i = 0; i < rounds; ++i) c += __popcll(__ballot(fetch(i) >= cand));
    }
    c = total(c, bit & 1);
    if (c >= kept) least = cand;
  }
  {
    int c = 0;
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) c += __popcll(__ballot(key[i] > least));
    } else {
      for (int i = 0; i < rounds; ++i) c += __popcll(__ballot(fetch(i) > least));
    }
    above = total(c, 1);
  }
  const int ties = kept - above;  // of the keys that equal `least`, the first in slot order
  // 1024 slots at a time, in order
  int tied = 0, done = 0;
  const uint64_t lower = (1ull << lane) - 1;
  auto place = [&](int i, uint32_t k) {
    const uint64_t eq = __ballot(k == least && k != 0), gt = __ballot(k > least);
    if (lane == 0) {
      counts[i & 1][wave] = __popcll(eq);
      before[i & 1][wave] = __popcll(gt);
    }
    __syncthreads();
    int eq_under = 0, gt_under = 0, eq_all = 0, gt_all = 0;
#pragma unroll
    for (int j = 0; j < SEL_WAVES; ++j) {
      const int e = counts[i & 1][j], a = before[i & 1][j];
      eq_under += j < wave ? e : 0;
      gt_under += j < wave ? a : 0;
      eq_all += e;
      gt_all += a;
    }
    const int eq_rank = tied + eq_under + __popcll(eq & lower);
    const bool is_eq = (eq >> lane) & 1, is_gt = (gt >> lane) & 1;
    // ranks among the kept: greater ones before, and the tied ones before that are within the quota
    const int at_rank = done + gt_under + __popcll(gt & lower) + min(eq_rank, ties);
    if (is_gt || (is_eq && eq_rank < ties)) mine[at_rank] = i * SEL_THREADS + tid;
    tied += eq_all;
    done += gt_all;
  };
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (i < rounds) place(i, key[i]);
  } else {
    for (int i = 0; i < rounds; ++i) place(i, fetch(i));
  }
}

// Kept rows to their new pages: 16 bytes a thread, then each row's scales, position and weight.
__global__ void __launch_bounds__(THREADS)
move_kernel(Kv4Cache c, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ out_table,
            int out_width, const int32_t *__restrict__ ctx_len, int max_ctx, int keep,
            const int32_t *__restrict__ list, const float *__restrict__ weights, long w_seq, long w_head,
            float *__restrict__ out_weights, long o_seq, long o_head, int per_block) {
  const int g = blockIdx.y, b = blockIdx.z;
  const int kept = min(min(max(ctx_len[b], 0), max_ctx), keep);
  const int32_t *from = table + (long)b * width, *to = out_table + (long)b * out_width;
  const int32_t *mine = list + ((long)b * c.hkv + g) * keep;
  const int chunks = c.d / 32, lanes = 2 * chunks;  // 16-byte chunks of K's row, then of V's
  const int j0 = blockIdx.x * per_block, j1 = min(j0 + per_block, keep);
  for (int i = threadIdx.x; i < (j1 - j0) * lanes; i += THREADS) {
    const int j = j0 + i / lanes, l = i % lanes, chunk = l % chunks;
    float w = 0.f;
    if (j < kept) {
      const int slot = mine[j];
      const long src = row_of(c, from, g, slot), dst = row_of(c, to, g, j);
      if (src >= 0 && dst >= 0) {
        uint8_t *codes = l < chunks ? c.k : c.v, *scales = l < chunks ? c.ks : c.vs;
        *reinterpret_cast<u32x4 *>(codes + dst * (c.d / 2) + chunk * 16) =
            *reinterpret_cast<const u32x4 *>(codes + src * (c.d / 2) + chunk * 16);
        scales[dst * chunks + chunk] = scales[src * chunks + chunk];
        if (l == 0) c.pos[dst] = c.pos[src];
      }
      if (l == 0) w = weights[b * w_seq + g * w_head + slot];
    }
    if (l == 0) out_weights[b * o_seq + g * o_head + j] = w;
  }
}

}  // namespace

hipError_t dx_kv4_append_launch(const Kv4Cache &c, const Kv4Batch &q, const void *k, const void *v,
                                const int32_t *positions, long k_stride, long v_stride, bool f32, hipStream_t s) {
  const long items = (long)q.max_seq_len * (c.hkv * c.d / 8);
  const int per_block = items <= 8 * THREADS ? THREADS : 4 * THREADS;
  const dim3 grid((unsigned)((items + per_block - 1) / per_block), q.num_seqs);
  if (f32)
    append_kernel<<<grid, dim3(THREADS), 0, s>>>(c, q, static_cast<const float *>(k), static_cast<const float *>(v),
                                                 positions, k_stride, v_stride, per_block);
  else
    append_kernel<<<grid, dim3(THREADS), 0, s>>>(c, q, static_cast<const uint16_t *>(k),
                                                 static_cast<const uint16_t *>(v), positions, k_stride, v_stride,
                                                 per_block);
  return hipGetLastError();
}

hipError_t dx_kv4_read_launch(const Kv4Cache &c, const Kv4Batch &q, uint16_t *k, uint16_t *v, long k_stride,
                              long v_stride, hipStream_t s) {
  const long items = (long)q.max_seq_len * (c.hkv * c.d / 8);
  const int per_block = items <= 8 * THREADS ? THREADS : 4 * THREADS;
  const dim3 grid((unsigned)((items + per_block - 1) / per_block), q.num_seqs);
  read_kernel<<<grid, dim3(THREADS), 0, s>>>(c, q, k, v, k_stride, v_stride, per_block);
  return hipGetLastError();
}

hipError_t dx_kv4_evict_launch(const Kv4Cache &c, const int32_t *table, int width, const int32_t *out_table,
                               int out_width, const int32_t *ctx_len, int num_seqs, int max_ctx, int keep, int recent,
                               const float *weights, long w_seq, long w_head, float *out_weights, long o_seq,
                               long o_head, int32_t *out_len, int32_t *list, hipStream_t s) {
  const dim3 grid(c.hkv, num_seqs), block(SEL_THREADS);
  const int rounds = (max_ctx + SEL_THREADS - 1) / SEL_THREADS;
#define SELECT(N) \
  select_kernel<N><<<grid, block, 0, s>>>(weights, w_seq, w_head, ctx_len, max_ctx, keep, recent, list, out_len)
  if (rounds <= 4) SELECT(4);
  else if (rounds <= 16) SELECT(16);
  else if (rounds <= 64) SELECT(64);
  else SELECT(0);
#undef SELECT
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int per_block = 64;
  move_kernel<<<dim3((keep + per_block - 1) / per_block, c.hkv, num_seqs), dim3(THREADS), 0, s>>>(
      c, table, width, out_table, out_width, ctx_len, max_ctx, keep, list, weights, w_seq, w_head, out_weights, o_seq,
      o_head, per_block);
  return hipGetLastError();
}

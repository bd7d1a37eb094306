// Attention of a sequence's newest tokens over its paged 4-bit cache, for gfx950.
//
// For query head h of KV head g and newest token i of n (own slot a = ctx - n + i):
//   t_j = scale q . k_j, softcap tanh(t_j / softcap) with a soft-cap, for the slots j <= a (with a window also j > a -
//   window and position_j > position_a - window); out = sum_j e^{t_j} v_j / sum_j e^{t_j}; a row that sees nothing is 0.
// All query heads of a KV head and all new tokens are rows of one product: row r is token r / G, head g G + r % G.
//
// kv4_attn_kernel: a workgroup owns 16 rows and one span of the keys, its four waves take 32 keys in turn, each with a
// softmax of its own (running maximum and sum in base 2), joined through LDS at the end; spans are joined by
// kv4_join_kernel. How keys are split follows from the sequence alone (`spans`), so a row's result does not depend on
// its batch.
//
// Per 32 keys, with 16x16x32 MFMAs (A: 16 rows, lane l row l % 16 and eight k of group l / 16; C: lane l column l % 16,
// rows 4 (l / 16) + r):
//   S^T = K Q^T. The order of the reduction is free as long as both sides share it: lane group l / 16 takes a whole
//     block of 32 dimensions, so a lane reads 16 bytes of one key, one scale, and feeds four products from registers.
//   A lane then holds, for query l % 16, keys 4 (l / 16) .. + 3 of both 16-key halves: as eight k of the product
//     O^T = V^T P^T they stay in the lane. P needs no exchange; the other operand wants V by columns, so V is decoded to
//     bf16 into LDS by rows and read back transposed (ds_read_b64_tr_b16: 16 lanes read four rows of 16 columns, lane i
//     gets column i).
// fp32 queries: what the cache stands for is exact in bf16, so the query and P alone are split, each in three bf16, and
// three products are summed in fp32.
#include "kv4.h"

namespace {

using namespace kv4;

constexpr int THREADS = 256, WAVES = 4;
constexpr float LOG2E = 1.4426950408889634f;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// How a sequence's keys are split: [lo, ctx) in `count` spans of `keys`.
struct Spans {
  int lo, keys, count;
};

constexpr int SPAN = 256, MAX_SPANS = 32, SPLIT_ROWS = 2048;

__host__ __device__ inline int most_spans(int rows) {
  const int most = SPLIT_ROWS / (rows > 0 ? rows : 1);
  return most < 1 ? 1 : most > MAX_SPANS ? MAX_SPANS : most;
}

__host__ __device__ inline Spans spans(int ctx, int n, int rows, int window) {
  int lo = window > 0 && ctx - n - window + 1 > 0 ? ctx - n - window + 1 : 0;
  lo &= ~63;
  const int len = ctx - lo, most = most_spans(rows);
  int keys = SPAN;
  while ((long)keys * most < len) keys *= 2;
  const int count = (len + keys - 1) / keys;
  return {lo, keys, count < 1 ? 1 : count};
}

DX_DEVICE floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The bf16 V tile of a wave: [32 keys][D], in 32-byte units (the 16 columns one transposed read takes of a row), unit u
// of row r at u ^ (r & 7) (r >> 1 at D 64, where a row is half the banks): the rows that a read touches fall on
// different banks.
template <int D>
DX_DEVICE int unit_at(int row, int unit) {
  if constexpr (D == 64) return row * D + ((unit ^ ((row >> 1) & 3)) << 4);
  else return row * D + ((unit ^ (row & 7)) << 4);
}

DX_DEVICE s16x4 read_transposed(const uint16_t *p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
#else
  return s16x4{};
#endif
}

// x = x0 + x1 + x2 in bf16 parts (24 bits and more), or its one rounding.
template <int NS>
DX_DEVICE void split8(const float (&x)[8], bf16x8 (&out)[NS]) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf2(rest[2 * i], rest[2 * i + 1]);
    out[n] = as_bf16x8(w);
    if (n + 1 < NS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rest[2 * i] -= lo_bf(w[i]);
        rest[2 * i + 1] -= hi_bf(w[i]);
      }
    }
  }
}

// Eight consecutive query elements as NS bf16 operands.
template <int NS>
DX_DEVICE void load_query(const void *base, long at, bf16x8 (&out)[NS]) {
  if constexpr (NS == 1) {
    out[0] = as_bf16x8(*reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(base) + at));
  } else {
    const float *p = static_cast<const float *>(base) + at;
    const floatx4 a = *reinterpret_cast<const floatx4 *>(p), b = *reinterpret_cast<const floatx4 *>(p + 4);
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    split8<NS>(x, out);
  }
}

// 32 keys of a page as a wave holds them before use.
template <int D>
struct Raw {
  static constexpr int KJ = D == 256 ? 2 : 1;   // K loads a 16-key half: lane l has key l % 16
  static constexpr int VJ = D / 64;             // V loads: lane l has 32 dimensions of one key, rows in order
  u32x4 k[2][KJ], v[VJ];
  uint32_t ks[2][KJ], vs[VJ];
};

template <int D>
DX_DEVICE void load_keys(Raw<D> &w, const Kv4Cache &c, long row0, int lane) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const long row = row0 + t * 16 + (lane & 15);
    if constexpr (D == 64) {  // a lane group takes half a block
      const u32x2 x = *reinterpret_cast<const u32x2 *>(c.k + row * 32 + (lane >> 4) * 8);
      w.k[t][0] = u32x4{x[0], x[1], 0, 0};
      w.ks[t][0] = c.ks[row * 2 + (lane >> 5)];
    } else {
#pragma unroll
      for (int j = 0; j < Raw<D>::KJ; ++j) {
        w.k[t][j] = *reinterpret_cast<const u32x4 *>(c.k + row * (D / 2) + (j * 4 + (lane >> 4)) * 16);
        w.ks[t][j] = c.ks[row * (D / 32) + j * 4 + (lane >> 4)];
      }
    }
  }
}

template <int D>
DX_DEVICE void load_values(Raw<D> &w, const Kv4Cache &c, long row0, int lane) {
#pragma unroll
  for (int j = 0; j < Raw<D>::VJ; ++j) {
    w.v[j] = *reinterpret_cast<const u32x4 *>(c.v + row0 * (D / 2) + (j * 64 + lane) * 16);
    w.vs[j] = c.vs[row0 * (D / 32) + j * 64 + lane];
  }
}

// Dimension of element 0 of lane group `grp` in the i-th product of a 16-key half (eight consecutive ones follow).
template <int D>
DX_DEVICE int product_dim(int i, int grp) {
  return D == 64 ? grp * 16 + i * 8 : ((i >> 2) * 4 + grp) * 32 + (i & 3) * 8;
}

// Scores of one 16-key half, in base 2. The product is read in the block that issued it: where a uniform branch came
// between the two, the compiler left out the wait states that a matrix result needs before it is read (a path of 6
// instead of 8 was there, and the last two of the four values were stale).
template <int D, int NS, bool CAP>
DX_DEVICE void key_scores(const Raw<D> &w, int t, const bf16x8 (&q)[D / 32][NS], float scale, float softcap,
                          float (&t2)[4]) {
  floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int j = D == 64 ? 0 : i >> 2;
    const bf16x8 a = as_bf16x8(decode8(w.k[t][j][i & 3], scale_of(w.ks[t][j])));
#pragma unroll
    for (int n = 0; n < NS; ++n) s = mfma16(a, q[i][n], s);
  }
  const float c = CAP ? scale / softcap : scale * LOG2E;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    t2[r] = s[r] * c;
    asm volatile("" : "+v"(t2[r]));  // here, not where a later block uses it
  }
  if constexpr (CAP) {
#pragma unroll
    for (int r = 0; r < 4; ++r) t2[r] = softcap * LOG2E * tanhf(t2[r]);
  }
}

template <int D, int NS, bool CAP>
__global__ void __launch_bounds__(THREADS) kv4_attn_kernel(Kv4Attn a) {
  constexpr int LPK = D / 32;  // lanes (blocks) a key in a V load
  __shared__ __attribute__((aligned(1024))) uint16_t tile[WAVES][STEP * D];
  __shared__ float join_m[WAVES][16], join_l[WAVES][16];
  const int g = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % a.max_splits, row_tile = blockIdx.x / a.max_splits;
  const Sequence s = sequence(a.q, b, a.c.shift);
  const int group = a.hq / a.c.hkv, rows = s.n * group, r0 = row_tile * 16;
  if (r0 >= rows) return;
  const Spans sp = spans(s.ctx, s.n, rows, a.slots);
  if (split >= sp.count) return;
  const int32_t *table = a.q.table + (long)b * a.q.table_width;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int k0 = sp.lo + split * sp.keys, k1 = min(s.ctx, k0 + sp.keys);

  const int row = r0 + col, token = row / group;
  const bool real = row < rows && s.start + token >= 0 && s.start + token < a.q.rows;
  const int own = s.ctx - s.n + token;  // the row's own slot
  bf16x8 q[D / 32][NS];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    if (real) load_query<NS>(a.query, (s.start + token) * a.q_stride + (long)(g * group + row % group) * D +
                                          product_dim<D>(i, grp), q[i]);
    else
#pragma unroll
      for (int n = 0; n < NS; ++n) q[i][n] = as_bf16x8(u32x4{0, 0, 0, 0});
  }
  int own_pos = 0;
  if (a.window > 0 && real && own >= 0) {
    const long r = row_of(a.c, table, g, own);
    own_pos = r >= 0 ? a.c.pos[r] : 0;
  }
  // keys below `open` are seen by every row of the tile, as far as the order of tokens goes
  const int open = s.ctx - s.n + r0 / group + 1;

  floatx4 o[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  uint16_t *mine = tile[wave];

  for (int kb = k0 + wave * STEP; kb < k1; kb += WAVES * STEP) {
    const long row0 = row_of(a.c, table, g, kb);
    if (row0 < 0) continue;
    Raw<D> w;
    load_keys<D>(w, a.c, row0, lane);
    load_values<D>(w, a.c, row0, lane);
    float t2[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float half[4];
      key_scores<D, NS, CAP>(w, t, q, a.scale, a.softcap, half);
#pragma unroll
      for (int r = 0; r < 4; ++r) t2[t * 4 + r] = half[r];
    }
    const bool masked = a.window > 0 || kb + STEP > open;
    uint32_t seen = 0xff;  // of this lane's eight keys
    if (masked) {
      seen = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = kb + t * 16 + grp * 4;
        int pos[4] = {0, 0, 0, 0};
        if (a.window > 0) {
          const int4 p = *reinterpret_cast<const int4 *>(a.c.pos + row0 + t * 16 + grp * 4);
          pos[0] = p.x, pos[1] = p.y, pos[2] = p.z, pos[3] = p.w;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bool see = key + r <= own;
          if (a.window > 0)
            see = see && key + r > own - a.slots && (long)pos[r] > (long)own_pos - a.window;
          if (!see) t2[t * 4 + r] = -INFINITY;
          seen |= (uint32_t)see << (t * 4 + r);
        }
      }
    }
    float top = t2[0];
#pragma unroll
    for (int r = 1; r < 8; ++r) top = fmaxf(top, t2[r]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m)) {
      const float next = fmaxf(m, top);
      const float f = next == -INFINITY ? 1.f : fast_exp2(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      p[r] = fast_exp2(t2[r] - base);
      l += p[r];
    }
    bf16x8 pb[NS];
    split8<NS>(p, pb);

    // V to LDS. Slots behind the sequence hold anything: zeros here. A block of NaN may stand behind a row's own token
    // too, where 0 NaN would reach the row: such blocks are zero here and added below to the rows that see them.
    uint64_t nan_blocks[Raw<D>::VJ];
    bool any_nan = false;
#pragma unroll
    for (int j = 0; j < Raw<D>::VJ; ++j) {
      const int key = j * (64 / LPK) + lane / LPK;
      u32x4 x = w.v[j];
      uint32_t byte = w.vs[j];
      if (masked) {
        const bool inside = kb + key < s.ctx, bad = byte == 255;
        nan_blocks[j] = __ballot(inside && bad);
        any_nan = any_nan || nan_blocks[j] != 0;
        if (!inside || bad) {
          x = u32x4{0, 0, 0, 0};
          byte = 127;
        }
      }
      const int unit = (lane % LPK) * 2;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x4 *>(mine + unit_at<D>(key, unit + (i >> 1)) + (i & 1) * 8) =
            decode8(x[i], scale_of(byte));
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint16_t *p0 = mine + unit_at<D>(grp * 4 + (col >> 2), i) + (col & 3) * 4;
      const uint16_t *p1 = mine + unit_at<D>(16 + grp * 4 + (col >> 2), i) + (col & 3) * 4;
      const s16x4 v0 = read_transposed(p0), v1 = read_transposed(p1);
      const bf16x8 vt = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int n = 0; n < NS; ++n) o[i] = mfma16(vt, pb[n], o[i]);
    }
    if (masked && any_nan) {
#pragma unroll
      for (int blk = 0; blk < LPK; ++blk) {
        int hit = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int key = (r >> 2) * 16 + grp * 4 + (r & 3);
          uint64_t bits = nan_blocks[0];
#pragma unroll
          for (int j = 1; j < Raw<D>::VJ; ++j) bits = key / (64 / LPK) == j ? nan_blocks[j] : bits;
          hit |= (int)((bits >> (key % (64 / LPK) * LPK + blk)) & 1) & (int)((seen >> r) & 1);
        }
        hit |= __shfl_xor(hit, 16, 64);
        hit |= __shfl_xor(hit, 32, 64);
        if (hit) {
          o[2 * blk] += NAN;
          o[2 * blk + 1] += NAN;
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the four waves' parts, through LDS: [16 rows][D] fp32 a wave, where its V tile was
  if (grp == 0) {
    join_m[wave][col] = m;
    join_l[wave][col] = l;
  }
  __syncthreads();
  float top = join_m[0][col];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) top = fmaxf(top, join_m[w][col]);
  const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - top);
  float *part = reinterpret_cast<float *>(mine);
  static_assert(sizeof(tile[0]) >= 16 * D * sizeof(float), "a wave's rows fit its V tile");
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    *reinterpret_cast<floatx4 *>(part + col * D + i * 16 + grp * 4) = o[i] * f;
  __syncthreads();

  const int valid = min(16, rows - r0);
  for (int i = tid; i < valid * (D / 4); i += THREADS) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float mm = join_m[0][r], ll = 0.f;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, join_m[w][r]);
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float lw = join_l[w][r], mw = join_m[w][r];
      ll += lw * (mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : fast_exp2(mw - mm));
      acc += *reinterpret_cast<const floatx4 *>(reinterpret_cast<const float *>(tile[w]) + r * D + d);
    }
    const int tok = (r0 + r) / group, h = g * group + (r0 + r) % group;
    const long unit = (long)b * a.c.hkv + g;
    if (sp.count == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      acc *= inv;
      const long out_row = s.start + tok;
      if (out_row >= 0 && out_row < a.q.rows) {
        const long at = out_row * a.out_stride + (long)h * D + d;
        if constexpr (NS == 1) {
          const u32x2 y = {pack_bf2(acc[0], acc[1]), pack_bf2(acc[2], acc[3])};
          *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + at) = y;
        } else {
          *reinterpret_cast<floatx4 *>(static_cast<float *>(a.out) + at) = acc;
        }
      }
      if (a.w_out && d == 0) a.lse[unit * a.max_rows + r0 + r] = mm + log2f(ll);
    } else {
      const long p = unit * a.part_rows + (long)split * rows + r0 + r;
      *reinterpret_cast<floatx4 *>(a.partial + p * D + d) = acc;
      if (d == 0) {
        a.stats[p * 2] = mm;
        a.stats[p * 2 + 1] = ll;
      }
    }
  }
}

// Spans of one row to its output, in their order: one wave a row, D / 64 dimensions a lane.
template <int D, int NS>
__global__ void __launch_bounds__(THREADS) kv4_join_kernel(Kv4Attn a) {
  constexpr int E = D / 64;
  const int g = blockIdx.y, b = blockIdx.z;
  const Sequence s = sequence(a.q, b, a.c.shift);
  const int group = a.hq / a.c.hkv, rows = s.n * group;
  const int r = blockIdx.x * WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= rows) return;
  const Spans sp = spans(s.ctx, s.n, rows, a.slots);
  if (sp.count == 1) return;
  const long unit = (long)b * a.c.hkv + g, first = unit * a.part_rows + r;
  float m = -INFINITY, l = 0.f, acc[E] = {};
  // the spans' statistics a lane each; 32 at most
  float ms = -INFINITY, ls = 0.f;
  if (lane < sp.count) {
    ms = a.stats[(first + (long)lane * rows) * 2];
    ls = a.stats[(first + (long)lane * rows) * 2 + 1];
  }
  m = wave_max(ms);
  const float f = ms == -INFINITY ? (ls == 0.f ? 0.f : 1.f) : fast_exp2(ms - m);
  l = wave_sum(ls * f);
  for (int i = 0; i < sp.count; ++i) {
    const float fi = __shfl(f, i, 64);
    const float *p = a.partial + (first + (long)i * rows) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += p[e] * fi;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long out_row = s.start + r / group;
  if (out_row >= 0 && out_row < a.q.rows) {
    const long at = out_row * a.out_stride + (long)(g * group + r % group) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (NS == 1) static_cast<uint16_t *>(a.out)[at + e] = f2bf(acc[e] * inv);
      else static_cast<float *>(a.out)[at + e] = acc[e] * inv;
    }
  }
  if (a.w_out && lane == 0) a.lse[unit * a.max_rows + r] = m + log2f(l);
}

// weights_out_j = weights_in_j (0 for the newest slots) + sum over the rows that see j of e^{t_j} / sum e^t. A wave owns
// 32 keys and walks all rows, so every sum has one owner and one order.
template <int D, int NS, bool CAP>
__global__ void __launch_bounds__(THREADS) kv4_weights_kernel(Kv4Attn a) {
  const int g = blockIdx.y, b = blockIdx.z;
  const Sequence s = sequence(a.q, b, a.c.shift);
  const int32_t *table = a.q.table + (long)b * a.q.table_width;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = a.hq / a.c.hkv, rows = s.n * group;
  const int kb = (blockIdx.x * WAVES + wave) * STEP;
  if (kb >= s.ctx) return;
  const long unit = (long)b * a.c.hkv + g;
  const long row0 = row_of(a.c, table, g, kb);
  const int lo = a.window > 0 ? s.ctx - s.n - a.slots + 1 : 0;
  float sum[8] = {};
  if (row0 >= 0 && kb + STEP > lo) {
    Raw<D> w;
    load_keys<D>(w, a.c, row0, lane);
    int pos[8] = {};
    if (a.window > 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int4 p = *reinterpret_cast<const int4 *>(a.c.pos + row0 + t * 16 + grp * 4);
        pos[t * 4] = p.x, pos[t * 4 + 1] = p.y, pos[t * 4 + 2] = p.z, pos[t * 4 + 3] = p.w;
      }
    }
    // the first row that can see a key here
    const int first = max(0, kb - (s.ctx - s.n)) * group;
    for (int r0 = first & ~15; r0 < rows; r0 += 16) {
      const int row = r0 + col, token = row / group, own = s.ctx - s.n + token;
      const bool real = row < rows && s.start + token >= 0 && s.start + token < a.q.rows;
      bf16x8 q[D / 32][NS];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        if (real) load_query<NS>(a.query, (s.start + token) * a.q_stride + (long)(g * group + row % group) * D +
                                              product_dim<D>(i, grp), q[i]);
        else
#pragma unroll
          for (int n = 0; n < NS; ++n) q[i][n] = as_bf16x8(u32x4{0, 0, 0, 0});
      }
      const float lse = real ? a.lse[unit * a.max_rows + row] : 0.f;
      int own_pos = 0;
      if (a.window > 0 && real && own >= 0) {
        const long r = row_of(a.c, table, g, own);
        own_pos = r >= 0 ? a.c.pos[r] : 0;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float t2[4];
        key_scores<D, NS, CAP>(w, t, q, a.scale, a.softcap, t2);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = kb + t * 16 + grp * 4 + r;
          bool see = real && key <= own;
          if (a.window > 0)
            see = see && key > own - a.slots && (long)pos[t * 4 + r] > (long)own_pos - a.window;
          sum[t * 4 + r] += see ? fast_exp2(t2[r] - lse) : 0.f;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int off = 1; off < 16; off *= 2) sum[i] += __shfl_xor(sum[i], off, 64);
  if (col < 8) {  // lane col of a group stores the group's key of that index
    const int key = kb + (col >> 2) * 16 + grp * 4 + (col & 3);
    float mine = sum[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mine = col == i ? sum[i] : mine;
    if (key < s.ctx) {
      const float old = key < s.ctx - s.n ? a.w_in[b * a.wi_seq + g * a.wi_head + key] : 0.f;
      a.w_out[b * a.wo_seq + g * a.wo_head + key] = old + mine;
    }
  }
}

template <int D, int NS, bool CAP>
hipError_t launch(const Kv4Attn &a, hipStream_t s) {
  const int tiles = (a.max_rows + 15) / 16;
  hipError_t e = hipSuccess;
  if (tiles > 0) {
    kv4_attn_kernel<D, NS, CAP><<<dim3(a.max_splits * tiles, a.c.hkv, a.q.num_seqs), dim3(THREADS), 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && tiles > 0 && a.max_splits > 1) {
    const int split_rows = min(a.max_rows, SPLIT_ROWS / 2);  // rows with more than one span
    kv4_join_kernel<D, NS><<<dim3((split_rows + WAVES - 1) / WAVES, a.c.hkv, a.q.num_seqs), dim3(THREADS), 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.w_out && a.q.max_ctx > 0) {
    kv4_weights_kernel<D, NS, CAP>
        <<<dim3((a.q.max_ctx + WAVES * STEP - 1) / (WAVES * STEP), a.c.hkv, a.q.num_seqs), dim3(THREADS), 0, s>>>(a);
    e = hipGetLastError();
  }
  return e;
}

template <int D>
hipError_t by_type(const Kv4Attn &a, bool f32, hipStream_t s) {
  if (f32) return a.softcap > 0.f ? launch<D, 3, true>(a, s) : launch<D, 3, false>(a, s);
  return a.softcap > 0.f ? launch<D, 1, true>(a, s) : launch<D, 1, false>(a, s);
}

}  // namespace

Kv4Plan dx_kv4_attn_plan(int max_seq_len, int max_ctx, int group, int window) {
  Kv4Plan p;
  p.max_rows = max_seq_len * group;
  // a window's span starts at a multiple of 64 below it and ends with the newest tokens
  const long seen = window > 0 ? (long)window + 64 + max_seq_len : max_ctx;
  const long len = seen < max_ctx ? seen : max_ctx, most = (len + SPAN - 1) / SPAN;
  p.max_splits = most < 1 ? 1 : most > MAX_SPANS ? MAX_SPANS : (int)most;  // a shorter sequence may have more than a longer
  const long rows = (long)p.max_splits * p.max_rows;
  p.part_rows = p.max_splits == 1 ? 0 : (int)(rows < SPLIT_ROWS ? rows : SPLIT_ROWS);
  return p;
}

hipError_t dx_kv4_attn_launch(const Kv4Attn &a, bool f32, hipStream_t s) {
  if (a.c.d == 64) return by_type<64>(a, f32, s);
  if (a.c.d == 128) return by_type<128>(a, f32, s);
  return by_type<256>(a, f32, s);
}

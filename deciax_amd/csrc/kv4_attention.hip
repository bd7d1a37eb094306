// Attention of a sequence's newest tokens over its paged 4-bit cache, for gfx950.
//
// For query head h of KV head g and newest token i of n (own slot a = ctx - n + i):
//   t_j = scale q . k_j, softcap tanh(t_j / softcap) with a soft-cap, for the slots j <= a (with a window also j > a -
//   window and position_j > position_a - window); out = sum_j e^{t_j} v_j / sum_j e^{t_j}; a row that sees nothing is 0.
// All query heads of a KV head and all new tokens are rows of one product: row r is token r / G, head g G + r % G.
//
// kv4_attn_kernel: a workgroup owns 16 rows and one span of the keys (or two, one after the other), its four waves take 32
// keys in turn, each with a softmax of its own (running maximum and sum in base 2), joined through LDS at the end; spans
// are joined by kv4_join_kernel. kv4_attn_tile_kernel: a workgroup owns 64 or 128 rows and decodes keys once for all. How
// keys are split follows from the sequence alone (`spans`), so a row's result does not depend on its batch.
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

// Rows of a KV head up to which waves share rows and split keys (kv4_attn_kernel), by the row tiles that a wave has
// beyond. Two waste more when rows are few. 24 sequences of 24 rows over 3000 keys: D = 256, one tile, 92 us here and 87
// there; D = 128, two, 87 and 146. 8 of 40 rows over 4000: 66 and 54; 63 and 90.
template <int NT>
constexpr int few_rows() { return NT == 1 ? 32 : 48; }

// Workgroups of kv4_attn_tile_kernel at most: 4 rounds of two a CU.
constexpr int TILE_GROUPS = 2048;
DX_DEVICE floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// bf16 tiles in LDS: [keys][columns] in 16-byte chunks, chunk c of row r at c ^ swizzle(r), over banks of 16 chunks.
// V in kv4_attn_kernel: 16 lanes write a chunk each, of four rows and four blocks (chunks 4 apart; 64 columns: eight rows,
// two blocks, and two rows share the banks); 32 lanes read the halves of two neighbouring chunks of eight rows, transposed.
// So the low two bits differ over the four rows, and the bits above the lowest over the eight. In the tile kernel's tiles
// 16 lanes write, and of K read, one chunk each of 16 rows.
template <int W>
DX_DEVICE int swizzle(int r) {
  if constexpr (W == 64) {
    const int t = r >> 1;
    return (t & 3) | (t & 1) << 2;
  } else {
    return (r & 3) | (r & 1) << 2 | (r & 4) << 1;
  }
}
template <int W>
DX_DEVICE int v_chunk(int r, int c) { return r * W + ((c ^ swizzle<W>(r)) << 3); }
template <int W>
DX_DEVICE int k_chunk(int r, int c) { return r * W + ((c ^ (W == 64 ? (r >> 1) & 7 : r & 15)) << 3); }

DX_DEVICE s16x4 read_transposed(const uint16_t *p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
#else
  return s16x4{};
#endif
}

// A barrier for what went through LDS. __syncthreads() would wait for the loads and stores on their way as well: the next
// keys' and this span's outputs'.
DX_DEVICE void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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

// The keys of 32 slots as a wave holds them before use: lane l has key l % 16 of each 16-key half, 16 bytes a load.
template <int D>
struct Keys {
  static constexpr int N = D == 256 ? 2 : 1;
  u32x4 k[2][N];
  float scale[2][N];
};

// From memory; row0 is the same in all lanes.
template <int D>
DX_DEVICE void load_keys(Keys<D> &w, const Kv4Cache &c, long row0, int lane) {
  const uint8_t *codes = c.k + row0 * (D / 2), *scales = c.ks + row0 * (D / 32);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t row = t * 16 + (lane & 15), grp = lane >> 4;
    if constexpr (D == 64) {  // a lane group takes half a block
      const u32x2 x = *reinterpret_cast<const u32x2 *>(codes + (row * 32 + grp * 8));
      w.k[t][0] = u32x4{x[0], x[1], 0, 0};
      w.scale[t][0] = scale_of(scales[row * 2 + (grp >> 1)]);
    } else {
#pragma unroll
      for (int j = 0; j < Keys<D>::N; ++j) {
        w.k[t][j] = *reinterpret_cast<const u32x4 *>(codes + (row * (D / 2) + (j * 4 + grp) * 16));
        w.scale[t][j] = scale_of(scales[row * (D / 32) + j * 4 + grp]);
      }
    }
  }
}

// The wait for these loads here and not at their first use: inside a loop it would be a wait for the loop's own loads.
template <int N, int NS>
DX_DEVICE void settle(bf16x8 (&q)[N][NS]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int n = 0; n < NS; ++n) asm volatile("" : "+v"(q[i][n]));
}

// Dimension of element 0 of lane group `grp` in the i-th product of a 16-key half (eight consecutive ones follow).
template <int D>
DX_DEVICE int product_dim(int i, int grp) {
  return D == 64 ? grp * 16 + i * 8 : ((i >> 2) * 4 + grp) * 32 + (i & 3) * 8;
}

// cap2 tanh(x) of four values. The continued fraction of tanh, cut after x^9, is x (y^2 + 105 y + 945) / (15 (y^2 + 28 y +
// 63)) with y = x^2, off by 2.4e-8 of the value at |x| <= 0.9 (scores up to 0.9 of the cap) and by fp32's rounding
// below that: relative precision where scores are small, which 1 - 2 / (1 + e^2x) has not. That form serves beyond, in a
// branch that real scores do not take.
DX_DEVICE void capped(float (&x)[4], float cap2) {
  float t[4];
  const float far = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float y = x[r] * x[r];
    const float n = __builtin_fmaf(y + 105.f, y, 945.f), m = __builtin_fmaf(y + 28.f, y, 63.f);
    t[r] = x[r] * (cap2 * (1.f / 15.f)) * n * fast_rcp(m);
  }
  if (__any(!(far <= 0.9f))) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float e = 1.f - 2.f * fast_rcp(1.f + fast_exp2(2.f * LOG2E * fabsf(x[r])));
      t[r] = fabsf(x[r]) <= 0.9f ? t[r] : cap2 * copysignf(e, x[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = t[r];
}

// Products to what the soft-cap takes, or to scores in base 2. They are read in the block that issued them: where a
// uniform branch came between, the compiler left out the wait states that a matrix result needs before it is read (a path
// of 6 instead of 7 was there, and the last two of the four values were stale).
template <int N, bool CAP>
DX_DEVICE void products(const floatx4 (&s)[N], float scale, float softcap, float (&x)[N][4]) {
  const float c = CAP ? scale / softcap : scale * LOG2E;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[n][r] = s[n][r] * c;
      asm volatile("" : "+v"(x[n][r]));  // here, not where a later block uses it
    }
}

// Scores of 32 keys: element 4 t + r is key 16 t + 4 (lane / 16) + r.
template <int D, int NS, bool CAP>
DX_DEVICE void key_scores(const Keys<D> &w, const bf16x8 (&q)[D / 32][NS], float scale, float softcap,
                          float (&t2)[2][4]) {
  floatx4 s[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int j = D == 64 ? 0 : i >> 2;
      const bf16x8 a = as_bf16x8(decode8(w.k[t][j][i & 3], w.scale[t][j]));
#pragma unroll
      for (int n = 0; n < NS; ++n) s[t] = mfma16(a, q[i][n], s[t]);
    }
  products<2, CAP>(s, scale, softcap, t2);
  if constexpr (CAP) {
    capped(t2[0], softcap * LOG2E);
    capped(t2[1], softcap * LOG2E);
  }
}

// The pages of a span, a lane each (64 at a time), so that the loop over keys looks none up in memory.
struct Pages {
  const int32_t *table;
  int width, first;
  long base;  // of this lane: the first row of page table[first + lane] for one head, -1 for none

  DX_DEVICE void load(const Kv4Cache &c, int g, int at, int lane) {
    first = at;
    const int page = at + lane < width ? table[at + lane] : -1;
    base = page >= 0 && page < c.pages ? ((long)page * c.hkv + g) << c.shift : -1;
  }
  // row_of(slot), for a slot that is the same in all lanes
  DX_DEVICE long row(const Kv4Cache &c, int g, int slot, int lane) {
    const int at = slot >> c.shift;
    if (at - first >= 64) {  // slots only rise
      load(c, g, at, lane);
      // wait here: behind the branch the wait would be for all loads on their way, taken or not
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    }
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)base, at - first);
    const int hi = __builtin_amdgcn_readlane((int)(base >> 32), at - first);
    const long row = (long)hi << 32 | lo;
    return hi < 0 ? -1 : row + (slot & ((1 << c.shift) - 1));
  }
};

// One query row as the mask and the addresses need it.
struct Row {
  bool real;    // a row of the packed q
  int own;      // its own slot
  int first;     // with a window: the first slot in it
  int first_pos;  // and the lowest position
  long at;      // its first element in q
};

DX_DEVICE Row query_row(const Kv4Attn &a, const Sequence &s, const int32_t *table, int g, int row, int rows, int group) {
  Row r;
  const int token = row / group;
  r.real = row < rows && s.start + token >= 0 && s.start + token < a.q.rows;
  r.own = s.ctx - s.n + token;
  r.first = r.first_pos = 0;
  if (a.window > 0 && r.real && r.own >= 0) {
    const long at = row_of(a.c, table, g, r.own);
    r.first = a.slots > 0 ? r.own - a.slots + 1 : 0;
    r.first_pos = (int)max((long)(at >= 0 ? a.c.pos[at] : 0) - a.window + 1, -0x80000000L);
  }
  // a row that is none reads the first one: its column of the products goes nowhere
  r.at = r.real ? (s.start + token) * a.q_stride + (long)(g * group + row % group) * a.c.d : 0;
  return r;
}

// Which of the four keys from `key` on (positions `pos`) a row sees; the scores of the others become -inf.
template <bool WIN>
DX_DEVICE uint32_t mask4(const Row &row, int key, const int4 &pos, float (&t2)[4]) {
  const int p[4] = {pos.x, pos.y, pos.z, pos.w};
  uint32_t seen = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    bool see = key + r <= row.own;
    if constexpr (WIN) see = see && key + r >= row.first && p[r] >= row.first_pos;
    if (!see) t2[r] = -INFINITY;
    seen |= (uint32_t)see << r;
  }
  return seen;
}

// The largest of the lanes l % 16 of all four lane groups: rows of 16 lanes, then of 32, exchanged in registers.
DX_DEVICE float max_of_groups(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
#endif
  return x;
}

// The softmax of eight more scores a lane (32 keys a row): raises the running maximum `m` once it is SLACK behind in some
// row, scales what was summed, and gives P as the matrix operand: 2^SLACK at most, as precise as below 1. The lanes of a
// row keep partial sums `l`, joined at the end. (Raised at every new maximum, 16 rows did so in every second step of 90.)
constexpr float SLACK = 8.f;

template <int ND, int NS>
DX_DEVICE void softmax_step(const float (&t2)[2][4], float &m, float &l, floatx4 (&o)[ND], bf16x8 (&pb)[NS]) {
  float top = t2[0][0];
#pragma unroll
  for (int r = 1; r < 8; ++r) top = fmaxf(top, t2[r >> 2][r & 3]);
  top = max_of_groups(top);
  if (__any(top > m + SLACK)) {
    const float next = fmaxf(m, top);
    const float f = next == -INFINITY ? 1.f : fast_exp2(m - next);
    m = next;
    l *= f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] *= f;
  }
  const float base = m == -INFINITY ? 0.f : m;
  float p[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    p[r] = fast_exp2(t2[r >> 2][r & 3] - base);
    l += p[r];
  }
  split8<NS>(p, pb);
}

// How much a part with maximum m and sum l weighs beside a maximum `top`: 0 for one that saw nothing.
DX_DEVICE float part_weight(float m, float l, float top) {
  return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - top);
}

// Four dimensions of one row: to the output where its keys are one span, else to the workspace.
template <int D, int NS>
DX_DEVICE void store_row(const Kv4Attn &a, const Sequence &s, const Spans &sp, long unit, int g, int group, int rows,
                         int split, int row, int d, floatx4 acc, float m, float l) {
  if (sp.count == 1) {
    acc *= l == 0.f ? 0.f : 1.f / l;
    const long out_row = s.start + row / group;
    if (out_row >= 0 && out_row < a.q.rows) {
      const long at = out_row * a.out_stride + (long)(g * group + row % group) * D + d;
      if constexpr (NS == 1) {
        const u32x2 y = {pack_bf2(acc[0], acc[1]), pack_bf2(acc[2], acc[3])};
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + at) = y;
      } else {
        *reinterpret_cast<floatx4 *>(static_cast<float *>(a.out) + at) = acc;
      }
    }
    if (a.w_out && d == 0) a.lse[unit * a.max_rows + row] = m + log2f(l);
  } else {
    const long p = unit * a.part_rows + (long)split * rows + row;
    *reinterpret_cast<floatx4 *>(a.partial + p * D + d) = acc;
    if (d == 0) {
      a.stats[p * 2] = m;
      a.stats[p * 2 + 1] = l;
    }
  }
}

// Few rows: the four waves share 16 rows and take 32 keys in turn. What bounds this kernel is the time that a step's loads
// take, so a step's registers are filled with the next one's as soon as they have been used: K's at the step's start, V's
// once it is decoded. 32 sequences of up to 16384 slots, 8 heads of 256: 222 us (3.9 TB/s, where a copy reaches 5.0); 24
// with a window of 4096, 16 heads of 128: 52 us; one of 2111: 12 us, of which 3 pass before the first keys are there. Loads
// are contiguous over the lanes (16 rows of one chunk, as the product wants K, made the vector cache look at each lane by
// itself: 865 accesses a step where 140 do); K gets its order in LDS.
template <int D>
struct Stage {  // of a wave
  static constexpr int VW = D < 128 ? D : 128;  // columns of V in bf16 at a time
  alignas(1024) uint8_t k[STEP * D / 2];
  uint16_t vt[STEP * VW];
};

template <int D, int NS, bool CAP, bool WIN>
__global__ void __launch_bounds__(THREADS, D == 256 && NS > 1 ? 1 : 2) kv4_attn_kernel(Kv4Attn a) {
  constexpr int LPK = D / 32, VW = Stage<D>::VW, VB = VW / 32;  // blocks of a key, columns and blocks of V at a time
  constexpr int KL = D / 64;                                    // loads of a step's K
  constexpr int VK = 64 / VB, VJ = STEP / VK;                   // keys of one load of V, loads of VW columns
  __shared__ union {
    Stage<D> stage;
    float part[16 * D];
  } stages[WAVES];
  __shared__ float join_m[WAVES][16], join_l[WAVES][16];
  const int g = blockIdx.y, b = blockIdx.z;
  const int tiles = a.few_tiles, row_tile = blockIdx.x % tiles;
  const Sequence s = sequence(a.q, b, a.c.shift);
  const int group = a.hq / a.c.hkv, rows = s.n * group, r0 = row_tile * 16;
  if (r0 >= rows || rows > a.few_rows) return;
  const Spans sp = spans(s.ctx, s.n, rows, a.slots);
  const int first_span = blockIdx.x / tiles * a.spans_each, end_span = min(first_span + a.spans_each, sp.count);
  if (first_span >= sp.count) return;
  const int32_t *table = a.q.table + (long)b * a.q.table_width;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  // this workgroup's spans: their keys follow each other, and so do its waves' steps
  const int k0 = sp.lo + first_span * sp.keys, k1 = min(s.ctx, sp.lo + end_span * sp.keys);
  Pages pages{table, a.q.table_width, 0, -1};
  pages.load(a.c, g, k0 >> a.c.shift, lane);
  Stage<D> &st = stages[wave].stage;

  // Where 16-byte chunk x of 32 rows of K stands in the stage: a row's chunks are exchanged so that 16 rows' reads of one
  // chunk fall on all banks.
  auto k_slot = [](int x) {
    if constexpr (D == 256) return ((x & ~7) | ((x & 7) ^ ((x >> 4) & 7))) * 16;
    else if constexpr (D == 128) return ((x & ~3) | ((x & 3) ^ ((x >> 4) & 3))) * 16;
    else return x * 16;
  };
  u32x4 kr[KL], vr[D / VW][VJ];
  uint32_t ks[2][Keys<D>::N], vs[D / VW][VJ];
  int4 pos[2] = {};
  // A step without a page, or past the last span's end, reads the pool's first rows instead: nothing of them is seen. No
  // branch goes round the loads, behind which the compiler could only wait for all of them.
  auto fetch_keys = [&](int kb) {
    const long row0 = kb < k1 ? pages.row(a.c, g, kb, lane) : -1, at = max(row0, 0L);
    const uint8_t *codes = a.c.k + at * (D / 2), *scales = a.c.ks + at * LPK;
#pragma unroll
    for (int i = 0; i < KL; ++i) kr[i] = *reinterpret_cast<const u32x4 *>(codes + (uint32_t)(i * 64 + lane) * 16);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < Keys<D>::N; ++j)
        ks[t][j] = scales[(uint32_t)((t * 16 + col) * LPK + (D == 64 ? grp >> 1 : j * 4 + grp))];
    if constexpr (WIN) {
#pragma unroll
      for (int t = 0; t < 2; ++t) pos[t] = *reinterpret_cast<const int4 *>(a.c.pos + at + t * 16 + grp * 4);
    }
    return row0;
  };
  auto fetch_values = [&](long row0) {
    const long at = max(row0, 0L);
    const uint8_t *codes = a.c.v + at * (D / 2), *scales = a.c.vs + at * LPK;
#pragma unroll
    for (int h = 0; h < D / VW; ++h)
#pragma unroll
      for (int j = 0; j < VJ; ++j) {
        const uint32_t block = (j * VK + lane / VB) * LPK + h * VB + lane % VB;
        vr[h][j] = *reinterpret_cast<const u32x4 *>(codes + block * 16);
        vs[h][j] = scales[block];
      }
  };

  const Row row = query_row(a, s, table, g, r0 + col, rows, group);
  bf16x8 q[D / 32][NS];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) load_query<NS>(a.query, row.at + product_dim<D>(i, grp), q[i]);
  int kb = k0 + wave * STEP;
  long row0 = fetch_keys(kb);
  fetch_values(row0);
  settle(q);
  // keys below `open` are seen by every row of the tile, as far as the order of tokens goes
  const int open = s.ctx - s.n + r0 / group + 1;

  for (int span = first_span; span < end_span; ++span) {
    floatx4 o[D / 16];
  #pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int span_end = min(s.ctx, sp.lo + (span + 1) * sp.keys);

    for (; kb < span_end; kb += WAVES * STEP) {
      const bool page = row0 >= 0;
      Keys<D> w;
  #pragma unroll
      for (int i = 0; i < KL; ++i) *reinterpret_cast<u32x4 *>(st.k + k_slot(i * 64 + lane)) = kr[i];
      __builtin_amdgcn_wave_barrier();
  #pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = t * 16 + col;
        if constexpr (D == 64) {
          const u32x2 x = *reinterpret_cast<const u32x2 *>(st.k + r * 32 + grp * 8);
          w.k[t][0] = u32x4{x[0], x[1], 0, 0};
        } else {
  #pragma unroll
          for (int j = 0; j < Keys<D>::N; ++j)
            w.k[t][j] = *reinterpret_cast<const u32x4 *>(st.k + k_slot(r * LPK + j * 4 + grp));
        }
  #pragma unroll
        for (int j = 0; j < Keys<D>::N; ++j) {
          w.scale[t][j] = scale_of(ks[t][j]);
          asm volatile("" : "+v"(w.scale[t][j]));  // before the next ones are asked for, not with a copy of them
        }
      }
      int4 here[2] = {pos[0], pos[1]};
      if constexpr (WIN) {
  #pragma unroll
        for (int t = 0; t < 2; ++t) asm volatile("" : "+v"(here[t].x), "+v"(here[t].y), "+v"(here[t].z), "+v"(here[t].w));
      }
      const long next = fetch_keys(kb + WAVES * STEP);

      float t2[2][4];
      key_scores<D, NS, CAP>(w, q, a.scale, a.softcap, t2);
      const bool masked = WIN || kb + STEP > open || !page;
      uint32_t seen = 0xff;  // of this lane's eight keys
      if (masked) {
        seen = 0;
  #pragma unroll
        for (int t = 0; t < 2; ++t)
          seen |= mask4<WIN>(row, page ? kb + t * 16 + grp * 4 : 0x7ffffff0, here[t], t2[t]) << (4 * t);
      }
      if (a.scores && rows <= SCORE_ROWS && col < rows) {
        float *to = a.scores + (((long)b * a.c.hkv + g) * a.score_rows + col) * a.score_slots + kb + grp * 4;
  #pragma unroll
        for (int t = 0; t < 2; ++t)
          *reinterpret_cast<floatx4 *>(to + t * 16) = floatx4{t2[t][0], t2[t][1], t2[t][2], t2[t][3]};
      }
      bf16x8 pb[NS];
      softmax_step<D / 16, NS>(t2, m, l, o, pb);

      // V to bf16, VW columns at a time. Slots behind the sequence hold anything: zeros here. A block of NaN may stand
      // behind a row's own token too, where 0 NaN would reach the row: such blocks are zero here and added below to the
      // rows that see them.
      uint64_t nan_blocks[D / VW][VJ];
      bool any_nan = false;
  #pragma unroll
      for (int h = 0; h < D / VW; ++h) {
  #pragma unroll
        for (int j = 0; j < VJ; ++j) {
          const int key = j * VK + lane / VB;
          u32x4 x = vr[h][j];
          uint32_t byte = vs[h][j];
          if (masked) {
            const bool inside = page && kb + key < s.ctx, bad = byte == 255;
            nan_blocks[h][j] = __ballot(inside && bad);
            any_nan = any_nan || nan_blocks[h][j] != 0;
            if (!inside || bad) {
              x = u32x4{0, 0, 0, 0};
              byte = 127;
            }
          }
  #pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x4 *>(st.vt + v_chunk<VW>(key, lane % VB * 4 + i)) = decode8(x[i], scale_of(byte));
        }
        if (h == D / VW - 1) fetch_values(next);
        __builtin_amdgcn_wave_barrier();
  #pragma unroll
        for (int i = 0; i < VW / 16; ++i) {
          const uint16_t *p0 = st.vt + v_chunk<VW>(grp * 4 + (col >> 2), 2 * i + ((col >> 1) & 1)) + (col & 1) * 4;
          const s16x4 v0 = read_transposed(p0), v1 = read_transposed(p0 + 16 * VW);  // 16 rows on: the same place
          const bf16x8 vt = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
  #pragma unroll
          for (int n = 0; n < NS; ++n) o[h * (VW / 16) + i] = mfma16(vt, pb[n], o[h * (VW / 16) + i]);
        }
        __builtin_amdgcn_wave_barrier();
      }
      if (masked && any_nan) {
  #pragma unroll
        for (int blk = 0; blk < LPK; ++blk) {
          int hit = 0;
  #pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int key = (r >> 2) * 16 + grp * 4 + (r & 3);
            uint64_t bits = nan_blocks[blk / VB][0];
  #pragma unroll
            for (int j = 1; j < VJ; ++j) bits = key / VK == j ? nan_blocks[blk / VB][j] : bits;
            hit |= (int)((bits >> (key % VK * VB + blk % VB)) & 1) & (int)((seen >> r) & 1);
          }
          hit |= __shfl_xor(hit, 16, 64);
          hit |= __shfl_xor(hit, 32, 64);
          if (hit) {
            o[2 * blk] += NAN;
            o[2 * blk + 1] += NAN;
          }
        }
      }
      row0 = next;
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // the four waves' parts, through LDS: [16 rows][D] fp32 a wave, where its stage was
    if (grp == 0) {
      join_m[wave][col] = m;
      join_l[wave][col] = l;
    }
    lds_barrier();
    float top = join_m[0][col];
  #pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, join_m[w][col]);
    const float f = part_weight(m, l, top);
    float *part = stages[wave].part;
    const int valid = min(16, rows - r0);
    if (col < valid) {
  #pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<floatx4 *>(part + col * D + i * 16 + grp * 4) = o[i] * f;
    }
    lds_barrier();

    for (int i = tid; i < valid * (D / 4); i += THREADS) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float mm = join_m[0][r], ll = 0.f;
  #pragma unroll
      for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, join_m[w][r]);
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  #pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        ll += join_l[w][r] * part_weight(join_m[w][r], join_l[w][r], mm);
        acc += *reinterpret_cast<const floatx4 *>(stages[w].part + r * D + d);
      }
      store_row<D, NS>(a, s, sp, (long)b * a.c.hkv + g, g, group, rows, span, r0 + r, d, acc, mm, ll);
    }
    lds_barrier();
  }
}

// Many rows: TW waves of 16 NT rows each walk the same keys, decoded once a workgroup to bf16 in LDS, TK keys at a time: a
// tile's codes are on their way while the one before is used, and go over it afterwards. Two workgroups a CU, in step with
// themselves alone, hide each other's waits; twice the rows a workgroup (half the decoding) or two tiles in turn (no wait
// between use and decoding) were no faster: 6 questions of up to 611 tokens over up to 8803, D = 256, 358 us either way.
// Now 295 to 302 us: 4 sequences of 400 tokens over 6000 slots reach 410 TFLOP/s. Of its time the vector units work 47% (277
// instructions a wave and 32 keys: soft-cap 100, softmax 75, decoding 60), LDS 38%, the matrix units 20%; two waves a SIMD
// (236 registers) leave the rest to waits.
template <int D>
constexpr int tile_keys() { return D == 256 ? 32 : 64; }

template <int D, int NS, bool CAP, int NT, int TW>
__global__ void __launch_bounds__(64 * TW, D == 256 ? (NS > 1 ? 1 : 2) : 2) kv4_attn_tile_kernel(Kv4Attn a) {
  constexpr int TK = tile_keys<D>(), LPK = D / 32, T = 64 * TW;
  constexpr int CHUNKS = TK * LPK;        // 16-byte chunks (blocks) of K, and of V, in a tile
  constexpr int LOADS = 2 * CHUNKS / T;   // of a thread
  constexpr int KW = 64 / LPK;            // keys of a wave's load
  static_assert(2 * CHUNKS % T == 0 && CHUNKS % 64 == 0, "whole waves load K or V");
  __shared__ __attribute__((aligned(1024))) uint16_t kt[TK * D], vt[TK * D];
  __shared__ uint8_t nan_block[CHUNKS];
  __shared__ uint8_t nan_wave[TW];
  constexpr int ROWS = 16 * NT * TW;
  const int group = a.hq / a.c.hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  // Which row tile, span and head of which sequence: work items of all sequences, counted from their lengths.
  for (int item = blockIdx.x;; item += gridDim.x) {
    int b = 0, before = 0;  // items of the sequences before
    for (int b0 = 0;; b0 += 64) {
      if (b0 >= a.q.num_seqs) return;
      int mine = 0;
      if (b0 + lane < a.q.num_seqs) {
        const Sequence s = sequence(a.q, b0 + lane, a.c.shift);
        const int rows = s.n * group;
        if (rows > a.few_rows) mine = (rows + ROWS - 1) / ROWS * spans(s.ctx, s.n, rows, a.slots).count * a.c.hkv;
      }
      int upto = mine;
#pragma unroll
      for (int off = 1; off < 64; off *= 2) {
        const int x = __shfl_up(upto, off, 64);
        upto += lane >= off ? x : 0;
      }
      const uint64_t behind = __ballot(item - before < upto);
      if (behind) {
        const int at = __ffsll((unsigned long long)behind) - 1;
        b = b0 + at;
        before += __shfl(upto - mine, at, 64);
        break;
      }
      before += __shfl(upto, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const Sequence s = sequence(a.q, b, a.c.shift);
    const int rows = s.n * group, tiles = (rows + ROWS - 1) / ROWS;
    const Spans sp = spans(s.ctx, s.n, rows, a.slots);
    const int place = __builtin_amdgcn_readfirstlane(item - before);
    const int r0 = place % tiles * ROWS, split = place / tiles % sp.count, g = place / tiles / sp.count;
    const int32_t *table = a.q.table + (long)b * a.q.table_width;
    // the span's keys that some row of this workgroup sees
    const int last_own = s.ctx - s.n + (min(r0 + ROWS, rows) - 1) / group;
    const int first_own = s.ctx - s.n + r0 / group;
    int k0 = sp.lo + split * sp.keys;
    const int k1 = min(min(s.ctx, k0 + sp.keys), last_own + 1);
    if (a.window > 0) k0 = max(k0, (first_own - a.slots + 1) & ~63);
    Pages pages{table, a.q.table_width, 0, -1};
    pages.load(a.c, g, max(k0, 0) >> a.c.shift, lane);

    const int w0 = r0 + wave * 16 * NT;  // this wave's first row
    Row row[NT];
    bf16x8 q[NT][D / 32][NS];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      row[n] = query_row(a, s, table, g, w0 + n * 16 + col, rows, group);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) load_query<NS>(a.query, row[n].at + i * 32 + grp * 8, q[n][i]);
    }
    const int open = s.ctx - s.n + w0 / group + 1;                               // as above, for the wave's rows
    const int shut = s.ctx - s.n + (min(w0 + 16 * NT, rows) - 1) / group + 1;  // keys from here on no row sees
    const bool idle = w0 >= rows;

    floatx4 o[NT][D / 16];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[n][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    u32x4 raw[LOADS];
    uint32_t byte[LOADS];
    // A wave's load has KW keys, a lane block lane / KW of key lane % KW: neighbours write the same columns of different
    // rows of LDS, which the swizzle spreads over the banks (neighbouring blocks of one row: 4.9 conflict cycles where 0.8
    // are left, and 9% of the kernel's time). A tile lies in one page.
    const uint32_t in_wave = lane % KW * LPK + lane / KW;
    auto fetch = [&](int kb) {
      const long row0 = kb < k1 ? pages.row(a.c, g, kb, lane) : -1, from = max(row0, 0L);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int c = i * T + tid;
        const uint32_t chunk = (c & ~63) % CHUNKS + in_wave;
        const bool keys = __builtin_amdgcn_readfirstlane(c) < CHUNKS;
        raw[i] = *reinterpret_cast<const u32x4 *>((keys ? a.c.k : a.c.v) + from * (D / 2) + chunk * 16);
        byte[i] = ((keys ? a.c.ks : a.c.vs) + from * LPK)[chunk];
      }
      return row0;
    };
    auto decode = [&](int kb) {
      bool bad_here = false;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int c = i * T + tid, chunk = (c & ~63) % CHUNKS + in_wave, key = chunk / LPK, blk = chunk % LPK;
        if (c < CHUNKS) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<u32x4 *>(kt + k_chunk<D>(key, blk * 4 + x)) = decode8(raw[i][x], scale_of(byte[i]));
        } else {
          const bool inside = kb + key < k1, bad = inside && byte[i] == 255;
          if (!inside || bad) {
            raw[i] = u32x4{0, 0, 0, 0};
            byte[i] = 127;
          }
          nan_block[key * LPK + blk] = bad;
          bad_here = bad_here || bad;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<u32x4 *>(vt + v_chunk<D>(key, blk * 4 + x)) = decode8(raw[i][x], scale_of(byte[i]));
        }
      }
      const bool any = __any(bad_here);
      if (lane == 0) nan_wave[wave] = any;
    };

    // 32 keys of the tile in `half`, from row `at` of it, for this wave's rows: their scores, then what they do to the rows
    float t2[NT][2][4];
    uint32_t seen[NT];
    auto scores = [&](int at, int kb, long row0) {
      if (idle || row0 < 0 || kb >= shut || kb >= k1) return;
      const bool masked = a.window > 0 || kb + STEP > open;
#pragma unroll
      for (int n = 0; n < NT; ++n) seen[n] = 0xff;
      // K's operands four at a time, the next four on their way while these are used: left to itself the compiler reads
      // each one right before its product, and V's below likewise (6 questions of up to 611 tokens: 358 us, not 304)
      constexpr int KG = D / 64;
      bf16x8 kf[2][4];
      auto load_k = [&](int x, bf16x8 (&f)[4]) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int i = 2 * x + y / 2, r = (y & 1) * 16 + col;
          // column 16-byte chunk 4 i + grp; the swizzle is below 16, so chunks 16 on are at a constant distance
          const uint16_t *p = kt + at * D + k_chunk<D>(r, (i & 3) * 4 + grp) + (i & ~3) * 32;
          f[y] = as_bf16x8(*reinterpret_cast<const u32x4 *>(p));
        }
      };
      floatx4 sc[2][NT];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[t][n] = floatx4{0.f, 0.f, 0.f, 0.f};
      load_k(0, kf[0]);
#pragma unroll
      for (int x = 0; x < KG; ++x) {
        if (x + 1 < KG) load_k(x + 1, kf[(x + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int z = 0; z < NS; ++z) sc[y & 1][n] = mfma16(kf[x & 1][y], q[n][2 * x + y / 2][z], sc[y & 1][n]);
        __builtin_amdgcn_sched_barrier(0);
      }
      float part[2][NT][4];
      products<NT, CAP>(sc[0], a.scale, a.softcap, part[0]);
      products<NT, CAP>(sc[1], a.scale, a.softcap, part[1]);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        int4 pos{0, 0, 0, 0};
        if (a.window > 0) pos = *reinterpret_cast<const int4 *>(a.c.pos + row0 + t * 16 + grp * 4);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (CAP) capped(part[t][n], a.softcap * LOG2E);
          if (masked) {
            const uint32_t see = a.window > 0 ? mask4<true>(row[n], kb + t * 16 + grp * 4, pos, part[t][n])
                                              : mask4<false>(row[n], kb + t * 16 + grp * 4, pos, part[t][n]);
            seen[n] = t == 0 ? see : seen[n] | see << 4;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) t2[n][t][r] = part[t][n][r];
        }
      }
    };
    auto values = [&](int at, int kb, long row0) {
      if (idle || row0 < 0 || kb >= shut || kb >= k1) return;
      constexpr int VG = D / 64;
      bf16x8 vf[2][4];
      auto load_v = [&](int x, bf16x8 (&f)[4]) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int i = 4 * x + y;
          const int chunk = 2 * (i & 7) + ((col >> 1) & 1);
          const uint16_t *p0 = vt + at * D + v_chunk<D>(grp * 4 + (col >> 2), chunk) + (col & 1) * 4 + (i & ~7) * 16;
          const s16x4 v0 = read_transposed(p0), v1 = read_transposed(p0 + 16 * D);
          f[y] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        }
      };
      load_v(0, vf[0]);
      bf16x8 pb[NT][NS];
#pragma unroll
      for (int n = 0; n < NT; ++n) softmax_step<D / 16, NS>(t2[n], m[n], l[n], o[n], pb[n]);
#pragma unroll
      for (int x = 0; x < VG; ++x) {
        if (x + 1 < VG) load_v(x + 1, vf[(x + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int z = 0; z < NS; ++z) o[n][4 * x + y] = mfma16(vf[x & 1][y], pb[n][z], o[n][4 * x + y]);
        __builtin_amdgcn_sched_barrier(0);
      }
      uint32_t flags = 0;
#pragma unroll
      for (int w = 0; w < TW; ++w) flags |= nan_wave[w];
      if (flags) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int blk = 0; blk < LPK; ++blk) {
            int hit = 0;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const int key = at + (r >> 2) * 16 + grp * 4 + (r & 3);
              hit |= (int)nan_block[key * LPK + blk] & (int)((seen[n] >> r) & 1);
            }
            hit |= __shfl_xor(hit, 16, 64);
            hit |= __shfl_xor(hit, 32, 64);
            if (hit) {
              o[n][2 * blk] += NAN;
              o[n][2 * blk + 1] += NAN;
            }
          }
      }
    };

#pragma unroll
    for (int n = 0; n < NT; ++n) settle(q[n]);
    if (k0 < k1) {
      long here = fetch(k0);
      decode(k0);
      lds_barrier();
      for (int kb = k0; kb < k1; kb += TK) {
        const long next = fetch(kb + TK);
#pragma unroll
        for (int at = 0; at < TK; at += STEP) {
          scores(at, kb + at, here < 0 ? -1 : here + at);
          values(at, kb + at, here < 0 ? -1 : here + at);
        }
        lds_barrier();
        decode(kb + TK);
        here = next;
        lds_barrier();
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] += __shfl_xor(l[n], 16, 64);
      l[n] += __shfl_xor(l[n], 32, 64);
      const int r = w0 + n * 16 + col;
      if (r >= rows) continue;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        store_row<D, NS>(a, s, sp, (long)b * a.c.hkv + g, g, group, rows, split, r, i * 16 + grp * 4, o[n][i], m[n], l[n]);
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
  const float f = lane < sp.count ? part_weight(ms, ls, m) : 0.f;
  l = wave_sum(ls * f);
  for (int i0 = 0; i0 < sp.count; i0 += 8) {  // eight spans' loads at a time
    float x[8][E];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float *p = a.partial + (first + (long)min(i0 + i, sp.count - 1) * rows) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = p[e];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float fi = __shfl(f, i0 + i, 64);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = i0 + i < sp.count ? __builtin_fmaf(x[i][e], fi, acc[e]) : acc[e];
    }
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

// weights_out_j = weights_in_j (0 for the newest slots) + sum over the rows that see j of e^{t_j} / sum e^t, for sequences
// of few rows, whose scores kv4_attn_kernel kept: 4 bytes a row and slot in the place of the key's 34, 68 or 136.
__global__ void __launch_bounds__(THREADS) kv4_score_weights_kernel(Kv4Attn a) {
  constexpr int ITER = 4;
  const int g = blockIdx.y, b = blockIdx.z;
  const Sequence s = sequence(a.q, b, a.c.shift);
  const int group = a.hq / a.c.hkv, rows = s.n * group;
  const int j0 = blockIdx.x * (ITER * THREADS) + threadIdx.x;
  if (rows > SCORE_ROWS || j0 >= s.ctx) return;
  const Spans sp = spans(s.ctx, s.n, rows, a.slots);
  const long unit = (long)b * a.c.hkv + g;
  const float *scores = a.scores + unit * a.score_rows * a.score_slots, *lse = a.lse + unit * a.max_rows;
  const float *old = a.w_in + b * a.wi_seq + g * a.wi_head;
  float sum[ITER] = {}, was[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) was[i] = old[min(j0 + i * THREADS, s.ctx - 1)];
  for (int r = 0; r < rows; ++r) {
    if (s.start + r / group < 0 || s.start + r / group >= a.q.rows) continue;  // no row of the packed q
    const float base = lse[r];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int j = j0 + i * THREADS;
      // no score below the window's first tile; a row that saw nothing has a base of -inf and scores of -inf
      const float t = scores[(long)r * a.score_slots + min(max(j, sp.lo), s.ctx - 1)];
      sum[i] += j >= sp.lo && t != -INFINITY ? fast_exp2(t - base) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int j = j0 + i * THREADS;
    if (j < s.ctx) a.w_out[b * a.wo_seq + g * a.wo_head + j] = (j < s.ctx - s.n ? was[i] : 0.f) + sum[i];
  }
}

// The same for sequences of more rows, from the keys. A wave owns 32 keys, decoded once, and walks all rows, so every sum
// has one owner and one order. Its workgroup brings the rows through LDS, 32 at a time and the next 32 on their way: read
// by each wave as its products want them (16 rows of one chunk) they cost the vector cache a look at every lane: 261 us
// where this takes 176, for 6 questions of up to 611 tokens over up to 8803; with three waves a SIMD 147.
template <int D, int NS, bool CAP>
__global__ void __launch_bounds__(THREADS, NS == 1 ? 3 : 1) kv4_weights_kernel(Kv4Attn a) {
  constexpr int ROWS = 32, BYTES = NS == 1 ? 2 : 4, CHUNKS = D * BYTES / 16;  // 16-byte chunks of a row
  constexpr int LOADS = ROWS * CHUNKS / THREADS;                               // of a thread
  __shared__ u32x4 qs[2][ROWS * CHUNKS];  // chunk c of row r at c ^ (r % 8)
  __shared__ float lses[2][ROWS];
  const int g = blockIdx.y, b = blockIdx.z;
  const Sequence s = sequence(a.q, b, a.c.shift);
  const int32_t *table = a.q.table + (long)b * a.q.table_width;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = a.hq / a.c.hkv, rows = s.n * group;
  const int kb0 = blockIdx.x * (WAVES * STEP), kb = kb0 + wave * STEP;
  if (kb0 >= s.ctx || (a.scores && rows <= SCORE_ROWS)) return;
  const long unit = (long)b * a.c.hkv + g;
  const long row0 = kb < s.ctx ? row_of(a.c, table, g, kb) : -1;
  const int lo = a.window > 0 ? s.ctx - s.n - a.slots + 1 : 0;
  const bool live = row0 >= 0 && kb + STEP > lo;
  float sum[8] = {};
  if (a.q.rows > 0 && kb0 + WAVES * STEP > lo) {
    bf16x8 k[2][D / 32];
    int4 pos[2] = {};
    {
      const long at = max(row0, 0L);
      Keys<D> w;
      load_keys<D>(w, a.c, at, lane);
      if (a.window > 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) pos[t] = *reinterpret_cast<const int4 *>(a.c.pos + at + t * 16 + grp * 4);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const int j = D == 64 ? 0 : i >> 2;
          k[t][i] = as_bf16x8(decode8(w.k[t][j][i & 3], w.scale[t][j]));
        }
    }
    const bool packed = s.start >= 0 && (long)s.start + s.n <= a.q.rows;
    u32x4 raw[LOADS];
    float raw_lse = 0.f;
    auto fetch = [&](int r0) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int x = i * THREADS + tid, r = r0 + x / CHUNKS, token = r / group;
        const bool real = r < rows && s.start + token >= 0 && s.start + token < a.q.rows;
        const long at = real ? (s.start + token) * a.q_stride + (long)(g * group + r - token * group) * D : 0;
        raw[i] = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.query) + at * BYTES + x % CHUNKS * 16);
      }
      raw_lse = a.lse[unit * a.max_rows + min(r0 + (tid & (ROWS - 1)), rows - 1)];
    };
    auto keep = [&](int half) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int x = i * THREADS + tid, r = x / CHUNKS, c = x % CHUNKS;
        qs[half][r * CHUNKS + (c ^ (r & 7))] = raw[i];
      }
      if (tid < ROWS) lses[half][tid] = raw_lse;
    };
    auto add = [&](int half, int sub, int r0) {
      const int r = sub + col;
      auto load_q = [&](int i, bf16x8 (&q)[NS]) {
        const u32x4 *p = qs[half] + r * CHUNKS;
        const int c = product_dim<D>(i, grp) * BYTES / 16;
        if constexpr (NS == 1) {
          q[0] = as_bf16x8(p[c ^ (r & 7)]);
        } else {
          const floatx4 x = __builtin_bit_cast(floatx4, p[c ^ (r & 7)]);
          const floatx4 y = __builtin_bit_cast(floatx4, p[(c + 1) ^ (r & 7)]);
          const float z[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
          split8<NS>(z, q);
        }
      };
      bf16x8 q[2][2][NS];  // two products' rows at a time, the next two on their way
      floatx4 sc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
      load_q(0, q[0][0]);
      load_q(1, q[0][1]);
      const float lse = lses[half][r];
#pragma unroll
      for (int i = 0; i < D / 32; i += 2) {
        if (i + 2 < D / 32) {
          load_q(i + 2, q[(i / 2 + 1) & 1][0]);
          load_q(i + 3, q[(i / 2 + 1) & 1][1]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int t = 0; t < 2; ++t) sc[t] = mfma16(k[t][i + x], q[i / 2 & 1][x][n], sc[t]);
        __builtin_amdgcn_sched_barrier(0);
      }
      float t2[2][4];
      products<2, CAP>(sc, a.scale, a.softcap, t2);
      // whether some row of these does not see some key of these
      const bool masked = a.window > 0 || !packed || r0 + 16 > rows || kb + STEP > s.ctx - s.n + r0 / group + 1;
      Row row;
      if (masked) row = query_row(a, s, table, g, r0 + col, rows, group);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (CAP) capped(t2[t], a.softcap * LOG2E);
        if (masked) {
          const int key = kb + t * 16 + grp * 4;
          const uint32_t seen = a.window > 0 ? mask4<true>(row, key, pos[t], t2[t])
                                             : mask4<false>(row, key, pos[t], t2[t]);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[t * 4 + r] += row.real && (seen >> r) & 1 ? fast_exp2(t2[t][r] - lse) : 0.f;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[t * 4 + r] += fast_exp2(t2[t][r] - lse);
        }
      }
    };
    // the first row that can see a key of the workgroup's
    const int first = min(max(0, kb0 - (s.ctx - s.n)), s.n) * group & ~(ROWS - 1);
    if (first < rows) {
      fetch(first);
      keep(0);
      lds_barrier();
      int half = 0;
      for (int r0 = first; r0 < rows; r0 += ROWS) {
        fetch(r0 + ROWS);
        if (live) {
          add(half, 0, r0);
          if (r0 + 16 < rows) add(half, 16, r0 + 16);
        }
        half ^= 1;
        keep(half);
        lds_barrier();
      }
    }
  }
  if (kb >= s.ctx) return;
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

// kv4_attn_kernel's workgroups are listed by row tile, then by span: a sequence of many rows has few spans, and the
// workgroups that have work then follow each other over the XCDs (listed by span first they were every 32nd one, all on one
// XCD).
// Sequences of few rows take kv4_attn_kernel, of more kv4_attn_tile_kernel; a batch of both launches both.
template <int D, int NS, bool CAP>
hipError_t launch(Kv4Attn a, hipStream_t s) {
  constexpr int NT = NS == 1 && D < 256 ? 2 : 1, TW = 4;
  a.few_rows = few_rows<NT>();
  const int few = a.q.rows > 0 ? (min(a.max_rows, a.few_rows) + 15) / 16 : 0;  // without rows: the weights alone
  const int tiles = a.q.rows > 0 && a.max_rows > a.few_rows ? (a.max_rows + 16 * NT * TW - 1) / (16 * NT * TW) : 0;
  a.few_tiles = few;
  // Two spans a workgroup where there are many workgroups: a workgroup's start (lengths, page, query and first keys, each
  // after the other) takes 3 us of some 13. 64 x 4000 137 -> 128 us, 32 x 14000 217 -> 206, 16 x 8000 64.3 -> 62.2;
  // 4 x 16384 (1024 workgroups) 42.6 -> 44.3.
  a.spans_each = (long)a.max_splits * few * a.c.hkv * a.q.num_seqs >= 2048 ? 2 : 1;
  hipError_t e = hipSuccess;
  if (few > 0) {
    const dim3 grid((a.max_splits + a.spans_each - 1) / a.spans_each * few, a.c.hkv, a.q.num_seqs);
    if (a.window > 0) kv4_attn_kernel<D, NS, CAP, true><<<grid, dim3(THREADS), 0, s>>>(a);
    else kv4_attn_kernel<D, NS, CAP, false><<<grid, dim3(THREADS), 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && tiles > 0) {
    const long items = (long)a.max_splits * tiles * a.c.hkv * a.q.num_seqs;
    kv4_attn_tile_kernel<D, NS, CAP, NT, TW>
        <<<dim3((int)min(items, (long)TILE_GROUPS)), dim3(64 * TW), 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && few > 0 && a.max_splits > 1) {
    const int split_rows = min(a.max_rows, MOST_SPLIT_ROWS);
    kv4_join_kernel<D, NS><<<dim3((split_rows + WAVES - 1) / WAVES, a.c.hkv, a.q.num_seqs), dim3(THREADS), 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.w_out && a.q.max_ctx > 0 && a.scores) {
    kv4_score_weights_kernel<<<dim3((a.q.max_ctx + 4 * THREADS - 1) / (4 * THREADS), a.c.hkv, a.q.num_seqs),
                               dim3(THREADS), 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.w_out && a.q.max_ctx > 0 && (!a.scores || a.max_rows > SCORE_ROWS)) {
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

hipError_t dx_kv4_attn_launch(const Kv4Attn &a, bool f32, hipStream_t s) {
  if (a.c.d == 64) return by_type<64>(a, f32, s);
  if (a.c.d == 128) return by_type<128>(a, f32, s);
  return by_type<256>(a, f32, s);
}

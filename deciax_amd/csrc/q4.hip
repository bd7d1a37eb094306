// Weights in 4 bits with one scale and zero point a group, and products with them.
//
// Format: W[n, k] = scale (code - zero), code and zero 0..15; a group is 32, 64 or 128 neighbouring k of a row. Codes lie
// in tiles of 16 rows and 128 columns, 1 KB each, [n / 16][k / 128][64 lanes][16 bytes]: lane 16 q + r holds row r, its
// dword j the columns 32 j + 8 q + 0..7, which is the second operand of the j-th 16x16x32 product of the tile. Within a
// dword the nibbles are the columns 0, 2, 4, 6, 1, 3, 5, 7, so that one shift, one mask and one or make two bf16 values.
// A group's word [n / 16][k / group][16] is its scale (a bf16 or fp16 number) as fp32 with the zero in the lowest four
// bits. Missing rows and columns of a tile have code 0; missing rows word 0.
#include "common.h"
#include "kernels.h"

namespace {

constexpr int WAVES = 8, THREADS = 64 * WAVES;

DX_DEVICE floatx4 mfma16(u32x4 a, u32x4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// Eight codes as bf16 numbers 8 + code / 2: a code's four bits are the highest of the mantissa of a number in [8, 16).
DX_DEVICE u32x4 halves(uint32_t w) {
  constexpr uint32_t MASK = 0x00780078u, EIGHT = 0x41004100u;
  return u32x4{((w << 3) & MASK) | EIGHT, ((w >> 1) & MASK) | EIGHT, ((w >> 5) & MASK) | EIGHT,
               ((w >> 9) & MASK) | EIGHT};
}

DX_DEVICE float scale_of(uint32_t word) { return __uint_as_float(word & ~15u); }
DX_DEVICE float zero_of(uint32_t word) { return (float)(word & 15u); }

// y = x W^T on 16x16x32 products (first operand x: lane l has row l % 16 and the columns 8 (l / 16) .. of a step of 32; second
// W, the same; the result's lane l has column l % 16, rows 4 (l / 16) + e).
//
// Eight sums are taken: of the tiles 0, 8, 16, .. of the columns, of 1, 9, 17, .., and so on, each in this order, and added
// in theirs. So the order of a sum goes by k alone, and a row of y depends on its row of x alone, whichever kernel has it:
// with few rows the eight waves of a workgroup have a sum each, with many a wave takes them one after the other.
//
// The products are of x and 8 + code / 2, both exact: with X the group's sum of x (one more product, by ones),
// sum x (code - zero) = 2 (sum x (8 + code / 2) - (8 + zero / 2) X), the difference rounded once, and only then the scale.
// All sums in fp32. An infinity or a NaN in a row of x makes that row of y NaN.
//
// Reads of a weight's tiles t and groups of one tile row, and of x, as buffers: what lies behind the last column reads as 0,
// without a branch, so that every load stays on its way until it is used.
struct TileRow {
  __amdgpu_buffer_rsrc_t codes, words;
};
DX_DEVICE TileRow tile_row(const u32x4 *codes, const uint32_t *words, long tile, int tiles_k, int groups) {
  return TileRow{__builtin_amdgcn_make_buffer_rsrc((void *)(codes + tile * tiles_k * 64), (short)0, tiles_k * 1024, 0x00020000),
                 __builtin_amdgcn_make_buffer_rsrc((void *)(words + tile * groups * 16), (short)0, groups * 64, 0x00020000)};
}
DX_DEVICE u32x4 load16(__amdgpu_buffer_rsrc_t from, uint32_t bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_raw_buffer_load_b128(from, bytes, 0, 0);
#else
  return u32x4{};
#endif
}
DX_DEVICE uint32_t load4(__amdgpu_buffer_rsrc_t from, uint32_t bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_raw_buffer_load_b32(from, bytes, 0, 0);
#else
  return 0;
#endif
}

// A tile's codes and words.
template <int GROUPS>
struct Codes {
  u32x4 raw;
  uint32_t word[GROUPS];
  DX_DEVICE void load(const TileRow &from, uint32_t t, int lane) {
    raw = load16(from.codes, t * 1024 + lane * 16);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) word[g] = load4(from.words, (t * GROUPS + g) * 64 + (lane & 15) * 4);
  }
};

// Columns 128 t .. of 16 rows of x. Read as they are multiplied, a lane its row, 16 rows' pieces of 64 bytes would take four
// times as long as whole rows of 256: so 16 lanes read a row, and the wave turns the tile in LDS, chunk c of row r at c ^ r.
struct Columns {
  u32x4 part[4];
  // at: the rows' bytes before their columns; rows behind the last stand for it and are not stored.
  DX_DEVICE static void places(uint32_t (&at)[4], int m, long ldx, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + (lane >> 4);
      at[i] = min(r, m - 1) * (uint32_t)ldx * 2 + 16 * ((lane & 15) ^ r);
    }
  }
  DX_DEVICE void load(__amdgpu_buffer_rsrc_t x, const uint32_t (&at)[4], int t, int k, int lane) {
    const int left = k - 128 * t;  // columns, at most 0 behind the last tile
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 8 * ((lane & 15) ^ (4 * i + (lane >> 4)));
      part[i] = load16(x, col < left ? at[i] + 256 * t : 0x7fffffffu);
    }
  }
  DX_DEVICE void turn(u32x4 *lds, u32x4 (&step)[4], int lane) const {
    const int c = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[64 * i + lane] = part[i];
#pragma unroll
    for (int s = 0; s < 4; ++s) step[s] = lds[16 * c + ((4 * s + q) ^ c)];
  }
};

template <int MT, int NT, int SPG>
DX_DEVICE void multiply(const Codes<4 / SPG> (&w)[NT], const u32x4 (&x)[MT][4], floatx4 (&sum)[MT][NT]) {
  const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
  for (int g = 0; g < 4 / SPG; ++g) {
    floatx4 acc[MT][NT], xs[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      xs[i] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{0, 0, 0, 0};
    }
#pragma unroll
    for (int s = g * SPG; s < (g + 1) * SPG; ++s) {
#pragma unroll
      for (int i = 0; i < MT; ++i) xs[i] = mfma16(x[i][s], ones, xs[i]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const u32x4 b = halves(w[j].raw[s]);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = mfma16(x[i][s], b, acc[i][j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float s2 = 2.f * scale_of(w[j].word[g]), off = -8.f - 0.5f * zero_of(w[j].word[g]);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][j][e] = fmaf(s2, fmaf(off, xs[i][e], acc[i][j][e]), sum[i][j][e]);
    }
  }
}

// The waves' sums of a tile, added in their order and stored. The next tile takes the other buffer: what this one held is
// read before its barrier.
template <typename OUT>
DX_DEVICE void join(float (&parts)[WAVES][256], const floatx4 &sum, OUT *y, int tile, int m, int n, long ldy) {
  const int at = threadIdx.x, lane = at & 63;
#pragma unroll
  for (int e = 0; e < 4; ++e) parts[at >> 6][64 * e + lane] = sum[e];  // row 4 (lane / 16) + e
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (at >= 16 * m) return;
  const int o = 16 * tile + (at & 15), from = 64 * ((at >> 4) & 3) + 16 * (at >> 6) + (at & 15);
  float v = parts[0][from];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v += parts[w][from];
  if (o >= n) return;
  if constexpr (sizeof(OUT) == 2)
    y[(long)(at >> 4) * ldy + o] = f2bf(v);
  else
    y[(long)(at >> 4) * ldy + o] = v;
}

// Up to 16 rows, TPW tiles of columns a wave: x stays in registers, and the workgroup walks tiles of 16 rows of W, one in
// `gridDim.x`; the next one's codes are on their way while this one's are multiplied. Bound by the reads of the codes, once
// there are enough: 4 rows x 256000 x 3584 (481 MB) 92 us, 5.2 TB/s; 1 x 28672 x 3584 12.0 us, half of them the first
// tile's latency and the launch; 1 x 3584 x 4096 4.3 us, where an empty launch takes 3.4. Read again for each tile of W, x
// takes the first to 189 us.
template <int TPW, int SPG, typename OUT>
__global__ void __launch_bounds__(THREADS)
linear_q4_few_kernel(const uint16_t *__restrict__ x, const u32x4 *__restrict__ codes, const uint32_t *__restrict__ words,
                     OUT *__restrict__ y, int m, int n, int k, long ldx, long ldy) {
  __shared__ __align__(16) float parts[2][WAVES][256];
  __shared__ u32x4 turned[WAVES][256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_k = (k + 127) >> 7, tiles_n = (n + 15) >> 4, groups = k / (32 * SPG);
  Codes<4 / SPG> w[TPW][1];
  TileRow from = tile_row(codes, words, blockIdx.x, tiles_k, groups);
#pragma unroll
  for (int d = 0; d < TPW; ++d) w[d][0].load(from, wave + d * WAVES, lane);
  const auto rows = __builtin_amdgcn_make_buffer_rsrc((void *)x, (short)0, (int)(((m - 1) * ldx + k) * 2), 0x00020000);
  uint32_t at[4];
  Columns::places(at, m, ldx, lane);
  Columns read[TPW];
#pragma unroll
  for (int d = 0; d < TPW; ++d) read[d].load(rows, at, wave + d * WAVES, k, lane);
  u32x4 xs[TPW][1][4];
#pragma unroll
  for (int d = 0; d < TPW; ++d) read[d].turn(turned[wave], xs[d][0], lane);
  int buffer = 0;
  for (int tile = blockIdx.x; tile < tiles_n; tile += gridDim.x, buffer ^= 1) {
    floatx4 sum[1][1] = {{{0, 0, 0, 0}}};
    const int next = tile + (int)gridDim.x;
    from = tile_row(codes, words, min(next, tiles_n - 1), next < tiles_n ? tiles_k : 0, next < tiles_n ? groups : 0);
#pragma unroll
    for (int d = 0; d < TPW; ++d) {
      multiply<1, 1, SPG>(w[d], xs[d], sum);
      w[d][0].load(from, wave + d * WAVES, lane);
    }
    join(parts[buffer], sum[0][0], y, tile, m, n, ldy);
  }
}

// Up to 16 rows and more columns than that: one tile of W a workgroup, codes and x two tiles ahead. Bound by the chain of
// a wave's tiles (a load's way, the turn, the products): 13 x 3585 x 14336 with groups of 32 11.4 us of 30 MB, 16 x 28672 x
// 9216 37 us (3.8 TB/s). Codes further ahead take the registers of a second workgroup a CU and unroll more code: four tiles
// 14.1 and 57 us, eight 15.5 and 79. One ahead 12.6 and 38.2.
template <int SPG, typename OUT>
__global__ void __launch_bounds__(THREADS)
linear_q4_long_kernel(const uint16_t *__restrict__ x, const u32x4 *__restrict__ codes, const uint32_t *__restrict__ words,
                      OUT *__restrict__ y, int m, int n, int k, long ldx, long ldy) {
  constexpr int AHEAD = 2;
  __shared__ __align__(16) float parts[WAVES][256];
  __shared__ u32x4 turned[WAVES][256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_k = (k + 127) >> 7, groups = k / (32 * SPG);
  const TileRow from = tile_row(codes, words, blockIdx.x, tiles_k, groups);
  const auto rows = __builtin_amdgcn_make_buffer_rsrc((void *)x, (short)0, (int)(((m - 1) * ldx + k) * 2), 0x00020000);
  uint32_t at[4];
  Columns::places(at, m, ldx, lane);
  Codes<4 / SPG> w[AHEAD][1];
  Columns xs[AHEAD];
#pragma unroll
  for (int d = 0; d < AHEAD; ++d) w[d][0].load(from, wave + d * WAVES, lane);
#pragma unroll
  for (int d = 0; d < AHEAD; ++d) xs[d].load(rows, at, wave + d * WAVES, k, lane);
  floatx4 sum[1][1] = {{{0, 0, 0, 0}}};
  for (int t = wave; t < tiles_k; t += AHEAD * WAVES) {
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {  // tiles behind the last add 0
      const int tile = t + d * WAVES;
      __builtin_amdgcn_sched_barrier(0);  // one tile after the other: both turned at once a tenth more
      u32x4 step[1][4];
      xs[d % AHEAD].turn(turned[wave], step[0], lane);
      xs[d % AHEAD].load(rows, at, tile + AHEAD * WAVES, k, lane);
      multiply<1, 1, SPG>(w[d], step, sum);
      w[d][0].load(from, tile + AHEAD * WAVES, lane);
    }
  }
  join(parts, sum[0][0], y, blockIdx.x, m, n, ldy);
}

// What a wave holds of 16 MT rows and 16 NT columns: the codes of two tiles, x of one on its way.
template <int MT, int NT, int SPG>
struct Block {
  TileRow from[NT];
  __amdgpu_buffer_rsrc_t rows[MT];
  Codes<4 / SPG> w[2][NT];
  Columns read[MT];
  uint32_t at[4];  // of whole tiles of rows; those that are not whole have their last rows' places cut below
  int k, lane;

  DX_DEVICE Block(const uint16_t *x, const u32x4 *codes, const uint32_t *words, long m0, long m, int tile0, int n, int k,
                  int groups, long ldx)
      : k(k), lane(threadIdx.x & 63) {
    const int tiles_k = (k + 127) >> 7, tiles_n = (n + 15) >> 4;
#pragma unroll
    for (int j = 0; j < NT; ++j) from[j] = tile_row(codes, words, min(tile0 + j, tiles_n - 1), tiles_k, groups);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const long first = min(m0 + 16 * i, m - 1);
      const int left = (int)min(m - first, 16L);
      rows[i] = __builtin_amdgcn_make_buffer_rsrc((void *)(x + first * ldx), (short)0, (int)(((left - 1) * ldx + k) * 2),
                                                  0x00020000);
    }
    Columns::places(at, 16, ldx, lane);  // rows behind the last lie behind the buffer: they read as 0 and are not stored
  }
  DX_DEVICE void load_x(int t) {
#pragma unroll
    for (int i = 0; i < MT; ++i) read[i].load(rows[i], at, t, k, lane);
  }
  DX_DEVICE void load_w(int set, int t) {
#pragma unroll
    for (int j = 0; j < NT; ++j) w[set][j].load(from[j], t, lane);
  }
  // One tile of columns, while the next one's x and the codes of `next` come.
  DX_DEVICE void step(int set, int next, u32x4 *turned, floatx4 (&sum)[MT][NT]) {
    u32x4 x[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) read[i].turn(turned, x[i], lane);
    load_x(next);
    load_w(set ^ 1, next);
    multiply<MT, NT, SPG>(w[set], x, sum);
  }
};

// More rows: the eight waves' sums of 16 MT rows and 16 NT columns. Bound by the x that each workgroup reads from L2 and turns
// for only 16 NT columns and by its waves' short chains: 17 to 32 rows x 28672 x 3584 22 us, 33 to 64, which read and make the
// codes bf16 twice, 41 (bf16 weights of that size would take 37 to read); 64 x 8192 x 3584 10.5, 128 x 3584 x 14336 27.
template <int MT, int NT, int SPG, typename OUT>
__global__ void __launch_bounds__(THREADS)
linear_q4_some_kernel(const uint16_t *__restrict__ x, const u32x4 *__restrict__ codes, const uint32_t *__restrict__ words,
                      OUT *__restrict__ y, long m, int n, int k, long ldx, long ldy) {
  __shared__ float parts[WAVES][16][16 * NT + 1];
  __shared__ u32x4 turned[WAVES][256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_k = (k + 127) >> 7;
  const long m0 = (long)blockIdx.y * (16 * MT);
  Block<MT, NT, SPG> b(x, codes, words, m0, m, blockIdx.x * NT, n, k, k / (32 * SPG), ldx);
  floatx4 sum[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sum[i][j] = floatx4{0, 0, 0, 0};
  b.load_w(0, wave);
  b.load_x(wave);
  for (int t = wave; t < tiles_k; t += 2 * WAVES) {
    b.step(0, t + WAVES, turned[wave], sum);
    b.step(1, t + 2 * WAVES, turned[wave], sum);  // behind the last tile it adds 0
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (i > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) parts[wave][4 * (lane >> 4) + e][16 * j + (lane & 15)] = sum[i][j][e];
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * NT; at += THREADS) {
      const int row = at / (16 * NT), col = at % (16 * NT), o = blockIdx.x * NT * 16 + col;
      const long r = m0 + 16 * i + row;
      if (r >= m || o >= n) continue;
      float v = parts[0][row][col];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v += parts[w][row][col];
      if constexpr (sizeof(OUT) == 2)
        y[r * ldy + o] = f2bf(v);
      else
        y[r * ldy + o] = v;
    }
  }
}

// Many rows: four waves of 16 MT rows each and the same 16 NT columns, each with all eight sums, one after the other. Bound
// by the vector unit: per tile and wave 128 instructions make the codes bf16 and 32 MT NT / SPG apply the zeros and scales,
// 4 cycles each, beside 40 products of 16 cycles. 2048 x 8192 x 3584 190 us (630 TFLOP/s); 611 rows with groups of 64 82 us,
// in 640 workgroups where 512 fit at once (the library's product of bf16 weights of that size takes 40). Larger tiles lose the second
// workgroup of a CU: 16 MT x 16 NT of 64 x 32, 64 x 64 and 32 x 128 take 125, 125 and 135 us for those 82.
template <int MT, int NT, int SPG, typename OUT>
__global__ void __launch_bounds__(256, 2)
linear_q4_many_kernel(const uint16_t *__restrict__ x, const u32x4 *__restrict__ codes, const uint32_t *__restrict__ words,
                      OUT *__restrict__ y, long m, int n, int k, long ldx, long ldy) {
  __shared__ u32x4 turned[4][256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_k = (k + 127) >> 7;
  const long m0 = ((long)blockIdx.y * 4 + wave) * (16 * MT);
  if (m0 >= m) return;
  Block<MT, NT, SPG> b(x, codes, words, m0, m, blockIdx.x * NT, n, k, k / (32 * SPG), ldx);
  floatx4 sum[MT][NT], total[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sum[i][j] = total[i][j] = floatx4{0, 0, 0, 0};
  int t = 0;
  auto one = [&](int set) {
    const bool last = t + WAVES >= tiles_k;  // of its sum
    const int next = !last ? t + WAVES : t % WAVES + 1 < WAVES ? t % WAVES + 1 : tiles_k;
    b.step(set, next, turned[wave], sum);
    if (last) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          total[i][j] += sum[i][j];
          sum[i][j] = floatx4{0, 0, 0, 0};
        }
    }
    t = next;
  };
  b.load_w(0, 0);
  b.load_x(0);
  for (int i = 0; i < tiles_k; i += 2) {
    one(0);
    if (i + 1 < tiles_k) one(1);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long r = m0 + 16 * i + 4 * (lane >> 4) + e;
        const int o = (blockIdx.x * NT + j) * 16 + (lane & 15);
        if (r >= m || o >= n) continue;
        if constexpr (sizeof(OUT) == 2)
          y[r * ldy + o] = f2bf(total[i][j][e]);
        else
          y[r * ldy + o] = total[i][j][e];
      }
}

// A wave lays out one tile: lane 16 q + r the codes that the products read as its.
// Once a weight, so it is not tuned: one of 28672 x 3584 is quantised in 70 us, packed from a byte a code in 192 and read as
// fp32 in 108, where the bytes alone take 46, 28 and 83.
struct Place {
  int row, col;  // of the lane's first value of step 0
  bool in;       // the row exists
};

DX_DEVICE Place place(long tile, int tiles_k, int n) {
  const int lane = threadIdx.x & 63;
  const int row = (int)(tile / tiles_k) * 16 + (lane & 15);
  return Place{row, (int)(tile % tiles_k) * 128 + 8 * (lane >> 4), row < n};
}

DX_DEVICE uint32_t nibbles(const uint32_t (&code)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= code[e] << (4 * (e / 2) + 16 * (e % 2));
  return w;
}

// Each group's range is widened to hold 0; scale = bf16((hi - lo) / 15), zero = round(-lo / scale), code = round(w / scale)
// + zero, cut to 0..15 (the scale's own rounding can pass them by one). A group that holds an infinity or a NaN has a NaN
// for its scale and reads as NaN; one whose scale rounds to 0 reads as 0.
template <int SPG>
__global__ void __launch_bounds__(256)
quantize_q4_kernel(const uint16_t *__restrict__ w, long ldw, u32x4 *__restrict__ codes, uint32_t *__restrict__ words,
                   int n, int k, long tiles) {
  const long tile = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int tiles_k = (k + 127) >> 7, lane = threadIdx.x & 63, groups = k / (32 * SPG);
  const Place p = place(tile, tiles_k, n);
  float v[4][8];
  float lo[4 / SPG], hi[4 / SPG];
  bool fine[4 / SPG];
#pragma unroll
  for (int g = 0; g < 4 / SPG; ++g) {
    lo[g] = hi[g] = 0.f;
    fine[g] = true;
#pragma unroll
    for (int s = g * SPG; s < (g + 1) * SPG; ++s) {
      const int col = p.col + 32 * s;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] = 0.f;
      if (p.in && col < k) {
        const u32x4 r = *reinterpret_cast<const u32x4 *>(w + p.row * ldw + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[s][2 * e] = lo_bf(r[e]);
          v[s][2 * e + 1] = hi_bf(r[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[g] = fminf(lo[g], v[s][e]);
        hi[g] = fmaxf(hi[g], v[s][e]);
        fine[g] &= fabsf(v[s][e]) < INFINITY;
      }
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {  // the four lanes of a row
      lo[g] = fminf(lo[g], __shfl_xor(lo[g], off, 64));
      hi[g] = fmaxf(hi[g], __shfl_xor(hi[g], off, 64));
      fine[g] &= __shfl_xor((int)fine[g], off, 64) != 0;
    }
  }
  u32x4 out;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int g = s / SPG;
    const float scale = round_bf(hi[g] / 15.f - lo[g] / 15.f);
    const bool real = fine[g] && scale > 0.f;
    const float zero = real ? fminf(rintf(-lo[g] / scale), 15.f) : 0.f;
    uint32_t code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      code[e] = real && p.in && p.col + 32 * s < k ? (uint32_t)fminf(fmaxf(rintf(v[s][e] / scale) + zero, 0.f), 15.f) : 0u;
    out[s] = nibbles(code);
    const int group = (p.col + 32 * s) / (32 * SPG);
    if (s % SPG == 0 && lane < 16 && group < groups)
      words[((tile / tiles_k) * groups + group) * 16 + lane] =
          !p.in ? 0u : !fine[g] ? 0x7fc00000u : __float_as_uint(real ? scale : 0.f) | (uint32_t)zero;
  }
  codes[tile * 64 + lane] = out;
}

// Given codes (a byte each, its low four bits), scales (bf16, or fp16) and zeros (a byte a group; 8 without them).
template <int SPG, bool HALF>
__global__ void __launch_bounds__(256)
pack_q4_kernel(const uint8_t *__restrict__ code, const uint16_t *__restrict__ scales, const uint8_t *__restrict__ zeros,
               u32x4 *__restrict__ codes, uint32_t *__restrict__ words, int n, int k, long tiles) {
  const long tile = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int tiles_k = (k + 127) >> 7, lane = threadIdx.x & 63, groups = k / (32 * SPG);
  const Place p = place(tile, tiles_k, n);
  u32x4 out;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int col = p.col + 32 * s;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = p.in && col < k ? code[(long)p.row * k + col + e] & 15u : 0u;
    out[s] = nibbles(c);
    const int group = col / (32 * SPG);
    if (s % SPG == 0 && lane < 16 && group < groups) {
      uint32_t word = 0;
      if (p.in) {
        const uint16_t b = scales[(long)p.row * groups + group];
        const float scale = HALF ? (float)__builtin_bit_cast(_Float16, b) : bf2f(b);
        word = (__float_as_uint(scale) & ~15u) | (zeros ? zeros[(long)p.row * groups + group] & 15u : 8u);
      }
      words[((tile / tiles_k) * groups + group) * 16 + lane] = word;
    }
  }
  codes[tile * 64 + lane] = out;
}

template <int SPG>
__global__ void __launch_bounds__(256)
q4_values_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ words, float *__restrict__ w, int n, int k,
                 long ldw, long tiles) {
  const long tile = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int tiles_k = (k + 127) >> 7, lane = threadIdx.x & 63, groups = k / (32 * SPG);
  const Place p = place(tile, tiles_k, n);
  const u32x4 raw = codes[tile * 64 + lane];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int col = p.col + 32 * s;
    if (!p.in || col >= k) continue;
    const uint32_t word = words[((tile / tiles_k) * groups + col / (32 * SPG)) * 16 + (lane & 15)];
    const u32x4 h = halves(raw[s]);
    const float off = 16.f + zero_of(word);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[p.row * ldw + col + 2 * e] = (2.f * lo_bf(h[e]) - off) * scale_of(word);
      w[p.row * ldw + col + 2 * e + 1] = (2.f * hi_bf(h[e]) - off) * scale_of(word);
    }
  }
}

template <int MT, int NT, int SPG>
hipError_t run_some(const Q4Weight &w, const uint16_t *x, void *y, long m, long ldx, long ldy, bool f32, hipStream_t s) {
  const dim3 grid((unsigned)dx_ceil_div(w.n, 16 * NT), (unsigned)dx_ceil_div(m, 16 * MT));
  const u32x4 *codes = static_cast<const u32x4 *>(w.codes);
  if (f32)
    linear_q4_some_kernel<MT, NT, SPG, float>
        <<<grid, dim3(THREADS), 0, s>>>(x, codes, w.words, static_cast<float *>(y), m, w.n, w.k, ldx, ldy);
  else
    linear_q4_some_kernel<MT, NT, SPG, uint16_t>
        <<<grid, dim3(THREADS), 0, s>>>(x, codes, w.words, static_cast<uint16_t *>(y), m, w.n, w.k, ldx, ldy);
  return hipGetLastError();
}

template <int MT, int NT, int SPG>
hipError_t run_many(const Q4Weight &w, const uint16_t *x, void *y, long m, long ldx, long ldy, bool f32, hipStream_t s) {
  const dim3 grid((unsigned)dx_ceil_div(w.n, 16 * NT), (unsigned)dx_ceil_div(m, 64 * MT));
  const u32x4 *codes = static_cast<const u32x4 *>(w.codes);
  if (f32)
    linear_q4_many_kernel<MT, NT, SPG, float>
        <<<grid, dim3(256), 0, s>>>(x, codes, w.words, static_cast<float *>(y), m, w.n, w.k, ldx, ldy);
  else
    linear_q4_many_kernel<MT, NT, SPG, uint16_t>
        <<<grid, dim3(256), 0, s>>>(x, codes, w.words, static_cast<uint16_t *>(y), m, w.n, w.k, ldx, ldy);
  return hipGetLastError();
}

// Two workgroups a CU where their registers fit (up to four tiles of x a wave) and each still has four tiles of W or more;
// else one, with more of them: 40000 columns of 2048 9.9 us with two and 10.9 with one, 256000 of 3584 96 and 108, but 8192
// of 3584 6.4 and 5.8.
template <int TPW, int SPG>
hipError_t run_few(const Q4Weight &w, const uint16_t *x, void *y, long m, long ldx, long ldy, bool f32, hipStream_t s) {
  const int tiles = dx_ceil_div(w.n, 16), most = TPW <= 4 && tiles > 2048 ? 512 : 256;
  const int each = dx_ceil_div(tiles, most);
  const dim3 grid((unsigned)dx_ceil_div(tiles, each));
  const u32x4 *codes = static_cast<const u32x4 *>(w.codes);
  if (f32)
    linear_q4_few_kernel<TPW, SPG, float>
        <<<grid, dim3(THREADS), 0, s>>>(x, codes, w.words, static_cast<float *>(y), (int)m, w.n, w.k, ldx, ldy);
  else
    linear_q4_few_kernel<TPW, SPG, uint16_t>
        <<<grid, dim3(THREADS), 0, s>>>(x, codes, w.words, static_cast<uint16_t *>(y), (int)m, w.n, w.k, ldx, ldy);
  return hipGetLastError();
}

template <int SPG>
hipError_t run_long(const Q4Weight &w, const uint16_t *x, void *y, long m, long ldx, long ldy, bool f32, hipStream_t s) {
  const dim3 grid((unsigned)dx_ceil_div(w.n, 16));
  const u32x4 *codes = static_cast<const u32x4 *>(w.codes);
  if (f32)
    linear_q4_long_kernel<SPG, float>
        <<<grid, dim3(THREADS), 0, s>>>(x, codes, w.words, static_cast<float *>(y), (int)m, w.n, w.k, ldx, ldy);
  else
    linear_q4_long_kernel<SPG, uint16_t>
        <<<grid, dim3(THREADS), 0, s>>>(x, codes, w.words, static_cast<uint16_t *>(y), (int)m, w.n, w.k, ldx, ldy);
  return hipGetLastError();
}

// Up to 16 rows: x in registers up to 8192 columns (28672 rows of W: 2048 columns 8.6 us against 13.0 with x read again,
// 8192 28 against 33), but where each workgroup has one tile of W anyway and more than 4096 columns not (3584 rows of W and
// 8192 columns, 16 rows of x: 7.3 against 6.8 read as it is multiplied; 2048 columns 3.6 against 3.7).
//
// More: tiles of 128 x 64 where there is one for every CU and more than half of their rows are in use, else eight waves a
// tile (us of the one and the other: 128 x 16384 x 3584 37 and 39, 128 x 28672 x 3584 50 and 73, 611 x 8192 x 3584 83 and
// 100, but 200 x 3584 x 4096 37 and 18, 64 x 28672 x 3584 43 and 41). These of 32 x 64, or of 32 x 32 where the smaller ones
// are no more than the CUs (17 x 3584 x 4096 9.4 and 8.0, 32 x 8192 x 3584 10.0 and 8.5, but 64 x 8192 x 3584 10.9 and 12.9).
template <int SPG>
hipError_t by_rows(const Q4Weight &w, const uint16_t *x, void *y, long m, long ldx, long ldy, bool f32, hipStream_t s) {
  const int tiles = dx_ceil_div(w.k, 128 * WAVES);  // of a wave
  if (m <= 16) {
    if (tiles <= 2) return run_few<2, SPG>(w, x, y, m, ldx, ldy, f32, s);
    if (tiles <= 4) return run_few<4, SPG>(w, x, y, m, ldx, ldy, f32, s);
    if (tiles <= 6 && w.n > 4096) return run_few<6, SPG>(w, x, y, m, ldx, ldy, f32, s);
    if (tiles <= 8 && w.n > 4096) return run_few<8, SPG>(w, x, y, m, ldx, ldy, f32, s);
    return run_long<SPG>(w, x, y, m, ldx, ldy, f32, s);
  }
  const bool many = m > 64 && (long)dx_ceil_div(w.n, 64) * dx_ceil_div(m, 128) >= 256;
  if (many) return run_many<2, 4, SPG>(w, x, y, m, ldx, ldy, f32, s);
  if ((long)dx_ceil_div(w.n, 32) * dx_ceil_div(m, 32) <= 256) return run_some<2, 2, SPG>(w, x, y, m, ldx, ldy, f32, s);
  return run_some<2, 4, SPG>(w, x, y, m, ldx, ldy, f32, s);
}

inline long tiles_of(const Q4Weight &w) { return (long)dx_ceil_div(w.n, 16) * dx_ceil_div(w.k, 128); }

}  // namespace

hipError_t dx_linear_q4_launch(const Q4Weight &w, const uint16_t *x, void *y, long m, long ldx, long ldy, bool f32,
                               hipStream_t s) {
  if (w.group == 32) return by_rows<1>(w, x, y, m, ldx, ldy, f32, s);
  if (w.group == 64) return by_rows<2>(w, x, y, m, ldx, ldy, f32, s);
  return by_rows<4>(w, x, y, m, ldx, ldy, f32, s);
}

hipError_t dx_quantize_q4_launch(const Q4Weight &w, const uint16_t *values, long ldw, hipStream_t s) {
  const long tiles = tiles_of(w);
  const dim3 grid((unsigned)dx_ceil_div(tiles, 4));
  u32x4 *codes = static_cast<u32x4 *>(w.codes);
  auto go = [&](auto kernel) { kernel<<<grid, dim3(256), 0, s>>>(values, ldw, codes, w.words, w.n, w.k, tiles); };
  if (w.group == 32) go(quantize_q4_kernel<1>);
  else if (w.group == 64) go(quantize_q4_kernel<2>);
  else go(quantize_q4_kernel<4>);
  return hipGetLastError();
}

hipError_t dx_pack_q4_launch(const Q4Weight &w, const uint8_t *code, const uint16_t *scales, bool half,
                             const uint8_t *zeros, hipStream_t s) {
  const long tiles = tiles_of(w);
  const dim3 grid((unsigned)dx_ceil_div(tiles, 4));
  u32x4 *codes = static_cast<u32x4 *>(w.codes);
  auto go = [&](auto kernel) { kernel<<<grid, dim3(256), 0, s>>>(code, scales, zeros, codes, w.words, w.n, w.k, tiles); };
  if (w.group == 32) half ? go(pack_q4_kernel<1, true>) : go(pack_q4_kernel<1, false>);
  else if (w.group == 64) half ? go(pack_q4_kernel<2, true>) : go(pack_q4_kernel<2, false>);
  else half ? go(pack_q4_kernel<4, true>) : go(pack_q4_kernel<4, false>);
  return hipGetLastError();
}

hipError_t dx_q4_values_launch(const Q4Weight &w, float *values, long ldw, hipStream_t s) {
  const long tiles = tiles_of(w);
  const dim3 grid((unsigned)dx_ceil_div(tiles, 4));
  const u32x4 *codes = static_cast<const u32x4 *>(w.codes);
  auto go = [&](auto kernel) { kernel<<<grid, dim3(256), 0, s>>>(codes, w.words, values, w.n, w.k, ldw, tiles); };
  if (w.group == 32) go(q4_values_kernel<1>);
  else if (w.group == 64) go(q4_values_kernel<2>);
  else go(q4_values_kernel<4>);
  return hipGetLastError();
}

// Log probabilities of given tokens, entropy and the best alternatives, from rows of logits.
//
// t = x, or cap tanh(x / cap) with a soft-cap (-inf stays -inf: no alternative); with M = max t,
//   S = sum e^{t - M} = 1 + R, E = sum (t - M) e^{t - M}:   log p_j = (t_j - M) - log(1 + R), H = log(1 + R) - E / (1 + R).
// R, the weights beside the largest one's own, is kept instead of S: where one token is all but certain, its log probability
// and the entropy are as small as R, which 1 + R has lost. All terms have one sign, so log p <= 0 and H >= 0.
// With a cap of up to 40, t = cap - 2 cap r with r = 1 / (1 + e^{2x / cap}), and t - M = 2 cap (r_M - r): off by a few
// roundings of the cap. Beyond, t by `capped`, off by a few of itself.
// The logits are read once. Two launches:
//   parts_kernel: a wave takes 2048 neighbouring logits of a row in registers, its M, R and E, and the largest logit of each
//     32 neighbours.
//   row_kernel: one workgroup a row joins the parts in their order and finds the alternatives from those largest ones: the
//     k-th largest of the threads' largest bounds the k best from below, so only the groups that reach it (a few more than
//     k) are looked at again, each wave keeping a sorted list of its best, one a lane.
// Chunks follow from the vocabulary alone, so a row's result does not depend on the others.
// Bound: 1500 rows of 256000 bf16 logits, soft-capped: parts 215 us (3.6 TB/s; two exponentials and a reciprocal a logit
// keep the vector units as busy as the memory), rows 23 us. One row: 4.6 and 8.2 us, loads that wait for each other.
#include "common.h"
#include "kernels.h"

namespace {

constexpr int THREADS = 256, WAVES = 4;
constexpr int CHUNK = 2048, LANE = CHUNK / 64;  // logits of a wave, of a lane
constexpr int GROUP = 32;                       // neighbouring logits with one largest value
constexpr int MOST_TOP = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// A logit as a whole number that orders as it does (-0 equals 0). NaN rows have no alternatives: any order will do.
DX_DEVICE uint32_t order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

DX_DEVICE bool by_cap(float cap) { return cap > 0.f && cap <= 40.f; }  // whether t is taken by its distance to the cap

// cap tanh(x / cap), -inf staying -inf, to a few roundings of itself: with y = x / cap the continued fraction of tanh cut
// after y^9, y (y^4 + 105 y^2 + 945) / (15 (y^4 + 28 y^2 + 63)), off by 2.4e-8 of the value at |y| <= 0.9, and the
// exponential's form beyond. One value for one x wherever it is computed: the difference of a row's largest logit to
// itself is 0 in both kernels, so no product here may join a later difference.
DX_DEVICE float capped(float x, float cap) {
#pragma clang fp contract(off)
  const float y = x * (1.f / cap), z = y * y;
  const float n = __builtin_fmaf(z + 105.f, z, 945.f), m = __builtin_fmaf(z + 28.f, z, 63.f);
  const float far = cap * copysignf(1.f - 2.f * fast_rcp(1.f + fast_exp2(2.f * LOG2E * fabsf(y))), x);
  return x == -INFINITY ? x : fabsf(y) > 0.9f ? far : x * ((1.f / 15.f) * n * fast_rcp(m));
}

// Where a logit stands: t = constant + unit level, whose differences are as accurate as said above. -inf for -inf.
DX_DEVICE float unit_of(float cap) { return by_cap(cap) ? 2.f * cap : 1.f; }
DX_DEVICE float fall(float x, float c1) { return fast_rcp(1.f + fast_exp2(c1 * x)); }  // r, with c1 = 2 log2(e) / cap
DX_DEVICE float level(float x, float cap) {
  if (cap == 0.f || x == -INFINITY) return x;
  return by_cap(cap) ? -fall(x, 2.f * LOG2E / cap) : capped(x, cap);
}

// A difference of levels, bounded below so that a weight of 0 times it is 0; NaN stays.
DX_DEVICE float below(float v, float top) {
  const float d = v - top;
  return d < -1e30f ? -1e30f : d;
}

template <int N>
struct Number {
  static constexpr int value = N;
};

// Reductions over a wave in registers, all lanes the same result: pairs, quads, eights and rows of 16 by DPP, then rows and
// halves exchanged. The largest logit is needed before the sums start: with shuffles through LDS 1500 x 256000 in bf16 take
// 225 us instead of 215, one row 13.6 instead of 12.8.
template <typename F>
DX_DEVICE float over_wave(float x, F f) {
#if defined(__HIP_DEVICE_COMPILE__)
  auto moved = [&](auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = f(x, moved(Number<0xb1>{}));   // quad_perm 1 0 3 2
  x = f(x, moved(Number<0x4e>{}));   // quad_perm 2 3 0 1
  x = f(x, moved(Number<0x141>{}));  // row_half_mirror
  x = f(x, moved(Number<0x140>{}));  // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
#endif
  return x;
}
DX_DEVICE float max_of_wave(float x) { return over_wave(x, [](float a, float b) { return fmaxf(a, b); }); }
DX_DEVICE float sum_of_wave(float x) { return over_wave(x, [](float a, float b) { return a + b; }); }

DX_DEVICE float to_float(uint16_t x) { return bf2f(x); }
DX_DEVICE float to_float(float x) { return x; }

template <typename T>
__global__ void __launch_bounds__(THREADS)
parts_kernel(const T *__restrict__ logits, int vocab, long ld, float cap, int chunks, int groups,
             float *__restrict__ parts, float *__restrict__ largest) {
  constexpr int V = 16 / sizeof(T), NV = LANE / V;  // values a 16-byte load, loads a lane
  constexpr int QUAD = GROUP / V;                   // lanes that share a group in one load
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long row = blockIdx.y;
  const int chunk = blockIdx.x * WAVES + wave;
  if (chunk >= chunks) return;
  const T *p = logits + row * ld;
  const int c0 = chunk * CHUNK;
  float x[NV][V];
  const bool whole = c0 + CHUNK <= vocab;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = c0 + (j * 64 + lane) * V;
    if (whole) {
      // rows of an odd length start anywhere: a 16-byte load needs no alignment beyond its element's
      struct __attribute__((packed, aligned(sizeof(T)))) Wide {
        u32x4 w;
      };
      const u32x4 w = reinterpret_cast<const Wide *>(p + at)->w;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (sizeof(T) == 2) x[j][i] = i & 1 ? hi_bf(w[i / 2]) : lo_bf(w[i / 2]);
        else x[j][i] = __uint_as_float(w[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[j][i] = at + i < vocab ? to_float(p[at + i]) : -INFINITY;
    }
  }
  float top = -INFINITY, low = INFINITY, mine[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float g = x[j][0];
#pragma unroll
    for (int i = 1; i < V; ++i) g = fmaxf(g, x[j][i]);
#pragma unroll
    for (int i = 0; i < V; ++i) low = fminf(low, x[j][i]);
    top = fmaxf(top, g);
#pragma unroll
    for (int off = 1; off < QUAD; off *= 2) g = fmaxf(g, __shfl_xor(g, off, 64));
    mine[j] = g;
  }
  if (largest) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int g = c0 / GROUP + (j * 64 + lane) / QUAD;
      if (lane % QUAD == 0 && g < groups) largest[row * groups + g] = mine[j];
    }
  }
  float s = 0.f, e = 0.f;
  top = max_of_wave(top);
  if (cap > 0.f) top = level(top, cap);
  const float base = top == -INFINITY ? 0.f : top, unit = unit_of(cap) * LOG2E;
  if (by_cap(cap)) {
    // u = unit (r_M - r) in one instruction, the rounding of its constant taken out of the sums afterwards
    const float c1 = 2.f * LOG2E / cap, shift = -unit * base, off = __builtin_fmaf(unit, base, shift);
    // most chunks have no -inf, and do not look for it again
    auto add = [&](auto banned) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = __builtin_fmaf(-unit, fall(x[j][i], c1), shift);
          float w = fast_exp2(u);
          if constexpr (decltype(banned)::value) w = x[j][i] == -INFINITY ? 0.f : w;
          s += w;
          e = __builtin_fmaf(w, u, e);
        }
    };
    if (__any(low == -INFINITY)) add(Number<1>{});
    else add(Number<0>{});
    const float f = fast_exp2(-off);
    e = (e - off * s) * f;
    s *= f;
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (cap > 0.f) x[j][i] = capped(x[j][i], cap);
        const float u = below(x[j][i], base) * LOG2E, w = fast_exp2(u);
        s += w;
        e = __builtin_fmaf(w, u, e);
      }
  }
  s = sum_of_wave(s);
  e = sum_of_wave(e);
  float rest = top == -INFINITY ? s : s - 1.f;  // no logit at all: 0, or NaN
  if (s < 1.0625f && top != -INFINITY) {        // the sums' roundings are too much of these: all but the largest again
    rest = e = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = below(by_cap(cap) ? level(x[j][i], cap) : x[j][i], base) * unit;
        const float w = u < 0.f ? fast_exp2(u) : 0.f;
        rest += w;
        e = __builtin_fmaf(w, u, e);
      }
    rest = sum_of_wave(rest);
    e = sum_of_wave(e);
  }
  if (lane == 0) {
    float *out = parts + (row * chunks + chunk) * 3;
    out[0] = top;
    out[1] = rest;
    out[2] = e;  // in base 2
  }
}

// The logit that order() made.
DX_DEVICE float logit_of(uint32_t v) { return __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v); }

constexpr int ROW_WAVES = 8, ROW_THREADS = 64 * ROW_WAVES;
constexpr int HELD = 16;  // groups that a thread keeps in registers: all of them up to a vocabulary of 262144

// The workgroup's sums of three numbers a thread, in the waves' order.
DX_DEVICE void block_sums(float (&x)[3], float (&red)[3][ROW_WAVES]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    x[i] = sum_of_wave(x[i]);
    if ((threadIdx.x & 63) == 0) red[i][threadIdx.x >> 6] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    x[i] = 0.f;
#pragma unroll
    for (int w = 0; w < ROW_WAVES; ++w) x[i] += red[i][w];
  }
}

DX_DEVICE uint64_t from_lane(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}

// Each lane its lower neighbour's value (lane 0 anything).
DX_DEVICE uint64_t from_below(uint64_t v) {
  constexpr int SHIFT = 0x138;  // DPP: the whole wave by one lane
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, SHIFT, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), SHIFT, 0xf, 0xf, false);
  return (uint64_t)hi << 32 | lo;
}

// Insert v (the same in all lanes) into the wave's list, lane i its i-th largest; the last one falls off.
DX_DEVICE void insert(uint64_t &list, uint64_t v, int lane) {
  const uint64_t above = from_below(list);
  const bool moves = list < v;
  list = moves ? (lane == 0 || above >= v ? v : above) : list;
}

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS)
row_kernel(const T *__restrict__ logits, const int32_t *__restrict__ targets, int vocab, long ld, float cap, int top,
           int chunks, int groups, const float *__restrict__ parts, const float *__restrict__ largest,
           float *__restrict__ logprobs, float *__restrict__ entropy, int32_t *__restrict__ ids,
           float *__restrict__ top_logprobs) {
  __shared__ float red[3][ROW_WAVES], reds[ROW_WAVES];
  __shared__ uint32_t lane_best[ROW_THREADS];
  __shared__ uint64_t reach[ROW_WAVES][HELD];
  __shared__ uint64_t best[ROW_WAVES][MOST_TOP];
  const long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T *p = logits + row * ld;
  const float *part = parts + row * chunks * 3, *big = largest + row * groups;

  // What is known to be needed is asked for at once: a kernel's first loads come from memory, some 2 us each if one waits
  // for the other (this row, its target's logit, its parts and groups in turn made a single row 14 us).
  const int target = targets[row];
  const float target_logit = to_float(p[min(max(target, 0), vocab - 1)]);
  float first[3] = {-INFINITY, 0.f, 0.f};  // this thread's first part
  if (tid < chunks) {
#pragma unroll
    for (int i = 0; i < 3; ++i) first[i] = part[tid * 3 + i];
  }
  // a thread's groups are tid, tid + 512, ...
  constexpr int BLOCK = HELD * ROW_THREADS;
  const int blocks = (groups + BLOCK - 1) / BLOCK;
  uint32_t v[HELD];
  auto hold = [&](int block) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int i = block * BLOCK + j * ROW_THREADS + tid;
      const uint32_t x = order(big[min(i, groups - 1)]);  // no branch: sixteen loads on their way at once
      v[j] = i < groups ? x : 0;
    }
  };
  if (top > 0) {
    uint32_t mine = 0;
    for (int block = 0; block < blocks; ++block) {
      hold(block);
#pragma unroll
      for (int j = 0; j < HELD; ++j) mine = max(mine, v[j]);
    }
    lane_best[tid] = mine;
  }
  // join: every thread the same highest level, then sums in the threads' order
  float most = first[0];
  for (int i = tid + ROW_THREADS; i < chunks; i += ROW_THREADS) most = fmaxf(most, part[i * 3]);
  most = max_of_wave(most);
  if (lane == 0) reds[wave] = most;
  __syncthreads();
  most = reds[0];
#pragma unroll
  for (int w = 1; w < ROW_WAVES; ++w) most = fmaxf(most, reds[w]);
  const float unit = unit_of(cap);
  float sums[3] = {0.f, 0.f, 0.f};  // of R, of E, and of the parts that hold the largest t: one 1 of theirs is 1 + R's
  auto add = [&](float top_i, float rest_i, float e_i) {
    if (top_i == -INFINITY) {
      sums[0] += rest_i;  // 0, or NaN
      return;
    }
    // a part of masked logits may lie as far below as numbers go
    const bool holds = top_i == most;
    const float d = below(top_i, most) * unit * LOG2E, f = fast_exp2(d);
    sums[0] += holds ? rest_i : (1.f + rest_i) * f;
    sums[1] += f * (e_i + (1.f + rest_i) * d);
    sums[2] += holds ? 1.f : 0.f;
  };
  add(first[0], first[1], first[2]);
  for (int i = tid + ROW_THREADS; i < chunks; i += ROW_THREADS) add(part[i * 3], part[i * 3 + 1], part[i * 3 + 2]);
  block_sums(sums, red);
  // no finite logit at all: no token has any probability
  const bool empty = most == -INFINITY && sums[0] == 0.f, lost = sums[0] != sums[0];
  const float rest = sums[0] + (sums[2] - 1.f), log_s = log1pf(rest), e = sums[1] * LN2;
  if (tid == 0) {
    float lp = 0.f;
    if (target < -1 || target >= vocab) lp = NAN;
    else if (target >= 0) lp = empty ? -INFINITY : (level(target_logit, cap) - most) * unit - log_s;
    logprobs[row] = lost && target != -1 ? NAN : lp;
    entropy[row] = lost ? NAN : empty ? 0.f : log_s - e / (1.f + rest);
  }
  if (top == 0) return;
  int32_t *out = ids + row * top;
  float *out_lp = top_logprobs + row * top;
  if (empty || lost) {
    for (int i = tid; i < top; i += ROW_THREADS) {
      out[i] = -1;
      out_lp[i] = lost ? NAN : -INFINITY;
    }
    return;
  }
  // The `top`-th largest of the threads' largest logits, bit by bit from the top: that many logits are as large, so the
  // best ones are, and only groups that reach it are looked at. (Fewer threads with groups than `top`: all groups.) Half
  // the bits, 0.1 us each, are near enough: 8 of a mantissa.
  uint32_t least = 0;
  {
    uint32_t x[ROW_WAVES];
#pragma unroll
    for (int w = 0; w < ROW_WAVES; ++w) x[w] = lane_best[w * 64 + lane];
    for (int bit = 31; bit >= 15; --bit) {
      const uint32_t cand = least | (1u << bit);
      int c = 0;
#pragma unroll
      for (int w = 0; w < ROW_WAVES; ++w) c += __popcll(__ballot(x[w] >= cand));
      if (c >= top) least = cand;
    }
  }
  // a wave's own best, over its share of the groups, two groups of 32 at a time
  uint64_t list = 0;
  auto look = [&](int g0, int g1) {  // g1 = g0: one group
    const int g = lane < 32 ? g0 : g1, token = g * GROUP + (lane & 31);
    uint64_t key = 0;
    if (token < vocab && (lane < 32 || g1 != g0))
      key = ((uint64_t)order(to_float(p[token])) << 32) | (uint32_t)~token;
    uint64_t in = __ballot(key > from_lane(list, top - 1) && (uint32_t)(key >> 32) >= least);
    while (in) {
      const int src = __ffsll((unsigned long long)in) - 1;
      in &= in - 1;
      insert(list, from_lane(key, src), lane);
    }
  };
  int held = -1;  // a group that waits for a second one
  for (int block = blocks - 1; block >= 0; --block) {
    if (block < blocks - 1) hold(block);  // the last one still is
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const uint64_t in = __ballot(v[j] >= least && v[j] != 0);
      if (lane == 0) reach[wave][j] = in;
    }
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < HELD; ++j) {
      uint64_t in = from_lane(reach[wave][j], 0);
      while (in) {
        const int g = block * BLOCK + j * ROW_THREADS + wave * 64 + __ffsll((unsigned long long)in) - 1;
        in &= in - 1;
        if (held < 0) {
          held = g;
        } else {
          look(held, g);
          held = -1;
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (held >= 0) look(held, held);
  best[wave][lane] = lane < top ? list : 0;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < ROW_WAVES; ++w) {
    const uint64_t theirs = best[w][lane];
    for (int i = 0; i < top; ++i) {
      const uint64_t v = from_lane(theirs, i);
      if (v <= from_lane(list, top - 1)) break;  // the rest is smaller still
      insert(list, v, lane);
    }
  }
  if (lane < top) {
    const int token = (int)~(uint32_t)list;
    const bool none = list == 0 || (uint32_t)(list >> 32) <= order(-INFINITY);
    out[lane] = none ? -1 : token;
    out_lp[lane] = none ? -INFINITY : (level(logit_of((uint32_t)(list >> 32)), cap) - most) * unit - log_s;
  }
}

}  // namespace

hipError_t dx_token_logprobs_launch(const void *logits, const int32_t *targets, long rows, int vocab, long ld, float cap,
                                    int top, float *logprobs, float *entropy, int32_t *ids, float *top_logprobs,
                                    float *parts, float *groups, bool f32, hipStream_t s) {
  const int chunks = (vocab + CHUNK - 1) / CHUNK, ngroups = (vocab + GROUP - 1) / GROUP;
  // rows beyond a grid's y dimension go in further launches
  for (long r0 = 0; r0 < rows; r0 += 65535) {
    const dim3 grid((chunks + WAVES - 1) / WAVES, (unsigned)min(rows - r0, 65535L));
    float *pr = parts + r0 * chunks * 3, *gr = top > 0 ? groups + r0 * ngroups : nullptr;
    if (f32)
      parts_kernel<<<grid, dim3(THREADS), 0, s>>>(static_cast<const float *>(logits) + r0 * ld, vocab, ld, cap, chunks,
                                                  ngroups, pr, gr);
    else
      parts_kernel<<<grid, dim3(THREADS), 0, s>>>(static_cast<const uint16_t *>(logits) + r0 * ld, vocab, ld, cap,
                                                  chunks, ngroups, pr, gr);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  // a launch's threads are counted in 32 bits
  constexpr long MOST_ROWS = (1L << 32) / ROW_THREADS / 2;
  for (long r0 = 0; r0 < rows; r0 += MOST_ROWS) {
    const dim3 grid((unsigned)min(rows - r0, MOST_ROWS)), block(ROW_THREADS);
    const float *pr = parts + r0 * chunks * 3, *gr = groups + (top > 0 ? r0 * ngroups : 0);
    int32_t *id = top > 0 ? ids + r0 * top : nullptr;
    float *tl = top > 0 ? top_logprobs + r0 * top : nullptr;
    if (f32)
      row_kernel<<<grid, block, 0, s>>>(static_cast<const float *>(logits) + r0 * ld, targets + r0, vocab, ld, cap, top, chunks,
                                        ngroups, pr, gr, logprobs + r0, entropy + r0, id, tl);
    else
      row_kernel<<<grid, block, 0, s>>>(static_cast<const uint16_t *>(logits) + r0 * ld, targets + r0, vocab, ld, cap, top,
                                        chunks, ngroups, pr, gr, logprobs + r0, entropy + r0, id, tl);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

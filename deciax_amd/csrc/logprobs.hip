// Log probabilities of given tokens, entropy and the best alternatives, from rows of logits.
//
// t = x, or cap tanh(x / cap) with a soft-cap (-inf stays -inf: no alternative); with M >= max t,
//   S = sum e^{t - M}, E = sum (t - M) e^{t - M}:   log p_j = (t_j - M) - log S,   H = log S - E / S.
// The logits are read once. Two launches:
//   parts_kernel: a wave takes 2048 neighbouring logits of a row in registers, its M (with a cap of up to 40, where e^{-2
//     cap} is well above the smallest numbers, the cap itself: t - cap = -2 cap / (1 + e^{2x / cap}); else its largest t),
//     S and E, and the largest logit of each 32 neighbours.
//   row_kernel: one workgroup a row joins the parts in their order and finds the alternatives from those largest ones: the
//     k-th largest of the threads' largest bounds the k best from below, so only the groups that reach it (a few more than
//     k) are looked at again, each wave keeping a sorted list of its best, one a lane.
// Chunks follow from the vocabulary alone, so a row's result does not depend on the others.
// Bound: 1500 rows of 256000 bf16 logits, soft-capped: parts 200 us (3.9 TB/s; two exponentials and a reciprocal a logit
// keep the vector units as busy as the memory), rows 22 us. One row: 4.3 and 7.6 us, loads that wait for each other.
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

DX_DEVICE bool by_cap(float cap) { return cap > 0.f && cap <= 40.f; }  // whether M is the cap

// cap tanh(x / cap), -inf staying -inf, to a few roundings of itself: with y = x / cap the continued fraction of tanh cut
// after y^9, y (y^4 + 105 y^2 + 945) / (15 (y^4 + 28 y^2 + 63)), off by 2.4e-8 of the value at |y| <= 0.9, and the
// exponential's form beyond.
DX_DEVICE float capped(float x, float cap) {
  const float y = x * (1.f / cap), z = y * y;
  const float n = __builtin_fmaf(z + 105.f, z, 945.f), m = __builtin_fmaf(z + 28.f, z, 63.f);
  const float far = cap * copysignf(1.f - 2.f * fast_rcp(1.f + fast_exp2(2.f * LOG2E * fabsf(y))), x);
  return x == -INFINITY ? x : fabsf(y) > 0.9f ? far : x * ((1.f / 15.f) * n * fast_rcp(m));
}

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

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
  float shift = cap, s = 0.f, e = 0.f;
  if (by_cap(cap)) {
    // 1.5 of some 19 vector instructions' time a logit (three are transcendental, four each), 1500 x 256000 in bf16: a
    // chunk without -inf, most are, does not look for it again
    const float c1 = 2.f * LOG2E / cap, c2 = -2.f * LOG2E * cap;
    auto add = [&](auto banned) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = c2 * fast_rcp(1.f + fast_exp2(c1 * x[j][i]));
          float w = fast_exp2(u);
          if constexpr (decltype(banned)::value) w = x[j][i] == -INFINITY ? 0.f : w;
          s += w;
          e = __builtin_fmaf(w, u, e);
        }
    };
    if (__any(low == -INFINITY)) add(Flag<true>{});
    else add(Flag<false>{});
  } else {
    if (cap > 0.f) {
      top = -INFINITY;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[j][i] = capped(x[j][i], cap);
          top = fmaxf(top, x[j][i]);
        }
    }
    shift = wave_max(top);
    const float base = shift == -INFINITY ? 0.f : shift;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = fmaxf(x[j][i] - base, -1e30f) * LOG2E;
        const float w = fast_exp2(u);
        s += w;
        e = __builtin_fmaf(w, u, e);
      }
    // fmaxf passes over a NaN: keep it (and inf - inf)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s = x[j][i] != x[j][i] ? NAN : s;
    if (base == INFINITY) s = NAN;
  }
  s = wave_sum(s);
  e = wave_sum(e);
  if (lane == 0) {
    float *out = parts + (row * chunks + chunk) * 3;
    out[0] = shift;
    out[1] = s;
    out[2] = e;  // in base 2
  }
}

// The logit that order() made.
DX_DEVICE float logit_of(uint32_t v) { return __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v); }

// t - shift of a logit, as accurate as parts_kernel's sum is.
DX_DEVICE float shifted(float x, float cap, float shift) {
  if (x == -INFINITY) return -INFINITY;
  if (by_cap(cap)) return -2.f * cap / (1.f + expf(2.f * x / cap));
  return (cap > 0.f ? capped(x, cap) : x) - shift;
}

constexpr int ROW_WAVES = 8, ROW_THREADS = 64 * ROW_WAVES;
constexpr int HELD = 16;  // groups that a thread keeps in registers: all of them up to a vocabulary of 262144

// The workgroup's sums of a and of b, in the waves' order.
DX_DEVICE void block_sums(float &a, float &b, float (&red)[2][ROW_WAVES]) {
  a = wave_sum(a);
  b = wave_sum(b);
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = a;
    red[1][threadIdx.x >> 6] = b;
  }
  __syncthreads();
  a = b = 0.f;
#pragma unroll
  for (int w = 0; w < ROW_WAVES; ++w) {
    a += red[0][w];
    b += red[1][w];
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
  __shared__ float red[2][ROW_WAVES], reds[ROW_WAVES];
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
  // join: every thread the same largest shift, then sums in the threads' order
  float shift = cap;
  if (!by_cap(cap)) {
    float m = first[0];
    for (int i = tid + ROW_THREADS; i < chunks; i += ROW_THREADS) m = fmaxf(m, part[i * 3]);
    m = wave_max(m);
    if (lane == 0) reds[wave] = m;
    __syncthreads();
    shift = reds[0];
#pragma unroll
    for (int w = 1; w < ROW_WAVES; ++w) shift = fmaxf(shift, reds[w]);
  }
  float s = 0.f, e = 0.f;
  auto add = [&](float top_i, float s_i, float e_i) {
    // a part of masked logits may lie as far below as numbers go: the same bound as a logit's there
    const float d = top_i == -INFINITY ? 0.f : top_i - shift < -1e30f ? -1e30f : (top_i - shift) * LOG2E;
    const float f = fast_exp2(d), si = s_i * f;
    s += si;
    e += e_i * f + si * d;
  };
  add(first[0], first[1], first[2]);
  for (int i = tid + ROW_THREADS; i < chunks; i += ROW_THREADS) add(part[i * 3], part[i * 3 + 1], part[i * 3 + 2]);
  block_sums(s, e, red);
  e *= LN2;
  // no finite logit at all: no token has any probability
  const bool empty = s == 0.f, lost = s != s;
  const float log_s = logf(s);
  if (tid == 0) {
    float lp = 0.f;
    if (target < -1 || target >= vocab) lp = NAN;
    else if (target >= 0) lp = empty ? -INFINITY : shifted(target_logit, cap, shift) - log_s;
    logprobs[row] = lost && target != -1 ? NAN : lp;
    entropy[row] = lost ? NAN : empty ? 0.f : log_s - e / s;
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
    out_lp[lane] = none ? -INFINITY : shifted(logit_of((uint32_t)(list >> 32)), cap, shift) - log_s;
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
  if (f32)
    row_kernel<<<dim3((unsigned)rows), dim3(ROW_THREADS), 0, s>>>(static_cast<const float *>(logits), targets, vocab, ld,
                                                              cap, top, chunks, ngroups, parts, groups, logprobs,
                                                              entropy, ids, top_logprobs);
  else
    row_kernel<<<dim3((unsigned)rows), dim3(ROW_THREADS), 0, s>>>(static_cast<const uint16_t *>(logits), targets, vocab, ld,
                                                              cap, top, chunks, ngroups, parts, groups, logprobs,
                                                              entropy, ids, top_logprobs);
  return hipGetLastError();
}

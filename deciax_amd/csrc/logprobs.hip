// Log probabilities of given tokens, entropy and the best alternatives, from rows of logits.
//
// t = x, or cap tanh(x / cap) with a soft-cap (-inf stays -inf: no alternative); with M >= max t,
//   S = sum e^{t - M}, E = sum (t - M) e^{t - M}:   log p_j = (t_j - M) - log S,   H = log S - E / S.
// The logits are read once. Two launches:
//   parts_kernel: a wave takes 2048 neighbouring logits of a row in registers, its M (the shift is the cap itself with
//     one: t - cap = -2 cap / (1 + e^{2x / cap}), which keeps its relative precision where the weight is), S and E, and
//     the largest logit of each 32 neighbours.
//   row_kernel: one workgroup a row joins the parts in their order and finds the alternatives from those largest ones:
//     with k alternatives wanted, their k-th largest value L bounds what can be among the k best from below, so only the
//     groups above L (fewer than k) and the first k groups that equal L are looked at again.
// Chunks follow from the vocabulary alone, so a row's result does not depend on the others.
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
  float top = -INFINITY, mine[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float g = x[j][0];
#pragma unroll
    for (int i = 1; i < V; ++i) g = fmaxf(g, x[j][i]);
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
  if (cap > 0.f) {
    const float c1 = 2.f * LOG2E / cap, c2 = -2.f * LOG2E * cap;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = c2 * fast_rcp(1.f + fast_exp2(c1 * x[j][i]));
        const float w = x[j][i] == -INFINITY ? 0.f : fast_exp2(u);
        s += w;
        e = __builtin_fmaf(w, u, e);
      }
  } else {
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

DX_DEVICE float block_sum(float v, float *red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

DX_DEVICE int block_count(int wave_count, int *red) {
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = wave_count;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// t - shift of a logit, as accurate as parts_kernel's sum is.
DX_DEVICE float shifted(float x, float cap, float shift) {
  if (x == -INFINITY) return -INFINITY;
  return cap > 0.f ? -2.f * cap / (1.f + expf(2.f * x / cap)) : x - shift;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
row_kernel(const T *__restrict__ logits, const int32_t *__restrict__ targets, int vocab, long ld, float cap, int top,
           int chunks, int groups, const float *__restrict__ parts, const float *__restrict__ largest,
           float *__restrict__ logprobs, float *__restrict__ entropy, int32_t *__restrict__ ids,
           float *__restrict__ top_logprobs) {
  __shared__ float red[WAVES];
  __shared__ int redi[WAVES];
  __shared__ int found[2 * MOST_TOP];
  __shared__ uint64_t best[WAVES][MOST_TOP];
  const long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T *p = logits + row * ld;
  const float *part = parts + row * chunks * 3;
  // join: every thread the same largest shift, then sums in the threads' order
  float shift = cap;
  if (!(cap > 0.f)) {
    float m = -INFINITY;
    for (int i = tid; i < chunks; i += THREADS) m = fmaxf(m, part[i * 3]);
    m = wave_max(m);
    if (lane == 0) red[wave] = m;
    __syncthreads();
    shift = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  }
  float s = 0.f, e = 0.f;
  for (int i = tid; i < chunks; i += THREADS) {
    const float d = part[i * 3] == -INFINITY ? 0.f : (part[i * 3] - shift) * LOG2E;
    const float f = fast_exp2(d), si = part[i * 3 + 1] * f;
    s += si;
    e += part[i * 3 + 2] * f + si * d;
  }
  s = block_sum(s, red);
  e = block_sum(e, red) * LN2;
  // no finite logit at all: no token has any probability
  const bool empty = s == 0.f, lost = s != s;
  const float log_s = logf(s);
  if (tid == 0) {
    const int target = targets[row];
    float lp = 0.f;
    if (target < -1 || target >= vocab) lp = NAN;
    else if (target >= 0) lp = empty ? -INFINITY : shifted(to_float(p[target]), cap, shift) - log_s;
    logprobs[row] = lost && target != -1 ? NAN : lp;
    entropy[row] = lost ? NAN : empty ? 0.f : log_s - e / s;
  }
  if (top == 0) return;
  int32_t *out = ids + row * top;
  float *out_lp = top_logprobs + row * top;
  if (empty || lost) {
    for (int i = tid; i < top; i += THREADS) {
      out[i] = -1;
      out_lp[i] = lost ? NAN : -INFINITY;
    }
    return;
  }
  // the k-th largest of the groups' largest, bit by bit
  const float *big = largest + row * groups;
  const int k = min(top, groups);
  uint32_t least = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = least | (1u << bit);
    int c = 0;
    for (int i = tid; i < groups; i += THREADS) c += order(big[i]) >= cand;
    c = (int)wave_sum((float)c);
    if (block_count(c, redi) >= k) least = cand;
  }
  // groups above it in any order, then the first k that equal it: thread t looks at groups t, t + 256, ...
  int have = 0;  // entries of found
  int equal = 0;
  for (int i0 = 0; i0 < groups; i0 += THREADS) {
    const int i = i0 + tid;
    const uint32_t v = i < groups ? order(big[i]) : 0u;
    const bool more = i < groups && v > least, same = i < groups && v == least;
    const uint64_t bm = __ballot(more), bs = __ballot(same), lower = (1ull << lane) - 1;
    __syncthreads();
    if (lane == 0) {
      redi[wave] = __popcll(bm) | (__popcll(bs) << 16);
    }
    __syncthreads();
    int um = 0, us = 0, am = 0, as = 0;
    for (int w = 0; w < WAVES; ++w) {
      const int x = redi[w];
      um += w < wave ? x & 0xffff : 0;
      us += w < wave ? x >> 16 : 0;
      am += x & 0xffff;
      as += x >> 16;
    }
    if (more) found[have + um + __popcll(bm & lower)] = i;
    const int rank = equal + us + __popcll(bs & lower);
    if (same && rank < k) found[2 * MOST_TOP - 1 - rank] = i;
    have += am;
    equal += as;
  }
  __syncthreads();
  const int tied = min(equal, k), cands = have + tied;
  // each wave the best of its share of the groups: lane i holds the i-th best as (logit, lower token first)
  uint64_t list = 0;
  const uint32_t floor = top <= groups ? least : 0;  // that many groups have a logit this large
  for (int c = wave; c < (cands + 1) / 2; c += WAVES) {  // two groups of 32 at a time
    const int which = c * 2 + (lane >> 5);
    uint64_t key = 0;
    if (which < cands) {
      const int g = which < have ? found[which] : found[2 * MOST_TOP - 1 - (which - have)];
      const int token = g * GROUP + (lane & 31);
      if (token < vocab) key = ((uint64_t)order(to_float(p[token])) << 32) | (uint32_t)~token;
    }
    uint64_t worst = __shfl(list, top - 1, 64);
    uint64_t in = __ballot(key > worst && (uint32_t)(key >> 32) >= floor);
    while (in) {
      const int src = __ffsll((unsigned long long)in) - 1;
      in &= in - 1;
      const uint64_t v = __shfl(key, src, 64);
      const uint64_t above = __shfl_up(list, 1, 64);
      // lanes whose entry is below v move down by one
      const bool below = list < v;
      const bool first = below && (lane == 0 || above >= v);
      list = first ? v : below ? above : list;
    }
  }
  if (lane < MOST_TOP) best[wave][lane] = lane < top ? list : 0;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < WAVES; ++w)
    for (int i = 0; i < top; ++i) {
      const uint64_t v = best[w][i];
      if (v == 0 || v <= __shfl(list, top - 1, 64)) break;
      const uint64_t above = __shfl_up(list, 1, 64);
      const bool below = list < v;
      const bool first = below && (lane == 0 || above >= v);
      list = first ? v : below ? above : list;
    }
  if (lane < top) {
    const int token = (int)~(uint32_t)list;
    const bool none = list == 0 || (uint32_t)(list >> 32) <= order(-INFINITY);
    out[lane] = none ? -1 : token;
    out_lp[lane] = none ? -INFINITY : shifted(to_float(p[token]), cap, shift) - log_s;
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
    row_kernel<<<dim3((unsigned)rows), dim3(THREADS), 0, s>>>(static_cast<const float *>(logits), targets, vocab, ld,
                                                              cap, top, chunks, ngroups, parts, groups, logprobs,
                                                              entropy, ids, top_logprobs);
  else
    row_kernel<<<dim3((unsigned)rows), dim3(THREADS), 0, s>>>(static_cast<const uint16_t *>(logits), targets, vocab, ld,
                                                              cap, top, chunks, ngroups, parts, groups, logprobs,
                                                              entropy, ids, top_logprobs);
  return hipGetLastError();
}

// Linear attention with a decay for each token and head, over packed sequences with a kept state:
//   S_t = e^g_t S_(t-1) + k_t v_t^T,   o_t = scale q_t S_t,   S [DK, DV] fp32.
//
// In chunks: with G_i the sum of g over the chunk's tokens up to i,
//   o_i = scale (e^G_i q_i S + sum_(j <= i) e^(G_i - G_j) (q_i . k_j) v_j),   S' = e^G_C S + sum_j e^(G_C - G_j) k_j v_j^T.
// Sums and differences of g are taken in 64 bits: behind a strong decay they are small differences of large numbers. The
// state is multiplied by e^G_C as a sum of two floats: rounded to one, the same error in every chunk of a head of constant
// decay adds up over all the chunks that the state remembers.
//
// A long sequence is cut into segments (linear_attention_plan.h): kernel 1 finds what each adds to the state, kernel 2
// joins them to every segment's start, kernel 3 runs each from there. The cut follows from the sequence's own length, so a
// result does not depend on the batch.
#include "common.h"
#include "kernels.h"
#include "linear_attention_plan.h"

namespace {

constexpr int THREADS = 256, COLS = 64;  // columns of the state a workgroup has
constexpr float NO_DECAY_BELOW = -1e4f;  // e^g is 0 from there on, and sums of g stay exact enough

struct Sequence {
  long start, slot;  // first packed row, state (-1: none)
  int len;
};

// A sequence that reaches outside the packed rows has none.
DX_DEVICE Sequence sequence(const LinearAttn &a, int b) {
  Sequence s;
  s.start = a.seq_start[b];
  s.len = min(max(a.seq_len[b], 0), a.max_len);
  if (s.start < 0 || s.start + s.len > a.rows) s.len = 0;
  s.slot = a.index ? a.index[b] : b;
  if (s.slot < 0 || s.slot >= a.slots) s.slot = -1;
  return s;
}

// The head and the first column of a workgroup that has W of them. Those that read the same rows of q and k are hk apart
// in the grid: where hk is a multiple of 8, on the same XCD, whose L2 holds the rows.
struct Unit {
  int head, col0;
};
template <int W>
DX_DEVICE Unit unit(const LinearAttn &a) {
  const int kh = blockIdx.x % a.hk, rest = blockIdx.x / a.hk, blocks = a.dv / W;
  return Unit{kh * (a.h / a.hk) + rest / blocks, rest % blocks * W};
}

DX_DEVICE float decay_of(float g) { return g < NO_DECAY_BELOW ? NO_DECAY_BELOW : g; }

template <typename T>
DX_DEVICE float value(const T *p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}
template <typename T>
DX_DEVICE void put(T *p, float x) {
  if constexpr (sizeof(T) == 2) *p = f2bf(x);
  else *p = x;
}

// x = e^g as the sum of two floats.
struct Factor {
  float hi, lo;
};
DX_DEVICE Factor factor_of(double g) {
  const double e = exp(g);
  const float hi = (float)e;
  return Factor{hi, hi < INFINITY ? (float)(e - (double)hi) : 0.f};  // NaN and infinity as they are
}
DX_DEVICE float times(float x, Factor f) { return fmaf(x, f.hi, x * f.lo); }

// Token by token: thread 16 r + c of 256 has four columns and the rows r, r + 16, .., all fp32. Bound by the state, read and
// written once: 48 sequences of 1 token, 32 heads of 128 by 128 (202 MB) 42 us, 4.8 TB/s.
template <int DK>
constexpr int STEP_LDS = 2 * DK + 4 * COLS;  // floats
template <typename T, int DK>
DX_DEVICE void step_body(const LinearAttn &a, const Sequence &s, int head, int col0, float *lds) {
  constexpr int R = DK / 16;
  float *kq = lds;                    // [2][DK]
  float *part = lds + 2 * DK;         // [4 waves][COLS]
  const int tid = threadIdx.x % THREADS, c = tid & 15, r = tid >> 4, wave = tid >> 6;
  const int kh = head / (a.h / a.hk);
  const long at = ((s.slot * a.h + head) * DK + r) * (long)a.dv + col0 + 4 * c;
  floatx4 st[R];
#pragma unroll
  for (int i = 0; i < R; ++i) st[i] = floatx4{0, 0, 0, 0};
  if (s.slot >= 0)  // one branch around all loads
#pragma unroll
    for (int i = 0; i < R; ++i) st[i] = *reinterpret_cast<const floatx4 *>(a.state_in + at + 16L * i * a.dv);
  for (int t = 0; t < s.len; ++t) {
    const long row = s.start + t;
    const T *q = static_cast<const T *>(a.q) + row * a.qs + kh * DK, *k = static_cast<const T *>(a.k) + row * a.ks + kh * DK;
    if (t > 0) __syncthreads();
    for (int i = tid; i < 2 * DK; i += THREADS) kq[i] = i < DK ? value(k + i) : value(q + i - DK);
    const T *v = static_cast<const T *>(a.v) + row * a.vs + head * a.dv + col0 + 4 * c;
    floatx4 vv;
#pragma unroll
    for (int e = 0; e < 4; ++e) vv[e] = value(v + e);
    const Factor d = factor_of((double)decay_of(a.decay[row * a.ds + head]));
    __syncthreads();
    floatx4 o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float kk = kq[r + 16 * i], qq = kq[DK + r + 16 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[i][e] = fmaf(kk, vv[e], times(st[i][e], d));
        o[e] = fmaf(qq, st[i][e], o[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += __shfl_xor(o[e], 16, 64);
      o[e] += __shfl_xor(o[e], 32, 64);
    }
    if ((tid & 63) < 16) *reinterpret_cast<floatx4 *>(part + wave * COLS + 4 * c) = o;
    __syncthreads();
    if (tid < COLS)
      put(static_cast<T *>(a.out) + row * a.os + head * a.dv + col0 + tid,
          a.scale * ((part[tid] + part[COLS + tid]) + (part[2 * COLS + tid] + part[3 * COLS + tid])));
  }
  if (s.slot >= 0)
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<floatx4 *>(a.state_out + at + 16L * i * a.dv) = st[i];
}

template <typename T, int DK>
__global__ void __launch_bounds__(THREADS) step_kernel(LinearAttn a) {
  __shared__ __align__(16) float lds[STEP_LDS<DK>];
  const int blocks = a.dv / COLS;
  step_body<T, DK>(a, sequence(a, blockIdx.y), blockIdx.x / blocks, blockIdx.x % blocks * COLS, lds);
}

// A barrier for what went through LDS alone: loads of the next chunk stay on their way.
DX_DEVICE void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ------------------------------------------------------------------------------------------ fp32, chunks of 32 tokens
//
// fp32 products (v_mfma_f32_16x16x4_f32: lane l has row or column l % 16 of an operand and k l / 16, and of the result
// column l % 16, rows 4 (l / 16) + r). Four products take 16 k, of which group l / 16 has 4 (l / 16) .. + 3: rows of LDS are
// read 16 bytes a lane, and a result tile is the four second operands of the next product as it lies. Wave w has the
// columns 16 w .. of the state, in registers. Bound by the chain of a sequence's chunks, of which one is 2.3 to 2.9 us at keys of
// 64 dimensions: rows are asked for a chunk ahead. 4161 tokens of 3 heads of 64 by 256 60 us, 2111 of 32 heads of 128 by 128
// 144; 5 sequences of 3 to 37 tokens 10.
DX_DEVICE floatx4 mfma_f32(float x, float y, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0); }

// Rows as a buffer of n of them: those behind read as zeros and are not written, without a branch. An offset stays below
// 2^31, since strides are below 2^24.
DX_DEVICE __amdgpu_buffer_rsrc_t rows_of(const void *first, int n, long stride_bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)first, (short)0, (int)(n * stride_bytes), 0x00020000);
}

// What a chunk's decays come to, found by one wave: lane i has token i. Powers of two.
struct Sums {
  double upto, end;  // of this lane's token and of the chunk
};
template <int N>
DX_DEVICE Sums sum_of(float g) {
  const int lane = threadIdx.x & 63;
  double sum = (double)decay_of(g) * 1.4426950408889634;
#pragma unroll
  for (int off = 1; off < N; off <<= 1) {
    const double y = __shfl_up(sum, off, 64);
    if (lane >= off) sum += y;
  }
  return Sums{sum, __shfl(sum, N - 1, 64)};
}

template <int DK>
struct alignas(16) Chunk {
  static constexpr int TOKENS = 32, W = DK + 4, VW = COLS + 4, PW = TOKENS + 4;  // rows 16 bytes on: on other banks
  float q[TOKENS][W], k[TOKENS][W], v[TOKENS][VW], p[TOKENS][PW];
  struct Decay {
    double sum[TOKENS], total;
    float from_start[TOKENS], to_end[TOKENS];  // 2^G_i, 2^(G_C - G_j)
    Factor all;
  } decay[2];  // this chunk's and the next one's
  int lost[2];  // whether a value is no finite number
  static_assert(W % 4 == 0 && VW % 4 == 0 && PW % 4 == 0, "rows are read and written 16 bytes at a time");
};
static_assert(alignof(Chunk<64>) % 16 == 0 && alignof(Chunk<128>) % 16 == 0 && alignof(Chunk<256>) % 16 == 0,
              "rows are read and written 16 bytes at a time");

// The wave's columns of the state: tile i has rows 16 i + 4 (l / 16) + r, column 16 wave + l % 16.
DX_DEVICE long state_at(const LinearAttn &a, int i, int r, int col0) {
  const int lane = threadIdx.x & 63;
  return (long)(16 * i + 4 * (lane >> 4) + r) * a.dv + col0 + 16 * (threadIdx.x >> 6) + (lane & 15);
}

// A chunk's rows on their way from memory.
template <int DK, bool OUT>
struct FetchedF32 {
  static constexpr int KI = DK / 32, KR = 4 * THREADS / DK, VR = 4 * THREADS / COLS;  // loads of q and k; rows a load
  floatx4 q[OUT ? KI : 1], k[KI], v[2];

  DX_DEVICE void load(const LinearAttn &a, long row, int n, int head, int kh, int col0) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t tid = threadIdx.x, kr = tid / (DK / 4), kc = 16 * (tid % (DK / 4)), vr = tid / 16, vc = 16 * (tid % 16);
    const uint32_t qs = 4 * (uint32_t)a.qs, ks = 4 * (uint32_t)a.ks, vs = 4 * (uint32_t)a.vs;
    const auto qp = rows_of(static_cast<const float *>(a.q) + row * a.qs + kh * DK, n, 4 * a.qs);
    const auto kp = rows_of(static_cast<const float *>(a.k) + row * a.ks + kh * DK, n, 4 * a.ks);
    const auto vp = rows_of(static_cast<const float *>(a.v) + row * a.vs + head * a.dv + col0, n, 4 * a.vs);
    auto at = [](__amdgpu_buffer_rsrc_t from, uint32_t bytes) {
      return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(from, bytes, 0, 0));
    };
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      if (OUT) q[i] = at(qp, (kr + KR * i) * qs + kc);
      k[i] = at(kp, (kr + KR * i) * ks + kc);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] = at(vp, (vr + VR * i) * vs + vc);
#endif
  }

  DX_DEVICE void store(Chunk<DK> &m, int par) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int r = tid / (DK / 4) + KR * i, c = 4 * (tid % (DK / 4));
      if (OUT) *reinterpret_cast<floatx4 *>(&m.q[r][c]) = q[i];
      *reinterpret_cast<floatx4 *>(&m.k[r][c]) = k[i];
    }
    bool lost = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<floatx4 *>(&m.v[tid / 16 + VR * i][4 * (tid % 16)]) = v[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) lost |= !(fabsf(v[i][e]) < INFINITY);
    }
    if (lost) m.lost[par] = 1;
  }
};

// Tokens [t0, t1) of a sequence from the state st on; OUT: with their outputs. Returns the sum of their g, in powers of two.
template <int DK, bool OUT>
DX_DEVICE double chunks(const LinearAttn &a, const Sequence &s, int head, int col0, int t0, int t1, floatx4 (&st)[DK / 16],
                        Chunk<DK> &m) {
  constexpr int N = Chunk<DK>::TOKENS;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int kh = head / (a.h / a.hk);
  auto decay = [&](int t) { return wave == 1 && lane < N && t + lane < t1 ? a.decay[(s.start + t + lane) * a.ds + head] : 0.f; };
  auto sums = [&](typename Chunk<DK>::Decay &d, float x) {
    const Sums sum = sum_of<N>(x);
    if (lane < N) {
      d.sum[lane] = sum.upto;
      d.from_start[lane] = exp2f((float)sum.upto);
      d.to_end[lane] = exp2f((float)(sum.end - sum.upto));
    }
    if (lane == 0) {
      d.all = factor_of(sum.end * 0.6931471805599453);
      d.total = sum.end;
    }
  };
  FetchedF32<DK, OUT> f;
  f.load(a, s.start + t0, min(N, t1 - t0), head, kh, col0);
  float next = decay(t0);
  if (wave == 1) sums(m.decay[0], next);
  next = decay(t0 + N);
  if (tid < 2) m.lost[tid] = 0;
  __syncthreads();
  double total = 0.0;
  int par = 0;
  for (int t = t0; t < t1; t += N, par ^= 1) {
    const int n = min(N, t1 - t);
    const long row = s.start + t;
    f.store(m, par);
    lds_barrier();
    f.load(a, row + N, max(min(N, t1 - t - N), 0), head, kh, col0);  // none behind the last chunk
    const typename Chunk<DK>::Decay &d = m.decay[par];
    total += d.total;
    floatx4 o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (wave == 1) {  // whose tile of the weights is that of later tokens
      sums(m.decay[par ^ 1], next);
      next = decay(t + 2 * N);
    }
    if constexpr (OUT) {
      const int i0 = 16 * (wave >> 1), j0 = 16 * (wave & 1);
      floatx4 p[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      if (wave != 1)
#pragma unroll
        for (int x = 0; x < DK; x += 16) {
          const floatx4 qx = *reinterpret_cast<const floatx4 *>(&m.q[i0 + c][x + 4 * g]);
          const floatx4 kx = *reinterpret_cast<const floatx4 *>(&m.k[j0 + c][x + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e & 1] = mfma_f32(qx[e], kx[e], p[e & 1]);
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * g + r, j = j0 + c;
        const float weight = (p[0][r] + p[1][r]) * exp2f((float)(d.sum[i] - d.sum[j]));
        m.p[i][j] = j <= i ? weight : 0.f;
      }
#pragma unroll
      for (int x = 0; x < DK / 16; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const floatx4 qx = *reinterpret_cast<const floatx4 *>(&m.q[16 * i + c][16 * x + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i] = mfma_f32(qx[e], st[x][e], o[i]);
        }
    }
    lds_barrier();
    float v[2][4];  // rows 16 j + 4 g + e of the wave's columns
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = m.v[16 * j + 4 * g + e][16 * wave + c];
    if constexpr (OUT) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] *= d.from_start[16 * i + 4 * g + r];
      if (!m.lost[par]) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const floatx4 px = *reinterpret_cast<const floatx4 *>(&m.p[16 * i + c][16 * j + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i] = mfma_f32(px[e], v[j][e], o[i]);
          }
      } else {  // a weight of 0 would carry a later token's infinity or NaN to this one
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            for (int j = 0; j <= 16 * i + 4 * g + r; ++j)
              o[i][r] = fmaf(m.p[16 * i + 4 * g + r][j], m.v[j][16 * wave + c], o[i][r]);
      }
#if defined(__HIP_DEVICE_COMPILE__)
      const auto out = rows_of(static_cast<float *>(a.out) + row * a.os + head * a.dv + col0, n, 4 * a.os);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(a.scale * o[i][r]), out,
                                                4 * ((16 * i + 4 * g + r) * (uint32_t)a.os + 16 * wave + c), 0, 0);
#endif
    }
    const Factor all = d.all;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[i][r] = times(st[i][r], all);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = v[j][e] * d.to_end[16 * j + 4 * g + e];
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) st[i] = mfma_f32(m.k[16 * j + 4 * g + e][16 * i + c], y, st[i]);
      }
    lds_barrier();
    if (tid == 0) m.lost[par] = 0;  // set again behind the next chunk's barriers
  }
  return total;
}

// ------------------------------------------------------------------------------------------ bf16, chunks of 64 tokens
//
// bf16 products (16x16x32: lane l has row or column l % 16 of an operand and eight k of group g = l / 16; of the result
// column l % 16, rows 4 g + r). Wave w has the columns 16 NC w .. of the state, in registers, as results S[DK rows, column].
//   Weights P^T = K Q^T: wave w the queries 16 w .., all earlier keys. A lane holds keys 4 g + r of a query, which is what
//     the product O^T = V^T P^T takes as eight k when V is read back transposed by the same rows; P goes through LDS as
//     two bf16 parts, since every wave needs all of it.
//   O^T += S^T Q^T: two tiles of S are eight k of a lane as they lie, again as two bf16 parts; Q is read by the same rows.
//   S = K^T (w V): both read transposed; w V, w = e^(G_C - G_j), as three bf16 parts: the state keeps fp32's precision.
// P and S as one part each would be off by 2^-8 of the mass of an output (its sums of absolute values), which the output's own
// rounding does not hide. As two they are off by up to 2^-16 of it: below that rounding unless the terms cancel to less than
// 2^-8 of them. A third part of both would be some 29% more products.
//
// Bound by the wave's own instructions: at keys of 128 dimensions the matrix unit is busy 32% of the time and the vector
// unit 46% (splitting into parts, decays, addresses), both at once 11%; at keys of 256, whose one workgroup a CU has no
// other beside it, 21%, 27% and 5%. 12 sequences of 517 to 16384 tokens, 46000 in all, 32 heads of 128 by 128: 660 us, of which
// 400 here, 195 the segments' own part, 60 the join; without the products for the state 115 less, without stores of outputs 90.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

DX_DEVICE floatx4 mfma16(bf16x8 x, bf16x8 y, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }

// 16 lanes read four rows of 16 values, lane i gets column i.
DX_DEVICE s16x4 read_transposed(const uint16_t *p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
#else
  return s16x4{};
#endif
}

// Rows of W values in 16-byte chunks, chunk c of row r at c ^ f(r): 16 rows' reads of one chunk, and eight rows' transposed
// reads of two neighbouring ones, fall on all banks (a line of them is 16 chunks).
template <int W>
DX_DEVICE int place(int r, int c) {
  const int f = W == 64 ? ((r >> 1) & 3) << 1 | ((r >> 3) & 1) : (r & 7) << 1 | ((r >> 3) & 1);
  return r * W + ((c ^ f) << 3);
}

DX_DEVICE bf16x8 both(s16x4 x, s16x4 y) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Queries lie in the order in which two tiles of the state are eight k of a lane: chunk 4 u + g of a row has the dimensions
// 32 u + 4 g .. and 32 u + 16 + 4 g .. (one read), where the four dimensions h of a row are half (h >> 2) & 1 of chunk
// 4 u + (h & 3).
template <int W>
DX_DEVICE int q_half(int r, int h) {
  return place<W>(r, 4 * (h >> 3) + (h & 3)) + ((h >> 2) & 1) * 4;
}

// Columns 16 t .. of the rows 32 a + 4 g .. and 32 a + 16 + 4 g .. as eight k.
template <int W>
DX_DEVICE bf16x8 columns(const uint16_t *rows, int a, int t, int lane) {
  const int c = lane & 15, r = 32 * a + 4 * (lane >> 4) + (c >> 2);
  const uint16_t *p = rows + place<W>(r, 2 * t + ((c >> 1) & 1)) + (c & 1) * 4;
  return both(read_transposed(p), read_transposed(p + 16 * W));  // 16 rows on: the same place
}

// x = the sum of N bf16 parts, nearly: what N parts cannot hold is below 2^(-8 N) of it.
template <int N>
DX_DEVICE void split(const float (&x)[8], bf16x8 (&out)[N]) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = pack_bf2(rest[2 * e], rest[2 * e + 1]);
      if (n + 1 < N) {
        rest[2 * e] -= lo_bf(w[e]);
        rest[2 * e + 1] -= hi_bf(w[e]);
      }
    }
    out[n] = as_bf16x8(w);
  }
}

// Asks for N times one matrix instruction and V others of the vector unit, in the block between two barriers of the
// schedule: each runs while the other does.
template <int N, int V>
DX_DEVICE void interleave() {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
  }
#endif
}

template <int DK, int NC, int WAVES>
struct Tile {
  static constexpr int TOKENS = 64, W = 16 * NC * WAVES;
  uint16_t q[TOKENS * (DK > W ? DK : W)], k[TOKENS * DK], v[TOKENS * W];  // q: behind the products with it, outputs
  u32x4 p[4][2][2][64];  // [16 queries][32 keys][part][lane]
  struct Decay {
    double sum[TOKENS];  // of g, in powers of two
    float from_start[TOKENS], to_end[TOKENS];
    int shift;
    double total, rest;  // of g; of the state's scale behind the chunk
  } decay[2];  // this chunk's and the next one's
  int lost[2];  // whether a value is no finite number
};

// A chunk's rows on their way from memory.
template <int DK, int NC, int WAVES, bool OUT>
struct Fetched {
  using Shared = Tile<DK, NC, WAVES>;
  static constexpr int THREADS = 64 * WAVES, W = Shared::W;
  static constexpr int KR = THREADS / (DK / 8), VR = THREADS / (W / 8), KI = 64 / KR, VI = 64 / VR;  // rows a load, loads
  u32x4 q[OUT ? KI : 1], k[KI], v[VI];

  DX_DEVICE void load(const LinearAttn &a, long row, int n, int head, int kh, int col0, uint32_t tid) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t kr = tid / (DK / 8), kc = 16 * (tid % (DK / 8)), vr = tid / (W / 8), vc = 16 * (tid % (W / 8));
    const uint32_t qs = 2 * (uint32_t)a.qs, ks = 2 * (uint32_t)a.ks, vs = 2 * (uint32_t)a.vs;
    const auto qp = rows_of(static_cast<const uint16_t *>(a.q) + row * a.qs + kh * DK, n, 2 * a.qs);
    const auto kp = rows_of(static_cast<const uint16_t *>(a.k) + row * a.ks + kh * DK, n, 2 * a.ks);
    const auto vp = rows_of(static_cast<const uint16_t *>(a.v) + row * a.vs + head * a.dv + col0, n, 2 * a.vs);
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      if (OUT) q[i] = __builtin_amdgcn_raw_buffer_load_b128(qp, (kr + KR * i) * qs + kc, 0, 0);
      k[i] = __builtin_amdgcn_raw_buffer_load_b128(kp, (kr + KR * i) * ks + kc, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(vp, (vr + VR * i) * vs + vc, 0, 0);
#endif
  }

  // The first wave's: what the chunk's decays come to. The state is 2^x times what the registers hold: a chunk moves x, and
  // the registers are shifted by whole powers of two when x leaves [0, 1). So no rounding of a decay is ever multiplied
  // in, and a head that forgets slowly has hardly anything to multiply. With x below 0 the registers, and v times its
  // weight on the way to them, would pass fp32's range where the state does not.
  DX_DEVICE static double sums(typename Shared::Decay &d, float g, double x, float log2_scale) {
    const int lane = threadIdx.x;
    const auto [sum, end] = sum_of<64>(g);
    d.sum[lane] = sum;
    d.from_start[lane] = fast_exp2((float)(sum + x + log2_scale));
    x += end;
    const double whole = x < 0.0 || x >= 1.0 ? floor(x) : 0.0;
    x -= whole;
    d.to_end[lane] = fast_exp2((float)(end - sum - x));
    if (lane == 0) {
      d.shift = (int)fmin(fmax(whole, -4096.0), 4096.0);
      d.total = end;
      d.rest = x;
    }
    return x;
  }

  DX_DEVICE void store(Shared &m, uint32_t tid, int par) const {
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const uint32_t at = tid + THREADS * i, r = at / (DK / 8), c = at % (DK / 8);
      if (OUT) {  // by halves: see q_half
        *reinterpret_cast<u32x2 *>(m.q + q_half<DK>(r, 2 * c)) = u32x2{q[i][0], q[i][1]};
        *reinterpret_cast<u32x2 *>(m.q + q_half<DK>(r, 2 * c + 1)) = u32x2{q[i][2], q[i][3]};
      }
      *reinterpret_cast<u32x4 *>(m.k + place<DK>(r, c)) = k[i];
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const uint32_t at = tid + THREADS * i, r = at / (W / 8), c = at % (W / 8);
      *reinterpret_cast<u32x4 *>(m.v + place<W>(r, c)) = v[i];
    }
    const bf16x8 nothing = as_bf16x8(u32x4{0, 0, 0, 0});
    floatx4 sum = {0, 0, 0, 0};  // 0 times each value: NaN where one is no finite number
#pragma unroll
    for (int i = 0; i < VI; ++i) sum = mfma16(nothing, as_bf16x8(v[i]), sum);
    if (sum[0] != 0.f) m.lost[par] = 1;
  }
};

// Tokens [t0, t1) of a sequence from the state st on, the first chunk's rows on their way; OUT: with their outputs. Returns
// the sum of their g, in powers of two.
template <int DK, int NC, int WAVES, bool OUT>
DX_DEVICE double tiles(const LinearAttn &a, const Sequence &s, int head, int col0, int t0, int t1,
                       floatx4 (&st)[DK / 16][NC], Fetched<DK, NC, WAVES, OUT> &f, Tile<DK, NC, WAVES> &m) {
  constexpr int N = 64, W = Tile<DK, NC, WAVES>::W;
  constexpr bool AHEAD = DK < 256;  // operands are made ready while others are multiplied; at 256 registers are short
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kh = head / (a.h / a.hk);
  const float log2_scale = log2f(a.scale);
  double total = 0.0, next = 0.0, rest = 0.0;  // next: the first wave's, behind the chunk that it has summed last
  // g of a chunk's tokens, a chunk earlier than its rows, so that no sum of them waits for the rows
  auto decay = [&](int t) {
    float g = 0.f;
#if defined(__HIP_DEVICE_COMPILE__)
    const int n = max(min(N, t1 - t), 0), lane = threadIdx.x & 63;
    const auto rows = __builtin_amdgcn_make_buffer_rsrc((void *)(a.decay + (s.start + t) * a.ds + head), (short)0,
                                                        n > 0 ? (int)((n - 1) * a.ds + 1) * 4 : 0, 0x00020000);
    g = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, 4 * (uint32_t)lane * (uint32_t)a.ds, 0, 0));
#endif
    return g;
  };
  auto sums = [&](typename Tile<DK, NC, WAVES>::Decay &d, float g, int t, double x) {
    return Fetched<DK, NC, WAVES, OUT>::sums(d, t + (int)threadIdx.x < t1 ? g : 0.f, x, log2_scale);  // rows of stride 0 have no end
  };
  float g1 = decay(t0), g2 = decay(t0 + N);
  if (wave == 0) next = sums(m.decay[0], g1, t0, 0.0);
  if (threadIdx.x < 2) m.lost[threadIdx.x] = 0;
  // waited for here: the loop's own wait for these rows is then not one for the outputs stored before it
  __builtin_amdgcn_s_waitcnt(0x0f70);
  lds_barrier();
  int par = 0;
  for (int t = t0; t < t1; t += N, par ^= 1) {
    const int n = min(N, t1 - t);
    const long row = s.start + t;
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // places in LDS are found again for every chunk: held over all of them they take registers
    tid &= 64 * WAVES - 1;
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    f.store(m, tid, par);
    lds_barrier();
    g1 = g2;
    g2 = decay(t + 2 * N);
    f.load(a, row + N, max(min(N, t1 - t - N), 0), head, kh, col0, tid);  // none behind the last chunk
    const typename Tile<DK, NC, WAVES>::Decay &d = m.decay[par];
    total += d.total;
    // A weight of 0 would carry a later token's infinity or NaN to an earlier one: such values are taken out of the wave's
    // columns, and what they reach is NaN.
    const bool lost = __builtin_amdgcn_readfirstlane(m.lost[par]) != 0;
    int first = N;  // of the wave's column lane % (16 NC): the first token whose value is lost
    if (lost) {
      const int col = 16 * NC * wave + lane % (16 * NC);
      for (int j = N - 1; j >= 0; --j) {
        uint16_t &v = m.v[place<W>(j, col >> 3) + (col & 7)];
        if ((v & 0x7f80) == 0x7f80) {
          first = j;
          v = 0;  // by all lanes of a column alike
        }
      }
    }
    floatx4 o[4][NC];
    if constexpr (OUT) {
      const int mine = wave & 3;  // its 16 queries; eight waves share them by 32 keys
      bf16x8 qf[DK / 32];
#pragma unroll
      for (int u = 0; u < DK / 32; ++u)
        qf[u] = both(*reinterpret_cast<const s16x4 *>(m.q + q_half<DK>(16 * mine + c, 8 * u + 2 * g)),
                     *reinterpret_cast<const s16x4 *>(m.q + q_half<DK>(16 * mine + c, 8 * u + 2 * g + 1)));
      const double upto = d.sum[16 * mine + c] + log2_scale;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (2 * b > mine) break;
        if (WAVES == 8 && b != wave >> 2) continue;
        double sum[8];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[4 * j + r] = d.sum[32 * b + 16 * j + 4 * g + r];
        floatx4 w[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        constexpr int AT_ONCE = DK / 32 < 4 ? DK / 32 : 4;  // reads on their way together
#pragma unroll
        for (int u0 = 0; u0 < DK / 32; u0 += AT_ONCE) {
          bf16x8 kf[AT_ONCE][2];
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              kf[u][j] = as_bf16x8(
                  *reinterpret_cast<const u32x4 *>(m.k + place<DK>(32 * b + 16 * j + c, 4 * (u0 + u) + g)));
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) w[j] = mfma16(kf[u][j], qf[u0 + u], w[j]);  // keys behind the queries: 0 below
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = fast_exp2((float)(upto - sum[e]));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float weight = w[e >> 2][e & 3] * p[e];  // before the choice: no branch around it
          p[e] = 32 * b + 16 * (e >> 2) + 4 * g + (e & 3) <= 16 * mine + c ? weight : 0.f;
        }
        bf16x8 parts[2];
        split(p, parts);
#pragma unroll
        for (int z = 0; z < 2; ++z) m.p[mine][b][z][lane] = __builtin_bit_cast(u32x4, parts[z]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int y = 0; y < NC; ++y) o[i][y] = floatx4{0, 0, 0, 0};
      // Two tiles of the state at a time: while the matrix cores multiply one pair, the next is split and its queries read.
      bf16x8 sf[2][NC][2], qx[2][4];
      auto ready = [&](int u, int at) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          qx[at][i] = as_bf16x8(*reinterpret_cast<const u32x4 *>(m.q + place<DK>(16 * i + c, 4 * u + g)));
#pragma unroll
        for (int y = 0; y < NC; ++y) {
          float pair[8];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            pair[r] = st[2 * u][y][r];
            pair[4 + r] = st[2 * u + 1][y][r];
          }
          split(pair, sf[at][y]);
        }
      };
      ready(0, 0);
#pragma unroll
      for (int u = 0; u < DK / 32; ++u) {
        __builtin_amdgcn_sched_barrier(0);
        if (u + 1 < DK / 32) ready(u + 1, (u + 1) & 1);
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int y = 0; y < NC; ++y) o[i][y] = mfma16(sf[u & 1][y][z], qx[u & 1][i], o[i][y]);
        if (u + 1 < DK / 32) interleave<8 * NC, 3>();
      }
    }
    if (wave == 0 && t + N < t1) next = sums(m.decay[par ^ 1], g1, t + N, next);
    lds_barrier();
    const int shift = __builtin_amdgcn_readfirstlane(d.shift);
    if (shift != 0)
#pragma unroll
      for (int u = 0; u < DK / 16; ++u)
#pragma unroll
        for (int y = 0; y < NC; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[u][y][r] = ldexpf(st[u][y][r], shift);
    bf16x8 vf[2][NC];
    floatx4 weight[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int y = 0; y < NC; ++y) vf[b][y] = columns<W>(m.v, b, NC * wave + y, lane);
#pragma unroll
      for (int j = 0; j < 2; ++j) weight[b][j] = *reinterpret_cast<const floatx4 *>(d.to_end + 32 * b + 16 * j + 4 * g);
    }
    bf16x8 wv[2][NC][3];
    auto weigh = [&](int b) {
#pragma unroll
      for (int y = 0; y < NC; ++y) {
        const u32x4 raw = __builtin_bit_cast(u32x4, vf[b][y]);
        float p[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[2 * e] = lo_bf(raw[e]) * weight[b][e >> 1][(2 * e) & 3];
          p[2 * e + 1] = hi_bf(raw[e]) * weight[b][e >> 1][(2 * e + 1) & 3];
        }
        split(p, wv[b][y]);
      }
    };
    __builtin_amdgcn_sched_barrier(0);
    if (AHEAD) weigh(0);
    if constexpr (OUT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float from = d.from_start[16 * i + c];
#pragma unroll
        for (int y = 0; y < NC; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][y][r] *= from;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int i = 2 * b; i < 4; ++i) {
            const bf16x8 p = as_bf16x8(m.p[i][b][z][lane]);
#pragma unroll
            for (int y = 0; y < NC; ++y) o[i][y] = mfma16(vf[b][y], p, o[i][y]);
          }
      if (AHEAD) {
        interleave<12 * NC, 5>();
#pragma unroll
        for (int y = 0; y < NC; ++y)
#pragma unroll
          for (int z = 0; z < 3; ++z) asm volatile("" ::"v"(__builtin_bit_cast(u32x4, wv[0][y][z])));  // here, not below
      }
      if (lost)
#pragma unroll
        for (int y = 0; y < NC; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = __shfl(first, 16 * y + 4 * g + r, 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i][y][r] = 16 * i + c >= at ? NAN : o[i][y][r];
          }
      // The wave's outputs through its own part of q: stored as they lie, 8 bytes a lane in pieces of 32, they took an
      // eighth of the kernel's time. Chunk x of row r at x ^ f(r), over banks of 16 chunks.
      constexpr int CH = 2 * NC, LINE = 16 / CH;  // chunks of a row, rows of a line of banks
      uint16_t *own = m.q + wave * (N * CH * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int y = 0; y < NC; ++y) {
          const int r = 16 * i + c, x = 2 * y + (g >> 1);
          *reinterpret_cast<u32x2 *>(own + (r * CH + (x ^ (r / LINE % CH))) * 8 + (g & 1) * 4) =
              u32x2{pack_bf2(o[i][y][0], o[i][y][1]), pack_bf2(o[i][y][2], o[i][y][3])};
        }
#if defined(__HIP_DEVICE_COMPILE__)
      const auto out = rows_of(static_cast<uint16_t *>(a.out) + row * a.os + head * a.dv + col0, n, 2 * a.os);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const uint32_t r = (64 * i + lane) / CH, x = lane % CH;
        __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4 *>(own + (r * CH + (x ^ (r / LINE % CH))) * 8),
                                               out, 2 * (r * (uint32_t)a.os + 16 * NC * wave + 8 * x), 0, 0);
      }
#endif
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      __builtin_amdgcn_sched_barrier(0);
      if (!AHEAD || b == 0) weigh(AHEAD ? 1 : b);
      constexpr int AT_ONCE = 2;
#pragma unroll
      for (int u0 = 0; u0 < DK / 16; u0 += AT_ONCE) {
        bf16x8 kt[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) kt[u] = columns<DK>(m.k, b, u0 + u, lane);
#pragma unroll
        for (int z = 2; z >= 0; --z)
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int y = 0; y < NC; ++y) st[u0 + u][y] = mfma16(kt[u], wv[b][y][z], st[u0 + u][y]);
      }
      if (AHEAD && b == 0) interleave<DK / 16 * 3 * NC, 3>();
    }
    if (lost)
#pragma unroll
      for (int y = 0; y < NC; ++y) {
        const float gone = __shfl(first, 16 * y + c, 64) < N ? NAN : 0.f;
#pragma unroll
        for (int u = 0; u < DK / 16; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[u][y][r] += gone;
      }
    rest = d.rest;
    if (tid == 0) m.lost[par] = 0;
    lds_barrier();
  }
  const Factor scale = factor_of(rest * 0.6931471805599453);
#pragma unroll
  for (int u = 0; u < DK / 16; ++u)
#pragma unroll
    for (int y = 0; y < NC; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[u][y][r] = times(st[u][y][r], scale);
  return total;
}

// Element r of the wave's result tile (x, y) in a state.
template <int NC>
DX_DEVICE long tile_at(const LinearAttn &a, int x, int y, int r, int col0) {
  const int lane = threadIdx.x & 63;
  return (long)(16 * x + 4 * (lane >> 4) + r) * a.dv + col0 + 16 * (NC * (threadIdx.x >> 6) + y) + (lane & 15);
}

template <int DK, int NC, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, DK == 256 ? 1 : 2)
segment_bf16_kernel(LinearAttn a, float *parts, double *sums, int most) {
  __shared__ __align__(16) Tile<DK, NC, WAVES> m;
  const int b = blockIdx.z, i = blockIdx.y;
  const auto [head, col0] = unit<16 * NC * WAVES>(a);
  const Sequence s = sequence(a, b);
  const la::Segments seg = la::segments(s.len, la::limit(DK));
  if (s.len <= la::STEP || i >= seg.count - 1) return;
  Fetched<DK, NC, WAVES, false> f;
  f.load(a, s.start + i * seg.tokens, 64, head, head / (a.h / a.hk), col0, threadIdx.x);
  floatx4 st[DK / 16][NC];
#pragma unroll
  for (int x = 0; x < DK / 16; ++x)
#pragma unroll
    for (int y = 0; y < NC; ++y) st[x][y] = floatx4{0, 0, 0, 0};
  const double total = tiles<DK, NC, WAVES, false>(a, s, head, col0, i * seg.tokens, (i + 1) * seg.tokens, st, f, m);
  const long unit = ((long)b * most + i) * a.h + head;
  float *to = parts + unit * DK * a.dv;
#pragma unroll
  for (int x = 0; x < DK / 16; ++x)
#pragma unroll
    for (int y = 0; y < NC; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) to[tile_at<NC>(a, x, y, r, col0)] = st[x][y][r];
  if (col0 == 0 && threadIdx.x == 0) sums[unit] = total * 0.6931471805599453;
}

template <int DK, int NC, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, DK == 256 ? 1 : 2)
chunk_bf16_kernel(LinearAttn a, const float *parts, int most) {
  __shared__ __align__(16) Tile<DK, NC, WAVES> m;
  const int b = blockIdx.z, i = blockIdx.y;
  const auto [head, col0] = unit<16 * NC * WAVES>(a);
  const Sequence s = sequence(a, b);
  if (s.len <= la::STEP) {
    if (i > 0) return;
    // 256 threads have COLS columns: the workgroup's halves side by side, or one after the other
    const int half = threadIdx.x / THREADS;
    for (int y = half; y < 16 * NC * WAVES / COLS; y += 64 * WAVES / THREADS) {
      if (y > half) __syncthreads();
      step_body<uint16_t, DK>(a, s, head, col0 + COLS * y, reinterpret_cast<float *>(&m) + half * STEP_LDS<DK>);
    }
    return;
  }
  const la::Segments seg = la::segments(s.len, la::limit(DK));
  if (i >= seg.count) return;
  const float *from = seg.count > 1 ? parts + (((long)b * most + i) * a.h + head) * DK * a.dv
                      : s.slot >= 0 ? a.state_in + (s.slot * a.h + head) * DK * a.dv : nullptr;
  const int t0 = i * seg.tokens, t1 = min(t0 + seg.tokens, s.len);
  Fetched<DK, NC, WAVES, true> f;
  f.load(a, s.start + t0, min(64, t1 - t0), head, head / (a.h / a.hk), col0, threadIdx.x);
  floatx4 st[DK / 16][NC];
#pragma unroll
  for (int x = 0; x < DK / 16; ++x)
#pragma unroll
    for (int y = 0; y < NC; ++y) st[x][y] = floatx4{0, 0, 0, 0};
  if (from)  // one branch around all loads
#pragma unroll
    for (int x = 0; x < DK / 16; ++x)
#pragma unroll
      for (int y = 0; y < NC; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[x][y][r] = from[tile_at<NC>(a, x, y, r, col0)];
  tiles<DK, NC, WAVES, true>(a, s, head, col0, t0, t1, st, f, m);
  if (i == seg.count - 1 && s.slot >= 0) {
    float *to = a.state_out + (s.slot * a.h + head) * DK * a.dv;
#pragma unroll
    for (int x = 0; x < DK / 16; ++x)
#pragma unroll
      for (int y = 0; y < NC; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) to[tile_at<NC>(a, x, y, r, col0)] = st[x][y][r];
  }
}

// ------------------------------------------------------------------------------------------ segments

// What each segment but the last adds to the state, and the sum of its g.
template <int DK>
__global__ void __launch_bounds__(THREADS) segment_f32_kernel(LinearAttn a, float *parts, double *sums, int most) {
  __shared__ __align__(16) Chunk<DK> m;
  const int b = blockIdx.z, i = blockIdx.y;
  const auto [head, col0] = unit<COLS>(a);
  const Sequence s = sequence(a, b);
  const la::Segments seg = la::segments(s.len, la::limit(DK));
  if (s.len <= la::STEP_F32 || i >= seg.count - 1) return;
  floatx4 st[DK / 16];
#pragma unroll
  for (int x = 0; x < DK / 16; ++x) st[x] = floatx4{0, 0, 0, 0};
  const double total = chunks<DK, false>(a, s, head, col0, i * seg.tokens, (i + 1) * seg.tokens, st, m);
  const long unit = ((long)b * most + i) * a.h + head;
  float *to = parts + unit * DK * a.dv;
#pragma unroll
  for (int x = 0; x < DK / 16; ++x)
#pragma unroll
    for (int r = 0; r < 4; ++r) to[state_at(a, x, r, col0)] = st[x][r];
  if (col0 == 0 && threadIdx.x == 0) sums[unit] = total * 0.6931471805599453;
}

// In the place of each segment's part the state that it starts from. Four values a thread, four parts on their way together
// (eight ask for parts that are not there: 41.3 us in all for 40.3 at 1024 tokens), the decays found once a workgroup; bound
// by the bytes of the parts: 12 sequences of 517 to 16384 tokens 60 us. Part after part, 8192 tokens take 122 us in all for 121.
__global__ void __launch_bounds__(THREADS) join_kernel(LinearAttn a, float *parts, const double *sums, int most) {
  constexpr int AT_ONCE = 4;
  __shared__ Factor decay[la::MOST_SEGMENTS];
  const int b = blockIdx.z, head = blockIdx.y;
  const Sequence s = sequence(a, b);
  const int last = la::segments(s.len, la::limit(a.dk)).count - 1;  // it adds nothing to a later one
  if (last == 0) return;
  const long size = (long)a.dk * a.dv, at = ((long)blockIdx.x * THREADS + threadIdx.x) * 4;  // size: a multiple of 4 THREADS
  const long first = (long)b * most * a.h + head;
  auto part = [&](int i) { return reinterpret_cast<floatx4 *>(parts + (first + (long)i * a.h) * size + at); };
  floatx4 next[AT_ONCE];
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) next[i] = *part(min(i, last - 1));
  floatx4 st = {0, 0, 0, 0};
  if (s.slot >= 0) st = *reinterpret_cast<const floatx4 *>(a.state_in + (s.slot * a.h + head) * size + at);
  if (threadIdx.x < last) decay[threadIdx.x] = factor_of(sums[first + (long)threadIdx.x * a.h]);
  __syncthreads();
  for (int i0 = 0; i0 < last; i0 += AT_ONCE) {
    if (i0 > 0)
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) next[i] = *part(min(i0 + i, last - 1));
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      if (i0 + i >= last) break;
      *part(i0 + i) = st;
#pragma unroll
      for (int e = 0; e < 4; ++e) st[e] = next[i][e] + times(st[e], decay[i0 + i]);
    }
  }
  *part(last) = st;
}

template <int DK>
__global__ void __launch_bounds__(THREADS) chunk_f32_kernel(LinearAttn a, const float *parts, int most) {
  __shared__ __align__(16) Chunk<DK> m;
  const int b = blockIdx.z, i = blockIdx.y;
  const auto [head, col0] = unit<COLS>(a);
  const Sequence s = sequence(a, b);
  if (s.len <= la::STEP_F32) {
    if (i == 0) step_body<float, DK>(a, s, head, col0, &m.q[0][0]);
    return;
  }
  const la::Segments seg = la::segments(s.len, la::limit(DK));
  if (i >= seg.count) return;
  const float *from = seg.count > 1 ? parts + (((long)b * most + i) * a.h + head) * DK * a.dv
                      : s.slot >= 0 ? a.state_in + (s.slot * a.h + head) * DK * a.dv : nullptr;
  floatx4 st[DK / 16];
#pragma unroll
  for (int x = 0; x < DK / 16; ++x) st[x] = floatx4{0, 0, 0, 0};
  if (from)
#pragma unroll
    for (int x = 0; x < DK / 16; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[x][r] = from[state_at(a, x, r, col0)];
  chunks<DK, true>(a, s, head, col0, i * seg.tokens, min((i + 1) * seg.tokens, s.len), st, m);
  if (i == seg.count - 1 && s.slot >= 0) {
    float *to = a.state_out + (s.slot * a.h + head) * DK * a.dv;
#pragma unroll
    for (int x = 0; x < DK / 16; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r) to[state_at(a, x, r, col0)] = st[x][r];
  }
}

template <typename T, int DK>
hipError_t run(const LinearAttn &a, hipStream_t s) {
  unsigned x = (unsigned)(a.h * (a.dv / COLS));
  if (a.max_len <= (sizeof(T) == 2 ? la::STEP : la::STEP_F32)) {
    step_kernel<T, DK><<<dim3(x, a.num_seqs), dim3(THREADS), 0, s>>>(a);
    return hipGetLastError();
  }
  const int most = la::most_segments(a.max_len, la::limit(DK));
  // Columns of a workgroup: 2 COLS share the rows of q and k and their weights, but where COLS make no more workgroups than
  // there are CUs they are faster (32 heads of 128 by 128, 200 tokens: 1 sequence 20 us against 24, 4 22 and 26, 5 28 and
  // 27; 12 of 3000 727 and 586). A column's sums are the same.
  const bool two = sizeof(T) == 2 && a.dv > COLS && (long)x * most * a.num_seqs > 256;
  if (two) x /= 2;
  // 2 COLS columns: four waves of 32, two workgroups a CU (12 of 3000: 581 us, eight waves of 16 664); at DK 256, where one
  // fills the registers, eight of 16 (2111 tokens 80 us, four of 32 91)
  constexpr int NC = DK == 256 ? 1 : 2, WAVES = DK == 256 ? 8 : 4;
  const dim3 grid(x, most, a.num_seqs), before(x, most - 1, a.num_seqs), block(THREADS), wide(64 * WAVES);
  if (most > 1) {
    if constexpr (sizeof(T) == 2) {
      if (two) segment_bf16_kernel<DK, NC, WAVES><<<before, wide, 0, s>>>(a, a.parts, a.sums, most);
      else segment_bf16_kernel<DK, 1, 4><<<before, block, 0, s>>>(a, a.parts, a.sums, most);
    } else {
      segment_f32_kernel<DK><<<before, block, 0, s>>>(a, a.parts, a.sums, most);
    }
    const unsigned y = (unsigned)dx_ceil_div((long)a.dk * a.dv, 4 * THREADS);
    join_kernel<<<dim3(y, a.h, a.num_seqs), block, 0, s>>>(a, a.parts, a.sums, most);
  }
  if constexpr (sizeof(T) == 2) {
    if (two) chunk_bf16_kernel<DK, NC, WAVES><<<grid, wide, 0, s>>>(a, a.parts, most);
    else chunk_bf16_kernel<DK, 1, 4><<<grid, block, 0, s>>>(a, a.parts, most);
  } else {
    chunk_f32_kernel<DK><<<grid, block, 0, s>>>(a, a.parts, most);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t by_dim(const LinearAttn &a, hipStream_t s) {
  if (a.dk == 64) return run<T, 64>(a, s);
  if (a.dk == 128) return run<T, 128>(a, s);
  return run<T, 256>(a, s);
}

}  // namespace

hipError_t dx_linear_attn_launch(const LinearAttn &a, bool f32, hipStream_t s) {
  return f32 ? by_dim<float>(a, s) : by_dim<uint16_t>(a, s);
}

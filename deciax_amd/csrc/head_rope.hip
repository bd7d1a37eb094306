// Norms of query and key heads and the rotation by position, in one pass.
//
// Per head: u = x / sqrt(mean x^2 + eps) (1 + w) (without norm weights u = x), then the first 2 `pairs` dimensions turn by
// position * inv_freq[j]: pairs (j, j + pairs), or neighbours (2 j, 2 j + 1); cos and sin times `factor`. fp32 throughout,
// rounded once. The angle is taken in 64 bits, as a share of a turn: in fp32 it is off by 0.06 at position 10^6. What fp32
// cannot hold of the share turns its cosine and sine on: else each is off by up to 2^-23.3, whatever its own size.
#include "common.h"
#include "kernels.h"

namespace {

constexpr int THREADS = 256, MAX_PAIRS = 128;

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

template <typename T>
DX_DEVICE void store8(T *p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4 *>(p) = w;
  } else {
    *reinterpret_cast<floatx4 *>(p) = floatx4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<floatx4 *>(p + 4) = floatx4{x[4], x[5], x[6], x[7]};
  }
}

// A workgroup takes ROWS rows: their cosines and sines once into LDS, then eight dimensions of a head a thread, a head's
// D / 8 lanes side by side. A row may be read and written in place: a lane writes what it read, and takes its partner's
// half from the partner's registers. Bound by the bytes of the rows, each read and written once: 70471 rows of 24 heads of
// 256 (1.73 GB), a quarter of each turned, 311 us, 5.6 TB/s. Turned whole 467: a lane reads eight cosines and sines in a row,
// and the lanes' reads meet on the same banks of LDS (72% of its cycles). A small call is the launch and one chain of
// loads: 48 rows 4.9 us, with norms 5.4.
template <typename T, int D, int ROWS, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_kernel(HeadRope a) {
  constexpr int LANES = D / 8;
  __shared__ float2 turns[ROWS][MAX_PAIRS];
  const long row0 = (long)blockIdx.x * ROWS;
  const int rows = (int)min((long)ROWS, a.rows - row0), heads = a.hq + a.hkv, pairs = a.pairs;
  for (int i = threadIdx.x; i < rows * pairs; i += THREADS) {
    const int r = i / pairs, j = i - r * pairs;
    double t = (double)a.positions[row0 + r] * a.inv_freq[j] * 0.15915494309189535;  // turns: by 1 / (2 pi)
    t -= rint(t);
    const float angle = (float)(2.0 * t), rest = (float)(2.0 * t - angle) * 3.14159274f;
    float s, c;
    sincospif(angle, &s, &c);
    turns[r][j] = float2{fmaf(-s, rest, c) * a.factor, fmaf(c, rest, s) * a.factor};
  }
  const int part = threadIdx.x % LANES, dim = 8 * part;
  float wq[8], wk[8];
  if (a.q_norm) {
    load8(static_cast<const T *>(a.q_norm) + dim, wq);
    load8(static_cast<const T *>(a.k_norm) + dim, wk);
  }
  __syncthreads();
  const int items = rows * heads * LANES;
  for (int i = threadIdx.x; i < items; i += THREADS) {
    const int unit = i / LANES, r = unit / heads, head = unit - r * heads;
    float x[8];
    load8(static_cast<const T *>(a.x) + (row0 + r) * a.x_stride + head * D + dim, x);
    if (a.q_norm) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
      for (int off = LANES / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
      const float inv = rsqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (1.f + (head < a.hq ? wq[e] : wk[e]));
    }
    if constexpr (INTERLEAVED) {
      if (dim < 2 * pairs) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 t = turns[r][dim / 2 + e / 2];
          const float p = x[e], q = x[e + 1];
          x[e] = p * t.x - q * t.y;
          x[e + 1] = q * t.x + p * t.y;
        }
      }
    } else {
      // lanes of the first half take p cos - q sin, those of the second q cos + p sin
      const bool second = dim >= pairs;
      const int lane = (threadIdx.x & 63) + (second ? -pairs / 8 : pairs / 8);
      float other[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) other[e] = __shfl(x[e], lane, 64);
      if (dim < 2 * pairs) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = turns[r][(second ? dim - pairs : dim) + e];
          x[e] = second ? x[e] * t.x + other[e] * t.y : x[e] * t.x - other[e] * t.y;
        }
      }
    }
    store8(static_cast<T *>(a.out) + (row0 + r) * a.out_stride + head * D + dim, x);
  }
}

template <typename T, int D, int ROWS>
hipError_t run(const HeadRope &a, hipStream_t s) {
  const dim3 grid((unsigned)dx_ceil_div(a.rows, ROWS));
  if (a.interleaved)
    qk_norm_rope_kernel<T, D, ROWS, true><<<grid, dim3(THREADS), 0, s>>>(a);
  else
    qk_norm_rope_kernel<T, D, ROWS, false><<<grid, dim3(THREADS), 0, s>>>(a);
  return hipGetLastError();
}

// One row a workgroup up to 1024 rows (four would leave CUs without work: 24 heads of 256, 48 rows 5.4 us against 13.4, 1024
// 11.2 and 16.0) and where a row keeps the threads busy twice or more (70471 rows, turned whole, 469 us against 471). Narrow
// rows share the start: 30000 of 20 heads of 128 84 us one by one and 66 four at a time, of 6 heads of 64 28 and 16.
template <typename T, int D>
hipError_t by_rows(const HeadRope &a, hipStream_t s) {
  return a.rows <= 1024 || (a.hq + a.hkv) * D >= 4096 ? run<T, D, 1>(a, s) : run<T, D, 4>(a, s);
}

template <typename T>
hipError_t by_dim(const HeadRope &a, hipStream_t s) {
  if (a.d == 64) return by_rows<T, 64>(a, s);
  if (a.d == 128) return by_rows<T, 128>(a, s);
  return by_rows<T, 256>(a, s);
}

}  // namespace

hipError_t dx_qk_norm_rope_launch(const HeadRope &a, bool f32, hipStream_t s) {
  return f32 ? by_dim<float>(a, s) : by_dim<uint16_t>(a, s);
}

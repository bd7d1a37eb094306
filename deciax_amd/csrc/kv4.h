// The paged 4-bit cache, and what its kernels share.
//
// Format: 32 neighbouring values of one head of one token share a scale 2^e, e the smallest integer with
// amax <= 6 2^e, kept in [-119, 125] and stored as the byte e + 127; a value is the 4-bit code of the nearest of
// +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} in units of the scale (a tie takes the even code), the even dimension in the low half
// of its byte. These are the values that v_cvt_scalef32_pk_bf16_fp4 and its inverse convert; each is a bf16 number, so
// what the kernels multiply is exactly what the cache stands for. The ends of e keep the least value a normal bf16
// number and the largest a finite one. A block that holds an infinity or a NaN has the scale byte 255 and reads as NaN.
//
// Slot j of a sequence is row j % page of page table[j / page]; a page holds [kv heads][page slots] rows of each array.
// Table entries outside the pool are never followed: a slot there is not written and not seen.
#pragma once

#include "common.h"
#include "kernels.h"
#include "kv4_plan.h"

namespace kv4 {

constexpr int STEP = 32;  // keys that a wave takes at a time; pages hold a multiple of 64

struct Sequence {
  int n, ctx;  // newest tokens, slots with them
  long start;  // the newest tokens' first packed row
};

DX_DEVICE Sequence sequence(const Kv4Batch &q, int b, int shift) {
  Sequence s;
  s.n = min(max(q.seq_len[b], 0), q.max_seq_len);
  s.ctx = min(max(q.ctx_len[b], 0), min(q.max_ctx, (int)min((long)q.table_width << shift, 0x7fffffffL)));
  s.start = q.seq_start[b];
  return s;
}

// First row of the page that holds `slot` (whose place in it is added), or -1 for a page outside the pool.
DX_DEVICE long row_of(const Kv4Cache &c, const int32_t *table, int g, int slot) {
  const int page = table[slot >> c.shift];
  if (page < 0 || page >= c.pages) return -1;
  return (((long)page * c.hkv + g) << c.shift) + (slot & ((1 << c.shift) - 1));
}

// The scale of a byte, as the conversions take it: a float with that exponent.
DX_DEVICE float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight 4-bit values of one block to bf16.
DX_DEVICE u32x4 decode8(uint32_t w, float scale) {
  u32x4 r = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
#endif
  return r;
}

DX_DEVICE uint32_t encode8(const float (&x)[8], float scale) {
  uint32_t w = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
#endif
  return w;
}

// The scale byte for the largest |value| of a block, given as its bits (any infinity or NaN compares above all).
DX_DEVICE uint32_t scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255;
  // amax = m 2^E: 6 2^e >= amax from e = E - 2 where m <= 1.5, from E - 1 above
  const int byte = (int)(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x400000u);
  return (uint32_t)min(max(byte, 127 - 119), 127 + 125);
}

}  // namespace kv4

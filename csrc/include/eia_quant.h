// The 8-bit key/value cache.  A row is the D values of one token and kv head: e4m3 codes of x / 2^e and one byte
// e + 127, where e is the smallest whole number for which the row's largest magnitude is at most 448 * 2^e, held to
// [-100, 119].  A power of two costs a floating-point code nothing but its smallest magnitudes and makes every value
// code * 2^e exact in bf16: matrix products take bf16 operands made by v_cvt_scalef32_pk_bf16_fp8, whose scale operand is
// the byte in the exponent field, and lose nothing of what the cache holds.  (A scale of amax / 448 would be a factor
// behind each product.)
// Byte 255 marks a token and head of which a key or value is not finite: in k_scale, for both rows, so that a query
// that sees the token becomes NaN through its score and one that does not sees nothing of it; codes are 0 then.
//   keys    k[page][head][token][D]                values  v[page][head][token / 16][D][token % 16]
//   bytes   k_scale, v_scale[page][head][token]
// Sixteen tokens of a value channel are 16 contiguous bytes: the operand of two 16x16x32 products, in one load, for
// pages of any multiple of 16 tokens.
#pragma once
#include "eia_common.h"

constexpr int QUANT_GROUP = 16;        // tokens of a value tile
constexpr unsigned QUANT_POISON = 255;

struct QuantCache {
  uint8_t *k, *v, *ks, *vs;
  long codes, scales;                  // bytes from a page to the next
  int Hkv, bs;
  EIA_DEV uint8_t* key(int page, int h, int off, int D) const { return k + page * codes + ((long)h * bs + off) * D; }
  // channel 0 of the sixteen tokens from off on
  EIA_DEV uint8_t* values(int page, int h, int off, int D) const { return v + page * codes + ((long)h * bs + off) * D; }
  EIA_DEV uint8_t* kscale(int page, int h, int off) const { return ks + page * scales + (long)h * bs + off; }
  EIA_DEV uint8_t* vscale(int page, int h, int off) const { return vs + page * scales + (long)h * bs + off; }
};

// A table's entry, held to the pool: what it names outside of it is not read.
EIA_DEV int quant_page(int page, unsigned top) { return (int)min((unsigned)page, top); }

// 16 bytes that are read once and leave nothing in the caches, or as usual.
template <bool ONCE> EIA_DEV uint4 quant_load(const void* p) {
  typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
  if constexpr (ONCE) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
  return *reinterpret_cast<const uint4*>(p);
}

// Byte of a row whose largest magnitude has these bits (a row that is not finite: 0x7f800000 or more, not asked here).
// 448 = 1.75 * 2^8: a mantissa over 1.75 carries into the exponent.
EIA_DEV unsigned quant_byte(unsigned amax_bits) {
  const int b = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
  return (unsigned)min(max(b, 27), 246);
}
EIA_DEV float quant_inverse(unsigned byte) { return __uint_as_float((254 - byte) << 23); }    // 2^-e, byte in [27, 246]

// A double as the float on its way to a code: cut off, and its last bit set if anything was, so that the nearest code of the float is
// that of the double (rounded to the nearest twice, a value beside a border would come to lie on it: one key in a million.  4096 tokens 20.4 -> 20.8 us).
EIA_DEV float quant_odd(double x) {
  const unsigned hi = (unsigned)__double2hiint(x), lo = (unsigned)__double2loint(x);
  return (float)__hiloint2double((int)hi, (int)((lo & 0xe0000000u) | (min(lo << 3, 1u) << 29)));
}

// Four values, scaled, as codes.  Nothing scaled passes 448 but rows beyond 448 * 2^119.
EIA_DEV unsigned quant_pack(float a, float b, float c, float d, float inv) {
  auto held = [&](float x) { return fminf(fmaxf(x * inv, -448.f), 448.f); };
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(held(a), held(b), 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(held(c), held(d), r, true);
}

// Two codes of a word (the low or the high two) times the power of two whose bits `scale` holds.
template <bool HI> EIA_DEV unsigned quant_pair(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
EIA_DEV bf16x8 quant_eight(unsigned a, unsigned b, float scale) {
  return __builtin_bit_cast(bf16x8, make_uint4(quant_pair<false>(a, scale), quant_pair<true>(a, scale), quant_pair<false>(b, scale),
                                               quant_pair<true>(b, scale)));
}
EIA_DEV float quant_scale(unsigned byte) { return __uint_as_float(byte << 23); }

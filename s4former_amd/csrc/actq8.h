// 8-bit activation checkpoints: groups of 32 consecutive channels of a row share one power-of-two scale.
//
//   amax = max |x| over the group,  s = the least power of two with round(amax / s) <= 127,  code = round-to-even(x / s)
//
// x / s and code * s are exact (a shift of the exponent), so |x - code s| <= s / 2, and code * s has at most seven significant bits: it is
// exact in bf16, a restored value or matrix operand is never rounded again.  Where s is not clamped, amax / 127.5 < s <= amax / 63.75 and
// the error is at most amax / 127.5.  s stops at 2^121 above, where codes stop at 127 (with 2^122 the largest magnitudes would restore as
// infinity) and the bound stands, and at 2^-126 below, where it is 2^-127 instead: a group of magnitudes up to 2^-127 restores as zeros.
// The scale byte is the biased exponent of s (1 .. 248; groups of zeros take 1); 255 marks a group that
// held an infinity or a NaN: all its 32 values come back as NaN, so that a diverged pass is not hidden.  Byte 0 is never written and
// stands for zeros.
#pragma once
#include "common.h"
#include <initializer_list>

#define ACTQ8_GROUP 32

// host side of the argument checks: a piece of memory, and whether two have a byte in common
struct Piece { const char* p; int64_t n; };
inline Piece piece(const void* p, int64_t n) { return {(const char*)p, p ? n : 0}; }
// [rows, cols] with a row stride of ld elements of es bytes, from its first byte to its last
inline Piece piece(const void* p, int64_t rows, int64_t ld, int64_t cols, int es) { return piece(p, ((rows - 1) * ld + cols) * es); }
inline bool meet(const Piece& a, const Piece& b) { return a.n > 0 && b.n > 0 && a.p < b.p + b.n && b.p < a.p + a.n; }
inline bool meet(const Piece& a, std::initializer_list<Piece> l) {
  for (const Piece& b : l)
    if (meet(a, b)) return true;
  return false;
}
// two [rows, cols] matrices are the same one, or no element of one lies in the other (two column slices of one buffer, say)
inline bool same_or_apart(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int64_t cols, int es) {
  if ((a == b && (lda == ldb || rows == 1)) || !meet(piece(a, rows, lda, cols, es), piece(b, rows, ldb, cols, es))) return true;
  if (lda != ldb || lda < 2 * cols) return false;
  const int64_t ld = lda * es, d = (((const char*)b - (const char*)a) % ld + ld) % ld;
  return d >= cols * es && d <= ld - cols * es;
}

// lanes l ^ 1, l ^ 2 by quad permutes; after both, the halves of eight lanes by a mirror (the four lanes of a quad agree by then)
template <int CTRL> __device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float dpp_f32(float v) {
  return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(v)));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141;

// maximum over the LANES (4 or 8) neighbouring lanes that hold one group; |x| as its bit pattern: an unsigned maximum orders
// magnitudes, puts infinity above every number and NaN above infinity, where a float maximum would drop the NaN
template <int LANES> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
  v = max(v, dpp_u32<DPP_XOR1>(v));
  v = max(v, dpp_u32<DPP_XOR2>(v));
  if constexpr (LANES == 8) v = max(v, dpp_u32<DPP_HALF_MIRROR>(v));
  return v;
}
template <int LANES> __device__ __forceinline__ float group_sum(float v) {
  v += dpp_f32<DPP_XOR1>(v);
  v += dpp_f32<DPP_XOR2>(v);
  if constexpr (LANES == 8) v += dpp_f32<DPP_HALF_MIRROR>(v);
  return v;
}

__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// scale byte of a group from the bits of its largest magnitude.  The carry of + 0x10000 out of the mantissa is the test
// amax / 2^(e - 6) >= 127.5, e = floor(log2 amax)
__device__ __forceinline__ uint32_t q8_scale_byte(uint32_t amax_bits) {
  const int b = (int)((amax_bits + 0x10000u) >> 23) - 6;
  return amax_bits >= 0x7f800000u ? 255u : (uint32_t)min(max(b, 1), 248);
}
// 1 / s
__device__ __forceinline__ float q8_inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// s (NaN for a group that was not finite, zero for byte 0)
__device__ __forceinline__ float q8_scale(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }

// x / s + 1.5 * 2^23 rounds x / s to a whole number, ties to even, whose two's complement stands in the low bits of the sum
__device__ __forceinline__ uint32_t q8_code_bits(float x, float inv) {
  return __float_as_uint(__builtin_amdgcn_fmed3f(fmaf(x, inv, 12582912.f), 12582912.f - 127.f, 12582912.f + 127.f));
}
// four codes in the bytes of a word
__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __builtin_amdgcn_perm(q8_code_bits(b, inv), q8_code_bits(a, inv), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(q8_code_bits(d, inv), q8_code_bits(c, inv), 0x04000c0cu);
  return lo | hi;
}
// code e (0..3) of a word as a float
__device__ __forceinline__ float q8_code(uint32_t w, int e) { return (float)(int)(int8_t)(w >> (8 * e)); }
// two values that are exact in bf16 -> one word (the low halves of the floats are zero)
__device__ __forceinline__ uint32_t pack_exact_bf16(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

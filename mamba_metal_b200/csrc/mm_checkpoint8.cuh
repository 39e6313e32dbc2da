// 8-bit activation checkpoints: the block format's arithmetic (the header gives its definition).
// Scales are powers of two, so scaling a value up or down is exact and the one rounding is the one to the
// code: every reader and writer of the format agrees to the bit, whatever it fuses the conversion with. A
// scale of max/127 would use the codes' range better (up to one bit) but round twice.
#pragma once

#include "mm_common.cuh"

namespace mm {

constexpr int kCkBlock = MM_CHECKPOINT8_BLOCK;
constexpr unsigned kCkNonFinite = 255;

// Exponent byte of a block whose largest |x| has the given float bits. 127 = 0x1.fcp6: with
// max = m 2^k, m in [1, 2), the least e is k - 6, or k - 5 when m > 0x1.fc. Subnormal maxima (k field 0)
// end below the clamp.
MM_DEV unsigned ck_exponent(unsigned max_bits) {
  const int k = (int)(max_bits >> 23);
  const int e = k - 6 + ((max_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return k == 255 ? kCkNonFinite : (unsigned)max(e, 1);
}
// 2^-e and 2^e for exponent byte e + 127. A non-finite block's codes are never used.
MM_DEV float ck_inverse_scale(unsigned byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }
MM_DEV float ck_scale(unsigned byte) {
  return byte == kCkNonFinite ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}
MM_DEV int ck_code(float x, float inverse_scale) { return __float2int_rn(x * inverse_scale); }
MM_DEV unsigned ck_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

MM_DEV unsigned ck_pack4(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
MM_DEV int ck_byte(unsigned w, int i) { return (int)(w << (24 - 8 * i)) >> 24; }

// The element of type T that a code stands for: exact, except past T's largest finite value, which is
// restored instead (amax near the top of the range can round up to a code past it).
template <typename T> struct CkMax;
template <> struct CkMax<float> { static constexpr float v = 3.40282347e38f; };
template <> struct CkMax<__half> { static constexpr float v = 65504.f; };
template <> struct CkMax<__nv_bfloat16> { static constexpr float v = 3.38953139e38f; };
template <typename T> MM_DEV float ck_restore(int code, float scale) {
  const float v = (float)code * scale;
  return v > CkMax<T>::v ? CkMax<T>::v : v < -CkMax<T>::v ? -CkMax<T>::v : v;  // NaN passes both
}

inline bool ck_rows_aligned(const void* p, const int64_t* st, int64_t batch, int64_t dim, int elem, int align) {
  return (reinterpret_cast<uintptr_t>(p) % align) == 0 && (batch <= 1 || (st[0] * elem) % align == 0) &&
         (dim <= 1 || (st[1] * elem) % align == 0);
}

// Access of a tensor's rows (contiguous along time where n of them have more than one step)
inline Access ck_access(const void* p, const int64_t* st, int64_t batch, int64_t dim, int64_t steps, int elem) {
  if (steps > 1 && st[2] != 1) return kAnyStride;
  return ck_rows_aligned(p, st, batch, dim, elem, 16) ? kAligned : kContiguous;
}

}  // namespace mm

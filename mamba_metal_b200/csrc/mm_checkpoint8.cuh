// 8-bit activation checkpoints: the block format's arithmetic (the header gives its definition).
// Scales are powers of two, so scaling a value up or down is exact and the one rounding is the one to the
// code: every reader and writer of the format agrees to the bit, whatever it fuses the conversion with. A
// scale of max/127 would use the codes' range better (up to one bit) but round twice.
#pragma once

#include <type_traits>

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
// The low byte is the code: the scaled value is at most 127, so beside 1.5 * 2^23 the sum's one rounding, to even, leaves
// whole numbers, in two's complement. (The conversion instruction runs at an eighth of an addition's rate.)
constexpr float kCkWhole = 12582912.f;
MM_DEV unsigned ck_code(float x, float inverse_scale) { return __float_as_uint(fmaf(x, inverse_scale, kCkWhole)); }
MM_DEV uint2 ck_code_pair(f2_t x, f2_t inverse_scale) {
  const float2 v = f2_unpack(f2_fma(x, inverse_scale, f2_pack(kCkWhole, kCkWhole)));
  return make_uint2(__float_as_uint(v.x), __float_as_uint(v.y));
}
MM_DEV unsigned ck_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The largest |x| of eight values, as float bits; 16-bit types two at a time, in their own bits
template <typename T> MM_DEV unsigned ck_max_bits(const Raw8<T>& r) {
  unsigned m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, u4_word(r.v[k / 4], k % 4) & 0x7fffffffu);
    return m;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) m = __vmaxu2(m, u4_word(r.v[0], k) & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    return std::is_same<T, __half>::value ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))) : m << 16;
  }
}

MM_DEV unsigned ck_pack4(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Code i of a word of four: through the low byte of 2^23 + 128 + code, or by the conversion instruction, which suits
// kernels that keep the ALU busy (restoring bf16 10240 x 32768 163 and 180 us; conv gradient, channels last, bf16
// 4x5120x5601 343 and 271 when it was chosen)
MM_DEV float ck_converted(unsigned w, int i) { return (float)((int)(w << (24 - 8 * i)) >> 24); }
MM_DEV float ck_value(unsigned w, int i) {
  return __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7650 + i)) - 8388736.f;
}

// The element of type T that a code stands for: exact in the type that was packed, except past T's largest finite value, which is
// restored instead (amax near the top of the range can round up to a code past it). Every reader of codes goes by this
// or, where a block is known to stay in range, by the product alone.
template <typename T> struct CkMax;
template <> struct CkMax<float> { static constexpr float v = 3.40282347e38f; };
template <> struct CkMax<__half> { static constexpr float v = 65504.f; };
template <> struct CkMax<__nv_bfloat16> { static constexpr float v = 3.38953139e38f; };
template <typename T> MM_DEV float ck_limited(float v) {  // the lesser of the magnitudes, v's sign; NaN stays
  float r;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(CkMax<T>::v));
  return r;
}
template <typename T> MM_DEV float ck_restore(float code, float scale) { return ck_limited<T>(code * scale); }

// Whether no code of such a block stands for more than that (127 2^9 = 65024, 127 2^121 = 0x1.fcp127)
template <typename T> MM_DEV bool ck_in_range(unsigned byte) { return byte <= (std::is_same<T, __half>::value ? 136u : 248u); }

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

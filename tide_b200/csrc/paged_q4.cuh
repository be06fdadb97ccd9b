// The paged cache in 4 bits: how a token's key and value lie in it.
//
// A group is 32 neighbouring channels of a token's key or value in one head,
// held as codes c and a zero point z in 0..15 and a scale s; it stands for
// (c - z) s.  With lo and hi the least and the largest value, 0 among them, and
// t = (hi - lo) / 15,
//   s = t rounded up to four significant bits,  z = round(-lo / s),
//   c = round(x / s) + z, within 0..15:
// off by s / 2 at most, zero held as zero.  |c - z| <= 15 has four bits, as s
// has, so that a value has eight and both 16-bit types hold it exactly (fp16
// from s = 2^-21 on, the least scale that is given there): nothing is rounded
// when the cache is read, and the tensor cores' operands are its values.
//
// A scale and its zero point are 16 bits: a bf16 whose last four mantissa bits
// are zero, and z in their place.  So d channels are 9 d / 16 bytes, 4.5 bits
// a value.  A group with a value that is not finite has the scale NaN.
//
// Sixteen tokens of a head are a block of 18 d bytes, so that one copy brings
// all of it: the codes of the keys [16][d / 2], of the values, the scales of
// the keys [d / 32][token % 4][token / 4], of the values.  Eight channels are
// 32 bits, lowest first channels 0, 2, 4, 6, 1, 3, 5, 7: one shift and one mask
// give two neighbours in the halves of a register.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace tide {
namespace q4 {

constexpr int kBlock = 16;  // tokens of a block
constexpr int kGroup = 32;  // channels of a group

template <int D>
struct Layout {
  static constexpr int kRow = D / 2;           // bytes of a token's codes, key or value
  static constexpr int kCodes = kBlock * kRow; // of a block's, key or value
  static constexpr int kScales = D;            // bytes of a block's scales, key or value
  static constexpr int kBytes = 2 * kCodes + 2 * kScales;
  // side 0: keys, 1: values
  static __device__ __forceinline__ int codes(int side, int token) {
    return side * kCodes + token * kRow;
  }
  static __device__ __forceinline__ int scale(int side, int group, int token) {
    return 2 * kCodes + side * kScales + 2 * (group * kBlock + token % 4 * 4 + token / 4);
  }
};

template <typename T>
using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;

template <typename T>
__device__ __forceinline__ Pair<T> as_pair(uint32_t v) {
  return *reinterpret_cast<Pair<T> *>(&v);
}
template <typename P2>
__device__ __forceinline__ uint32_t as_bits(P2 v) {
  return *reinterpret_cast<uint32_t *>(&v);
}

// A number of the type's whose last bits are a code (and so 2^7 or 2^10 more
// than it), in both halves.
template <typename T>
constexpr uint32_t kMagic = std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u;

// x's codes as such numbers: one instruction, if the number is not a constant to
// the compiler (which would load it anew each time, or use two).
template <uint32_t MASK = 0x000f000fu>
__device__ __forceinline__ uint32_t numbers(uint32_t x, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(MASK), "r"(magic));
  return r;
}

// What two codes need: their zero points plus that number, and their scales.
template <typename T>
struct Pars {
  Pair<T> zero, scale;
};
// Of two 16-bit scales in the halves of p.
template <typename T>
__device__ __forceinline__ Pars<T> pars(uint32_t p, uint32_t magic = kMagic<T>) {
  Pars<T> r;
  r.zero = as_pair<T>(numbers(p, magic));
  if constexpr (std::is_same<T, __half>::value)
    r.scale = __floats2half2_rn(__uint_as_float((p & 0xfff0u) << 16), __uint_as_float(p & 0xfff00000u));
  else
    r.scale = as_pair<T>(p & 0xfff0fff0u);
  return r;
}
// Two values whose codes are the lowest four bits of x's halves.
template <typename T>
__device__ __forceinline__ uint32_t value2(uint32_t x, const Pars<T> &p, uint32_t magic = kMagic<T>) {
  const Pair<T> c = as_pair<T>(numbers(x, magic));
  return as_bits(__hmul2(__hsub2(c, p.zero), p.scale));
}
// The same of nibbles `at` and at + 4 of a word, at < 4.  fp16 has bits enough to
// take those with an odd number where they lie: 2^10 + 16 c.
template <typename T>
__device__ __forceinline__ uint32_t value2_at(uint32_t w, int at, const Pars<T> &p, uint32_t magic = kMagic<T>) {
  if constexpr (std::is_same<T, __half>::value) {
    if (at & 1) {
      const Pair<T> c = as_pair<T>(numbers<0x00f000f0u>(w >> 4 * (at - 1), magic));
      // (64 + c) - (64 + z), the latter being (1024 + z) - 960
      const Pair<T> d = __hfma2(c, __float2half2_rn(0.0625f), __hsub2(__float2half2_rn(960.f), p.zero));
      return as_bits(__hmul2(d, p.scale));
    }
  }
  return value2<T>(w >> 4 * at, p, magic);
}
// The eight channels of a word.
template <typename T>
__device__ __forceinline__ uint4 value8(uint32_t w, const Pars<T> &p) {
  return make_uint4(value2_at<T>(w, 0, p), value2_at<T>(w, 1, p), value2_at<T>(w, 2, p), value2_at<T>(w, 3, p));
}

}  // namespace q4
}  // namespace tide

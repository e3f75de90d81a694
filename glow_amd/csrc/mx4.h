// Microscaled 4-bit rows (laid out as mx4_layout.h says): the conversions and the checks of
// arguments that the kernels over them share.
#ifndef GLOW_MI355X_MX4_H
#define GLOW_MI355X_MX4_H

#include "common.h"
#include "mx4_layout.h"

#include <type_traits>

namespace mi355x {

// ---- element types ---------------------------------------------------------------

// E::Eight: eight neighbouring values in the registers they fill, from any address that is
// one of an element (loads of sixteen bytes need no more alignment than that).
typedef float mx_v8f __attribute__((ext_vector_type(8)));
typedef _Float16 mx_v8h __attribute__((ext_vector_type(8)));
typedef uint32_t mx_v4u __attribute__((ext_vector_type(4)));

struct F32 {
  typedef float T;
  typedef mx_v8f Eight;
  typedef Eight Eight1 __attribute__((aligned(4)));
  static constexpr int kSize = 4;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
  static __device__ __forceinline__ float get(const Eight &e, int j) { return e[j]; }
  static __device__ __forceinline__ Eight put(const float (&x)[8]) {
    return Eight{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
  }
};
struct F16 {
  typedef _Float16 T;
  typedef mx_v8h Eight;
  typedef Eight Eight1 __attribute__((aligned(2)));
  static constexpr int kSize = 2;
  static __device__ __forceinline__ float to(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from(float v) { return (_Float16)v; }
  static __device__ __forceinline__ float get(const Eight &e, int j) { return (float)e[j]; }
  // magnitudes of a pair as a word of whole numbers, and the float's bits of one of them
  static __device__ __forceinline__ uint32_t pair(const Eight &e, int i) {
    return __builtin_bit_cast(mx_v4u, e)[i];
  }
  static __device__ __forceinline__ uint32_t float_bits(uint32_t half) {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)half));
  }
  template <int SEL> static __device__ __forceinline__ uint32_t codes2(uint32_t old, uint32_t two, float scale) {
    typedef _Float16 Two __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(Two, two), scale, SEL);
  }
  static __device__ __forceinline__ Eight put(const float (&x)[8]) {
    Eight e;
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = (_Float16)x[j];
    return e;
  }
};
struct BF16 {
  typedef __bf16 T;
  typedef mx_v4u Eight;                     // a value is the upper half of its float's bits
  typedef Eight Eight1 __attribute__((aligned(2)));
  static constexpr int kSize = 2;
  static __device__ __forceinline__ float to(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 from(float v) { return (__bf16)v; }
  static __device__ __forceinline__ float get(const Eight &e, int j) {
    return __uint_as_float(j & 1 ? e[j >> 1] & 0xffff0000u : e[j >> 1] << 16);
  }
  static __device__ __forceinline__ uint32_t pair(const Eight &e, int i) { return e[i]; }
  static __device__ __forceinline__ uint32_t float_bits(uint32_t half) { return half << 16; }
  template <int SEL> static __device__ __forceinline__ uint32_t codes2(uint32_t old, uint32_t two, float scale) {
    typedef __bf16 Two __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(Two, two), scale, SEL);
  }
  static __device__ __forceinline__ Eight put(const float (&x)[8]) {
    typedef __bf16 Two __attribute__((ext_vector_type(2)));
    Eight e;
#pragma unroll
    for (int j = 0; j < 4; j++)
      e[j] = __builtin_bit_cast(uint32_t, Two{(__bf16)x[2 * j], (__bf16)x[2 * j + 1]});
    return e;
  }
};
struct MX4 {
  typedef uint8_t T;
  static constexpr int kSize = 0;
};

template <class E> __device__ __forceinline__ typename E::Eight load_eight(const typename E::T *p) {
  return *reinterpret_cast<const typename E::Eight1 *>(p);
}
// The same at the end of a row: `left` values (none where it is not positive), zeros behind.
template <class E> __device__ __forceinline__ typename E::Eight load_eight_end(const typename E::T *p, int left) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = j < left ? E::to(p[j]) : 0.0f;
  return E::put(x);                          // (exact: the values are of the type)
}
template <class E> __device__ __forceinline__ void load8(float (&x)[8], const typename E::T *p) {
  const typename E::Eight e = load_eight<E>(p);
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = E::get(e, j);
}
template <class E> __device__ __forceinline__ void load8_end(float (&x)[8], const typename E::T *p, int left) {
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = j < left ? E::to(p[j]) : 0.0f;
}
template <class E> __device__ __forceinline__ void store8(typename E::T *p, const float (&x)[8]) {
  *reinterpret_cast<typename E::Eight1 *>(p) = E::put(x);
}
template <class E>
__device__ __forceinline__ void store8_end(typename E::T *p, const float (&x)[8], int left) {
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < left) p[j] = E::from(x[j]);
}

// v / (1 + exp(-v)) with the hardware's exp2 and reciprocal, two instructions for the twenty of a
// correctly rounded quotient. In steps of 2^-24: 1.23 |v| from the exponent (its product's
// rounding and the constant's), 2 each from exp2 and the reciprocal, 1 each from the sum and the
// last product, so 1.23 |v| + 6 at most; next to nothing beside a 16- or 4-bit result's own rounding,
// and what a 32-bit result is off by. Below -87 the reciprocal is no normal number, or exp2 an
// infinity: -0 for magnitudes under 2^-119.
__device__ __forceinline__ float silu(float v) {
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}
__device__ __forceinline__ float relu(float v) { return v < 0 ? 0.0f : v; } // NaN stays
template <int ACT> __device__ __forceinline__ float activate(float v) {
  return ACT == MI355X_ACT_RELU ? relu(v) : ACT == MI355X_ACT_SILU ? silu(v) : v;
}
// f(std::integral_constant<int, ACT>) of the activation: the choice is made once, outside of
// loops (inside one the compiler computes all of them for every value: 8 of 17 us of a
// 256x256 tile without a K loop).
template <class F> __device__ __forceinline__ void with_activation(int act, F &&f) {
  if (act == MI355X_ACT_RELU) f(std::integral_constant<int, MI355X_ACT_RELU>());
  else if (act == MI355X_ACT_SILU) f(std::integral_constant<int, MI355X_ACT_SILU>());
  else f(std::integral_constant<int, MI355X_ACT_NONE>());
}

// ---- blocks ------------------------------------------------------------------------

// The largest magnitude as its bits: of IEEE numbers without their signs these are ordered
// as whole numbers are, infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t largest8(const float (&x)[8]) {
  // (maximum, unlike max, gives NaN as soon as one is NaN)
  float m = __builtin_fabsf(x[0]);
#pragma unroll
  for (int j = 1; j < 8; j++) m = __builtin_elementwise_maximum(m, __builtin_fabsf(x[j]));
  return magnitude_bits(m);
}
// The scale byte of a block whose largest magnitude has these bits: its exponent less the 2
// of E2M1's largest value, 0 at least; 255, NaN, for infinities and NaN.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t bits) {
  const uint32_t e = bits >> 23;
  return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}
// 2^(byte - 127); 2^-127 is no normal number. NaN blocks have codes of zero, whatever the
// values: their scale here is any that makes codes of zeros.
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// Eight values as codes, rounded to nearest with ties to even and saturated at 6 by the
// conversion instruction.
__device__ __forceinline__ uint32_t mx4_codes8(const float (&x)[8], uint32_t byte) {
  const float s = mx4_scale(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return byte == 255 ? 0 : w;
}
// The same of eight values in their own type's registers. 16-bit types are never widened: the
// largest magnitude is found two values at a time and the conversion takes pairs (half the
// instructions of the way through floats).
template <class E> __device__ __forceinline__ uint32_t largest8(const typename E::Eight &e) {
  if constexpr (E::kSize == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, magnitude_bits(e[j]));
    return m;
  } else {
    typedef uint16_t Two __attribute__((ext_vector_type(2)));
    Two m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(Two, E::pair(e, i) & 0x7fff7fffu));
    return max((uint32_t)m[0], (uint32_t)m[1]);
  }
}
// What largest8 gives as a float's bits (16-bit types: after the maximum over the block).
template <class E> __device__ __forceinline__ uint32_t largest_bits(uint32_t m) {
  if constexpr (E::kSize == 4) return m;
  else return E::float_bits(m);
}
template <class E> __device__ __forceinline__ uint32_t mx4_codes8_of(const typename E::Eight &e, uint32_t byte) {
  uint32_t w = 0;
  const float s = mx4_scale(byte);
  if constexpr (E::kSize == 4) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, e[0], e[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, e[2], e[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, e[4], e[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, e[6], e[7], s, 3);
  } else {
    w = E::template codes2<0>(w, E::pair(e, 0), s);
    w = E::template codes2<1>(w, E::pair(e, 1), s);
    w = E::template codes2<2>(w, E::pair(e, 2), s);
    w = E::template codes2<3>(w, E::pair(e, 3), s);
  }
  return byte == 255 ? 0 : w;
}
typedef float mx4_v2f __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void mx4_values8(float (&x)[8], uint32_t codes, uint32_t byte) {
  const float s = mx4_scale(byte);
  const mx4_v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0);
  const mx4_v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
  const mx4_v2f c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2);
  const mx4_v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
  const float nan = __builtin_nanf("");
#pragma unroll
  for (int j = 0; j < 2; j++) {
    x[j] = byte == 255 ? nan : a[j];
    x[2 + j] = byte == 255 ? nan : b[j];
    x[4 + j] = byte == 255 ? nan : c[j];
    x[6 + j] = byte == 255 ? nan : d[j];
  }
}
// A value with its counterpart 16 or 32 lanes away, in both: x and the one swapped in.
__device__ __forceinline__ uint32_t max_across16(uint32_t m) {
  const auto s = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return max((uint32_t)s[0], (uint32_t)s[1]);
}
__device__ __forceinline__ uint32_t max_across32(uint32_t m) {
  const auto s = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return max((uint32_t)s[0], (uint32_t)s[1]);
}
__device__ __forceinline__ float add_across16(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float add_across32(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// x + x of the lane N further on in the row of sixteen: the lanes of a row N apart hold their
// sum once this is done for 8, 4, .. down to N.
template <int N> __device__ __forceinline__ float add_rotated(float x) {
  return x + __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), 0x120 + N, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = add_rotated<1>(add_rotated<2>(add_rotated<4>(add_rotated<8>(x))));
  return add_across32(add_across16(x));
}
// The largest of four neighbouring lanes, in all four.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true)); // lanes 1 0 3 2
  return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true)); // 2 3 0 1
}

// A group's sixteen lanes, eight columns each, write it: codes, the word of scales, and
// behind the last group the zeros that fill the row up. `l` is the lane of the group.
template <class E>
__device__ __forceinline__ void mx4_store_group(uint8_t *row, int groups, int g, int l,
                                                const typename E::Eight &x) {
  const uint32_t byte = mx4_scale_byte(largest_bits<E>(quad_max(largest8<E>(x))));
  reinterpret_cast<uint32_t *>(row + (size_t)g * kMxGroupBytes)[l] = mx4_codes8_of<E>(x, byte);
  // lanes 0, 4, 8, 12 hold the four scales: each lane's byte in its place, joined by or
  uint32_t word = (l & 3) == 0 ? byte << (8 * (l >> 2)) : 0;
  word |= (uint32_t)__builtin_amdgcn_mov_dpp((int)word, 0x124, 0xf, 0xf, true); // row_ror:4
  word |= (uint32_t)__builtin_amdgcn_mov_dpp((int)word, 0x128, 0xf, 0xf, true); // row_ror:8
  uint32_t *scales = reinterpret_cast<uint32_t *>(row + (size_t)groups * kMxGroupBytes);
  if (l == 0) scales[g] = word;
  else if (g == groups - 1 && l < 4 && l <= ((-groups) & 3)) scales[g + l] = 0;
}

// ---- checks of arguments -----------------------------------------------------------

inline bool float_type(int type) { return type == MI355X_F32 || type == MI355X_F16 || type == MI355X_BF16; }
inline size_t float_size(int type) { return type == MI355X_F32 ? 4 : 2; }

// Whether a tensor of rows can be addressed: pointer, distance between rows. Says why not.
inline int check_rows(const char *what, const void *p, int type, size_t row_bytes, size_t rows, size_t cols) {
  MI355X_REQUIRE(type == MI355X_MX4 || float_type(type), "%s: unknown element type %d", what, type);
  MI355X_REQUIRE(cols <= 0x7fffffff && rows <= 0x7fffffff,
                 "%s: %zu x %zu, up to 2^31 - 1 each are supported", what, rows, cols);
  const size_t align = type == MI355X_MX4 ? 16 : float_size(type);
  const size_t least = type == MI355X_MX4 ? mx4_row_bytes_of(cols) : cols * align;
  MI355X_REQUIRE(row_bytes >= least, "%s: rows %zu bytes apart, %zu columns take %zu", what, row_bytes, cols, least);
  MI355X_REQUIRE(row_bytes % align == 0 && (uintptr_t)p % align == 0,
                 "%s: the address and the distance between rows have to be multiples of %zu", what, align);
  size_t span;
  MI355X_REQUIRE(!__builtin_mul_overflow(rows, row_bytes, &span) && span <= PTRDIFF_MAX,
                 "%s: %zu rows %zu bytes apart", what, rows, row_bytes);
  MI355X_REQUIRE(p || rows == 0 || least == 0, "%s: NULL", what);
  return MI355X_OK;
}
// Bytes from the first to the last one that a tensor of rows uses.
inline size_t rows_span(int type, size_t row_bytes, size_t rows, size_t cols) {
  if (!rows) return 0;
  return (rows - 1) * row_bytes + (type == MI355X_MX4 ? mx4_row_bytes_of(cols) : cols * float_size(type));
}
inline bool overlaps(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a_bytes && b_bytes && a && b && x < y + b_bytes && y < x + a_bytes;
}

// Launches the quantisation of checked rows (mx4.hip).
int mx4_quantize_launch(uint8_t *dst, size_t dst_row_bytes, const void *src, int src_type,
                        size_t src_row_bytes, size_t rows, size_t cols, hipStream_t st);

} // namespace mi355x

#endif

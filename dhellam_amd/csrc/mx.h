// Microscaled floating point (the OCP MX formats): a row is cut into blocks of 32 elements along its columns; a block has one
// power of two as its scale (an exponent code e: 2^(e - 127), 255 for NaN) and its elements in e4m3 (8 bits) or e2m1 (4 bits).
//
// In memory, for a matrix of `rows` x `cols`, with kp = cols rounded up to 128:
//   codes   [rows][kp] bytes (e4m3) or [rows][kp / 2] bytes (e2m1, the even column in the low half), zeros behind cols
//   scales  [kp / 128][rows4 / 4][4][4] bytes, rows4 = rows rounded up to 4: the code of block i of columns 128 c .. of row r
//           is at [c][r / 4][i][r % 4]; zeros for rows and blocks that are not there
// A cell of 16 bytes holds four rows' scales of 128 columns with the rows inside: a lane of a matrix instruction that owns
// block i of rows 4 r .. 4 r + 3 (one of each of four operand blocks) takes the four scales as one dword, which the
// instruction picks bytes from by itself, and the 64 lanes of a wavefront read 256 consecutive bytes.
#pragma once
#include "common.h"

namespace dh {

// e8m0 code of a block from the bits of its largest magnitude in fp32: floor(log2) less the exponent of the format's largest
// element (the rule of the specification, under which the largest elements may saturate), one more where `cover` asks that
// nothing saturates and the largest element lies past 1.75 x 2^8 or 1.5 x 2^2 of it.  Magnitudes below the smallest scale
// share 2^-127.  Not finite: 255.
template <bool E4> __device__ __forceinline__ uint32_t mx_scale_code(uint32_t top, int cover) {
  int e = (int)(top >> 23) - (E4 ? 8 : 2);
  if (cover && (top & 0x7fffffu) > (E4 ? 0x600000u : 0x400000u)) e += 1;
  e = e < 0 ? 0 : e;
  return top >= 0x7f800000u ? 255u : (uint32_t)e;
}
// 2^(127 - code), by which the block's values are multiplied: exact but for what lies far below the smallest element.
// (A finite block's code is at most 253, e2m1's under `cover`, so this is a normal number.  For 255 it is none: the codes are cleared.)
__device__ __forceinline__ float mx_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// Four consecutive elements, already scaled, to e4m3 (round to nearest even, saturating at 448).
__device__ __forceinline__ uint32_t mx_e4m3x4(float a, float b, float c, float d) {
  a = __builtin_amdgcn_fmed3f(a, -448.f, 448.f);
  b = __builtin_amdgcn_fmed3f(b, -448.f, 448.f);
  c = __builtin_amdgcn_fmed3f(c, -448.f, 448.f);
  d = __builtin_amdgcn_fmed3f(d, -448.f, 448.f);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// Eight consecutive elements, already scaled, to e2m1 (round to nearest even; the conversion saturates at 6).
__device__ __forceinline__ uint32_t mx_e2m1x8(const float *v) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
  return r;
}

// Eight consecutive values of a block with the given code: 8 bytes of e4m3 (lo, hi) or 4 bytes of e2m1 (lo).
template <bool E4> struct MxPack { uint32_t lo, hi; };
template <bool E4> __device__ __forceinline__ MxPack<E4> mx_pack(const float (&v)[8], uint32_t code) {
  const float inv = mx_inverse(code);
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = v[j] * inv;
  MxPack<E4> o;
  if constexpr (E4) {
    o.lo = mx_e4m3x4(s[0], s[1], s[2], s[3]);
    o.hi = mx_e4m3x4(s[4], s[5], s[6], s[7]);
    o.hi = code == 255u ? 0u : o.hi;
  } else {
    o.lo = mx_e2m1x8(s);
    o.hi = 0;
  }
  o.lo = code == 255u ? 0u : o.lo;
  return o;
}

// Largest of a value over four neighbouring lanes (quad exchanges inside the vector ALU).
__device__ __forceinline__ uint32_t quad_umax(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);      // lanes 1 0 3 2
  v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);               // lanes 2 3 0 1
  return v > o ? v : o;
}

// Largest over the lanes l, l ^ 16, l ^ 32 and l ^ 48, in the vector ALU as well: a swap leaves a lane its own value in one result and the
// other lane's in the other.  PAIRS: two 16-bit values a lane.
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
template <bool PAIRS> __device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) {
  if constexpr (PAIRS) return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, a), __builtin_bit_cast(ushort2v, b)));
  else return a > b ? a : b;
}
template <bool PAIRS> __device__ __forceinline__ uint32_t column_umax(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = umax<PAIRS>(r[0], r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return umax<PAIRS>(q[0], q[1]);
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 8 values of type T at any address that suits T: 16-byte loads, which the hardware takes at any alignment.
template <typename T> struct alignas(sizeof(T)) Loose8 { T v[8]; };
typedef uint32_t loose2_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t loose4_u32x4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct LooseU4 { using type = loose4_u32x4; };
template <> struct LooseU4<bf16_t> { using type = loose2_u32x4; };
template <> struct LooseU4<f16_t> { using type = loose2_u32x4; };
template <typename T> __device__ __forceinline__ Loose8<T> load_nt(const T *p) {
  using V = typename LooseU4<T>::type;
  Loose8<T> x;
#pragma unroll
  for (int i = 0; i < (int)sizeof(x) / 16; ++i) {
    const dh_u32x4 q = __builtin_nontemporal_load(reinterpret_cast<const V *>(p) + i);
    __builtin_memcpy(reinterpret_cast<char *>(&x) + 16 * i, &q, 16);
  }
  return x;
}
template <typename T> __device__ __forceinline__ void store_nt(T *p, const Loose8<T> &x) {
  using V = typename LooseU4<T>::type;
#pragma unroll
  for (int i = 0; i < (int)sizeof(x) / 16; ++i) {
    dh_u32x4 q;
    __builtin_memcpy(&q, reinterpret_cast<const char *>(&x) + 16 * i, 16);
    __builtin_nontemporal_store(q, reinterpret_cast<V *>(p) + i);
  }
}
static inline int64_t mx_rows4(int64_t rows) { return (rows + 3) / 4 * 4; }

}  // namespace dh

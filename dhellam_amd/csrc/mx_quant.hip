// Quantisation to microscaled floating point, along the rows of a matrix, along its columns, or both in one pass over it, and the
// RMS norm (with the residual's addition) that writes its result in 8 bits with scales.  Format and rounding: mx.h.
#include <algorithm>
#include <type_traits>

#include "mx.h"

namespace dh {

// ---- quantisation -------------------------------------------------------------------------------------------------------
// A workgroup takes 128 x 128 elements, a wavefront 32 rows of them, a lane 8 rows x 8 columns (row group lane / 16, column
// group lane % 16), so that each of its 8 loads brings 4 rows of 128 elements.  A block along a row lies in the 4 lanes of a
// quad, a block along a column in the lanes l, l ^ 16, l ^ 32, l ^ 48 (8 rows each): both maxima are a few exchanges between
// lanes, and no element goes through LDS before it is rounded.  What a lane holds of a column are 8 neighbouring elements
// of the transposed result: they are packed in registers and go through LDS as 8 (4) bytes, so that memory gets
// 128 (64) bytes of a row of the transpose at a time.
// Bound by memory: 4096 x 7168 in bf16 to e4m3, along both directions 25 to 27 us (119 MB; 23.0 at what a copy of 1 GiB reaches, 5.2 TB/s); 4096 x 8192
// along the rows 18.5 (101 MB; 19.5).  4096 x 7168 in other forms: bf16 to e2m1 14.8 along the rows (5.0 TB/s) and 20.7 along both (4.3), fp32 to e4m3
// 22.6 (6.5) and 31.8 (5.6).  A few rows: 4 to 5 us, most of it the launch.  Five or six workgroups on a
// compute unit by fewer registers were slower.
struct QuantParams {
  const void *x;
  int64_t rows, cols, ldx;
  uint8_t *codes, *scales, *codes_t, *scales_t;
  int cover;
  int tiles_c;
};

// What a lane holds of a row: 8 values, 16-bit ones in pairs as they came.
template <typename T> struct Held8 {
  static constexpr bool PAIRS = sizeof(T) == 2;
  static constexpr int N = PAIRS ? 4 : 8;                  // registers
  uint32_t v[N];
  __device__ __forceinline__ void load(const T *p) {
    const Loose8<T> x = *reinterpret_cast<const Loose8<T> *>(p);
    __builtin_memcpy(v, &x, sizeof(x));
  }
  __device__ __forceinline__ void load_first(const T *p, int n) {
    T x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? p[j] : from_f<T>(0.f);
    __builtin_memcpy(v, x, sizeof(x));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0;
  }
  // the first n values (0..8) away, zeros behind the last
  template <int BY> __device__ __forceinline__ void drop_registers(bool yes) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = yes ? (i + BY < N ? v[(i + BY) % N] : 0u) : v[i];
  }
  __device__ __forceinline__ void drop(int n) {
    if constexpr (PAIRS) {
      drop_registers<2>(n & 4);
      drop_registers<1>(n & 2);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = n & 1 ? v[i] >> 16 | (i + 1 < N ? v[(i + 1) % N] << 16 : 0u) : v[i];
    } else {
      drop_registers<4>(n & 4);
      drop_registers<2>(n & 2);
      drop_registers<1>(n & 1);
    }
    if (n >= 8) clear();
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (!PAIRS) return __uint_as_float(v[j]);
    else return to_f(__builtin_bit_cast(T, (uint16_t)(v[j >> 1] >> (16 * (j & 1)))));
  }
};
// Magnitudes of a register, and the fp32 bits of the one in its half h.
template <typename T> __device__ __forceinline__ uint32_t mags(uint32_t v) { return v & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu); }
template <typename T> __device__ __forceinline__ uint32_t mag_bits(uint32_t m, int h) {
  if constexpr (sizeof(T) == 4) return m;
  else return __float_as_uint(to_f(__builtin_bit_cast(T, (uint16_t)(m >> (16 * h)))));
}

// Where 8 rows' codes of a column lie in LDS: column c of 16 units of CB bytes.  The 64 lanes that write at once have c = 8 cg + j (cg of 0..15) and
// units 4 w + rg (rg of 0..3): slots and units are exchanged by bits of cg, so that they fall on all 64 banks; 16 bytes stay together.
template <bool E4> __device__ __forceinline__ int mx_tile_at(int c, int unit) {
  if constexpr (E4) return (c ^ ((c >> 3) & 1)) * 128 + ((unit ^ (((c >> 4) & 7) << 1)) << 3);
  else return (c ^ ((c >> 3) & 3)) * 64 + ((unit ^ (((c >> 5) & 3) << 2)) << 2);
}

template <typename T, bool E4, bool ROWS, bool COLS>
__global__ void __launch_bounds__(256) mx_quantise_kernel(const QuantParams p) {
  using H = Held8<T>;
  constexpr bool PAIRS = H::PAIRS;
  constexpr int CB = E4 ? 8 : 4;                           // bytes of 8 codes
  __shared__ __attribute__((aligned(16))) uint8_t tile[COLS ? 128 * 16 * CB : 16];
  __shared__ __attribute__((aligned(16))) uint8_t sr[ROWS ? 512 : 16], sc[COLS ? 512 : 16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int rg = lane >> 4, cg = lane & 15;
  const int64_t tr = blockIdx.x / p.tiles_c, tc = blockIdx.x % p.tiles_c;
  const int64_t r0 = tr * 128, c0 = tc * 128;
  const int64_t row0 = r0 + 32 * w + 8 * rg, col0 = c0 + 8 * cg;
  const T *x = reinterpret_cast<const T *>(p.x);
  H v[8];
  if (r0 + 128 <= p.rows && c0 + 128 <= p.cols) {          // (of the workgroup: no load waits for a comparison)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(x + (row0 + i) * p.ldx + col0);
  } else if (p.cols >= 8) {
    // nor here: what lies past the end is loaded from before it and taken away behind the loads (24 x 3584 4.8 us,
    // 5.4 with loads in branches; 1999 x 1001 5.3 and 6.2)
    const int64_t at = std::min(col0, p.cols - 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(x + std::min(row0 + i, p.rows - 1) * p.ldx + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].drop(row0 + i < p.rows ? (int)std::min<int64_t>(col0 - at, 8) : 8);
  } else {
    const int64_t left = p.cols - col0;                    // (fewer than 8)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row0 + i < p.rows && left > 0) v[i].load_first(x + (row0 + i) * p.ldx + col0, (int)left);
      else v[i].clear();
    }
  }
  if constexpr (ROWS) {
    const int64_t kp = (int64_t)p.tiles_c * 128;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < H::N; ++j) top = umax<PAIRS>(top, mags<T>(v[i].v[j]));
      if constexpr (PAIRS) top = top > (top << 16) ? top >> 16 : top & 0xffffu;      // the larger half, below
      const uint32_t code = mx_scale_code<E4>(mag_bits<T>(quad_umax(top), 0), p.cover);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[i].at(j);
      const MxPack<E4> o = mx_pack<E4>(f, code);
      const int r = 32 * w + 8 * rg + i;
      if (r0 + r < p.rows) {
        uint8_t *dst = p.codes + (r0 + r) * (E4 ? kp : kp / 2) + (c0 + 8 * cg) / (E4 ? 1 : 2);
        if constexpr (E4) *reinterpret_cast<uint2 *>(dst) = uint2{o.lo, o.hi};
        else *reinterpret_cast<uint32_t *>(dst) = o.lo;
      }
      if ((cg & 3) == 0) sr[(r >> 2) * 16 + (cg >> 2) * 4 + (r & 3)] = (uint8_t)code;
    }
  }
  if constexpr (COLS) {
    uint32_t top[H::N];
#pragma unroll
    for (int j = 0; j < H::N; ++j) {
      top[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top[j] = umax<PAIRS>(top[j], mags<T>(v[i].v[j]));
      top[j] = column_umax<PAIRS>(top[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t code = mx_scale_code<E4>(mag_bits<T>(top[PAIRS ? j >> 1 : j], j & 1), p.cover);
      float col[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) col[i] = v[i].at(j);
      const MxPack<E4> o = mx_pack<E4>(col, code);
      const int c = 8 * cg + j;
      uint8_t *dst = tile + mx_tile_at<E4>(c, 4 * w + rg);
      if constexpr (E4) *reinterpret_cast<uint2 *>(dst) = uint2{o.lo, o.hi};
      else *reinterpret_cast<uint32_t *>(dst) = o.lo;
      if (rg == 0) sc[(c >> 2) * 16 + w * 4 + (c & 3)] = (uint8_t)code;
    }
  }
  __syncthreads();
  if constexpr (ROWS) {
    // the tile's 32 cells of scales, one behind the other
    const int64_t cells = (p.rows + 3) / 4;
    if (tid < 32 && r0 / 4 + tid < cells)
      *reinterpret_cast<dh_u32x4 *>(p.scales + (tc * cells + r0 / 4 + tid) * 16) = *reinterpret_cast<const dh_u32x4 *>(sr + tid * 16);
  }
  if constexpr (COLS) {
    const int64_t cells = (p.cols + 3) / 4, kpt = (p.rows + 127) / 128 * 128, ldt = E4 ? kpt : kpt / 2;
    if (tid >= 64 && tid < 96 && c0 / 4 + tid - 64 < cells)
      *reinterpret_cast<dh_u32x4 *>(p.scales_t + (tr * cells + c0 / 4 + tid - 64) * 16) = *reinterpret_cast<const dh_u32x4 *>(sc + (tid - 64) * 16);
    constexpr int LPR = CB;                                // lanes of 16 bytes a row of the transpose takes
#pragma unroll
    for (int it = 0; it < 128 * LPR / 256; ++it) {
      const int c = (it * 256 + tid) / LPR, b = (it * 256 + tid) % LPR;
      if (c0 + c < p.cols)
        *reinterpret_cast<dh_u32x4 *>(p.codes_t + (c0 + c) * ldt + tr * (16 * CB) + b * 16) =
            *reinterpret_cast<const dh_u32x4 *>(tile + mx_tile_at<E4>(c, b * (16 / CB)));
    }
  }
}

template <typename T, bool E4> static void launch_quantise(const QuantParams &p, hipStream_t st) {
  const dim3 grid((unsigned)(cdiv(p.rows, 128) * p.tiles_c)), block(256);
  if (p.codes && p.codes_t) hipLaunchKernelGGL((mx_quantise_kernel<T, E4, true, true>), grid, block, 0, st, p);
  else if (p.codes) hipLaunchKernelGGL((mx_quantise_kernel<T, E4, true, false>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((mx_quantise_kernel<T, E4, false, true>), grid, block, 0, st, p);
}

// ---- residual addition, RMS norm, 8 bits with scales -----------------------------------------------------------------------
// A row belongs to TPR threads, a thread holds VPT groups of 8 columns of it (group t + i TPR) from the first load to the last
// store.  A block of 32 lies in the 4 lanes of a quad, the four blocks of a dword of scales in 16 lanes.
// Bound by memory: 8192 x 8192 in bf16 with a residual 89 us, 5.3 TB/s (118 with the loads in branches, whose waits come one by one, and less exact: so whole
// rows have a form without), in fp32 180 us (4.9 TB/s).  One row of 8192: 4.5 us, the launch and two trips to memory; 256 rows of 1024 threads 7, 512 and 1024
// rows of 256 threads 15 and 21, a few rows a compute unit one behind the other.
struct NormMxParams {
  const void *x, *residual, *gamma;
  void *sum_out, *y;
  uint8_t *codes, *scales;
  float *rsigma;
  int64_t rows;
  int cols, cover;
  float eps, shift;
};

// (without NT the accesses keep their lines in the caches; with it, where a call moves more than these hold, they do not displace others)
template <typename T, bool NT> __device__ __forceinline__ void store8(T *p, const Loose8<T> &o, int n) {
  if (n >= 8) {
    if constexpr (NT) store_nt(p, o);
    else *reinterpret_cast<Loose8<T> *>(p) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = o.v[j];
  }
}
template <typename T> __device__ __forceinline__ Loose8<T> rounded8(const float (&f)[8]) {
  Loose8<T> o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o.v[j] = from_f<T>(f[j]);
  return o;
}
// 8 columns of which n exist (WHOLE: all or none), zeros for the others
template <typename T, bool WHOLE, bool NT> __device__ __forceinline__ Loose8<T> fetch8(const T *p, int n) {
  Loose8<T> x;
  if (n >= 8) {
    x = NT ? load_nt(p) : *reinterpret_cast<const Loose8<T> *>(p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x.v[j] = from_f<T>(0.f);
    if (!WHOLE)
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < n) x.v[j] = p[j];
  }
  return x;
}
// x + residual, rounded to T as a separate addition stores it
template <typename T> __device__ __forceinline__ Loose8<T> sum8(const Loose8<T> &a, const Loose8<T> &b) {
  Loose8<T> o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o.v[j] = from_f<T>(to_f(a.v[j]) + to_f(b.v[j]));
  return o;
}
// The sum of 8 squares, in 64 bits as everything up to 1/rms.
template <typename T> __device__ __forceinline__ double squares8(const Loose8<T> &a) {
  double s[2] = {0.0, 0.0};
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j & 1] = fma((double)to_f(a.v[j]), (double)to_f(a.v[j]), s[j & 1]);
  return s[0] + s[1];
}
template <int CTRL> __device__ __forceinline__ double dpp64(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)bits, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(bits >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// All 64 lanes' sum (a quad's, two quads', a row's of 16, the four rows').
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<0xb1>(v);      // lanes l ^ 1
  v += dpp64<0x4e>(v);      // l ^ 2
  v += dpp64<0x141>(v);     // 7 - l of the half row
  v += dpp64<0x140>(v);     // 15 - l of the row
  return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}
// 1 / sqrt(a) to 2^-44 for any a of 64 bits: fp32's for a brought to [0.5, 2) by an even power of two, and one step of Newton's iteration
// (fp32's alone where that is 0, infinite or NaN: a row that holds an infinity has 1/rms = 0).
__device__ __forceinline__ double rsqrt64(double a) {
  const int even = __builtin_amdgcn_frexp_exp(a) & ~1;     // (0 for what is not finite)
  const double m = ldexp(a, -even);
  const float r0 = 1.0f / sqrtf((float)m);
  const double r = (double)r0;
  return ldexp(r0 > 0.f && r0 < INFINITY ? fma(r * 0.5, fma(-m * r, r, 1.0), r) : r, -(even >> 1));
}
// What was computed from x before is computed again behind this, not kept: a row and gamma in 32 and in 64 bits do not fit the registers.
template <typename T> __device__ __forceinline__ void keep_packed(Loose8<T> &x) {
  uint32_t v[sizeof(x) / 4];
  __builtin_memcpy(v, &x, sizeof(x));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(x) / 4); ++i) asm volatile("" : "+v"(v[i]));
  __builtin_memcpy(&x, v, sizeof(x));
}
// v to fp32, rounded to the neighbour whose last bit is set where v lies between two: a rounding to fewer bits behind it gives what it gives for v itself.
__device__ __forceinline__ float to_odd(double v) {
  const float f = (float)v;
  const uint32_t bits = __float_as_uint(f);
  const double back = (double)f;
  const bool as_it_is = back == v || (bits & 1) || f == 0.f || !(fabsf(f) < INFINITY);
  const uint32_t odd = (v > back) == (f > 0.f) ? bits + 1 : bits - 1;
  return __uint_as_float(as_it_is ? bits : odd);
}
// The magnitude (fp32 bits) past which the largest of a block makes its elements' fp32 arithmetic safe from the smallest numbers: where x / rms or the
// result is subnormal it is off by more than 2^-22 of itself, but by 2^-150 of the largest |gamma| (or of 1) at most, and it is a zero
// under a scale of 2^-109 of that.  The larger of the quad's, from the gammas that its threads hold.  (None for a row whose 1/rms may not be normal in fp32.)
template <typename T> __device__ __forceinline__ float gamma_top(const Loose8<T> &gamma, float shift, float top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(to_f(gamma.v[j]) + shift));
  return top;
}
__device__ __forceinline__ uint32_t norm_safe_above(float gamma_top) { return __float_as_uint(0x1p-100f * __uint_as_float(quad_umax(magnitude(gamma_top)))); }
__device__ __forceinline__ uint32_t norm_safe_row(uint32_t safe_above, double rs) { return rs >= 0x1p-100 && rs <= 0x1p100 ? safe_above : ~0u; }
// Not 0 where one of the values is not a zero.
template <typename T> __device__ __forceinline__ uint32_t any_bits(const Loose8<T> &x) {
  uint32_t v[sizeof(x) / 4], any = 0;
  __builtin_memcpy(v, &x, sizeof(x));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(x) / 4); ++i) any |= mags<T>(v[i]);
  return any;
}
// The result of 8 columns (n exist) of a row: y, codes; returns the block's scale code (the same in the quad).
// fp32's y is off by 2^-22 of itself at most: 1/rms rounded, gamma + 1 rounded, two products.  Every place where a scale or an element changes has
// zeros behind its fourth bit; a y that comes that near to one is formed again in 64 bits, so that codes and scales are those of
// the exact y (to 2^-43).  One wavefront in 115 has such an element among its 512 (zeros count as near too, but are not formed again); without, 1 to 3
// elements in 2 million were the neighbour.  `lowest`: the least of the largest magnitudes of the blocks so far; where fp32 does not do for
// a block (norm_safe_row), the row is formed again by the form of EXACT, all in 64 bits.  A result past fp32's largest number is not finite.
// 8192 x 8192 in bf16 with a residual: 80 us in fp32 throughout, 87 with the sums and near elements in 64 bits, 89 with the range test and the form of
// EXACT (90 with that test at every block, and 5.5 for one row instead of 4.5); 512 x 8192 15 to 16.  All four groups' y before one test for near ones were slower.
template <typename T, bool EXACT = false> __device__ __forceinline__ uint32_t norm_out8(const NormMxParams &p, Loose8<T> x, Loose8<T> gamma, double rs64,
                                                                                        uint32_t &lowest, int64_t row, int g, int64_t kp, bool active) {
  const int n = p.cols - 8 * g;
  const float rs = (float)rs64;
  constexpr uint32_t NEAR = 4;                             // steps of fp32: 2^-22 of y at most
  keep_packed(x);
  keep_packed(gamma);
  float y[8];
  uint32_t near = ~0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (EXACT) y[j] = to_odd((double)to_f(x.v[j]) * rs64 * ((double)to_f(gamma.v[j]) + (double)p.shift));
    else y[j] = to_f(x.v[j]) * rs * (to_f(gamma.v[j]) + p.shift);
    if (n < 8 && j >= n) y[j] = 0.f;                       // (a row of infinities or NaN makes products of zeros NaN)
    else near = std::min(near, (__float_as_uint(y[j]) + NEAR) << 13);
  }
  if (!EXACT && near <= 2 * NEAR << 13 && active) {
    keep_packed(x);
    keep_packed(gamma);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n && (__float_as_uint(y[j]) + NEAR) << 13 <= 2 * NEAR << 13 && y[j] != 0.f)
        y[j] = to_odd((double)to_f(x.v[j]) * rs64 * ((double)to_f(gamma.v[j]) + (double)p.shift));
  }
  if (p.y && active && n > 0) store8<T, false>(reinterpret_cast<T *>(p.y) + row * p.cols + 8 * g, rounded8<T>(y), n);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t m = magnitude(y[j]);
    top = top > m ? top : m;
  }
  top = quad_umax(top);
  if (!EXACT && 8 * (g & ~3) < p.cols) lowest = std::min(lowest, top);
  const uint32_t code = mx_scale_code<true>(top, p.cover);
  if (active) {
    const MxPack<true> o = mx_pack<true>(y, code);
    *reinterpret_cast<uint2 *>(p.codes + row * kp + 8 * g) = uint2{o.lo, o.hi};
  }
  return active ? code : 0u;
}

// TPR threads a row, ROWS rows a workgroup; gamma stays in registers.  All loads of a row go out before anything waits for one.
template <typename T, int TPR, int VPT, int ROWS, bool WHOLE, bool RES, bool NT>
__global__ void __launch_bounds__(TPR *ROWS, VPT == 4 ? (sizeof(T) == 4 ? 3 : 4) : 1) norm_mx_kernel(const NormMxParams p) {
  constexpr int WPR = TPR / 64;
  __shared__ double red[2][WPR * ROWS];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int groups = (p.cols + 127) / 128 * 16;
  const int64_t kp = (int64_t)groups * 8, cells = (p.rows + 3) / 4;
  const double inv_cols = 1.0 / (double)p.cols;
  const T *x = reinterpret_cast<const T *>(p.x), *res = reinterpret_cast<const T *>(p.residual);
  Loose8<T> gamma[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int g = lane + i * TPR;
    gamma[i] = fetch8<T, WHOLE, false>(reinterpret_cast<const T *>(p.gamma) + 8 * g, p.cols - 8 * g);
  }
  uint32_t safe_above = 0;
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < 4 * cells; row0 += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    const int64_t row = row0 + sub;
    const bool active = row < p.rows;
    Loose8<T> held[VPT], add[RES ? VPT : 1];               // the row as it is normalised, in its own type
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = lane + i * TPR, n = active ? p.cols - 8 * g : 0;
      held[i] = fetch8<T, WHOLE, NT>(x + row * p.cols + 8 * g, n);
      if constexpr (RES) add[i] = fetch8<T, WHOLE, NT>(res + row * p.cols + 8 * g, n);
    }
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = lane + i * TPR, n = active ? p.cols - 8 * g : 0;
      if constexpr (RES) {
        held[i] = sum8(held[i], add[i]);
        if (n > 0) store8<T, NT>(reinterpret_cast<T *>(p.sum_out) + row * p.cols + 8 * g, held[i], n);
      }
      mine += squares8(held[i]);
    }
    double s = wave_sum64(mine);
    if constexpr (WPR > 1) {                               // (two sets of sums: the next row's are written before every wavefront has read these)
      if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = s;
      __syncthreads();
      s = 0.0;
#pragma unroll
      for (int i = 0; i < WPR; ++i) s += red[turn][sub * WPR + i];
    }
    const double rs = rsqrt64(s * inv_cols + (double)p.eps);
    if (row0 == (int64_t)blockIdx.x * ROWS) {              // (behind the first row's loads, which do not wait for gamma)
      float largest = 1.f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) largest = gamma_top(gamma[i], p.shift, largest);
      safe_above = norm_safe_above(largest);
    }
    uint32_t lowest = ~0u;
    auto out = [&](auto exact) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int g = lane + i * TPR;
        if (g >= groups) continue;                         // (16 lanes at a time: groups is a multiple of 16)
        const uint32_t code = norm_out8<T, decltype(exact)::value>(p, held[i], gamma[i], rs, lowest, row, g, kp, active);
        if ((lane & 3) == 0 && row < 4 * cells)
          p.scales[((int64_t)(g >> 4) * cells + (row >> 2)) * 16 + ((g >> 2) & 3) * 4 + (row & 3)] = (uint8_t)code;
      }
    };
    out(std::false_type{});
    const uint32_t safe_row = norm_safe_row(safe_above, rs);
    if (__builtin_expect(active && !(lowest > safe_row), 0)) {      // (the same in the quad)
      uint32_t any = 0;                                    // (zeros, a masked row's, are what they are)
#pragma unroll
      for (int i = 0; i < VPT; ++i) any |= any_bits(held[i]);
      if (safe_row == ~0u || quad_umax(any)) out(std::true_type{});
    }
    if (active && lane == 0) p.rsigma[row] = (float)rs;
  }
}

// Rows of any length: one workgroup a row, read once for its statistics and again, from the cache, for its result.  2048 x 20000 in bf16 with a residual
// 99 us, 2.9 TB/s: a row's two passes wait for one another, and 16 wavefronts of these registers fill a compute unit.
template <typename T, bool RES>
__global__ void __launch_bounds__(1024) norm_mx_long_kernel(const NormMxParams p) {
  __shared__ double red[16];
  const int groups = (p.cols + 127) / 128 * 16;
  const int64_t kp = (int64_t)groups * 8, cells = (p.rows + 3) / 4;
  const T *res = reinterpret_cast<const T *>(p.residual);
  for (int64_t row = blockIdx.x; row < 4 * cells; row += gridDim.x) {
    const bool active = row < p.rows;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.cols;
    double s = 0.0;
    for (int g = threadIdx.x; active && g < groups; g += 1024) {
      const int n = p.cols - 8 * g;
      Loose8<T> v = fetch8<T, false, false>(x + 8 * g, n);
      if constexpr (RES) {
        v = sum8(v, fetch8<T, false, false>(res + row * p.cols + 8 * g, n));
        if (n > 0) store8<T, false>(reinterpret_cast<T *>(p.sum_out) + row * p.cols + 8 * g, v, n);
      }
      s += squares8(v);
    }
    s = wave_sum64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i];
    __syncthreads();                                       // (the next row's are written behind these reads)
    const double rs = rsqrt64(s / (double)p.cols + (double)p.eps);
    if (RES) x = reinterpret_cast<const T *>(p.sum_out) + row * p.cols;      // a thread reads what it wrote itself
    for (int g = threadIdx.x; g < groups; g += 1024) {
      const int n = p.cols - 8 * g;
      const Loose8<T> v = fetch8<T, false, false>(x + 8 * g, active ? n : 0), gamma = fetch8<T, false, false>(reinterpret_cast<const T *>(p.gamma) + 8 * g, n);
      uint32_t lowest = ~0u, code = norm_out8<T>(p, v, gamma, rs, lowest, row, g, kp, active);
      if (__builtin_expect(active && !(lowest > norm_safe_row(norm_safe_above(gamma_top(gamma, p.shift, 1.f)), rs)), 0))
        code = norm_out8<T, true>(p, v, gamma, rs, lowest, row, g, kp, active);
      if ((threadIdx.x & 3) == 0)
        p.scales[((int64_t)(g >> 4) * cells + (row >> 2)) * 16 + ((g >> 2) & 3) * 4 + (row & 3)] = (uint8_t)code;
    }
    if (active && threadIdx.x == 0) p.rsigma[row] = (float)rs;
  }
}

template <typename T, bool WHOLE, bool RES> static void launch_norm_mx(const NormMxParams &p, hipStream_t st) {
  const int64_t rows4 = mx_rows4(p.rows);
  const bool nt = stream_hint(p.rows * p.cols * (int64_t)(sizeof(T) * (RES ? 3 : 1) + 1));
  auto grid = [&](int64_t per, int64_t most) { return dim3((unsigned)std::min(cdiv(rows4, per), most)); };
#define DH_NORM_MX(TPR, VPT, ROWS)                                                                                                                      \
  do {                                                                                                                                                \
    const dim3 g = grid(ROWS, 256 * 8);                                                                                                                 \
    if (nt) hipLaunchKernelGGL((norm_mx_kernel<T, TPR, VPT, ROWS, WHOLE, RES, true>), g, dim3(TPR * ROWS), 0, st, p);                                    \
    else hipLaunchKernelGGL((norm_mx_kernel<T, TPR, VPT, ROWS, WHOLE, RES, false>), g, dim3(TPR * ROWS), 0, st, p);                                      \
  } while (0)
  if (p.cols <= 512) DH_NORM_MX(64, 1, 4);
  else if (p.cols <= 1024) DH_NORM_MX(64, 2, 4);
  else if (p.cols <= 8192 && p.rows <= 256) DH_NORM_MX(1024, 1, 1);
  else if (p.cols <= 2048) DH_NORM_MX(256, 1, 1);
  else if (p.cols <= 4096) DH_NORM_MX(256, 2, 1);
  else if (p.cols <= 8192) DH_NORM_MX(256, 4, 1);
  else if (p.cols <= 16384) DH_NORM_MX(1024, 2, 1);
  else hipLaunchKernelGGL((norm_mx_long_kernel<T, RES>), grid(1, 256 * 16), dim3(1024), 0, st, p);
#undef DH_NORM_MX
}

}  // namespace dh

extern "C" int dh_mx_quantise(const void *x, int64_t rows, int64_t cols, int64_t ldx, int dtype, int format, int cover, void *codes, void *scales,
                              void *codes_t, void *scales_t, void *stream) {
  DH_CHECK(rows >= 0 && cols >= 0, "rows %lld, cols %lld", (long long)rows, (long long)cols);
  DH_CHECK(format == DH_MX_E4M3 || format == DH_MX_E2M1, "unknown format %d", format);
  DH_CHECK(dtype == DH_F32 || dtype == DH_BF16 || dtype == DH_F16, "unknown dtype %d", dtype);
  if (rows == 0 || cols == 0) return DH_OK;
  DH_CHECK(rows < (1ll << 31) && cols < (1ll << 31), "sizes of 2^31 and more: rows %lld, cols %lld", (long long)rows, (long long)cols);
  DH_CHECK(dh::cdiv(rows, 128) * dh::cdiv(cols, 128) < (1ll << 24), "more than 2^24 tiles of 128 x 128, which a launch of 256 threads each takes");
  DH_CHECK(x && (codes || codes_t), "null pointer");
  DH_CHECK(!codes == !scales && !codes_t == !scales_t, "codes and scales come in pairs");
  DH_CHECK(ldx >= cols || rows == 1, "row stride %lld of %lld columns", (long long)ldx, (long long)cols);
  DH_CHECK(dh::aligned16(codes) && dh::aligned16(scales) && dh::aligned16(codes_t) && dh::aligned16(scales_t), "codes and scales must be 16-byte aligned");
  const dh::QuantParams p{x, rows, cols, ldx, (uint8_t *)codes, (uint8_t *)scales, (uint8_t *)codes_t, (uint8_t *)scales_t, cover, (int)dh::cdiv(cols, 128)};
  DH_DISPATCH_DTYPE(dtype, if (format == DH_MX_E4M3) dh::launch_quantise<T, true>(p, (hipStream_t)stream);
                    else dh::launch_quantise<T, false>(p, (hipStream_t)stream));
  DH_LAUNCH_CHECK();
  return DH_OK;
}

extern "C" int dh_rmsnorm_mx(const void *x, const void *residual, void *sum_out, const void *gamma, void *y, void *codes, void *scales, float *rsigma,
                             int64_t rows, int64_t cols, float eps, int zero_centered_gamma, int cover, int dtype, void *stream) {
  DH_CHECK(rows >= 0 && cols >= 0, "rows %lld, cols %lld", (long long)rows, (long long)cols);
  DH_CHECK(dtype == DH_F32 || dtype == DH_BF16 || dtype == DH_F16, "unknown dtype %d", dtype);
  if (rows == 0 || cols == 0) return DH_OK;
  DH_CHECK(rows < (1ll << 31) && cols <= (1ll << 24), "sizes: rows %lld < 2^31, cols %lld <= 2^24", (long long)rows, (long long)cols);
  DH_CHECK(x && gamma && codes && scales && rsigma, "null pointer");
  DH_CHECK(!residual == !sum_out, "a residual and a place for the sum come together");
  DH_CHECK(dh::aligned16(codes) && dh::aligned16(scales), "codes and scales must be 16-byte aligned");
  const dh::NormMxParams p{x, residual, gamma, sum_out, y, (uint8_t *)codes, (uint8_t *)scales, rsigma, rows, (int)cols, cover, eps,
                           zero_centered_gamma ? 1.0f : 0.0f};
  const hipStream_t st = (hipStream_t)stream;
  DH_DISPATCH_DTYPE(dtype, if (cols % 8 == 0) { if (residual) dh::launch_norm_mx<T, true, true>(p, st); else dh::launch_norm_mx<T, true, false>(p, st); }
                    else { if (residual) dh::launch_norm_mx<T, false, true>(p, st); else dh::launch_norm_mx<T, false, false>(p, st); });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

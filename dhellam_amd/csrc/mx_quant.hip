// Quantisation to microscaled floating point, along the rows of a matrix, along its columns, or both in one pass over it, and the
// RMS norm (with the residual's addition) that writes its result in 8 bits with scales.  Format and rounding: mx.h.
#include <algorithm>

#include "mx.h"

namespace dh {

// ---- quantisation -------------------------------------------------------------------------------------------------------
// A workgroup takes 128 x 128 elements, a wavefront 32 rows of them, a lane 8 rows x 8 columns (row group lane / 16, column
// group lane % 16), so that each of its 8 loads brings 4 rows of 128 elements.  A block along a row lies in the 4 lanes of a
// quad, a block along a column in the lanes l, l ^ 16, l ^ 32, l ^ 48 (8 rows each): both maxima are a few exchanges between
// lanes, and no element goes through LDS before it is rounded.  What a lane holds of a column are 8 neighbouring elements
// of the transposed result: they are packed in registers and go through LDS as 8 (4) bytes, so that memory gets
// 128 (64) bytes of a row of the transpose at a time.
struct QuantParams {
  const void *x;
  int64_t rows, cols, ldx;
  uint8_t *codes, *scales, *codes_t, *scales_t;
  int cover;
  int tiles_c;
};

template <typename T, bool E4, bool ROWS, bool COLS>
__global__ void __launch_bounds__(256) mx_quantise_kernel(const QuantParams p) {
  constexpr int CB = E4 ? 8 : 4;                           // bytes of 8 codes
  __shared__ __attribute__((aligned(16))) uint8_t tile[COLS ? 128 * (16 * CB + 16) : 16];
  __shared__ __attribute__((aligned(16))) uint8_t sr[ROWS ? 512 : 16], sc[COLS ? 512 : 16];
  constexpr int TP = 16 * CB + 16;                         // bytes from one row of the tile to the next
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int rg = lane >> 4, cg = lane & 15;
  const int64_t tr = blockIdx.x / p.tiles_c, tc = blockIdx.x % p.tiles_c;
  const int64_t r0 = tr * 128, c0 = tc * 128;
  const int64_t row0 = r0 + 32 * w + 8 * rg, col0 = c0 + 8 * cg;
  const T *x = reinterpret_cast<const T *>(p.x);
  float v[8][8];
  const int64_t left = p.cols - col0;
  if (left >= 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row0 + i < p.rows) load8(v[i], x + (row0 + i) * p.ldx + col0);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = row0 + i < p.rows && left > 0;
      load8_first(v[i], in ? x + (row0 + i) * p.ldx + col0 : x, in ? (int)left : 0);
    }
  }
  if constexpr (ROWS) {
    const int64_t kp = (int64_t)p.tiles_c * 128;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) { const uint32_t m = magnitude(v[i][j]); top = top > m ? top : m; }
      const uint32_t code = mx_scale_code<E4>(quad_umax(top), p.cover);
      const MxPack<E4> o = mx_pack<E4>(v[i], code);
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
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) { const uint32_t m = magnitude(v[i][j]); top = top > m ? top : m; }
      uint32_t o1 = (uint32_t)__shfl_xor((int)top, 16, 64);
      top = top > o1 ? top : o1;
      o1 = (uint32_t)__shfl_xor((int)top, 32, 64);
      top = top > o1 ? top : o1;
      const uint32_t code = mx_scale_code<E4>(top, p.cover);
      float col[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) col[i] = v[i][j];
      const MxPack<E4> o = mx_pack<E4>(col, code);
      const int c = 8 * cg + j;
      uint8_t *dst = tile + c * TP + (4 * w + rg) * CB;
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
        *reinterpret_cast<dh_u32x4 *>(p.codes_t + (c0 + c) * ldt + tr * (16 * CB) + b * 16) = *reinterpret_cast<const dh_u32x4 *>(tile + c * TP + b * 16);
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
struct NormMxParams {
  const void *x, *residual, *gamma;
  void *sum_out, *y;
  uint8_t *codes, *scales;
  float *rsigma;
  int64_t rows;
  int cols, cover;
  float eps, shift;
};

template <typename T> __device__ __forceinline__ void store8(T *p, const float (&f)[8], int n) {
  if (n >= 8) {
    Loose8<T> o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = from_f<T>(f[j]);
    *reinterpret_cast<Loose8<T> *>(p) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = from_f<T>(f[j]);
  }
}

// x + residual of 8 columns, rounded to T as a separate addition stores it
template <typename T, bool RES>
__device__ __forceinline__ void norm_row8(float (&f)[8], const NormMxParams &p, int64_t at, int n) {
  const T *x = reinterpret_cast<const T *>(p.x) + at;
  if (n >= 8) load8(f, x);
  else load8_first(f, n > 0 ? x : reinterpret_cast<const T *>(p.x), n);
  if constexpr (RES) {
    if (n > 0) {
      float r[8];
      const T *q = reinterpret_cast<const T *>(p.residual) + at;
      if (n >= 8) load8(r, q);
      else load8_first(r, q, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = to_f(from_f<T>(f[j] + r[j]));
    }
  }
}

template <typename T, int BT, int TPR, int VPT, bool RES>
__global__ void __launch_bounds__(BT) norm_mx_kernel(const NormMxParams p) {
  constexpr int RPB = BT / TPR;
  __shared__ float red[BT / 64];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int groups = (p.cols + 127) / 128 * 16;
  const int64_t kp = (int64_t)groups * 8, cells = (p.rows + 3) / 4;
  const float inv_cols = 1.0f / (float)p.cols;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < 4 * cells; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + sub;
    const bool active = row < p.rows;
    float v[VPT][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = lane + i * TPR;
      const int n = active ? p.cols - 8 * g : 0;
      norm_row8<T, RES>(v[i], p, row * p.cols + 8 * g, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j] * v[i][j];
      if (RES && n > 0) store8(reinterpret_cast<T *>(p.sum_out) + row * p.cols + 8 * g, v[i], n);
    }
    s = TPR == 64 ? wave_sum(s) : block_sum<BT>(s, red);
    const float rs = 1.0f / sqrtf(s * inv_cols + p.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = lane + i * TPR;
      if (g >= groups || row >= 4 * cells) continue;       // (16 lanes at a time: groups is a multiple of 16)
      const int n = p.cols - 8 * g;
      float gm[8];
      const T *gamma = reinterpret_cast<const T *>(p.gamma) + 8 * g;
      if (n >= 8) load8(gm, gamma);
      else load8_first(gm, n > 0 ? gamma : reinterpret_cast<const T *>(p.gamma), n);
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = n > j && active ? v[i][j] * rs * (gm[j] + p.shift) : 0.f;
        const uint32_t m = magnitude(v[i][j]);
        top = top > m ? top : m;
      }
      if (p.y && active && n > 0) store8(reinterpret_cast<T *>(p.y) + row * p.cols + 8 * g, v[i], n);
      const uint32_t code = mx_scale_code<true>(quad_umax(top), p.cover);
      if (active) {
        const MxPack<true> o = mx_pack<true>(v[i], code);
        *reinterpret_cast<uint2 *>(p.codes + row * kp + 8 * g) = uint2{o.lo, o.hi};
      }
      if ((lane & 3) == 0)
        p.scales[((int64_t)(g >> 4) * cells + (row >> 2)) * 16 + ((g >> 2) & 3) * 4 + (row & 3)] = active ? (uint8_t)code : 0;
    }
    if (active && lane == 0) p.rsigma[row] = rs;
  }
}

// Rows of any length: one workgroup a row, read once for its statistics and again, from the cache, for its result.
template <typename T, bool RES>
__global__ void __launch_bounds__(1024) norm_mx_long_kernel(const NormMxParams p) {
  __shared__ float red[16];
  const int groups = (p.cols + 127) / 128 * 16;
  const int64_t kp = (int64_t)groups * 8, cells = (p.rows + 3) / 4;
  for (int64_t row = blockIdx.x; row < 4 * cells; row += gridDim.x) {
    const bool active = row < p.rows;
    float s = 0.f;
    for (int g = threadIdx.x; active && g < groups; g += 1024) {
      float v[8];
      const int n = p.cols - 8 * g;
      norm_row8<T, RES>(v, p, row * p.cols + 8 * g, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j] * v[j];
      if (RES && n > 0) store8(reinterpret_cast<T *>(p.sum_out) + row * p.cols + 8 * g, v, n);
    }
    s = block_sum<1024>(s, red);
    const float rs = 1.0f / sqrtf(s / (float)p.cols + p.eps);
    NormMxParams q = p;
    if (RES) q.x = p.sum_out;                              // a thread reads what it wrote itself
    for (int g = threadIdx.x; g < groups; g += 1024) {
      float v[8], gm[8];
      const int n = p.cols - 8 * g;
      norm_row8<T, false>(v, q, row * p.cols + 8 * g, active ? n : 0);
      const T *gamma = reinterpret_cast<const T *>(p.gamma) + 8 * g;
      if (n >= 8) load8(gm, gamma);
      else load8_first(gm, n > 0 ? gamma : reinterpret_cast<const T *>(p.gamma), n);
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = n > j && active ? v[j] * rs * (gm[j] + p.shift) : 0.f;
        const uint32_t m = magnitude(v[j]);
        top = top > m ? top : m;
      }
      if (p.y && active && n > 0) store8(reinterpret_cast<T *>(p.y) + row * p.cols + 8 * g, v, n);
      const uint32_t code = mx_scale_code<true>(quad_umax(top), p.cover);
      if (active) {
        const MxPack<true> o = mx_pack<true>(v, code);
        *reinterpret_cast<uint2 *>(p.codes + row * kp + 8 * g) = uint2{o.lo, o.hi};
      }
      if ((threadIdx.x & 3) == 0)
        p.scales[((int64_t)(g >> 4) * cells + (row >> 2)) * 16 + ((g >> 2) & 3) * 4 + (row & 3)] = active ? (uint8_t)code : 0;
    }
    if (active && threadIdx.x == 0) p.rsigma[row] = rs;
  }
}

template <typename T, bool RES> static void launch_norm_mx(const NormMxParams &p, hipStream_t st) {
  const int64_t rows4 = mx_rows4(p.rows);
  const int64_t most = 256 * 16;
  auto grid = [&](int64_t per) { return dim3((unsigned)std::min(cdiv(rows4, per), most)); };
#define DH_NORM_MX(BT, TPR, VPT) hipLaunchKernelGGL((norm_mx_kernel<T, BT, TPR, VPT, RES>), grid(BT / TPR), dim3(BT), 0, st, p)
  if (p.cols <= 512) DH_NORM_MX(256, 64, 1);
  else if (p.cols <= 1024) DH_NORM_MX(256, 64, 2);
  else if (p.cols <= 2048) DH_NORM_MX(256, 256, 1);
  else if (p.cols <= 4096) DH_NORM_MX(256, 256, 2);
  else if (p.cols <= 8192) DH_NORM_MX(256, 256, 4);
  else if (p.cols <= 16384) DH_NORM_MX(1024, 1024, 2);
  else hipLaunchKernelGGL((norm_mx_long_kernel<T, RES>), grid(1), dim3(1024), 0, st, p);
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
  DH_CHECK(dh::cdiv(rows, 128) * dh::cdiv(cols, 128) < (1ll << 31), "more than 2^31 tiles");
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
  DH_DISPATCH_DTYPE(dtype, if (residual) dh::launch_norm_mx<T, true>(p, (hipStream_t)stream);
                    else dh::launch_norm_mx<T, false>(p, (hipStream_t)stream));
  DH_LAUNCH_CHECK();
  return DH_OK;
}

// What a step does with its gradients before the optimiser: the norm of all of them together and their clipping, over lists of
// tensors of any number, size and type.
//
//   sum_sq = sum over all elements of g^2           norm = |scale| sqrt(sum_sq)
//   factor = scale min(1, max_norm / (norm + 1e-6)) out = factor g
//
// with the norm and the factor in 64 bits; a norm that fp32 cannot hold counts as not finite, and a factor that rounds to 0 in fp32 as 0.
// Both passes cut every tensor into pieces of 32768 elements, a workgroup each; a launch takes up to 80 tensors from a table in
// its arguments.  Squares are added in 64 bits (an fp32 square overflows from 1.8e19 on), a workgroup's sum is written to its own
// place and one workgroup adds these up in order: the result is the same bits every time.  Bound by memory: 16-byte loads at any alignment.
// 559 M elements in bf16 (1.12 GB) to fp32: norm 155 to 165 us (6.8 to 7.2 TB/s read), the join of 17073 sums 5, clipping 645 (5.2 TB/s read and written, a
// copy's rate).  Clipping in reverse order, for what the norm's pass left on the chip, gained nothing.
#include <cmath>

#include "mx.h"

namespace dh {

constexpr int GRAD_TABLE = 80;
constexpr int64_t GRAD_PIECE = 32768;

struct GradTable {
  const void *g[GRAD_TABLE];
  void *out[GRAD_TABLE];
  int64_t n[GRAD_TABLE];
  int first[GRAD_TABLE];             // the tensor's first workgroup in the launch
  uint8_t type[GRAD_TABLE], out_type[GRAD_TABLE];
  int count, blocks;
};

// The tensor that a workgroup belongs to.
__device__ __forceinline__ int grad_find(const GradTable &t, int block) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// N consecutive elements at any address that suits T, 16 bytes or 8; NT: without a place in the caches.
template <typename T, int N> struct alignas(sizeof(T)) Run { T v[N]; };
template <bool NT, typename T, int N> __device__ __forceinline__ Run<T, N> grad_load(const T *p) {
  Run<T, N> x;
  if constexpr (NT && sizeof(x) == 16) {
    const dh_u32x4 q = __builtin_nontemporal_load(reinterpret_cast<const typename LooseU4<T>::type *>(p));
    __builtin_memcpy(&x, &q, 16);
  } else {
    x = *reinterpret_cast<const Run<T, N> *>(p);
  }
  return x;
}

template <typename T, bool NT> __device__ __forceinline__ double grad_piece_sum(const T *g, int64_t n) {
  constexpr int N = 16 / (int)sizeof(T), STEP = 256 * N;
  double s[2] = {0.0, 0.0};
#pragma unroll 8
  for (int i = 0; i < (int)GRAD_PIECE / STEP; ++i) {
    const int64_t at = (int64_t)i * STEP + threadIdx.x * N;
    if (at + N <= n) {
      const Run<T, N> x = grad_load<NT, T, N>(g + at);
#pragma unroll
      for (int j = 0; j < N; ++j) s[j & 1] = fma((double)to_f(x.v[j]), (double)to_f(x.v[j]), s[j & 1]);
    } else {
      for (int64_t j = at; j < n; ++j) s[0] = fma((double)to_f(g[j]), (double)to_f(g[j]), s[0]);
    }
  }
  return s[0] + s[1];
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <bool NT> __global__ void __launch_bounds__(256) grad_norm_kernel(const GradTable t, double *partial) {
  __shared__ double red[4];
  const int i = grad_find(t, (int)blockIdx.x);
  const int64_t at = (int64_t)((int)blockIdx.x - t.first[i]) * GRAD_PIECE, n = t.n[i] - at;
  double s = 0.0;
  if (t.type[i] == DH_F32) s = grad_piece_sum<float, NT>(reinterpret_cast<const float *>(t.g[i]) + at, n);
  else if (t.type[i] == DH_BF16) s = grad_piece_sum<bf16_t, NT>(reinterpret_cast<const bf16_t *>(t.g[i]) + at, n);
  else s = grad_piece_sum<f16_t, NT>(reinterpret_cast<const f16_t *>(t.g[i]) + at, n);
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__global__ void __launch_bounds__(1024) grad_join_kernel(const double *partial, int64_t n, double *sum_sq) {
  __shared__ double red[16];
  double s = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i];
    sum_sq[0] = s;
  }
}

// (a lane stores 16 bytes, so that a wavefront's store is one run of memory: fp32 from 16 bits in pieces of 32 bytes a lane ran at 4.7 TB/s)
template <typename T, typename TO, bool NT> __device__ __forceinline__ void grad_piece_scale(const T *g, TO *out, int64_t n, float factor, float behind) {
  constexpr int N = 16 / (int)sizeof(TO), STEP = 256 * N;
#pragma unroll 8
  for (int i = 0; i < (int)GRAD_PIECE / STEP; ++i) {
    const int64_t at = (int64_t)i * STEP + threadIdx.x * N;
    if (at + N <= n) {
      const Run<T, N> x = grad_load<NT, T, N>(g + at);
      Run<TO, N> o;
#pragma unroll
      for (int j = 0; j < N; ++j) o.v[j] = factor == 0.f ? from_f<TO>(0.f) : from_f<TO>(to_f(x.v[j]) * factor * behind);
      if constexpr (NT) {
        dh_u32x4 q;
        __builtin_memcpy(&q, &o, 16);
        __builtin_nontemporal_store(q, reinterpret_cast<typename LooseU4<TO>::type *>(out + at));
      } else {
        *reinterpret_cast<Run<TO, N> *>(out + at) = o;
      }
    } else {
      for (int64_t j = at; j < n; ++j) out[j] = factor == 0.f ? from_f<TO>(0.f) : from_f<TO>(to_f(g[j]) * factor * behind);
    }
  }
}

template <bool NT> __global__ void __launch_bounds__(256) grad_clip_kernel(const GradTable t, const double *sum_sq, double max_norm, double scale, float *found) {
  const double norm = fabs(scale) * sqrt(sum_sq[0]);
  double factor = scale * fmin(1.0, max_norm / (norm + 1e-6));
  if (!((float)norm < INFINITY) || (float)factor == 0.f) factor = 0.0;
  if (found && blockIdx.x == 0 && threadIdx.x == 0) {
    found[0] = (float)norm;
    found[1] = (float)factor;
  }
  if (t.blocks == 0) return;
  // a factor below fp32's normal numbers in two steps, so that it keeps its 24 bits (the second is a power of two)
  const float behind = fabs(factor) < 0x1p-126 ? 0x1p-64f : 1.f, f = (float)(behind == 1.f ? factor : factor * 0x1p64);
  const int i = grad_find(t, (int)blockIdx.x);
  const int64_t at = (int64_t)((int)blockIdx.x - t.first[i]) * GRAD_PIECE, n = t.n[i] - at;
  if (f == 1.f && t.g[i] == t.out[i]) return;              // in place, nothing to change
#define GRAD_SCALE(T, TO) grad_piece_scale<T, TO, NT>(reinterpret_cast<const T *>(t.g[i]) + at, reinterpret_cast<TO *>(t.out[i]) + at, n, f, behind)
  if (t.type[i] == DH_F32) GRAD_SCALE(float, float);
  else if (t.type[i] == DH_BF16) {
    if (t.out_type[i] == DH_F32) GRAD_SCALE(bf16_t, float);
    else GRAD_SCALE(bf16_t, bf16_t);
  } else {
    if (t.out_type[i] == DH_F32) GRAD_SCALE(f16_t, float);
    else GRAD_SCALE(f16_t, f16_t);
  }
#undef GRAD_SCALE
}

// The whole list, before the first table is launched: a call that is refused has changed nothing.
static int grad_check(const void *const *g, void *const *out, const int64_t *counts, const int *types, const int *out_types, int n) {
  for (int i = 0; i < n; ++i) {
    DH_CHECK(counts[i] >= 0, "tensor %d: %lld elements", i, (long long)counts[i]);
    DH_CHECK(types[i] == DH_F32 || types[i] == DH_BF16 || types[i] == DH_F16, "tensor %d: unknown dtype %d", i, types[i]);
    DH_CHECK(!out || out_types[i] == types[i] || out_types[i] == DH_F32, "tensor %d: results are of its own type or fp32", i);
    DH_CHECK(counts[i] == 0 || (g[i] && (!out || out[i])), "tensor %d: null pointer", i);
    DH_CHECK(counts[i] < GRAD_PIECE << 23, "tensor %d is too large", i);
  }
  return DH_OK;
}

// Calls fn(table) for the lists in tables of up to GRAD_TABLE tensors that are not empty.
template <typename F>
static int grad_tables(const void *const *g, void *const *out, const int64_t *counts, const int *types, const int *out_types, int n, F &&fn) {
  for (int i = 0; i < n;) {
    GradTable t{};
    int64_t blocks = 0;
    for (; i < n && t.count < GRAD_TABLE; ++i) {
      if (counts[i] == 0) continue;
      const int64_t b = cdiv(counts[i], GRAD_PIECE);
      if (blocks + b >= (1ll << 24)) break;                 // (a launch holds fewer than 2^32 threads; one tensor has half of that at most)
      t.g[t.count] = g[i];
      t.out[t.count] = out ? out[i] : nullptr;
      t.n[t.count] = counts[i];
      t.type[t.count] = (uint8_t)types[i];
      t.out_type[t.count] = (uint8_t)(out ? out_types[i] : 0);
      t.first[t.count++] = (int)blocks;
      blocks += b;
    }
    t.blocks = (int)blocks;
    if (t.count > 0)
      if (const int rc = fn(t)) return rc;
  }
  return DH_OK;
}

}  // namespace dh

extern "C" size_t dh_grad_norm_workspace_bytes(const int64_t *counts, int n) {
  int64_t blocks = 0;
  for (int i = 0; i < n; ++i) blocks += counts[i] > 0 ? dh::cdiv(counts[i], dh::GRAD_PIECE) : 0;
  return (size_t)blocks * 8;
}

extern "C" int dh_grad_norm(const void *const *grads, const int64_t *counts, const int *dtypes, int n, double *sum_sq, void *workspace,
                            size_t workspace_bytes, void *stream) {
  using namespace dh;
  DH_CHECK(n >= 0 && (n == 0 || (grads && counts && dtypes)) && sum_sq, "bad list");
  if (const int rc = grad_check(grads, nullptr, counts, dtypes, nullptr, n)) return rc;
  const size_t need = dh_grad_norm_workspace_bytes(counts, n);
  DH_CHECK(need == 0 || (workspace && (uintptr_t)workspace % 8 == 0 && workspace_bytes >= need), "workspace of %zu bytes, %zu are needed", workspace_bytes,
           need);
  double *partial = reinterpret_cast<double *>(workspace);
  // gradients that the last-level cache holds stay there for the clipping: 215 MB in 16 bits to fp32 132 us (165 read past it), 1.1 GB 808 (835)
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += counts[i] * (int64_t)dtype_size(dtypes[i]);
  const bool nt = stream_hint(bytes);
  int64_t done = 0;
  const hipStream_t st = (hipStream_t)stream;
  const int rc = grad_tables(grads, nullptr, counts, dtypes, nullptr, n, [&](const GradTable &t) -> int {
    if (nt) hipLaunchKernelGGL((grad_norm_kernel<true>), dim3((unsigned)t.blocks), dim3(256), 0, st, t, partial + done);
    else hipLaunchKernelGGL((grad_norm_kernel<false>), dim3((unsigned)t.blocks), dim3(256), 0, st, t, partial + done);
    done += t.blocks;
    DH_LAUNCH_CHECK();
    return DH_OK;
  });
  if (rc) return rc;
  hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(1024), 0, st, partial, done, sum_sq);
  DH_LAUNCH_CHECK();
  return DH_OK;
}

extern "C" int dh_grad_clip(const void *const *grads, void *const *out, const int64_t *counts, const int *dtypes, const int *out_dtypes, int n,
                            const double *sum_sq, double max_norm, double scale, float *found, void *stream) {
  using namespace dh;
  DH_CHECK(n >= 0 && (n == 0 || (grads && out && counts && dtypes && out_dtypes)) && sum_sq && found, "bad list");
  DH_CHECK(max_norm >= 0, "max_norm %g", max_norm);
  DH_CHECK(std::isfinite((float)scale), "scale %g", scale);
  if (const int rc = grad_check(grads, out, counts, dtypes, out_dtypes, n)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  float *say = found;
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += counts[i] * (int64_t)(dtype_size(dtypes[i]) + dtype_size(out_dtypes[i]));
  const bool nt = stream_hint(bytes);
  const int rc = grad_tables(grads, out, counts, dtypes, out_dtypes, n, [&](const GradTable &t) -> int {
    if (nt) hipLaunchKernelGGL((grad_clip_kernel<true>), dim3((unsigned)t.blocks), dim3(256), 0, st, t, sum_sq, max_norm, scale, say);
    else hipLaunchKernelGGL((grad_clip_kernel<false>), dim3((unsigned)t.blocks), dim3(256), 0, st, t, sum_sq, max_norm, scale, say);
    say = nullptr;
    DH_LAUNCH_CHECK();
    return DH_OK;
  });
  if (rc) return rc;
  if (say) {
    hipLaunchKernelGGL((grad_clip_kernel<false>), dim3(1), dim3(64), 0, st, GradTable{}, sum_sq, max_norm, scale, say);
    DH_LAUNCH_CHECK();
  }
  return DH_OK;
}

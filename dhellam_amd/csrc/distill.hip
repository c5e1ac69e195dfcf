// Distillation from a teacher's top logits, mixed with the labels' cross entropy, over a (slice of a) vocabulary.
//
// A row has student logits x_c, K teacher entries (id_k, t_k), a temperature tau and a share alpha:
//   p_k = exp(t_k / tau - l),  l = log sum_k exp(t_k / tau), or the teacher's over its whole vocabulary when the caller has it
//   q = softmax(x / tau),  M = sum_k p_k
//   loss = alpha tau^2 sum_k p_k (log p_k - log q_k) + (1 - alpha) (log sum_c exp(x_c) - x_target)
//   d loss / d x_c = alpha tau (M q_c - sum_{k: id_k = c} p_k) + (1 - alpha) (softmax(x)_c - [c = target])
//
// Entries with an id outside the vocabulary do not exist (padding).  Bound by memory: the forward reads the row
// once with a running maximum and one or two sums of exponentials beside it, and K single logits; the backward reads it once more
// and writes the gradient.  The K listed columns (and the target's) are corrected behind the row's stores, so nothing
// per element depends on the column.
#include "common.h"

namespace dh {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int BT = 256, MAX_K = 1024, SLOTS = MAX_K / BT;      // threads of a row's workgroup; entries of a list; of a thread

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes aligned as single elements are: rows of any pitch and any start.
typedef uint32_t raw16 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> __device__ __forceinline__ Vec<T> load16(const T *p) {
  return __builtin_bit_cast(Vec<T>, *reinterpret_cast<const raw16 *>(p));
}
template <typename T> __device__ __forceinline__ void store16(T *p, const Vec<T> &x) {
  *reinterpret_cast<raw16 *>(p) = __builtin_bit_cast(raw16, x);
}

__device__ __forceinline__ float block_max(float v, float *red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

struct Teacher {
  const void *ids, *logits;
  const float *lse;
  const int64_t *target;
  int64_t vocab_start, vocab_total, cols;
  int k, wide_ids, dtype;
  float inv_tau, tau, alpha;

  __device__ __forceinline__ int64_t id(int64_t r, int j) const {
    const int64_t at = r * k + j;
    return wide_ids ? ((const int64_t *)ids)[at] : ((const int32_t *)ids)[at];
  }
  // t / tau
  __device__ __forceinline__ float logit(int64_t r, int j) const {
    const int64_t at = r * k + j;
    const float t = dtype == DH_F32 ? ((const float *)logits)[at]
                                    : dtype == DH_BF16 ? to_f(((const bf16_t *)logits)[at]) : to_f(((const f16_t *)logits)[at]);
    return t * inv_tau;
  }
  __device__ __forceinline__ bool there(int64_t id) const { return id >= 0 && id < vocab_total; }
  // the local column of an id, -1 on other ranks' slices
  __device__ __forceinline__ int64_t column(int64_t id) const {
    const int64_t c = id - vocab_start;
    return c >= 0 && c < cols ? c : -1;
  }
};

// The per-row statistics, `pitch` floats apart.
enum { LOSS, ROW_MAX, SUM_TAU, SUM_ONE, NORM, MASS, DOT, MASS_LOCAL, ENTROPY, PREDICTED, N_STATS };

// Running maximum and sums of exponentials against it: s at the temperature, s1 at one (TWO).
template <bool TWO> struct Running {
  float m = -INFINITY, s = 0.f, s1 = 0.f;
  __device__ __forceinline__ void move(float to, float k) {
    s *= exp2_fast((m - to) * k);
    if (TWO) s1 *= exp2_fast((m - to) * LOG2E);
    m = to;
  }
  template <int N> __device__ __forceinline__ void add(const float *x, float k) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > m) move(top, k);                      // m = -inf: 0 * exp2(-inf) = 0
    if (m == -INFINITY && top == -INFINITY) return;      // nothing but -inf so far
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // (x - m) first: the difference of two close numbers is exact
      s += exp2_fast((x[i] - m) * k);
      if (TWO) s1 += exp2_fast((x[i] - m) * LOG2E);
    }
  }
  // brought to a maximum that others share
  __device__ __forceinline__ void align(float to, float k) {
    if (m > -INFINITY) move(to, k);
  }
};

template <bool TWO, typename T>
__device__ __forceinline__ void scan_row(const T *row, int64_t from, int64_t to, float k, Running<TWO> &run) {
  constexpr int N = Vec<T>::N, U = 4;                // vectors in flight
  const int64_t nvec = (to - from) / N;
  const T *base = row + from;
  int64_t v = threadIdx.x;
  for (; v + (U - 1) * BT < nvec; v += U * BT) {
    Vec<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load16(base + (v + u * BT) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = to_f(x[u].v[e]);
      run.template add<N>(f, k);
    }
  }
  for (; v < nvec; v += BT) {
    const Vec<T> x = load16(base + v * N);
    float f[N];
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = to_f(x.v[e]);
    run.template add<N>(f, k);
  }
  for (int64_t c = nvec * N + threadIdx.x; c < to - from; c += BT) {
    const float f = to_f(base[c]);
    run.template add<1>(&f, k);
  }
}

// The row's statistics from its maximum and sums, by a whole workgroup.
template <typename T>
__device__ __forceinline__ void finish_row(const Teacher &t, const T *row, int64_t r, float m, float s, float s1, float *stats,
                                           int64_t pitch, float *red) {
  float a[SLOTS], x[SLOTS];                          // t / tau, the student's logit (local entries)
  bool local[SLOTS];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = i * BT + (int)threadIdx.x;
    a[i] = -INFINITY;
    x[i] = 0.f;
    local[i] = false;
    if (j < t.k) {
      const int64_t id = t.id(r, j);
      if (t.there(id)) {
        a[i] = t.logit(r, j);
        const int64_t c = t.column(id);
        local[i] = c >= 0;
        if (local[i]) x[i] = to_f(row[c]);
      }
    }
    top = fmaxf(top, a[i]);
  }
  float norm;
  if (t.lse) {
    norm = t.lse[r];
  } else {
    top = block_max(top, red);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (a[i] != -INFINITY) sum += expf(a[i] - top);
    sum = block_sum<BT>(sum, red);
    norm = sum != 0.f ? top + logf(sum) : 0.f;       // no entries: no mass either
  }
  float mass = 0.f, mine = 0.f, dot = 0.f, ent = 0.f;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
    if (a[i] != -INFINITY) {
      const float p = expf(a[i] - norm);
      if (p != 0.f) {
        mass += p;
        ent += p * (a[i] - norm);
        if (local[i]) {
          mine += p;
          dot += p * ((x[i] - m) * t.inv_tau);
        }
      }
    }
  mass = block_sum<BT>(mass, red);
  mine = block_sum<BT>(mine, red);
  dot = block_sum<BT>(dot, red);
  ent = block_sum<BT>(ent, red);
  if (threadIdx.x == 0) {
    float loss = 0.f, pred = 0.f;
    if (mass != 0.f && t.alpha > 0.f) loss = t.alpha * t.tau * t.tau * (ent - dot + mass * logf(s));
    if (t.target) {
      const int64_t c = t.column(t.target[r]);
      if (c >= 0) pred = to_f(row[c]) - m;
      loss += (1.f - t.alpha) * (logf(s1) - pred);
    }
    float *o = stats + r;
    o[LOSS * pitch] = loss;
    o[ROW_MAX * pitch] = m;
    o[SUM_TAU * pitch] = s;
    o[SUM_ONE * pitch] = s1;
    o[NORM * pitch] = norm;
    o[MASS * pitch] = mass;
    o[DOT * pitch] = dot;
    o[MASS_LOCAL * pitch] = mine;
    o[ENTROPY * pitch] = ent;
    o[PREDICTED * pitch] = pred;
  }
}

// One workgroup a row, or a segment of one (partial sums in `parts`: [rows][segments][3]).
template <typename T, bool TWO>
__global__ void __launch_bounds__(BT)
distill_fwd_kernel(const T *__restrict__ logits, int64_t ld, int64_t segment, Teacher t, float *__restrict__ stats, int64_t pitch,
                   float *__restrict__ parts) {
  __shared__ float red[4];
  const int64_t r = blockIdx.x;
  const T *row = logits + r * ld;
  const float k = t.inv_tau * LOG2E;
  const int64_t from = (int64_t)blockIdx.y * segment, to = from + segment < t.cols ? from + segment : t.cols;
  Running<TWO> run;
  scan_row<TWO>(row, from, to, k, run);
  const float m = block_max(run.m, red);
  run.align(m, k);
  const float s = block_sum<BT>(run.s, red), s1 = TWO ? block_sum<BT>(run.s1, red) : s;
  if (parts) {
    if (threadIdx.x == 0) {
      float *o = parts + (r * gridDim.y + blockIdx.y) * 3;
      o[0] = m;
      o[1] = s;
      o[2] = s1;
    }
    return;
  }
  finish_row(t, row, r, m, s, s1, stats, pitch, red);
}

// The segments of a row, joined, and the row's statistics.
template <typename T>
__global__ void __launch_bounds__(BT)
distill_join_kernel(const T *__restrict__ logits, int64_t ld, int segments, Teacher t, float *__restrict__ stats, int64_t pitch,
                    const float *__restrict__ parts) {
  __shared__ float red[4];
  const int64_t r = blockIdx.x;
  const float k = t.inv_tau * LOG2E, *p = parts + r * segments * 3;
  Running<true> run;
  for (int i = threadIdx.x; i < segments; i += BT) {
    const float m = p[3 * i], to = fmaxf(m, run.m);
    float s = p[3 * i + 1], s1 = p[3 * i + 2];
    if (m > -INFINITY) {
      s *= exp2_fast((m - to) * k);
      s1 *= exp2_fast((m - to) * LOG2E);
    }
    run.align(to, k);
    run.m = to;
    run.s += s;
    run.s1 += s1;
  }
  const float m = block_max(run.m, red);
  run.align(m, k);
  const float s = block_sum<BT>(run.s, red), s1 = block_sum<BT>(run.s1, red);
  finish_row(t, logits + r * ld, r, m, s, s1, stats, pitch, red);
}

// One workgroup a segment of a row.  grad may be the logits (each element is read, then written, by the same thread; the listed
// ones are read before any store of the row).
template <typename T, bool TWO>
__global__ void __launch_bounds__(BT)
distill_bwd_kernel(const T *logits, int64_t ld, int64_t segment, Teacher t, const float *__restrict__ stats, int64_t pitch,
                   const float *__restrict__ dout, T *grad, int64_t ld_grad) {
  constexpr int N = Vec<T>::N, U = 4, HOLD = SLOTS + 1;      // + 1: the target
  __shared__ int32_t cols_of[MAX_K + 4];                     // columns of the segment, -1 elsewhere
  __shared__ float weight[MAX_K + 4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t from = (int64_t)blockIdx.y * segment, to = from + segment < t.cols ? from + segment : t.cols;
  const T *row = logits + r * ld + from;
  T *out = grad + r * ld_grad + from;
  const float *st = stats + r;
  const float m = st[ROW_MAX * pitch], mass = st[MASS * pitch], norm = st[NORM * pitch], d = dout[r];
  const float k = t.inv_tau * LOG2E;
  const float scale = mass != 0.f ? t.alpha * t.tau * d : 0.f;
  const float ks = scale != 0.f ? scale * mass / st[SUM_TAU * pitch] : 0.f;
  const float hard = t.target ? (1.f - t.alpha) * d : 0.f;
  const float k1 = hard != 0.f ? hard / st[SUM_ONE * pitch] : 0.f;
  const int64_t len = to - from, nvec = len / N;
  if (d == 0.f || (scale == 0.f && hard == 0.f)) {           // a row that is left out: zeros, whatever it holds
    Vec<T> zero;
#pragma unroll
    for (int e = 0; e < N; ++e) zero.v[e] = from_f<T>(0.f);
    for (int64_t v = tid; v < nvec; v += BT) store16(out + v * N, zero);
    for (int64_t c = nvec * N + tid; c < len; c += BT) out[c] = from_f<T>(0.f);
    return;
  }
  auto value = [&](float x) {
    if (TWO) return fmaf(exp2_fast((x - m) * k), ks, exp2_fast((x - m) * LOG2E) * k1);
    return exp2_fast((x - m) * k) * (ks + k1);
  };
  // the entries that lie in this segment: weight and value without them, from the logits before they are overwritten
  const int entries = t.k + (t.target ? 1 : 0);
  float base[HOLD];
#pragma unroll
  for (int i = 0; i < HOLD; ++i) {
    const int j = i * BT + tid;
    base[i] = 0.f;
    if (j < entries) {
      int64_t c = -1;
      float w = 0.f;
      if (j == t.k) {
        c = t.column(t.target[r]);
        w = hard;
      } else {
        const int64_t id = t.id(r, j);
        if (t.there(id)) {
          c = t.column(id);
          const float a = t.logit(r, j);
          w = a != -INFINITY ? scale * expf(a - norm) : 0.f;
        }
      }
      if (c < from || c >= to) c = -1;
      else base[i] = value(to_f(row[c - from]));
      cols_of[j] = c < 0 ? -1 : (int32_t)(c - from);
      weight[j] = w;
    }
  }
  if (tid < 4 && entries + tid < MAX_K + 4) cols_of[entries + tid] = -1;
  __syncthreads();
  int64_t v = tid;
  auto emit = [&](int64_t at, const Vec<T> &x) {
    Vec<T> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = from_f<T>(value(to_f(x.v[e])));
    store16(out + at * N, o);
  };
  for (; v + (U - 1) * BT < nvec; v += U * BT) {
    Vec<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load16(row + (v + u * BT) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) emit(v + u * BT, x[u]);
  }
  for (; v < nvec; v += BT) emit(v, load16(row + v * N));
  for (int64_t c = nvec * N + tid; c < len; c += BT) out[c] = from_f<T>(value(to_f(row[c])));
  __syncthreads();                                           // the segment's stores are complete
  // the first entry of a column takes off the weights of all that name it, in the list's order
#pragma unroll
  for (int i = 0; i < HOLD; ++i) {
    const int j = i * BT + tid;
    const int c = j < entries ? cols_of[j] : -1;
    if (c >= 0) {
      bool first = true;
      float w = 0.f;
      for (int o = 0; o < entries; ++o)
        if (cols_of[o] == c) {
          first &= o >= j;
          w += weight[o];
        }
      if (first) out[c] = from_f<T>(base[i] - w);
    }
  }
}

// Segments of a row: one where the rows alone fill the chip; then pieces of at least 4096 columns until they do.
int64_t segments_of(int64_t rows, int64_t cols, int64_t least, int64_t want) {
  int64_t n = cdiv(want, rows);
  const int64_t most = cdiv(cols, least);
  if (n > most) n = most;
  return n < 1 ? 1 : n > 65535 ? 65535 : n;
}
int64_t fwd_segments(int64_t rows, int64_t cols) { return rows >= 1024 ? 1 : segments_of(rows, cols, 4096, 2048); }
// a segment's length, whole 16-byte pieces of any type
int64_t segment_of(int64_t cols, int64_t segments) { return cdiv(cdiv(cols, segments), 8) * 8; }

}  // namespace
}  // namespace dh

using namespace dh;

static int distill_check(const void *logits, int64_t ld, const void *ids, int id_bytes, const void *teacher, int teacher_dtype,
                         int64_t rows, int64_t cols, int k, int64_t vocab_start, int64_t vocab_total, const int64_t *target,
                         float temperature, float alpha, int dtype, const float *stats, int64_t pitch) {
  DH_CHECK(rows >= 0 && cols > 0 && ld >= cols && rows < (1ll << 24) && cols < (1ll << 30), "rows=%lld cols=%lld ld=%lld",
           (long long)rows, (long long)cols, (long long)ld);
  DH_CHECK(k >= 1 && k <= MAX_K, "%d teacher entries a row: 1 to %d", k, MAX_K);
  DH_CHECK(id_bytes == 4 || id_bytes == 8, "ids of %d bytes", id_bytes);
  DH_CHECK(teacher_dtype == DH_F32 || teacher_dtype == DH_BF16 || teacher_dtype == DH_F16, "unknown teacher dtype %d", teacher_dtype);
  DH_CHECK(dtype == DH_F32 || dtype == DH_BF16 || dtype == DH_F16, "unknown dtype %d", dtype);
  DH_CHECK(vocab_start >= 0 && vocab_total >= vocab_start + cols, "columns %lld to %lld of a vocabulary of %lld", (long long)vocab_start,
           (long long)(vocab_start + cols), (long long)vocab_total);
  DH_CHECK(temperature >= 1e-6f && temperature <= 1e6f, "temperature %g outside [1e-6, 1e6]", temperature);
  DH_CHECK(alpha >= 0.f && alpha <= 1.f, "alpha %g outside [0, 1]", alpha);
  DH_CHECK(alpha == 1.f || target || rows == 0, "alpha %g without targets", alpha);
  DH_CHECK(rows == 0 || (logits && ids && teacher && stats), "null pointer");
  DH_CHECK(pitch >= rows, "pitch=%lld < rows", (long long)pitch);
  return DH_OK;
}

extern "C" size_t dh_distill_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t n = fwd_segments(rows, cols);
  return n > 1 ? (size_t)(rows * n * 3 * (int64_t)sizeof(float)) : 0;
}

extern "C" int dh_distill_fwd(const void *logits, int64_t ld, const void *ids, int id_bytes, const void *teacher, int teacher_dtype,
                              const float *teacher_lse, const int64_t *target, int64_t rows, int64_t cols, int k, int64_t vocab_start,
                              int64_t vocab_total, float temperature, float alpha, int dtype, float *stats, int64_t pitch,
                              void *workspace, size_t workspace_bytes, void *stream) {
  if (const int rc = distill_check(logits, ld, ids, id_bytes, teacher, teacher_dtype, rows, cols, k, vocab_start, vocab_total, target,
                                   temperature, alpha, dtype, stats, pitch))
    return rc;
  if (rows == 0) return DH_OK;
  const size_t need = dh_distill_workspace_bytes(rows, cols);
  DH_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  const Teacher t{ids, teacher, teacher_lse, alpha < 1.f ? target : nullptr, vocab_start, vocab_total, cols, k, id_bytes == 8,
                  teacher_dtype, 1.f / temperature, temperature, alpha};
  const int64_t segment = segment_of(cols, fwd_segments(rows, cols)), n = cdiv(cols, segment);
  const bool two = alpha < 1.f && temperature != 1.f;
  float *parts = need ? (float *)workspace : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  DH_DISPATCH_DTYPE(dtype, {
    const auto kernel = two ? distill_fwd_kernel<T, true> : distill_fwd_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows, (unsigned)n), dim3(BT), 0, st, (const T *)logits, ld, segment, t, stats, pitch,
                       parts);
    if (parts)
      hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)rows), dim3(BT), 0, st, (const T *)logits, ld, (int)n, t, stats,
                         pitch, (const float *)parts);
  });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

extern "C" int dh_distill_bwd(const void *logits, int64_t ld, const void *ids, int id_bytes, const void *teacher, int teacher_dtype,
                              const int64_t *target, const float *stats, int64_t pitch, const float *dout, int64_t rows, int64_t cols,
                              int k, int64_t vocab_start, int64_t vocab_total, float temperature, float alpha, int dtype, void *grad,
                              int64_t ld_grad, void *stream) {
  if (const int rc = distill_check(logits, ld, ids, id_bytes, teacher, teacher_dtype, rows, cols, k, vocab_start, vocab_total, target,
                                   temperature, alpha, dtype, stats, pitch))
    return rc;
  if (rows == 0) return DH_OK;
  DH_CHECK(dout && grad && ld_grad >= cols, "dout or grad null, or ld_grad=%lld < cols", (long long)ld_grad);
  {
    const char *a = (const char *)logits, *b = (const char *)grad;
    const int64_t e = (int64_t)dtype_size(dtype);
    DH_CHECK((a == b && ld_grad == ld) || a + ((rows - 1) * ld + cols) * e <= b || b + ((rows - 1) * ld_grad + cols) * e <= a,
             "grad is either the logits (same pitch) or does not overlap them");
  }
  const Teacher t{ids, teacher, nullptr, alpha < 1.f ? target : nullptr, vocab_start, vocab_total, cols, k, id_bytes == 8,
                  teacher_dtype, 1.f / temperature, temperature, alpha};
  const int64_t want = segments_of(rows, cols, 2048, 2048), whole = cdiv(cols, 16384);
  const int64_t segment = segment_of(cols, want > whole ? want : whole), n = cdiv(cols, segment);
  DH_CHECK(n <= 65535, "too many columns");
  const bool two = alpha < 1.f && temperature != 1.f;
  const hipStream_t st = (hipStream_t)stream;
  DH_DISPATCH_DTYPE(dtype, {
    const auto kernel = two ? distill_bwd_kernel<T, true> : distill_bwd_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows, (unsigned)n), dim3(BT), 0, st, (const T *)logits, ld, segment, t, stats, pitch, dout,
                       (T *)grad, ld_grad);
  });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

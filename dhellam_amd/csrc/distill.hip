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
//
// 4096 x 128256 in bf16, K = 128, alpha 0.5, tau 1: forward 163 us (6.4 TB/s), backward 356 us (5.9 TB/s); a copy on this card 5.9 TB/s.
#include "common.h"

namespace dh {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_K = 1024;                // entries of a list
constexpr float LOWEST = -3.402823466e38f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes aligned as single elements are: rows of any pitch and any start.
typedef uint32_t raw16 __attribute__((ext_vector_type(4), aligned(2)));
template <bool NT, typename T> __device__ __forceinline__ Vec<T> load16(const T *p) {
  const raw16 *q = reinterpret_cast<const raw16 *>(p);
  return __builtin_bit_cast(Vec<T>, NT ? __builtin_nontemporal_load(q) : *q);
}
template <bool NT, typename T> __device__ __forceinline__ void store16(T *p, const Vec<T> &x) {
  const raw16 v = __builtin_bit_cast(raw16, x);
  if (NT) __builtin_nontemporal_store(v, reinterpret_cast<raw16 *>(p));
  else *reinterpret_cast<raw16 *>(p) = v;
}

// How the exponential at temperature one comes from that at tau, e: it is the same (tau 1, or no targets), e^2 (tau 2), e^4 (tau 4), or
// needs one of its own.  An exponential is four of the fifteen issue slots that an element takes with two of them, which is
// more than its two bytes take to arrive: forward of 4096 x 16032 in bf16 at tau 2, alpha 0.5, 32.4 us with two, 29.8 squared.
enum Hard { SAME, SQUARE, FOURTH, OWN };
Hard hard_of(float temperature, float alpha) {
  if (alpha == 1.f || temperature == 1.f) return SAME;
  return temperature == 2.f ? SQUARE : temperature == 4.f ? FOURTH : OWN;
}
template <Hard H> __device__ __forceinline__ float exp_one(float e, float y) {      // y = x - reference
  if (H == SAME) return e;
  if (H == SQUARE) return e * e;
  if (H == FOURTH) return (e * e) * (e * e);
  return exp2_fast(y * LOG2E);
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

// Sums of exponentials, s at the temperature and s1 at one, against a reference m that is moved only when a value
// passes it by 2^16: the sums are then as exact as against the maximum (a float's precision does not depend on its scale), and a
// wavefront hardly ever branches once it has seen its first values.  The lowest float to begin with, for the reference and for the
// maximum: -inf adds nothing to it, a row of lowest floats is a row of equal ones, and x - m is a number for every x, also where a
// rank's slice holds nothing but -inf.
template <Hard H> struct Running {
  float m = LOWEST, top = LOWEST, s = 0.f, s1 = 0.f;
  __device__ __forceinline__ void move(float to, float k) {
    s *= exp2_fast((m - to) * k);
    if (H != SAME) s1 *= exp2_fast((m - to) * LOG2E);
    m = to;
  }
  template <int N> __device__ __forceinline__ void add(const float *x, float k, float slack) {
    float t = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) t = fmaxf(t, x[i]);
    top = fmaxf(top, t);
    if (t > m + slack) move(t, k);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // (x - m) first: the difference of two close numbers is exact
      const float y = x[i] - m;
      const float e = exp2_fast(y * k);
      s += e;
      if (H != SAME) s1 += exp_one<H>(e, y);
    }
  }
};

template <bool NT, int BT, Hard H, typename T>
__device__ __forceinline__ void scan_row(const T *row, int64_t from, int64_t to, float k, Running<H> &run) {
  constexpr int N = Vec<T>::N, U = 2;                // vectors in flight: 4096 x 16032 in bf16, not in any cache, 29.8 us, with 4 32.3, with 8 38.6
  const float slack = 16.f / fmaxf(k, LOG2E);        // 2^16 at either temperature
  const int nvec = (int)((to - from) / N);
  const T *base = row + from;
  for (int v = threadIdx.x; v < nvec; v += U * BT) {
    Vec<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * BT < nvec) x[u] = load16<NT>(base + (int64_t)(v + u * BT) * N);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * BT < nvec) {
        float f[N];
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = to_f(x[u].v[e]);
        run.template add<N>(f, k, slack);
      }
  }
  for (int64_t c = (int64_t)nvec * N + threadIdx.x; c < to - from; c += BT) {
    const float f = to_f(base[c]);
    run.template add<1>(&f, k, slack);
  }
}

// A row's teacher entries, by one wavefront, 256 at a time: what is read is asked for before the row is scanned.
struct Entries {
  static constexpr int U = 4;
  float a[U], x[U];                                  // t / tau (-inf: none), the student's logit
  uint32_t local;                                    // bit i: entry i lies in this slice
  template <typename T> __device__ __forceinline__ void load(const Teacher &t, const T *row, int64_t r, int first) {
    int64_t id[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = first + i * 64 + (int)(threadIdx.x & 63);
      id[i] = -1;
      a[i] = -INFINITY;
      if (j < t.k) {
        id[i] = t.id(r, j);
        a[i] = t.logit(r, j);
      }
    }
    local = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      x[i] = 0.f;
      if (!t.there(id[i])) {
        a[i] = -INFINITY;
        continue;
      }
      const int64_t c = t.column(id[i]);
      if (c >= 0) {
        x[i] = to_f(row[c]);
        local |= 1u << i;
      }
    }
  }
};

// The sums over a row's entries in one pass: weights exp(a - ref) against a running reference, logits against `m`, the row's maximum, or
// (FIND) against the largest logit of an entry that has a weight, which m then is.
struct Sums {
  float norm, mass, dot, mine, ent;
  template <bool FIND, typename T>
  __device__ __forceinline__ void run(const Teacher &t, const T *row, int64_t r, float &m, Entries &e) {
    float ref = -INFINITY, w0 = 0.f, wa = 0.f, wx = 0.f, wl = 0.f;
    for (int first = 0;;) {
      float top = fmaxf(fmaxf(e.a[0], e.a[1]), fmaxf(e.a[2], e.a[3]));
      top = fmaxf(wave_max(top), ref);
      if (ref > -INFINITY) {
        const float f = expf(ref - top);
        wa = (wa + (ref - top) * w0) * f;
        w0 *= f, wx *= f, wl *= f;
      }
      ref = top;
      if (FIND) {
        float to = m;
#pragma unroll
        for (int i = 0; i < Entries::U; ++i)
          if (e.a[i] != -INFINITY && (e.local >> i & 1)) to = fmaxf(to, e.x[i]);
        to = wave_max(to);
        if (wl != 0.f) wx += wl * ((m - to) * t.inv_tau);
        m = to;
      }
#pragma unroll
      for (int i = 0; i < Entries::U; ++i)
        if (e.a[i] != -INFINITY) {
          const float y = e.a[i] - ref, w = expf(y);
          if (w != 0.f) {
            w0 += w;
            wa += w * y;
            if (e.local >> i & 1) {
              wl += w;
              wx += w * ((e.x[i] - m) * t.inv_tau);
            }
          }
        }
      first += Entries::U * 64;
      if (first >= t.k) break;
      e.load(t, row, r, first);
    }
    w0 = wave_sum(w0), wa = wave_sum(wa), wx = wave_sum(wx), wl = wave_sum(wl);
    norm = mass = dot = mine = ent = 0.f;
    if (w0 == 0.f) return;                           // no entries
    norm = t.lse ? t.lse[r] : ref + logf(w0);
    const float scale = t.lse ? expf(ref - norm) : 1.f / w0;
    mass = t.lse ? w0 * scale : 1.f;
    dot = wx * scale;
    mine = t.lse || wl != w0 ? wl * scale : 1.f;
    ent = wa * scale + (ref - norm) * mass;
  }
};

__device__ __forceinline__ void write_stats(const Teacher &t, float *stats, int64_t pitch, float m, float s, float s1, const Sums &e,
                                            float pred) {
  float loss = 0.f;
  if (e.mass != 0.f && t.alpha > 0.f) loss = t.alpha * t.tau * t.tau * (e.ent - e.dot + e.mass * logf(s));
  if (t.target) loss += (1.f - t.alpha) * (logf(s1) - pred);
  stats[LOSS * pitch] = loss;
  stats[ROW_MAX * pitch] = m;
  stats[SUM_TAU * pitch] = s;
  stats[SUM_ONE * pitch] = s1;
  stats[NORM * pitch] = e.norm;
  stats[MASS * pitch] = e.mass;
  stats[DOT * pitch] = e.dot;
  stats[MASS_LOCAL * pitch] = e.mine;
  stats[ENTROPY * pitch] = e.ent;
  stats[PREDICTED * pitch] = pred;
}

// What a row's segments leave for the join: three floats each, and the first one's sums over the entries, with dot against a reference of
// the entries' own, for the first segment's maximum may be any low value.
enum { PART_NORM, PART_MASS, PART_DOT, PART_MINE, PART_ENT, PART_REF, PART_TARGET, PART_SUMS };

// One workgroup a row, or a segment of one.
template <typename T, Hard H, bool NT, int BT>
__global__ void __launch_bounds__(BT)
distill_fwd_kernel(const T *__restrict__ logits, int64_t ld, int64_t segment, int segments, Teacher t, float *__restrict__ stats,
                   int64_t pitch, float *__restrict__ parts) {
  __shared__ float red[BT / 64][3];
  const int64_t r = blockIdx.x / (unsigned)segments;
  const int y = blockIdx.x % (unsigned)segments, w = threadIdx.x >> 6;
  const T *row = logits + r * ld;
  const float k = t.inv_tau * LOG2E;
  const int64_t from = (int64_t)y * segment, to = from + segment < t.cols ? from + segment : t.cols;
  Entries e;
  float xt = 0.f;
  bool has_target = false;
  if (y == 0 && w == 0) {
    e.load(t, row, r, 0);
    if (t.target) {
      const int64_t c = t.column(t.target[r]);
      has_target = c >= 0;
      if (has_target) xt = to_f(row[c]);
    }
  }
  Running<H> run;
  scan_row<NT, BT>(row, from, to, k, run);
  float m = wave_max(run.top);
  run.move(m, k);
  float s = wave_sum(run.s), s1 = H != SAME ? wave_sum(run.s1) : s;
  if ((threadIdx.x & 63) == 0) {
    red[w][0] = m;
    red[w][1] = s;
    red[w][2] = s1;
  }
  __syncthreads();
  if (w != 0) return;
  m = red[0][0];
#pragma unroll
  for (int i = 1; i < BT / 64; ++i) m = fmaxf(m, red[i][0]);
  s = s1 = 0.f;
#pragma unroll
  for (int i = 0; i < BT / 64; ++i) {
    const float d = red[i][0] - m;
    s += red[i][1] * exp2_fast(d * k);               // (a wavefront of -inf only adds nothing)
    if (H != SAME) s1 += red[i][2] * exp2_fast(d * LOG2E);
  }
  if (H == SAME) s1 = s;
  float *o = parts ? parts + (r * segments + y) * 3 : nullptr;
  if (parts && threadIdx.x == 0) {
    o[0] = m;
    o[1] = s;
    o[2] = s1;
  }
  if (y != 0) return;
  Sums sums;
  if (!parts) {
    sums.run<false>(t, row, r, m, e);
    if (threadIdx.x == 0) write_stats(t, stats + r, pitch, m, s, s1, sums, has_target ? xt - m : 0.f);
    return;
  }
  float ref = LOWEST;
  sums.run<true>(t, row, r, ref, e);
  if (threadIdx.x == 0) {
    o = parts + (int64_t)gridDim.x * 3 + r * PART_SUMS;
    o[PART_NORM] = sums.norm;
    o[PART_MASS] = sums.mass;
    o[PART_DOT] = sums.dot;
    o[PART_MINE] = sums.mine;
    o[PART_ENT] = sums.ent;
    o[PART_REF] = ref;
    o[PART_TARGET] = xt;
  }
}

// The segments of a row, joined by one wavefront.
__global__ void __launch_bounds__(64)
distill_join_kernel(int segments, Teacher t, float *__restrict__ stats, int64_t pitch, const float *__restrict__ parts) {
  const int64_t r = blockIdx.x;
  const float k = t.inv_tau * LOG2E, *p = parts + r * segments * 3, *e = parts + (int64_t)gridDim.x * segments * 3 + r * PART_SUMS;
  float top = LOWEST;
  for (int i = threadIdx.x; i < segments; i += 64) top = fmaxf(top, p[3 * i]);
  const float m = wave_max(top);
  float s = 0.f, s1 = 0.f;
  for (int i = threadIdx.x; i < segments; i += 64) {
    const float d = p[3 * i] - m;
    s += p[3 * i + 1] * exp2_fast(d * k);
    s1 += p[3 * i + 2] * exp2_fast(d * LOG2E);
  }
  s = wave_sum(s), s1 = wave_sum(s1);
  if (threadIdx.x != 0) return;
  Sums sums;
  sums.norm = e[PART_NORM], sums.mass = e[PART_MASS], sums.mine = e[PART_MINE], sums.ent = e[PART_ENT];
  sums.dot = sums.mine != 0.f ? e[PART_DOT] + sums.mine * ((e[PART_REF] - m) * t.inv_tau) : 0.f;
  write_stats(t, stats + r, pitch, m, s, s1, sums, t.target && t.column(t.target[r]) >= 0 ? e[PART_TARGET] - m : 0.f);
}

// One workgroup a segment of a row.  Its wavefronts look up the listed columns that lie in the segment, 64 each, then all stream the
// segment, and behind its stores the listed columns are corrected.  grad may be the logits: the listed ones are read before any store.
// A segment is short, four vectors a thread, so that the workgroups of a moment read and write neighbouring memory, at the price of
// looking at a row's list once a segment.  us by KB a segment, inputs in no cache, before the wait below: 4096 x 128256 in bf16, 129 columns a row, 8 406, 12 354,
// 16 353 (6.0 TB/s, what a copy reaches), 24 382, 32 404, 128 431; 4096 x 16032, 65 columns, 8 52, 16 55, 32 59, but with the forward in
// front 8 87, 16 84, 32 87; 1000 x 50257 in fp32 8 70, 16 77, 32 83 (99.5, 101.7, 104.3).
constexpr int64_t BWD_BYTES = 16384;
template <typename T, Hard H, bool NT, int BT>
__global__ void __launch_bounds__(BT)
distill_bwd_kernel(const T *logits, int64_t ld, int64_t segment, int segments, Teacher t, const float *__restrict__ stats,
                   int64_t pitch, const float *__restrict__ dout, T *grad, int64_t ld_grad) {
  constexpr int N = Vec<T>::N, U = 4;                        // vectors in flight
  __shared__ __align__(16) int32_t cols_of[MAX_K];           // columns in the segment, -1 elsewhere
  __shared__ __align__(16) float weight[MAX_K];              // what is taken off them
  __shared__ uint32_t named[BWD_BYTES / 2 / 32];             // a bit a column: listed
  __shared__ int twice;                                      // a column is listed twice
  const int64_t r = blockIdx.x / (unsigned)segments;
  const int tid = threadIdx.x;
  const int64_t from = (int64_t)(blockIdx.x % (unsigned)segments) * segment, to = from + segment < t.cols ? from + segment : t.cols;
  const T *row = logits + r * ld + from;
  T *out = grad + r * ld_grad + from;
  const float *st = stats + r;
  const float m = st[ROW_MAX * pitch], mass = st[MASS * pitch], norm = st[NORM * pitch], d = dout[r];
  const float k = t.inv_tau * LOG2E;
  const float scale = mass != 0.f ? t.alpha * t.tau * d : 0.f;
  const float hard = t.target ? (1.f - t.alpha) * d : 0.f;
  const int len = (int)(to - from), nvec = len / N;
  if (d == 0.f || (scale == 0.f && hard == 0.f)) {           // a row that is left out: zeros, whatever it holds
    Vec<T> zero;
#pragma unroll
    for (int e = 0; e < N; ++e) zero.v[e] = from_f<T>(0.f);
    for (int v = tid; v < nvec; v += BT) store16<NT>(out + (int64_t)v * N, zero);
    for (int c = nvec * N + tid; c < len; c += BT) out[c] = from_f<T>(0.f);
    return;
  }
  const float ks = scale != 0.f ? scale * mass / st[SUM_TAU * pitch] : 0.f;
  const float k1 = hard != 0.f ? hard / st[SUM_ONE * pitch] : 0.f;
  auto value = [&](float x) {
    const float e = exp2_fast((x - m) * k);
    if (H == SAME) return e * (ks + k1);
    return fmaf(e, ks, exp_one<H>(e, x - m) * k1);
  };
#pragma unroll
  for (int i = 0; i < BWD_BYTES / 2 / 32; i += BT) named[i + tid] = 0;
  if (tid == 0) twice = 0;
  __syncthreads();
  constexpr int SLOTS = 4;                                   // entries of a thread: lists of up to 4 BT
  float base[SLOTS];                                         // of the thread's entries: the value without what is taken off
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = i * BT + tid;
    base[i] = 0.f;
    if (i * BT < t.k && j < ((t.k + 3) & ~3)) {
      int64_t c = -1;
      float w = 0.f;
      if (j < t.k) {
        const int64_t id = t.id(r, j);
        const float a = t.logit(r, j);
        if (t.there(id)) c = id - t.vocab_start - from;
        w = a != -INFINITY ? scale * expf(a - norm) : 0.f;
      }
      if (c < 0 || c >= len) {
        c = -1;
      } else {
        base[i] = value(to_f(row[c]));
        const uint32_t bit = 1u << (c & 31);
        if (atomicOr(&named[c >> 5], bit) & bit) twice = 1;
      }
      cols_of[j] = (int32_t)c;
      weight[j] = w;
    }
  }
  int target = -1;                                           // the label's column
  float at_target = 0.f;
  if (t.target) {
    const int64_t c = t.target[r] - t.vocab_start - from;
    if (c >= 0 && c < len) {
      target = (int)c;
      at_target = value(to_f(row[c]));
    }
  }
  if (logits == grad) {                                      // every listed value has arrived before any wavefront writes
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  for (int v = tid; v < nvec; v += U * BT) {
    Vec<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * BT < nvec) x[u] = load16<false>(row + (int64_t)(v + u * BT) * N);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * BT < nvec) {
        Vec<T> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = from_f<T>(value(to_f(x[u].v[e])));
        store16<NT>(out + (int64_t)(v + u * BT) * N, o);
      }
  }
  for (int c = nvec * N + tid; c < len; c += BT) out[c] = from_f<T>(value(to_f(row[c])));
  // the segment's stores are complete, the lists too.  (Both barriers of global memory wait for it themselves: __syncthreads() compiles to a wait for
  // LDS alone, and neither two stores nor a read and a store of one address are to depend on the order that the memory keeps.  Backward, us,
  // without this wait / with it: 4096 x 128256 in bf16 352 / 356, 4096 x 16032 53.8 / 54.6.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  // the label's weight goes with the entry of its column, or alone
  if (tid == 0 && target >= 0 && !(named[target >> 5] >> (target & 31) & 1)) out[target] = from_f<T>(at_target - hard);
  // no column twice, as a rule; else the first entry of a column takes off the weights of all that name it, in the list's order.  (Without the
  // bits, every entry looking for others of its column, 2000 x 4001 with 256 entries a row took 70 us, so 12.)
  const bool once = twice == 0;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    if (i * BT >= t.k) break;
    const int j = i * BT + tid;
    const int c = j < t.k ? cols_of[j] : -1;
    if (c < 0) continue;
    bool first = true;
    float off = once ? weight[j] : 0.f;
    for (int o = 0; !once && o < t.k; o += 4) {
      const int4 cc = *reinterpret_cast<const int4 *>(cols_of + o);
      const float4 ww = *reinterpret_cast<const float4 *>(weight + o);
      off += cc.x == c ? ww.x : 0.f;
      off += cc.y == c ? ww.y : 0.f;
      off += cc.z == c ? ww.z : 0.f;
      off += cc.w == c ? ww.w : 0.f;
      first &= !((cc.x == c && o < j) || (cc.y == c && o + 1 < j) || (cc.z == c && o + 2 < j) || (cc.w == c && o + 3 < j));
    }
    if (first) out[c] = from_f<T>(base[i] - (c == target ? off + hard : off));
  }
}

template <typename T, Hard H> auto fwd_kernel(int threads, bool nt) {
  return threads == 64     ? distill_fwd_kernel<T, H, false, 64>
         : threads == 1024 ? (nt ? distill_fwd_kernel<T, H, true, 1024> : distill_fwd_kernel<T, H, false, 1024>)
                           : (nt ? distill_fwd_kernel<T, H, true, 256> : distill_fwd_kernel<T, H, false, 256>);
}
template <typename T, Hard H> auto bwd_kernel(int threads, bool nt) {
  return threads == 64 ? distill_bwd_kernel<T, H, false, 64> : nt ? distill_bwd_kernel<T, H, true, 256> : distill_bwd_kernel<T, H, false, 256>;
}
#define DISTILL_PICK(pick, hard, threads, nt)                                                       \
  (hard == SAME ? pick<T, SAME>(threads, nt) : hard == SQUARE ? pick<T, SQUARE>(threads, nt)        \
   : hard == FOURTH ? pick<T, FOURTH>(threads, nt) : pick<T, OWN>(threads, nt))

// Segments of a row: at least `least` columns, no more of them than make `want` workgroups of all rows.
int64_t segments_of(int64_t rows, int64_t cols, int64_t least, int64_t want) {
  int64_t n = cdiv(want, rows);
  const int64_t most = cdiv(cols, least);
  if (n > most) n = most;
  return n < 1 ? 1 : n;
}
// a segment's length, whole cache lines of any type (4096 x 128256 backward, when it was 398 us: -10)
int64_t segment_of(int64_t cols, int64_t segments) { return cdiv(cdiv(cols, segments), 64) * 64; }
// The forward's: one, but for few rows of very many columns, where joining them costs a launch.  us, one workgroup of 1024 threads a row / segments
// of 4096, bf16: 16 rows of 50257 7.5 / 8.3, of 70000 8.1 / 7.9, of 128256 11.4 / 7.8, of 262144 19.3 / 8.1; 64 rows of 70000 8.1 / 8.4, of 128256
// 11.4 / 9.7, of 262144 20.1 / 11.7; 99 rows 8.1 / 9.1, 12.2 / 10.5, 20.8 / 15.9; 128 rows 8.1 / 10.7, 12.3 / 11.9, 20.1 / 18.8; 200 rows 8.5 / 11.6,
// 12.8 / 15.9, 23.1 / 23.6
int64_t fwd_segment(int64_t rows, int64_t cols) { return segment_of(cols, rows < 100 && cols > 65536 ? segments_of(rows, cols, 4096, 2048) : 1); }
// Threads of a row's workgroup in the forward.  A wavefront where rows are short, for four of them mostly wait for each other: us, 256 threads / 64,
// bf16: 2000 x 1000 5.8 / 5.2, 8000 x 1000 14.4 / 8.7, 8000 x 2000 17.2 / 11.2, 8000 x 4001 21.5 / 16.9, but 2000 x 4001 7.3 / 7.9, 512 x 8008 5.3 / 7.3.
// 1024 where there are no more rows than stand on the chip at once, or long ones: us, 256 / 1024: bf16, 64 x 10000 5.2 / 5.0, 128 x 32000 9.0 / 6.4, 512 x 50257
// 17.7 / 13.1, 700 x 128256 44.5 / 36.6, 4096 x 128256 167 / 161, but 700 x 16032 8.6 / 9.9, 3000 x 50257 67 / 73; fp32, 3000 x 50257 99 / 94.
int fwd_threads(int64_t rows, int64_t cols, int64_t bytes) {
  if (cols <= 2048 || (cols <= 4096 && rows >= 4096)) return 64;
  return (rows <= 512 && cols > 8192) || bytes >= 192 << 10 ? 1024 : 256;
}

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
  const int64_t n = cdiv(cols, fwd_segment(rows, cols));
  return n > 1 ? (size_t)(rows * (n * 3 + PART_SUMS) * (int64_t)sizeof(float)) : 0;
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
  const int64_t segment = fwd_segment(rows, cols), n = cdiv(cols, segment);
  float *parts = need ? (float *)workspace : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  DH_DISPATCH_DTYPE(dtype, {
    // rows that do not fit in the last-level cache do not go through it: 4096 x 128256 in bf16 183 -> 163 us; 1000 x 50257 in fp32 with the
    // hint 38.0 -> 35.4, but the backward then finds nothing of it (102 -> 113 both)
    const int threads = n > 1 ? 256 : fwd_threads(rows, cols, cols * (int64_t)sizeof(T));
    const auto kernel = DISTILL_PICK(fwd_kernel, hard_of(temperature, alpha), threads, threads > 64 && stream_hint(rows * cols * (int64_t)sizeof(T)));
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * n)), dim3(threads), 0, st, (const T *)logits, ld, segment, (int)n, t, stats, pitch, parts);
  });
  if (parts)
    hipLaunchKernelGGL(distill_join_kernel, dim3((unsigned)rows), dim3(64), 0, st, (int)n, t, stats, pitch, (const float *)parts);
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
  const int64_t want = segments_of(rows, cols, 2048, 2048), whole = cdiv(cols * (int64_t)dtype_size(dtype), BWD_BYTES);
  const int64_t segment = segment_of(cols, want > whole ? want : whole), n = cdiv(cols, segment);
  DH_CHECK(rows * n < 1ll << 24, "rows=%lld of cols=%lld: too many for one call", (long long)rows, (long long)cols);
  const hipStream_t st = (hipStream_t)stream;
  DH_DISPATCH_DTYPE(dtype, {
    // the gradient's stores go past the caches where that and the logits are more than a part of the last one.  us, forward, backward and a
    // reader of the gradient behind them, in the caches / past them, 16032 columns in bf16: 1024 rows 36.4 / 38.7, 2048 64.0 / 63.2, 4096
    // 107.6 / 106.7 (90.2 / 83.8 without the reader), 8192 220 / 208; 1000 x 50257 in fp32 154 / 140
    const bool nt = 2 * rows * cols * (int64_t)sizeof(T) > 96ll << 20;
    // a wavefront for short rows as in the forward: 2000 x 1000 6.1 / 4.8 us, 8000 x 1000 17.0 / 11.5, 8000 x 2000 19.6 / 16.0, 8000 x 4001 29.0 /
    // 29.1; it holds lists of up to 256
    const int threads = cols <= 2048 && k <= 256 ? 64 : 256;
    const auto kernel = DISTILL_PICK(bwd_kernel, hard_of(temperature, alpha), threads, nt && threads == 256);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * n)), dim3(threads), 0, st, (const T *)logits, ld, segment, (int)n, t, stats, pitch, dout,
                       (T *)grad, ld_grad);
  });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

// The router's training side: losses that keep the experts in balance, counts, and the gradient of the logits.
//
//   p_t = softmax(logits_t),  lse_t = log sum exp(logits_t),  N = tokens that count
//   counts_e = choices of expert e,  P_e = sum_t p_te           (over the tokens that count)
//   balance = a E / (k N^2) sum_e counts_e P_e,   z = b / N sum_t lse_t^2
//   d balance / d logit_te = a E / (k N^2) p_te (counts_e - sum_f counts_f p_tf),   d z / d logit_te = 2 b / N lse_t p_te
//   and through the gates, g = softmax of the chosen logits:  d logit of choice j = g_j (dg_j - sum_i g_i dg_i)
//
// A token's row of up to 64 logits is held by L lanes of 4 each: 16-byte loads, exchanges over L lanes only.  Sums over tokens
// stay in registers, then LDS, then one partial sum a workgroup (one of 1024 threads a compute unit) that a second launch adds in order: no
// atomics on floats, the same result every time.
//
// 131072 tokens x 64 experts, k 8: losses 14.1 us (38 MB; 3 of them the second launch), gradient 15.5 us (80 MB, 5.2 TB/s).  Small calls are
// launches: 64 tokens x 8 experts 3.9 and 2.9 us.
#include "common.h"

namespace dh {
namespace {

constexpr int BAL_MAX_E = 64, BAL_MAX_K = 8, BAL_BT = 1024, BAL_MAX_BLOCKS = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct BalancePartial {
  float prob[BAL_MAX_E];
  int32_t counts[BAL_MAX_E];
  float z;
  int32_t n;
};

// The four logits of a lane, -inf past the last expert.
__device__ __forceinline__ void load_row(const float *logits, int64_t t, int e0, int E, bool vec, float x[4]) {
  const float *row = logits + t * E;
  if (vec) {
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (e0 < E) v = *reinterpret_cast<const float4 *>(row + e0);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = e0 + i < E ? row[e0 + i] : -INFINITY;
  }
}

// Reductions over L neighbouring lanes, without LDS: exchanges with the neighbour, the other pair, the mirror image in 8 and in 16.
template <int CTRL> __device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int L> __device__ __forceinline__ float lanes_max(float v) {
  if (L >= 2) v = fmaxf(v, moved<0xB1>(v));
  if (L >= 4) v = fmaxf(v, moved<0x4E>(v));
  if (L >= 8) v = fmaxf(v, moved<0x141>(v));
  if (L >= 16) v = fmaxf(v, moved<0x140>(v));
  return v;
}
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
  if (L >= 2) v += moved<0xB1>(v);
  if (L >= 4) v += moved<0x4E>(v);
  if (L >= 8) v += moved<0x141>(v);
  if (L >= 16) v += moved<0x140>(v);
  return v;
}

// Totals in LDS -> the outputs, by the first wavefront.
__device__ __forceinline__ void balance_finish(const float *prob, const int *counts, float z, int n, int E, int K, float a, float b,
                                               float *losses, int32_t *counts_out, float *prob_out, int32_t *tokens_out) {
  const int e = threadIdx.x;
  if (e >= 64) return;
  const float p = e < E ? prob[e] : 0.f;
  const int c = e < E ? counts[e] : 0;
  const float inv = n > 0 ? 1.f / (float)n : 0.f;
  const float s = wave_sum(n > 0 ? ((float)c * inv) * (p * inv) : 0.f);
  if (e < E) {
    counts_out[e] = c;
    prob_out[e] = p;
  }
  if (e == 0) {
    losses[0] = a * (float)E / (float)K * s;
    losses[1] = n > 0 ? b * z * inv : 0.f;
    tokens_out[0] = n;
  }
}

template <int L, int BT>
__global__ void __launch_bounds__(BT)
balance_fwd_kernel(const float *__restrict__ logits, const int32_t *__restrict__ idx, const uint8_t *__restrict__ mask, int64_t tokens,
                   int E, int K, float a, float b, float *__restrict__ lse_out, BalancePartial *__restrict__ partials,
                   float *__restrict__ losses, int32_t *__restrict__ counts_out, float *__restrict__ prob_out,
                   int32_t *__restrict__ tokens_out, bool vec) {
  constexpr int WAVES = BT / 64, TPB = BT / L;
  __shared__ int cnt[WAVES][BAL_MAX_E];
  __shared__ float prob[WAVES][BAL_MAX_E];
  __shared__ float red_z[WAVES];
  __shared__ int red_n[WAVES];
  const int tid = threadIdx.x, w = tid >> 6, l = tid % L, e0 = 4 * l;
  cnt[w][tid & 63] = 0;
  prob[w][tid & 63] = 0.f;
  __syncthreads();
  // sums of a lane: of up to 64 terms, then those of these, so that none has more than 64 + tokens / 2^20 additions behind one another
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, z = 0.f, far[4] = {0.f, 0.f, 0.f, 0.f}, far_z = 0.f;
  int n = 0, terms = 0;
  constexpr int S = (BAL_MAX_K + L - 1) / L;        // choices of a token that a lane counts
  for (int64_t t0 = (int64_t)blockIdx.x * TPB; t0 < tokens; t0 += (int64_t)gridDim.x * TPB) {
    const int64_t t = t0 + tid / L;
    const bool in = t < tokens;
    bool on = in;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    int e[S];
#pragma unroll
    for (int s = 0; s < S; ++s) e[s] = in && l + s * L < K ? idx[t * K + l + s * L] : -1;
    if (in) {
      load_row(logits, t, e0, E, vec, x);
      if (mask) on = mask[t] != 0;
    }
    const float m = lanes_max<L>(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    float ex[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ex[i] = __builtin_amdgcn_exp2f((x[i] - m) * LOG2E);
    const float sum = lanes_sum<L>((ex[0] + ex[1]) + (ex[2] + ex[3]));
    const float lse = m + __builtin_amdgcn_logf(sum) * LN2, inv = __builtin_amdgcn_rcpf(sum);
    if (in && l == 0) lse_out[t] = lse;
    if (on) {                                       // (a masked row may hold anything)
#pragma unroll
      for (int s = 0; s < S; ++s)
        if ((unsigned)e[s] < (unsigned)E) atomicAdd(&cnt[w][e[s]], 1);      // (whole numbers: any order)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += ex[i] * inv;
      if (l == 0) {
        z += lse * lse;
        n += 1;
      }
    }
    if (++terms == 64) {
#pragma unroll
      for (int i = 0; i < 4; ++i) far[i] += acc[i], acc[i] = 0.f;
      far_z += z;
      z = 0.f;
      terms = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] += far[i];
  z += far_z;
#pragma unroll
  for (int o = 32; o >= L; o >>= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
  z = wave_sum(z);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((tid & 63) < L)
#pragma unroll
    for (int i = 0; i < 4; ++i) prob[w][e0 + i] = acc[i];
  if ((tid & 63) == 0) {
    red_z[w] = z;
    red_n[w] = n;
  }
  __syncthreads();
  if (tid < 64) {
    float p = 0.f;
    int c = 0;
    z = 0.f;
    n = 0;
    for (int i = 0; i < WAVES; ++i) {
      p += prob[i][tid];
      c += cnt[i][tid];
      z += red_z[i];
      n += red_n[i];
    }
    if (partials) {
      BalancePartial &out = partials[blockIdx.x];
      out.prob[tid] = p;
      out.counts[tid] = c;
      if (tid == 0) {
        out.z = z;
        out.n = n;
      }
    } else {
      prob[0][tid] = p;
      cnt[0][tid] = c;
      __builtin_amdgcn_wave_barrier();
      balance_finish(prob[0], cnt[0], z, n, E, K, a, b, losses, counts_out, prob_out, tokens_out);
    }
  }
}

// The workgroups' sums, added in their order: 16 wavefronts take every 16th, a lane an expert.
__global__ void __launch_bounds__(1024)
balance_join_kernel(const BalancePartial *__restrict__ partials, int blocks, int E, int K, float a, float b, float *__restrict__ losses,
                    int32_t *__restrict__ counts_out, float *__restrict__ prob_out, int32_t *__restrict__ tokens_out) {
  __shared__ float prob[16][64];
  __shared__ int cnt[16][64];
  __shared__ float red_z[16];
  __shared__ int red_n[16];
  constexpr int U = BAL_MAX_BLOCKS / 16;
  const int e = threadIdx.x & 63, w = threadIdx.x >> 6;
  float p = 0.f, z = 0.f, pp[U];
  int c = 0, n = 0, cc[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {                     // all asked for before any is added
    pp[i] = 0.f;
    cc[i] = 0;
    if (w + 16 * i < blocks) {
      pp[i] = partials[w + 16 * i].prob[e];
      cc[i] = partials[w + 16 * i].counts[e];
    }
  }
  if (e < U && w + 16 * e < blocks) {
    z = partials[w + 16 * e].z;
    n = partials[w + 16 * e].n;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    p += pp[i];
    c += cc[i];
  }
  z = wave_sum(z);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  prob[w][e] = p;
  cnt[w][e] = c;
  if (e == 0) {
    red_z[w] = z;
    red_n[w] = n;
  }
  __syncthreads();
  if (w == 0) {
    p = 0.f, z = 0.f;
    c = 0, n = 0;
    for (int i = 0; i < 16; ++i) {
      p += prob[i][e];
      c += cnt[i][e];
      z += red_z[i];
      n += red_n[i];
    }
    prob[0][e] = p;
    cnt[0][e] = c;
    __builtin_amdgcn_wave_barrier();
    balance_finish(prob[0], cnt[0], z, n, E, K, a, b, losses, counts_out, prob_out, tokens_out);
  }
}

// What a wavefront writes to LDS before this, its lanes read behind it (they access it in order; the compiler is to keep that).
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int L>
__global__ void __launch_bounds__(256)
route_bwd_kernel(const float *__restrict__ logits, const int32_t *__restrict__ idx, const float *__restrict__ gates,
                 const float *__restrict__ dgates, const uint8_t *__restrict__ mask, const float *__restrict__ lse,
                 const int32_t *__restrict__ counts, const int32_t *__restrict__ n_tokens, const float *__restrict__ dlosses,
                 int64_t tokens, int E, int K, float a, float b, float *__restrict__ dlogits, bool vec) {
  constexpr int TPB = 256 / L, S = (BAL_MAX_K + L - 1) / L;       // choices a lane holds
  __shared__ __align__(16) float tile[L >= 8 ? TPB : 1][4 * L];    // a token's gradient through its gates; all zero between tokens
  __shared__ int32_t marks[L >= 8 ? TPB : 1][4 * L];
  const int tid = threadIdx.x, l = tid % L, e0 = 4 * l, first = (tid & 63) - l;
  if constexpr (L >= 8) {
    *reinterpret_cast<float4 *>(&tile[tid / L][e0]) = make_float4(0.f, 0.f, 0.f, 0.f);
    wave_order();                                   // (a token's lanes are of one wavefront)
  }
  float ca = 0.f, cb = 0.f, c[4] = {0.f, 0.f, 0.f, 0.f};
  if (lse) {
    const int n = n_tokens[0];
    const float inv = n > 0 ? 1.f / (float)n : 0.f;
    ca = a * (float)E / (float)K * inv * (dlosses ? dlosses[0] : 1.f);
    cb = 2.f * b * inv * (dlosses ? dlosses[1] : 1.f);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e0 + i < E) c[i] = (float)counts[e0 + i] * inv;
  }
  for (int64_t t0 = (int64_t)blockIdx.x * TPB; t0 < tokens; t0 += (int64_t)gridDim.x * TPB) {
    const int64_t t = t0 + tid / L;
    const bool in = t < tokens;
    bool on = in;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, d[4] = {0.f, 0.f, 0.f, 0.f}, z = 0.f, g[S], v[S];
    int e[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int j = l + s * L;
      e[s] = -1;
      g[s] = v[s] = 0.f;
      if (dgates && in && j < K) {
        e[s] = idx[t * K + j];
        g[s] = gates[t * K + j];
        v[s] = dgates[t * K + j];
      }
    }
    if (lse) {
      if (in) {
        load_row(logits, t, e0, E, vec, x);
        z = lse[t];
        if (mask) on = mask[t] != 0;
      }
      // the log-sum-exp is one rounded float, off by up to 2^-24 of itself: it serves as the reference, and the row's own sum
      // (one but for that) makes probabilities of the exponentials, whatever the size of the logits
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f((x[i] - z) * LOG2E);
      const float inv = __builtin_amdgcn_rcpf(lanes_sum<L>((p[0] + p[1]) + (p[2] + p[3])));
      const float mean = lanes_sum<L>((c[0] * p[0] + c[1] * p[1]) + (c[2] * p[2] + c[3] * p[3])) * inv;
      if (on)                                       // (a masked row may hold anything)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = p[i] * inv * (ca * (c[i] - mean) + cb * z);
    }
    if (dgates) {
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) sum += g[s] * v[s];
      sum = lanes_sum<L>(sum);
#pragma unroll
      for (int s = 0; s < S; ++s) v[s] = g[s] * (v[s] - sum);
      bool spread = false;
      if constexpr (L >= 8) {
        // a choice a lane: through a row of LDS, where no expert is chosen twice (each lane finds its own mark there); 131072 tokens x 64
        // experts, k 8, by exchanges and four comparisons a choice 17.6 us, so 15.7 (both before the probabilities had a sum of their own)
        const bool chose = (unsigned)e[0] < (unsigned)E;
        float *to = tile[tid / L];
        int32_t *mark = marks[tid / L];
        if (chose) {
          to[e[0]] = v[0];
          mark[e[0]] = l;
        }
        wave_order();
        spread = !__any(chose && mark[e[0]] != l);
        if (spread) {
          const float4 got = *reinterpret_cast<const float4 *>(to + e0);
          d[0] += got.x, d[1] += got.y, d[2] += got.z, d[3] += got.w;
        }
        wave_order();
        if (chose) to[e[0]] = 0.f;
        wave_order();
      }
#pragma unroll
      for (int j = 0; j < BAL_MAX_K; ++j)
        if (!spread && j < K) {                     // choice j, to the lane that holds its expert
          const int to = __shfl(e[j / L], first + j % L, 64) - e0;
          const float val = __shfl(v[j / L], first + j % L, 64);
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] += to == i ? val : 0.f;
        }
    }
    if (in) {
      float *row = dlogits + t * E;
      if (vec) {
        if (e0 < E) *reinterpret_cast<float4 *>(row + e0) = make_float4(d[0], d[1], d[2], d[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e0 + i < E) row[e0 + i] = d[i];
      }
    }
  }
}

int lanes_of(int E) { return E <= 4 ? 1 : E <= 8 ? 2 : E <= 16 ? 4 : E <= 32 ? 8 : 16; }

// One workgroup, one launch, for up to four rounds of it: us with it / in two launches, 2048 tokens x 8 experts 5.8 / 6.5; beyond it grows by the
// round, two launches stay at 7 to 16384 tokens.
bool balance_one(int64_t tokens, int E) { return tokens * lanes_of(E) <= 4 * BAL_BT; }

#define BAL_LANES(E, ...)                                  \
  switch (lanes_of(E)) {                                   \
    case 1: { constexpr int L = 1; __VA_ARGS__; } break;   \
    case 2: { constexpr int L = 2; __VA_ARGS__; } break;   \
    case 4: { constexpr int L = 4; __VA_ARGS__; } break;   \
    case 8: { constexpr int L = 8; __VA_ARGS__; } break;   \
    default: { constexpr int L = 16; __VA_ARGS__; }        \
  }

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" size_t dh_balance_loss_workspace_bytes(int64_t tokens, int experts) {
  if (tokens <= 0 || experts < 1 || experts > BAL_MAX_E || balance_one(tokens, experts)) return 0;
  return BAL_MAX_BLOCKS * sizeof(BalancePartial);
}

extern "C" int dh_balance_loss_fwd(const float *logits, const int32_t *topk_idx, const uint8_t *mask, int64_t tokens, int experts,
                                   int k, float balance_coef, float z_coef, float *losses, int32_t *counts, float *prob_sum,
                                   int32_t *n_tokens, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  DH_CHECK(tokens >= 0 && tokens < (1ll << 31) / BAL_MAX_K, "tokens=%lld", (long long)tokens);
  DH_CHECK(experts >= 1 && experts <= BAL_MAX_E, "experts=%d must be in [1, %d]", experts, BAL_MAX_E);
  DH_CHECK(k >= 1 && k <= BAL_MAX_K && k <= experts, "k=%d must be in [1, min(%d, experts)]", k, BAL_MAX_K);
  DH_CHECK(losses && counts && prob_sum && n_tokens && (tokens == 0 || (logits && topk_idx && lse)), "null pointer");
  const size_t need = dh_balance_loss_workspace_bytes(tokens, experts);
  DH_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  const bool vec = experts % 4 == 0 && aligned16(logits);
  const hipStream_t st = (hipStream_t)stream;
  BAL_LANES(experts, {
    if (need == 0) {
      hipLaunchKernelGGL((balance_fwd_kernel<L, BAL_BT>), dim3(1), dim3(BAL_BT), 0, st, logits, topk_idx, mask, tokens, experts,
                         k, balance_coef, z_coef, lse, nullptr, losses, counts, prob_sum, n_tokens, vec);
    } else {
      int64_t blocks = cdiv(tokens * L, BAL_BT);
      if (blocks > BAL_MAX_BLOCKS) blocks = BAL_MAX_BLOCKS;
      hipLaunchKernelGGL((balance_fwd_kernel<L, BAL_BT>), dim3((unsigned)blocks), dim3(BAL_BT), 0, st, logits, topk_idx, mask, tokens, experts,
                         k, balance_coef, z_coef, lse, (BalancePartial *)workspace, losses, counts, prob_sum, n_tokens, vec);
      hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(1024), 0, st, (const BalancePartial *)workspace, (int)blocks, experts, k,
                         balance_coef, z_coef, losses, counts, prob_sum, n_tokens);
    }
  });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

extern "C" int dh_moe_route_bwd(const float *logits, const int32_t *topk_idx, const float *gates, const float *dgates,
                                const uint8_t *mask, const float *lse, const int32_t *counts, const int32_t *n_tokens,
                                const float *dlosses, int64_t tokens, int experts, int k, float balance_coef, float z_coef,
                                float *dlogits, void *stream) {
  DH_CHECK(tokens >= 0 && tokens < (1ll << 31) / BAL_MAX_K, "tokens=%lld", (long long)tokens);
  DH_CHECK(experts >= 1 && experts <= BAL_MAX_E, "experts=%d must be in [1, %d]", experts, BAL_MAX_E);
  DH_CHECK(k >= 1 && k <= BAL_MAX_K && k <= experts, "k=%d must be in [1, min(%d, experts)]", k, BAL_MAX_K);
  if (tokens == 0) return DH_OK;
  DH_CHECK(topk_idx && dlogits, "null pointer");
  DH_CHECK(!dgates || gates, "dgates without gates");
  DH_CHECK(!lse || (logits && counts && n_tokens), "the losses' gradient needs the logits, counts and n_tokens");
  DH_CHECK(dgates || lse, "neither dgates nor the losses' statistics: there is no gradient");
  const bool vec = experts % 4 == 0 && aligned16(logits) && aligned16(dlogits);
  const hipStream_t st = (hipStream_t)stream;
  BAL_LANES(experts, {
    int64_t blocks = cdiv(tokens * L, 256);
    if (blocks > 2048) blocks = 2048;              // eight a compute unit; 131072 tokens x 64 experts, k 8: 1024 19.6 us, 2048 17.3, 4096 18.7, 16384 20.7
    hipLaunchKernelGGL((route_bwd_kernel<L>), dim3((unsigned)blocks), dim3(256), 0, st, logits, topk_idx, gates, dgates, mask, lse,
                       counts, n_tokens, dlosses, tokens, experts, k, balance_coef, z_coef, dlogits, vec);
  });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

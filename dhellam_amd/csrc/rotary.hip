// Rotary positions in their general form: the two halves or the interleaved pairs of the first `rot` elements of a head, the rest
// passed through, angles from a table of whole numbers.
//
//   y_a = f (x_a cos - x_b sin),  y_b = f (x_b cos + x_a sin),  angle = position * frequency_j
//   (a, b) = (j, j + rot / 2) or (2j, 2j + 1);  backward: sin -> -sin
//
// A pair's frequency is kept as u = frequency / 2 pi in units of 2^-64 turns.  position * u modulo 2^64 is then the angle less its
// whole turns, exactly, whatever the position: two 32-bit multiplies for its upper half, against an fp32 product that is off
// by position * 2^-25 of the frequency (0.03 rad at a million) and a reduction after it.
//
// Bound by memory: every element is read and written once.  A lane owns a piece of W elements of the pairs (both halves of
// it, or interleaved), forms its angles once and walks heads of the same token with them.
#include "common.h"

namespace dh {
namespace {

// W elements in one access, aligned as single elements are: rows of any pitch and any start.
template <typename T, int W> struct Piece {
  T v[W];
};
template <int BYTES> struct Raw;
template <> struct Raw<2> { typedef uint16_t type; };
template <> struct Raw<4> { typedef uint32_t type __attribute__((aligned(2))); };
template <> struct Raw<8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Raw<16> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <typename T, int W> __device__ __forceinline__ Piece<T, W> load_piece(const T *p) {
  typedef typename Raw<sizeof(T) * W>::type R;
  return __builtin_bit_cast(Piece<T, W>, *reinterpret_cast<const R *>(p));
}
template <typename T, int W> __device__ __forceinline__ void store_piece(T *p, const Piece<T, W> &x) {
  typedef typename Raw<sizeof(T) * W>::type R;
  *reinterpret_cast<R *>(p) = __builtin_bit_cast(R, x);
}

// cos and sin of an angle in 2^-32 turns.  16-bit results: the hardware's instructions (about 1e-6 off, a hundredth of fp16's rounding).
// fp32: the nearest eighth turns are taken off in integers, what is left (at most pi / 4) goes into the two Taylor series, whose next
// terms are below 2e-9.
template <bool EXACT> __device__ __forceinline__ void turn(int32_t a, float factor, float &c, float &s) {
  if constexpr (!EXACT) {
    const float rev = (float)a * 0x1p-32f;
    c = __builtin_amdgcn_cosf(rev) * factor;
    s = __builtin_amdgcn_sinf(rev) * factor;
  } else {
    const uint32_t quarter = ((uint32_t)a + 0x20000000u) >> 30;
    const float x = (float)(int32_t)((uint32_t)a - (quarter << 30)) * 1.46291807926715968105e-9f;      // 2 pi / 2^32
    const float z = x * x;
    const float sx = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880 - z * (1.f / 39916800)))));
    const float cx = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
    const float c1 = quarter & 1 ? sx : cx, s1 = quarter & 1 ? cx : sx;
    c = (quarter == 1 || quarter == 2 ? -c1 : c1) * factor;
    s = (quarter >= 2 ? -s1 : s1) * factor;
  }
}

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  const uint64_t *steps;
  const void *positions;
  int64_t tokens, seq_len;
  int64_t q_tok, q_head, k_tok, k_head, qo_tok, qo_head, ko_tok, ko_head;
  int hq, hk, d, rot, wide_positions;
  uint32_t pieces, rot_pieces, slots, lanes;      // of a head; of its turned part; lanes that share a token's heads; lanes of a token
  float factor, sign;
};

template <typename T, int W, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  constexpr int NP = INTER ? W / 2 : W;            // pairs of a piece
  constexpr int HG = 4;                            // heads in flight
  const uint32_t heads = a.hq + a.hk;
  for (int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x; item < a.tokens * a.lanes; item += (int64_t)gridDim.x * 256) {
    const int64_t t = item / a.lanes;
    const uint32_t r = (uint32_t)(item - t * a.lanes), c = r % a.pieces, slot = r / a.pieces;
    auto src_of = [&](uint32_t h) {
      return h < (uint32_t)a.hq ? (const T *)a.q + t * a.q_tok + h * a.q_head : (const T *)a.k + t * a.k_tok + (h - a.hq) * a.k_head;
    };
    auto dst_of = [&](uint32_t h) {
      return h < (uint32_t)a.hq ? (T *)a.qo + t * a.qo_tok + h * a.qo_head : (T *)a.ko + t * a.ko_tok + (h - a.hq) * a.ko_head;
    };
    if (c >= a.rot_pieces) {                       // what is not turned: copied, the last piece element by element
      const int at = a.rot + (int)(c - a.rot_pieces) * W, n = a.d - at < W ? a.d - at : W;
      for (uint32_t h = slot; h < heads; h += a.slots) {
        const T *src = src_of(h) + at;
        T *dst = dst_of(h) + at;
        if (n == W) {
          store_piece<T, W>(dst, load_piece<T, W>(src));
        } else {
          for (int i = 0; i < n; ++i) dst[i] = src[i];
        }
      }
      continue;
    }
    const int lo = (int)c * W, hi = lo + (INTER ? 0 : a.rot / 2);
    Piece<T, W> x[HG], y[HG];
    auto load_group = [&](uint32_t h0) {
#pragma unroll
      for (int g = 0; g < HG; ++g)
        if (h0 + g * a.slots < heads) {
          const T *src = src_of(h0 + g * a.slots);
          x[g] = load_piece<T, W>(src + lo);
          if constexpr (!INTER) y[g] = load_piece<T, W>(src + hi);
        }
    };
    load_group(slot);
    int64_t pos;
    if (a.positions) pos = a.wide_positions ? ((const int64_t *)a.positions)[t] : ((const int32_t *)a.positions)[t];
    else pos = a.seq_len > 0 ? t % a.seq_len : t;
    float cs[NP], sn[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      turn<sizeof(T) == 4>((int32_t)(((uint64_t)pos * a.steps[c * NP + j]) >> 32), a.factor, cs[j], sn[j]);
      sn[j] *= a.sign;
    }
    for (uint32_t h0 = slot; h0 < heads; h0 += HG * a.slots) {
      if (h0 != slot) load_group(h0);
#pragma unroll
      for (int g = 0; g < HG; ++g)
        if (h0 + g * a.slots < heads) {
          T *dst = dst_of(h0 + g * a.slots);
          Piece<T, W> u, v;
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const float p = to_f(x[g].v[INTER ? 2 * j : j]), q = to_f(INTER ? x[g].v[2 * j + 1] : y[g].v[j]);
            const T up = from_f<T>(p * cs[j] - q * sn[j]), vq = from_f<T>(q * cs[j] + p * sn[j]);
            if constexpr (INTER) {
              u.v[2 * j] = up;
              u.v[2 * j + 1] = vq;
            } else {
              u.v[j] = up;
              v.v[j] = vq;
            }
          }
          store_piece<T, W>(dst + lo, u);
          if constexpr (!INTER) store_piece<T, W>(dst + hi, v);
        }
    }
  }
}

template <typename T, int W> void rotary_launch(const RotaryArgs &a, bool inter, int64_t blocks, hipStream_t st) {
  if constexpr (W >= 2)
    if (inter) {
      hipLaunchKernelGGL((rotary_kernel<T, W, true>), dim3((unsigned)blocks), dim3(256), 0, st, a);
      return;
    }
  hipLaunchKernelGGL((rotary_kernel<T, W, false>), dim3((unsigned)blocks), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace dh

extern "C" int dh_rotary(const void *q, const void *k, void *q_out, void *k_out, const uint64_t *steps, const void *positions,
                         int position_bytes, int64_t tokens, int hq, int hk, int d, int rot, int64_t q_token, int64_t q_head,
                         int64_t k_token, int64_t k_head, int64_t qo_token, int64_t qo_head, int64_t ko_token, int64_t ko_head,
                         int64_t seq_len, int interleaved, int backward, float factor, int dtype, void *stream) {
  using namespace dh;
  DH_CHECK(tokens >= 0 && hq >= 0 && hk >= 0 && d > 0 && hq < (1 << 20) && hk < (1 << 20) && d < (1 << 20),
           "bad shape tokens=%lld hq=%d hk=%d d=%d", (long long)tokens, hq, hk, d);
  DH_CHECK(rot >= 2 && rot % 2 == 0 && rot <= d, "%d turned elements of a head of %d: an even number, at least 2", rot, d);
  DH_CHECK(dtype == DH_F32 || dtype == DH_BF16 || dtype == DH_F16, "unknown dtype %d", dtype);
  if (tokens == 0 || hq + hk == 0) return DH_OK;
  DH_CHECK(steps, "steps is null");
  DH_CHECK(hq == 0 || (q && q_out), "q/q_out null with hq > 0");
  DH_CHECK(hk == 0 || (k && k_out), "k/k_out null with hk > 0");
  DH_CHECK(!positions || position_bytes == 4 || position_bytes == 8, "positions of %d bytes", position_bytes);
  // the widest piece that cuts the turned part (a half of it) without a rest
  const int n = 16 / (int)dtype_size(dtype), part = interleaved ? rot : rot / 2;
  int w = n;
  while (part % w) w /= 2;
  RotaryArgs a{q, k, q_out, k_out, steps, positions, tokens, seq_len, q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token,
               ko_head, hq, hk, d, rot, position_bytes == 8, 0, 0, 0, 0, factor, backward ? -1.f : 1.f};
  a.rot_pieces = (uint32_t)(part / w);
  const bool inplace = (hq == 0 || q == q_out) && (hk == 0 || k == k_out);
  a.pieces = a.rot_pieces + (inplace ? 0 : (uint32_t)((d - rot + w - 1) / w));
  const int heads = hq + hk;
  // lanes that share a token's heads: until the chip is full, then four heads a lane
  a.slots = 1;
  while ((int)a.slots < heads && tokens * a.pieces * a.slots < 256ll * 256 * 2) ++a.slots;
  a.lanes = a.pieces * a.slots;
  int64_t blocks = cdiv(tokens * (int64_t)a.lanes, 256);
  if (blocks > 1 << 20) blocks = 1 << 20;
  const hipStream_t st = (hipStream_t)stream;
  DH_DISPATCH_DTYPE(dtype, {
    switch (w) {
      case 8:
        if constexpr (sizeof(T) == 2) rotary_launch<T, 8>(a, interleaved, blocks, st);
        break;
      case 4: rotary_launch<T, 4>(a, interleaved, blocks, st); break;
      case 2: rotary_launch<T, 2>(a, interleaved, blocks, st); break;
      default: rotary_launch<T, 1>(a, interleaved, blocks, st);
    }
  });
  DH_LAUNCH_CHECK();
  return DH_OK;
}

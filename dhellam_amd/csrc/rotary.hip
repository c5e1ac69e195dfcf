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
// Bound by memory: every element is read and written once.  A lane owns a piece of 16 bytes of the pairs (of both halves, or
// interleaved), forms its angles once and turns that piece of one or two heads with them.  65536 tokens x 40 heads of 128 in bf16 (1.34 GB):
// 220 us, 6.1 TB/s; a copy on this card 5.9 TB/s.  Small calls are a launch: 1 token 2.6 us.
#include <type_traits>

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
template <bool NT, int W, typename T> __device__ __forceinline__ Piece<T, W> load_piece(const T *p) {
  typedef typename Raw<sizeof(T) * W>::type R;
  const R *q = reinterpret_cast<const R *>(p);
  return __builtin_bit_cast(Piece<T, W>, NT ? __builtin_nontemporal_load(q) : *q);
}
template <bool NT, int W, typename T> __device__ __forceinline__ void store_piece(T *p, const Piece<T, W> &x) {
  typedef typename Raw<sizeof(T) * W>::type R;
  const R v = __builtin_bit_cast(R, x);
  if (NT) __builtin_nontemporal_store(v, reinterpret_cast<R *>(p));
  else *reinterpret_cast<R *>(p) = v;
}

// The rounding to 16 bits as a step of its own.  The compiler fuses that to fp16 into the sum before it for some elements of a piece and not
// for others; an element's bits would then depend on where in a piece it lies, so on the number of tokens, on in place or not, and, where
// pieces overlap, on which lane comes last.
template <typename T> __device__ __forceinline__ T rounded(float x) {
  if constexpr (std::is_same_v<T, f16_t>) asm("" : "+v"(x));
  return from_f<T>(x);
}

// n / d for n < 2^31 by a product with floor(2^32 (2^l - d) / d) + 1, 2^l the first power of two from d on (Granlund and Montgomery, Division
// by invariant integers using multiplication, 1994).
struct Divider {
  uint32_t d, m, l;
  explicit Divider(uint32_t by) : d(by < 1 ? 1 : by), m(0), l(0) {
    while ((1ull << l) < d) ++l;
    m = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> l; }
};

// cos and sin of an angle in 2^-32 turns.  16-bit results: the hardware's instructions (about 1e-6 off, a hundredth of fp16's rounding).
// fp32: the nearest eighth turns are taken off in integers, what is left (at most pi / 4) goes into the two Taylor series, whose next
// terms are below 2e-9.
template <bool EXACT> __device__ __forceinline__ void turn(int32_t a, float &c, float &s) {
  if constexpr (!EXACT) {
    const float rev = (float)a * 0x1p-32f;
    c = __builtin_amdgcn_cosf(rev);
    s = __builtin_amdgcn_sinf(rev);
  } else {
    const uint32_t quarter = ((uint32_t)a + 0x20000000u) >> 30;
    const float x = (float)(int32_t)((uint32_t)a - (quarter << 30)) * 1.46291807926715968105e-9f;      // 2 pi / 2^32
    const float z = x * x;
    const float sx = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880 - z * (1.f / 39916800)))));
    const float cx = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
    const float c1 = quarter & 1 ? sx : cx, s1 = quarter & 1 ? cx : sx;
    c = quarter == 1 || quarter == 2 ? -c1 : c1;
    s = quarter >= 2 ? -s1 : s1;
  }
}

struct RotaryTensor {
  const char *in;
  char *out;
  int64_t in_tok, in_head, out_tok, out_head;      // bytes
  int heads;
};
struct RotaryArgs {
  RotaryTensor q, k;
  const uint64_t *steps;
  const void *positions;
  int64_t first, seq_len;                          // the launch's first token
  int d, rot, wide_positions;
  // Lanes: a token's behind one another, in them those of its heads' pieces, turned ones first.  Or tokens in groups of 64, in a group first
  // all lanes of turned pieces (then a token has `lanes` of them and a head `pieces`) and then all others: wavefronts of one kind.
  uint32_t items, tokens, group_tokens, turned, q_slots, k_slots;      // turned: pieces of a head that turn, or lanes of a group; slots: lanes that share heads
  Divider group, lanes, pieces, rest_lanes, rest_pieces;
  float factor, sin_factor;
};

// H: heads of a lane, `slots` apart; REST: there is a rest of the head, to be copied
template <typename T, int W, bool INTER, bool REST, bool NT, int H>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  constexpr int NP = INTER ? W / 2 : W;            // pairs of a piece
  constexpr int WT = 16 / sizeof(T);               // elements of a piece that is not turned
  const uint32_t item = blockIdx.x * 256 + threadIdx.x;
  if (item >= a.items) return;
  bool rest = false;
  Divider lanes = a.lanes, pieces = a.pieces;
  uint32_t r = item, tl = 0;
  if constexpr (REST)
    if (a.group_tokens > 1) {
      const uint32_t group = a.group.div(item);
      r -= group * a.group.d;
      tl = group * a.group_tokens;
      rest = r >= a.turned;
      if (rest) {
        r -= a.turned;
        lanes = a.rest_lanes;
        pieces = a.rest_pieces;
      }
    }
  const uint32_t in_group = lanes.div(r);
  r -= in_group * lanes.d;
  tl += in_group;
  if (REST && tl >= a.tokens) return;
  uint32_t slot = pieces.div(r), c = r - slot * pieces.d;
  if constexpr (REST)
    if (a.group_tokens == 1 && c >= a.turned) {
      rest = true;
      c -= a.turned;
    }
  const bool of_k = slot >= a.q_slots;
  const char *src = of_k ? a.k.in : a.q.in;
  char *dst = of_k ? a.k.out : a.q.out;
  const int64_t in_head = of_k ? a.k.in_head : a.q.in_head, out_head = of_k ? a.k.out_head : a.q.out_head;
  const uint32_t slots = of_k ? a.k_slots : a.q_slots;
  if (of_k) slot -= a.q_slots;
  src += (int64_t)tl * (of_k ? a.k.in_tok : a.q.in_tok) + (int64_t)slot * in_head;
  dst += (int64_t)tl * (of_k ? a.k.out_tok : a.q.out_tok) + (int64_t)slot * out_head;
  const int n_heads = ((of_k ? a.k.heads : a.q.heads) - (int)slot + (int)slots - 1) / (int)slots;
  const int64_t in_step = in_head * slots, out_step = out_head * slots;
  // (out of place the last piece of a part may begin in the one before it: the same values twice)
  if (rest) {                                      // what is not turned: copied
    const int n = a.d - a.rot;
    int at = (int)c * WT;
    if (n >= WT && at > n - WT) at = n - WT;
    const T *s = (const T *)src + a.rot + at;
    T *o = (T *)dst + a.rot + at;
    if (n >= WT) {
      Piece<T, WT> x[H];
#pragma unroll
      for (int g = 0; g < H; ++g)
        if (g < n_heads) x[g] = load_piece<NT, WT>((const T *)((const char *)s + g * in_step));
#pragma unroll
      for (int g = 0; g < H; ++g)
        if (g < n_heads) store_piece<NT, WT>((T *)((char *)o + g * out_step), x[g]);
    } else {
      for (int g = 0; g < n_heads; ++g)
        for (int i = 0; i < n; ++i) ((T *)((char *)o + g * out_step))[i] = ((const T *)((const char *)s + g * in_step))[i];
    }
    return;
  }
  const int part = INTER ? a.rot : a.rot / 2, lo = (int)c * W < part - W ? (int)c * W : part - W, hi = lo + (INTER ? 0 : part);
  Piece<T, W> x[H], y[H];
#pragma unroll
  for (int g = 0; g < H; ++g)
    if (g < n_heads) {
      const T *s = (const T *)(src + g * in_step);
      x[g] = load_piece<NT, W>(s + lo);
      if constexpr (!INTER) y[g] = load_piece<NT, W>(s + hi);
    }
  const int64_t t = a.first + tl;
  int64_t pos;
  if (a.positions) pos = a.wide_positions ? ((const int64_t *)a.positions)[t] : ((const int32_t *)a.positions)[t];
  else pos = a.seq_len > 0 ? t % a.seq_len : t;
  float cs[NP], sn[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    turn<sizeof(T) == 4>((int32_t)(((uint64_t)pos * a.steps[(INTER ? lo / 2 : lo) + j]) >> 32), cs[j], sn[j]);
    cs[j] *= a.factor;
    sn[j] *= a.sin_factor;
  }
#pragma unroll
  for (int g = 0; g < H; ++g)
    if (g < n_heads) {
      T *o = (T *)(dst + g * out_step);
      Piece<T, W> u, v;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const float p = to_f(x[g].v[INTER ? 2 * j : j]), q = to_f(INTER ? x[g].v[2 * j + 1] : y[g].v[j]);
        const T up = rounded<T>(fmaf(p, cs[j], -(q * sn[j]))), vq = rounded<T>(fmaf(q, cs[j], p * sn[j]));
        if constexpr (INTER) {
          u.v[2 * j] = up;
          u.v[2 * j + 1] = vq;
        } else {
          u.v[j] = up;
          v.v[j] = vq;
        }
      }
      store_piece<NT, W>(o + lo, u);
      if constexpr (!INTER) store_piece<NT, W>(o + hi, v);
    }
}

template <typename T, int W, bool INTER, bool REST> void rotary_launch(const RotaryArgs &a, int heads, bool nt, hipStream_t st) {
  const auto kernel = heads == 1 ? rotary_kernel<T, W, INTER, REST, false, 1>
                    : nt         ? rotary_kernel<T, W, INTER, REST, true, 2> : rotary_kernel<T, W, INTER, REST, false, 2>;
  hipLaunchKernelGGL(kernel, dim3((a.items + 255) / 256), dim3(256), 0, st, a);
}
template <typename T, int W> void rotary_launch(const RotaryArgs &a, bool inter, bool rest, int heads, bool nt, hipStream_t st) {
  if constexpr (W >= 2)
    if (inter) return rest ? rotary_launch<T, W, true, true>(a, heads, nt, st) : rotary_launch<T, W, true, false>(a, heads, nt, st);
  if (rest) rotary_launch<T, W, false, true>(a, heads, nt, st);
  else rotary_launch<T, W, false, false>(a, heads, nt, st);
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
  // pieces of 16 bytes, or the widest power of two that the turned part (a half of it) holds; in place one that cuts it without a rest
  const bool q_inplace = hq > 0 && q == q_out, k_inplace = hk > 0 && k == k_out, inplace = (hq == 0 || q_inplace) && (hk == 0 || k_inplace);
  DH_CHECK(!q_inplace || (q_token == qo_token && q_head == qo_head), "q in place with other strides");
  DH_CHECK(!k_inplace || (k_token == ko_token && k_head == ko_head), "k in place with other strides");
  const int n = 16 / (int)dtype_size(dtype), part = interleaved ? rot : rot / 2;
  int w = n;
  while (q_inplace || k_inplace ? part % w : w > part) w /= 2;
  const uint32_t turned_pieces = (uint32_t)cdiv(part, w), rest_pieces = inplace ? 0 : (uint32_t)cdiv(d - rot, n);
  const int64_t pieces = turned_pieces + rest_pieces, e = (int64_t)dtype_size(dtype), bytes = 2 * tokens * (hq + hk) * d * e;
  // heads of a lane: two, which share the angles and twice the bytes in flight; one while that leaves the chip half empty.  us, one / two /
  // four: bf16, d 128: 1 token x 40 heads 2.6 / 2.8 / 3.3, 512 x 40 4.6 / 4.8 / 5.3, 4096 x 9 6.4 / 6.1 / 6.4, 65536 x 40 221 / 218 / 236,
  // interleaved 246 / 226 / 233; fp32, 1000 x 32 heads of 64 5.4 / 5.1 / 5.2
  const int per_lane = tokens * pieces * (hq + hk) <= 1 << 18 ? 1 : 2;
  const uint32_t q_slots = (uint32_t)cdiv(hq, per_lane), k_slots = (uint32_t)cdiv(hk, per_lane);
  const uint64_t lanes = (uint64_t)pieces * (q_slots + k_slots);
  DH_CHECK(lanes < 1u << 22, "hq=%d hk=%d heads of %d are too many", hq, hk, d);
  // where the two parts of a head do not share its memory's 64-byte pieces: us by single tokens / by groups, bf16, 60000 x 40 heads of 64, 32 of
  // them turned, 162 / 138 (pairs 134 / 129), 16384 x 40 of 128, 64 turned, 63 / 61, but 4096 x 40 of 64 9.7 / 11.2; fp16, 60000 x 40 of 80, 20
  // turned, 196 / 273 (pairs 187 / 278), 30000 x 40 of 96, 48 turned, 125 / 139
  const uint32_t group = rest_pieces && tokens >= 64 && rot * e % 64 == 0 && d * e % 64 == 0 ? 64 : 1, turned_lanes = turned_pieces * (q_slots + k_slots);
  const bool grouped = group > 1;
  RotaryArgs a{{(const char *)q, (char *)q_out, q_token * e, q_head * e, qo_token * e, qo_head * e, hq},
               {(const char *)k, (char *)k_out, k_token * e, k_head * e, ko_token * e, ko_head * e, hk},
               steps, positions, 0, seq_len, d, rot, position_bytes == 8, 0, 0, group, grouped ? group * turned_lanes : turned_pieces, q_slots,
               k_slots, Divider(group * (uint32_t)lanes), Divider(grouped ? turned_lanes : (uint32_t)lanes),
               Divider(grouped ? turned_pieces : (uint32_t)pieces), Divider((uint32_t)lanes - turned_lanes), Divider(rest_pieces), factor,
               backward ? -factor : factor};
  // past the caches where the tensors do not fit there, but only in whole cache lines: 12 + 4 heads of 96 in fp16, whose halves are 96
  // bytes, 60000 tokens, 76 us, past them 96; 32 + 8 heads of 128 in bf16, 65536, 245, past them 218
  const bool nt = stream_hint(bytes) && (interleaved ? rot : rot / 2) * e % 128 == 0 && (d - rot) * e % 128 == 0;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t most = (int64_t)((1u << 30) / (group * lanes)) * group;      // tokens of a launch
  for (; a.first < tokens; a.first += most) {
    if (a.first) {
      a.q.in += most * a.q.in_tok, a.q.out += most * a.q.out_tok;
      a.k.in += most * a.k.in_tok, a.k.out += most * a.k.out_tok;
    }
    a.tokens = (uint32_t)(tokens - a.first < most ? tokens - a.first : most);
    a.items = (uint32_t)(cdiv(a.tokens, group) * group * (int64_t)lanes);
    DH_DISPATCH_DTYPE(dtype, {
      switch (w) {
        case 8:
          if constexpr (sizeof(T) == 2) rotary_launch<T, 8>(a, interleaved, rest_pieces > 0, per_lane, nt, st);
          break;
        case 4: rotary_launch<T, 4>(a, interleaved, rest_pieces > 0, per_lane, nt, st); break;
        case 2: rotary_launch<T, 2>(a, interleaved, rest_pieces > 0, per_lane, nt, st); break;
        default: rotary_launch<T, 1>(a, interleaved, rest_pieces > 0, per_lane, nt, st);
      }
    });
  }
  DH_LAUNCH_CHECK();
  return DH_OK;
}

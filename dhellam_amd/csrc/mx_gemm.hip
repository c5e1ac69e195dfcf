// Products of microscaled operands on gfx950's scaled matrix instructions: c[m, n] (+)= sum_k a[m, k] * b[n, k], a and b each in
// e4m3 or e2m1 with a scale a block of 32 along k (mx.h), fp32 sums, c in fp32, bf16 or fp16.
//
// v_mfma_scale_f32_16x16x128_f8f6f4, lane l (r = l % 16, g = l / 16): the operand's row (column) r; an 8-bit operand's 32 bytes are
// k = 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15, a 4-bit operand's 16 bytes k = 32 g .. 32 g + 31; the scale of block g of row r is a
// byte of the lane's scale register, chosen by the instruction.  D: 4 floats, D[row = 4 g + v][col = r].  A scale of 255 makes its own
// row (column) NaN, whatever the elements are.  The product is formed as C^T (b in the first slot), so that a lane holds neighbouring
// columns of one row of c.
//
// How exact it is: of the products of e4m3 elements the instruction adds 8 or 16 at a time aligned to the largest, and drops what lies more than
// 13 bits below that one's leading bit (measured, and the same for its unscaled form): on normal data a sum is off by 1.5e-5 to
// 2.5e-5 of itself, whatever its length, with one 4-bit operand by 7e-6; products of two 4-bit operands are exact.  A result in 16 bits is
// rounded to 2^-9 (2^-12), far above that.  A result in fp32 is promised to 1e-5 everywhere else in this library, so with an 8-bit
// operand it is formed from the elements in bf16, which hold them and their scales exactly (mx_wide below).
#include <algorithm>
#include <type_traits>

#include "mma.h"
#include "mx.h"
#include "tile_order.h"

namespace dh {

typedef int mx_v8i __attribute__((ext_vector_type(8)));

struct MxGemmParams {
  const uint8_t *a, *as, *b, *bs;     // codes and scales
  void *c;
  float *ws;                          // partial tiles where k is split
  int64_t m, n, ldc;
  int64_t cells_a, cells_b;           // 16-byte cells of scales in a group of 128 columns
  int steps;                          // k / 128, rounded up
  int accumulate, vec;                // vec: rows of c take 16-byte accesses
  int tiles_m, tiles_n, pieces;       // (of k; one where tiles are of 256 x 256)
};

template <int BITS> struct MxBytes { static constexpr int STEP = BITS * 16; };   // bytes of 128 columns

// A lane's share of 128 columns of one row: chunk 0 (and 1) of 16 bytes.
template <int BITS> struct MxFrag { int4v q[BITS / 4]; };
template <int BITS> __device__ __forceinline__ mx_v8i mx_operand(const MxFrag<BITS> &f) {
  if constexpr (BITS == 8) return mx_v8i{f.q[0][0], f.q[0][1], f.q[0][2], f.q[0][3], f.q[1][0], f.q[1][1], f.q[1][2], f.q[1][3]};
  else return mx_v8i{f.q[0][0], f.q[0][1], f.q[0][2], f.q[0][3], 0, 0, 0, 0};
}
// format field of the instruction: 0 e4m3, 4 e2m1
template <int FA, int FB, int SELB, int SELA>
__device__ __forceinline__ floatx4 mx_mma(const MxFrag<FB> &b, uint32_t sb, const MxFrag<FA> &a, uint32_t sa, const floatx4 &c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(b), mx_operand(a), c, FB == 8 ? 0 : 4, FA == 8 ? 0 : 4, SELB, (int)sb, SELA, (int)sa);
}
template <int FA, int FB>
__device__ __forceinline__ floatx4 mx_mma_sel(int selb, int sela, const MxFrag<FB> &b, uint32_t sb, const MxFrag<FA> &a, uint32_t sa, const floatx4 &c) {
#define MX_SEL(x, y) if (selb == x && sela == y) return mx_mma<FA, FB, x, y>(b, sb, a, sa, c)
  MX_SEL(0, 0); MX_SEL(0, 1); MX_SEL(0, 2); MX_SEL(0, 3);
  MX_SEL(1, 0); MX_SEL(1, 1); MX_SEL(1, 2); MX_SEL(1, 3);
  MX_SEL(2, 0); MX_SEL(2, 1); MX_SEL(2, 2); MX_SEL(2, 3);
  MX_SEL(3, 0); MX_SEL(3, 1); MX_SEL(3, 2);
#undef MX_SEL
  return mx_mma<FA, FB, 3, 3>(b, sb, a, sa, c);
}

// The same 128 columns in four v_mfma_f32_16x16x32_bf16: a lane takes the 32 columns of block g, whose elements times their scale are exact in
// bf16 unless they lie below its smallest normal number (2^-126; all is lost below 2^-133), and products are added in fp32.
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fc00000u : code == 0u ? 0x400000u : code << 23);
}
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
template <int BITS> struct MxWide { bf16x8 v[4]; };
template <int BITS> __device__ __forceinline__ MxWide<BITS> mx_wide(const MxFrag<BITS> &f, float scale) {
  MxWide<BITS> o;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    mx_bf16x2 x[4];
    if constexpr (BITS == 8) {
      const int lo = f.q[t >> 1][2 * (t & 1)], hi = f.q[t >> 1][2 * (t & 1) + 1];
      x[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
      x[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
      x[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
      x[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    } else {
      const uint32_t q = (uint32_t)f.q[0][t];
      x[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
      x[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
      x[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
      x[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o.v[t][2 * i] = x[i][0];
      o.v[t][2 * i + 1] = x[i][1];
    }
  }
  return o;
}

// The same instruction as assembly whose sum stays in its registers: with the builtin the compiler moved accumulators about and ran out
// of registers in mx_w8_kernel.  It does not know these for matrix instructions: what reads a sum waits first.
template <int FA, int FB, int SELB, int SELA, typename VB, typename VA>
__device__ __forceinline__ void mx_mma_tied(const VB &b, uint32_t sb, const VA &a, uint32_t sa, floatx4 &c) {
#ifdef __HIP_DEVICE_COMPILE__                                       // (the host's compiler has no registers for such operands)
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%c5,%c6,0] op_sel_hi:[%c7,%c8,0] cbsz:%c9 blgp:%c10"
               : "+v"(c)
               : "v"(b), "v"(a), "v"(sb), "v"(sa), "n"(SELB & 1), "n"(SELA & 1), "n"(SELB >> 1), "n"(SELA >> 1), "n"(FB == 8 ? 0 : 4), "n"(FA == 8 ? 0 : 4));
#endif
}
// 32 x 32 x 64 of 4 bits, for which this is the faster form: lane l holds block l / 32 (k = 32 (l / 32) and on) of row l % 32; D[row = 8 (v / 4) + 4
// (l / 32) + v % 4][col = l % 32].  In a loop of nothing else the matrix pipes are busy for 91 to 94 % of the time with it and 53 to 72 % with 16 x
// 16 x 128 (one to four wavefronts a SIMD), whose instruction takes longer to issue than its 16 cycles; on random data, where the board's power
// bounds both, 6.5 against 5.9 PFLOP/s.  (With an 8-bit operand it is the other way round: 4.05 against 4.36.)
template <int SELB, int SELA> __device__ __forceinline__ void mx_mma32_tied(const int4v &b, uint32_t sb, const int4v &a, uint32_t sa, floatx16 &c) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%c5,%c6,0] op_sel_hi:[%c7,%c8,0] cbsz:4 blgp:4"
               : "+v"(c)
               : "v"(b), "v"(a), "v"(sb), "v"(sa), "n"(SELB & 1), "n"(SELA & 1), "n"(SELB >> 1), "n"(SELA >> 1));
#endif
}
// The four dwords of a cell are blocks 0..3 of its 128 columns, a row a byte.  Of a lane's two rows y and y + 2: bytes [block][row] of blocks 0, 1
// and 2, 3.  Of its one row y: the four blocks.
__device__ __forceinline__ void mx_cell_rows2(uint32_t (&s)[2], const int4v &cell, uint32_t y) {
  const uint32_t sel = 0x06040200u + y * 0x01010101u;
  s[0] = __builtin_amdgcn_perm((uint32_t)cell[1], (uint32_t)cell[0], sel);
  s[1] = __builtin_amdgcn_perm((uint32_t)cell[3], (uint32_t)cell[2], sel);
}
__device__ __forceinline__ uint32_t mx_cell_row1(const int4v &cell, uint32_t y) {
  const uint32_t sel = 0x0400u + y * 0x0101u;
  const uint32_t lo = __builtin_amdgcn_perm((uint32_t)cell[1], (uint32_t)cell[0], sel), hi = __builtin_amdgcn_perm((uint32_t)cell[3], (uint32_t)cell[2], sel);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
template <int BITS> __device__ __forceinline__ auto mx_narrow(const int4v *q, int ks) {
  if constexpr (BITS == 8) return mx_v8i{q[0][0], q[0][1], q[0][2], q[0][3], q[1][0], q[1][1], q[1][2], q[1][3]};
  else return q[ks];
}

// What the chunks of a row in slot s are XORed with, rows of 128 bytes and of 64.  A read of 16 bytes a lane is served 16 lanes at a time, the first 16
// being lanes 0..3, 12..15, 20..23 and 24..27, the next the rest of the first 32; their chunks have to differ where lanes 0..15 read one chunk of
// 16 slots and lanes 16..31 its neighbour (16 x 16 x 128), the next but one (mx_wide), or 32 lanes one (32 x 32 x 64).  (slot / 2) % 8 alone costs mx_wide a second
// pass a read; with slot / 4 % 4 a fifth of LDS's cycles at 4096 x 7168 x 8192 in 8 x 4 bits were conflicts.
__device__ __forceinline__ int mx_turn8(int s) { return 0x32765410 >> (4 * ((s >> 1) & 7)) & 7; }
__device__ __forceinline__ int mx_turn4(int s) { return 0x78 >> (2 * ((s >> 2) & 3)) & 3; }

// c's element: added to if asked, rounded once.
template <typename TO> __device__ __forceinline__ TO mx_out(float v, const TO *old, int accumulate) {
  return from_f<TO>(accumulate ? v + to_f(*old) : v);
}
// N consecutive columns of a row, the first `left` of which exist
template <typename TO, int N> __device__ __forceinline__ void mx_store(TO *p, const float (&v)[N], int64_t left, int vec, int accumulate) {
  constexpr int E = 16 / (int)sizeof(TO);
  static_assert(N % E == 0 || N < E, "whole vectors");
  if constexpr (N % E == 0) {
    if (vec && left >= N) {
#pragma unroll
      for (int i = 0; i < N / E; ++i) {
        Vec<TO> o;
        if (accumulate) {
          const Vec<TO> old = ldg(p + E * i);
#pragma unroll
          for (int j = 0; j < E; ++j) o.v[j] = from_f<TO>(v[E * i + j] + to_f(old.v[j]));
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) o.v[j] = from_f<TO>(v[E * i + j]);
        }
        stg(p + E * i, o);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < left) p[j] = mx_out<TO>(v[j], p + j, accumulate);
}

// ---- few rows: operands straight to registers -----------------------------------------------------------------------------
// A workgroup makes a tile of 16 MT rows of a by 16 NT rows of b; its W wavefronts share the steps of 128 along k between them, one
// after the other, and add up through LDS in the order of the wavefronts.  Operand block i of MT (NT) takes the rows MT r + i, so that
// the scales of a lane's blocks lie side by side.  Where even so there are few workgroups, k is cut into pieces over workgroups as
// well, and mx_join_kernel adds these in order.
// Bound by the weights' bytes for a few rows: 1 x 7168 x 8192 with 4-bit weights 8 to 9 us for 31 MB (a copy's rate: 6.0), and by launch and the latency
// of a handful of loads for smaller ones (1 x 1280 x 8192 5 to 6).  Loads of the next step before this step's products did not help where the
// wavefronts of a compute unit are eight already (1 x 7168 x 8192, 777 x 1001 x 2080), nor did sixteen wavefronts.
// Step x of the P that a wavefront takes at a time.  With P of 2 the two steps' eight blocks are dealt out so that a lane's block of step x is
// block 2 g + x of them: its 4-bit elements of both steps are 32 consecutive bytes, a row's 128.
template <int BITS, int P, bool WIDE> __device__ __forceinline__ void mx_load(MxFrag<BITS> &f, const uint8_t *row, int g, int x) {
  if constexpr (BITS == 4) f.q[0] = *reinterpret_cast<const int4v *>(row + (P * g + x) * 16);
  else
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // (the instruction's 8-bit lane has the half g % 2 of blocks g / 2 and 2 + g / 2)
      const int block = WIDE ? P * g + x : P * (2 * i + (g >> 1)) + x, half = WIDE ? i : g & 1;
      f.q[i] = *reinterpret_cast<const int4v *>(row + block * 32 + half * 16);
    }
}
// The scales of a lane's block of step x, NB rows from `row` on; cells: from the unit's first group of 128 columns on.
template <int NB, int P> __device__ __forceinline__ uint32_t mx_scales(const uint8_t *s, int64_t cells, int64_t row, int g, int x) {
  const int block = P * g + x;
  const uint8_t *p = s + (block >> 2) * cells * 16 + (row >> 2) * 16 + (block & 3) * 4 + (row & 3);
  if constexpr (NB == 4) return *reinterpret_cast<const uint32_t *>(p);
  else if constexpr (NB == 2) return *reinterpret_cast<const uint16_t *>(p);
  else return *p;
}

template <int FA, int FB, int MT, int NT, int W, bool WIDE, typename TO>
__global__ void __launch_bounds__(64 * W) mx_direct_kernel(const MxGemmParams p) {
  constexpr int TM = 16 * MT, TN = 16 * NT, PITCH = TN + 4;
  constexpr int P = FB == 4 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float red[W * TM * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int t = blockIdx.x, piece = blockIdx.y;
  const int64_t m0 = (int64_t)(t % p.tiles_m) * TM, n0 = (int64_t)(t / p.tiles_m) * TN;
  const int64_t lda = (int64_t)p.steps * MxBytes<FA>::STEP, ldb = (int64_t)p.steps * MxBytes<FB>::STEP;
  const int64_t ra = m0 + MT * r, rb = n0 + NT * r;
  // rows past the end: those of the last row, into outputs that are not stored
  const uint8_t *ap[MT], *bp[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) ap[i] = p.a + std::min(ra + i, p.m - 1) * lda;
#pragma unroll
  for (int i = 0; i < NT; ++i) bp[i] = p.b + std::min(rb + i, p.n - 1) * ldb;
  const int64_t sra = std::min(ra, 4 * p.cells_a - MT), srb = std::min(rb, 4 * p.cells_b - NT);
  floatx4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  // U steps from s on
  auto unit = [&](auto u_, int64_t s) {
    constexpr int U = decltype(u_)::value;
    MxFrag<FA> fa[U][MT];
    MxFrag<FB> fb[U][NT];
    uint32_t sa[U], sb[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
#pragma unroll
      for (int j = 0; j < NT; ++j) mx_load<FB, U, WIDE>(fb[x][j], bp[j] + s * MxBytes<FB>::STEP, g, x);
      sb[x] = mx_scales<NT, U>(p.bs + s * p.cells_b * 16, p.cells_b, srb, g, x);
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
#pragma unroll
      for (int i = 0; i < MT; ++i) mx_load<FA, U, WIDE>(fa[x][i], ap[i] + s * MxBytes<FA>::STEP, g, x);
      sa[x] = mx_scales<MT, U>(p.as + s * p.cells_a * 16, p.cells_a, sra, g, x);
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      if constexpr (WIDE) {
        MxWide<FB> wb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) wb[j] = mx_wide<FB>(fb[x][j], mx_scale_value(sb[x] >> (8 * j) & 0xffu));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const MxWide<FA> wa = mx_wide<FA>(fa[x][i], mx_scale_value(sa[x] >> (8 * i) & 0xffu));
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = Mma<bf16_t>::mma16(wb[j].v[e], wa.v[e], acc[i][j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = mx_mma_sel<FA, FB>(j, i, fb[x][j], sb[x], fa[x][i], sa[x], acc[i][j]);
      }
    }
  };
  // the piece's units, one wavefront after the other; an odd last step is a unit of its own
  const int units = (p.steps + P - 1) / P;
  const int u0 = (int)((int64_t)piece * units / p.pieces), u1 = (int)((int64_t)(piece + 1) * units / p.pieces);
  for (int u = u0 + w; u < u1; u += W) {
    if (P == 2 && 2 * u + 1 == p.steps) unit(std::integral_constant<int, 1>{}, 2 * u);
    else unit(std::integral_constant<int, P>{}, (int64_t)P * u);
  }
  // D[row = 4 g + v] of block j is column NT (4 g + v) + j, its column r row MT r + i
  float *mine = red + w * TM * PITCH;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int j = 0; j < NT; ++j) mine[(MT * r + i) * PITCH + NT * (4 * g + v) + j] = acc[i][j][v];
  __syncthreads();
  constexpr int VPR = TN / 4;                              // groups of 4 columns in a row
  for (int u = tid; u < TM * VPR; u += 64 * W) {
    const int row = u / VPR, col = u % VPR * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const floatx4 q = *reinterpret_cast<const floatx4 *>(red + (x * TM + row) * PITCH + col);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += q[j];
    }
    if (m0 + row >= p.m || n0 + col >= p.n) continue;
    if (p.pieces > 1) {
      float *dst = p.ws + ((int64_t)piece * p.m + m0 + row) * (4 * p.cells_b) + n0 + col;
      *reinterpret_cast<floatx4 *>(dst) = floatx4{v[0], v[1], v[2], v[3]};
    } else {
      TO *dst = reinterpret_cast<TO *>(p.c) + (m0 + row) * p.ldc + n0 + col;
      mx_store<TO, 4>(dst, v, p.n - n0 - col, p.vec, p.accumulate);
    }
  }
}

// ---- 256 x 256 tiles: eight wavefronts in two alternating groups -------------------------------------------------------------
// The schedule of grouped_gemm_w8_kernel (grouped_gemm.hip, where its order of reads, waits, copies and barriers is argued): a wavefront has
// 128 x 64 outputs in four quarters, a quarter of a slice is [reads of fragments, copies | its MFMAs, more reads among them],
// and the wavefronts 4..7 run one barrier behind the others.  A slice is 128 bytes of a row here too: 256 columns where both operands have
// 4 bits (8 MFMAs of 32 x 32 x 64 in a quarter), 128 columns otherwise (8 of 16 x 16 x 128; a 4-bit operand's rows then have 64 bytes).
//
// LDS: regions of [128 slots][row bytes] for either half of the tile's rows of a and of b, two stages of them, and the scales in a ring
// of three.  Slots are dealt out so that the blocks a lane multiplies are neighbouring rows, whose scales lie in one cell, and a lane's outputs
// neighbouring columns.  16 x 16: slot s holds row 64 (s / 64) + 4 (s % 16) + s / 16 % 4 of a's half, row 32 (s / 32) + 2 (s % 16) + s / 16 % 2 of
// b's; the four (two) blocks' scales are read as one dword (half of one).  32 x 32: row 64 (s / 64) + 4 (s % 16) + 2 (s / 32 % 2) + s / 16 % 2 of
// a's half, row 32 (s / 32) + 4 (s % 8) + s / 8 % 4 of b's; a lane reads a whole cell, [4 blocks of 32][4 rows], and takes its rows' bytes out of
// it behind the next wait.  16-byte chunks are XORed with mx_turn8 (mx_turn4 in rows of 64 bytes): the lanes of a
// fragment read that LDS serves at once hit different chunks of 256 bytes.  Scales come as whole cells, 256 bytes a copy.
// Scales follow their fragments: those of the half that is read next lie in LDS since the wait two clusters before, and a slot of the
// ring is written again three slices later, long after its last read.
//
// Measured, 8192 x 8192 x 8192 to bf16: 8 x 8 bits 370 to 450 us with the board and the data's values (2.4 to 3.0 PFLOP/s), 4 x 4 bits 245 to
// 290 (3.8 to 4.5; 275 in blocks of 16 x 16 x 128 where these take 264).  Bound by power in 8 bits: the clock falls to 1.76 GHz of 2.4 and the matrix pipes are busy for 78 % of
// the time; in 4 bits they are busy for half of it at 1.95 GHz.  A tile costs about 10 us beside its slices (first copies, stores of c), which
// do not overlap with another's: one workgroup fills a compute unit's LDS.  From k of 4096 to 8192 8 x 8 bits run at 3.3 PFLOP/s, 4 x 4 at 5.2.
// Did not help: c by rows of 512 bytes through LDS (4 us a tile slower), copies a cluster earlier.
// 64 lanes x 4 bytes, as copy_1k
__device__ __forceinline__ void copy_256(uint32_t lane_off, const int4v &rsrc, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
               :
               : "v"(lane_off), "s"(rsrc), "s"(off), "s"(dst)
               : "memory", "m0");
}

template <int FA, int FB, typename TO>
__global__ void __launch_bounds__(512) mx_w8_kernel(const MxGemmParams p) {
  constexpr int KS = FA == 4 && FB == 4 ? 2 : 1;                 // steps of 128 columns in a slice
  constexpr int RA = KS * MxBytes<FA>::STEP, RB = KS * MxBytes<FB>::STEP;      // bytes of a row in a slice
  constexpr int NA = RA / 64, NB = RB / 64;                      // copies a wavefront issues for a region; 16-byte reads a fragment takes
  constexpr uint32_t REGA = 128 * RA, REGB = 128 * RB, OFF_B = 2 * REGA, STAGEB = OFF_B + 2 * REGB;
  constexpr uint32_t RING = 2 * STAGEB, SLOT = KS * 2048;        // scales of a slice: a's, then b's
  constexpr int COPIES = KS + 2 * NA + 2 * NB;                   // of a wavefront a slice
  constexpr bool B32 = KS == 2;                                  // in blocks of 32 x 32 x 64; else 16 x 16 x 128
  constexpr int SIDE = B32 ? 32 : 16, ABLK = 64 / SIDE, BBLK = 32 / SIDE;      // blocks of a half's 64 rows of a, 32 of b
  constexpr int APART = B32 ? 4 : NA, BPART = B32 ? 4 : NB;      // 16-byte reads of a block
  using Acc = std::conditional_t<B32, floatx16, floatx4>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[RING + 3 * SLOT];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w >> 2, wn = w & 3;
  const int c = lane & (SIDE - 1), g4 = lane / SIDE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
  const uint32_t lda = (uint32_t)p.steps * MxBytes<FA>::STEP, ldb = (uint32_t)p.steps * MxBytes<FB>::STEP;

  // ---- copies: a region is blocks of 1 KB, 8 slots of 128 bytes or 16 of 64; a wavefront takes NA (NB) neighbouring ones
  uint32_t ca[NA], cb[NB];
#pragma unroll
  for (int x = 0; x < NA; ++x) {
    const int s = NA == 2 ? 8 * (2 * w + x) + (lane >> 3) : 16 * w + (lane >> 2);
    const int chunk = NA == 2 ? (lane & 7) ^ mx_turn8(s) : (lane & 3) ^ mx_turn4(s);
    ca[x] = (uint32_t)(64 * (s >> 6) + 4 * (s & 15) + (B32 ? 2 * ((s >> 5) & 1) + ((s >> 4) & 1) : (s >> 4) & 3)) * lda + (uint32_t)(chunk * 16);
  }
#pragma unroll
  for (int x = 0; x < NB; ++x) {
    const int s = NB == 2 ? 8 * (2 * w + x) + (lane >> 3) : 16 * w + (lane >> 2);
    const int chunk = NB == 2 ? (lane & 7) ^ mx_turn8(s) : (lane & 3) ^ mx_turn4(s);
    cb[x] = (uint32_t)(32 * (s >> 5) + (B32 ? 4 * (s & 7) + ((s >> 3) & 3) : 2 * (s & 15) + ((s >> 4) & 1))) * ldb + (uint32_t)(chunk * 16);
  }
  const uint32_t cs = (uint32_t)(lane * 4);

  // ---- fragments and scales
  // chunk of a block's first read; the next: B32 the next chunk (a lane's half is one of the slice's two steps), else 4 chunks on
  constexpr uint32_t NEXT = B32 ? 16 : 64;
  const uint32_t qa = NA == 2 ? (B32 ? 4 * g4 : g4) ^ mx_turn8(c) : g4 ^ mx_turn4(c), qb = NB == 2 ? (B32 ? 4 * g4 : g4) ^ mx_turn8(c) : g4 ^ mx_turn4(c);
  const uint32_t fa_lane = (uint32_t)((wm * 64 + c) * RA) + qa * 16, fb_lane = (uint32_t)((wn * 32 + c) * RB) + qb * 16;
  // half: + 512; 16 x 16: step: + 1024
  const uint32_t sa_lane = (uint32_t)(wm * 256 + (c & 15) * 16) + (uint32_t)(B32 ? g4 * 1024 : g4 * 4);
  const uint32_t sb_lane = (uint32_t)(KS * 1024 + wn * 128) + (uint32_t)(B32 ? g4 * 1024 + (c & 7) * 16 : (c >> 1) * 16 + g4 * 4 + 2 * (c & 1));
  typedef __attribute__((address_space(3))) const int4v *lds_chunk;
  typedef __attribute__((address_space(3))) const uint32_t *lds_dword;
  typedef __attribute__((address_space(3))) const uint16_t *lds_half;

  const int pid = gg_xcd_chunk((int)blockIdx.x, p.tiles_m * p.tiles_n);
  int tm, tn;
  gg_tile_of(pid, p.tiles_m, p.tiles_n, tm, tn);
  const int cnt = (p.steps + KS - 1) / KS;                       // slices
  const int64_t m0 = (int64_t)tm * 256, n0 = (int64_t)tn * 256;
  // descriptors, cut at the operands' last rows: rows past them read as zeros
  int4v rsa = raw_rsrc(p.a + m0 * lda, std::min<int64_t>(p.m - m0, 256) * lda), rsb = raw_rsrc(p.b + n0 * ldb, std::min<int64_t>(p.n - n0, 256) * ldb);
  // (of the scales: a's and b's, where one copy a wavefront does, the one the wavefront copies)
  const bool sb_first = KS == 1 && w >= 4;
  int4v rss0 = raw_rsrc(sb_first ? p.bs + n0 * 4 : p.as + m0 * 4, sb_first ? (int64_t)p.steps * p.cells_b * 16 - n0 * 4 : (int64_t)p.steps * p.cells_a * 16 - m0 * 4);
  int4v rss1 = raw_rsrc(p.bs + n0 * 4, (int64_t)p.steps * p.cells_b * 16 - n0 * 4);
  const uint32_t gs0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)((sb_first ? p.cells_b : p.cells_a) * 16)), gs1 = (uint32_t)p.cells_b * 16;
  // they come out of v_readfirstlane, which the copies from assembly have to keep their distance from
  asm volatile("s_nop 4" : "+s"(rsa), "+s"(rsb), "+s"(rss0), "+s"(rss1));

  // before the copies of slice s
  auto turn_to = [&](int s) {
    if (s >= cnt) {
      rsa[2] = rsb[2] = rss0[2] = rss1[2] = 0;
    } else if (KS == 2 && (p.steps & 1) && s == cnt - 1) {
      // the last step of an odd number: chunks 4..7 are not there
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int ch = (lane & 7) ^ mx_turn8(8 * (2 * w + x) + (lane >> 3));
        if (ch >= 4) ca[x % NA] = cb[x % NB] = 0x80000000u;      // past any descriptor's end
      }
    }
  };
  auto copy_a = [&](int h, int s, uint32_t stage) {
#pragma unroll
    for (int x = 0; x < NA; ++x)
      copy_1k(ca[x], rsa, (uint32_t)s * RA + (uint32_t)h * 128 * lda, lds0 + stage + (uint32_t)h * REGA + (uint32_t)(NA * w + x) * 1024);
  };
  auto copy_b = [&](int h, int s, uint32_t stage) {
#pragma unroll
    for (int x = 0; x < NB; ++x)
      copy_1k(cb[x], rsb, (uint32_t)s * RB + (uint32_t)h * 128 * ldb, lds0 + stage + OFF_B + (uint32_t)h * REGB + (uint32_t)(NB * w + x) * 1024);
  };
  auto copy_s = [&](int s, uint32_t slot) {
    const uint32_t at = lds0 + slot, quarter = (uint32_t)(w & 3) * 256, to = (uint32_t)(w >> 2) * 1024 + quarter;
    if constexpr (KS == 2) {
      const uint32_t step = (uint32_t)(2 * s + (w >> 2));
      copy_256(cs, rss0, step * gs0 + quarter, at + to);
      copy_256(cs, rss1, step * gs1 + quarter, at + 2048 + to);
    } else {
      copy_256(cs, rss0, (uint32_t)s * gs0 + quarter, at + to);
    }
  };
  Acc acc[2][2][ABLK][BBLK];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < ABLK; ++b)
#pragma unroll
      for (int j = 0; j < BBLK; ++j) acc[i >> 1][i & 1][b][j] = Acc{};
  int4v fa[2][ABLK][APART], fb[2][BBLK][BPART];
  // scales as the instructions take them: 16 x 16: [half][step], a byte a block; 32 x 32: a's [half][steps 0, 1 / 2, 3 of 64], b's four steps in one;
  // a cell just read is taken apart behind the next wait
  uint32_t sa[2][2], sb[2][KS];
  int4v cell;
  auto mma_quarter = [&](int qm, int qn, auto rd) {
    __builtin_amdgcn_s_setprio(1);
    if constexpr (B32) {
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int t = x >> 1, b = x & 1;
#define MX_SEL(j, i) if (t == j && b == i) mx_mma32_tied<j, 2 * (j & 1) + i>(fb[qn][0][t], sb[qn][0], fa[qm][b][t], sa[qm][t >> 1], acc[qm][qn][b][0])
        MX_SEL(0, 0); MX_SEL(0, 1); MX_SEL(1, 0); MX_SEL(1, 1);
        MX_SEL(2, 0); MX_SEL(2, 1); MX_SEL(3, 0); MX_SEL(3, 1);
#undef MX_SEL
        __builtin_amdgcn_sched_barrier(0);
        rd(x);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int mi = x >> 1, nj = x & 1;
        const auto vb = mx_narrow<FB>(fb[qn][nj], 0);
        const auto va = mx_narrow<FA>(fa[qm][mi], 0);
        floatx4 &sum = acc[qm][qn][mi][nj];
#define MX_SEL(j, i) if (nj == j && mi == i) mx_mma_tied<FA, FB, j, i>(vb, sb[qn][0], va, sa[qm][0], sum)
        MX_SEL(0, 0); MX_SEL(0, 1); MX_SEL(0, 2); MX_SEL(0, 3);
        MX_SEL(1, 0); MX_SEL(1, 1); MX_SEL(1, 2); MX_SEL(1, 3);
#undef MX_SEL
        __builtin_amdgcn_sched_barrier(0);
        rd(x);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto read_a = [&](int h, uint32_t region, int x0, int x1) {    // reads x0..x1 of the half's ABLK APART
#pragma unroll
    for (int x = x0; x < x1; ++x)
      if (x < ABLK * APART)
        fa[h][x % ABLK][x / ABLK] = *(lds_chunk)(region + (fa_lane ^ (uint32_t)(x / ABLK) * NEXT) + (uint32_t)(x % ABLK * SIDE * RA));
  };
  auto read_b = [&](int h, uint32_t region, uint32_t slot) {
#pragma unroll
    for (int i = 0; i < BPART; ++i)
#pragma unroll
      for (int nj = 0; nj < BBLK; ++nj) fb[h][nj][i] = *(lds_chunk)(region + (fb_lane ^ (uint32_t)i * NEXT) + (uint32_t)(nj * SIDE * RB));
    if constexpr (B32) cell = *(lds_chunk)(lds0 + slot + sb_lane + (uint32_t)(h * 512));
    else sb[h][0] = *(lds_half)(lds0 + slot + sb_lane + (uint32_t)(h * 512));
  };
  auto read_sa = [&](int h, uint32_t slot) {
    if constexpr (B32) cell = *(lds_chunk)(lds0 + slot + sa_lane + (uint32_t)(h * 512));
    else sa[h][0] = *(lds_dword)(lds0 + slot + sa_lane + (uint32_t)(h * 512));
  };
  auto take_sa = [&](int h) { if constexpr (B32) mx_cell_rows2(sa[h], cell, (uint32_t)c >> 4); };
  auto take_sb = [&](int h) { if constexpr (B32) sb[h][0] = mx_cell_row1(cell, (uint32_t)c >> 3); };
#define MX_BARRIER()                        \
  do {                                      \
    __builtin_amdgcn_sched_barrier(0);      \
    asm volatile("s_barrier" ::: "memory"); \
    __builtin_amdgcn_sched_barrier(0);      \
  } while (0)
#define MX_READS_DONE() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")
#define MX_WAIT_BARRIER()                                                              \
  do {                                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                 \
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(COPIES) : "memory");         \
    __builtin_amdgcn_sched_barrier(0);                                                 \
  } while (0)

  uint32_t r0 = RING, r1 = RING + SLOT, r2 = RING + 2 * SLOT;    // the ring's slots of slices s, s + 1, s + 2
  turn_to(0);
  copy_s(0, r0); copy_a(0, 0, 0); copy_b(0, 0, 0); copy_b(1, 0, 0); copy_a(1, 0, 0);
  turn_to(1);
  copy_s(1, r1); copy_a(0, 1, STAGEB); copy_b(1, 1, STAGEB); copy_b(0, 1, STAGEB); copy_a(1, 1, STAGEB);
  MX_WAIT_BARRIER();
  if (w >= 4) MX_BARRIER();
  read_a(0, lds0, 0, 8);
  read_sa(0, r0);
  take_sa(0);
  read_b(0, lds0 + OFF_B, r0);
  uint32_t cur = 0;
  auto slice = [&](auto fc, int s) {
    constexpr int F = decltype(fc)::value, G = F ^ 1;            // the half of b that is multiplied first (s % 2), and the other
    const uint32_t nxt = STAGEB - cur, a0 = lds0 + cur, b0 = a0 + OFF_B, na = lds0 + nxt, nb = na + OFF_B;
    turn_to(s + 2);
    MX_READS_DONE();
    take_sb(F);
    read_b(G, b0 + G * REGB, r0);
    MX_BARRIER();
    mma_quarter(0, F, [&](int x) { if (x < 3) read_a(1, a0 + REGA, x, x + 1); });
    MX_BARRIER();
    MX_READS_DONE();
    take_sb(G);
    read_a(1, a0 + REGA, 3, 6);
    read_sa(1, r0);
    copy_s(s + 2, r2);
    copy_a(0, s + 2, cur);
    MX_WAIT_BARRIER();
    mma_quarter(0, G, [&](int x) { if (x < 2) read_a(1, a0 + REGA, 6 + x, 7 + x); });
    MX_BARRIER();
    MX_READS_DONE();
    take_sa(1);
    read_a(0, na, 0, 3);
    read_sa(0, r1);
    copy_b(F, s + 2, cur);
    MX_WAIT_BARRIER();
    mma_quarter(1, G, [&](int x) { if (x < 3) read_a(0, na, 3 + x, 4 + x); });
    MX_BARRIER();
    MX_READS_DONE();
    take_sa(0);
    read_b(G, nb + G * REGB, r1);
    copy_b(G, s + 2, cur);
    copy_a(1, s + 2, cur);
    MX_WAIT_BARRIER();
    mma_quarter(1, F, [&](int x) { if (x < 2) read_a(0, na, 6 + x, 7 + x); });
    MX_BARRIER();
    cur = nxt;
    const uint32_t r = r0;
    r0 = r1;
    r1 = r2;
    r2 = r;
  };
  int s = 0;
#pragma unroll 1
  for (; s + 1 < cnt; s += 2) {
    slice(std::integral_constant<int, 0>{}, s);
    slice(std::integral_constant<int, 1>{}, s + 1);
  }
  if (s < cnt) slice(std::integral_constant<int, 0>{}, s);
  if (w < 4) MX_BARRIER();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // the last copies have landed before the workgroup gives its LDS back

  // the last sums are there: 16 passes of 4 cycles behind the last instruction at most, and nothing reads them before
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < ABLK; ++b)
#pragma unroll
      for (int j = 0; j < BBLK; ++j) asm volatile("" : "+v"(acc[i >> 1][i & 1][b][j]));
  // a lane's columns of a row of a quarter's 64 rows x 32 columns: 16 x 16: 8 g4 .. + 7 of row 4 c + block; 32 x 32: 16 g4 .. + 15 of row 4 (c % 16) +
  // 2 block + c / 16
  constexpr int COLS = B32 ? 16 : 8;
#pragma unroll
  for (int qm = 0; qm < 2; ++qm)
#pragma unroll
    for (int b = 0; b < ABLK; ++b) {
      const int64_t row = m0 + 128 * qm + 64 * wm + (B32 ? 4 * (c & 15) + 2 * b + (c >> 4) : 4 * c + b);
      if (row >= p.m) continue;
#pragma unroll
      for (int qn = 0; qn < 2; ++qn) {
        const int64_t col = n0 + 128 * qn + 32 * wn + COLS * g4;
        if (col >= p.n) continue;
        float v[COLS];
#pragma unroll
        for (int i = 0; i < COLS; ++i) v[i] = B32 ? acc[qm][qn][b][0][4 * (i & 3) + (i >> 2)] : acc[qm][qn][b][(i & 1) % BBLK][(i >> 1) & 3];
        mx_store<TO, COLS>(reinterpret_cast<TO *>(p.c) + row * p.ldc + col, v, p.n - col, p.vec, p.accumulate);
      }
    }
#undef MX_BARRIER
#undef MX_READS_DONE
#undef MX_WAIT_BARRIER
}

// ---- 128 x 128 tiles: four wavefronts of 64 x 64 outputs, two workgroups on a compute unit -------------------------------------
// For products of too few 256 x 256 tiles, and for fp32 results of 8-bit operands.  Two stages of LDS; the fragments of slice s + 1 are read
// among the matrix instructions of slice s, into the other of two sets of registers.  One barrier a slice: a wavefront passes it when its
// reads of slice s are in registers, so the stage of slice s may be written again (by the copies of slice s + 2, which go out next), and when
// its own copies of slice s + 1 have landed, so that slice may be read.  What a workgroup waits for the other one of the compute unit fills:
// with four stages and one workgroup 2048 x 4096 x 8192 took 79 us in 8 bits and 58 in 4, with two and two it takes 58 and 40.
// Bound by LDS: a slice moves 34 KB into it and 72 KB out of it for 512 cycles of matrix instructions a SIMD; 2048 x 4096 x 8192 runs at 2.4
// (8 bits) and 3.4 PFLOP/s.  WIDE: by the bf16 matrix instructions, 1024 cycles of a slice a SIMD and workgroup, and the conversions, some 700 of
// the vector ALU beside them; 8192 x 1024 x 8192 117 us, 1.17 PFLOP/s (a bf16 product of the library's 1.3 to 1.4).
// Both operands' slots hold row 64 (s / 64) + 4 (s % 16) + s / 16 % 4 in blocks of 16 x 16 (four blocks' scales are one dword), 64 (s / 64) +
// 4 (s % 16) + 2 (s / 32 % 2) + s / 16 % 2 in blocks of 32 x 32 (scales as cells, taken apart behind the wait, as in mx_w8_kernel).
template <int FA, int FB, bool WIDE, typename TO>
__global__ void __launch_bounds__(256, 2) mx_t128_kernel(const MxGemmParams p) {
  constexpr int KS = FA == 4 && FB == 4 ? 2 : 1;
  constexpr int RA = KS * MxBytes<FA>::STEP, RB = KS * MxBytes<FB>::STEP, NA = RA / 64, NB = RB / 64;
  constexpr uint32_t REGA = 128 * RA, REGB = 128 * RB, OFF_S = REGA + REGB, STAGEB = OFF_S + KS * 1024;
  constexpr bool B32 = KS == 2;                                  // in blocks of 32 x 32 x 64, as in mx_w8_kernel; else 16 x 16 x 128
  constexpr int SIDE = B32 ? 32 : 16, BLK = 64 / SIDE, APART = B32 ? 4 : NA, BPART = B32 ? 4 : NB;
  using Acc = std::conditional_t<B32, floatx16, floatx4>;
  constexpr int STAGES = 2, COPIES = KS + 2 * NA + 2 * NB;      // of a wavefront a slice
  __shared__ __attribute__((aligned(1024))) unsigned char smem[STAGES * STAGEB];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w >> 1, wn = w & 1;
  const int c = lane & (SIDE - 1), g4 = lane / SIDE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
  const uint32_t lda = (uint32_t)p.steps * MxBytes<FA>::STEP, ldb = (uint32_t)p.steps * MxBytes<FB>::STEP;
  auto row_of = [](int s) { return (uint32_t)(64 * (s >> 6) + 4 * (s & 15) + (B32 ? 2 * ((s >> 5) & 1) + ((s >> 4) & 1) : (s >> 4) & 3)); };   // of a slot
  uint32_t ca[2 * NA], cb[2 * NB];
#pragma unroll
  for (int x = 0; x < 2 * NA; ++x) {
    const int s = NA == 2 ? 8 * (4 * w + x) + (lane >> 3) : 16 * (2 * w + x) + (lane >> 2);
    const int chunk = NA == 2 ? (lane & 7) ^ mx_turn8(s) : (lane & 3) ^ mx_turn4(s);
    ca[x] = row_of(s) * lda + (uint32_t)(chunk * 16);
  }
#pragma unroll
  for (int x = 0; x < 2 * NB; ++x) {
    const int s = NB == 2 ? 8 * (4 * w + x) + (lane >> 3) : 16 * (2 * w + x) + (lane >> 2);
    const int chunk = NB == 2 ? (lane & 7) ^ mx_turn8(s) : (lane & 3) ^ mx_turn4(s);
    cb[x] = row_of(s) * ldb + (uint32_t)(chunk * 16);
  }
  // chunk of a block's first read; the next: 32 x 32 and bf16 (a lane takes block g4) the next chunk, else 4 chunks on
  constexpr uint32_t NEXT = B32 || WIDE ? 16 : 64;
  const int q0 = B32 ? 4 * g4 : g4;
  const uint32_t qa = NA == 2 ? (WIDE ? 2 * g4 : q0) ^ mx_turn8(c) : g4 ^ mx_turn4(c), qb = NB == 2 ? (WIDE ? 2 * g4 : q0) ^ mx_turn8(c) : g4 ^ mx_turn4(c);
  const uint32_t fa_lane = (uint32_t)((wm * 64 + c) * RA) + qa * 16;
  const uint32_t fb_lane = REGA + (uint32_t)((wn * 64 + c) * RB) + qb * 16;
  // scales of a slice: [step][a's 512 bytes, b's]
  const uint32_t s_lane = OFF_S + (uint32_t)((c & 15) * 16) + (uint32_t)(B32 ? g4 * 1024 : g4 * 4);
  const uint32_t sa_lane = s_lane + (uint32_t)(wm * 256), sb_lane = s_lane + (uint32_t)(512 + wn * 256);
  typedef __attribute__((address_space(3))) const int4v *lds_chunk;
  typedef __attribute__((address_space(3))) const uint32_t *lds_dword;

  const int pid = gg_xcd_chunk((int)blockIdx.x, p.tiles_m * p.tiles_n), piece = blockIdx.y;
  int tm, tn;
  gg_tile_of(pid, p.tiles_m, p.tiles_n, tm, tn);
  const int nsl = (p.steps + KS - 1) / KS;
  const int s0 = (int)((int64_t)piece * nsl / p.pieces), cnt = (int)((int64_t)(piece + 1) * nsl / p.pieces) - s0;
  const int64_t m0 = (int64_t)tm * 128, n0 = (int64_t)tn * 128;
  int4v rsa = raw_rsrc(p.a + m0 * lda, std::min<int64_t>(p.m - m0, 128) * lda), rsb = raw_rsrc(p.b + n0 * ldb, std::min<int64_t>(p.n - n0, 128) * ldb);
  // a wavefront copies scales of one operand: 256 bytes of a step
  const bool of_b = w >= 2;
  int4v rss = raw_rsrc(of_b ? p.bs + n0 * 4 : p.as + m0 * 4, of_b ? (int64_t)p.steps * p.cells_b * 16 - n0 * 4 : (int64_t)p.steps * p.cells_a * 16 - m0 * 4);
  const uint32_t gs = (uint32_t)__builtin_amdgcn_readfirstlane((int)((of_b ? p.cells_b : p.cells_a) * 16));
  asm volatile("s_nop 4" : "+s"(rsa), "+s"(rsb), "+s"(rss));
  auto turn_to = [&](int s) {
    if (s >= cnt) {
      rsa[2] = rsb[2] = rss[2] = 0;
    } else if (KS == 2 && (p.steps & 1) && s0 + s == nsl - 1) {      // chunks 4..7 are not there
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int ch = (lane & 7) ^ mx_turn8(8 * (4 * w + x) + (lane >> 3));
        if (ch >= 4) ca[x % (2 * NA)] = cb[x % (2 * NB)] = 0x80000000u;
      }
    }
  };
  auto copy = [&](int s, uint32_t stage) {
    const uint32_t at = lds0 + stage;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      copy_256((uint32_t)(lane * 4), rss, (uint32_t)(KS * (s0 + s) + ks) * gs + (uint32_t)(w & 1) * 256, at + OFF_S + (uint32_t)(ks * 1024 + w * 256));
#pragma unroll
    for (int x = 0; x < 2 * NA; ++x) copy_1k(ca[x], rsa, (uint32_t)(s0 + s) * RA, at + (uint32_t)(2 * NA * w + x) * 1024);
#pragma unroll
    for (int x = 0; x < 2 * NB; ++x) copy_1k(cb[x], rsb, (uint32_t)(s0 + s) * RB, at + REGA + (uint32_t)(2 * NB * w + x) * 1024);
  };
  Acc acc[BLK][BLK];
#pragma unroll
  for (int i = 0; i < BLK * BLK; ++i) acc[i / BLK][i % BLK] = Acc{};
  int4v fa[2][BLK][APART], fb[2][BLK][BPART];
  uint32_t sa[2], sb[2], na[2], nb[2];                           // this slice's scales, and (16 x 16) the next one's as they come
  int4v ca_next, cb_next;                                        // (32 x 32) the next one's cells
  constexpr int READS = 2 + BLK * APART + BLK * BPART;
  auto read = [&](int set, uint32_t at, int x) {                // read x of READS: the scales, then step by step what is multiplied first
    if (x == 0) {
      if constexpr (B32) ca_next = *(lds_chunk)(at + sa_lane);
      else na[0] = *(lds_dword)(at + sa_lane);
    } else if (x == 1) {
      if constexpr (B32) cb_next = *(lds_chunk)(at + sb_lane);
      else nb[0] = *(lds_dword)(at + sb_lane);
    } else if (x < 2 + BLK * BPART) {
      const int y = x - 2;
      fb[set][y % BLK][y / BLK] = *(lds_chunk)(at + (fb_lane ^ (uint32_t)(y / BLK) * NEXT) + (uint32_t)(y % BLK * SIDE * RB));
    } else if (x < READS) {
      const int y = x - 2 - BLK * BPART;
      fa[set][y % BLK][y / BLK] = *(lds_chunk)(at + (fa_lane ^ (uint32_t)(y / BLK) * NEXT) + (uint32_t)(y % BLK * SIDE * RA));
    }
  };
  uint32_t stage = 0;                                            // of slice s
  auto after = [&](uint32_t st) { return st == (STAGES - 1) * STAGEB ? 0u : st + STAGEB; };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    turn_to(s);
    copy(s, (uint32_t)s * STAGEB);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 2) * COPIES) : "memory");
#pragma unroll
  for (int x = 0; x < READS; ++x) read(0, lds0, x);
  turn_to(STAGES - 1);
  copy(STAGES - 1, (STAGES - 1) * STAGEB);
  auto slice = [&](auto set_, int s) {
    constexpr int SET = decltype(set_)::value;
    const uint32_t next = after(stage);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 2) * COPIES) : "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (B32) {
      mx_cell_rows2(sa, ca_next, (uint32_t)c >> 4);
      mx_cell_rows2(sb, cb_next, (uint32_t)c >> 4);
    } else {
      sa[0] = na[0];
      sb[0] = nb[0];
    }
    turn_to(s + STAGES);
    copy(s + STAGES, stage);
    if constexpr (WIDE) {
      MxWide<FB> wb[4];
#pragma unroll
      for (int nj = 0; nj < 4; ++nj) {
        MxFrag<FB> f;
#pragma unroll
        for (int i = 0; i < NB; ++i) f.q[i] = fb[SET][nj][i];
        wb[nj] = mx_wide<FB>(f, mx_scale_value(sb[0] >> (8 * nj) & 0xffu));
      }
#pragma unroll
      for (int mi = 0; mi < 4; ++mi) {
        MxFrag<FA> f;
#pragma unroll
        for (int i = 0; i < NA; ++i) f.q[i] = fa[SET][mi][i];
        const MxWide<FA> wa = mx_wide<FA>(f, mx_scale_value(sa[0] >> (8 * mi) & 0xffu));
        constexpr int PER = (READS + 3) / 4;                     // with all reads before the conversions 4 % slower
#pragma unroll
        for (int y = 0; y < PER; ++y) read(SET ^ 1, lds0 + next, PER * mi + y);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int nj = 0; nj < 4; ++nj) acc[mi][nj] = Mma<bf16_t>::mma16(wb[nj].v[t], wa.v[t], acc[mi][nj]);
      }
      stage = next;
      return;
    }
    // two wait states between what put the scales into their registers and the first product: the compiler keeps none for assembly
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      if constexpr (B32) {
        const int t = x >> 2, bm = (x >> 1) & 1, bn = x & 1;
#define MX_SEL(j, i, k) if (t == j && bm == i && bn == k) mx_mma32_tied<2 * (j & 1) + k, 2 * (j & 1) + i>(fb[SET][bn][t], sb[t >> 1], fa[SET][bm][t], sa[t >> 1], acc[bm][bn])
#define MX_SEL4(j) MX_SEL(j, 0, 0); MX_SEL(j, 0, 1); MX_SEL(j, 1, 0); MX_SEL(j, 1, 1)
        MX_SEL4(0); MX_SEL4(1); MX_SEL4(2); MX_SEL4(3);
#undef MX_SEL4
#undef MX_SEL
      } else {
        const int mi = x >> 2, nj = x & 3;
        const auto vb = mx_narrow<FB>(fb[SET][nj], 0);
        const auto va = mx_narrow<FA>(fa[SET][mi], 0);
        floatx4 &sum = acc[mi][nj];
#define MX_SEL(j, i) if (nj == j && mi == i) mx_mma_tied<FA, FB, j, i>(vb, sb[0], va, sa[0], sum)
        MX_SEL(0, 0); MX_SEL(0, 1); MX_SEL(0, 2); MX_SEL(0, 3);
        MX_SEL(1, 0); MX_SEL(1, 1); MX_SEL(1, 2); MX_SEL(1, 3);
        MX_SEL(2, 0); MX_SEL(2, 1); MX_SEL(2, 2); MX_SEL(2, 3);
        MX_SEL(3, 0); MX_SEL(3, 1); MX_SEL(3, 2); MX_SEL(3, 3);
#undef MX_SEL
      }
      __builtin_amdgcn_sched_barrier(0);
      constexpr int PER = (READS + 15) / 16;
#pragma unroll
      for (int y = 0; y < PER; ++y) read(SET ^ 1, lds0 + next, PER * x + y);
      __builtin_amdgcn_sched_barrier(0);
    }
    stage = next;
  };
  int s = 0;
#pragma unroll 1
  for (; s + 1 < cnt; s += 2) {
    slice(std::integral_constant<int, 0>{}, s);
    slice(std::integral_constant<int, 1>{}, s + 1);
  }
  if (s < cnt) slice(std::integral_constant<int, 0>{}, s);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // the last copies have landed before LDS is used again,
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");             // and the last sums are there
#pragma unroll
  for (int i = 0; i < BLK * BLK; ++i) asm volatile("" : "+v"(acc[i / BLK][i % BLK]));
  __syncthreads();
  // 32 rows of a wavefront's 64 at a time through LDS of its own, so that a store writes whole lines: a lane holds columns 16 g4 + 4 v + nj of
  // rows 4 c + mi, and stores 16 bytes of a row
  constexpr int PITCH = 68;
  float *mine = reinterpret_cast<float *>(smem) + w * 32 * PITCH;
  auto store = [&](auto *out, int64_t ld, int64_t cols, int vec, int accumulate) {
    using TS = std::remove_pointer_t<decltype(out)>;
    constexpr int E = 16 / (int)sizeof(TS), LPR = 64 / E;        // columns of a lane, lanes of a row
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if constexpr (B32) {
        // columns 32 x + 16 g4 + 4 v + .. of row 4 (c % 16) + 2 block + c / 16
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<floatx4 *>(mine + (2 * (c & 15) + (c >> 4)) * PITCH + 32 * (i >> 2) + 16 * g4 + 4 * (i & 3)) =
              floatx4{acc[half][0][i], acc[half][0][i + 8], acc[half][1][i], acc[half][1][i + 8]};
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const auto &s = acc[(2 * half + i) % BLK];
            *reinterpret_cast<floatx4 *>(mine + (2 * c + i) * PITCH + 16 * g4 + 4 * v) = floatx4{s[0][v], s[1 % BLK][v], s[2 % BLK][v], s[3 % BLK][v]};
          }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int it = 0; it < 32 * LPR / 64; ++it) {
        const int r = it * (64 / LPR) + lane / LPR, e = lane % LPR * E;
        const int64_t row = m0 + 64 * wm + 4 * (r >> 1) + 2 * half + (r & 1), col = n0 + 64 * wn + e;
        float v[E];
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          const floatx4 x = *reinterpret_cast<const floatx4 *>(mine + r * PITCH + e + 4 * q);
#pragma unroll
          for (int y = 0; y < 4; ++y) v[4 * q + y] = x[y];
        }
        if (row < p.m && col < cols) mx_store<TS, E>(out + row * ld + col, v, cols - col, vec, accumulate);
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (p.pieces > 1) store(p.ws + (int64_t)piece * p.m * (4 * p.cells_b), 4 * p.cells_b, 4 * p.cells_b, 1, 0);
  else store(reinterpret_cast<TO *>(p.c), p.ldc, p.n, p.vec, p.accumulate);
}

// c (+)= the pieces' sums, in order; a thread 4 columns.
template <typename TO> __global__ void __launch_bounds__(256) mx_join_kernel(const MxGemmParams p) {
  const int64_t groups = p.cells_b, u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= p.m * groups) return;
  const int64_t row = u / groups, col = u % groups * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int x = 0; x < p.pieces; ++x) {
    const floatx4 q = *reinterpret_cast<const floatx4 *>(p.ws + ((int64_t)x * p.m + row) * (4 * groups) + col);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += q[j];
  }
  mx_store<TO, 4>(reinterpret_cast<TO *>(p.c) + row * p.ldc + col, v, p.n - col, p.vec, p.accumulate);
}

// c = 0 where there is nothing to sum (k of 0).
template <typename TO> __global__ void __launch_bounds__(256) mx_zero_kernel(const MxGemmParams p) {
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < p.m * p.n; u += (int64_t)gridDim.x * 256)
    reinterpret_cast<TO *>(p.c)[u / p.n * p.ldc + u % p.n] = from_f<TO>(0.f);
}

constexpr int MX_MAX_PIECES = 16;

// Which kernel a product takes: `side` 256 is mx_w8_kernel, 128 mx_t128_kernel, 0 mx_direct_kernel with mt, nt and waves.  Measured on 1 to
// 8192 rows, widths of 512 to 8192 and k of 512 to 8192, in us for 8 x 8, 8 x 4 and 4 x 4 bits.
struct MxPlan { int side, mt, nt, waves, pieces; };
static bool mx_wide_needed(int fa, int fb, int out) { return out == DH_F32 && (fa == DH_MX_E4M3 || fb == DH_MX_E4M3); }
static MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int fa, int fb, int out) {
  const bool wide = mx_wide_needed(fa, fb, out), b4 = fb == DH_MX_E2M1;
  const int64_t steps = cdiv(k, 128);
  const int64_t big = cdiv(m, 256) * cdiv(n, 256), mid = cdiv(m, 128) * cdiv(n, 128);
  // Tokens of a few sequences.  32 columns a workgroup where that still fills the chip, else 16: 1 x 8192 x 3584 5.0 against 7.0 (8 x 4), 16 x
  // 7168 x 8192 11.1 against 14.0; but 8-bit weights, whose loads alone keep a compute unit busy, lose at 224 workgroups (13.5 against 17.8).
  MxPlan q{0, 1, 1, 8, 1};
  bool direct = m <= 16;
  if (direct) {
    if (cdiv(n, 32) >= (b4 ? 224 : 256)) q.nt = 2;
  } else if (m <= 32 || cdiv(m, 32) * cdiv(n, 32) <= 128) {
    // 24 x 8192 x 3584 9.4 / 8.1 / 6.5 against 11.3 / 10.7 / 9.5 in tiles of 32 x 64 and pieces of k; 65 x 1280 x 1024 4.7 / 4.5 / 4.4 against 7.6 / 7.1 / 6.6
    // in tiles of 128
    direct = true;
    q.mt = q.nt = 2;
  } else if (steps <= 32 && cdiv(m, 64) * cdiv(n, 32) <= 256) {
    // 512 x 512 x 512 5.1 / 5.0 / 4.5 against 6.2 / 6.0 / 5.8 in tiles of 128; past one workgroup a compute unit 1000 x 520 x 1999 13.9 / 15.4 / 9.5 against
    // 11.3 / 10.4 / 8.8, and at long k 64 x 7168 x 8192 26.7 / 22.9 / 16.5 against 20.0 / 17.1 / 16.4
    direct = true;
    q.mt = 4, q.nt = 2;
  } else if (wide && steps < 32 && mid < 128) {
    // 777 x 1001 x 2080 14 against 24.7 (15.5 by four wavefronts)
    direct = true;
    q.mt = q.nt = 4;
  }
  if (direct) {
    // k in pieces where few workgroups have long sums: 32 x 1280 x 8192 17.5 / 14.1 / 10.6 whole, 10.0 / 9.3 / 9.1 in up to 4 pieces
    const int64_t tiles = cdiv(m, 16 * q.mt) * cdiv(n, 16 * q.nt), units = b4 ? (steps + 1) / 2 : steps;
    if (tiles <= 64) q.pieces = (int)std::max<int64_t>(1, std::min<int64_t>({256 / tiles, units / (2 * q.waves), MX_MAX_PIECES}));
    return q;
  }
  // A round of the chip is 256 tiles of 256 x 256, or 512 of 128 x 128 in 0.6 of its time: 4096 x 7168 x 8192 (2 rounds and 4) 168 / 155 / 115 against
  // 204 / 176 / 124, 2048 x 4096 x 8192 (half a round and one) 73 / 69 / 59 against 58 / 55 / 40
  if (!wide && 5 * cdiv(big, 256) <= 3 * cdiv(mid, 512)) return {256, 0, 0, 8, 1};
  q = {128, 0, 0, 4, 1};
  // k in pieces, of 8 slices at least, while they have a compute unit each: 128 x 7168 x 8192 42 whole, 23 in four (8 x 8); 777 x 1001 x 2080 13.8 whole, 15.6
  // in two: the pieces' sums are written and read once more
  const int64_t slices = fa == DH_MX_E2M1 && b4 ? (steps + 1) / 2 : steps;
  // Two workgroups on a compute unit where what they save, 0.2 us a slice of a piece, pays for the further pieces' bytes, 3 us a hundred tiles: 2000 x 1024 x
  // 8192 34.3 in two, 32.9 in four, 300 x 4096 x 8192 29.5 and 25.8; but 2000 x 1024 x 4096 23.6 and 25.6, 512 x 7168 x 4096 24.9 whole and 30.7 in two
  auto pays = [&] { return mid * q.pieces <= 256 && 8 * slices >= mid * q.pieces * std::max(q.pieces, 2); };
  if (slices >= 24)
    while (q.pieces < MX_MAX_PIECES && slices >= 16 * q.pieces && (mid * q.pieces <= 128 || pays())) q.pieces *= 2;
  return q;
}

template <int FA, int FB, typename TO> static void mx_launch(MxGemmParams p, const MxPlan &q, hipStream_t st) {
  constexpr bool WIDE = sizeof(TO) == 4 && (FA == 8 || FB == 8);
  const int side_m = q.side ? q.side : 16 * q.mt, side_n = q.side ? q.side : 16 * q.nt;
  p.tiles_m = (int)cdiv(p.m, side_m);
  p.tiles_n = (int)cdiv(p.n, side_n);
  p.pieces = q.pieces;
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)q.pieces), block((unsigned)(64 * q.waves));
  if (q.side) {
    if constexpr (!WIDE) {
      if (q.side == 256) hipLaunchKernelGGL((mx_w8_kernel<FA, FB, TO>), grid, block, 0, st, p);
    }
    if (q.side == 128) hipLaunchKernelGGL((mx_t128_kernel<FA, FB, WIDE, TO>), grid, block, 0, st, p);
  }
#define MX_DIRECT(MT, NT, W) \
  if (!q.side && q.mt == MT && q.nt == NT && q.waves == W) hipLaunchKernelGGL((mx_direct_kernel<FA, FB, MT, NT, W, WIDE, TO>), grid, block, 0, st, p)
  MX_DIRECT(1, 1, 8);
  MX_DIRECT(1, 2, 8);
  MX_DIRECT(2, 2, 8);
  MX_DIRECT(4, 2, 8);
  if constexpr (WIDE) { MX_DIRECT(4, 4, 8); }
#undef MX_DIRECT
  if (q.pieces > 1) hipLaunchKernelGGL((mx_join_kernel<TO>), dim3((unsigned)cdiv(p.m * p.cells_b, 256)), dim3(256), 0, st, p);
}

}  // namespace dh

static int mx_gemm_sizes(int64_t m, int64_t n, int64_t k) {
  DH_CHECK(m >= 0 && n >= 0 && k >= 0, "m %lld, n %lld, k %lld", (long long)m, (long long)n, (long long)k);
  DH_CHECK(m < (1ll << 31) && n < (1ll << 31) && k <= (1ll << 22), "sizes: m %lld and n %lld < 2^31, k %lld <= 2^22", (long long)m, (long long)n,
           (long long)k);
  DH_CHECK(dh::cdiv(m, 16) * dh::cdiv(n, 16) < (1ll << 31), "more than 2^31 tiles");
  return DH_OK;
}

extern "C" size_t dh_mx_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k, int a_format, int b_format, int out_dtype) {
  if (m <= 0 || n <= 0 || k <= 0 || mx_gemm_sizes(m, n, k) != DH_OK) return 0;
  const dh::MxPlan q = dh::mx_plan(m, n, k, a_format, b_format, out_dtype);
  return q.pieces > 1 ? (size_t)q.pieces * (size_t)m * (size_t)dh::mx_rows4(n) * 4 : 0;
}

extern "C" int dh_mx_gemm_path(int64_t m, int64_t n, int64_t k, int a_format, int b_format, int out_dtype) {
  if (m <= 0 || n <= 0 || k <= 0 || mx_gemm_sizes(m, n, k) != DH_OK) return 0;
  const dh::MxPlan q = dh::mx_plan(m, n, k, a_format, b_format, out_dtype);
  return (q.side ? q.side : 10 * q.mt + q.nt) * 100 + q.pieces;
}

extern "C" int dh_mx_gemm_nt(const void *a_codes, const void *a_scales, int a_format, const void *b_codes, const void *b_scales, int b_format, void *c,
                             int64_t m, int64_t n, int64_t k, int64_t ldc, int out_dtype, int accumulate, void *workspace, size_t workspace_bytes,
                             void *stream) {
  using namespace dh;
  if (const int rc = mx_gemm_sizes(m, n, k)) return rc;
  DH_CHECK((a_format == DH_MX_E4M3 || a_format == DH_MX_E2M1) && (b_format == DH_MX_E4M3 || b_format == DH_MX_E2M1), "unknown format %d / %d", a_format,
           b_format);
  DH_CHECK(out_dtype == DH_F32 || out_dtype == DH_BF16 || out_dtype == DH_F16, "unknown dtype %d", out_dtype);
  if (m == 0 || n == 0) return DH_OK;
  DH_CHECK(c, "null pointer");
  DH_CHECK(ldc >= n || m == 1, "row stride %lld of %lld columns", (long long)ldc, (long long)n);
  MxGemmParams p{};
  p.c = c; p.m = m; p.n = n; p.ldc = ldc; p.accumulate = accumulate;
  const hipStream_t st = (hipStream_t)stream;
  if (k == 0) {
    if (!accumulate) {
      const dim3 grid((unsigned)std::min<int64_t>(cdiv(m * n, 256), 1 << 20));
      DH_DISPATCH_DTYPE(out_dtype, hipLaunchKernelGGL((mx_zero_kernel<T>), grid, dim3(256), 0, st, p));
      DH_LAUNCH_CHECK();
    }
    return DH_OK;
  }
  DH_CHECK(a_codes && a_scales && b_codes && b_scales, "null pointer");
  DH_CHECK(aligned16(a_codes) && aligned16(a_scales) && aligned16(b_codes) && aligned16(b_scales), "codes and scales must be 16-byte aligned");
  p.a = (const uint8_t *)a_codes; p.as = (const uint8_t *)a_scales; p.b = (const uint8_t *)b_codes; p.bs = (const uint8_t *)b_scales;
  p.cells_a = mx_rows4(m) / 4; p.cells_b = mx_rows4(n) / 4; p.steps = (int)cdiv(k, 128);
  p.vec = aligned16(c) && ldc * (int64_t)dtype_size(out_dtype) % 16 == 0;
  DH_CHECK(p.steps * std::max(p.cells_a, p.cells_b) * 16 < (1ll << 31), "scales of 2 GiB and more");
  const MxPlan q = mx_plan(m, n, k, a_format, b_format, out_dtype);
  // (a launch holds 2^32 - 1 threads a dimension; where k is split there are few tiles and a row's sums are joined by far fewer)
  const int64_t tiles = cdiv(m, q.side ? q.side : 16 * q.mt) * cdiv(n, q.side ? q.side : 16 * q.nt);
  DH_CHECK(tiles * 64 * q.waves < (1ll << 32), "%lld tiles are more than a launch takes: m %lld, n %lld", (long long)tiles, (long long)m, (long long)n);
  if (q.pieces > 1) {
    const size_t need = dh_mx_gemm_workspace_bytes(m, n, k, a_format, b_format, out_dtype);
    DH_CHECK(workspace && aligned16(workspace) && workspace_bytes >= need, "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    p.ws = (float *)workspace;
  }
#define MX_FORMATS(TO)                                                                  \
  if (a_format == DH_MX_E4M3 && b_format == DH_MX_E4M3) mx_launch<8, 8, TO>(p, q, st);  \
  else if (a_format == DH_MX_E4M3) mx_launch<8, 4, TO>(p, q, st);                       \
  else if (b_format == DH_MX_E4M3) mx_launch<4, 8, TO>(p, q, st);                       \
  else mx_launch<4, 4, TO>(p, q, st)
  DH_DISPATCH_DTYPE(out_dtype, MX_FORMATS(T));
#undef MX_FORMATS
  DH_LAUNCH_CHECK();
  return DH_OK;
}

// Linear read-out joined with its softmax cross-entropy (gncde_linear_cross_entropy, .._grad).
//
//   l_rv = sum_h x_rh W_vh + b_v,   lse_r = log sum_v exp l_rv,   loss_r = S_r lse_r - sum_v y_rv l_rv
//   dl_rv = g_r (S_r exp(l_rv - lse_r) - y_rv),   gx = dl W,   gW = dl^T x,   gb_v = sum_r dl_rv
//
// replacing log_softmax over materialised logits [rows, classes] (trainer_tgb.py:42-60) and its reverse mode.  The
// logits are never stored: the loss keeps, per row and tile of classes, the largest logit and the sum of exponentials
// relative to it; the gradient makes the logits once more, a piece of the classes at a time, and stores that piece's
// dl as a bf16 matrix operand.  All four products are one kernel, C^T = B A^T on v_mfma_f32_16x16x32_bf16 with fp32
// accumulation; where an operand's rows lie along the contraction it is read as it lies, and where they lie across it,
// LDS reads turn it, so one stored form of x, W and dl serves every product:
//
//   product   A (rows of the tile)     B (columns)          contraction   epilogue
//   logits    W       [classes, H]     x       [rows, H]    H             largest logit, sum of exponentials
//   logits    W piece [Vc, H]          x       [rows, H]    H             dl piece [rows, Vc]
//   gx        W piece, turned          dl      [rows, Vc]   Vc            fp32 sums / gx
//   gW        x, turned                dl, turned           rows          gW
//
// fp32 inputs are split into three bf16 parts each (8 bits of the significand a part, rounded to nearest: nothing is
// lost) and the six products above 2^-24 of |a||b| are summed, smallest first: fp32-class results on the bf16 matrix
// rate (16 times the fp32 one, so 2.7 times faster than fp32 MFMA at equal utilisation).
#include "gncde_internal.h"

#include <algorithm>
#include <type_traits>

namespace gncde {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int kPad = 64;  // packed contractions are padded to a multiple of this
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint16_t to_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float from_bf16(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// x = p0 + p1 + p2 in bf16 parts.  A finite x that would round to inf (above 3.39e38) is cut instead; an inf or NaN
// stays in p0 alone.
template <int NP>
__device__ __forceinline__ void split(float x, uint16_t (&p)[NP]) {
  p[0] = to_bf16(x);
  if (NP == 3) {
    if ((p[0] & 0x7f80) == 0x7f80 && (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u)
      p[0] = (uint16_t)(__float_as_uint(x) >> 16);
    const bool whole = (p[0] & 0x7f80) != 0x7f80;
    const float r1 = whole ? x - from_bf16(p[0]) : 0.f;
    p[NP > 1 ? 1 : 0] = NP > 1 ? to_bf16(r1) : p[0];
    const float r2 = r1 - from_bf16(p[NP > 1 ? 1 : 0]);
    p[NP > 2 ? 2 : 0] = NP > 2 ? to_bf16(r2) : p[0];
  }
}

// ---- logits far from zero ---------------------------------------------------------------------------------------
// A row's logits count relative to its largest before anything is rounded: loss = S log sum - sum y (l - top).  top + log sum
// and sum y l would each carry the rounding of a number of the logits' size: 3e-5 near 1000, where a row sure of its class
// has a loss of 1e-9.

// What logits are taken relative to: their largest, 0 where there is none.
__device__ __forceinline__ float reference(float top) { return top == -INFINITY ? 0.f : top; }

// exp(l - top), or exp(l - lse), as exp2(l by + off) rest, one fused product a logit: off is -top log2 e rounded, and rest,
// a factor of the whole row, what that rounding took from the exponent (the constant's own error meets l - top alone).  From
// 2^30 on, where off rounds by more than the exponential takes and ends past fp32's range, logits lie at least 64 apart:
// their difference as the exponent of two tells equal ones from smaller ones just as well.
struct Exponent {
  float by, off;
  __device__ __forceinline__ static bool far(float top) { return fabsf(top) >= 0x1p30f && fabsf(top) < INFINITY; }
  __device__ __forceinline__ explicit Exponent(float top) : by(far(top) ? 1.f : kLog2e), off(-top * by) {}
  __device__ __forceinline__ float rest(float top) const { return __builtin_amdgcn_exp2f(fmaf(-top, by, -off)); }
};

// The mass that goes with lse = top + log sum, as rounded, into the gradient: S exp(lse - (top + log sum)).  exp(l - lse) by
// itself has the rounding of a number of the logits' size: 6e-5 of a probability near 1000.
__device__ __forceinline__ float mass_beside(float lse, float top, float log_sum, float mass) {
  const float b = lse - top, lost = (top - (lse - b)) + (log_sum - b);  // exactly what the sum's rounding dropped
  return lost == lost ? mass * expf(-lost) : mass;
}

// sum y (l - top) relative to another logit, mass being sum y.
__device__ __forceinline__ float moved(float dot, float mass, float top, float to) {
  return mass == 0.f ? dot : fmaf(mass, reference(top) - to, dot);
}

// ---- targets and rows left out ----------------------------------------------------------------------------------
struct Rows {
  const void* target;
  const uint8_t* mask;
  int32_t kind;
};

__device__ __forceinline__ int64_t row_index(const Rows& r, int64_t n) {
  return r.kind == GNCDE_TARGET_INDEX32 ? (int64_t) static_cast<const int32_t*>(r.target)[n]
                                        : static_cast<const int64_t*>(r.target)[n];
}

__device__ __forceinline__ bool row_counts(const Rows& r, int64_t n) {
  if (r.mask && r.mask[n] == 0) return false;
  return r.kind == GNCDE_TARGET_ROWS || row_index(r, n) >= 0;
}

// ---- operand layout ---------------------------------------------------------------------------------------------
template <bool F32>
__device__ __forceinline__ float value(const void* p, int64_t i) {
  return F32 ? static_cast<const float*>(p)[i] : from_bf16(static_cast<const uint16_t*>(p)[i]);
}

// Values at p[i..i+3], zeros from `to` on.
template <bool F32>
__device__ __forceinline__ floatx4 four(const void* p, int64_t i, int64_t to) {
  typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));
  if (i + 4 <= to) {
    if (F32) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
      return floatx4{v[0], v[1], v[2], v[3]};
    }
    const u16x4u v = *reinterpret_cast<const u16x4u*>(static_cast<const uint16_t*>(p) + i);
    return floatx4{from_bf16(v[0]), from_bf16(v[1]), from_bf16(v[2]), from_bf16(v[3])};
  }
  floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (i + q < to) v[q] = value<F32>(p, i + q);
  return v;
}

// v to p[i..i+3], up to `to`.
template <bool F32>
__device__ __forceinline__ void put(void* p, int64_t i, int64_t to, floatx4 v) {
  typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));
  if (i + 4 <= to) {
    if (F32) *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = f32x4{v[0], v[1], v[2], v[3]};
    else
      *reinterpret_cast<u16x4u*>(static_cast<uint16_t*>(p) + i) =
          u16x4u{to_bf16(v[0]), to_bf16(v[1]), to_bf16(v[2]), to_bf16(v[3])};
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (i + q < to) {
      if (F32) static_cast<float*>(p)[i + q] = v[q];
      else static_cast<uint16_t*>(p)[i + q] = to_bf16(v[q]);
    }
}

// Packed operands: rows of Kp values (zeros behind the contraction), or for three parts rows of 3 Kp with 32 values of
// each part side by side: value k of part q at (k / 32) * 96 + q * 32 + k % 32.
template <int NP>
__device__ __forceinline__ int64_t packed(int64_t k, int q) {
  return NP == 1 ? k : (k >> 5) * 96 + q * 32 + (k & 31);
}

// The scale of dl: the largest |g| of the rows that count (1 where that is no use).  bf16 dl is stored over it, so that
// the equal cotangents of a mean leave the target's entry, nearly all of dl, near -1 and not at a rounded -g: the
// gradients' error is then that of their own rounding (2e-3 instead of 3e-3 of the norm at 8192 rows).  256 threads.
__device__ __forceinline__ void largest_cotangent(int64_t N, const Rows& rows, const float* __restrict__ g,
                                                  float* __restrict__ scale) {
  __shared__ float red[4];
  float m = 0.f;
  for (int64_t n0 = threadIdx.x; n0 < N; n0 += 2048) {
    float v[8];
    bool in[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // side by side: one wait for all
      const int64_t n = n0 + 256 * i < N ? n0 + 256 * i : n0;
      v[i] = fabsf(g[n]);
      in[i] = !rows.mask || rows.mask[n] != 0;
      if (rows.kind != GNCDE_TARGET_ROWS) in[i] &= row_index(rows, n) >= 0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, in[i] ? v[i] : 0.f);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (threadIdx.x == 0) *scale = m > 1e-30f && m < 1e30f ? m : 1.f;
}

// src [R, H] -> packed [R][Kp]; with `left`, rows left out are zeros, whatever they hold.
struct PackJob {
  const void* src;
  uint16_t* dst;
  int64_t R;
  int32_t left;
  uint32_t blocks;
};

// x and W in one launch, either may have no blocks.  With `scale`, one workgroup more in front finds that.
template <bool F32, int NP>
__global__ void __launch_bounds__(256) k_xent_pack(PackJob x, PackJob w, int H, int Kp, Rows rows, int64_t N,
                                                   const float* __restrict__ g, float* __restrict__ scale) {
  if (scale && blockIdx.x == 0) {
    largest_cotangent(N, rows, g, scale);
    return;
  }
  const uint32_t at = blockIdx.x - (scale ? 1 : 0);
  const bool is_x = at < x.blocks;
  const int64_t block = is_x ? at : at - x.blocks, blocks = is_x ? x.blocks : w.blocks, R = is_x ? x.R : w.R;
  const void* src = is_x ? x.src : w.src;
  uint16_t* dst = is_x ? x.dst : w.dst;
  const bool left = is_x ? x.left != 0 : w.left != 0;
  const int cpr = Kp / 8;
  for (int64_t e = block * 256 + threadIdx.x; e < R * cpr; e += blocks * 256) {
    const int64_t r = e / cpr;
    const int h0 = (int)(e - r * cpr) * 8;
    const bool keep = !left || row_counts(rows, r);
    u16x8 o[NP];
    floatx4 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] = keep && h0 + 4 * i < H ? four<F32>(src, r * H + h0 + 4 * i, r * H + H) : floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint16_t p[NP];
      split<NP>(v[i >> 2][i & 3], p);
#pragma unroll
      for (int q = 0; q < NP; ++q) o[q][i] = p[q];
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) *reinterpret_cast<u16x8*>(dst + r * NP * Kp + packed<NP>(h0, q)) = o[q];
  }
}

// ---- the product ------------------------------------------------------------------------------------------------
enum { E_LSE = 0, E_DL = 1, E_GX = 2, E_GW = 3 };
constexpr int kLeftOut = -2;

// A row's target within the piece (-1: none there; kLeftOut) and whether its logits are far, in one word.
__device__ __forceinline__ float row_word(int target, bool far) { return __int_as_float((target + 2) | (far ? 1 << 30 : 0)); }
__device__ __forceinline__ int word_target(float w) { return (__float_as_int(w) & ~(1 << 30)) - 2; }
__device__ __forceinline__ bool word_far(float w) { return __float_as_int(w) & (1 << 30); }

struct GemmArgs {
  const uint16_t* A;
  const uint16_t* B;
  int64_t lda, ldb;          // row strides in values (of packed rows: of all parts); dl has none
  int64_t M, N;              // rows of A and of B
  int K;                     // contraction: a multiple of 8 of the logits, the rows of turned operands
  int kt;                    // steps over K
  int per_split, splits;     // steps a workgroup of one split takes
  int64_t tm, tn;            // tiles
  // logits
  Rows rows;
  const void* bias;          // this piece's
  int64_t v0, V;             // first class of the piece, classes in all
  float2* part;              // E_LSE: [N][part_ld] (largest, sum of exponentials), this launch's tiles from part_at
  float2* part_y;            // E_LSE, label rows: likewise (sum y (l - largest), sum y)
  int64_t part_ld, part_at;
  float* hit;                // E_LSE, indices: [N] the target's logit
  const float* stats;        // E_DL
  const float* g;
  const float* scale;        // E_DL: dl is stored over it; E_GX, E_GW: the result is multiplied by it (may be NULL: 1)
  uint16_t* P;               // E_DL: [class / 32][block][part][32], classes zero-padded to mp
  int64_t mp;
  int64_t block;             // rows of a block of dl, the rows of x or more
  float* part_b;             // E_DL: [tn * WN][M] sums over this tile's rows of dl (may be NULL)
  // products
  void* out;                 // [N][ldo]
  float* acc;                // fp32 [split][N][lda_c]; NULL: write `out`
  int64_t ldo, ldacc;
  int32_t add;               // acc += instead of =
};

// One tile of C^T.  A step brings S::K values of every row of A and B into LDS: for one part 64 values, for three parts
// 32 of each part, which lie side by side in the packed operands; of a turned operand as many of its rows, the tile wide.
// Two LDS buffers; a wave's fragments are read one half-step (one part: a third of the products) before they are
// multiplied, and the barrier that hands a buffer over lies between two runs of products whose fragments are in registers
// already.  Workgroups stay for all their tiles, and the next tile's first operands are on their way while this one's
// products are put out.
//
// Tiles of 256 x 256 (three parts: 256 x 128), eight waves of 128 x 64 (64 x 64) each: what a step reads from LDS and
// brings there (256 KB at 128 bytes a cycle) takes as long as its products, so smaller tiles are bound by LDS; four waves
// of 128 x 128 read a third less and were slower, with nothing to run while one waits.  128 x 128 tiles, two workgroups a
// CU, and 128 x 64 ones (the logits) serve where larger ones leave CUs idle.
//
// Measured at 8192 x 4096 x 131072 bf16 (8.8 TFLOP a product): logits of the loss 6.6 ms (1.33 PFLOP/s), dl 6.9 (1.28),
// gx 6.6 (1.33), gW 7.5 (1.18), where a library product of such operands reaches 1.4 to 1.6 and, turned as gW's are,
// 0.94.  The logits are bound by power: their matrix units are busy 70 % of the cycles, and the clock falls to 1.65 GHz.
// The turned products wait for their operands, two LDS reads a fragment instead of one; gW's, with both turned, takes all 256
// registers and is the one kernel here with scratch (two registers, written and read once a tile, outside the loop over
// steps).  Turning W, x and dl in memory instead cost 0.5 ms of copies and 0.8 ms for dl's second form here, a tenth of the
// gradient at 1021 x 333 x 50021.
//
// The one-part products with turned operands (gx, gW) take steps of half that and four buffers (DEEP): their loads are
// then two to three steps on their way instead of one, and a hand-over leaves those of two steps there (gW 8.6 -> 7.5 ms,
// gx 7.5 -> 6.6).  dl lies in blocks of 32 classes for that, [class / 32][row][part][32]: a step's rows of it are one run
// of memory.  The logits' operands lie as their rows do and would be read in pieces of half a cache line (7.1 -> 7.6 ms).
template <int NP, bool DEEP>
struct Step {
  static constexpr int K = NP == 1 && !DEEP ? 64 : 32;  // contraction a step
  static constexpr int ROW = K * NP;              // values a row in LDS
  static constexpr int CH = ROW / 8;              // 16-byte chunks a row
  // A row's chunk c lies at place(c, row): rows that one LDS cycle reads together then differ in bank.
  static __device__ __forceinline__ int place(int c, int row) {
    return NP == 1 ? (DEEP ? c ^ (-(row >> 2) & 3) : c ^ (row & 7)) : (c & ~3) | ((c & 3) ^ ((row >> 1) & 3));
  }
  // A turned operand's step is K rows of the tile's width times NP values.  Its row k's chunk c lies at c ^ turn(k): the
  // eight rows that one LDS cycle reads 32 bytes each of then cover all banks.
  static __device__ __forceinline__ int turn(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) << 1; }
  // dl's, in blocks of 32 columns: [block][row][32 values of every part].
  static __device__ __forceinline__ int turn_dl(int k) { return ((k >> 3) & 1) << 1; }
};

// Lane l of 16 hands in the address of four values of row l / 4 and gets value l of the four rows' 16.
__device__ __forceinline__ u16x4 read_tr(const uint16_t* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)const_cast<uint16_t*>(p)));
}

// A barrier for what went through LDS alone: stores to memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The order within a half-step of MMS products: an LDS read behind every product or two, and the LOADS loads of the
// step after next behind them, or in front (EARLY): that hides more of their latency and is 4 % on the logits' products
// (8192 x 4096 x 131072), but of turned operands, with twice the reads, it is 3 to 40 % slower.
template <int MMS, int READS, int LOADS, bool EARLY>
__device__ __forceinline__ void interleave() {
  constexpr int PER = LOADS > 0 || MMS < 2 * READS ? 1 : 2;
  constexpr int LATER = MMS >= READS + 2 * LOADS && !EARLY ? 2 : 1;
  if constexpr (EARLY) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  if constexpr (!EARLY) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, LATER, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
  }
  __builtin_amdgcn_sched_group_barrier(0x008, MMS, 0);
}

// The sum over each run of 16 lanes, in all of them (lane exchanges within the run: pairs, quads, halves, mirror).
__device__ __forceinline__ float sum16(float x) {
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xb1, 0xf, 0xf, true));
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4e, 0xf, 0xf, true));
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xf, 0xf, true));
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xf, 0xf, true));
  return x;
}

// A value of the lane's own that the compiler takes for new: what follows from it is worked out again for every tile and
// does not stay in registers over the products.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// LDS of k_xent_mm, in 16-bit values: two buffers of a step, the second one shared with the staged dl; the rows' and the
// classes' data, twice.
template <int BM, int BN, int EPI, int NP>
struct Space {
  static constexpr bool DEEP = EPI >= E_GX && NP == 1;
  static constexpr int TILE = (BM + BN) * Step<NP, DEEP>::ROW;
  static constexpr int PAD = 16;  // values a staged row of dl is longer
  // dl is staged beside the first buffer, which already takes the next tile: in two halves where one does not fit
  static constexpr int HALVES = BM + BN >= 512 ? 2 : 1;
  static constexpr int STAGE = EPI != E_DL ? 0 : BN / HALVES * (BM + PAD);
  static constexpr int HALF = (DEEP ? 2 : 1) * TILE;  // of the buffers
  static constexpr int BUFS = (HALF + (HALF > STAGE ? HALF : STAGE) + 7) / 8 * 8;
  static constexpr int INFO = EPI >= E_GX ? 0 : BN, BIAS = EPI >= E_GX ? 0 : BM;
  static constexpr int ALL = BUFS + 2 * INFO * 8 + 2 * BIAS * 2;
};

// Tiles `first`, `first` + `step`, ... of a product.  SOFT: the targets are label rows.
template <int BM, int BN, int WM, int WN, int EPI, int NP, bool F32, bool SOFT>
__device__ __forceinline__ void mm_tiles(const GemmArgs& a, uint16_t* lds, const uint32_t first, const uint32_t step) {
  typedef Space<BM, BN, EPI, NP> L;
  constexpr bool DEEP = L::DEEP;
  typedef Step<NP, DEEP> S;
  constexpr int NW = WM * WN, RT = BM / WM / 16, CT = BN / WN / 16;
  constexpr int IA = BM * S::CH / 64 / NW, IT = IA + BN * S::CH / 64 / NW;  // 1 KB loads a wave: A's, then B's
  constexpr bool OUT = EPI == E_GX || EPI == E_GW;
  constexpr bool TA = OUT, TB = EPI == E_GW;  // turned operands
  static_assert(RT % 4 == 0 && IA * 64 * NW == BM * S::CH && IT * 64 * NW == (BM + BN) * S::CH,
                "chunks divide over the waves");
  constexpr int TILE = L::TILE, PAD = L::PAD, HALVES = L::HALVES, BUFS = L::BUFS, INFO = L::INFO, BIAS = L::BIAS;
  uint16_t* const stage = lds + L::HALF;
  // What the logits' epilogues need of a row of x: lse's exponent, g over the scale, the same times the mass and the
  // exponent's rest, and the row's word.  Fetched with the tile's first operands, one tile ahead.
  floatx4* const info = reinterpret_cast<floatx4*>(lds + BUFS);
  float* const bias = reinterpret_cast<float*>(lds + BUFS + 2 * INFO * 8);  // of the tile's classes, likewise
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const uint32_t all = (uint32_t)(a.tm * a.tn) * (uint32_t)a.splits;

  // The tile in hand, and what its loads need: this lane's chunks of a step as byte offsets from the tile's first row of
  // A or B (rows behind the last read the last one's values: their results are never written), and buffer descriptors of
  // the tile's rows; a load behind the last step goes through one of no bytes and reads nothing.
  int64_t m0, n0;
  int tile_m, tile_n, split_k, k_from, k_to;
  uint32_t off[IT];
  const int col = ((lane & 7) ^ (lane >> 3)) * 8;  // one part: first value of all of them within the step
  const uint16_t *base_a, *base_b;
  auto place_of = [&](int i, int lane) {  // this lane's chunk of the buffer
    return i < IA ? (wave * IA + i) * 64 + lane : BM * S::CH + (wave * (IT - IA) + i - IA) * 64 + lane;
  };
  auto turned_row = [&](int i, int lane) {  // a turned operand's: its row of the step
    return i < IA ? place_of(i, lane) / (BM * NP / 8) : (place_of(i, lane) - BM * S::CH) / S::CH % 32;
  };
  // Tile `bid`: consecutive workgroups go round the eight XCDs, so each XCD takes a run of the order: split by split, and
  // within one in blocks of eight tiles of A by all of B.  What an XCD reads at a time stays in its cache.
  auto take = [&](uint32_t bid) {
    const uint32_t nt = (uint32_t)(a.tm * a.tn), tn = (uint32_t)a.tn;
    const uint32_t q = all >> 3, r = all & 7, xcd = bid & 7;
    uint32_t lin = xcd * q + (xcd < r ? xcd : r) + (bid >> 3);
    const uint32_t sp = lin / nt;
    lin -= sp * nt;
    const uint32_t grp = lin / (8 * tn), in = lin - grp * 8 * tn;
    const uint32_t left = (uint32_t)a.tm - grp * 8, gm = left < 8 ? left : 8;
    tile_m = __builtin_amdgcn_readfirstlane((int)(grp * 8 + in % gm));
    tile_n = __builtin_amdgcn_readfirstlane((int)(in / gm));
    split_k = __builtin_amdgcn_readfirstlane((int)sp);
    m0 = (int64_t)tile_m * BM, n0 = (int64_t)tile_n * BN;
    const int lane = fresh(threadIdx.x) & 63;
    const int most_a = (int)(a.M - m0 < BM ? a.M - m0 : BM) - 1, most_b = (int)(a.N - n0 < BN ? a.N - n0 : BN) - 1;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int slot = place_of(i, lane), row = slot / S::CH;
      if (i < IA && TA) {
        const int k = turned_row(i, lane);
        const int c = (slot - k * (BM * NP / 8)) ^ S::turn(k);
        off[i] = ((uint32_t)k * (uint32_t)a.lda + c * 8) * 2u;
        continue;
      }
      if (i >= IA && TB) {
        const int at = slot - BM * S::CH, block = at / (32 * S::CH), k = turned_row(i, lane);
        const int c = (at % S::CH) ^ S::turn_dl(k);
        off[i] = (((uint32_t)block * (uint32_t)a.block + k) * (uint32_t)S::ROW + c * 8) * 2u;
        continue;
      }
      const int c = S::place(slot - row * S::CH, row);  // place() is its own inverse
      const int rr = i < IA ? row : row - BM, most = i < IA ? most_a : most_b;
      off[i] = ((uint32_t)(rr < most ? rr : most) * (uint32_t)(i < IA ? a.lda : OUT ? S::ROW : a.ldb) + c * 8) * 2u;
    }
    k_from = split_k * a.per_split;
    k_to = k_from + a.per_split < a.kt ? k_from + a.per_split : a.kt;
    base_a = a.A + m0 * (TA ? NP : a.lda);
    base_b = a.B + n0 * (TB ? a.block * NP : OUT ? S::ROW : a.ldb);
  };

  auto load = [&](int k, int buf) {
    const int bytes = __builtin_amdgcn_readfirstlane((k - k_to) >> 31);  // all of 2^32, or none
    __amdgpu_buffer_rsrc_t ra, rb;
    if constexpr (TA) {  // the step's rows that there are, to the end of the last one
      const int64_t left = (int64_t)a.K - (int64_t)k * S::K, rows = left < S::K ? left : S::K;
      const int64_t all = (rows * a.lda - m0 * NP) * 2;
      const int some = k < k_to && all > 0 ? (int)all : 0;
      ra = __builtin_amdgcn_make_buffer_rsrc((void*)(base_a + (int64_t)k * S::K * a.lda), 0,
                                             __builtin_amdgcn_readfirstlane(some), 0x00020000);
    } else {
      ra = __builtin_amdgcn_make_buffer_rsrc((void*)base_a, 0, bytes, 0x00020000);
    }
    if constexpr (TB) {  // to the end of dl
      const int64_t all = ((((a.N + 63) / 64 * 64 - n0) / 32) * a.block - (int64_t)k * 32) * S::ROW * 2;
      const int64_t most = all < 0xffffffffll ? all : 0xffffffffll;
      rb = __builtin_amdgcn_make_buffer_rsrc((void*)(base_b + (int64_t)k * 32 * S::ROW), 0,
                                             __builtin_amdgcn_readfirstlane(k < k_to ? (int)(uint32_t)most : 0), 0x00020000);
    } else if constexpr (OUT) {
      rb = __builtin_amdgcn_make_buffer_rsrc((void*)(base_b + (int64_t)k * a.block * S::ROW), 0, bytes, 0x00020000);
    } else {
      rb = __builtin_amdgcn_make_buffer_rsrc((void*)base_b, 0, bytes, 0x00020000);
    }
    const uint32_t at = (uint32_t)k * (S::ROW * 2);
    // of a ragged last step's chunks behind the end, one that is there: zeroed below
    const uint32_t behind = k * S::K + col >= a.K ? (uint32_t)col * 2u : 0u;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      uint32_t o = off[i];
      if (NP == 1 && !OUT) o -= behind;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          i < IA ? ra : rb, (__attribute__((address_space(3))) void*)(lds + buf * TILE + place_of(i, 0) * 8), 16, o,
          OUT ? 0 : at, 0, 0);
    }
  };
  // The rows of x that the tile in hand has, into info[at].
  auto fetch_rows = [&](int at) {
    if constexpr (!OUT) {
      if (a.bias)
        for (int r = fresh(threadIdx.x); r < BM; r += NW * 64)
          bias[at * BIAS + r] = m0 + r < a.M ? value<F32>(a.bias, m0 + r) : 0.f;
      for (int r = fresh(threadIdx.x); r < BN; r += NW * 64) {
        const int64_t n = n0 + r < a.N ? n0 + r : a.N - 1;
        const bool kept = !a.rows.mask || a.rows.mask[n] != 0;
        const int64_t c = SOFT ? 0 : row_index(a.rows, n);
        floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
        if (EPI == E_DL) {
          const float lse = a.stats[2 * n], mass = a.stats[2 * n + 1];
          const float gv = a.g[n] / (a.scale ? *a.scale : 1.f);
          const Exponent e(lse);
          v = floatx4{e.off, gv, gv * mass * e.rest(lse), lse};
        }
        const bool in = n0 + r < a.N && kept && c >= 0;
        const int64_t t = c - a.v0;
        if (!in) v = floatx4{0.f, 0.f, 0.f, 0.f};
        v[3] = row_word(!in ? kLeftOut : !SOFT && t >= 0 && t < a.M ? (int)t : -1, Exponent::far(v[3]));
        info[at * INFO + r] = v;
      }
    }
  };
  // The buffer of step k is complete for every wave, and everybody has read the other one.
  auto hand_over = [&](int k, int buf, auto on_their_way) {
    constexpr int LEFT = decltype(on_their_way)::value;  // newer loads, which stay on their way
    static_assert(LEFT < 16, "fits the count's low bits");
    __builtin_amdgcn_s_waitcnt(0x0070 | LEFT);  // vmcnt(LEFT) lgkmcnt(0)
    if ((NP == 1 || TA || TB) && (k + 1) * S::K > a.K) {  // what lies behind the contraction's end
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const bool turned = i < IA ? TA : TB;
        const bool behind = turned ? k * S::K + turned_row(i, lane) >= a.K : NP == 1 && !OUT && k * S::K + col >= a.K;
        if (behind) *reinterpret_cast<u16x8*>(lds + buf * TILE + place_of(i, lane) * 8) = u16x8{};
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  floatx4 acc[RT][CT];

  const int fr = lane & 15, fk = lane >> 4;
  const uint16_t* la = lds + (wm * (BM / WM) + fr) * S::ROW;
  const uint16_t* lb = lds + (BM + wn * (BN / WN) + fr) * S::ROW;
  // A turned operand's: the lane's place in its first row, and which way its chunks are turned.
  const int turn = S::turn(fk * 8 + (fr >> 2)) * 8;
  const uint16_t* ta = lds + (fk * 8 + (fr >> 2)) * (BM * NP) + (fr & 3) * 4;
  const uint16_t* tb = lds + BM * S::ROW + (fk * 8 + (fr >> 2)) * S::ROW + (fr & 3) * 4;
  // Its 16 columns from `t` * 16 on over 32 rows: rows 8 fk .. 8 fk + 3 of them and the four behind.
  auto columns = [&](const uint16_t* p, int width) {
    const u16x4 u = read_tr(p), v = read_tr(p + 4 * width);
    return __builtin_bit_cast(bf16x8, u16x8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]});
  };
  auto columns_a = [&](int t, int q, int buf) {
    const int pair = NP == 1 ? t : (t >> 1) * 6 + q * 2 + (t & 1);
    return columns(ta + buf * TILE + (pair * 16 ^ turn), BM * NP);
  };
  auto columns_b = [&](int t, int q, int buf) {
    return columns(tb + buf * TILE + (t >> 1) * (32 * S::ROW) + q * 32 + ((t & 1) * 16 ^ S::turn_dl(fk * 8) * 8), S::ROW);
  };
  // Fragment set q: of one part the half-step q, of three parts the part q.
  constexpr bool EARLY = !OUT;
  typedef std::integral_constant<int, 0> None;
  constexpr int READS = (TA ? 2 : 1) * RT + (TB ? 2 : 1) * CT;
  auto read = [&](int q, int buf, bf16x8(&fa)[RT], bf16x8(&fb)[CT]) {
    const int c = S::place(q * 4 + fk, fr) * 8 + buf * TILE;  // tile rows are multiples of 16: place() sees fr
#pragma unroll
    for (int j = 0; j < CT; ++j)
      fb[j] = TB ? columns_b(wn * CT + j, q, buf) : *reinterpret_cast<const bf16x8*>(lb + j * 16 * S::ROW + c);
#pragma unroll
    for (int i = 0; i < RT; ++i)
      fa[i] = TA ? columns_a(wm * RT + i, q, buf) : *reinterpret_cast<const bf16x8*>(la + i * 16 * S::ROW + c);
  };
  auto multiply = [&](const bf16x8(&fa)[RT], const bf16x8(&fb)[CT]) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
  };

  // Puts out the products of tile (m0, n0); info[at] has its rows.
  auto put_out = [&](const int64_t m0, const int64_t n0, const int tile_m, const int tile_n, const int split_k,
                     const int at) {
    const int tid = fresh(threadIdx.x), lane = tid & 63, fr = lane & 15, fk = lane >> 4;
    const int64_t mb = m0 + wm * (BM / WM) + fk * 4;  // first of this lane's four rows of A in tile row 0
    const int64_t nb = n0 + wn * (BN / WN) + fr;

    if constexpr (OUT) {
      const float scale = a.scale ? *a.scale : 1.f;
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const int64_t n = nb + j * 16;
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const int64_t m = mb + i * 16;
          if (m >= a.M) continue;
          floatx4 v = acc[i][j] * scale;
          if (a.acc) {
            floatx4* p = reinterpret_cast<floatx4*>(a.acc + ((int64_t)split_k * a.N + n) * a.ldacc + m);
            if (a.add) v += *p;
            *p = v;
          } else if (F32) {
            put<true>(static_cast<float*>(a.out) + n * a.ldo, m, a.M, v);
          } else {
            put<false>(static_cast<uint16_t*>(a.out) + n * a.ldo, m, a.M, v);
          }
        }
      }
      return;
    }

    // logits: the bias, and classes behind the last at -inf
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const floatx4 bv = *reinterpret_cast<const floatx4*>(bias + at * BIAS + wm * (BM / WM) + fk * 4 + i * 16);
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] += bv;
      }
    }
    if (m0 + BM > a.M) {
      const int left = (int)(a.M - mb);  // of this lane's rows of A
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bool in = i * 16 + q < left;
#pragma unroll
          for (int j = 0; j < CT; ++j) acc[i][j][q] = in ? acc[i][j][q] : -INFINITY;
        }
    }

    // Hands use(i, y) the label row's values beside acc[i][j], four i at a time on their way (more would take registers
    // that are not there); of a row that is not `in`, another's.
    auto labels = [&](int j, bool in, auto use) {
      typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
      const float* row = static_cast<const float*>(a.rows.target) + (in ? nb + j * 16 : 0) * a.V + a.v0 + mb;
      if (m0 + BM <= a.M) {
#pragma unroll
        for (int i0 = 0; i0 < RT; i0 += 4) {
          f32x4 y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = *reinterpret_cast<const f32x4*>(row + (i0 + i) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) use(i0 + i, floatx4{y[i][0], y[i][1], y[i][2], y[i][3]});
        }
        return;
      }
      const int left = fresh((int)(a.M - mb));  // of this lane's classes
      if (a.V < 4) {
        floatx4 y;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = q < left ? row[q] : 0.f;
        use(0, y);
        return;
      }
      // four values that end with the piece's last one where they would go beyond it, moved to their places
#pragma unroll
      for (int i0 = 0; i0 < RT; i0 += 4) {
        f32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = (i0 + i) * 16;
          v[i] = *reinterpret_cast<const f32x4*>(row + (from < left - 4 ? from : left - 4));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int by = (i0 + i) * 16 - (left - 4);
          floatx4 y = floatx4{v[i][0], v[i][1], v[i][2], v[i][3]};
          if (__any(by > 0)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float s = by <= 0 ? v[i][q] : 0.f;
#pragma unroll
              for (int k = 1; q + k < 4; ++k) s = by == k ? v[i][q + k] : s;
              y[q] = s;
            }
          }
          use(i0 + i, y);
        }
      }
    };

    if constexpr (EPI == E_LSE) {
      float* sm = reinterpret_cast<float*>(stage);  // [4][WM][BN]
      float top[CT], sum[CT], dot[CT] = {}, mass[CT] = {};
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        top[j] = -INFINITY, sum[j] = 0.f;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) top[j] = fmaxf(top[j], acc[i][j][q]);
      }
#pragma unroll
      for (int d = 16; d < 64; d <<= 1) {
        float other[CT];
#pragma unroll
        for (int j = 0; j < CT; ++j) other[j] = __shfl_xor(top[j], d);
#pragma unroll
        for (int j = 0; j < CT; ++j) top[j] = fmaxf(top[j], other[j]);
      }
      if constexpr (SOFT) {
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const bool in = word_target(info[at * INFO + wn * (BN / WN) + j * 16 + fr][3]) != kLeftOut;
          const float ref = reference(top[j]);
          labels(j, in, [&](int i, floatx4 y) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float v = in ? y[q] : 0.f;
              mass[j] += v;
              dot[j] += v == 0.f ? 0.f : v * (acc[i][j][q] - ref);  // a class at -inf without mass adds nothing
            }
          });
        }
#pragma unroll
        for (int d = 16; d < 64; d <<= 1)
#pragma unroll
          for (int j = 0; j < CT; ++j) {
            dot[j] += __shfl_xor(dot[j], d);
            mass[j] += __shfl_xor(mass[j], d);
          }
      }
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const float ref = reference(top[j]);
        const Exponent e(ref);
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) part[q] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][q], e.by, e.off));
        sum[j] = ((part[0] + part[1]) + (part[2] + part[3])) * e.rest(ref);
      }
      if constexpr (!SOFT) {
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const int target = word_target(info[at * INFO + wn * (BN / WN) + j * 16 + fr][3]), t = target - (int)mb;
          if (__any(target >= 0 && t >= 0 && t < RT * 16)) {  // few tiles hold a target
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (target >= 0 && t == i * 16 + q) a.hit[nb + j * 16] = acc[i][j][q];
          }
        }
      }
#pragma unroll
      for (int d = 16; d < 64; d <<= 1) {
        float other[CT];
#pragma unroll
        for (int j = 0; j < CT; ++j) other[j] = __shfl_xor(sum[j], d);
#pragma unroll
        for (int j = 0; j < CT; ++j) sum[j] += other[j];
      }
      if (fk == 0) {
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const int c = wn * (BN / WN) + j * 16 + fr;
          sm[wm * BN + c] = top[j];
          sm[(WM + wm) * BN + c] = sum[j];
          sm[(2 * WM + wm) * BN + c] = dot[j];
          sm[(3 * WM + wm) * BN + c] = mass[j];
        }
      }
      __syncthreads();
      for (int col = tid; col < BN; col += NW * 64) {
        if (n0 + col >= a.N) break;
        float top = sm[col];
#pragma unroll
        for (int w = 1; w < WM; ++w) top = fmaxf(top, sm[w * BN + col]);
        const float ref = reference(top);
        float sum = 0.f, dot = 0.f, mass = 0.f;
#pragma unroll
        for (int w = 0; w < WM; ++w) {
          const float tw = sm[w * BN + col], mw = sm[(3 * WM + w) * BN + col];
          sum += sm[(WM + w) * BN + col] * (tw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((tw - ref) * kLog2e));
          dot += moved(sm[(2 * WM + w) * BN + col], mw, tw, ref);
          mass += mw;
        }
        a.part[(n0 + col) * a.part_ld + a.part_at + tile_m] = make_float2(top, sum);
        if (SOFT) a.part_y[(n0 + col) * a.part_ld + a.part_at + tile_m] = make_float2(dot, mass);
      }
      return;
    }

    if constexpr (EPI == E_DL) {
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const floatx4 row = info[at * INFO + wn * (BN / WN) + j * 16 + fr];
        const int target = word_target(row[3]);
        const float by = word_far(row[3]) ? 1.f : kLog2e, off = row[0], gv = row[1], gs = row[2];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            acc[i][j][q] = gs * __builtin_amdgcn_exp2f(fmaf(acc[i][j][q], by, off));
        if constexpr (!SOFT) {
          const int t = target - (int)mb;
          if (__any(target >= 0 && t >= 0 && t < RT * 16)) {  // few tiles hold a target
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) acc[i][j][q] -= target >= 0 && t == i * 16 + q ? gv : 0.f;
          }
        }
      }
      if constexpr (SOFT) {
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const floatx4 row = info[at * INFO + wn * (BN / WN) + j * 16 + fr];
#pragma unroll
          for (int i = 0; i < RT; ++i) asm volatile("" : "+v"(acc[i][j]));  // the exponentials first: not the labels wait
          labels(j, word_target(row[3]) != kLeftOut, [&](int i, floatx4 y) {
            acc[i][j] -= row[1] * y;
            asm volatile("" : "+v"(acc[i][j]));
          });
        }
      }
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const bool in = word_target(info[at * INFO + wn * (BN / WN) + j * 16 + fr][3]) != kLeftOut;
        if (!__all(in)) {  // rows left out, whatever their logits
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][j][q] = in ? acc[i][j][q] : 0.f;
        }
      }
      if (m0 + BM > a.M) {  // classes behind the last: an lse of NaN must not reach them
        const int left = (int)(a.M - mb);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < CT; ++j) acc[i][j][q] = i * 16 + q < left ? acc[i][j][q] : 0.f;
      }
      if (a.part_b) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          floatx4 s = acc[i][0];
#pragma unroll
          for (int j = 1; j < CT; ++j) s += acc[i][j];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float r = sum16(s[q]);
            const int64_t m = mb + i * 16 + q;
            if (fr == 0 && m < a.M) a.part_b[(int64_t)(tile_n * WN + wn) * a.M + m] = r;
          }
        }
      }
      // dl goes out through LDS in whole 16-byte chunks: from the registers it would be 8-byte pieces of 16 rows.
      constexpr int THREADS = NW * 64, HN = BN / HALVES;
      const int lm = wm * (BM / WM) + fk * 4, ln = wn * (BN / WN) + fr;
#pragma unroll
      for (int s = 0; s < NP; ++s) {
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          if (s + half > 0) lds_barrier();
          if (wn * (BN / WN) / HN == half) {
#pragma unroll
            for (int j = 0; j < CT; ++j)
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                u16x4 part;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  part[q] = to_bf16(acc[i][j][q]);
                  if (NP > 1) acc[i][j][q] -= from_bf16(part[q]);  // what the next part holds
                }
                *reinterpret_cast<u16x4*>(stage + (ln - half * HN + j * 16) * (BM + PAD) + lm + i * 16) = part;
              }
          }
          lds_barrier();
#pragma unroll 2
          for (int e = tid; e < HN * (BM / 8); e += THREADS) {  // 16 rows of a block a wave: 1 KB
            const int row = (e >> 2) % HN, c = (e >> 2) / HN * 32 + (e & 3) * 8;
            const int64_t n = n0 + half * HN + row;
            if (n < a.N && m0 + c < a.mp)
              *reinterpret_cast<u16x8*>(a.P + ((m0 + c) / 32 * a.block + n) * (32 * NP) + s * 32 + (c & 31)) =
                  *reinterpret_cast<const u16x8*>(stage + row * (BM + PAD) + c);
          }
        }
      }
    }
  };

  take(first);
  if (k_from < k_to) load(k_from, 0);
  if (DEEP && k_from < k_to) load(k_from + 1, 1);
  fetch_rows(0);
  int at = 0;
  for (uint32_t bid = first; bid < all; bid += step, at ^= 1) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (k_from < k_to) {
      hand_over(k_from, 0, None());
      if (!DEEP) load(k_from + 1, 1);
      if constexpr (DEEP) {
        load(k_from + 2, 2);
        load(k_from + 3, 3);
        bf16x8 fa0[RT], fb0[CT], fa1[RT], fb1[CT];
        read(0, 0, fa0, fb0);
        // step k's products; step k + 1 is read and step k + 4 sent for
        auto go = [&](int k, const bf16x8(&fa)[RT], const bf16x8(&fb)[CT], bf16x8(&na)[RT], bf16x8(&nb)[CT]) {
          const int buf = (k - k_from) & 3;
          hand_over(k + 1, (buf + 1) & 3, std::integral_constant<int, 2 * IT>());
          read(0, (buf + 1) & 3, na, nb);  // behind the last step: what lies there, never multiplied
          load(k + 4, buf);
          multiply(fa, fb);
          interleave<RT * CT, READS, IT, EARLY>();
        };
        for (int k = k_from; k < k_to; k += 2) {
          go(k, fa0, fb0, fa1, fb1);
          if (k + 1 < k_to) go(k + 1, fa1, fb1, fa0, fb0);
        }
      } else if constexpr (NP == 1) {
        bf16x8 fa0[RT], fb0[CT], fa1[RT], fb1[CT];
        read(0, 0, fa0, fb0);
        for (int k = k_from; k < k_to; ++k) {
          const int buf = (k - k_from) & 1;
          read(1, buf, fa1, fb1);
          multiply(fa0, fb0);
          interleave<RT * CT, READS, 0, EARLY>();
          hand_over(k + 1, buf ^ 1, None());
          if (EARLY) load(k + 2, buf);
          read(0, buf ^ 1, fa0, fb0);  // behind the last step: what lies there, never multiplied
          if (!EARLY) load(k + 2, buf);
          multiply(fa1, fb1);
          interleave<RT * CT, READS, IT, EARLY>();
        }
      } else {
        bf16x8 ha[RT], hb[CT], ma[RT], mb[CT], sa[RT], sb[CT];
        read(1, 0, ma, mb);
        for (int k = k_from; k < k_to; ++k) {
          const int buf = (k - k_from) & 1;
          read(0, buf, ha, hb);
          multiply(ma, mb);
          interleave<RT * CT, READS, 0, EARLY>();
          read(2, buf, sa, sb);
          multiply(ma, hb);
          multiply(ha, mb);
          interleave<2 * RT * CT, READS, 0, EARLY>();
          hand_over(k + 1, buf ^ 1, None());
          if (EARLY) load(k + 2, buf);
          read(1, buf ^ 1, ma, mb);
          if (!EARLY) load(k + 2, buf);
          multiply(sa, hb);
          multiply(ha, sb);
          multiply(ha, hb);
          interleave<3 * RT * CT, READS, IT, EARLY>();
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();

    // The next tile's first operands and rows are on their way while this one's products are put out.
    const int64_t m0_now = m0, n0_now = n0;
    const int tm_now = tile_m, tn_now = tile_n, split_now = split_k;
    if (bid + step < all) {
      take(bid + step);
      if (k_from < k_to) load(k_from, 0);
      if (DEEP && k_from < k_to) load(k_from + 1, 1);
      fetch_rows(at ^ 1);
    }
    put_out(m0_now, n0_now, tm_now, tn_now, split_now, at);
  }
}

// (One LDS object: with two, the compiler waits for every load into LDS before any read of it.)
template <int BM, int BN, int WM, int WN, int EPI, int NP, bool F32, bool SOFT>
__global__ void __launch_bounds__(WM* WN * 64, NP == 1 || BM == 256 ? 2 : 1) k_xent_mm(GemmArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Space<BM, BN, EPI, NP>::ALL];
  mm_tiles<BM, BN, WM, WN, EPI, NP, F32, SOFT>(a, lds, blockIdx.x, gridDim.x);
}

// gx and gW of a piece side by side, gx's in the first `groups` workgroups.
template <int NP, bool F32>
__global__ void __launch_bounds__(256, NP == 1 ? 2 : 1) k_xent_both(GemmArgs x, GemmArgs w, uint32_t groups) {
  static_assert(Space<128, 128, E_GX, NP>::ALL == Space<128, 128, E_GW, NP>::ALL, "one space for either");
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Space<128, 128, E_GW, NP>::ALL];
  if (blockIdx.x < groups) mm_tiles<128, 128, 2, 2, E_GX, NP, F32, false>(x, lds, blockIdx.x, groups);
  else mm_tiles<128, 128, 2, 2, E_GW, NP, F32, false>(w, lds, blockIdx.x - groups, gridDim.x - groups);
}

// A pair (largest, sum of exponentials relative to it) joined with another.
__device__ __forceinline__ void join_pair(float& top, float& sum, float top2, float sum2) {
  const float nt = fmaxf(top, top2), ref = reference(nt);
  sum = sum * (top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((top - ref) * kLog2e)) +
        sum2 * (top2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((top2 - ref) * kLog2e));
  top = nt;
}

// Likewise with (sum y (l - largest), sum y).
__device__ __forceinline__ void join_row(float& top, float& sum, float& dot, float& mass, float top2, float sum2, float dot2,
                                         float mass2) {
  const float ref = reference(fmaxf(top, top2));
  dot = moved(dot, mass, top, ref) + moved(dot2, mass2, top2, ref);
  mass += mass2;
  join_pair(top, sum, top2, sum2);
}

// ---- joins ------------------------------------------------------------------------------------------------------
// One wave a row: the tiles' (largest, sum) pairs into the row's running pair; at the last piece, lse and the loss.
__global__ void __launch_bounds__(256) k_xent_join(int64_t N, int64_t tiles, const float2* __restrict__ part,
                                                   const float2* __restrict__ part_y, const float* __restrict__ hit,
                                                   Rows rows, int64_t V, float4* __restrict__ run, int first, int last,
                                                   float* __restrict__ loss, float* __restrict__ stats) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  float top = -INFINITY, sum = 0.f, dot = 0.f, mass = 0.f;
  if (!first && lane == 0) {
    const float4 r = run[n];
    top = r.x, sum = r.y, dot = r.z, mass = r.w;
  }
  for (int64_t i = lane; i < tiles; i += 64) {
    const float2 p = part[n * tiles + i];
    const float2 q = part_y ? part_y[n * tiles + i] : make_float2(0.f, 0.f);
    join_row(top, sum, dot, mass, p.x, p.y, q.x, q.y);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
    join_row(top, sum, dot, mass, __shfl_xor(top, d), __shfl_xor(sum, d), __shfl_xor(dot, d), __shfl_xor(mass, d));
  if (lane != 0) return;
  if (!last) {
    run[n] = make_float4(top, sum, dot, mass);
    return;
  }
  const bool counts = row_counts(rows, n);
  const float ls = logf(sum);
  float lse = top + ls;
  if (rows.kind != GNCDE_TARGET_ROWS && counts) {
    const bool in = row_index(rows, n) < V;
    lse = in ? lse : NAN;
    dot = in ? hit[n] - top : NAN;
    mass = 1.f;
  }
  loss[n] = counts ? mass * ls - dot : 0.f;
  stats[2 * n] = counts ? lse : 0.f;
  stats[2 * n + 1] = counts ? mass_beside(lse, top, ls, mass) : 0.f;
}

// out[i] = sum over splits of acc[s][i], in the split order, times the scale: up to four such jobs a launch.
struct SumJob {
  int64_t N, M;
  int64_t ldacc, stride, ldo;
  const float* acc;
  const float* scale;  // may be NULL
  void* out;
  int32_t splits;
  uint32_t blocks;
};

struct SumJobs {
  SumJob job[4];
};

template <bool F32>
__global__ void __launch_bounds__(256) k_xent_sum(SumJobs jobs) {
  uint32_t at = blockIdx.x;
  int q = 0;
  while (q < 3 && at >= jobs.job[q].blocks) at -= jobs.job[q++].blocks;
  const SumJob& j = jobs.job[q];
  const float by = j.scale ? *j.scale : 1.f;
  const int splits = j.splits;
  for (int64_t e = (int64_t)at * 256 + threadIdx.x; e < j.N * j.M; e += (int64_t)j.blocks * 256) {
    const int64_t n = e / j.M, m = e - n * j.M;
    float s = 0.f;
    for (int k0 = 0; k0 < splits; k0 += 8) {  // eight loads side by side: 64 splits of 100 x 512 18 -> 6 us
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k0 + k < splits ? j.acc[(k0 + k) * j.stride + n * j.ldacc + m] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    s *= by;
    if (F32) static_cast<float*>(j.out)[n * j.ldo + m] = s;
    else static_cast<uint16_t*>(j.out)[n * j.ldo + m] = to_bf16(s);
  }
}

// ---- few classes and a narrow hidden row: everything in LDS -----------------------------------------------------
// W (as fp32), 16 rows of x and their dl stay in LDS and all four products run on v_mfma_f32_16x16x4f32 (either type:
// the products of bf16 values are exact there), so nothing but the results goes to memory: the loss is one launch, the
// gradient two (the second adds the workgroups' gW and gb).  TGB's read-out (classes = nodes, hidden 32) is this size,
// where the tiled kernels above are eleven launches of a few microseconds.  255 x 32 x 255 (the loss) takes 6 us and the
// gradient of 4080 x 32 x 255 14 and 4, of which launches, the first reads and the last writes are all but a few.
//
// Sixteen waves a workgroup; a row tile's classes go round the waves by 16, two rounds at most.
constexpr int kSmallLds = 20480;     // floats: W [Vp][Hs], x [16][Hs], dl [16][Vs], joins
constexpr int kSmallJoin = 5120;     // [16][16][4] of the loss, [16 / (Hp / 16)][16][Hs] of gx
constexpr int kSmallTiles = 4;       // 16 x 16 tiles of gW a wave holds
constexpr int kSmallThreads = 1024, kSmallWaves = 16;

struct SmallSize {
  int Vp, Hp, Hs, Vs;  // padded to 16; row strides of W / x and of dl, 4 floats off a multiple of 16 (banks)
};

__host__ __device__ __forceinline__ SmallSize small_size(int H, int V) {
  SmallSize z;
  z.Vp = (V + 15) / 16 * 16, z.Hp = (H + 15) / 16 * 16;
  z.Hs = z.Hp + 4, z.Vs = z.Vp + 4;
  return z;
}

bool small_fits(int64_t H, int64_t V) {
  if (H > 128 || V > 2 * 16 * kSmallWaves) return false;
  const SmallSize z = small_size((int)H, (int)V);
  return z.Vp * z.Hs + 16 * z.Hs + 16 * z.Vs + kSmallJoin <= kSmallLds &&
         (z.Vp / 16) * (z.Hp / 16) <= kSmallWaves * kSmallTiles;
}

struct SmallArgs {
  const void *x, *W, *b;
  Rows rows;
  int64_t N;
  int H, V;
  float *loss, *stats;         // the loss writes both
  const float *row_stats, *g;  // the gradient reads both
  void* gx;                    // may be NULL
  float* part;                 // [workgroups][V H + V]; NULL without gW and gb
};

template <bool F32, bool GRAD>
__global__ void __launch_bounds__(kSmallThreads) k_xent_small(SmallArgs a) {
  __shared__ __attribute__((aligned(16))) float sm[kSmallLds];
  const SmallSize z = small_size(a.H, a.V);
  float* w = sm;
  float* x = w + z.Vp * z.Hs;
  float* d = x + 16 * z.Hs;
  float* join = d + 16 * z.Vs;
  const int lane = threadIdx.x & 63, fr = lane & 15, fk = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int vt = z.Vp / 16, ht = z.Hp / 16, hq = z.Hp / 4;
  const int lr = threadIdx.x / hq, lh = (threadIdx.x - lr * hq) * 4;  // this thread's row and values of W and x
  for (int v = lr; v < z.Vp; v += kSmallThreads / hq) {
    if (lr >= kSmallThreads / hq) break;
    *reinterpret_cast<floatx4*>(w + v * z.Hs + lh) =
        v < a.V && lh < a.H ? four<F32>(a.W, (int64_t)v * a.H + lh, (int64_t)v * a.H + a.H) : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  floatx4 bias[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int v = (wave + kSmallWaves * i) * 16 + fk * 4;
    bias[i] = a.b && v < a.V ? four<F32>(a.b, v, a.V) : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const bool soft = a.rows.kind == GNCDE_TARGET_ROWS;
  floatx4 gw[kSmallTiles];
  float gb = 0.f;  // of class threadIdx.x
#pragma unroll
  for (int i = 0; i < kSmallTiles; ++i) gw[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int64_t tiles = (a.N + 15) / 16;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t r0 = t * 16, n = r0 + fr;  // n: this lane's row
    const bool in = n < a.N && row_counts(a.rows, n);
    const int64_t hit = in && !soft ? row_index(a.rows, n) : -1;
    floatx4 y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int v = (wave + kSmallWaves * i) * 16 + fk * 4;
      y[i] = floatx4{0.f, 0.f, 0.f, 0.f};
      if (soft && in && v < a.V) y[i] = four<true>(a.rows.target, n * a.V + v, n * a.V + a.V);
    }
    float lse = 0.f, gv = 0.f, gs = 0.f;
    if (GRAD && in) {
      lse = a.row_stats[2 * n];
      gv = a.g[n];
      gs = gv * a.row_stats[2 * n + 1];
    }
    floatx4 xv = floatx4{0.f, 0.f, 0.f, 0.f};
    if (lr < 16 && r0 + lr < a.N && lh < a.H && (!GRAD || row_counts(a.rows, r0 + lr)))
      xv = four<F32>(a.x, (r0 + lr) * a.H + lh, (r0 + lr) * a.H + a.H);
    __syncthreads();  // the last tile's x, dl and joins have been read
    if (lr < 16) *reinterpret_cast<floatx4*>(x + lr * z.Hs + lh) = xv;
    __syncthreads();
    float top = -INFINITY, sum = 0.f, dot = 0.f, mass = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tile = wave + kSmallWaves * i;
      if (tile >= vt) break;
      floatx4 l = floatx4{0.f, 0.f, 0.f, 0.f}, l1 = l;
      const float* wa = w + (tile * 16 + fr) * z.Hs + fk;
      const float* xb = x + fr * z.Hs + fk;
      for (int h = 0; h < z.Hp; h += 16) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          l = __builtin_amdgcn_mfma_f32_16x16x4f32(wa[h + 8 * k], xb[h + 8 * k], l, 0, 0, 0);
          l1 = __builtin_amdgcn_mfma_f32_16x16x4f32(wa[h + 8 * k + 4], xb[h + 8 * k + 4], l1, 0, 0, 0);
        }
      }
      const int v = tile * 16 + fk * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) l[q] = v + q < a.V ? l[q] + l1[q] + bias[i][q] : -INFINITY;
      if (GRAD) {
        floatx4 dv;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          dv[q] = gs * __builtin_amdgcn_exp2f((l[q] - lse) * kLog2e);
          if (soft) dv[q] -= gv * y[i][q];
          else dv[q] -= hit == v + q ? gv : 0.f;
          dv[q] = in && v + q < a.V ? dv[q] : 0.f;
        }
        *reinterpret_cast<floatx4*>(d + fr * z.Vs + v) = dv;
      } else {
        const float tt = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), ref = reference(tt);
        float ts = 0.f, td = 0.f, tm = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          ts += __builtin_amdgcn_exp2f((l[q] - ref) * kLog2e);
          const float yq = soft ? y[i][q] : hit == v + q ? 1.f : 0.f;
          tm += yq;
          td += yq == 0.f ? 0.f : yq * (l[q] - ref);  // a class at -inf without mass adds nothing
        }
        join_row(top, sum, dot, mass, tt, ts, td, tm);
      }
    }
    if (!GRAD) {
#pragma unroll
      for (int s = 16; s < 64; s <<= 1)
        join_row(top, sum, dot, mass, __shfl_xor(top, s), __shfl_xor(sum, s), __shfl_xor(dot, s), __shfl_xor(mass, s));
      if (fk == 0) *reinterpret_cast<floatx4*>(join + (wave * 16 + fr) * 4) = floatx4{top, sum, dot, mass};
      __syncthreads();
      if (wave == 0) {  // four of the waves' joins a lane, then the four lanes of a row
        top = -INFINITY, sum = dot = mass = 0.f;
#pragma unroll
        for (int i = 0; i < kSmallWaves / 4; ++i) {
          const floatx4 q = *reinterpret_cast<const floatx4*>(join + ((fk * 4 + i) * 16 + fr) * 4);
          join_row(top, sum, dot, mass, q[0], q[1], q[2], q[3]);
        }
#pragma unroll
        for (int s = 16; s < 64; s <<= 1)
          join_row(top, sum, dot, mass, __shfl_xor(top, s), __shfl_xor(sum, s), __shfl_xor(dot, s), __shfl_xor(mass, s));
        if (fk == 0 && n < a.N) {
          const float ls = logf(sum);
          lse = top + ls;
          if (!soft) {
            mass = 1.f;
            if (in && hit >= a.V) lse = dot = NAN;
          }
          a.loss[n] = in ? mass * ls - dot : 0.f;
          a.stats[2 * n] = in ? lse : 0.f;
          a.stats[2 * n + 1] = in ? mass_beside(lse, top, ls, mass) : 0.f;
        }
      }
    } else {
      __syncthreads();
      const int parts = kSmallWaves / ht;  // waves that share a hidden tile of gx, each with its share of the classes
      if (a.gx && wave < parts * ht) {     // gx^T [hidden][16 rows]
        const int i = wave % ht, part = wave / ht;
        floatx4 o0 = floatx4{0.f, 0.f, 0.f, 0.f}, o1 = o0;
        const float* wa = w + fk * z.Hs + i * 16 + fr;
        const float* db = d + fr * z.Vs + fk;
        for (int v = part * 16; v < z.Vp; v += parts * 16) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            o0 = __builtin_amdgcn_mfma_f32_16x16x4f32(wa[(v + 8 * k) * z.Hs], db[v + 8 * k], o0, 0, 0, 0);
            o1 = __builtin_amdgcn_mfma_f32_16x16x4f32(wa[(v + 8 * k + 4) * z.Hs], db[v + 8 * k + 4], o1, 0, 0, 0);
          }
        }
        *reinterpret_cast<floatx4*>(join + (part * 16 + fr) * z.Hs + i * 16 + fk * 4) = o0 + o1;
      }
      if (a.part) {
#pragma unroll
        for (int i = 0; i < kSmallTiles; ++i) {  // gW [classes][hidden]: tiles round the waves
          const int tile = wave + kSmallWaves * i;
          if (tile >= vt * ht) break;
          const int v = tile / ht * 16, h = tile % ht * 16;
#pragma unroll
          for (int k = 0; k < 16; k += 4)
            gw[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(d[(k + fk) * z.Vs + v + fr], x[(k + fk) * z.Hs + h + fr],
                                                         gw[i], 0, 0, 0);
        }
        if (threadIdx.x < a.V) {
          float s = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) s += d[r * z.Vs + threadIdx.x];
          gb += s;
        }
      }
      __syncthreads();
      if (a.gx && lr < 16 && r0 + lr < a.N) {
        floatx4 o = *reinterpret_cast<const floatx4*>(join + lr * z.Hs + lh);
        for (int q = 1; q < parts; ++q) o += *reinterpret_cast<const floatx4*>(join + (q * 16 + lr) * z.Hs + lh);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (lh + q < a.H) {
            if (F32) static_cast<float*>(a.gx)[(r0 + lr) * a.H + lh + q] = o[q];
            else static_cast<uint16_t*>(a.gx)[(r0 + lr) * a.H + lh + q] = to_bf16(o[q]);
          }
      }
    }
  }
  if (GRAD && a.part) {
    float* out = a.part + (int64_t)blockIdx.x * ((int64_t)a.V * a.H + a.V);
#pragma unroll
    for (int i = 0; i < kSmallTiles; ++i) {
      const int tile = wave + kSmallWaves * i;
      if (tile >= vt * ht) break;
      const int v = tile / ht * 16 + fk * 4, h = tile % ht * 16 + fr;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (v + q < a.V && h < a.H) out[(v + q) * a.H + h] = gw[i][q];
    }
    if (threadIdx.x < a.V) out[a.V * a.H + threadIdx.x] = gb;
  }
}

// VH values of gW and V of gb (or gx's, with V 0) from the workgroups' parts: 64 values a workgroup, sixteen runs of
// parts side by side, added in order.
template <bool F32>
__global__ void __launch_bounds__(1024) k_xent_parts_sum(int parts, int VH, int V, const float* __restrict__ part,
                                                         void* __restrict__ gW, void* __restrict__ gb) {
  __shared__ float run[16][64];
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int e = blockIdx.x * 64 + c, len = VH + V;
  const int per = (parts + 15) / 16, to = per * (q + 1) < parts ? per * (q + 1) : parts;
  float s = 0.f;
  if (e < len) {
    for (int i = per * q; i < to; i += 8) {  // eight loads side by side
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i + u < to ? part[(int64_t)(i + u) * len + e] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  }
  run[q][c] = s;
  __syncthreads();
  if (q != 0 || e >= len) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += run[i][c];
  void* out = e < VH ? gW : gb;
  const int at = e < VH ? e : e - VH;
  if (!out) return;
  if (F32) static_cast<float*>(out)[at] = s;
  else static_cast<uint16_t*>(out)[at] = to_bf16(s);
}

// ---- few rows ---------------------------------------------------------------------------------------------------
// Up to 16 rows: one matrix tile's columns, and the weight's bytes are all there is.  Every wave streams its own W rows
// from memory into matrix operands (16 classes, 16 bytes a lane; LDS holds x alone), eight loads ahead of the products;
// where the classes are too few for all waves, ks of them share a tile's contraction.  The gradient reads W once for dl
// and once more, row by row, for gx, writing gW in the same loop: a VALU product, which for so few rows hides behind
// the bytes, and needs no transposed copy of W.  One row of 4096 against 131072 classes in bf16: 210 us
// with the join's 5, 5.2 TB/s of the stream, where reads alone reach 6.4.
constexpr int kFewRows = 16;
constexpr int kFewWaves = 16;
constexpr int kFewLds = 147456;   // bytes of x
constexpr int kFewAhead = 8;      // loads in flight a lane

template <bool F32>
struct Few {
  static constexpr int K = F32 ? 16 : 32;  // contraction a load of all lanes
  static constexpr int C = F32 ? 4 : 8;    // values a lane
  static constexpr int SZ = F32 ? 4 : 2;
};

struct FewArgs {
  const void *x, *W, *b;
  Rows rows;
  int N, H, ks, xs;            // ks: waves that share a tile; xs: values a row of x in LDS
  int64_t V, tiles;
  float2 *part, *part_y;       // the loss: [N][workgroups]
  float* hit;
  const float *stats, *g;      // the gradient
  float* d;                    // [N][V]
  void* gb;
};

template <bool F32, bool GRAD>
__global__ void __launch_bounds__(kFewWaves * 64) k_xent_few(FewArgs a) {
  typedef Few<F32> S;
  typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef __bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
  extern __shared__ __attribute__((aligned(16))) char few_lds[];
  char* xl = few_lds;
  __shared__ __attribute__((aligned(16))) float join[kFewWaves * 64 * 4];
  const int lane = threadIdx.x & 63, fr = lane & 15, fk = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int xs = a.xs;
  for (int e = threadIdx.x; e < a.N * xs; e += kFewWaves * 64) {
    const int n = e / xs, h = e - n * xs;
    const bool in = h < a.H;
    if (F32) reinterpret_cast<float*>(xl)[e] = in ? static_cast<const float*>(a.x)[n * a.H + h] : 0.f;
    else reinterpret_cast<uint16_t*>(xl)[e] = in ? static_cast<const uint16_t*>(a.x)[n * a.H + h] : (uint16_t)0;
  }
  __syncthreads();
  const int64_t n = fr;
  const bool in = n < a.N && row_counts(a.rows, n);
  const bool soft = a.rows.kind == GNCDE_TARGET_ROWS;
  const int64_t hit = in && !soft ? row_index(a.rows, n) : -1;
  const float* y = in && soft ? static_cast<const float*>(a.rows.target) + n * a.V : nullptr;
  float lse = 0.f, gv = 0.f, gs = 0.f;
  if (GRAD && in) {
    lse = a.stats[2 * n];
    gv = a.g[n];
    gs = gv * a.stats[2 * n + 1];
  }
  float top = -INFINITY, sum = 0.f, dot = 0.f, mass = 0.f;
  const int group = wave / a.ks, share = wave % a.ks, groups = kFewWaves / a.ks;
  const int ksteps = (a.H + S::K - 1) / S::K, per = (ksteps + a.ks - 1) / a.ks;
  const int s_from = share * per, s_to = s_from + per < ksteps ? s_from + per : ksteps;
  const char* xrow = xl + (fr < a.N ? fr : a.N - 1) * xs * S::SZ + fk * 16;
  for (int64_t t0 = (int64_t)blockIdx.x * groups; t0 < a.tiles; t0 += (int64_t)gridDim.x * groups) {
    const int64_t tile = t0 + group, v0 = tile * 16;
    floatx4 acc0 = floatx4{0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    if (tile < a.tiles) {
      const int64_t row = v0 + fr < a.V ? v0 + fr : a.V - 1;
      const char* wrow = static_cast<const char*>(a.W) + (row * a.H + fk * S::C) * S::SZ;
      auto get = [&](int s, u16x8& o) {  // 16 bytes of this lane's W row, zeros behind its end
        const int h = s * S::K + fk * S::C;
        const char* p = wrow + (int64_t)s * S::K * S::SZ;
        if (h + S::C <= a.H) {
          if (F32) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(p);
            o = __builtin_bit_cast(u16x8, floatx4{v[0], v[1], v[2], v[3]});
          } else {
            const bf16x8u v = *reinterpret_cast<const bf16x8u*>(p);
            o = __builtin_bit_cast(u16x8, v);
          }
        } else {
          o = u16x8{};
          if (F32) {
            floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (h + q < a.H) v[q] = reinterpret_cast<const float*>(p)[q];
            o = __builtin_bit_cast(u16x8, v);
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (h + q < a.H) o[q] = reinterpret_cast<const uint16_t*>(p)[q];
          }
        }
      };
      auto use = [&](int s, const u16x8& o, floatx4& acc) {
        const u16x8 xv = *reinterpret_cast<const u16x8*>(xrow + s * S::K * S::SZ);
        if (F32) {
          const floatx4 wf = __builtin_bit_cast(floatx4, o), xf = __builtin_bit_cast(floatx4, xv);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[q], xf[q], acc, 0, 0, 0);
        } else {
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o), __builtin_bit_cast(bf16x8, xv),
                                                        acc, 0, 0, 0);
        }
      };
      u16x8 now[kFewAhead], next[kFewAhead];
      int s = s_from;
      const int whole = s_from + (s_to - s_from) / kFewAhead * kFewAhead;
      if (s < whole) {
#pragma unroll
        for (int u = 0; u < kFewAhead; ++u) get(s + u, now[u]);
      }
      for (; s < whole; s += kFewAhead) {
        if (s + kFewAhead < whole) {
#pragma unroll
          for (int u = 0; u < kFewAhead; ++u) get(s + kFewAhead + u, next[u]);
        }
#pragma unroll
        for (int u = 0; u < kFewAhead; ++u) use(s + u, now[u], u & 1 ? acc1 : acc0);
#pragma unroll
        for (int u = 0; u < kFewAhead; ++u) now[u] = next[u];
      }
      for (; s < s_to; ++s) {
        u16x8 o;
        get(s, o);
        use(s, o, acc0);
      }
    }
    floatx4 l = acc0 + acc1;
    if (a.ks > 1) {  // the shares of a tile, added in order by its first wave
      __syncthreads();
      *reinterpret_cast<floatx4*>(join + (wave * 64 + lane) * 4) = l;
      __syncthreads();
      if (share != 0) continue;
      for (int q = 1; q < a.ks; ++q) l += *reinterpret_cast<const floatx4*>(join + ((wave + q) * 64 + lane) * 4);
    }
    if (tile >= a.tiles) continue;
    const int64_t v = v0 + fk * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      l[q] = v + q < a.V ? l[q] + (a.b ? value<F32>(a.b, v + q) : 0.f) : -INFINITY;
    if (GRAD) {
      float dv[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        dv[q] = gs * __builtin_amdgcn_exp2f((l[q] - lse) * kLog2e);
        if (soft) dv[q] -= in && v + q < a.V ? gv * y[v + q] : 0.f;
        else dv[q] -= hit == v + q ? gv : 0.f;
        dv[q] = in && v + q < a.V ? dv[q] : 0.f;
        if (n < a.N && v + q < a.V) a.d[n * a.V + v + q] = dv[q];
      }
      if (a.gb) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float r = dv[q];
#pragma unroll
          for (int i = 1; i < 16; i <<= 1) r += __shfl_xor(r, i);
          if (fr == 0 && v + q < a.V) {
            if (F32) static_cast<float*>(a.gb)[v + q] = r;
            else static_cast<uint16_t*>(a.gb)[v + q] = to_bf16(r);
          }
        }
      }
    } else {
      const float tt = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), ref = reference(tt);
      float ts = 0.f, td = 0.f, tm = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        ts += __builtin_amdgcn_exp2f((l[q] - ref) * kLog2e);
        if (soft) {
          const float yv = in && v + q < a.V ? y[v + q] : 0.f;
          tm += yv;
          td += yv == 0.f ? 0.f : yv * (l[q] - ref);  // a class at -inf without mass adds nothing
        } else if (hit == v + q) {
          a.hit[n] = l[q];
        }
      }
      join_row(top, sum, dot, mass, tt, ts, td, tm);
    }
  }
  if (GRAD) return;
#pragma unroll
  for (int s = 16; s < 64; s <<= 1)
    join_row(top, sum, dot, mass, __shfl_xor(top, s), __shfl_xor(sum, s), __shfl_xor(dot, s), __shfl_xor(mass, s));
  __syncthreads();
  if (fk == 0) *reinterpret_cast<floatx4*>(join + (wave * 16 + fr) * 4) = floatx4{top, sum, dot, mass};
  __syncthreads();
  if (threadIdx.x < a.N) {
    top = -INFINITY, sum = dot = mass = 0.f;
    for (int w = 0; w < kFewWaves; ++w) {
      const floatx4 q = *reinterpret_cast<const floatx4*>(join + (w * 16 + threadIdx.x) * 4);
      join_row(top, sum, dot, mass, q[0], q[1], q[2], q[3]);
    }
    a.part[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = make_float2(top, sum);
    if (soft) a.part_y[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = make_float2(dot, mass);
  }
}

// gx and gW from dl, W streamed once: a workgroup takes a run of classes (blockIdx.x) and 256 C columns (blockIdx.y).
template <bool F32, int NR, int C>
__global__ void __launch_bounds__(256) k_xent_few_out(int N, int H, int64_t V, int64_t per, const float* __restrict__ d,
                                                      const void* __restrict__ x, const void* __restrict__ W,
                                                      Rows rows, float* __restrict__ part, void* __restrict__ gW) {
  const int h = (blockIdx.y * 256 + threadIdx.x) * C;
  if (h >= H) return;
  const int64_t v_from = blockIdx.x * per, v_to = v_from + per < V ? v_from + per : V;
  float xv[NR][C], gx[NR][C];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const bool in = n < N && row_counts(rows, n);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      xv[n][c] = in && h + c < H ? value<F32>(x, (int64_t)n * H + h + c) : 0.f;
      gx[n][c] = 0.f;
    }
  }
  auto get = [&](int64_t v, float (&w)[C]) {
#pragma unroll
    for (int c = 0; c < C; c += 4) {
      const floatx4 q = four<F32>(W, v * H + h + c, v * H + H);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[c + i] = q[i];
    }
  };
  typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));
  auto out = [&](int64_t v, const float (&w)[C]) {
    float o[C];
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float dv = n < N ? d[n * V + v] : 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        gx[n][c] = fmaf(dv, w[c], gx[n][c]);
        o[c] = fmaf(dv, xv[n][c], o[c]);
      }
    }
    if (!gW) return;
#pragma unroll
    for (int c = 0; c < C; c += 4) {
      if (h + c + 4 <= H) {
        if (F32) *reinterpret_cast<f32x4*>(static_cast<float*>(gW) + v * H + h + c) = f32x4{o[c], o[c + 1], o[c + 2], o[c + 3]};
        else *reinterpret_cast<u16x4u*>(static_cast<uint16_t*>(gW) + v * H + h + c) =
            u16x4u{to_bf16(o[c]), to_bf16(o[c + 1]), to_bf16(o[c + 2]), to_bf16(o[c + 3])};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (h + c + i < H) {
            if (F32) static_cast<float*>(gW)[v * H + h + c + i] = o[c + i];
            else static_cast<uint16_t*>(gW)[v * H + h + c + i] = to_bf16(o[c + i]);
          }
      }
    }
  };
  int64_t v = v_from;
  for (; v + 4 <= v_to; v += 4) {
    float w[4][C];
#pragma unroll
    for (int u = 0; u < 4; ++u) get(v + u, w[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) out(v + u, w[u]);
  }
  for (; v < v_to; ++v) {
    float w[C];
    get(v, w);
    out(v, w);
  }
  if (!part) return;
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (n < N && h + c < H) part[((int64_t)blockIdx.x * N + n) * H + h + c] = gx[n][c];
}

// ---- host -------------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t div_up(int64_t x, int64_t by) { return (x + by - 1) / by; }

constexpr int64_t kCus = 256;
constexpr int64_t kMostBlocks = int64_t(1) << 20;  // of the element-wise kernels: the rest by their loops
constexpr int64_t kPieceBytes = int64_t(1) << 30;  // of a piece's operands: fewer pieces are fewer passes over gx's sums

struct Tile {
  int64_t bm, bn, wn;
};

enum { T_LARGE, T_SMALL, T_HALF };  // 256 x 256 (three parts: 256 x 128); 128 x 128; 128 x 64, of the logits alone

Tile tile_of(int tile, int np) {
  if (tile == T_LARGE) return Tile{256, np == 1 ? 256 : 128, np == 1 ? 4 : 2};
  return Tile{128, tile == T_SMALL ? 128 : 64, 2};
}

// Workgroups of a tile that a CU holds at once, by their LDS.
int64_t places(int tile, int np) {
  if (tile == T_LARGE) return 1;
  return (tile == T_HALF ? 2 : 1) + (np == 1 ? 1 : 0);
}


int64_t steps_of(int epi, int64_t K, int np) {
  return np == 1 ? div_up(K, epi == E_GX || epi == E_GW ? 32 : 64) : up(K, kPad) / 32;
}

struct Cfg {
  int tile = T_LARGE;
  int splits = 1;   // of the contraction
  double us = 0;    // what the model below says
};

// The model that chooses tiles, splits and pieces: rounds of workgroups over the CUs, each its steps and a fixed part,
// and the join of splits.  In us: a step of a 256 x 256 tile 1.45 (1.5 PFLOP/s over 256 CUs), of a 128 x 128 tile 0.83
// alone on its CU and 1.05 beside another, of a 128 x 64 tile 0.55, 0.65 and 0.95 beside two; of three parts 2.2 (256 x
// 128), 1.5 and 0.85 or 1.35 beside another.  The large tile is 1.4 to 2.3 times faster a product and loses where it
// leaves CUs without one: 784 tiles are four rounds of 256.  Against launches with one tile forced (ten shapes each, 100
// to 6000 rows, 500 to 50000 classes) the choices were the faster ones or within 10 %: the loss of 512 x 1024 x 32000
// takes 33 us in 256 x 256 tiles, 39 in 128 x 128 and 49 in 128 x 64; of 299 x 960 x 4333 in fp32 44 us in 128 x 128 and
// 30 in 128 x 64.
Cfg cost(int epi, int64_t M, int64_t N, int64_t kt, int np, int tile, int64_t splits) {
  const Tile t = tile_of(tile, np);
  const bool out = epi == E_GX || epi == E_GW;
  const int64_t groups = div_up(M, t.bm) * div_up(N, t.bn) * splits;
  const int64_t beside = std::min(places(tile, np), div_up(groups, kCus));  // workgroups that share a CU
  static const double kStep[2][3][3] = {{{1.45}, {0.83, 1.05}, {0.55, 0.65, 0.95}}, {{2.2}, {1.5}, {0.85, 1.35}}};
  const double step = kStep[np == 1 ? 0 : 1][tile][beside - 1] * (np == 1 && out ? 0.5 : 1);
  static const double kFixed[2][3] = {{7, 7, 5}, {16, 12, 7}};
  const double fixed = kFixed[epi == E_DL][tile];
  Cfg c{tile, (int)splits, (double)div_up(groups, beside * kCus) * ((double)div_up(kt, splits) * step + fixed)};
  if (splits > 1) c.us += 5 + (double)splits * (double)N * (double)M * 8 / 4.5e6;
  return c;
}

Cfg choose(int epi, int64_t M, int64_t N, int64_t kt, int np, int64_t most_splits) {
  const bool out = epi == E_GX || epi == E_GW;
  Cfg best = cost(epi, M, N, kt, np, T_LARGE, 1);
  const int64_t tiles = div_up(M, 256) * div_up(N, 256);
  for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (s > 1 && (s > most_splits || s * (np == 1 && out ? 4 : 2) > kt + 1 || tiles * s > 2 * kCus)) break;
    for (int tile = T_LARGE; tile <= (out ? T_SMALL : T_HALF); ++tile) {
      const Cfg c = cost(epi, M, N, kt, np, tile, div_up(kt, div_up(kt, s)));  // no split without a step
      if (c.us < best.us) best = c;
    }
  }
  return best;
}

// A piece's classes as whole rounds of large tiles and the rest in small ones, where that is faster than one launch.
struct Cover {
  int64_t first = 0;  // classes of the first launch; the others go to the second
  Cfg a, b;
  double us = 0;
};

Cover cover(int epi, int64_t vc, int64_t N, int64_t kt, int np) {
  Cover c;
  c.first = vc, c.a = choose(epi, vc, N, kt, np, 1), c.us = c.a.us;
  const int64_t tn = div_up(N, tile_of(T_LARGE, np).bn), rounds = div_up(vc, 256) * tn / kCus;
  const int64_t first = rounds * kCus / tn * 256;
  if (first > 0 && first < vc) {
    const Cfg a = cost(epi, first, N, kt, np, T_LARGE, 1), b = choose(epi, vc - first, N, kt, np, 1);
    if (a.us + b.us + 3 < c.us) c.first = first, c.a = a, c.b = b, c.us = a.us + b.us + 3;
  }
  return c;
}

struct PieceCfg {
  Cover dl;
  Cfg gx, gw;
  double us = 0;
};

PieceCfg piece_cfg(int64_t N, int64_t H, int64_t vc, int np, int64_t most_gx) {
  PieceCfg c;
  c.dl = cover(E_DL, vc, N, steps_of(E_DL, H, np), np);
  c.gx = choose(E_GX, H, N, steps_of(E_GX, vc, np), np, most_gx);
  c.gw = choose(E_GW, H, vc, steps_of(E_GW, N, np), np, 64);
  c.us = c.dl.us + c.gx.us + c.gw.us + (double)H * (double)N * 8 / 3e6;
  return c;
}

struct Plan {
  int64_t N, H, V;
  bool small = false;   // k_xent_small
  bool few = false;     // k_xent_few
  int64_t few_groups = 0, few_out = 0;  // workgroups of the loss / dl, runs of classes of gx and gW
  int ks = 1, xs = 0;
  bool f32, direct_ok;  // direct_ok: sizes allow x and W as operands as they lie (the pointers decide too)
  int np;
  int64_t Kp;           // packed contraction of x and W
  // rows of a block of dl: an odd multiple of 16, so that a tile's blocks do not all start on the same channels (8192
  // rows: dl and gW 2 to 3 % faster)
  int64_t block;
  int64_t piece, whole; // classes a piece; the loss's where W is used as it lies
  int64_t bytes = 0;
  // offsets
  int64_t o_x = 0, o_w = 0, o_part = 0, o_party = 0, o_hit = 0, o_run = 0;
  int64_t o_scale = 0, o_p = 0, o_gx = 0, o_gw = 0, o_b = 0;
  int64_t ldacc = 0;
  PieceCfg full, last;  // the gradient's products for a full piece and the last one

  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(std::max<int64_t>(n, 16), 256);
    return at;
  }
};

// Workgroups of the small gradient: one for each CU, each with its share of the row tiles and one part of gW.
int64_t small_groups(int64_t N) { return std::min(div_up(N, 16), kCus); }

// Rows of the bias's sums: tile columns times waves across, of either tile size.
int64_t bias_rows(int64_t N) { return 4 * div_up(N, 128); }

// Columns a thread of k_xent_few_out takes: what its rows of x and gx leave registers for.
int64_t few_cols(int64_t N) { return N > 4 ? 4 : 8; }

bool make_plan(int64_t N, int64_t H, int64_t V, int32_t dtype, bool grad, Plan& p) {
  // launches stay below 2^32 threads, and 256 rows of every operand below 2^32 bytes
  if (N < 0 || H <= 0 || V <= 0 || N > (int64_t(1) << 21) || H > (int64_t(1) << 16) || V > (int64_t(1) << 26) ||
      N * H > (int64_t(1) << 35) || V * H > (int64_t(1) << 35))
    return false;
  if (dtype != GNCDE_DTYPE_FP32 && dtype != GNCDE_DTYPE_BF16) return false;
  p = Plan{};
  p.N = N, p.H = H, p.V = V;
  p.f32 = dtype == GNCDE_DTYPE_FP32;
  p.np = p.f32 ? 3 : 1;
  p.direct_ok = !p.f32 && H % 8 == 0;
  p.Kp = up(H, 64);
  p.block = up(N, 16) | 16;
  if (N == 0) {  // nothing to plan: the gradient writes zeros
    p.take(0);
    return true;
  }
  p.small = small_fits(H, V);
  if (p.small) {
    p.o_b = p.take(grad ? 4 * small_groups(N) * (V * H + V) : 0);
    return true;
  }
  if (N <= kFewRows) {
    const int64_t sz = p.f32 ? 4 : 2, step = p.f32 ? 16 : 32;
    const int64_t xs = up(H, step) + 16 / sz;  // rows of x start in different banks
    if (N * xs * sz <= kFewLds) {
      p.few = true;
      p.xs = (int)xs;
      const int64_t tiles = div_up(V, 16);
      while (p.ks < kFewWaves && tiles * p.ks < kCus * kFewWaves && div_up(H, step) >= 2 * kFewAhead * p.ks) p.ks *= 2;
      p.few_groups = std::min(div_up(tiles * p.ks, kFewWaves), kCus);
      const int64_t cols = div_up(H, 256 * few_cols(N));
      p.few_out = std::min(div_up(V, 4), std::max<int64_t>(1, 4 * kCus / cols));
      if (!grad) {
        p.o_part = p.take(8 * N * p.few_groups);
        p.o_party = p.take(8 * N * p.few_groups);
        p.o_hit = p.take(4 * N);
      } else {
        p.o_p = p.take(4 * N * V);
        p.o_gx = p.take(4 * p.few_out * N * H);
      }
      return true;
    }
  }
  const int64_t plane = 2 * p.np;
  // Classes a piece: what the piece puts into the workspace stays within kPieceBytes.
  const int64_t per_class = plane * p.Kp + (grad ? plane * p.block : N / 8 + 24);
  const int64_t most = std::max<int64_t>(256, kPieceBytes / per_class / 256 * 256);
  p.piece = std::min(up(V, 256), most);
  p.whole = std::min(up(V, 256), std::max<int64_t>(256, kPieceBytes / (N / 8 + 24) / 256 * 256));
  if (grad && p.piece < V) {  // of several pieces: the size whose products fill the CUs best
    double best = 0;
    for (int64_t i = 0; i < 16; ++i) {
      const int64_t grain = i < 8 ? 2048 : 256, at = i < 8 ? 16 - i : 24 - i;
      const int64_t c = most * at / 16 / grain * grain;
      if (c < 256) continue;
      const int64_t n = V / c, rest = V - n * c;
      const double us = (double)n * piece_cfg(N, H, c, p.np, 64).us + (rest ? piece_cfg(N, H, rest, p.np, 64).us : 0);
      if (best == 0 || us < best) best = us, p.piece = c;
    }
  }
  // W as it lies may still be unusable (its address): the packed piece has its place in any case.
  p.o_x = p.take(plane * N * p.Kp);
  p.o_w = p.take(plane * std::min(p.piece, V) * p.Kp);
  if (!grad) {
    const int64_t tiles = std::max(p.piece, p.direct_ok ? p.whole : 0) / 128;
    p.o_part = p.take(8 * N * tiles);
    p.o_party = p.take(8 * N * tiles);
    p.o_hit = p.take(4 * N);
    p.o_run = p.take(16 * N);
  } else {
    const int64_t vc = std::min(p.piece, V), rest = V % p.piece ? V % p.piece : vc;
    p.full = piece_cfg(N, H, vc, p.np, 64);
    // the last one adds to the sums that the others left
    p.last = rest == vc ? p.full : piece_cfg(N, H, rest, p.np, p.full.gx.splits);
    p.o_scale = p.take(4);
    p.o_p = p.take(plane * p.block * up(p.piece, kPad));
    p.ldacc = up(H, 4);
    p.o_gx = p.take(4 * std::max(p.full.gx.splits, p.last.gx.splits) * N * p.ldacc);
    const int64_t a = p.full.gw.splits > 1 ? p.full.gw.splits * vc : 0;
    const int64_t b = p.last.gw.splits > 1 ? p.last.gw.splits * rest : 0;
    p.o_gw = p.take(4 * std::max(a, b) * p.ldacc);
    p.o_b = p.take(4 * bias_rows(N) * vc);
  }
  return true;
}

// The product's tiles and steps; returns its workgroups: one for every place the chip has (LDS: one large or two small
// ones a CU), each with its share of the tiles.
template <int EPI, int NP>
unsigned lay_out(GemmArgs& a, const Cfg& cfg) {
  const Tile t = tile_of(cfg.tile, NP);
  a.tm = div_up(a.M, t.bm), a.tn = div_up(a.N, t.bn);
  a.kt = (int)steps_of(EPI, a.K, NP);
  a.splits = cfg.splits;
  a.per_split = (int)div_up(a.kt, cfg.splits);
  return (unsigned)std::min(a.tm * a.tn * cfg.splits, places(cfg.tile, NP) * kCus);
}

template <int EPI, bool F32>
void mm(GemmArgs a, const Cfg& cfg, hipStream_t st) {
  constexpr int NP = F32 ? 3 : 1;
  const dim3 grid(lay_out<EPI, NP>(a, cfg));
  const auto launch = [&](auto soft) {
    constexpr bool SOFT = decltype(soft)::value;
    if (cfg.tile == T_SMALL) {
      hipLaunchKernelGGL((k_xent_mm<128, 128, 2, 2, EPI, NP, F32, SOFT>), grid, dim3(256), 0, st, a);
      return;
    }
    if constexpr (EPI == E_LSE || EPI == E_DL) {
      if (cfg.tile == T_HALF) {
        hipLaunchKernelGGL((k_xent_mm<128, 64, 2, 2, EPI, NP, F32, SOFT>), grid, dim3(256), 0, st, a);
        return;
      }
    }
    if constexpr (F32)
      hipLaunchKernelGGL((k_xent_mm<256, 128, 4, 2, EPI, NP, F32, SOFT>), grid, dim3(512), 0, st, a);
    else if constexpr (EPI == E_GX)  // the wave's shorter side turned, 16 LDS reads a half-step instead of 20: 5 % faster
      hipLaunchKernelGGL((k_xent_mm<256, 256, 4, 2, EPI, NP, F32, SOFT>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((k_xent_mm<256, 256, 2, 4, EPI, NP, F32, SOFT>), grid, dim3(512), 0, st, a);
  };
  if constexpr (EPI == E_LSE || EPI == E_DL) {
    if (a.rows.kind == GNCDE_TARGET_ROWS) return launch(std::true_type{});
  }
  launch(std::false_type{});
}

bool aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Small tiles leave room for both: 2903 x 51 x 1293 takes 13 us for the two instead of 22.
template <bool F32>
void mm_both(GemmArgs x, const Cfg& cx, GemmArgs w, const Cfg& cw, hipStream_t st) {
  constexpr int NP = F32 ? 3 : 1;
  const unsigned gx = lay_out<E_GX, NP>(x, cx), gw = lay_out<E_GW, NP>(w, cw);
  hipLaunchKernelGGL((k_xent_both<NP, F32>), dim3(gx + gw), dim3(256), 0, st, x, w, gx);
}

struct Call {
  const void *x, *W, *b;
  Rows rows;
  char* ws;
  hipStream_t st;
};

template <bool F32>
struct Operand {
  const uint16_t* p;
  int64_t ld;
  int K;
};

// x and a piece of W as the products' operands: as they lie where their rows start on 16 bytes (x: and no row is to be
// put aside), else packed, both in one launch.  With an x from an earlier piece, W alone.  The scale of dl is found
// beside them.
template <bool F32>
void operands(const Plan& p, const Call& c, const void* W, int64_t vc, bool aside, const float* g, float* scale,
              Operand<F32>& x, Operand<F32>& w) {
  PackJob jx = {}, jw = {};
  const auto job = [&](const void* src, int64_t R, int64_t at, bool left, PackJob& j, Operand<F32>& o) {
    if (!left && p.direct_ok && aligned(src, 16)) {
      o = {static_cast<const uint16_t*>(src), p.H, (int)p.H};
      return;
    }
    j = {src, reinterpret_cast<uint16_t*>(c.ws + at), R, left, (uint32_t)std::min(div_up(R * (p.Kp / 8), 256), kMostBlocks)};
    o = {j.dst, p.np * p.Kp, (int)p.Kp};
  };
  if (!x.p) job(c.x, p.N, p.o_x, aside, jx, x);
  job(W, vc, p.o_w, false, jw, w);
  const uint32_t blocks = jx.blocks + jw.blocks + (scale ? 1 : 0);
  if (blocks)
    hipLaunchKernelGGL((k_xent_pack<F32, F32 ? 3 : 1>), dim3(blocks), dim3(256), 0, c.st, jx, jw, (int)p.H, (int)p.Kp, c.rows,
                       p.N, g, scale);
}

// The logits of classes v0 + at .. of a piece that starts at v0.
template <bool F32>
GemmArgs logits_args(const Operand<F32>& w, const Operand<F32>& x, const Plan& p, const Call& c, int64_t v0, int64_t at,
                     int64_t n) {
  GemmArgs a = {};
  a.A = w.p + at * w.ld, a.lda = w.ld, a.M = n;
  a.B = x.p, a.ldb = x.ld, a.N = p.N;
  // one of the two may be packed (zeros behind H) and the other not
  a.K = std::min(w.K, x.K);
  a.rows = c.rows;
  a.bias = c.b ? static_cast<const char*>(c.b) + (v0 + at) * (F32 ? 4 : 2) : nullptr;
  a.v0 = v0 + at, a.V = p.V;
  return a;
}

SmallArgs small_args(const Plan& p, const Call& c) {
  SmallArgs a = {};
  a.x = c.x, a.W = c.W, a.b = c.b, a.rows = c.rows;
  a.N = p.N, a.H = (int)p.H, a.V = (int)p.V;
  return a;
}

FewArgs few_args(const Plan& p, const Call& c) {
  FewArgs a = {};
  a.x = c.x, a.W = c.W, a.b = c.b, a.rows = c.rows;
  a.N = (int)p.N, a.H = (int)p.H, a.ks = p.ks, a.xs = p.xs;
  a.V = p.V, a.tiles = div_up(p.V, 16);
  return a;
}

template <bool F32>
void forward(const Plan& p, const Call& c, float* loss, float* stats) {
  if (p.few) {
    FewArgs a = few_args(p, c);
    a.part = reinterpret_cast<float2*>(c.ws + p.o_part);
    a.part_y = reinterpret_cast<float2*>(c.ws + p.o_party);
    a.hit = reinterpret_cast<float*>(c.ws + p.o_hit);
    hipLaunchKernelGGL((k_xent_few<F32, false>), dim3((unsigned)p.few_groups), dim3(kFewWaves * 64),
                       (unsigned)(p.N * p.xs * (F32 ? 4 : 2)), c.st, a);
    hipLaunchKernelGGL(k_xent_join, dim3((unsigned)div_up(p.N, 4)), dim3(256), 0, c.st, p.N, p.few_groups, a.part,
                       c.rows.kind == GNCDE_TARGET_ROWS ? a.part_y : nullptr, a.hit, c.rows, p.V, nullptr, 1, 1, loss,
                       stats);
    return;
  }
  if (p.small) {
    SmallArgs a = small_args(p, c);
    a.loss = loss, a.stats = stats;
    hipLaunchKernelGGL((k_xent_small<F32, false>), dim3((unsigned)std::min(div_up(p.N, 16), 8 * kCus)),
                       dim3(kSmallThreads), 0, c.st, a);
    return;
  }
  Operand<F32> x = {}, w = {};
  const int64_t piece = p.direct_ok && aligned(c.W, 16) ? p.whole : p.piece;
  for (int64_t v0 = 0; v0 < p.V; v0 += piece) {
    const int64_t vc = std::min(piece, p.V - v0);
    operands<F32>(p, c, static_cast<const char*>(c.W) + v0 * p.H * (F32 ? 4 : 2), vc, false, nullptr, nullptr, x, w);
    const Cover cv = cover(E_LSE, vc, p.N, steps_of(E_LSE, std::min(w.K, x.K), p.np), p.np);
    const int64_t tiles_a = div_up(cv.first, tile_of(cv.a.tile, p.np).bm);
    const int64_t tiles = tiles_a + (cv.first < vc ? div_up(vc - cv.first, tile_of(cv.b.tile, p.np).bm) : 0);
    for (int64_t at = 0; at < vc; at += cv.first) {
      GemmArgs a = logits_args<F32>(w, x, p, c, v0, at, at == 0 ? cv.first : vc - cv.first);
      a.part = reinterpret_cast<float2*>(c.ws + p.o_part);
      a.part_y = reinterpret_cast<float2*>(c.ws + p.o_party);
      a.part_ld = tiles, a.part_at = at == 0 ? 0 : tiles_a;
      a.hit = reinterpret_cast<float*>(c.ws + p.o_hit);
      mm<E_LSE, F32>(a, at == 0 ? cv.a : cv.b, c.st);
      if (at != 0) break;
    }
    hipLaunchKernelGGL(k_xent_join, dim3((unsigned)div_up(p.N, 4)), dim3(256), 0, c.st, p.N, tiles,
                       reinterpret_cast<const float2*>(c.ws + p.o_part),
                       c.rows.kind == GNCDE_TARGET_ROWS ? reinterpret_cast<const float2*>(c.ws + p.o_party) : nullptr,
                       reinterpret_cast<const float*>(c.ws + p.o_hit), c.rows, p.V,
                       reinterpret_cast<float4*>(c.ws + p.o_run), v0 == 0, v0 + piece >= p.V, loss, stats);
  }
}

// Sums on their way into one launch.
template <bool F32>
struct Sums {
  SumJobs jobs = {};
  int n = 0;

  void add(int64_t N, int64_t M, int64_t splits, const float* acc, int64_t ldacc, int64_t stride, const float* scale,
           void* out, int64_t ldo) {
    jobs.job[n++] = {N,     M,   ldacc, stride, ldo, acc, scale, out, (int32_t)splits,
                     (uint32_t)std::min(div_up(N * M, 256), kMostBlocks)};
  }
  void launch(hipStream_t st) {
    uint32_t blocks = 0;
    for (int i = 0; i < n; ++i) blocks += jobs.job[i].blocks;
    if (n) hipLaunchKernelGGL((k_xent_sum<F32>), dim3(blocks), dim3(256), 0, st, jobs);
    *this = {};
  }
};

template <bool F32>
void backward(const Plan& p, const Call& c, const float* stats, const float* g, void* gx, void* gW, void* gb) {
  constexpr int64_t SZ = F32 ? 4 : 2;
  if (p.small) {
    SmallArgs a = small_args(p, c);
    a.row_stats = stats, a.g = g, a.gx = gx;
    a.part = gW || gb ? reinterpret_cast<float*>(c.ws + p.o_b) : nullptr;
    const int groups = (int)small_groups(p.N);
    hipLaunchKernelGGL((k_xent_small<F32, true>), dim3(groups), dim3(kSmallThreads), 0, c.st, a);
    const int VH = a.V * a.H;
    if (a.part)
      hipLaunchKernelGGL((k_xent_parts_sum<F32>), dim3((unsigned)div_up(VH + a.V, 64)), dim3(1024), 0, c.st, groups, VH,
                         a.V, a.part, gW, gb);
    return;
  }
  if (p.few) {
    FewArgs a = few_args(p, c);
    a.stats = stats, a.g = g, a.gb = gb;
    a.d = reinterpret_cast<float*>(c.ws + p.o_p);
    hipLaunchKernelGGL((k_xent_few<F32, true>), dim3((unsigned)p.few_groups), dim3(kFewWaves * 64),
                       (unsigned)(p.N * p.xs * SZ), c.st, a);
    if (!gx && !gW) return;
    float* part = gx ? reinterpret_cast<float*>(c.ws + p.o_gx) : nullptr;
    const int64_t per = div_up(p.V, p.few_out), runs = div_up(p.V, per);
    const dim3 grid((unsigned)runs, (unsigned)div_up(p.H, 256 * few_cols(p.N)));
    const auto out = [&](auto rows, auto cols) {
      hipLaunchKernelGGL((k_xent_few_out<F32, decltype(rows)::value, decltype(cols)::value>), grid, dim3(256), 0, c.st, a.N,
                         a.H, p.V, per, a.d, c.x, c.W, c.rows, part, gW);
    };
    // rows that are not there cost products all the same: 2 rows of 1856 against 85678 classes take 258 us as 4, 170 as 2
    typedef std::integral_constant<int, 4> Four;
    typedef std::integral_constant<int, 8> Eight;
    if (p.N == 1) out(std::integral_constant<int, 1>(), Eight());
    else if (p.N == 2) out(std::integral_constant<int, 2>(), Eight());
    else if (p.N <= 4) out(Four(), Eight());
    else if (p.N <= 8) out(Eight(), Four());
    else out(std::integral_constant<int, 16>(), Four());
    if (gx)
      hipLaunchKernelGGL((k_xent_parts_sum<F32>), dim3((unsigned)div_up(p.N * p.H, 64)), dim3(1024), 0, c.st, (int)runs,
                         (int)(p.N * p.H), 0, part, gx, nullptr);
    return;
  }
  // Three parts take dl as it is: an entry is off by 2^-25 of itself or 2^-134, whichever is more, and with the largest
  // cotangent at 2^-110 or above (8e-34) the latter is below 2^-24 of that.
  float* scale = F32 ? nullptr : reinterpret_cast<float*>(c.ws + p.o_scale);
  // gW multiplies every row of x, by zeros where it is left out: those rows are put aside, whatever they hold
  const bool aside = gW && (c.rows.mask || c.rows.kind != GNCDE_TARGET_ROWS);
  Operand<F32> x = {}, w = {};
  uint16_t* P = reinterpret_cast<uint16_t*>(c.ws + p.o_p);
  float* acc_x = reinterpret_cast<float*>(c.ws + p.o_gx);
  float* acc_w = reinterpret_cast<float*>(c.ws + p.o_gw);
  float* part_b = reinterpret_cast<float*>(c.ws + p.o_b);
  const bool one = p.piece >= p.V;
  Sums<F32> sums;
  for (int64_t v0 = 0; v0 < p.V; v0 += p.piece) {
    const int64_t vc = std::min(p.piece, p.V - v0), vp = up(vc, kPad);
    const char* wsrc = static_cast<const char*>(c.W) + v0 * p.H * SZ;
    const PieceCfg& cfg = v0 + p.piece >= p.V ? p.last : p.full;
    operands<F32>(p, c, wsrc, vc, aside, g, v0 == 0 ? scale : nullptr, x, w);
    for (int64_t at = 0; at < vc; at += cfg.dl.first) {
      const int64_t len = at == 0 ? cfg.dl.first : vc - cfg.dl.first;
      GemmArgs a = logits_args<F32>(w, x, p, c, v0, at, len);
      a.stats = stats, a.g = g;
      a.scale = scale;
      a.P = P + p.np * at * p.block, a.block = p.block, a.mp = at + len < vc ? len : vp - at;
      a.part_b = gb ? part_b + bias_rows(p.N) * at : nullptr;
      const Cfg& one_cfg = at == 0 ? cfg.dl.a : cfg.dl.b;
      mm<E_DL, F32>(a, one_cfg, c.st);
      if (gb) {
        const Tile t = tile_of(one_cfg.tile, p.np);
        sums.add(1, len, div_up(p.N, t.bn) * t.wn, a.part_b, len, len, scale, static_cast<char*>(gb) + (v0 + at) * SZ, len);
      }
      if (at != 0) break;
    }
    GemmArgs to_x = {}, to_w = {};
    if (gx) {
      GemmArgs& q = to_x;
      q.scale = scale;
      q.A = w.p, q.lda = w.ld, q.M = p.H;
      q.B = P, q.block = p.block, q.N = p.N;
      q.K = (int)vc;
      q.out = gx, q.ldo = p.H;
      // every piece's splits fill the same sums; the last piece may have fewer, and leaves the others as they are
      const bool kept = !one || cfg.gx.splits > 1;
      if (kept) q.acc = acc_x, q.ldacc = p.ldacc, q.add = v0 > 0;
      if (kept && v0 + p.piece >= p.V)
        sums.add(p.N, p.H, one ? p.last.gx.splits : p.full.gx.splits, acc_x, p.ldacc, p.N * p.ldacc, nullptr, gx, p.H);
    }
    if (gW) {
      GemmArgs& q = to_w;
      q.scale = scale;
      q.A = x.p, q.lda = x.ld, q.M = p.H;
      q.B = P, q.block = p.block, q.N = vc;
      q.K = (int)p.N;
      char* out = static_cast<char*>(gW) + v0 * p.H * SZ;
      q.out = out, q.ldo = p.H;
      const int sp = cfg.gw.splits;
      if (sp > 1) {
        q.acc = acc_w, q.ldacc = p.ldacc;
        sums.add(vc, p.H, sp, acc_w, p.ldacc, vc * p.ldacc, nullptr, out, p.H);
      }
    }
    if (gx && gW && cfg.gx.tile == T_SMALL && cfg.gw.tile == T_SMALL) {
      mm_both<F32>(to_x, cfg.gx, to_w, cfg.gw, c.st);
    } else {
      if (gx) mm<E_GX, F32>(to_x, cfg.gx, c.st);
      if (gW) mm<E_GW, F32>(to_w, cfg.gw, c.st);
    }
    sums.launch(c.st);
  }
}

int check(int64_t rows, int64_t hidden, int64_t classes, int32_t dtype, const void* x, const void* W, const void* b,
          int32_t kind, const void* target, bool grad, const void* ws, size_t ws_bytes, Plan& p) {
  if (rows < 0 || hidden <= 0 || classes <= 0) return GNCDE_ERR_SHAPE;
  if (kind < GNCDE_TARGET_INDEX32 || kind > GNCDE_TARGET_ROWS) return GNCDE_ERR_ARG;
  if (!make_plan(rows, hidden, classes, dtype, grad, p)) return GNCDE_ERR_UNSUPPORTED;
  const int64_t sz = p.f32 ? 4 : 2, tsz = kind == GNCDE_TARGET_INDEX64 ? 8 : 4;
  if (!W || !aligned(W, sz) || !aligned(b, sz)) return GNCDE_ERR_ARG;
  if (rows > 0 && (!x || !target || !aligned(x, sz) || !aligned(target, tsz))) return GNCDE_ERR_ARG;
  if (rows > 0 && (!ws || !aligned(ws, 256) || ws_bytes < (size_t)p.bytes)) return GNCDE_ERR_WORKSPACE;
  return GNCDE_OK;
}

}  // namespace
}  // namespace gncde

extern "C" {

size_t gncde_linear_cross_entropy_workspace_bytes(int64_t rows, int64_t hidden, int64_t classes, int32_t dtype,
                                                  int32_t grad) {
  gncde::Plan p;
  return gncde::make_plan(rows, hidden, classes, dtype, grad != 0, p) ? (size_t)p.bytes : 0;
}

int gncde_linear_cross_entropy(int64_t rows, int64_t hidden, int64_t classes, int32_t dtype, const void* x,
                               const void* W, const void* b, int32_t target_kind, const void* target,
                               const uint8_t* mask, float* loss, float* stats, void* workspace,
                               size_t workspace_bytes, void* stream) {
  gncde::Plan p;
  const int rc = gncde::check(rows, hidden, classes, dtype, x, W, b, target_kind, target, false, workspace,
                              workspace_bytes, p);
  if (rc != GNCDE_OK) return rc;
  if (rows == 0) return GNCDE_OK;
  if (!loss || !stats) return GNCDE_ERR_ARG;
  const gncde::Call c{x, W, b, {target, mask, target_kind}, static_cast<char*>(workspace),
                      static_cast<hipStream_t>(stream)};
  if (p.f32) gncde::forward<true>(p, c, loss, stats);
  else gncde::forward<false>(p, c, loss, stats);
  return hipGetLastError() == hipSuccess ? GNCDE_OK : GNCDE_ERR_HIP;
}

int gncde_linear_cross_entropy_grad(int64_t rows, int64_t hidden, int64_t classes, int32_t dtype, const void* x,
                                    const void* W, const void* b, int32_t target_kind, const void* target,
                                    const uint8_t* mask, const float* stats, const float* g, void* gx, void* gW,
                                    void* gb, void* workspace, size_t workspace_bytes, void* stream) {
  gncde::Plan p;
  const int rc = gncde::check(rows, hidden, classes, dtype, x, W, b, target_kind, target, true, workspace,
                              workspace_bytes, p);
  if (rc != GNCDE_OK) return rc;
  const int64_t sz = p.f32 ? 4 : 2;
  if (!gncde::aligned(gx, sz) || !gncde::aligned(gW, sz) || !gncde::aligned(gb, sz)) return GNCDE_ERR_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows == 0) {  // no row: gradients of nothing
    const auto zeros = [&](auto sums) {
      if (gW) sums.add(classes, hidden, 0, nullptr, 0, 0, nullptr, gW, hidden);
      if (gb) sums.add(1, classes, 0, nullptr, 0, 0, nullptr, gb, classes);
      sums.launch(st);
    };
    if (p.f32) zeros(gncde::Sums<true>());
    else zeros(gncde::Sums<false>());
    return hipGetLastError() == hipSuccess ? GNCDE_OK : GNCDE_ERR_HIP;
  }
  if (!stats || !g) return GNCDE_ERR_ARG;
  if (!gx && !gW && !gb) return GNCDE_OK;
  const gncde::Call c{x, W, b, {target, mask, target_kind}, static_cast<char*>(workspace), st};
  if (p.f32) gncde::backward<true>(p, c, stats, g, gx, gW, gb);
  else gncde::backward<false>(p, c, stats, g, gx, gW, gb);
  return hipGetLastError() == hipSuccess ? GNCDE_OK : GNCDE_ERR_HIP;
}

}  // extern "C"

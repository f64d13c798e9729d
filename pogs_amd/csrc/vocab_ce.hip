// Softmax cross entropy of feature rows over a large vocabulary of embeddings, without keeping the logits but for few rows
// (pr_vocab_ce_fwd / pr_vocab_ce_bwd).
//
//   z_pv  = scale <x_p, w_v>          p < P rows, v < V words, contraction over D features
//   lse_p = log sum_v exp z_pv        loss_p = lse_p - z_p,label(p)
//   with upstream gradients u_p of loss_p and l_p of lse_p, a_p = u_p + l_p, b_p = u_p:
//   G_pv  = a_p exp(z_pv - lse_p) - b_p [v = label(p)],   dX = scale G W,   dW = scale G^T X
//
// Few rows have kernels of their own (below).  All other products run on the matrix cores as v_mfma_f32_32x32x16 with
// float32 accumulators.  Operands are packed once per call into fragment order, 1 KB blocks [32 rows][16 of the
// contraction] with lane l's eight values consecutive, so that a block moves memory -> LDS by one direct 16-byte-a-lane load
// and LDS -> registers by one conflict-free ds_read_b128.
//
// The logits' operands: 16-bit input is packed as it is.  A float32 value becomes two float16 planes, head and residual, after
// its row has been scaled by the power of two that brings its largest magnitude to 2^13..2^14 (22 bits down to 2^-15 of the
// row's largest, below that to 2^-38 of it); head*head + head*residual + residual*head lose 2^-22.  A logit is the product's
// accumulator times both rows' powers of two: a row or a word that is far larger than the others takes nothing from them.
// X takes the scale's sign.  Values that are not finite stay so; rows with the ignored label are packed as zeros, whatever they
// hold.
//
// The gradients' operands are bfloat16 pieces, which have float32's range: the entries of G go from the probability of a
// word that nobody means to the largest row's weight, so a row's or a word's gradient would be lost under a common scale in
// float16.  G is kept in two pieces (three for float32 input), to 2^-16 (2^-24) of each entry, below half a step of the
// output's type, as one piece of 8 or 11 bits would not be: the label's entry carries most of a word's gradient, and its
// rounding would show.  W and X are one piece (bfloat16), two (float16) or three (float32), which hold every bit of the packed
// value, and two, three and six products of pieces are made.
//
// One product kernel with four epilogues:
//   STATS  64 to 320 words x 256 rows: the row of X is on the lane, so the maximum and sum over the words are taken in
//          registers; one (max, sum) pair per row and wavefront leaves, in the log2 domain
//   GRAD   the same product again for a piece of the vocabulary, turned into the pieces of G.  A lane's eight accumulators
//          are eight consecutive slots of the contraction of dX = G W as they stand, if W's packed copy uses the same slot
//          order; for dW = G^T X the tile is transposed by two products with the identity, which are exact
//   DX     partials of a gradient in float32, one plane per split of its contraction; dX's are added to over the pieces.
//          Two such products may share a launch: dX's and, where dW has too few tiles for the chip, dW's
//   DW     dW rows of the piece, contraction over all rows, written in the output type
// G of one piece of the vocabulary is all that is ever held of the P x V logits.
//
// Bound: the matrix cores, at the clock that the chip's power allows (1.75 to 1.8 GHz under these kernels, of 2.4).
// 8192 rows x 131072 words x 1024 dims, bfloat16, loss and both gradients, 11.1 ms: STATS 1.75 ms (1260 TFLOP/s), and for
// each of eight pieces GRAD 0.39 (710, with 1 GB of G to write), DX 0.40 and DW 0.38 (1390 and 1450, two products each);
// packing 0.10, transposing 0.09.  A library product of 8192^3 bfloat16 runs at 1290 on the same card.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "common.h"

namespace pr {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));

constexpr int TILE_V = 256;  // words of the packed copies are padded to it
constexpr int TILE_P = 256;  // rows per workgroup; rows of the packed copies are padded to it
constexpr int CUS = 256;
constexpr int TOP_EXP = 13;  // packed magnitudes are below 2^(TOP_EXP + 1)
constexpr float MAX_FLOOR = -3.0e38f;  // a maximum over nothing: exp2 of anything minus it is 0, not NaN
constexpr float LN2F = 0.69314718055994531f;
// The kernels for few rows read the vocabulary once for the scores and once for dX, where the packed path reads it three
// times and writes it twice before its products; they multiply 32, 64 or 128 rows, whatever there are.  131072 words x 1024
// dims, loss and both gradients: 1 row 453 against 1589 us (bfloat16 212 against 817, float16 228 against 902), 128 rows 686
// against 1658 (333 against 839, 409 against 936); loss alone, 128 rows: 220 against 495 (74 against 175).  256 rows have no
// kernel here; two such passes would still take less than packing (1703 and 862 us with gradients).
constexpr int FEW_ROWS = 128;
// Below so many elements of the vocabulary there is little to gain (2000 words x 256 dims: 42 against 64 us on the GPU,
// less than the host takes), and the packed path's backward pass has its own copy of the vocabulary.
// Narrow tables gain more (both gradients, 1 M words x 16 dims: 8 rows 0.22 against 3.40 ms, 128 rows 0.57 against 3.41;
// bfloat16 0.16 and 0.43 against 2.63): their logits are wider than they are, 512 bytes a word for 128 rows, but so is what
// packing holds, 320 bytes (bfloat16 128) for 32 dims or fewer and 1 GB of G.
constexpr int64_t FEW_VOCABULARY = 1 << 19;
constexpr int SCORE_ROWS = 64;      // rows that they take from any vocabulary where no backward pass follows
constexpr int SCORE_BLOCKS = 1024;  // workgroups of the score kernel: four per CU
// Workgroups of the others, where there is work for so many: two per CU.  (One row to 128 of 131072 words x 1024 dims,
// bfloat16, loss and gradients, G's second piece cut off: 223 to 322 us; 256 workgroups 267 to 386, 1024 workgroups 223 to
// 359.)
constexpr int FEW_BLOCKS = 512;
constexpr int AMAX_BLOCKS = 1024;  // partial maxima per tensor at most

struct Matrix {  // rows x cols with any strides (elements)
  const void *data;
  int64_t rows, cols, ld_row, ld_col;
};

// Operands of a product A B^T as sums of NA and NB planes (or pieces) of type E.  Of the planes' products those are made
// whose numbers add up to less than the larger count.
template <typename E_, int NA_, int NB_>
struct Form {
  typedef E_ E;
  typedef E_ E8 __attribute__((ext_vector_type(8)));
  static constexpr int NA = NA_, NB = NB_, MOST = NA > NB ? NA : NB;
  static constexpr int KB = MOST == 1 ? 2 : 1;   // 16-wide blocks of the contraction in a stage
  static constexpr int PRODUCTS = NA == 1 || NB == 1 ? MOST : MOST * (MOST + 1) / 2;
};
template <typename T>
struct Types {  // bfloat16
  typedef Form<__bf16, 1, 1> Logits;
  typedef Form<__bf16, 1, 2> Grads;
};
template <>
struct Types<_Float16> {
  typedef Form<_Float16, 1, 1> Logits;
  typedef Form<__bf16, 2, 2> Grads;
};
template <>
struct Types<float> {
  typedef Form<_Float16, 2, 2> Logits;
  typedef Form<__bf16, 3, 3> Grads;
};

__device__ __forceinline__ f16v mfma(h8v a, h8v b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16v mfma(b8v a, b8v b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// v as N bfloat16 pieces, 8 bits of it each: all but the last by truncation, so that the largest values do not overflow, the
// last one rounded.  Three hold all of a float32 value, two all of a float16 one and any other to 2^-16.
template <int N>
__device__ __forceinline__ void bf16_pieces(const float (&v)[8], b8v (&out)[N]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int n = 0; n + 1 < N; ++n) {
    u4v w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned a = __builtin_bit_cast(unsigned, r[2 * i]), b = __builtin_bit_cast(unsigned, r[2 * i + 1]);
      w[i] = __builtin_amdgcn_perm(b, a, 0x07060302);   // the upper halves
      r[2 * i] -= __builtin_bit_cast(float, a & 0xffff0000u), r[2 * i + 1] -= __builtin_bit_cast(float, b & 0xffff0000u);
    }
    out[n] = __builtin_bit_cast(b8v, w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) out[N - 1][i] = (__bf16)r[i];
}

// A factor as mantissa and exponent: applied together with a power of two that brings a result back, so that neither their
// product with the other comes near the ends of float32.
struct Scale {
  float m;
  int e;
  __host__ static Scale of(float v) {
    Scale s;
    s.m = frexpf(v, &s.e);
    return s;
  }
  __device__ __forceinline__ float times(float v, int exponent) const { return ldexpf(v * m, e + exponent); }
};

struct Scalars {  // per call, on the device
  int exp_x, exp_w;  // the transposed copies are value * 2^exp
  float n_valid;     // rows whose label is not the ignored one
};

// ---- packing --------------------------------------------------------------------------------------------------------
template <typename T>
struct Eight;  // eight consecutive elements as one or two 16-byte accesses, at any element's address
template <>
struct Eight<float> {
  typedef float f4v __attribute__((ext_vector_type(4)));
  typedef f4v f4_at __attribute__((aligned(4)));
  f4v a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = reinterpret_cast<const f4_at *>(p)[0];
    b = reinterpret_cast<const f4_at *>(p)[1];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
};
template <typename T>
struct Eight {
  typedef u4v u4_at __attribute__((aligned(2)));
  u4v a;
  __device__ __forceinline__ void load(const T *p) { a = *reinterpret_cast<const u4_at *>(p); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 t = __builtin_bit_cast(t8, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  }
};

template <typename T>
__device__ __forceinline__ void load8(const Matrix &m, int64_t row, int64_t k, float (&v)[8]) {
  const T *src = (const T *)m.data + row * m.ld_row;
  if (m.ld_col == 1 && k + 8 <= m.cols) {
    Eight<T> e;
    e.load(src + k);
    e.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < m.cols ? (float)src[(k + i) * m.ld_col] : 0.f;
  }
}

struct AmaxJob {
  Matrix m;
  const int64_t *labels;  // rows with the ignored label do not count (NULL: all do)
  int64_t ignore;
  int blocks;             // workgroups, one partial each
  int64_t padded;         // rows of the packed copy
  int *exps;              // their exponents
};

__device__ __forceinline__ float block_max(float top) {
  __shared__ float part[4];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

constexpr int OF_ZEROS = 200;  // exponent of a row without a finite value but zeros: above all others

// Largest finite magnitude of each row of W, then of X, as the exponent that the row is packed with, and of all rows of a
// workgroup.  `lanes` lanes (a power of two) take a row, a wavefront four rows for each of their groups.
template <typename T>
__global__ void __launch_bounds__(256) vce_amax_kernel(AmaxJob w, AmaxJob x, int lanes, float *__restrict__ partial) {
  const bool first = (int)blockIdx.x < w.blocks;
  const AmaxJob &j = first ? w : x;
  const int block = (int)blockIdx.x - (first ? 0 : w.blocks);
  const int groups = 64 / lanes, lane = threadIdx.x & (lanes - 1);
  float all = 0.f;
  for (int64_t r0 = ((int64_t)block * 4 + (threadIdx.x >> 6)) * 4 * groups + (threadIdx.x & 63) / lanes; r0 < j.padded;
       r0 += (int64_t)j.blocks * 16 * groups) {
    float top[4] = {0.f, 0.f, 0.f, 0.f};
    bool live[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t row = r0 + q * groups;
      live[q] = row < j.m.rows && !(j.labels && j.labels[row] == j.ignore);
    }
    for (int64_t k = lane * 8; k < j.m.cols; k += lanes * 8) {
      float v[4][8];
      if (j.m.ld_col == 1 && (j.m.cols & 7) == 0) {   // four loads under way
        Eight<T> e[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) e[q].load((const T *)j.m.data + min(r0 + q * groups, j.m.rows - 1) * j.m.ld_row + k);
#pragma unroll
        for (int q = 0; q < 4; ++q) e[q].get(v[q]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) load8<T>(j.m, min(r0 + q * groups, j.m.rows - 1), k, v[q]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) top[q] = fabsf(v[q][i]) < INFINITY ? fmaxf(top[q], fabsf(v[q][i])) : top[q];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!live[q]) top[q] = 0.f;
      for (int d = lanes / 2; d > 0; d >>= 1) top[q] = fmaxf(top[q], __shfl_xor(top[q], d));
      if (lane == 0 && r0 + q * groups < j.padded) j.exps[r0 + q * groups] = top[q] > 0.f ? TOP_EXP - ilogbf(top[q]) : OF_ZEROS;
      all = fmaxf(all, top[q]);
    }
  }
  all = block_max(all);
  if (threadIdx.x == 0) partial[blockIdx.x] = all;
}

__device__ __forceinline__ int top_exponent(const float *partial, int n) {
  float top = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) top = fmaxf(top, partial[i]);
  top = block_max(top);
  return top > 0.f ? TOP_EXP - ilogbf(top) : 0;
}

struct PackJob {
  Matrix m;
  const int64_t *labels;  // rows with the ignored label are zeros (NULL: all count)
  int64_t ignore;
  u4v *dst;
  int64_t plane;    // 16-byte units between the head and the residual plane
  int64_t units;    // (32-row tile, 64 columns) pairs
  int kblocks;      // 16-wide blocks of the contraction per 32-row tile
  int partials;     // of the largest magnitude
  const int *exps;  // of the rows (NULL: values are packed as they are)
  float sign;
};

// A wavefront takes 32 rows x 64 columns: eight lanes read 128 (float32: 256) consecutive bytes of a row and store them
// to the four blocks' places, 128 consecutive bytes for eight rows.
// Block (tile t, k step s), lane (m, h): row 32 t + m, columns 16 s + 8 h + 0..7.
template <typename T>
__global__ void __launch_bounds__(256) vce_pack_kernel(PackJob w, PackJob x, const float *__restrict__ partial,
                                                       Scalars *__restrict__ s) {
  typedef typename Types<T>::Logits F;
  typedef typename F::E8 E8;
  const int ew = top_exponent(partial, w.partials), ex = top_exponent(partial + w.partials, x.partials);
  if (blockIdx.x == 0 && threadIdx.x == 0) s->exp_w = ew, s->exp_x = ex;
  const int lane = threadIdx.x & 63, piece = lane & 7;
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < w.units + x.units; u += (int64_t)gridDim.x * 4) {
    const bool first = u < w.units;
    const PackJob &j = first ? w : x;
    const unsigned groups = (j.kblocks + 3) / 4, v = (unsigned)(first ? u : u - w.units), at = v / groups;  // units < 2^31
    const int64_t tile = at, kb = (v - at * groups) * 4 + piece / 2, k = kb * 16 + (piece & 1) * 8;
    if (kb >= j.kblocks) continue;
    u4v *dst = j.dst + (tile * j.kblocks + kb) * 64 + (piece & 1) * 32 + lane / 8;
    float val[4][8];
    int e[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t row = tile * 32 + q * 8 + lane / 8;
      e[q] = j.exps ? j.exps[row] : 0;
      const bool live = row < j.m.rows && k < j.m.cols && !(j.labels && j.labels[row] == j.ignore);
#pragma unroll
      for (int i = 0; i < 8; ++i) val[q][i] = 0.f;
      if (live) load8<T>(j.m, row, k, val[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      E8 hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = ldexpf(val[q][i], e[q]) * j.sign;
        hi[i] = (typename F::E)f;
        if (F::NA == 2) lo[i] = (typename F::E)(f - (float)hi[i]);
      }
      dst[q * 8] = __builtin_bit_cast(u4v, hi);
      if (F::NA == 2) dst[q * 8 + j.plane] = __builtin_bit_cast(u4v, lo);
    }
  }
}

// Place of slot i of lane half h in k step s of a 32-wide piece of the contraction, for operands that come out of (or
// meet one that comes out of) an accumulator: the order in which a 32x32 accumulator tile holds its rows.
__device__ __forceinline__ constexpr int slot_place(int s, int h, int i) { return 16 * s + 8 * (i >> 2) + 4 * h + (i & 3); }

struct TransposeJob {
  const u4v *src;     // [32-row tile][k block], contraction over the columns
  u4v *dst;           // [32-column tile][row block], contraction over the rows, in slot order
  int64_t plane;      // of both: they hold the same number of blocks
  int64_t row_tiles, col_tiles;
  const int *exps, *exp;   // of the rows and of the copy (exps NULL: as they are)
};

// The packed copies for the contraction over rows, from those over columns: one 32x32 tile per wavefront, every plane as two
// products with the identity.  Each value passes the matrix core as itself times one and its planes add up to it: exact.
// Here rows have to share an exponent, the largest row's; the pieces have room for what that takes from the others.
template <typename T>
__device__ __forceinline__ void transpose_tiles(const TransposeJob &w, const TransposeJob &x, int64_t u, int64_t step) {
  typedef typename Types<T>::Logits F;
  typedef typename F::E8 E8;
  constexpr int FROM = F::NA, TO = Types<T>::Grads::NA;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int64_t nw = w.row_tiles * w.col_tiles, nx = x.row_tiles * x.col_tiles;
  E8 ident[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) ident[s][i] = 16 * s + 8 * h + i == (lane & 31) ? (typename F::E)1.f : (typename F::E)0.f;
  for (; u < nw + nx; u += step) {
    const bool first = u < nw;
    const TransposeJob &j = first ? w : x;
    const unsigned q = (unsigned)(first ? u : u - nw), by = q / (unsigned)j.col_tiles;                 // tiles < 2^31
    const int64_t rt = by, ct = q - by * (unsigned)j.col_tiles;
    const u4v *src = j.src + (rt * j.col_tiles + ct) * 128 + lane;
    f16v tr;
#pragma unroll
    for (int r = 0; r < 16; ++r) tr[r] = 0.f;
#pragma unroll
    for (int pl = 0; pl < FROM; ++pl)
#pragma unroll
      for (int s = 0; s < 2; ++s) tr = mfma(__builtin_bit_cast(E8, src[pl * j.plane + s * 64]), ident[s], tr);
    u4v *dst = j.dst + (ct * j.row_tiles + rt) * 128 + lane;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float v[8];
      b8v o[TO];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = tr[8 * s + k];
      if constexpr (FROM == 2) {   // every row to the copy's scale
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], *j.exp - j.exps[rt * 32 + slot_place(s, h, k)]);
      }
      bf16_pieces<TO>(v, o);
#pragma unroll
      for (int pl = 0; pl < TO; ++pl) dst[pl * j.plane + s * 64] = __builtin_bit_cast(u4v, o[pl]);
    }
  }
}

struct CoefJob {
  int64_t P, Pp, V, ignore;
  const int64_t *labels;
  const float *g_loss, *g_lse;  // either may be NULL
  int per_row, mean;
  const Scalars *s;
  const float2 *stat;
  int *exp_g;
  float *a, *b;
  const float *tops;   // largest factors of parts of the rows, or NULL: every workgroup looks for the largest itself
  int n_tops;
  // G = ra exp2(logit - maximum) - rb at the label: the sum of the exponentials goes into ra
  __device__ __forceinline__ void row(int64_t p, float one, float &ra, float &rb) const {
    ra = rb = 0.f;
    if (p >= P || labels[p] == ignore) return;
    rb = !g_loss ? 0.f : per_row ? g_loss[p] : one;
    ra = (rb + (g_lse ? g_lse[p] : 0.f)) / stat[p].y;
    if (g_loss && (labels[p] < 0 || labels[p] >= V)) ra = NAN;   // no such word: the row's loss is NaN
  }
  // the loss's gradient of every row, where it is one for all
  __device__ __forceinline__ float one() const {
    return g_loss && !per_row ? *g_loss * (mean ? 1.f / s->n_valid : 1.f) : 0.f;
  }
  __device__ __forceinline__ void largest(int64_t p, float one, float &top) const {
    float ra, rb;
    row(p, one, ra, rb);
    ra = fabsf(ra), rb = fabsf(rb);
    if (ra < INFINITY) top = fmaxf(top, ra);
    if (rb < INFINITY) top = fmaxf(top, rb);
  }
};
// Brings the largest factor to 2^12..2^13 (|G| <= |ra| + |rb|).
__device__ __forceinline__ int coef_exponent(float top) { return top > 0.f ? TOP_EXP - 1 - ilogbf(top) : 0; }

constexpr int COEF_ROWS = 4096;  // rows whose factors one workgroup writes

// The largest row factors of many rows, one a workgroup.
__global__ void __launch_bounds__(1024) vce_largest_kernel(CoefJob c, float *__restrict__ tops) {
  const float one = c.one();
  float top = 0.f;
  for (int64_t p = (int64_t)blockIdx.x * 1024 + threadIdx.x; p < c.P; p += (int64_t)gridDim.x * 1024) c.largest(p, one, top);
  __shared__ float part[16];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, part[i]);
  tops[blockIdx.x] = top;
}

// Row factors of G, scaled by coef_exponent.  With one gradient for all rows there is no largest to look for.
__device__ __forceinline__ void row_factors(const CoefJob &c, int block) {
  const float one = c.one();
  float top = fabsf(one) < INFINITY ? fabsf(one) : 0.f;
  if (c.per_row || c.g_lse) {
    if (c.tops) top = (int)threadIdx.x < c.n_tops ? fmaxf(top, c.tops[threadIdx.x]) : top;
    else
      for (int64_t p = threadIdx.x; p < c.P; p += 1024) c.largest(p, one, top);
    __shared__ float part[16];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = part[0];
    for (int i = 1; i < 16; ++i) top = fmaxf(top, part[i]);
  }
  const int e = coef_exponent(top);
  if (block == 0 && threadIdx.x == 0) *c.exp_g = e;
  const int64_t end = min((int64_t)(block + 1) * COEF_ROWS, c.Pp);
  for (int64_t p = (int64_t)block * COEF_ROWS + threadIdx.x; p < end; p += 1024) {
    float a, b;
    c.row(p, one, a, b);
    c.a[p] = ldexpf(a, e);
    c.b[p] = ldexpf(b, e);
  }
}

// What the gradients' products need besides the packed operands, in one launch: the first workgroups write the row
// factors, the others the transposed copies.
template <typename T>
__global__ void __launch_bounds__(1024) vce_prepare_kernel(CoefJob c, TransposeJob w, TransposeJob x) {
  const int coef_blocks = (int)((c.Pp + COEF_ROWS - 1) / COEF_ROWS);
  if ((int)blockIdx.x < coef_blocks) {
    row_factors(c, blockIdx.x);
    return;
  }
  transpose_tiles<T>(w, x, (int64_t)(blockIdx.x - coef_blocks) * 16 + (threadIdx.x >> 6),
                     (int64_t)(gridDim.x - coef_blocks) * 16);
}

// ---- products -------------------------------------------------------------------------------------------------------
struct GemmArgs {
  const u4v *A, *B;            // operand blocks, already at the first block of the contraction
  int64_t plane_a, plane_b;    // 16-byte units between planes
  int64_t ld_a, ld_b;          // blocks per 32-row tile
  int a_tiles, b_tiles;        // 32-row tiles A and B have (tiles past them repeat the last one; results are not used)
  int kblocks, k_split;        // blocks of the contraction, and of each split of it (the last one may have fewer)
  int m_tiles, n_tiles, splits;
  const Scalars *scal;
  const int *exp_g;            // DW: packed gradient = G * 2^exp_g
  Scale scale;
  // STATS, GRAD: logit in the log2 domain = accumulator * 2^(exp_c - exps_a[word] - exps_b[row]) * c
  const int *exps_a, *exps_b;  // float32 input: from the first word of the piece on, and of the rows
  int exp_c;
  float c;
  int64_t P, V, v0;            // v0: first word of the piece
  const int64_t *labels;
  float2 *partial;             // STATS: [pair][Pp]
  float *target;               // STATS: [Pp], the label's logit in the log2 domain
  int64_t Pp;
  const float2 *stat;          // GRAD: maximum and sum of every row
  const float *coef_a, *coef_b;
  u4v *gx, *gw;                // GRAD: G as the operand of DX and of DW (either may be NULL)
  int64_t plane_gx, plane_gw, ld_gx, ld_gw;
  // DX
  float *acc;                  // [split][Pp][ld_acc]
  int64_t ld_acc;
  int add;
  // DW
  void *out;                   // [V][D], contiguous
  int64_t D;
};

typedef __attribute__((address_space(1))) const void *global_ptr;
typedef __attribute__((address_space(3))) void *lds_ptr;

template <typename T>
__device__ __forceinline__ void store4(T *dst, float a, float b, float c, float d) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<t4 *>(dst) = t4{(T)a, (T)b, (T)c, (T)d};
}

enum { STATS, GRAD, DX, DW };
template <typename T, int MODE>
struct FormOf {
  typedef typename Types<T>::Grads F;
};
template <typename T>
struct FormOf<T, STATS> {
  typedef typename Types<T>::Logits F;
};
template <typename T>
struct FormOf<T, GRAD> {
  typedef typename Types<T>::Logits F;
};
template <typename F, int MT>
constexpr int STAGE_BLOCKS = F::KB * (F::NA * 2 * MT + F::NB * 8);   // of 1 KB

// Eight wavefronts, 2 x 4, of MT x 2 accumulator tiles each: 64 MT rows of A by 256 rows of B.  LDS holds three stages of
// 16 or (one plane each) 32 of the contraction, filled by direct loads two stages ahead.  The wavefronts form two
// groups, one wavefront of each on every SIMD, that take turns between barriers: one reads its next stage from LDS while
// the other multiplies.  One workgroup a CU, which takes tile after tile and starts the next one's loads before it turns
// to the epilogue.
template <typename T, int MT, int MODE>
__global__ void __launch_bounds__(512, 2) vce_gemm_kernel(const GemmArgs g, const GemmArgs g2) {
#pragma clang fp contract(off)   // products are rounded before they are subtracted (the logits, below)
  extern __shared__ u4v lds[];
  typedef typename FormOf<T, MODE>::F F;
  typedef typename F::E8 E8;
  constexpr int WM = 2, WN = 4, NT = 2, WAVES = WM * WN, KB = F::KB, NA = F::NA, NB = F::NB;
  constexpr int A_TILES = WM * MT, B_TILES = WN * NT, A_BLOCKS = KB * NA * A_TILES;
  constexpr int STAGE = STAGE_BLOCKS<F, MT>, LOADS = (STAGE + WAVES - 1) / WAVES;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  const bool late = wave >= WAVES / 2;
  constexpr bool SCALED = (MODE == STATS || MODE == GRAD) && NA == 2;
  __shared__ __attribute__((aligned(16))) int word_exp[SCALED ? 2 : 1][SCALED ? 64 * MT : 1];   // of this tile and the next

  // Workgroups go to the eight XCDs in turn: each XCD takes a run of consecutive tiles, ordered as bands of eight
  // M tiles walked along N, so that its L2 holds the operands of the tiles it works on together.
  const unsigned tiles1 = (unsigned)g.m_tiles * g.n_tiles * g.splits;
  const unsigned tiles = tiles1 + (MODE == DX ? (unsigned)g2.m_tiles * g2.n_tiles * g2.splits : 0u), per_xcd = (tiles + 7) / 8;
  const unsigned lo = (blockIdx.x & 7) * per_xcd, hi = min(lo + per_xcd, tiles);
  unsigned tile = lo + (blockIdx.x >> 3);
  if (tile >= hi) return;

  int m_tile, n_tile, split, stages;
  bool other;             // DX: the tile is of the second product
  const u4v *src[LOADS];  // this wavefront's blocks of a stage, ordered [k block][plane][tile] for A, then for B
  auto place = [&](unsigned t) {
    other = MODE == DX && t >= tiles1;
    if (other) t -= tiles1;
    const unsigned m_tiles = other ? g2.m_tiles : g.m_tiles, n_tiles = other ? g2.n_tiles : g.n_tiles;
    const int k_split = other ? g2.k_split : g.k_split, kblocks = other ? g2.kblocks : g.kblocks;
    const int a_tiles = other ? g2.a_tiles : g.a_tiles, b_tiles = other ? g2.b_tiles : g.b_tiles;
    const u4v *A = other ? g2.A : g.A, *B = other ? g2.B : g.B;
    const int64_t plane_a = other ? g2.plane_a : g.plane_a, plane_b = other ? g2.plane_b : g.plane_b;
    const int64_t ld_a = other ? g2.ld_a : g.ld_a, ld_b = other ? g2.ld_b : g.ld_b;
    split = (int)(t / (m_tiles * n_tiles));
    t -= split * m_tiles * n_tiles;
    const unsigned band = t / (8u * n_tiles), in_band = t - band * 8u * n_tiles;
    const unsigned band_m = min(8u, m_tiles - band * 8u);
    m_tile = (int)(band * 8u + in_band % band_m), n_tile = (int)(in_band / band_m);
    stages = min(k_split, kblocks - split * k_split) / KB;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int j = min(wave * LOADS + l, STAGE - 1);  // (a share past the end repeats the last block, into its own place)
      const bool is_a = j < A_BLOCKS;
      const int q = is_a ? j : j - A_BLOCKS, per = is_a ? A_TILES : B_TILES, planes = is_a ? NA : NB;
      const int at = q % per, kb = q / per / planes, plane = q / per % planes;
      const int64_t row = is_a ? min(m_tile * A_TILES + at, a_tiles - 1) : min(n_tile * B_TILES + at, b_tiles - 1);
      const u4v *base = is_a ? A + plane * plane_a + row * ld_a * 64 : B + plane * plane_b + row * ld_b * 64;
      src[l] = base + ((int64_t)split * k_split + kb) * 64;
    }
  };
  auto fill = [&](int buf) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int j = min(wave * LOADS + l, STAGE - 1);
      __builtin_amdgcn_global_load_lds((global_ptr)(src[l] + lane), (lds_ptr)(lds + (buf * STAGE + j) * 64), 16, 0, 0);
      src[l] += KB * 64;
    }
    asm volatile("" ::: "memory");   // fills stay in order: the waits below count on it
  };
  struct Block {  // of the contraction
    E8 a[NA][MT], b[NB][NT];
  };
  auto read = [&](int buf, int kb, Block &f) {
    const u4v *sa = lds + (buf * STAGE + kb * NA * A_TILES + wm * MT) * 64 + lane;
    const u4v *sb = lds + (buf * STAGE + A_BLOCKS + kb * NB * B_TILES + wn * NT) * 64 + lane;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n) f.b[j][n] = __builtin_bit_cast(E8, sb[(j * B_TILES + n) * 64]);
#pragma unroll
    for (int j = 0; j < NA; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) f.a[j][i] = __builtin_bit_cast(E8, sa[(j * A_TILES + i) * 64]);
  };
  f16v acc[MT][NT];
  auto multiply = [&](const Block &f) {
#pragma unroll
    for (int sum = 0; sum < F::MOST; ++sum)     // the sum of the planes' numbers; more would be left out
#pragma unroll
      for (int j = 0; j < NA && j <= sum; ++j)
        if (sum - j < NB) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[i][n] = mfma(f.a[j][i], f.b[sum - j][n], acc[i][n]);
        }
  };
  // Waits for all but the youngest fill of this wavefront (`more`: there is one) and for its own LDS reads; after the
  // barrier both hold for all wavefronts that have come to it.
  auto arrive = [&](bool more) {
    if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  place(tile);
  fill(0);
  if (stages > 1) fill(1);
  for (int turn = 0;; turn ^= 1) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][n][r] = 0.f;
    const int m0 = (m_tile * WM + wm) * 32 * MT;                                   // first row of A of this wavefront
    const int64_t n0 = ((int64_t)n_tile * WN + wn) * 32 * NT + (lane & 31);        // this lane's row of B, tile 0
    const int of_split = split, of_m = m_tile, of_n = n_tile;
    const bool of_other = other;
    // what the epilogue needs of its rows, ahead of the loads that it would wait for otherwise
    int place_of[NT];             // the label's place among this wavefront's words, or something out of their range
    float top2[NT], coef_a[NT], coef_b[NT];
    int row_exp[NT];
    if constexpr (SCALED) {
      // (the other half is still being read by wavefronts that are an epilogue behind; they are done before the next write)
      if ((int)threadIdx.x < 64 * MT) word_exp[turn][threadIdx.x] = g.exps_a[min(m_tile * 64 * MT + (int)threadIdx.x, g.a_tiles * 32 - 1)];
#pragma unroll
      for (int n = 0; n < NT; ++n) row_exp[n] = g.exp_c - g.exps_b[n0 + 32 * n];
    }
    if constexpr (MODE == STATS || MODE == GRAD) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int64_t p = n0 + 32 * n, rel = (p < g.P ? g.labels[p] : -1) - (g.v0 + m0);
        place_of[n] = rel >= 0 && rel < 32 * MT ? (int)rel : -32;
        if constexpr (MODE == GRAD) top2[n] = g.stat[p].x, coef_a[n] = g.coef_a[p], coef_b[n] = g.coef_b[p];
      }
    }
    arrive(stages > 1);
    if (late) __builtin_amdgcn_s_barrier();    // the second group is one barrier behind
    int buf = 0;
    for (int st = 0; st < stages; ++st) {
      Block f[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) read(buf, kb, f[kb]);
      // into the stage before this one: this group has read it two barriers ago, the other one barrier ago
      if (st + 2 < stages) fill(buf == 0 ? 2 : buf - 1);
      __builtin_amdgcn_sched_barrier(0);
      // the stage after this one: this group reads it two barriers from now, and the other group waits for its loads of
      // it before the barrier in between
      arrive(st + 2 < stages);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) multiply(f[kb]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      buf = buf == 2 ? 0 : buf + 1;
    }
    if (!late) __builtin_amdgcn_s_barrier();   // in step again: every wavefront has read the last stage
    asm volatile("" ::: "memory");

    tile += gridDim.x >> 3;
    const bool again = tile < hi;
    if (again) {
      place(tile);
      fill(0);
      if (stages > 1) fill(1);
    }
    // accumulator register r of tile (i, n): row m0 + 32 i + (r & 3) + 8 (r >> 2) + 4 h of A, row n0 + 32 n of B

    if constexpr (MODE == STATS || MODE == GRAD) {
      const float c = g.c;
      // words of this wavefront that exist, from this lane's first one on: compared with constants below
      const int left = (int)min(g.V - (g.v0 + m0), (int64_t)(32 * MT)) - 4 * h;
      const bool whole = g.V - (g.v0 + m0) >= 32 * MT;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int64_t p = n0 + 32 * n;
        if constexpr (SCALED) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int4 e = *reinterpret_cast<const int4 *>(&word_exp[turn][wm * 32 * MT + 32 * i + 8 * q + 4 * h]);
              acc[i][n][4 * q] = ldexpf(acc[i][n][4 * q], row_exp[n] - e.x);
              acc[i][n][4 * q + 1] = ldexpf(acc[i][n][4 * q + 1], row_exp[n] - e.y);
              acc[i][n][4 * q + 2] = ldexpf(acc[i][n][4 * q + 2], row_exp[n] - e.z);
              acc[i][n][4 * q + 3] = ldexpf(acc[i][n][4 * q + 3], row_exp[n] - e.w);
            }
        }
        const bool mine = place_of[n] >= 0;
        const int at = place_of[n] - 4 * h;    // from this lane's first word on; the other half's places match no constant
        const bool here = __any(mine);
        // Logits, rounded: maximum, exponentials and G have to mean the same number, or the difference of logits of 2^24 and
        // more is not that of equal ones.
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][n][r] *= c;
        if constexpr (MODE == STATS) {
          if (here) {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r) z = at == 32 * i + (r & 3) + 8 * (r >> 2) ? acc[i][n][r] : z;
            if (mine && (at & 4) == 0) g.target[p] = z;
          }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (32 * i + (r & 3) + 8 * (r >> 2) >= left) acc[i][n][r] = -INFINITY;
          }
          float top = acc[0][n][0];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][n][r]);
          top = fmaxf(top, __shfl_xor(top, 32));
          top = fmaxf(top, MAX_FLOOR);
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(acc[i][n][r] - top);
          sum += __shfl_xor(sum, 32);
          if (h == 0) g.partial[(int64_t)(of_m * WM + wm) * g.Pp + p] = make_float2(top, sum);
        } else {
          const float m2 = top2[n], ca = coef_a[n], cb = coef_b[n];
          constexpr int NG = Types<T>::Grads::NB;
          b8v ident[2];
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) ident[s][i] = slot_place(s, h, i) == (lane & 31) ? (__bf16)1.f : (__bf16)0.f;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            float v[2][8];     // register r: slot r & 7 of step r >> 3
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r >> 3][r & 7] = ca * __builtin_amdgcn_exp2f(acc[i][n][r] - m2);
            if (here) {
#pragma unroll
              for (int r = 0; r < 16; ++r) v[r >> 3][r & 7] -= at == 32 * i + (r & 3) + 8 * (r >> 2) ? cb : 0.f;
            }
            if (!whole) {
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (32 * i + (r & 3) + 8 * (r >> 2) >= left) v[r >> 3][r & 7] = 0.f;
            }
            b8v f[2][NG];
#pragma unroll
            for (int s = 0; s < 2; ++s) bf16_pieces<NG>(v[s], f[s]);
            const int64_t pt = ((int64_t)of_n * WN + wn) * NT + n, vt = m0 / 32 + i;
            if (vt >= g.a_tiles) continue;     // past the piece
#pragma unroll
            for (int pl = 0; pl < NG; ++pl) {
              if (g.gx) {
                u4v *dst = g.gx + pl * g.plane_gx + (pt * g.ld_gx + vt * 2) * 64 + lane;
#pragma unroll
                for (int s = 0; s < 2; ++s) dst[s * 64] = __builtin_bit_cast(u4v, f[s][pl]);
              }
              if (g.gw) {
                f16v tr;
#pragma unroll
                for (int r = 0; r < 16; ++r) tr[r] = 0.f;
#pragma unroll
                for (int s = 0; s < 2; ++s) tr = mfma(f[s][pl], ident[s], tr);
                u4v *dst = g.gw + pl * g.plane_gw + (vt * g.ld_gw + pt * 2) * 64 + lane;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                  b8v o;
#pragma unroll
                  for (int k = 0; k < 8; ++k) o[k] = (__bf16)tr[8 * s + k];
                  dst[s * 64] = __builtin_bit_cast(u4v, o);
                }
              }
            }
          }
        }
      }
    } else if constexpr (MODE == DX) {
      const int64_t rows = of_other ? g2.Pp : g.Pp, ld = of_other ? g2.ld_acc : g.ld_acc;
      float *const to = (of_other ? g2.acc : g.acc) + ((int64_t)of_split * rows + n0) * ld;
      const bool add = of_other ? g2.add : g.add;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int d = m0 + 32 * i + 8 * q + 4 * h;
            if (d >= ld) continue;
            float4 *dst = reinterpret_cast<float4 *>(to + 32 * n * ld + d);
            float4 v = make_float4(acc[i][n][4 * q], acc[i][n][4 * q + 1], acc[i][n][4 * q + 2], acc[i][n][4 * q + 3]);
            if (add) {
              const float4 o = *dst;
              v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
            }
            *dst = v;
          }
      }
    } else {
      const int e = -(*g.exp_g + g.scal->exp_x);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int64_t v = g.v0 + n0 + 32 * n;
        if (v >= g.V) continue;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int d = m0 + 32 * i + 8 * q + 4 * h;
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = g.scale.times(acc[i][n][4 * q + k], e);
            T *dst = (T *)g.out + v * g.D + d;
            if ((g.D & 3) == 0) {
              if (d < g.D) store4<T>(dst, x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (d + k < g.D) dst[k] = (T)x[k];
            }
          }
      }
    }
    if (!again) return;
  }
}

// ---- few rows -------------------------------------------------------------------------------------------------------
// At most 32 NB rows: the vocabulary is read as it is, and nothing of its size is packed.  For the scores 16-bit operands go
// to the matrix cores in their own type; a float32 value is cut into three bfloat16 pieces that hold all its 24 bits (by
// truncation, so the largest values do not overflow), six products of which leave out less than 2^-21 of a product.  The
// gradients' operands are bfloat16 pieces as in the packed path: float16's range would lose rows of small weight.
//   SCORE   logits, maxima and sums of 32 words a wavefront.  For a backward pass the logits stay, 4 bytes for each word and
//           row: at 32 rows a 32nd of a float32 vocabulary of 1024 dims.
//   DX      32 words a step, 64 features a wavefront and 256 a workgroup, whose wavefronts make G of the step in LDS
//           together; reads the vocabulary once.  Partials per run of words, added by FINISH.
//   DW      32 words a wavefront: G of all rows is made from the logits in registers and multiplies the features, a 32- or
//           64-wide chunk at a time, which the workgroup shares through LDS, three stages deep.  Writes dW once.
// Bound: HBM for the fewest rows (131072 words x 1024 dims, one row: float32 SCORE 140 us, DX 112, DW 120 for 537 MB each,
// 3.8 to 4.8 TB/s; bfloat16 53, 65 and 54 for 268 MB, float16 80 and 56 for the gradients), the matrix cores and the
// conversions more and more from 64 rows on (128 rows: float32 205, 259 and 252 us; bfloat16 70, 134 and 114; float16, whose
// features take two pieces and DW so much LDS that a CU holds one workgroup, 154 and 203 for the gradients).  After a DW its
// lines are still on their way out of the cache, which a SCORE waits for (float32 210 us instead of 140).
template <typename T>
struct Operand;  // the pieces of eight consecutive values, ready for the matrix cores
template <>
struct Operand<float> {
  static constexpr int N = 3;
  u4v piece[N];
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned a[3], b[3];
      cut(v[2 * i], a), cut(v[2 * i + 1], b);
#pragma unroll
      for (int k = 0; k < 3; ++k) piece[k][i] = __builtin_amdgcn_perm(b[k], a[k], 0x07060302);  // the upper halves
    }
  }
  static __device__ __forceinline__ void cut(float v, unsigned (&p)[3]) {
    p[0] = __builtin_bit_cast(unsigned, v) & 0xffff0000u;
    v -= __builtin_bit_cast(float, p[0]);
    p[1] = __builtin_bit_cast(unsigned, v) & 0xffff0000u;
    p[2] = __builtin_bit_cast(unsigned, v - __builtin_bit_cast(float, p[1]));
  }
  static __device__ __forceinline__ f16v product(const Operand &a, const Operand &b, f16v acc) {
#pragma unroll
    for (int n = 2; n >= 0; --n)     // smallest first
#pragma unroll
      for (int k = 0; k <= n; ++k)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a.piece[k]),
                                                      __builtin_bit_cast(b8v, b.piece[n - k]), acc, 0, 0, 0);
    return acc;
  }
};
template <>
struct Operand<_Float16> {
  static constexpr int N = 1;
  u4v piece[N];
  __device__ __forceinline__ void set(const float (&v)[8]) {
    h8v z;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = (_Float16)v[i];
    piece[0] = __builtin_bit_cast(u4v, z);
  }
  static __device__ __forceinline__ f16v product(const Operand &a, const Operand &b, f16v acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a.piece[0]), __builtin_bit_cast(h8v, b.piece[0]),
                                                  acc, 0, 0, 0);
  }
};
template <>
struct Operand<__bf16> {
  static constexpr int N = 1;
  u4v piece[N];
  __device__ __forceinline__ void set(const float (&v)[8]) {
    b8v z;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = (__bf16)v[i];
    piece[0] = __builtin_bit_cast(u4v, z);
  }
  static __device__ __forceinline__ f16v product(const Operand &a, const Operand &b, f16v acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a.piece[0]), __builtin_bit_cast(b8v, b.piece[0]),
                                                   acc, 0, 0, 0);
  }
};

// Eight values of a gradient's operand in bfloat16 pieces, as in the packed path.
template <int N_>
struct Pieces {
  static constexpr int N = N_;
  u4v piece[N];
  __device__ __forceinline__ void set(const float (&v)[8]) {
    b8v o[N];
    bf16_pieces<N>(v, o);
#pragma unroll
    for (int k = 0; k < N; ++k) piece[k] = __builtin_bit_cast(u4v, o[k]);
  }
};
template <typename T>
using Factor = Pieces<Types<T>::Grads::NA>;        // of W or X
template <typename T>
using GradOperand = Pieces<Types<T>::Grads::NB>;   // of G
template <int NA, int NB>
__device__ __forceinline__ f16v times(const Pieces<NB> &g, const Pieces<NA> &x, f16v acc) {
#pragma unroll
  for (int n = (NA > NB ? NA : NB) - 1; n >= 0; --n)     // smallest first
#pragma unroll
    for (int k = 0; k <= n; ++k)
      if (k < NB && n - k < NA)
        acc = mfma(__builtin_bit_cast(b8v, g.piece[k]), __builtin_bit_cast(b8v, x.piece[n - k]), acc);
  return acc;
}

// Elements k..k+7 of a row as they are.  WIDE (unit column stride, eight columns at least): by 16-byte accesses.  Where
// they cross the end of the row the last eight columns are read in their place: few_column says which column a place holds,
// and the other factor is zero where that is one of an earlier place or none.
__device__ __forceinline__ int64_t few_column(int64_t k, int64_t cols) { return cols < 8 ? k : min(k, cols - 8); }
template <typename T, bool WIDE>
__device__ __forceinline__ Eight<T> fetch8(const Matrix &m, int64_t row, int64_t k) {
  const T *src = (const T *)m.data + row * m.ld_row;
  if (WIDE) {
    Eight<T> e;
    e.load(src + min(k, m.cols - 8));
    return e;
  }
  typedef T t8 __attribute__((ext_vector_type(8)));
  t8 z;
  const int64_t c = few_column(k, m.cols);
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = src[min(c + i, m.cols - 1) * m.ld_col];
  return __builtin_bit_cast(Eight<T>, z);
}
__device__ __forceinline__ Operand<float> operand(const Eight<float> &e) {
  float v[8];
  e.get(v);
  Operand<float> o;
  o.set(v);
  return o;
}
template <typename T>
__device__ __forceinline__ Operand<T> operand(const Eight<T> &e) {
  return Operand<T>{{e.a}};
}
template <typename O>
__device__ __forceinline__ O packed_operand(const u4v *src) {  // pieces 1 KB apart
  O o;
#pragma unroll
  for (int k = 0; k < O::N; ++k) o.piece[k] = src[k * 64];
  return o;
}
template <typename O>
__device__ __forceinline__ void store_operand(const O &o, u4v *dst) {
#pragma unroll
  for (int k = 0; k < O::N; ++k) dst[k * 64] = o.piece[k];
}

// Column of a 32-wide tile's lane, in the products whose columns are features: float32 tiles are 32 consecutive ones; two
// 16-bit tiles share 64, the even ones and the odd ones, so that a lane reads and writes both at once.
template <typename T>
__device__ __forceinline__ int64_t tile_column(int64_t tile, int lane) {
  return sizeof(T) == 4 ? tile * 32 + (lane & 31) : (tile >> 1) * 64 + 2 * (lane & 31) + (tile & 1);
}

struct FewPack {
  Matrix x;
  const int64_t *labels;  // rows with the ignored label are zeros
  int64_t ignore;
  int kblocks, row_blocks;  // 16 wide, of features and of rows
  u4v *xf, *xt;             // [32 rows][k block], [32 features][row block], pieces of 1 KB; either may be NULL
};

// A block of a packed copy of the features per wavefront.
template <typename T>
__global__ void __launch_bounds__(256) vce_few_pack_kernel(const FewPack j) {
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), nf = j.xf ? (int64_t)j.row_blocks / 2 * j.kblocks : 0;
  auto at = [&](int64_t row, int64_t col) {
    return row < j.x.rows && j.labels[row] != j.ignore ? (float)((const T *)j.x.data)[row * j.x.ld_row + col * j.x.ld_col] : 0.f;
  };
  float v[8];
  if (u < nf) {
    Operand<T> o;
    const int64_t n = u / j.kblocks, k = (u - n * j.kblocks) * 16 + 8 * h, c = few_column(k, j.x.cols);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i >= k && c + i < j.x.cols ? at(32 * n + (lane & 31), c + i) : 0.f;
    o.set(v);
    store_operand(o, j.xf + u * (Operand<T>::N * 64) + lane);
  } else if (j.xt && u - nf < (int64_t)j.kblocks / 2 * j.row_blocks) {
    const int64_t tile = (u - nf) / j.row_blocks, b = u - nf - tile * j.row_blocks, d = tile_column<T>(tile, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = d < j.x.cols ? at(16 * b + 8 * h + i, d) : 0.f;
    Factor<T> o;
    o.set(v);
    store_operand(o, j.xt + (u - nf) * (Factor<T>::N * 64) + lane);
  }
}

__device__ __forceinline__ void merge(float &m, float &s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  s = s * __builtin_amdgcn_exp2f(m - top) + s2 * __builtin_amdgcn_exp2f(m2 - top);
  m = top;
}

// SCORE for a small vocabulary: a workgroup takes 32 words at a time; its four wavefronts take the 64-wide pieces of the
// contraction in turn, add their tiles through LDS, and each keeps the running maximum and sum over a quarter of the words.
// XP: the features are packed (xf); otherwise they are read as they are, eight aligned columns at a time (D % 8 == 0), which
// saves a launch where it counts, with the fewest rows.
template <typename T, int NB, bool WIDE, bool XP>
__global__ void __launch_bounds__(256, 2) vce_score_kernel(Matrix w, Matrix x, const u4v *__restrict__ xf,
                                                           const int64_t *__restrict__ labels, int64_t ignore, float scale,
                                                           float2 *__restrict__ partial, float *__restrict__ target,
                                                           float *__restrict__ logits) {
#pragma clang fp contract(off)   // as in the product kernel
  constexpr int NJ = NB < 2 ? NB : 2;   // 32-row tiles that are added at once
  __shared__ float sum[4][NJ][16][64];
  __shared__ float2 join[4][NB][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const float c = scale * LOG2E;
  int64_t label[NB];
  float top[NB], tot[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int64_t p = 32 * n + (lane & 31);
    label[n] = p < x.rows ? labels[p] : -1;
    top[n] = MAX_FLOOR, tot[n] = 0.f;
  }
  const int64_t row = min((int64_t)(lane & 31), x.rows - 1);             // !XP
  const bool counts = label[0] != ignore && (lane & 31) < x.rows;
  const int64_t tiles = (w.rows + 31) / 32;
  const int groups = (int)((w.cols + 63) / 64);
  auto words = [&](int64_t t, int g, Eight<T> (&a)[4]) {
    const int64_t v = min(t * 32 + (lane & 31), w.rows - 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = fetch8<T, WIDE>(w, v, (int64_t)g * 64 + 16 * q + 8 * h);
  };
  Eight<T> a[4], next[4];
  if (wave < groups) words(blockIdx.x, wave, a);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    f16v acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][r] = 0.f;
    for (int g = wave; g < groups; g += 4) {
      // what comes next, of these words or of the next tile's, is on its way while this is multiplied and joined
      if (g + 4 < groups) words(t, g + 4, next);
      else if (t + gridDim.x < tiles) words(t + gridDim.x, wave, next);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const Operand<T> oa = operand(a[q]);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          Operand<T> ob;
          if (XP) {
            ob = packed_operand<Operand<T>>(xf + (((int64_t)n * groups + g) * 4 + q) * (Operand<T>::N * 64) + lane);
          } else {
            const int64_t k = (int64_t)g * 64 + 16 * q + 8 * h;
            ob = operand(fetch8<T, true>(x, row, k));
            const unsigned keep = counts && k < x.cols ? ~0u : 0u;
#pragma unroll
            for (int pc = 0; pc < Operand<T>::N; ++pc) ob.piece[pc] &= keep;
          }
          acc[n] = Operand<T>::product(oa, ob, acc[n]);
        }
        a[q] = next[q];
      }
    }
    // this wavefront's registers 4 wave..4 wave + 3: words 8 wave + 4 h + 0..3 of the tile
    const int64_t v0 = t * 32 + 8 * wave + 4 * h;
#pragma unroll
    for (int n0 = 0; n0 < NB; n0 += NJ) {
      __syncthreads();  // what was added before has been read
#pragma unroll
      for (int n = 0; n < NJ; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[wave][n][r][lane] = acc[n0 + n][r];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int n = n0 + j;
        float z[4], most = MAX_FLOOR;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 4 * wave + k;
          z[k] = ((sum[0][j][r][lane] + sum[1][j][r][lane]) + (sum[2][j][r][lane] + sum[3][j][r][lane])) * c;
          if (label[n] == v0 + k) target[32 * n + (lane & 31)] = z[k];
          if (v0 + k < w.rows) most = fmaxf(most, z[k]);
        }
        if (logits) store4<float>(logits + (t * 32 * NB + 32 * n + (lane & 31)) * 32 + 8 * wave + 4 * h, z[0], z[1], z[2], z[3]);
        float add = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) add += v0 + k < w.rows ? __builtin_amdgcn_exp2f(z[k] - most) : 0.f;
        merge(top[n], tot[n], most, add);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    merge(top[n], tot[n], __shfl_xor(top[n], 32), __shfl_xor(tot[n], 32));
    if (h == 0) join[wave][n][lane] = make_float2(top[n], tot[n]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * NB; i += 256) {
    float2 q = join[0][i / 32][i & 31];
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      const float2 o = join[k][i / 32][i & 31];
      merge(q.x, q.y, o.x, o.y);
    }
    if (i < x.rows) partial[(int64_t)i * gridDim.x + blockIdx.x] = q;
  }
}

template <typename T>
constexpr int few_blocks = sizeof(T) == 4 ? 2 : 4;     // 16-wide blocks in 128 bytes of a row
constexpr size_t score_lds(int nb, int blocks, int pieces) { return (size_t)2 * nb * blocks * pieces * 1024; }

// SCORE where there are enough words for the chip at 128 a workgroup: a wavefront has 32 words and the whole contraction,
// 128 bytes of each word's row at a time, and the four share the features' operands through LDS, where each wavefront of the
// kernel above reads all of them from L2 for every 32 words.
template <typename T, int NB, bool WIDE>
__global__ void __launch_bounds__(256, 2) vce_score_shared_kernel(Matrix w, int64_t rows, const u4v *__restrict__ xf,
                                                                  const int64_t *__restrict__ labels, float scale,
                                                                  float2 *__restrict__ partial, float *__restrict__ target,
                                                                  float *__restrict__ logits) {
#pragma clang fp contract(off)   // as in the product kernel
  typedef Operand<T> O;
  constexpr int Q = few_blocks<T>, STAGE = NB * Q * O::N, LOADS = (STAGE + 3) / 4;
  extern __shared__ u4v lds[];    // two stages
  __shared__ float2 join[4][NB][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const float c = scale * LOG2E;
  int label[NB];
  float top[NB], tot[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int64_t p = 32 * n + (lane & 31), y = p < rows ? labels[p] : -1;
    label[n] = y >= 0 && y < w.rows ? (int)y : -1;
    top[n] = MAX_FLOOR, tot[n] = 0.f;
  }
  const int64_t tiles = (w.rows + 127) / 128;
  const int chunks = (int)((w.cols + 63) / 64) * (4 / Q);
  auto fill = [&](int k, int buf) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int j = min(wave + 4 * l, STAGE - 1), n = j / (Q * O::N), at = j % (Q * O::N);   // (past the end: as in DW)
      __builtin_amdgcn_global_load_lds((global_ptr)(xf + ((int64_t)(n * chunks + k) * (Q * O::N) + at) * 64 + lane),
                                       (lds_ptr)(lds + (buf * STAGE + j) * 64), 16, 0, 0);
    }
    asm volatile("" ::: "memory");
  };
  auto words = [&](int64_t t, int k, Eight<T> (&a)[Q]) {
    const int64_t v = min(t * 128 + 32 * wave + (lane & 31), w.rows - 1);
#pragma unroll
    for (int q = 0; q < Q; ++q) a[q] = fetch8<T, WIDE>(w, v, (int64_t)k * (16 * Q) + 16 * q + 8 * h);
  };
  Eight<T> a[Q], next[Q];
  fill(0, 0);
  words(blockIdx.x, 0, a);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int buf = 0;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    f16v acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][r] = 0.f;
    for (int k = 0; k < chunks; ++k) {
      // the next chunk, of these words or of the next tile's, into the stage that was read before the last barrier
      const bool last = k + 1 == chunks;
      if (!last || t + gridDim.x < tiles) {
        fill(last ? 0 : k + 1, buf ^ 1);
        words(last ? t + gridDim.x : t, last ? 0 : k + 1, next);
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const O oa = operand(a[q]);
#pragma unroll
        for (int n = 0; n < NB; ++n)
          acc[n] = O::product(oa, packed_operand<O>(lds + (buf * STAGE + (n * Q + q) * O::N) * 64 + lane), acc[n]);
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __syncthreads();
      buf ^= 1;
#pragma unroll
      for (int q = 0; q < Q; ++q) a[q] = next[q];
    }
    const int64_t v0 = t * 128 + 32 * wave;
    const int left = (int)min(w.rows - v0, (int64_t)32) - 4 * h;     // words that exist, from this lane's first one on
    if (v0 >= w.rows) continue;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int at = label[n] - (int)v0 - 4 * h;
      float most = MAX_FLOOR;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[n][r] *= c;
        if (at == (r & 3) + 8 * (r >> 2)) target[32 * n + (lane & 31)] = acc[n][r];
        most = (r & 3) + 8 * (r >> 2) < left ? fmaxf(most, acc[n][r]) : most;
      }
      if (logits)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          store4<float>(logits + (v0 * NB + 32 * n + (lane & 31)) * 32 + 8 * q + 4 * h, acc[n][4 * q], acc[n][4 * q + 1],
                        acc[n][4 * q + 2], acc[n][4 * q + 3]);
      float add = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        add += (r & 3) + 8 * (r >> 2) < left ? __builtin_amdgcn_exp2f(acc[n][r] - most) : 0.f;
      merge(top[n], tot[n], most, add);
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    merge(top[n], tot[n], __shfl_xor(top[n], 32), __shfl_xor(tot[n], 32));
    if (h == 0) join[wave][n][lane] = make_float2(top[n], tot[n]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * NB; i += 256) {
    float2 q = join[0][i / 32][i & 31];
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      const float2 o = join[k][i / 32][i & 31];
      merge(q.x, q.y, o.x, o.y);
    }
    if (i < rows) partial[(int64_t)i * gridDim.x + blockIdx.x] = q;
  }
}

struct FewGrad {  // what G is made of
  CoefJob c;      // P, V, labels, upstream gradients
  int64_t D, Dk;
  const float *logits;
  // Row p as {maximum, ra, rb, label's bits}, made by every workgroup for itself (256 threads; a launch would cost more).
  __device__ __forceinline__ void rows(float4 *to, int n) const {
    const float one = c.one();
    for (int p = threadIdx.x; p < n; p += 256) {
      float a, b;
      c.row(p, one, a, b);
      const int64_t label = p < c.P ? c.labels[p] : -1;
      to[p] = make_float4(p < c.P ? c.stat[p].x : 0.f, a, b, __builtin_bit_cast(float, label >= 0 && label < c.V ? (int)label : -1));
    }
  }
  static __device__ __forceinline__ float entry(float z, const float4 &row, int word) {
    const float g = row.y * __builtin_amdgcn_exp2f(z - row.x);
    return __builtin_bit_cast(int, row.w) == word ? g - row.z : g;
  }
};

// A chunk of features of DW: a tile of 32, or a 16-bit pair of tiles.
template <typename T>
constexpr int few_tiles = sizeof(T) == 4 ? 1 : 2;
constexpr size_t dw_lds(int nb, int tiles, int pieces) { return (size_t)3 * 2 * nb * tiles * pieces * 1024; }

template <typename T, int NB>
__global__ void __launch_bounds__(256, 2) vce_few_dw_kernel(const FewGrad f, const u4v *__restrict__ xt, float scale,
                                                            T *__restrict__ out) {
  typedef Factor<T> X;
  constexpr int KB = 2 * NB, NT = few_tiles<T>, STAGE = NT * KB * X::N, LOADS = (STAGE + 3) / 4;
  __shared__ float4 rows[32 * NB];
  extern __shared__ u4v lds[];    // three stages, of a chunk of the features' operands each
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int64_t chunks = (f.D + 32 * NT - 1) / (32 * NT);
  auto fill = [&](int64_t c, int buf) {
    const u4v *src = xt + c * (STAGE * 64) + lane;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int j = min(wave + 4 * l, STAGE - 1);   // (past the end: the last block again, into its own place)
      __builtin_amdgcn_global_load_lds((global_ptr)(src + j * 64), (lds_ptr)(lds + (buf * STAGE + j) * 64), 16, 0, 0);
    }
    asm volatile("" ::: "memory");
  };
  fill(blockIdx.y, 0);
  if (blockIdx.y + gridDim.y < chunks) fill(blockIdx.y + gridDim.y, 1);
  f.rows(rows, 32 * NB);
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * 4 + wave, at = min(t, (f.c.V - 1) / 32);   // (past the end: not stored)
  GradOperand<T> ga[KB];
  const float *z = f.logits + at * (1024 * NB) + 256 * h + (lane & 31);
  float v[KB][8];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[b][i] = z[(16 * b + i) * 32];
#pragma unroll
  for (int b = 0; b < KB; ++b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[b][i] = FewGrad::entry(v[b][i], rows[16 * b + 8 * h + i], (int)(at * 32) + (lane & 31));
    ga[b].set(v[b]);
    // a block at a time: the row factors of all of them would not fit in registers
#pragma unroll
    for (int k = 0; k < GradOperand<T>::N; ++k) asm volatile("" : "+v"(ga[b].piece[k])::"memory");
    __builtin_amdgcn_sched_barrier(0);
  }
  const bool whole = t * 32 + 32 <= f.c.V;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  int buf = 0;
  for (int64_t c = blockIdx.y; c < chunks; c += gridDim.y) {
    // two chunks ahead, into the stage that was read before the last barrier
    const bool more = c + 2 * (int64_t)gridDim.y < chunks;
    if (more) fill(c + 2 * (int64_t)gridDim.y, buf == 0 ? 2 : buf - 1);
    f16v acc[2];     // of two tiles, or of the even and the odd blocks of one
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
    X x[2];
    x[0] = packed_operand<X>(lds + buf * STAGE * 64 + lane);
#pragma unroll
    for (int i = 0; i < NT * KB; ++i) {
      if (i + 1 < NT * KB) x[(i + 1) & 1] = packed_operand<X>(lds + (buf * STAGE + (i + 1) * X::N) * 64 + lane);
      const int j = NT == 1 ? i & 1 : i / KB;
      acc[j] = times(ga[i % KB], x[i & 1], acc[j]);
    }
    // all but the youngest fill have come, and what was written a chunk ago; this chunk's stores have until the next wait
    if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    buf = buf == 2 ? 0 : buf + 1;
    const int64_t d = tile_column<T>(NT * c, lane);
    if (d >= f.D) continue;
    T *dst = out + (t * 32 + 4 * h) * f.D + d;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int v = (r & 3) + 8 * (r >> 2);
      if (!whole && t * 32 + 4 * h + v >= f.c.V) continue;
      if constexpr (NT == 1) {
        dst[v * f.D] = (acc[0][r] + acc[1][r]) * scale;
      } else {
        typedef T t2 __attribute__((ext_vector_type(2)));
        const t2 g = {(T)(acc[0][r] * scale), (T)(acc[1][r] * scale)};
        if ((f.D & 1) == 0) {
          *reinterpret_cast<t2 *>(dst + v * f.D) = g;
        } else {
          dst[v * f.D] = g.x;
          if (d + 1 < f.D) dst[v * f.D + 1] = g.y;
        }
      }
    }
  }
}

// WIDE (unit column stride, two columns at least): a lane's two 16-bit columns by one access.
template <typename T, int NB, bool WIDE>
__global__ void __launch_bounds__(256, 2) vce_few_dx_kernel(const FewGrad f, Matrix w, int64_t steps,
                                                            float *__restrict__ acc_out) {
  typedef GradOperand<T> G;
  constexpr int R = 32 * NB, TASKS = (2 * NB + 3) / 4;     // (16 words, 32 rows) tiles of G for each wavefront
  constexpr bool PAIRS = sizeof(T) == 2;
  __shared__ float4 rows[R];
  __shared__ u4v g[2][2 * NB][G::N][64];
  f.rows(rows, R);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int64_t lo = blockIdx.y * steps, hi = min(lo + steps, (f.c.V + 31) / 32);
  const int64_t c0 = (int64_t)blockIdx.x * 256 + 64 * wave;
  const bool active = c0 < f.D;
  // this lane's two columns; the last ones again past the end
  const int64_t d0 = tile_column<T>(c0 / 32, lane), d1 = tile_column<T>(c0 / 32 + 1, lane);
  const int64_t at0 = WIDE && PAIRS ? min(d0, f.D - 2) : min(d0, f.D - 1), at1 = min(d1, f.D - 1);
  const unsigned shift = d0 == f.D - 1 ? 16 : 0;           // WIDE pairs: the last column of an odd number
  typedef unsigned u1_at __attribute__((aligned(2)));
  struct Raw {
    unsigned a[8], b[PAIRS && WIDE ? 1 : 8];
  };
  auto load = [&](int64_t step, int kb, Raw &raw) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T *src = (const T *)w.data + min(step * 32 + 16 * kb + 8 * h + i, f.c.V - 1) * w.ld_row;
      if constexpr (!PAIRS) {
        raw.a[i] = __builtin_bit_cast(unsigned, src[at0 * w.ld_col]);
        raw.b[i] = __builtin_bit_cast(unsigned, src[at1 * w.ld_col]);
      } else if constexpr (WIDE) {
        raw.a[i] = *reinterpret_cast<const u1_at *>(src + at0) >> shift;
      } else {
        raw.a[i] = __builtin_bit_cast(unsigned short, src[at0 * w.ld_col]);
        raw.b[i] = __builtin_bit_cast(unsigned short, src[at1 * w.ld_col]);
      }
    }
  };
  auto operands = [&](const Raw &raw, Factor<T> (&o)[2]) {
    if constexpr (Factor<T>::N == 2) {   // float16
      float v[2][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[0][i] = (float)__builtin_bit_cast(T, (unsigned short)raw.a[i]);
        v[1][i] = (float)__builtin_bit_cast(T, (unsigned short)(WIDE ? raw.a[i] >> 16 : raw.b[PAIRS && WIDE ? 0 : i]));
      }
      o[0].set(v[0]), o[1].set(v[1]);
    } else if constexpr (!PAIRS) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, raw.a[i]);
      o[0].set(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, raw.b[i]);
      o[1].set(v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[0].piece[0][i] = __builtin_amdgcn_perm(raw.a[2 * i + 1], raw.a[2 * i], 0x05040100);
        o[1].piece[0][i] = WIDE ? __builtin_amdgcn_perm(raw.a[2 * i + 1], raw.a[2 * i], 0x07060302)
                                : __builtin_amdgcn_perm(raw.b[PAIRS && WIDE ? 0 : 2 * i + 1], raw.b[PAIRS && WIDE ? 0 : 2 * i], 0x05040100);
      }
    }
  };
  struct Logits {
    float4 a[TASKS], b[TASKS];
  };
  auto logits = [&](int64_t step, Logits &z) {
#pragma unroll
    for (int k = 0; k < TASKS; ++k) {
      const int task = wave + 4 * k;
      if (task < 2 * NB) {
        const float *src = f.logits + (step * R + 32 * (task >> 1) + (lane & 31)) * 32 + 16 * (task & 1) + 8 * h;
        z.a[k] = reinterpret_cast<const float4 *>(src)[0], z.b[k] = reinterpret_cast<const float4 *>(src)[1];
      }
    }
  };
  auto make = [&](int64_t step, const Logits &z, int buf) {
#pragma unroll
    for (int k = 0; k < TASKS; ++k) {
      const int task = wave + 4 * k;
      if (task < 2 * NB) {
        const float4 row = rows[32 * (task >> 1) + (lane & 31)];
        const float v[8] = {z.a[k].x, z.a[k].y, z.a[k].z, z.a[k].w, z.b[k].x, z.b[k].y, z.b[k].z, z.b[k].w};
        const int word = (int)step * 32 + 16 * (task & 1) + 8 * h;
        float entry[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) entry[i] = word + i < f.c.V ? FewGrad::entry(v[i], row, word + i) : 0.f;
        G o;
        o.set(entry);
        store_operand(o, &g[buf][task][0][lane]);
      }
    }
  };
  f16v acc[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][j][r] = 0.f;
  Logits z;
  Raw raw[2];
  logits(lo, z);
  if (active) load(lo, 0, raw[0]);
  make(lo, z, 0);
  __syncthreads();
  int buf = 0;
  for (int64_t s = lo; s < hi; ++s) {
    const bool more = s + 1 < hi;
    if (more) logits(s + 1, z);
    if (active) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        if (kb == 0) load(s, 1, raw[1]);
        else if (more) load(s + 1, 0, raw[0]);
        Factor<T> o[2];
        operands(raw[kb], o);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const G ga = packed_operand<G>(&g[buf][2 * n + kb][0][lane]);
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[n][j] = times(ga, o[j], acc[n][j]);
        }
      }
    }
    if (more) make(s + 1, z, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  if (!active) return;
  float *dst = acc_out + (int64_t)blockIdx.y * R * f.Dk;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float *to = dst + (int64_t)(32 * n + (r & 3) + 8 * (r >> 2) + 4 * h) * f.Dk;
      if (PAIRS) *reinterpret_cast<float2 *>(to + d0) = make_float2(acc[n][0][r], acc[n][1][r]);
      else to[d0] = acc[n][0][r], to[d1] = acc[n][1][r];
    }
}

// dX = scale times the sum of the runs' partials, added in a fixed order: a row's 256 features per workgroup.
template <typename T>
__global__ void __launch_bounds__(1024) vce_few_finish_kernel(const FewGrad f, int64_t plane, int splits, float scale,
                                                              const float *__restrict__ acc, T *__restrict__ dx) {
  __shared__ float4 part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t p = blockIdx.y, d = (int64_t)blockIdx.x * 256 + 4 * lane;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < f.Dk)
#pragma unroll 8
    for (int k = wave; k < splits; k += 16) {
      const float4 q = *reinterpret_cast<const float4 *>(acc + k * plane + p * f.Dk + d);
      v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
    }
  part[wave][lane] = v;
  __syncthreads();
  if (wave != 0) return;
  for (int k = 1; k < 16; ++k) {
    const float4 q = part[k][lane];
    v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
  }
  const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (d + k < f.D) dx[p * f.D + d + k] = (T)(x[k] * scale);
}

// ---- rows -----------------------------------------------------------------------------------------------------------
struct RowsOut {
  int64_t P, V, ignore;
  const int64_t *labels;
  const float *target;
  float2 *stat;                  // maximum and sum of exp2(logit - maximum), log2 domain; may be NULL
  float *lse, *row_loss;         // lse may be NULL
};

__device__ __forceinline__ void finish_row(const RowsOut &o, int64_t p, float m, float s) {
  if (o.stat) o.stat[p] = p < o.P ? make_float2(m, s) : make_float2(0.f, 1.f);
  if (p >= o.P) return;
  const int64_t label = o.labels[p];
  const bool in = label != o.ignore;
  const float l = log2f(s);
  if (o.lse) o.lse[p] = in ? (m + l) * LN2F : 0.f;
  // a label outside the vocabulary has no logit: the row's loss is NaN
  o.row_loss[p] = !in ? 0.f : label < 0 || label >= o.V ? NAN : (l + (m - o.target[p])) * LN2F;
}

// Joins the (max, sum) pairs of the rows, [pair][Pp]: 8 rows x 32 lanes per workgroup.
__global__ void __launch_bounds__(256) vce_join_kernel(RowsOut o, int64_t Pp, int pairs, const float2 *__restrict__ partial) {
  const int row = threadIdx.x & 7, lane = threadIdx.x >> 3;
  const int64_t p = (int64_t)blockIdx.x * 8 + row;
  float m = MAX_FLOOR, s = 0.f;
#pragma unroll 4
  for (int j = lane; j < pairs; j += 32) {
    const float2 q = partial[(int64_t)j * Pp + p];
    merge(m, s, q.x, q.y);
  }
  __shared__ float2 part[32][8];
  part[lane][row] = make_float2(m, s);
  __syncthreads();
  for (int d = 16; d > 0; d >>= 1) {
    if (lane < d) {
      const float2 q = part[lane + d][row];
      merge(m, s, q.x, q.y);
      part[lane][row] = make_float2(m, s);
    }
    __syncthreads();
  }
  if (lane == 0) finish_row(o, p, m, s);
}

// The same for [row][pair], one row per workgroup.
__global__ void __launch_bounds__(256) vce_join_row_kernel(RowsOut o, int pairs, const float2 *__restrict__ partial) {
  const float2 *src = partial + (int64_t)blockIdx.x * pairs;
  float m = MAX_FLOOR, s = 0.f;
#pragma unroll 4
  for (int j = threadIdx.x; j < pairs; j += 256) merge(m, s, src[j].x, src[j].y);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) merge(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
  __shared__ float2 part[4];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x != 0) return;
  m = part[0].x, s = part[0].y;
#pragma unroll
  for (int k = 1; k < 4; ++k) merge(m, s, part[k].x, part[k].y);
  finish_row(o, blockIdx.x, m, s);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[16];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) v += part[i];
  return v;
}

__global__ void __launch_bounds__(1024) vce_reduce_kernel(int64_t P, const float *__restrict__ row_loss,
                                                          const int64_t *__restrict__ labels, int64_t ignore, int mean,
                                                          float *__restrict__ loss, Scalars *s) {
  double sum = 0., n = 0.;
  for (int64_t p = threadIdx.x; p < P; p += 1024) {
    sum += (double)row_loss[p];
    n += labels[p] != ignore ? 1. : 0.;
  }
  sum = block_sum(sum);
  n = block_sum(n);
  if (threadIdx.x != 0) return;
  if (s) s->n_valid = (float)n;
  *loss = (float)(mean ? sum / n : sum);
}

// Both for few rows, [row][pair]: a wavefront takes a row at a time, one workgroup all of them.
__global__ void __launch_bounds__(1024) vce_join_reduce_kernel(RowsOut o, int pairs, const float2 *__restrict__ partial,
                                                               int mean, float *__restrict__ loss, Scalars *sc) {
  const int lane = threadIdx.x & 63;
  for (int64_t p = threadIdx.x >> 6; p < o.P; p += 16) {
    const float2 *src = partial + p * pairs;
    float m = MAX_FLOOR, s = 0.f;
#pragma unroll 8
    for (int j = lane; j < pairs; j += 64) merge(m, s, src[j].x, src[j].y);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) merge(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
    if (lane == 0) finish_row(o, p, m, s);
  }
  __syncthreads();
  double sum = 0., n = 0.;
  for (int64_t p = threadIdx.x; p < o.P; p += 1024) {
    sum += (double)o.row_loss[p];
    n += o.labels[p] != o.ignore ? 1. : 0.;
  }
  sum = block_sum(sum);
  n = block_sum(n);
  if (threadIdx.x != 0) return;
  if (sc) sc->n_valid = (float)n;
  *loss = (float)(mean ? sum / n : sum);
}

struct FinishJob {
  int64_t rows, D, plane, ld;  // rows of the result; rows of a split and their stride in `acc`
  int splits;
  Scale scale;
  const float *acc;
  const int *exp_other, *exp_g;
  void *out;
};

// Rows of a gradient = sum of the splits, scaled, in the output type: a row per wavefront, four features per lane.  Up to
// two gradients a launch.
template <typename T>
__global__ void __launch_bounds__(256) vce_finish_kernel(const FinishJob a, const FinishJob b) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const bool first = row < a.rows;
  const FinishJob &j = first ? a : b;
  const int64_t p = first ? row : row - a.rows;
  if (p >= j.rows) return;
  const int e = -(*j.exp_g + *j.exp_other);
  for (int64_t d = (threadIdx.x & 63) * 4; d < j.D; d += 256) {
    const float *src = j.acc + p * j.ld + d;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < j.splits; ++k) {
      const float4 q = *reinterpret_cast<const float4 *>(src + k * j.plane * j.ld);
      v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
    }
    const float x[4] = {j.scale.times(v.x, e), j.scale.times(v.y, e), j.scale.times(v.z, e), j.scale.times(v.w, e)};
    T *dst = (T *)j.out + p * j.D + d;
    if ((j.D & 3) == 0) {
      store4<T>(dst, x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < j.D) dst[k] = (T)x[k];
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
int64_t round_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

struct Shape {
  int64_t P, V, D, Pp, Vp, Dk;
  int np, na, ng;   // planes of the logits' operands; pieces of the gradients' operands and of G
  Shape(int dtype, int64_t P_, int64_t V_, int64_t D_)
      : P(P_), V(V_), D(D_), Pp(round_up(P_, TILE_P)), Vp(round_up(V_, TILE_V)), Dk(round_up(D_, 32)) {
    if (dtype == PR_F32) of<float>();
    else if (dtype == PR_F16) of<_Float16>();
    else of<__bf16>();
  }
  template <typename T>
  void of() {
    np = Types<T>::Logits::NA, na = Types<T>::Grads::NA, ng = Types<T>::Grads::NB;
  }
  int64_t plane(int64_t rows) const { return rows * Dk / 8; }   // 16-byte units of one packed plane
};

bool valid_shape(int dtype, int64_t P, int64_t V, int64_t D) {
  return dtype >= PR_F32 && dtype <= PR_BF16 && P >= 0 && V >= 1 && D >= 1 && P < (1ll << 30) && V < (1ll << 30) &&
         D < (1ll << 20) && P * D < (1ll << 38) && V * D < (1ll << 38);
}

// Whether a call goes to the kernels for few rows, with a backward pass to come or without.
bool few(int64_t P, int64_t V, int64_t D) { return P <= FEW_ROWS && V * D >= FEW_VOCABULARY; }

struct Carve {  // consecutive 256-byte-aligned pieces of a buffer
  char *at;
  size_t used = 0;
  explicit Carve(void *base) : at((char *)base) {}
  template <typename T>
  T *take(int64_t n) {
    T *p = (T *)(at ? at + used : nullptr);
    used += (size_t)round_up((int64_t)sizeof(T) * n, 256);
    return p;
  }
};

struct Kept {  // what the forward pass leaves for the backward pass
  Scalars *scal;
  float2 *stat;
  u4v *xf, *wf;
  int *ex, *ew;   // float32: exponents of the packed rows
  Kept(Carve &c, const Shape &s) {
    scal = c.take<Scalars>(1);
    stat = c.take<float2>(s.Pp);
    xf = c.take<u4v>(s.np * s.plane(s.Pp));
    wf = c.take<u4v>(s.np * s.plane(s.Vp));
    ex = c.take<int>(s.np == 2 ? s.Pp : 0);
    ew = c.take<int>(s.np == 2 ? s.Vp : 0);
  }
  // what the logits' products need besides the operands; words from v0 on
  void scales(const Shape &s, float scale, int64_t v0, GemmArgs &g) const {
    g.c = fabsf(scale) * LOG2E, g.exp_c = 0;
    if (s.np == 2) g.exps_a = ew + v0, g.exps_b = ex, g.c = frexpf(g.c, &g.exp_c);
  }
};

int word_units(int planes, int64_t words, int64_t rows);

struct FwdScratch {
  float *amax, *target, *row_loss;
  float2 *partial;
  int pairs;
  FwdScratch(Carve &c, const Shape &s) {
    const int64_t words = 64 * word_units(s.np, s.Vp, s.Pp);
    pairs = (int)((s.Vp + words - 1) / words * 2);   // a wavefront's words each
    amax = c.take<float>(2 * AMAX_BLOCKS);
    target = c.take<float>(s.Pp);
    row_loss = c.take<float>(s.Pp);
    partial = c.take<float2>((int64_t)pairs * s.Pp);
  }
};

// G of one piece of the vocabulary, all copies and pieces (bfloat16, 8192 rows x 131072 words x 1024 dims, loss and both
// gradients: 11.0 ms with 1 GB, 11.9 with 512 MB).
constexpr int64_t PIECE_BYTES = 1024ll << 20;

// Splits of a contraction of `k` blocks, where its tiles alone are fewer than the CUs: as many, up to 16, as give each CU
// a tile at most, of at least four blocks each.  Every split writes and reads a partial result of its own, which costs
// more than CUs without work where there is a round of tiles already (50021 words x 768 dims, G in one piece: 1441 against 745 us).
struct Splits {
  int n, blocks;  // blocks of each but the last
};
Splits choose_splits(int64_t Dk, int64_t n_rows, int64_t k) {
  const int64_t tiles = round_up(Dk, 256) / 256 * ((n_rows + 255) / 256);
  const int64_t want = std::max<int64_t>(1, std::min({CUS / tiles, k / 4, (int64_t)16}));
  const int blocks = (int)round_up((k + want - 1) / want, 2);
  return Splits{(int)((k + blocks - 1) / blocks), blocks};
}

struct BwdScratch {
  int *exp_g;
  float *tops, *coef_a, *coef_b, *acc, *acc_w;
  u4v *xt, *wt, *gx, *gw;
  int64_t piece;  // words
  Splits split_words, split_rows;  // of the contractions of dX (a full piece's words) and of dW
  BwdScratch(Carve &c, const Shape &s, bool dx, bool dw) {
    const int64_t per_word = s.Pp * 2 * s.ng * (int(dx) + int(dw));
    piece = std::min(s.Vp, std::max<int64_t>(PIECE_BYTES / per_word / TILE_V, 1) * TILE_V);
    const int64_t pieces = (s.Vp + piece - 1) / piece;
    piece = round_up((s.Vp + pieces - 1) / pieces, TILE_V);   // of equal size
    split_words = choose_splits(s.Dk, s.Pp, piece / 16);
    split_rows = choose_splits(s.Dk, piece, s.Pp / 16);
    exp_g = c.take<int>(1);
    tops = c.take<float>(CUS);
    coef_a = c.take<float>(s.Pp);
    coef_b = c.take<float>(s.Pp);
    acc = c.take<float>(dx ? split_words.n * s.Pp * s.Dk : 0);
    acc_w = c.take<float>(dw && split_rows.n > 1 ? split_rows.n * piece * s.Dk : 0);
    wt = c.take<u4v>(dx ? s.na * s.plane(s.Vp) : 0);
    xt = c.take<u4v>(dw ? s.na * s.plane(s.Pp) : 0);
    gx = c.take<u4v>(dx ? s.ng * s.Pp * piece / 8 : 0);
    gw = c.take<u4v>(dw ? s.ng * s.Pp * piece / 8 : 0);
  }
};

// Launches a kernel whose dynamic LDS may be above the 64 KB that need no leave.
template <auto KERNEL, typename... Args>
int launch_lds(dim3 grid, dim3 block, size_t bytes, hipStream_t st, const Args &...args) {
  static std::atomic<uint64_t> known{0};   // devices that know the kernel's LDS size
  int device = 0;
  PR_HIP(hipGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(known.load(std::memory_order_acquire) & bit)) {
    PR_HIP(hipFuncSetAttribute((const void *)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    known.fetch_or(bit, std::memory_order_release);
  }
  hipLaunchKernelGGL(KERNEL, grid, block, bytes, st, args...);
  return check_launch("pr_vocab_ce");
}

struct Product {
  GemmArgs g;
  int64_t m_rows, n_rows;  // multiples of 32 and of 256
};

template <typename T, int MT, int MODE>
int launch_tiles(const Product &a, const Product *b, hipStream_t st) {
  const size_t bytes = (size_t)3 * STAGE_BLOCKS<typename FormOf<T, MODE>::F, MT> * 1024;
  auto cut = [](const Product &p) {
    GemmArgs g = p.g;
    g.m_tiles = (int)((p.m_rows + 64 * MT - 1) / (64 * MT)), g.n_tiles = (int)((p.n_rows + 255) / 256);
    g.a_tiles = (int)(p.m_rows / 32), g.b_tiles = (int)(p.n_rows / 32);
    return g;
  };
  const GemmArgs g = cut(a), g2 = b ? cut(*b) : GemmArgs{};
  const int64_t tiles = (int64_t)g.m_tiles * g.n_tiles * g.splits + (int64_t)g2.m_tiles * g2.n_tiles * g2.splits;
  if (tiles > (1ll << 30)) {
    set_error_text("pr_vocab_ce: too many tiles for one launch");
    return PR_EUNSUPPORTED;
  }
  return launch_lds<vce_gemm_kernel<T, MT, MODE>>(dim3((unsigned)std::min<int64_t>(CUS, (tiles + 7) / 8 * 8)), dim3(512),
                                                      bytes, st, g, g2);
}

// Time of so many tiles of 64 mt by 256, in arbitrary units.  A tile costs its products and the operand rows that it does
// not share, in units of one product of 64 rows: 1.5 with one plane each (256 features by 256 words against 128 by 256: 178 and
// 219 us for the same product), 1.8 with two and three of each (320 words by 256 rows against 256 by 256: 233 and 222 us), 6
// with one and two, where two thirds of what is loaded is not shared (the same as above: 390 and 560 us).
// The chip is bound by its power, so a last round that leaves CUs without work runs at a higher clock: three quarters of a
// full one.
double tile_time(int products, int64_t tiles, int mt) {
  const double own = products == 1 ? 1.5 : products == 2 ? 6. : 1.8;
  return ((double)(tiles / CUS) + (tiles % CUS ? 0.75 : 0.)) * (mt * products + own);
}

// Words per workgroup of STATS and GRAD, in units of 64: up to five, four with two planes, whose exponents take the registers.
int word_units(int planes, int64_t words, int64_t rows) {
  const int products = planes == 1 ? 1 : 3, most = planes == 1 ? 5 : 4;
  int best = 1;
  for (int mt = 2; mt <= most; ++mt) {
    auto time = [&](int m) { return tile_time(products, (words + 64 * m - 1) / (64 * m) * ((rows + 255) / 256), m); };
    if (time(mt) < time(best)) best = mt;
  }
  return best;
}
template <typename T, int MODE>
int launch_words(const GemmArgs &g, int64_t words, int64_t rows, hipStream_t st) {
  const Product p{g, words, rows};
  switch (word_units(Types<T>::Logits::NA, words, rows)) {
    case 1: return launch_tiles<T, 1, MODE>(p, nullptr, st);
    case 2: return launch_tiles<T, 2, MODE>(p, nullptr, st);
    case 3: return launch_tiles<T, 3, MODE>(p, nullptr, st);
    case 4: return launch_tiles<T, 4, MODE>(p, nullptr, st);
    default:
      if constexpr (Types<T>::Logits::NA == 1) return launch_tiles<T, 5, MODE>(p, nullptr, st);
      return PR_EUNSUPPORTED;   // (no choice of word_units)
  }
}

// The same for the products whose M rows are features.
template <typename T, int MODE>
int launch_features(const Product &a, const Product *b, hipStream_t st) {
  auto time = [&](int mt) {
    auto tiles = [mt](const Product &p) { return (p.m_rows + 64 * mt - 1) / (64 * mt) * ((p.n_rows + 255) / 256) * p.g.splits; };
    return tile_time(Types<T>::Grads::PRODUCTS, tiles(a) + (b ? tiles(*b) : 0), mt);
  };
  const int best = time(4) <= time(2) && time(4) <= time(1) ? 4 : time(2) <= time(1) ? 2 : 1;
  if (best == 4) return launch_tiles<T, 4, MODE>(a, b, st);
  if (best == 2) return launch_tiles<T, 2, MODE>(a, b, st);
  return launch_tiles<T, 1, MODE>(a, b, st);
}

struct Call {
  int dtype;
  int64_t P, V, D;
  Matrix x, w;
  const int64_t *labels;
  int64_t ignore;
  float scale;
};

#define PR_TRY(e)                  \
  do {                             \
    const int _rc = (e);           \
    if (_rc != PR_OK) return _rc;  \
  } while (0)

template <typename T>
int forward(const Call &c, int mean, Kept &k, FwdScratch &f, float *row_loss, float *lse, float *loss, hipStream_t st) {
  const Shape s(c.dtype, c.P, c.V, c.D);
  const int kb = (int)(s.Dk / 16);
  int w_blocks = 0, x_blocks = 0;
  if (s.np == 2) {
    int lanes = 1;
    while (lanes < 64 && lanes * 8 < c.D) lanes *= 2;
    const int rows = 16 * (64 / lanes);   // of a workgroup at a time
    auto blocks = [&](int64_t padded) { return (int)std::min<int64_t>(AMAX_BLOCKS, (padded + rows - 1) / rows); };
    w_blocks = blocks(s.Vp), x_blocks = blocks(s.Pp);
    const AmaxJob aw{c.w, nullptr, 0, w_blocks, s.Vp, k.ew}, ax{c.x, c.labels, c.ignore, x_blocks, s.Pp, k.ex};
    hipLaunchKernelGGL((vce_amax_kernel<T>), dim3(w_blocks + x_blocks), dim3(256), 0, st, aw, ax, lanes, f.amax);
    PR_TRY(check_launch("pr_vocab_ce"));
  }
  const PackJob jw{c.w, nullptr, 0, k.wf, s.plane(s.Vp), s.Vp / 32 * ((kb + 3) / 4), kb, w_blocks, s.np == 2 ? k.ew : nullptr, 1.f};
  const PackJob jx{c.x, c.labels, c.ignore, k.xf, s.plane(s.Pp), s.Pp / 32 * ((kb + 3) / 4), kb, x_blocks,
                   s.np == 2 ? k.ex : nullptr, c.scale < 0.f ? -1.f : 1.f};
  const int64_t pack_blocks = std::min<int64_t>(2048, (jw.units + jx.units + 3) / 4);
  hipLaunchKernelGGL((vce_pack_kernel<T>), dim3((unsigned)pack_blocks), dim3(256), 0, st, jw, jx, f.amax, k.scal);
  PR_TRY(check_launch("pr_vocab_ce"));
  GemmArgs g{};
  g.A = k.wf, g.B = k.xf, g.plane_a = s.plane(s.Vp), g.plane_b = s.plane(s.Pp), g.ld_a = g.ld_b = kb;
  g.kblocks = g.k_split = kb, g.splits = 1;
  g.P = c.P, g.V = c.V, g.labels = c.labels;
  g.partial = f.partial, g.target = f.target, g.Pp = s.Pp;
  k.scales(s, c.scale, 0, g);
  PR_TRY((launch_words<T, STATS>(g, s.Vp, s.Pp, st)));
  const RowsOut rows{c.P, c.V, c.ignore, c.labels, f.target, k.stat, lse, row_loss};
  hipLaunchKernelGGL(vce_join_kernel, dim3((unsigned)(s.Pp / 8)), dim3(256), 0, st, rows, s.Pp, f.pairs, f.partial);
  PR_TRY(check_launch("pr_vocab_ce"));
  if (!loss) return PR_OK;
  hipLaunchKernelGGL(vce_reduce_kernel, dim3(1), dim3(1024), 0, st, c.P, row_loss, c.labels, c.ignore, mean, loss, k.scal);
  return check_launch("pr_vocab_ce");
}

// 32-row tiles of the kernels for few rows, and the padded rows and features that go with them.
struct FewShape {
  int64_t P, V, D, R, Dk, tiles;
  int nb, pieces, factors;   // pieces of the features for the scores and for dW
  bool shared;   // which score kernel
  FewShape(int dtype, int64_t P_, int64_t V_, int64_t D_)
      : P(P_), V(V_), D(D_), Dk(round_up(D_, 64)), tiles((V_ + 31) / 32), nb(P_ <= 32 ? 1 : P_ <= 64 ? 2 : 4),
        pieces(dtype == PR_F32 ? 3 : 1), factors(Shape(dtype, P_, V_, D_).na) {
    R = 32 * nb;
    // Below, CUs would be without work (20011 words x 1024 dims: 64 rows 53 against 47 us, 24 bfloat16 rows 32 against 27;
    // 60000 x 512: 41 against 58, 25 against 28)
    shared = V >= 128 * CUS;
  }
  int64_t packed(int n) const { return R * Dk / 8 * n; }   // 16-byte units of a copy of the features in n pieces
};

struct FewKept {
  Scalars *scal;
  float2 *stat;
  float *logits;          // in the log2 domain: [32 words][R][32]
  u4v *xt;
  FewKept(Carve &c, const FewShape &s) {
    scal = c.take<Scalars>(1);
    stat = c.take<float2>(s.R);
    xt = c.take<u4v>(s.packed(s.factors));
    logits = c.take<float>(s.tiles * s.R * 32);
  }
};

struct ScoreScratch {  // of the forward pass for few rows
  float *target, *row_loss;
  float2 *partial;
  u4v *xf;
  int blocks;
  ScoreScratch(Carve &c, const FewShape &s) {
    blocks = (int)(s.shared ? std::min<int64_t>(FEW_BLOCKS, (s.V + 127) / 128) : std::min<int64_t>(SCORE_BLOCKS, s.tiles));
    target = c.take<float>(s.R);
    row_loss = c.take<float>(s.R);
    partial = c.take<float2>(blocks * s.R);
    xf = c.take<u4v>(s.packed(s.pieces));
  }
};

template <typename T, int NB>
int launch_score(const Call &c, const FewShape &s, ScoreScratch &f, FewKept *k, hipStream_t st) {
  const bool wide = c.D >= 8 && c.w.ld_col == 1, packed = NB > 1 || s.shared || !wide || c.x.ld_col != 1 || c.D % 8;
  if (packed || k) {
    const FewPack job{c.x, c.labels, c.ignore, (int)(s.Dk / 16), 2 * NB, packed ? f.xf : nullptr, k ? k->xt : nullptr};
    const int64_t units = s.Dk / 16 * NB * ((packed ? 1 : 0) + (k ? 1 : 0));
    hipLaunchKernelGGL((vce_few_pack_kernel<T>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, job);
    PR_TRY(check_launch("pr_vocab_ce"));
  }
  float *const logits = k ? k->logits : nullptr;
  if (s.shared) {
    const size_t bytes = score_lds(NB, few_blocks<T>, s.pieces);
    return wide ? launch_lds<vce_score_shared_kernel<T, NB, true>>(dim3(f.blocks), dim3(256), bytes, st, c.w, c.P,
                                                                   (const u4v *)f.xf, c.labels, c.scale, f.partial, f.target,
                                                                   logits)
                : launch_lds<vce_score_shared_kernel<T, NB, false>>(dim3(f.blocks), dim3(256), bytes, st, c.w, c.P,
                                                                    (const u4v *)f.xf, c.labels, c.scale, f.partial, f.target,
                                                                    logits);
  }
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(f.blocks), dim3(256), 0, st, c.w, c.x, f.xf, c.labels, c.ignore, c.scale, f.partial,
                       f.target, logits);
    return check_launch("pr_vocab_ce");
  };
  if constexpr (NB == 1)
    if (!packed) return launch(vce_score_kernel<T, NB, true, false>);
  return wide ? launch(vce_score_kernel<T, NB, true, true>) : launch(vce_score_kernel<T, NB, false, true>);
}

// k: for a backward pass, or NULL.
template <typename T>
int score(const Call &c, int mean, ScoreScratch &f, FewKept *k, float *row_loss, float *lse, float *loss, hipStream_t st) {
  const FewShape s(c.dtype, c.P, c.V, c.D);
  if (s.nb == 1) PR_TRY((launch_score<T, 1>(c, s, f, k, st)));
  else if (s.nb == 2) PR_TRY((launch_score<T, 2>(c, s, f, k, st)));
  else PR_TRY((launch_score<T, 4>(c, s, f, k, st)));
  const RowsOut rows{c.P, c.V, c.ignore, c.labels, f.target, k ? k->stat : nullptr, lse, row_loss};
  // (one workgroup for all rows: up to 32 no slower than two launches; 128 rows of 8000 words 15 us slower)
  if (loss && s.nb == 1) {
    hipLaunchKernelGGL(vce_join_reduce_kernel, dim3(1), dim3(1024), 0, st, rows, f.blocks, f.partial, mean, loss,
                       k ? k->scal : nullptr);
    return check_launch("pr_vocab_ce");
  }
  hipLaunchKernelGGL(vce_join_row_kernel, dim3((unsigned)c.P), dim3(256), 0, st, rows, f.blocks, f.partial);
  PR_TRY(check_launch("pr_vocab_ce"));
  if (!loss) return PR_OK;
  hipLaunchKernelGGL(vce_reduce_kernel, dim3(1), dim3(1024), 0, st, c.P, row_loss, c.labels, c.ignore, mean, loss,
                     k ? k->scal : nullptr);
  return check_launch("pr_vocab_ce");
}

struct FewBwdScratch {
  float *acc;
  int64_t steps;   // of 32 words, in a run of DX
  int splits;
  FewBwdScratch(Carve &c, const FewShape &s, bool dx) {
    const int64_t chunks = (s.Dk + 255) / 256, want = std::max<int64_t>(1, std::min<int64_t>(FEW_BLOCKS / chunks, s.tiles));
    steps = (s.tiles + want - 1) / want;
    splits = (int)((s.tiles + steps - 1) / steps);
    acc = c.take<float>(dx ? splits * s.R * s.Dk : 1);   // (no buffer of no bytes)
  }
};

template <typename T, int NB>
int few_gradients(const Call &c, const FewShape &s, const FewKept &k, const FewBwdScratch &b, const FewGrad &f, T *dx, T *dw,
                  hipStream_t st) {
  if (dx) {
    const dim3 grid((unsigned)((s.Dk + 255) / 256), b.splits);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, f, c.w, b.steps, b.acc);
      return check_launch("pr_vocab_ce");
    };
    if constexpr (sizeof(T) == 2)
      PR_TRY(c.w.ld_col == 1 && c.D >= 2 ? launch(vce_few_dx_kernel<T, NB, true>) : launch(vce_few_dx_kernel<T, NB, false>));
    else
      PR_TRY(launch(vce_few_dx_kernel<T, NB, false>));
    hipLaunchKernelGGL((vce_few_finish_kernel<T>), dim3(grid.x, (unsigned)c.P), dim3(1024), 0, st, f, s.R * s.Dk, b.splits,
                       c.scale, b.acc, dx);
    PR_TRY(check_launch("pr_vocab_ce"));
  }
  if (dw) {
    const unsigned blocks = (unsigned)((s.tiles + 3) / 4);
    // (a part has a chunk at least: of 32 float32 features, of 64 others)
    const unsigned parts = (unsigned)std::max<int64_t>(1, std::min<int64_t>(FEW_BLOCKS / blocks, c.D / 64));
    PR_TRY((launch_lds<vce_few_dw_kernel<T, NB>>(dim3(blocks, parts), dim3(256), dw_lds(NB, few_tiles<T>, s.factors), st, f,
                                                 (const u4v *)k.xt, c.scale, dw)));
  }
  return PR_OK;
}

template <typename T>
int few_backward(const Call &c, int per_row, int mean, const FewKept &k, const FewBwdScratch &b, const float *g_loss,
                 const float *g_lse, T *dx, T *dw, hipStream_t st) {
  const FewShape s(c.dtype, c.P, c.V, c.D);
  const FewGrad f{{c.P, s.R, c.V, c.ignore, c.labels, g_loss, g_lse, per_row, mean, k.scal, k.stat, nullptr, nullptr, nullptr, nullptr, 0},
                  c.D, s.Dk, k.logits};
  if (s.nb == 1) return few_gradients<T, 1>(c, s, k, b, f, dx, dw, st);
  if (s.nb == 2) return few_gradients<T, 2>(c, s, k, b, f, dx, dw, st);
  return few_gradients<T, 4>(c, s, k, b, f, dx, dw, st);
}

template <typename T>
int backward(const Call &c, int per_row, int mean, const Kept &k, BwdScratch &b, const float *g_loss, const float *g_lse, T *dx,
             T *dw, hipStream_t st) {
  const Shape s(c.dtype, c.P, c.V, c.D);
  const int kb = (int)(s.Dk / 16), kv = (int)(s.Vp / 16), kp = (int)(s.Pp / 16);
  // above one workgroup's rows the largest factor has a launch of its own (2 M rows of 100 words x 512 dims: 29.1 ms without,
  // when 507 workgroups each look through all rows)
  const bool search = (per_row || g_lse) && s.Pp > COEF_ROWS;
  const CoefJob coef{c.P, s.Pp, c.V, c.ignore, c.labels, g_loss, g_lse, per_row, mean, k.scal, k.stat, b.exp_g, b.coef_a, b.coef_b, search ? b.tops : nullptr,
                     (int)std::min<int64_t>(CUS, (c.P + 1023) / 1024)};
  if (search) {
    hipLaunchKernelGGL(vce_largest_kernel, dim3(coef.n_tops), dim3(1024), 0, st, coef, b.tops);
    PR_TRY(check_launch("pr_vocab_ce"));
  }
  const TransposeJob tw{k.wf, b.wt, s.plane(s.Vp), dx ? s.Vp / 32 : 0, s.Dk / 32, k.ew, &k.scal->exp_w};
  const TransposeJob tx{k.xf, b.xt, s.plane(s.Pp), dw ? s.Pp / 32 : 0, s.Dk / 32, k.ex, &k.scal->exp_x};
  const int64_t turns = ((tw.row_tiles + tx.row_tiles) * (s.Dk / 32) + 15) / 16;
  hipLaunchKernelGGL(vce_prepare_kernel<T>, dim3((unsigned)((s.Pp + COEF_ROWS - 1) / COEF_ROWS + std::min<int64_t>(1024, turns))),
                     dim3(1024), 0, st, coef, tw, tx);
  PR_TRY(check_launch("pr_vocab_ce"));
  const Scale abs_scale = Scale::of(fabsf(c.scale));   // X's copy has the sign
  for (int64_t v0 = 0; v0 < s.Vp; v0 += b.piece) {
    const int64_t words = std::min(b.piece, s.Vp - v0);
    GemmArgs g{};
    g.A = k.wf + v0 / 32 * kb * 64, g.B = k.xf, g.plane_a = s.plane(s.Vp), g.plane_b = s.plane(s.Pp), g.ld_a = g.ld_b = kb;
    g.kblocks = g.k_split = kb, g.splits = 1, g.P = c.P, g.V = c.V, g.v0 = v0, g.labels = c.labels, g.Pp = s.Pp;
    g.stat = k.stat, g.coef_a = b.coef_a, g.coef_b = b.coef_b;
    k.scales(s, c.scale, v0, g);
    g.gx = dx ? b.gx : nullptr, g.gw = dw ? b.gw : nullptr;
    g.plane_gx = g.plane_gw = s.Pp * b.piece / 8, g.ld_gx = b.piece / 16, g.ld_gw = kp;
    PR_TRY((launch_words<T, GRAD>(g, words, s.Pp, st)));
    const bool last = v0 + words >= s.Vp, split_dw = dw && b.split_rows.n > 1;
    Product px{{}, s.Dk, s.Pp}, pw{{}, s.Dk, words};
    GemmArgs &x = px.g, &w = pw.g;
    x.A = b.wt + v0 / 16 * 64, x.B = b.gx, x.plane_a = s.plane(s.Vp), x.plane_b = g.plane_gx, x.ld_a = kv, x.ld_b = g.ld_gx;
    x.acc = b.acc, x.Pp = s.Pp, x.ld_acc = s.Dk, x.add = v0 > 0;
    // the splits of a full piece; a shorter last piece leaves the rest of them as they are
    x.kblocks = (int)(words / 16), x.k_split = b.split_words.blocks, x.splits = (x.kblocks + x.k_split - 1) / x.k_split;
    w.A = b.xt, w.B = b.gw, w.plane_a = s.plane(s.Pp), w.plane_b = g.plane_gw, w.ld_a = w.ld_b = kp;
    w.kblocks = kp, w.k_split = b.split_rows.blocks, w.splits = b.split_rows.n;
    w.scal = k.scal, w.exp_g = b.exp_g, w.scale = abs_scale, w.V = c.V, w.v0 = v0, w.out = dw, w.D = c.D;
    w.acc = b.acc_w, w.Pp = words, w.ld_acc = s.Dk;
    if (dx || split_dw)
      PR_TRY((launch_features<T, DX>(dx ? px : pw, dx && split_dw ? &pw : nullptr, st)));
    if (dw && !split_dw) PR_TRY((launch_features<T, DW>(pw, nullptr, st)));
    FinishJob jobs[2] = {};
    int n = 0;
    if (dx && last) jobs[n++] = FinishJob{c.P, c.D, s.Pp, s.Dk, b.split_words.n, Scale::of(c.scale), b.acc, &k.scal->exp_w, b.exp_g, dx};
    if (split_dw)
      jobs[n++] = FinishJob{std::min(words, c.V - v0), c.D, words, s.Dk, w.splits, abs_scale, b.acc_w, &k.scal->exp_x,
                            b.exp_g, dw + v0 * c.D};
    if (n) {
      hipLaunchKernelGGL((vce_finish_kernel<T>), dim3((unsigned)((jobs[0].rows + jobs[1].rows + 3) / 4)), dim3(256), 0, st,
                         jobs[0], jobs[1]);
      PR_TRY(check_launch("pr_vocab_ce"));
    }
  }
  return PR_OK;
}

int check_call(const Call &c) {
  if (!valid_shape(c.dtype, c.P, c.V, c.D) || c.P < 1) return PR_EINVAL;
  if (!(fabsf(c.scale) <= 1e38f)) return PR_EINVAL;   // its product with log2(e) is finite
  return !c.labels || ((uintptr_t)c.labels & 7) ? PR_EINVAL : PR_OK;
}

int check_matrix(int dtype, const Matrix &m) {
  const uintptr_t mask = dtype == PR_F32 ? 3 : 1;
  return !m.data || ((uintptr_t)m.data & mask) || m.ld_row < 0 || m.ld_col < 0 ? PR_EINVAL : PR_OK;
}

}  // namespace
}  // namespace pr

extern "C" int pr_vocab_ce_keeps_vocabulary(int64_t P, int64_t V, int64_t D) { return !pr::few(P, V, D); }

extern "C" size_t pr_vocab_ce_kept_bytes(int dtype, int64_t P, int64_t V, int64_t D) {
  if (!pr::valid_shape(dtype, P, V, D)) return 0;
  pr::Carve c(nullptr);
  if (pr::few(P, V, D)) pr::FewKept k(c, pr::FewShape(dtype, P, V, D));
  else pr::Kept k(c, pr::Shape(dtype, P, V, D));
  return c.used;
}

extern "C" int pr_vocab_ce_score_rows(void) { return pr::SCORE_ROWS; }

extern "C" size_t pr_vocab_ce_fwd_scratch_bytes(int dtype, int64_t P, int64_t V, int64_t D) {
  if (!pr::valid_shape(dtype, P, V, D)) return 0;
  pr::Carve packed(nullptr), plain(nullptr);
  if (!pr::few(P, V, D)) pr::FwdScratch f(packed, pr::Shape(dtype, P, V, D));
  if (P <= pr::SCORE_ROWS || pr::few(P, V, D)) pr::ScoreScratch g(plain, pr::FewShape(dtype, P, V, D));
  return std::max(packed.used, plain.used);
}

extern "C" size_t pr_vocab_ce_bwd_scratch_bytes(int dtype, int64_t P, int64_t V, int64_t D, int want_dx, int want_dw) {
  if (!pr::valid_shape(dtype, P, V, D) || P < 1 || (!want_dx && !want_dw)) return 0;
  pr::Carve c(nullptr);
  if (pr::few(P, V, D)) pr::FewBwdScratch b(c, pr::FewShape(dtype, P, V, D), want_dx);
  else pr::BwdScratch b(c, pr::Shape(dtype, P, V, D), want_dx, want_dw);
  return c.used;
}

extern "C" int pr_vocab_ce_fwd(int dtype, int64_t P, int64_t V, int64_t D, const void *x, int64_t ldx_row, int64_t ldx_col,
                               const void *w, int64_t ldw_row, int64_t ldw_col, const int64_t *labels, int64_t ignore_index,
                               float scale, int mean, void *kept, size_t kept_bytes, void *scratch, size_t scratch_bytes,
                               float *row_loss, float *lse, float *loss, void *stream) {
  const pr::Call c{dtype, P, V, D, {x, P, D, ldx_row, ldx_col}, {w, V, D, ldw_row, ldw_col}, labels, ignore_index, scale};
  PR_TRY(pr::check_call(c));
  PR_TRY(pr::check_matrix(dtype, c.x));
  PR_TRY(pr::check_matrix(dtype, c.w));
  if ((!kept && P > pr::SCORE_ROWS && !pr::few(P, V, D)) || !scratch || (!row_loss && !loss) || ((uintptr_t)kept & 15) || ((uintptr_t)scratch & 15))
    return PR_EINVAL;
  if ((kept && kept_bytes < pr_vocab_ce_kept_bytes(dtype, P, V, D)) ||
      scratch_bytes < pr_vocab_ce_fwd_scratch_bytes(dtype, P, V, D))
    return PR_ESCRATCH;
  hipStream_t st = (hipStream_t)stream;
  pr::Carve ck(kept), cs(scratch);
  if (!kept || pr::few(P, V, D)) {
    const pr::FewShape s(dtype, P, V, D);
    pr::ScoreScratch f(cs, s);
    pr::FewKept few(ck, s), *k = kept ? &few : nullptr;
    if (!row_loss) row_loss = f.row_loss;
    if (dtype == PR_F32) return pr::score<float>(c, mean, f, k, row_loss, lse, loss, st);
    if (dtype == PR_F16) return pr::score<_Float16>(c, mean, f, k, row_loss, lse, loss, st);
    return pr::score<__bf16>(c, mean, f, k, row_loss, lse, loss, st);
  }
  const pr::Shape s(dtype, P, V, D);
  pr::Kept k(ck, s);
  pr::FwdScratch f(cs, s);
  if (!row_loss) row_loss = f.row_loss;
  if (dtype == PR_F32) return pr::forward<float>(c, mean, k, f, row_loss, lse, loss, st);
  if (dtype == PR_F16) return pr::forward<_Float16>(c, mean, k, f, row_loss, lse, loss, st);
  return pr::forward<__bf16>(c, mean, k, f, row_loss, lse, loss, st);
}

extern "C" int pr_vocab_ce_bwd(int dtype, int64_t P, int64_t V, int64_t D, const void *w, int64_t ldw_row, int64_t ldw_col,
                               const int64_t *labels, int64_t ignore_index, float scale, int mean, int per_row,
                               const void *kept, size_t kept_bytes, const float *g_loss, const float *g_lse, void *scratch,
                               size_t scratch_bytes, void *dx, void *dw, void *stream) {
  const pr::Call c{dtype, P, V, D, {}, {w, V, D, ldw_row, ldw_col}, labels, ignore_index, scale};
  PR_TRY(pr::check_call(c));
  if (!dx && !dw) return PR_OK;
  const bool few = pr::few(P, V, D);
  if (few && dx) PR_TRY(pr::check_matrix(dtype, c.w));
  if (!kept || !scratch || ((uintptr_t)kept & 15) || ((uintptr_t)scratch & 15)) return PR_EINVAL;
  if (((uintptr_t)dx & 15) || ((uintptr_t)dw & 15)) return PR_EINVAL;
  if (kept_bytes < pr_vocab_ce_kept_bytes(dtype, P, V, D) ||
      scratch_bytes < pr_vocab_ce_bwd_scratch_bytes(dtype, P, V, D, dx != nullptr, dw != nullptr))
    return PR_ESCRATCH;
  pr::Carve ck(const_cast<void *>(kept)), cs(scratch);
  hipStream_t st = (hipStream_t)stream;
  if (few) {
    const pr::FewShape s(dtype, P, V, D);
    const pr::FewKept k(ck, s);
    const pr::FewBwdScratch b(cs, s, dx != nullptr);
    if (dtype == PR_F32) return pr::few_backward<float>(c, per_row, mean, k, b, g_loss, g_lse, (float *)dx, (float *)dw, st);
    if (dtype == PR_F16)
      return pr::few_backward<_Float16>(c, per_row, mean, k, b, g_loss, g_lse, (_Float16 *)dx, (_Float16 *)dw, st);
    return pr::few_backward<__bf16>(c, per_row, mean, k, b, g_loss, g_lse, (__bf16 *)dx, (__bf16 *)dw, st);
  }
  const pr::Shape s(dtype, P, V, D);
  const pr::Kept k(ck, s);
  pr::BwdScratch b(cs, s, dx != nullptr, dw != nullptr);
  if (dtype == PR_F32) return pr::backward<float>(c, per_row, mean, k, b, g_loss, g_lse, (float *)dx, (float *)dw, st);
  if (dtype == PR_F16)
    return pr::backward<_Float16>(c, per_row, mean, k, b, g_loss, g_lse, (_Float16 *)dx, (_Float16 *)dw, st);
  return pr::backward<__bf16>(c, per_row, mean, k, b, g_loss, g_lse, (__bf16 *)dx, (__bf16 *)dw, st);
}

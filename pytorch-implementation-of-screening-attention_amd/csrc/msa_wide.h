// What the kernels around wide products share (msa_head.hip, msa_gated.hip): operands laid out for the matrix core,
// power-of-two scales, and the two products of a backward pass, dx = G W and dW = G^T x.
//
// Types: bf16 and fp16 rows are operands as they are (copied only where their rows are not 16-byte aligned or their
// width is no multiple of 32).  fp32 rows are taken in one of two formats, which the data decides on the device:
//   narrow: two fp16 terms, x s = h + 2^-11 l, with a power of two s for the whole matrix that brings its largest entry to
//     [2^14, 2^15): 22 bits of every entry down to 2^-28 of the largest, and three MFMA products where the fp32 MFMA would
//     take sixteen times as long;
//   wide: three bf16 terms, x = h + m + l, each the rest rounded: all 24 bits over fp32's whole range, six products.
// One scale ties the rows of a matrix to each other: next to a row 2^40 above it, a narrow row keeps 10 bits.  So a call
// is narrow only where its matrices are even (wide_mode), as model data is.
#pragma once

#include <type_traits>

#include "msa_internal.h"
#include "msa_matmul.h"

namespace msa {

// Operand type of an input type, and its number of terms.
template <typename T, bool WIDE = false> struct Wide { typedef T E; static constexpr int P = 1; };
template <> struct Wide<float, false> { typedef f16 E; static constexpr int P = 2; };
template <> struct Wide<float, true> { typedef bf16 E; static constexpr int P = 3; };
inline int planes_of(int dtype) { return dtype == 0 ? 3 : 1; }  // room for the terms of either format

// What every kernel of a call reads: rows that count, the format, and the scales of the operands (1 in the wide format).
struct WideMode {
  int live;
  int wide;
  float sx, sw, sg;
};

// What a block found in its rows of one matrix: the largest finite |entry| and row norm (of finite entries); fp32: 255 less
// the smallest exponent (as stored) of a nonzero row's largest entry (0: no such row), and how many nonzero entries lie
// below 2^-digits of their row's largest.  A place a block, joined in one kernel: 2700 atomics to one place take 40 us.
struct WidePart { float max, norm; int low, small; };
constexpr int kCopies = 4;
constexpr int64_t kMaxBlocks = 1024;  // of a matrix
constexpr int64_t kPartBytes = kCopies * kMaxBlocks * (int64_t)sizeof(WidePart);

// fn(std::bool_constant<wide>) in the call's format; uniform over the grid.
template <typename T, typename Fn>
__device__ inline void by_format(const WideMode* m, Fn fn) {
  if constexpr (__is_same(T, float)) {
    if (__builtin_amdgcn_readfirstlane(m->wide)) {
      fn(std::true_type());
      return;
    }
  }
  fn(std::false_type());
}

// p with a b c p in [2^(top-1), 2^top); 1 for 0.  The product itself may be too large or too small for a float.
__device__ inline float pow2_to(float a, float b, float c, int top) {
  if (!(a > 0.0f) || !(b > 0.0f) || !(c > 0.0f)) return 1.0f;
  int ea, eb, ec, em;
  const float m = frexpf(a, &ea) * frexpf(b, &eb) * frexpf(c, &ec);
  (void)frexpf(m, &em);
  int e = top - (ea + eb + ec + em);
  e = e > 120 ? 120 : (e < -120 ? -120 : e);
  return ldexpf(1.0f, e);
}
__device__ inline float pow2_to(float mx, int top) { return pow2_to(mx, 1.0f, 1.0f, top); }

// Scales of the operands.  fp16 gradients of logits lie in [-1, 1] and are kept times 2^15; those of the gated
// projections are bounded by max|dh| 1.13 max|x| max|w| (|act(g)| <= |g|, |act'| < 1.13).
template <typename T> __device__ inline float scale_x(const WideMode* m) {
  if constexpr (__is_same(T, float)) return m->sx;
  return 1.0f;
}
template <typename T> __device__ inline float scale_w(const WideMode* m) {
  if constexpr (__is_same(T, float)) return m->sw;
  return 1.0f;
}
template <typename T> __device__ inline float scale_g(const WideMode* m, int gated) {
  if constexpr (__is_same(T, bf16)) return 1.0f;
  if (__is_same(T, f16) && !gated) return 32768.0f;
  return m->sg;
}

// The N terms of v (already scaled) in an operand type.  v is held in a register first: formed inside, a product that makes v may be rounded
// to the first term straight from its exact value in one place and from the rounded one in another, and the others belong
// to one first term only.
template <typename E, int N> struct Terms {
  E t[N];
  __device__ explicit Terms(float v) {
    if constexpr (N == 1) {
      t[0] = (E)v;
      return;
    }
    asm("" : "+v"(v));
    t[0] = (E)v;
    if constexpr (N == 2) {
      t[1] = (E)((v - (float)t[0]) * 2048.0f);
    } else if constexpr (N == 3) {
      // past bf16's largest number, which is below fp32's, the first term is cut instead of rounded
      if (fabsf(v) < INFINITY && !(fabsf((float)t[0]) < INFINITY)) t[0] = (E)__uint_as_float(__float_as_uint(v) & 0xffff0000u);
      const float r = v - (float)t[0];
      t[1] = (E)r;
      t[2] = (E)(r - (float)t[1]);
    }
  }
};

// Terms of G.  2-byte types keep one, in their own type: beside the rounding of dx and dW themselves that makes their error
// sqrt(2) times as large on average (bf16 2.1e-3 where theirs alone is 1.7e-3; torch's products and cross entropy in the type,
// which round the logits too, 3.8e-3).  Two terms for all rows make dx and dW twice as long: 8192 rows of 512 by 50257 bf16 1.77 ->
// 2.86 ms a pass (torch's 2.90); a captured pass of less than 10 GFLOP a product 12 to 20% longer.  Few rows average over few roundings, and
// their products are short: two terms up to 256 rows.  Error of dx and dW over that of their own rounding, one term / two: 1.79
// / 1.00 for 2 rows, 1.48 / 1.00 for 18, 1.24 to 1.41 / 1.00 for 100 and more.  Time: 84 rows of 1024 by 51364 bf16 191 / 226 us,
// shorter calls alike (their launches).
constexpr int64_t kTwoTerms = 256;
inline int terms_of_g(int dtype, int64_t N) { return dtype == 0 || N <= kTwoTerms ? 2 : 1; }  // fp32: of the narrow format
inline int g_planes(int dtype, int64_t N) { return dtype == 0 ? 3 : terms_of_g(dtype, N); }   // that there is room for

// The products of one order of the wide format's three terms: h h (0); h m and m h (1); h l, l h and m m (2).
inline void add_wide_segs(MmSegs& s, int order, int64_t a, int64_t a_plane, int64_t b, int64_t b_plane) {
  for (int t = 0; t <= order; ++t) {
    s.a[s.n] = a + t * a_plane;
    s.b[s.n++] = b + (order - t) * b_plane;
  }
}

inline int64_t wide_dp(int64_t d) { return round_up(d, 32); }

// Matrices as operand rows of dp columns, in blocks of 32 columns (MmTile::Side) with blk bytes from block to block, their
// terms plane_bytes apart.  pos: null, or which row of the
// operand each row becomes (-1: none); rows from mode->live up to the next multiple of 128 are then zeroed.  slot (0: x, 1: w, 2:
// dh): whose scale it takes.
struct RowsCopy {
  const void* src; int64_t ld; int64_t rows; int d;
  char* dst; int64_t plane_bytes, blk;
  const int* pos; int slot, norms;
};
struct RowsCopies {
  RowsCopy m[kCopies];
  int n, dtype;
  const WideMode* mode;
  void add(const RowsCopy& c) { m[n++] = c; }
};
hipError_t launch_rows_copy(const RowsCopies& c, hipStream_t s);
// Looks over the matrices (slot 0: x, 1: w, 2: dh) and finds the scales and the format from it, into mode; live, if rows are
// taken out, is there.  parts: kPartBytes of scratch.  gated: G's scale is bounded by the maxima.
hipError_t launch_wide_mode(const RowsCopies& c, WidePart* parts, WideMode* mode, int gated, hipStream_t s);

// What G is to be multiplied with: *cmax; or dloss[0] factor, over the number of rows that count for a mean; or 1.
struct GradUnit {
  const float* dloss;
  float factor;
  int mode;  // 0: cmax, 1: mean, 2: sum, 3: one
};
__device__ inline float unit_of(const GradUnit& u, const WideMode* h, const float* cmax) {
  if (u.mode == 3) return 1.0f;
  if (u.mode == 0) return *cmax;
  if (u.mode == 2) return u.dloss[0] * u.factor;
  return h->live > 0 ? u.dloss[0] * u.factor / (float)h->live : 0.0f;  // a mean over no rows: gradients of zeros
}

// How the two products of a piece are cut: each of dx's tiles into dx_split ranges of its k, dW's into dw_split.  cost:
// stages (32 k of a tile) until the last of 256 blocks in flight (one a CU) has ended, as wide_share reckons.  Either a
// block for each range, the longer kind first; or, `slots` > 0, as many blocks as CUs: block s takes dW's ranges s, s + slots,
// ... and then range s / tiles of dx's tile s % tiles, the first n_a ranges `a` steps long (behind one more of dW's) and
// the others b.
struct WideShare {
  int dx_split, dw_split;
  bool dx_first;
  int64_t cost;
  int slots, n_a, a, b;
};
// segs: products that each tile adds up of one weight (MmSegs).
WideShare wide_share(int64_t N, int d, int64_t C, int halves, int segs, bool dx, bool dw);
// The columns of a piece of `rows` weight rows whose G takes `bytes_of_column` a column (fp32: of the narrow format): 1 GB of G, 512 or 256 MB, by cost, and 256 at least.
int64_t wide_piece(int64_t N, int d, int64_t rows, int halves, int segs, bool dx, bool dw, int64_t bytes_of_column, WideShare* share);

// The backward products of one piece of the weight's rows.
struct WideProducts {
  int dtype, gated;
  int64_t N, n_pad;  // tokens (operand rows), as padded in g
  int d;
  int64_t dp;
  int halves;        // weights: 1, or 2 (gate and up)
  int cols;          // weight rows of the piece
  int64_t C;         // columns of g: cols rounded up to 256
  const char* x; int64_t x_ld, x_blk, x_plane; int x_rows;    // bytes from row to row, from 32 columns on, to the second term; readable rows
  const char* w[2]; int64_t w_ld, w_blk, w_plane; int w_rows;        // the piece's first rows; readable rows from there
  const char* g; int64_t g_plane, g_half; int g_terms;        // [half][term][C / 32][n_pad][32]; terms of the narrow format
  float* dx_part; int dx_add;                                 // [share.dx_split][n_pad][dp], or null: no dx
  void* dw[2];                                                // the piece's rows of the gradients, or null
  float* dw_part;                                             // [share.dw_split][halves][C][dp] where that is over 1
  WideShare share;
  const WideMode* mode;
  GradUnit unit; const float* cmax;
  int use_live;  // tokens are mode->live
};
hipError_t launch_wide_products(const WideProducts& p, hipStream_t s);

// dx[n] = factor * sum of the parts' rows pos[n] (pos null: n); rows with pos < 0 are zero.
struct WideFinish {
  int dtype, gated;
  int64_t N, n_pad;
  int d;
  int64_t dp;
  int split;
  const float* part;
  const int* pos;
  const WideMode* mode;
  GradUnit unit; const float* cmax;
  void* dx;
};
hipError_t launch_wide_finish(const WideFinish& f, hipStream_t s);

}  // namespace msa

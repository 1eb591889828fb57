// Operand rows, scales and the backward products of the wide layers (msa_wide.h).
#include "msa_wide.h"

#include <string.h>

namespace msa {
namespace {

constexpr int kThreads = 256;
// Tokens (or weight rows) of a product's tile.  256 by 256, one block of 8 waves a CU, against two blocks of 256 by 128: a
// third less goes through LDS for each flop, and its one epilogue behind a long k costs little (the losses' own products,
// whose k is d, are better off with two blocks, one in its epilogue while the other multiplies).  us of a whole training
// pass, 128 / 256: 8192 x 50257 x 512 bf16 1855 / 1805, 32768 rows 7640 / 7270, 2867 fp32 rows 2500 / 2260.
constexpr int kTileN = 256, kProductThreads = 512;

// 8 neighbours of a row, zeros past its end.
template <typename T>
__device__ inline void load8(const T* in, int c, int d, bool vec, T (&x)[8]) {
  if (vec && c + 8 <= d) {
    typedef __attribute__((__vector_size__(16))) T T16;
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int q = 0; q < 8 / PER; ++q) {
      const T16 t = *reinterpret_cast<const T16*>(in + c + q * PER);
#pragma unroll
      for (int e = 0; e < PER; ++e) x[q * PER + e] = t[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T v = in[c + e < d ? c + e : d - 1];
      x[e] = c + e < d ? v : (T)0.0f;
    }
  }
}

struct RowsArgs {
  RowsCopy m[kCopies];
  int64_t first[kCopies + 1];  // blocks of each matrix
  int vec[kCopies];
  const WideMode* mode;
};
__device__ inline int matrix_of(const RowsArgs& a, int64_t block) {
  int i = 0;
#pragma unroll
  for (int k = 1; k < kCopies; ++k) i += block >= a.first[k] ? 1 : 0;
  return i;
}

// Below 2^-digits of its row's largest entry an entry is small (fp32): with rows' largest entries within 2^kEven of each other
// the rest keep their 22 bits in the narrow format.  dh is no operand, but rows and columns of G are as uneven as its own, and G
// keeps as many bits: G has the digits, and dh's share of kEvenG, to itself.
constexpr int kDigits = 18, kDigitsDh = 24, kEven = 10, kEvenG = 24;

// A wave takes rows in turn, of the matrix that its block belongs to.  Which entries of fp32 rows are small is seen once the
// largest is known: rows of up to 2048 are still in registers then, longer ones in the cache.
template <typename T>
__global__ void __launch_bounds__(kThreads) rows_max_kernel(RowsArgs a, WidePart* parts) {
  constexpr bool EVEN = __is_same(T, float);
  constexpr int HELD = EVEN ? 4 : 1;
  const int i = matrix_of(a, blockIdx.x), lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const RowsCopy m = a.m[i];
  const int64_t step = (a.first[i + 1] - a.first[i]) * 4;
  const float digits = m.slot == 2 ? 1.0f / (1 << kDigitsDh) : 1.0f / (1 << kDigits);
  float mx = 0.0f, nx = 0.0f;
  int low = 0, small = 0;
  for (int64_t r = ((int64_t)blockIdx.x - a.first[i]) * 4 + wave; r < m.rows; r += step) {
    if (m.pos != nullptr && m.pos[r] < 0) continue;
    const T* p = (const T*)m.src + r * m.ld;
    float ss = 0.0f, rx = 0.0f;
    T x[HELD][8];
    auto load = [&](int c0) {
#pragma unroll
      for (int q = 0; q < HELD; ++q) {
        const int c = c0 + q * 512 + lane * 8;
        if (c0 + q * 512 >= m.d) break;
        if (c < m.d) {
          load8(p, c, m.d, a.vec[i] != 0, x[q]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[q][e] = (T)0.0f;
        }
      }
    };
    for (int c0 = 0; c0 < m.d; c0 += HELD * 512) {
      load(c0);
#pragma unroll
      for (int q = 0; q < HELD; ++q) {
        if (c0 + q * 512 >= m.d) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = fabsf(to_f(x[q][e]));
          if (v < INFINITY) {
            rx = fmaxf(rx, v);
            ss = fmaf(v, v, ss);
          }
        }
      }
    }
    mx = fmaxf(mx, rx);
    if (m.norms || EVEN) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) rx = fmaxf(rx, __shfl_xor(rx, o));
    }
    if (m.norms) {
      ss = wave_sum(ss);
      if (ss > 1e-30f && ss < INFINITY) nx = fmaxf(nx, sqrtf(ss));
      else nx = fmaxf(nx, fminf(rx * sqrtf((float)m.d), 3e38f));  // squares left fp32's range: a bound that does not
    }
    if (EVEN && rx > 0.0f) {
      const int at = 255 - (int)(__float_as_uint(rx) >> 23);
      low = at > low ? at : low;
      const float least = rx * digits;
      for (int c0 = 0; c0 < m.d; c0 += HELD * 512) {
        if (m.d > HELD * 512) load(c0);
#pragma unroll
        for (int q = 0; q < HELD; ++q) {
          if (c0 + q * 512 >= m.d) break;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = fabsf(to_f(x[q][e]));
            small += v < least && v > 0.0f ? 1 : 0;
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  if constexpr (EVEN) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) small += __shfl_xor(small, o);
  }
  __shared__ WidePart found[4];
  if (lane == 0) found[wave] = WidePart{mx, nx, low, small};
  __syncthreads();
  if (threadIdx.x == 0) {
    WidePart f = found[0];
    for (int w = 1; w < 4; ++w)
      f = WidePart{fmaxf(f.max, found[w].max), fmaxf(f.norm, found[w].norm), f.low > found[w].low ? f.low : found[w].low, f.small + found[w].small};
    parts[blockIdx.x] = f;
  }
}

// The scales and the format.  Narrow is what has rows within 2^kEven of each other and fewer small entries than a quarter of
// a column would hold; with the gradient's rows besides, 2^kEvenG.  Model data lies far from both: rows behind a norm are
// within 2^3, and of normal entries 1e-5 are small, of which a quarter of a column is 1 / 4 d.  One block, four waves to a matrix.
template <typename T>
__global__ void __launch_bounds__(64 * 4 * kCopies) wide_mode_kernel(RowsArgs a, const WidePart* parts, WideMode* mode, int gated,
                                                                     int64_t rows_x, int64_t rows_w, int64_t rows_dh) {
  struct Sum { float max, norm; int low; long long small; };
  __shared__ Sum sums[4 * kCopies];
  auto join = [](Sum& x, float max, float norm, int low, long long small) {
    x = Sum{fmaxf(x.max, max), fmaxf(x.norm, norm), x.low > low ? x.low : low, x.small + small};
  };
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  Sum s = {0.0f, 0.0f, 0, 0};
  {
    const int64_t end = a.first[wave / 4 + 1], b = a.first[wave / 4] + wave % 4 * 64 + lane;
    constexpr int PER = (int)(kMaxBlocks / 256);
    WidePart p[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) p[q] = b + q * 256 < end ? parts[b + q * 256] : WidePart{0.0f, 0.0f, 0, 0};
#pragma unroll
    for (int q = 0; q < PER; ++q) join(s, p[q].max, p[q].norm, p[q].low, p[q].small);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) join(s, __shfl_xor(s.max, o), __shfl_xor(s.norm, o), __shfl_xor(s.low, o), __shfl_xor(s.small, o));
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  if (threadIdx.x > 0) return;
  Sum f[3] = {};
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    Sum m = sums[4 * i];
#pragma unroll
    for (int w = 1; w < 4; ++w) join(m, sums[4 * i + w].max, sums[4 * i + w].norm, sums[4 * i + w].low, sums[4 * i + w].small);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (a.m[i].slot == k) join(f[k], m.max, m.norm, m.low, m.small);  // a place without a matrix has zeros
  }
  bool wide = false;
  if constexpr (__is_same(T, float)) {
    const int64_t rows[3] = {rows_x >= 0 ? rows_x : mode->live, rows_w, rows_dh};  // -1: those that count
    int sum = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int uneven = f[k].low > 0 ? (int)(__float_as_uint(f[k].max) >> 23) + f[k].low - 255 : 0;
      wide = wide || f[k].small * 4 > rows[k] || (k < 2 && uneven > kEven);
      sum += uneven;
    }
    wide = wide || (rows_dh > 0 && sum > kEvenG);
  }
  mode->wide = wide ? 1 : 0;
  mode->sx = wide ? 1.0f : pow2_to(f[0].max, 15);
  mode->sw = wide ? 1.0f : pow2_to(f[1].max, 15);
  mode->sg = wide ? 1.0f : gated ? pow2_to(1.15f * fminf(f[2].max, 1e38f), f[0].norm, f[1].norm, 15) : 32768.0f;
}

// Rows to operand rows.  A wave per row, 8 columns a lane; a matrix's last blocks zero the rows behind the last one that
// counts, up to the next multiple of 128.
template <typename T>
__global__ void __launch_bounds__(kThreads) rows_copy_kernel(RowsArgs a, int dp) {
  const int i = matrix_of(a, blockIdx.x), lane = (int)threadIdx.x & 63;
  const RowsCopy m = a.m[i];
  const int64_t r = ((int64_t)blockIdx.x - a.first[i]) * 4 + (threadIdx.x >> 6);
  int64_t to = r;
  bool zero = false;
  if (r >= m.rows) {
    if (m.pos == nullptr) return;
    const int64_t live = a.mode->live;
    to = live + (r - m.rows);
    if (to >= (live + 127) / 128 * 128) return;
    zero = true;
  } else if (m.pos != nullptr) {
    to = m.pos[r];
    if (to < 0) return;
  }
  const float s = m.slot == 0 ? scale_x<T>(a.mode) : scale_w<T>(a.mode);
  char* const out = m.dst + to * 64;
  const T* in = (const T*)m.src + r * m.ld;
  for (int c = lane * 8; c < dp; c += 512) {
    T x[8];
    if (zero || c >= m.d) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (T)0.0f;
    } else {
      load8(in, c, m.d, a.vec[i] != 0, x);
    }
    by_format<T>(a.mode, [&](auto wide) {
      using F = Wide<T, decltype(wide)::value>;
      using E = typename F::E;
      typedef __attribute__((__vector_size__(16))) E E8;
      E8 t[F::P];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (F::P == 1) {
          t[0][e] = x[e];
        } else {
          const Terms<E, F::P> v(x[e] * s);
#pragma unroll
          for (int k = 0; k < F::P; ++k) t[k][e] = v.t[k];
        }
      }
#pragma unroll
      for (int k = 0; k < F::P; ++k) *reinterpret_cast<E8*>(out + (c >> 5) * m.blk + (c & 31) * 2 + k * m.plane_bytes) = t[k];
    });
  }
}

struct ProductArgs {
  int64_t N, n_pad;
  int d;
  int64_t dp;
  int tm, dx_tiles, dx_blocks, dw_blocks, dx_steps, dw_tn, halves, cols;
  int64_t C;
  WideShare share;
  MmSegs dx_segs[2], dw_segs[2];  // of the narrow and the wide format
  const char* x; int64_t x_ld, x_blk; int x_rows;
  const char* w; int64_t w_ld, w_blk; int w_rows;
  const char* g; int64_t g_half;
  float* dx_part; int dx_add;
  void* dw0; void* dw1;
  float* dw_part;
  const WideMode* mode;
  GradUnit unit; const float* cmax;
  int use_live, gated, vec;
};

// A block per tile and range of its k: dx[n][m] = sum_v G[n][v] W[v][m], and dW[v][m] = sum_n G[n][v] x[n][m].  Both in one
// launch, the longer blocks first, so that neither leaves CUs idle at its end.  Ranges of one tile, and tiles of one block
// of rows or columns of G, stand side by side: an XCD's blocks then read the same rows of W or x at the same time.  (Cut
// where equal shares end instead, the blocks start at places of their own in W: 12% slower at 8192 rows.)
template <typename T, bool WIDE>
struct Products {
  using E = typename Wide<T, WIDE>::E;
  using TX = MmTile<E, 256, kTileN, 2, 4, true, false, false, 4>;
  using TW = MmTile<E, 256, kTileN, 2, 4, true, true, false, 4>;

  // Steps [from, to) of dx's tile (tm, tn), as its part `part`.
  __device__ static inline void dx(const ProductArgs& p, LdsChar* lds, int64_t N, int tm, int tn, int part, int from, int to) {
    const int n0 = tn * kTileN, m0 = tm * 256;
    if (n0 >= N) return;
    typename TX::Acc acc;
    TX::clear(acc);
    const typename TX::Side A{p.w + (m0 >> 5) * p.w_blk, (int)(p.dp - m0), p.w_ld, p.w_blk, p.w_rows, 0};
    const typename TX::Side B{p.g + (int64_t)n0 * 64, (int)(p.n_pad - n0), 64, p.n_pad * 64, 0, 0};
    if (to > from) TX::run(acc, lds, A, B, p.dx_segs[WIDE], from * 32, to - from);
    float* out = p.dx_part + ((int64_t)part * p.n_pad + n0) * p.dp + m0;
    auto fn = [&](int i, int j, int g) { return quad<float>([&](int e) { return acc[i][j][4 * g + e]; }); };
    const int rows = (int)(N - n0 < kTileN ? N - n0 : kTileN);
    if (p.dx_add) TX::template store_rows<float, true>(lds, out, p.dp, rows, (int)(p.dp - m0), true, fn);
    else TX::template store_rows<float, false>(lds, out, p.dp, rows, (int)(p.dp - m0), true, fn);
  }

  // Range t % dw_split of a tile of dW.
  __device__ static inline void dw(const ProductArgs& p, LdsChar* lds, int64_t N, int64_t t) {
    const int split = (int)(t % p.share.dw_split);
    t /= p.share.dw_split;
    const int tm = (int)(t % p.tm);
    t /= p.tm;
    const int tn = (int)(t % p.dw_tn), half = (int)(t / p.dw_tn);
    const int n0 = tn * kTileN, m0 = tm * 256;
    const int steps = (int)((N + 31) / 32), from = (int)((int64_t)steps * split / p.share.dw_split),
              to = (int)((int64_t)steps * (split + 1) / p.share.dw_split);
    typename TW::Acc acc;
    TW::clear(acc);
    const typename TW::Side A{p.x + (m0 >> 5) * p.x_blk, (int)(p.dp - m0), p.x_ld, p.x_blk, p.x_rows, 0};
    const typename TW::Side B{p.g + half * p.g_half + (n0 >> 5) * p.n_pad * 64, (int)(p.C - n0), 64, p.n_pad * 64, (int)p.n_pad, 0};
    if (to > from) TW::run(acc, lds, A, B, p.dw_segs[WIDE], from * 32, to - from);
    const int rows = p.cols - n0 < kTileN ? p.cols - n0 : kTileN;
    if (p.share.dw_split > 1) {
      float* out = p.dw_part + (((int64_t)split * p.halves + half) * p.C + n0) * p.dp + m0;
      TW::template store_rows<float, false>(lds, out, p.dp, rows, (int)(p.dp - m0), true,
                                            [&](int i, int j, int g) { return quad<float>([&](int e) { return acc[i][j][4 * g + e]; }); });
    } else {
      const float f = unit_of(p.unit, p.mode, p.cmax) / scale_g<T>(p.mode, p.gated), fx = 1.0f / scale_x<T>(p.mode);
      T* out = (T*)(half ? p.dw1 : p.dw0) + (int64_t)n0 * p.d + m0;
      TW::template store_rows<T, false>(lds, out, p.d, rows, p.d - m0, p.vec != 0,
                                        [&](int i, int j, int g) { return quad<T>([&](int e) { return acc[i][j][4 * g + e] * f * fx; }); });
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kProductThreads, 2) products_kernel(ProductArgs p) {
  __shared__ char smem[Products<T, false>::TX::LDS];
  LdsChar* lds = (LdsChar*)smem;
  const int64_t N = p.use_live ? p.mode->live : p.N;
  const int first = p.share.dx_first ? p.dx_blocks : p.dw_blocks;
  const bool head = (int)blockIdx.x < first;
  const int64_t at = head ? blockIdx.x : (int64_t)blockIdx.x - first;
  by_format<T>(p.mode, [&](auto wide) {
    using P = Products<T, decltype(wide)::value>;
    if (head == p.share.dx_first) {
      int64_t t = xcd_order(at, p.dx_blocks);
      const int split = (int)(t % p.share.dx_split);
      t /= p.share.dx_split;
      const int from = (int)((int64_t)p.dx_steps * split / p.share.dx_split), to = (int)((int64_t)p.dx_steps * (split + 1) / p.share.dx_split);
      P::dx(p, lds, N, (int)(t % p.tm), (int)(t / p.tm), split, from, to);
    } else {
      P::dw(p, lds, N, xcd_order(at, p.dw_blocks));
    }
  });
}

// As many blocks as CUs, each with its share of both products (WideShare).  Blocks of an XCD hold one range of many tiles,
// so that they read the same rows of W at the same time.
template <typename T>
__global__ void __launch_bounds__(kProductThreads, 2) shares_kernel(ProductArgs p) {
  __shared__ char smem[Products<T, false>::TX::LDS];
  LdsChar* lds = (LdsChar*)smem;
  const int64_t N = p.use_live ? p.mode->live : p.N;
  const int slot = (int)xcd_order(blockIdx.x, p.share.slots);
  by_format<T>(p.mode, [&](auto wide) {
    using P = Products<T, decltype(wide)::value>;
    for (int t = slot; t < p.dw_blocks; t += p.share.slots) P::dw(p, lds, N, t);
    const int part = slot / p.dx_tiles, tile = slot - part * p.dx_tiles;
    if (part >= p.share.dx_split) return;
    const int a = p.share.a, b = p.share.b, n = p.share.n_a;
    int from = part < n ? part * a : n * a + (part - n) * b, to = part < n ? from + a : from + b;
    if (part == p.share.dx_split - 1 || to > p.dx_steps) to = p.dx_steps;
    if (from > to) from = to;
    P::dx(p, lds, N, tile % p.tm, tile / p.tm, part, from, to);
  });
}

// Sums of parts in their order, scaled, as rows of T.  A wave per row; the second matrix's rows follow the first's.
struct PartArgs {
  const float* part; int64_t part_stride, half_stride;
  int split;
  int64_t rows;
  int d, dp;
  const int* pos;
  const WideMode* mode;
  GradUnit unit; const float* cmax;
  int gated, by_x;
  void* out0; void* out1;
};
template <typename T>
__global__ void __launch_bounds__(kThreads) parts_kernel(PartArgs a) {
  int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  T* out = (T*)a.out0;
  const float* part = a.part;
  if (r >= a.rows) {
    if (a.out1 == nullptr || (r -= a.rows) >= a.rows) return;
    out = (T*)a.out1;
    part += a.half_stride;
  }
  const int64_t at = a.pos == nullptr ? r : a.pos[r];
  const float f = unit_of(a.unit, a.mode, a.cmax) / scale_g<T>(a.mode, a.gated), f2 = 1.0f / (a.by_x ? scale_x<T>(a.mode) : scale_w<T>(a.mode));
  for (int c = ((int)threadIdx.x & 63) * 4; c < a.d; c += 256) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at >= 0) {
#pragma unroll 4
      for (int s = 0; s < a.split; ++s) v += *reinterpret_cast<const f32x4*>(part + s * a.part_stride + at * a.dp + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = v[e] * f * f2;
    }
    T* o = out + r * a.d + c;
    if (c + 4 <= a.d && a.d % 4 == 0) store4(o, v[0], v[1], v[2], v[3]);
    else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.d) o[e] = from_f<T>(v[e]);
    }
  }
}

// Blocks of each matrix: a wave per row, at most `most` blocks.
RowsArgs rows_args(const RowsCopies& c, int64_t most, bool zeros, int64_t* blocks) {
  RowsArgs a = {};
  const int64_t es = c.dtype == 0 ? 4 : 2;
  int64_t at = 0;
  for (int i = 0; i < kCopies; ++i) {
    a.first[i] = at;
    if (i >= c.n) continue;
    a.m[i] = c.m[i];
    a.vec[i] = ((uintptr_t)c.m[i].src & 15) == 0 && c.m[i].ld * es % 16 == 0;
    const int64_t b = (c.m[i].rows + (zeros && c.m[i].pos != nullptr ? 128 : 0) + 3) / 4;
    at += b < most ? b : most;
  }
  a.first[kCopies] = at;
  for (int i = c.n; i < kCopies; ++i) a.first[i] = at;
  a.mode = c.mode;
  *blocks = at;
  return a;
}

template <typename T>
hipError_t rows_copy(const RowsCopies& c, hipStream_t s) {
  int64_t blocks;
  const RowsArgs a = rows_args(c, (int64_t)1 << 40, true, &blocks);
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL(rows_copy_kernel<T>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a, (int)wide_dp(c.m[0].d));
  return hipGetLastError();
}

template <typename T>
hipError_t wide_mode(const RowsCopies& c, WidePart* parts, WideMode* mode, int gated, hipStream_t s) {
  int64_t blocks, rows[3] = {0, 0, 0};
  const RowsArgs a = rows_args(c, kMaxBlocks, false, &blocks);
  if (blocks > 0) {
    hipLaunchKernelGGL(rows_max_kernel<T>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  for (int i = 0; i < c.n; ++i) rows[c.m[i].slot] += c.m[i].pos != nullptr ? -1 : c.m[i].rows;
  hipLaunchKernelGGL(wide_mode_kernel<T>, dim3(1), dim3(1024), 0, s, a, parts, mode, gated, rows[0], rows[1], rows[2]);
  return hipGetLastError();
}

template <typename T>
hipError_t products(const WideProducts& p, hipStream_t s) {
  constexpr int P = Wide<T>::P;
  const bool dx = p.dx_part != nullptr, dw = p.dw[0] != nullptr;
  if (!dx && !dw) return hipSuccess;
  ProductArgs a = {};
  a.N = p.N; a.n_pad = p.n_pad; a.d = p.d; a.dp = p.dp; a.share = p.share;
  a.tm = (int)((p.dp + 255) / 256);
  a.dx_tiles = dx ? a.tm * (int)((p.n_pad + kTileN - 1) / kTileN) : 0;
  a.dx_blocks = a.dx_tiles * p.share.dx_split;
  a.dx_steps = (p.cols + 63) / 64 * 2;  // columns of G that are there: the gated kernel fills 64 at a time
  a.dw_tn = (p.cols + kTileN - 1) / kTileN;
  a.dw_blocks = dw ? a.tm * a.dw_tn * p.halves * p.share.dw_split : 0;
  a.halves = p.halves; a.cols = p.cols;
  a.C = p.C;
  // (first, second) terms: low ones first
  int n = 0;
  for (int t = p.g_terms - 1; t >= 0; --t) {
    for (int half = 0; half < p.halves; ++half) {
      const int64_t wh = half ? p.w[1] - p.w[0] : 0, gh = half * p.g_half;
      a.dx_segs[0].a[n] = wh; a.dx_segs[0].b[n++] = gh + t * p.g_plane;
      if (t == 1 && P == 2) { a.dx_segs[0].a[n] = wh + p.w_plane; a.dx_segs[0].b[n++] = gh; }
    }
    if (t == 1) a.dx_segs[0].low = n;
  }
  a.dx_segs[0].n = n;
  n = 0;
  if (p.g_terms == 2) {
    a.dw_segs[0].a[n] = 0; a.dw_segs[0].b[n++] = p.g_plane;
    if (P == 2) { a.dw_segs[0].a[n] = p.x_plane; a.dw_segs[0].b[n++] = 0; }
  }
  a.dw_segs[0].low = n;
  a.dw_segs[0].a[n] = 0; a.dw_segs[0].b[n++] = 0;
  a.dw_segs[0].n = n;
  if (P == 2) {
    for (int order = 2; order >= 0; --order)
      for (int half = 0; half < p.halves; ++half)
        add_wide_segs(a.dx_segs[1], order, half ? p.w[1] - p.w[0] : 0, p.w_plane, half * p.g_half, p.g_plane);
    for (int order = 2; order >= 0; --order) add_wide_segs(a.dw_segs[1], order, 0, p.x_plane, 0, p.g_plane);
  }
  a.x = p.x; a.x_ld = p.x_ld; a.x_blk = p.x_blk; a.x_rows = p.x_rows;
  a.w = p.w[0]; a.w_ld = p.w_ld; a.w_blk = p.w_blk; a.w_rows = p.w_rows;
  a.g = p.g; a.g_half = p.g_half;
  a.dx_part = p.dx_part; a.dx_add = p.dx_add;
  a.dw0 = p.dw[0]; a.dw1 = p.dw[1]; a.dw_part = p.dw_part;
  a.mode = p.mode; a.unit = p.unit; a.cmax = p.cmax; a.use_live = p.use_live; a.gated = p.gated;
  a.vec = (int64_t)p.d * sizeof(T) % 16 == 0 && ((uintptr_t)p.dw[0] & 15) == 0 && ((uintptr_t)p.dw[1] & 15) == 0;
  if (p.share.slots > 0) hipLaunchKernelGGL(shares_kernel<T>, dim3((unsigned)p.share.slots), dim3(kProductThreads), 0, s, a);
  else hipLaunchKernelGGL(products_kernel<T>, dim3((unsigned)(a.dx_blocks + a.dw_blocks)), dim3(kProductThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !dw || p.share.dw_split == 1) return e;
  PartArgs q = {};
  q.part = p.dw_part; q.part_stride = (int64_t)p.halves * p.C * p.dp; q.half_stride = p.C * p.dp; q.split = p.share.dw_split;
  q.rows = p.cols; q.d = p.d; q.dp = (int)p.dp; q.mode = p.mode; q.unit = p.unit; q.cmax = p.cmax; q.gated = p.gated; q.by_x = 1;
  q.out0 = p.dw[0]; q.out1 = p.halves == 2 ? p.dw[1] : nullptr;
  hipLaunchKernelGGL(parts_kernel<T>, dim3((unsigned)((q.rows * p.halves + 3) / 4)), dim3(kThreads), 0, s, q);
  return hipGetLastError();
}

template <typename T>
hipError_t finish(const WideFinish& f, hipStream_t s) {
  if (f.N == 0) return hipSuccess;
  PartArgs q = {};
  q.part = f.part; q.part_stride = f.n_pad * f.dp; q.split = f.split;
  q.rows = f.N; q.d = f.d; q.dp = (int)f.dp; q.pos = f.pos; q.mode = f.mode; q.unit = f.unit; q.cmax = f.cmax; q.gated = f.gated;
  q.out0 = f.dx;
  hipLaunchKernelGGL(parts_kernel<T>, dim3((unsigned)((f.N + 3) / 4)), dim3(kThreads), 0, s, q);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rows_copy(const RowsCopies& c, hipStream_t s) {
  return c.dtype == 0 ? rows_copy<float>(c, s) : c.dtype == 1 ? rows_copy<bf16>(c, s) : rows_copy<f16>(c, s);
}
hipError_t launch_wide_mode(const RowsCopies& c, WidePart* parts, WideMode* mode, int gated, hipStream_t s) {
  return c.dtype == 0 ? wide_mode<float>(c, parts, mode, gated, s) : wide_mode<f16>(c, parts, mode, gated, s);
}
hipError_t launch_wide_products(const WideProducts& p, hipStream_t s) {
  return p.dtype == 0 ? products<float>(p, s) : p.dtype == 1 ? products<bf16>(p, s) : products<f16>(p, s);
}
hipError_t launch_wide_finish(const WideFinish& f, hipStream_t s) {
  return f.dtype == 0 ? finish<float>(f, s) : f.dtype == 1 ? finish<bf16>(f, s) : finish<f16>(f, s);
}

// Blocks in flight take the next block of the grid as they end: the time until all `n2` blocks of length l2 have ended that
// follow n1 of length l1.
constexpr int64_t kInFlight = 256;  // a block a CU
static int64_t two_kinds(int64_t n1, int64_t l1, int64_t n2, int64_t l2) {
  const int64_t r = n1 / kInFlight, more = n1 - r * kInFlight, few = kInFlight - more;
  const int64_t a = r * l1, b = a + l1;  // `more` places are free at b, the `few` others at a
  const int64_t end1 = more > 0 ? b : a;
  if (n2 == 0) return end1;
  auto fits = [&](int64_t t) { return few * ((t - a) / l2) + (t > b ? more * ((t - b) / l2) : 0) >= n2; };
  // without a remainder, then the next ends of both groups of places
  int64_t t = a + (n2 * l2 + few - 1) / few;
  if (t > b) t = (n2 * l2 + few * a + more * b + kInFlight - 1) / kInFlight;
  const int64_t ta = a + (t - a + l2 - 1) / l2 * l2, tb = t <= b ? b + l2 : b + (t - b + l2 - 1) / l2 * l2;
  int64_t lo = ta < tb ? ta : tb, hi = ta < tb ? tb : ta;
  if (more == 0) lo = hi = ta;
  t = fits(lo) ? lo : fits(hi) ? hi : lo + l2;
  return t > end1 ? t : end1;
}

WideShare wide_share(int64_t N, int d, int64_t C, int halves, int segs, bool dx, bool dw) {
  // What a block costs beside its stages, in stages of 0.7 us: 12 to fill and drain its pipeline, 5 to store a tile, and
  // where all CUs store fp32 tiles at once 20 more (64 MB at 4 TB/s); adding them up takes a launch, 8, and as much again.
  constexpr int64_t kFill = 12, kStore = 5, kFloat = 20, kLaunch = 8;
  const int64_t tm = (wide_dp(d) + 255) / 256;
  const int64_t tx = dx ? tm * ((N + kTileN - 1) / kTileN) : 0, kx = C / 32 * segs * halves;
  const int64_t tw = dw ? tm * (C / kTileN) * halves : 0, kw = (N + 31) / 32 * segs;
  constexpr int kCuts[] = {1, 2, 3, 4, 5, 6, 8, 11, 16, 24, 32, 48, 64};
  WideShare best = {1, 1, true, -1, 0, 0, 0, 0};
  for (const int sx : kCuts) {
    if (sx > 1 && (!dx || kx / sx < 8)) break;
    const int64_t nx = tx * sx;
    for (const int sw : kCuts) {
      if (sw > 1 && (!dw || kw / sw < 8)) break;
      const int64_t nw = tw * sw, floats = nx + (sw > 1 ? nw : 0), busy = kFloat * (floats < kInFlight ? floats : kInFlight) / kInFlight;
      const int64_t lx = (kx + sx - 1) / sx + kFill + kStore + busy;
      const int64_t lw = (kw + sw - 1) / sw + kFill + kStore + (sw > 1 ? busy : 0);
      const bool first = lx >= lw;
      const int64_t sum = kFloat * floats / kInFlight + (sw > 1 ? kLaunch : 0);
      const int64_t cost = sum + (first ? two_kinds(nx, lx, nw, lw) : two_kinds(nw, lw, nx, lx));
      if (best.cost < 0 || cost < best.cost) best = WideShare{sx, sw, first, cost, 0, 0, 0, 0};
    }
  }
  // shares of both: `ranges` of dx's tiles for each CU's block, and what dW's leave over
  const int64_t ranges = tx > 0 && tw > 0 ? kInFlight / tx : 0, xw = segs * halves, steps = C / 32;
  if (ranges < 2 || ranges > 64) return best;
  for (const int sw : kCuts) {
    if (sw > 1 && kw / sw < 8) break;
    const int64_t nw = tw * sw, floats = ranges * tx + (sw > 1 ? nw : 0), busy = kFloat * (floats < kInFlight ? floats : kInFlight) / kInFlight;
    const int64_t lw = (kw + sw - 1) / sw + kFill + kStore + (sw > 1 ? busy : 0), lx = kFill + kStore + busy;
    const int64_t q = nw / kInFlight, more = nw - q * kInFlight;  // `more` blocks have q + 1 ranges of dW
    int64_t n_a = (more + tx - 1) / tx;
    n_a = n_a < ranges ? n_a : ranges;
    const int64_t goal = (kx + (n_a * (q + 1) + (ranges - n_a) * q) * lw + ranges - 1) / ranges;
    const int64_t a = n_a > 0 ? (goal - (q + 1) * lw) / xw : 0;
    if (n_a > 0 && a * xw < 16) continue;
    const int64_t rest = n_a < ranges ? (steps - n_a * a + ranges - n_a - 1) / (ranges - n_a) : 0;
    if (n_a < ranges && (rest < 1 || steps - n_a * a < 1)) continue;
    const int64_t a_all = n_a == ranges ? (steps + ranges - 1) / ranges : a;
    const int64_t cost = goal + xw + lx + kFloat * floats / kInFlight + (sw > 1 ? kLaunch : 0);
    if (cost < best.cost)
      best = WideShare{(int)ranges, sw, false, cost, (int)kInFlight, (int)n_a, (int)a_all, (int)(rest > 0 ? rest : 1)};
  }
  return best;
}

int64_t wide_piece(int64_t N, int d, int64_t rows, int halves, int segs, bool dx, bool dw, int64_t bytes_of_column, WideShare* share) {
  // the sizes of the last call: a backward pass asks twice, for its workspace and for its launches
  struct Memo { int64_t key[8], C; WideShare share; };
  static thread_local Memo memo = {{-1}, 0, {}};
  const int64_t key[8] = {N, d, rows, halves, segs, dx, dw, bytes_of_column};
  if (memcmp(memo.key, key, sizeof(key)) == 0) {
    *share = memo.share;
    return memo.C;
  }
  const int64_t all = round_up(rows, 256);
  int64_t chosen = 0, cost = -1;
  for (int s = 30; s >= 28; --s) {
    int64_t C = ((int64_t)1 << s) / bytes_of_column / 256 * 256;
    C = C < 256 ? 256 : C > all ? all : C;
    const int64_t pieces = (all + C - 1) / C;  // of equal size
    C = round_up((all + pieces - 1) / pieces, 256);
    const WideShare w = wide_share(N, d, C, halves, segs, dx, dw);
    if (cost < 0 || w.cost * pieces < cost) {
      cost = w.cost * pieces;
      chosen = C;
      *share = w;
    }
  }
  memcpy(memo.key, key, sizeof(key));
  memo.C = chosen;
  memo.share = *share;
  return chosen;
}

}  // namespace msa

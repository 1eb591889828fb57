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

__global__ void hdr_clear_kernel(WideHdr* h) {
  for (int i = (int)threadIdx.x; i < kHdrWords; i += kThreads) reinterpret_cast<uint32_t*>(h)[i] = 0u;
}

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
  WideHdr* hdr;
};
__device__ inline int matrix_of(const RowsArgs& a, int64_t block) {
  int i = 0;
#pragma unroll
  for (int k = 1; k < kCopies; ++k) i += block >= a.first[k] ? 1 : 0;
  return i;
}

// A wave takes rows in turn, of the matrix that its block belongs to.
template <typename T>
__global__ void __launch_bounds__(kThreads) rows_max_kernel(RowsArgs a) {
  const int i = matrix_of(a, blockIdx.x), lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const RowsCopy m = a.m[i];
  const int64_t step = (a.first[i + 1] - a.first[i]) * 4;
  float mx = 0.0f, nx = 0.0f;
  for (int64_t r = ((int64_t)blockIdx.x - a.first[i]) * 4 + wave; r < m.rows; r += step) {
    if (m.pos != nullptr && m.pos[r] < 0) continue;
    const T* p = (const T*)m.src + r * m.ld;
    float ss = 0.0f, rx = 0.0f;
    for (int c = lane * 8; c < m.d; c += 512) {
      T x[8];
      load8(p, c, m.d, a.vec[i] != 0, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = fabsf(to_f(x[e]));
        if (v < INFINITY) {
          rx = fmaxf(rx, v);
          ss = fmaf(v, v, ss);
        }
      }
    }
    mx = fmaxf(mx, rx);
    if (m.norms) {
      ss = wave_sum(ss);
      if (ss > 1e-30f && ss < INFINITY) {
        nx = fmaxf(nx, sqrtf(ss));
      } else {  // squares left fp32's range: a bound that does not
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) rx = fmaxf(rx, __shfl_xor(rx, o));
        nx = fmaxf(nx, fminf(rx * sqrtf((float)m.d), 3e38f));
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  __shared__ float sm[4], sn[4];
  if (lane == 0) { sm[wave] = mx; sn[wave] = nx; }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int at = (int)blockIdx.x & (kSlots - 1);
    atomicMax(&a.hdr->max[m.slot][at][0], __float_as_uint(fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]))));
    if (m.norms) atomicMax(&a.hdr->max[kNormX + m.slot][at][0], __float_as_uint(fmaxf(fmaxf(sn[0], sn[1]), fmaxf(sn[2], sn[3]))));
  }
}

// Rows to operand rows.  A wave per row, 8 columns a lane; a matrix's last blocks zero the rows behind the last one that
// counts, up to the next multiple of 128.
template <typename T>
__global__ void __launch_bounds__(kThreads) rows_copy_kernel(RowsArgs a, int dp) {
  using E = typename Wide<T>::E;
  const int i = matrix_of(a, blockIdx.x), lane = (int)threadIdx.x & 63;
  const RowsCopy m = a.m[i];
  const int64_t r = ((int64_t)blockIdx.x - a.first[i]) * 4 + (threadIdx.x >> 6);
  int64_t to = r;
  bool zero = false;
  if (r >= m.rows) {
    if (m.pos == nullptr) return;
    const int64_t live = a.hdr->live;
    to = live + (r - m.rows);
    if (to >= (live + 127) / 128 * 128) return;
    zero = true;
  } else if (m.pos != nullptr) {
    to = m.pos[r];
    if (to < 0) return;
  }
  float s = 1.0f;
  if constexpr (Wide<T>::P == 2) s = m.slot == 0 ? scale_x<T>(a.hdr) : scale_w<T>(a.hdr);
  char* const out = m.dst + to * 64;
  const T* in = (const T*)m.src + r * m.ld;
  typedef __attribute__((__vector_size__(16))) E E8;
  for (int c = lane * 8; c < dp; c += 512) {
    T x[8];
    if (zero || c >= m.d) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (T)0.0f;
    } else {
      load8(in, c, m.d, a.vec[i] != 0, x);
    }
    E8 h;
    if constexpr (Wide<T>::P == 2) {
      E8 l;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Terms<E> t(x[e] * s);
        h[e] = t.h;
        l[e] = t.l;
      }
      *reinterpret_cast<E8*>(out + (c >> 5) * m.blk + (c & 31) * 2 + m.plane_bytes) = l;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = x[e];
    }
    *reinterpret_cast<E8*>(out + (c >> 5) * m.blk + (c & 31) * 2) = h;
  }
}

struct ProductArgs {
  int64_t N, n_pad;
  int d;
  int64_t dp;
  int tm, dx_tiles, dx_blocks, dw_blocks, dx_steps, dw_tn, halves, cols;
  int64_t C;
  WideShare share;
  MmSegs dx_segs, dw_segs;
  const char* x; int64_t x_ld, x_blk; int x_rows;
  const char* w; int64_t w_ld, w_blk; int w_rows;
  const char* g; int64_t g_half;
  float* dx_part; int dx_add;
  void* dw0; void* dw1;
  float* dw_part;
  const WideHdr* hdr;
  GradUnit unit; const float* cmax;
  int use_live, gated, vec;
};

// A block per tile and range of its k: dx[n][m] = sum_v G[n][v] W[v][m], and dW[v][m] = sum_n G[n][v] x[n][m].  Both in one
// launch, the longer blocks first, so that neither leaves CUs idle at its end.  Ranges of one tile, and tiles of one block
// of rows or columns of G, stand side by side: an XCD's blocks then read the same rows of W or x at the same time.  (Cut
// where equal shares end instead, the blocks start at places of their own in W: 12% slower at 8192 rows.)
template <typename T>
struct Products {
  using E = typename Wide<T>::E;
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
    if (to > from) TX::run(acc, lds, A, B, p.dx_segs, from * 32, to - from);
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
    if (to > from) TW::run(acc, lds, A, B, p.dw_segs, from * 32, to - from);
    const int rows = p.cols - n0 < kTileN ? p.cols - n0 : kTileN;
    if (p.share.dw_split > 1) {
      float* out = p.dw_part + (((int64_t)split * p.halves + half) * p.C + n0) * p.dp + m0;
      TW::template store_rows<float, false>(lds, out, p.dp, rows, (int)(p.dp - m0), true,
                                            [&](int i, int j, int g) { return quad<float>([&](int e) { return acc[i][j][4 * g + e]; }); });
    } else {
      const float f = unit_of(p.unit, p.hdr, p.cmax) / scale_g<T>(p.hdr, p.gated), fx = 1.0f / scale_x<T>(p.hdr);
      T* out = (T*)(half ? p.dw1 : p.dw0) + (int64_t)n0 * p.d + m0;
      TW::template store_rows<T, false>(lds, out, p.d, rows, p.d - m0, p.vec != 0,
                                        [&](int i, int j, int g) { return quad<T>([&](int e) { return acc[i][j][4 * g + e] * f * fx; }); });
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kProductThreads, 2) products_kernel(ProductArgs p) {
  __shared__ char smem[Products<T>::TX::LDS];
  LdsChar* lds = (LdsChar*)smem;
  const int64_t N = p.use_live ? p.hdr->live : p.N;
  const int first = p.share.dx_first ? p.dx_blocks : p.dw_blocks;
  const bool head = (int)blockIdx.x < first;
  const int64_t at = head ? blockIdx.x : (int64_t)blockIdx.x - first;
  if (head == p.share.dx_first) {
    int64_t t = xcd_order(at, p.dx_blocks);
    const int split = (int)(t % p.share.dx_split);
    t /= p.share.dx_split;
    const int from = (int)((int64_t)p.dx_steps * split / p.share.dx_split), to = (int)((int64_t)p.dx_steps * (split + 1) / p.share.dx_split);
    Products<T>::dx(p, lds, N, (int)(t % p.tm), (int)(t / p.tm), split, from, to);
  } else {
    Products<T>::dw(p, lds, N, xcd_order(at, p.dw_blocks));
  }
}

// As many blocks as CUs, each with its share of both products (WideShare).  Blocks of an XCD hold one range of many tiles,
// so that they read the same rows of W at the same time.
template <typename T>
__global__ void __launch_bounds__(kProductThreads, 2) shares_kernel(ProductArgs p) {
  __shared__ char smem[Products<T>::TX::LDS];
  LdsChar* lds = (LdsChar*)smem;
  const int64_t N = p.use_live ? p.hdr->live : p.N;
  const int slot = (int)xcd_order(blockIdx.x, p.share.slots);
  for (int t = slot; t < p.dw_blocks; t += p.share.slots) Products<T>::dw(p, lds, N, t);
  const int part = slot / p.dx_tiles, tile = slot - part * p.dx_tiles;
  if (part >= p.share.dx_split) return;
  const int a = p.share.a, b = p.share.b, n = p.share.n_a;
  int from = part < n ? part * a : n * a + (part - n) * b, to = part < n ? from + a : from + b;
  if (part == p.share.dx_split - 1 || to > p.dx_steps) to = p.dx_steps;
  if (from > to) from = to;
  Products<T>::dx(p, lds, N, tile % p.tm, tile / p.tm, part, from, to);
}

// Sums of parts in their order, scaled, as rows of T.  A wave per row; the second matrix's rows follow the first's.
struct PartArgs {
  const float* part; int64_t part_stride, half_stride;
  int split;
  int64_t rows;
  int d, dp;
  const int* pos;
  const WideHdr* hdr;
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
  const float f = unit_of(a.unit, a.hdr, a.cmax) / scale_g<T>(a.hdr, a.gated), f2 = 1.0f / (a.by_x ? scale_x<T>(a.hdr) : scale_w<T>(a.hdr));
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
  a.hdr = c.hdr;
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
hipError_t rows_max(const RowsCopies& c, hipStream_t s) {
  int64_t blocks;
  const RowsArgs a = rows_args(c, 1024, false, &blocks);
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL(rows_max_kernel<T>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
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
      a.dx_segs.a[n] = wh; a.dx_segs.b[n++] = gh + t * p.g_plane;
      if (t == 1 && P == 2) { a.dx_segs.a[n] = wh + p.w_plane; a.dx_segs.b[n++] = gh; }
    }
    if (t == 1) a.dx_segs.low = n;
  }
  a.dx_segs.n = n;
  n = 0;
  if (p.g_terms == 2) {
    a.dw_segs.a[n] = 0; a.dw_segs.b[n++] = p.g_plane;
    if (P == 2) { a.dw_segs.a[n] = p.x_plane; a.dw_segs.b[n++] = 0; }
  }
  a.dw_segs.low = n;
  a.dw_segs.a[n] = 0; a.dw_segs.b[n++] = 0;
  a.dw_segs.n = n;
  a.x = p.x; a.x_ld = p.x_ld; a.x_blk = p.x_blk; a.x_rows = p.x_rows;
  a.w = p.w[0]; a.w_ld = p.w_ld; a.w_blk = p.w_blk; a.w_rows = p.w_rows;
  a.g = p.g; a.g_half = p.g_half;
  a.dx_part = p.dx_part; a.dx_add = p.dx_add;
  a.dw0 = p.dw[0]; a.dw1 = p.dw[1]; a.dw_part = p.dw_part;
  a.hdr = p.hdr; a.unit = p.unit; a.cmax = p.cmax; a.use_live = p.use_live; a.gated = p.gated;
  a.vec = (int64_t)p.d * sizeof(T) % 16 == 0 && ((uintptr_t)p.dw[0] & 15) == 0 && ((uintptr_t)p.dw[1] & 15) == 0;
  if (p.share.slots > 0) hipLaunchKernelGGL(shares_kernel<T>, dim3((unsigned)p.share.slots), dim3(kProductThreads), 0, s, a);
  else hipLaunchKernelGGL(products_kernel<T>, dim3((unsigned)(a.dx_blocks + a.dw_blocks)), dim3(kProductThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !dw || p.share.dw_split == 1) return e;
  PartArgs q = {};
  q.part = p.dw_part; q.part_stride = (int64_t)p.halves * p.C * p.dp; q.half_stride = p.C * p.dp; q.split = p.share.dw_split;
  q.rows = p.cols; q.d = p.d; q.dp = (int)p.dp; q.hdr = p.hdr; q.unit = p.unit; q.cmax = p.cmax; q.gated = p.gated; q.by_x = 1;
  q.out0 = p.dw[0]; q.out1 = p.halves == 2 ? p.dw[1] : nullptr;
  hipLaunchKernelGGL(parts_kernel<T>, dim3((unsigned)((q.rows * p.halves + 3) / 4)), dim3(kThreads), 0, s, q);
  return hipGetLastError();
}

template <typename T>
hipError_t finish(const WideFinish& f, hipStream_t s) {
  if (f.N == 0) return hipSuccess;
  PartArgs q = {};
  q.part = f.part; q.part_stride = f.n_pad * f.dp; q.split = f.split;
  q.rows = f.N; q.d = f.d; q.dp = (int)f.dp; q.pos = f.pos; q.hdr = f.hdr; q.unit = f.unit; q.cmax = f.cmax; q.gated = f.gated;
  q.out0 = f.dx;
  hipLaunchKernelGGL(parts_kernel<T>, dim3((unsigned)((f.N + 3) / 4)), dim3(kThreads), 0, s, q);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_hdr_clear(WideHdr* hdr, hipStream_t s) {
  hipLaunchKernelGGL(hdr_clear_kernel, dim3(1), dim3(kThreads), 0, s, hdr);
  return hipGetLastError();
}
hipError_t launch_rows_copy(const RowsCopies& c, hipStream_t s) {
  return c.dtype == 0 ? rows_copy<float>(c, s) : c.dtype == 1 ? rows_copy<bf16>(c, s) : rows_copy<f16>(c, s);
}
hipError_t launch_rows_max(const RowsCopies& c, hipStream_t s) {
  return c.dtype == 0 ? rows_max<float>(c, s) : c.dtype == 1 ? rows_max<bf16>(c, s) : rows_max<f16>(c, s);
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

// Gated feed-forward: h = act(x Wg^T) * (x Wu^T) in one kernel, and its gradients.
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
// A tile's A rows alternate between the two weights by 16, so that a lane holds a feature's g and u of the same token and
// the activation and the product happen in registers: h is written once, g and u never.  The backward pass forms g
// and u again (keeping them rounded would cost 4 N F bytes and a rounding), in pieces of the features (up to 1 GB of dg and
// du, fp32 1.5 GB, or 256 features, whichever is more), then takes the two products of msa_wide.hip.
// The products bound it: 32768 rows of 512 to 2048 features, bf16: forward 161 us (850 TFLOP/s, matrix units busy 40% of the
// cycles: an epilogue for each 16 stages), dg and du 237 (27%: dh's loads and two stores), products 284 (965, 48%).  16 rows:
// latency, 6 to 7 us of kernel.
#include "msa_wide.h"

namespace msa {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// act(g) and act'(g): silu g / (1 + e^-g); gelu g (1 + erf(g / sqrt 2)) / 2, with erfc(x) = (a1 t + ... + a5 t^5) e^-x^2,
// t = 1 / (1 + p x), x >= 0 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26: within 1.5e-7): no
// branches, e^-x^2 also makes the slope, and the lower tail is not a difference.  slope of both kinds is c + what
// multiplies g in c'.
template <int ACT>
__device__ inline void act_slope(float g, float& a, float& s) {
  if constexpr (ACT == 0) {
    const float c = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
    a = g * c;
    s = fmaf(c, g - a, c);
  } else {
    const float e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * g * g);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(g), 1.0f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float tail = 0.5f * e * (p * t);  // erfc(|g| / sqrt 2) / 2
    const float c = g < 0.0f ? tail : 1.0f - tail;
    a = g * c;
    s = fmaf(g * 0.3989422804014327f, e, c);
  }
}
template <int ACT>
__device__ inline float act_of(float g) {
  float a, s;
  act_slope<ACT>(g, a, s);
  return a;
}

struct GatedArgs {
  const char* x; int64_t x_ld, x_blk; int64_t N, n_pad;
  const char* w; int64_t w_ld, w_blk, up;  // the gate's first row of the piece; from there to the other weight's
  int cols;                         // features of the piece
  MmSegs segs[2];                   // of the narrow and the wide format
  int ksteps, tiles_f, tiles_n;
  const WideMode* mode;
  void* h; int64_t h_ld; int vec;   // forward
  const void* dh; int64_t dh_ld;    // backward: the piece's first column
  char* g; int64_t plane, half;
};

// Tl: 128 features of 128 tokens, 64 of 128 where that shares the work better (smaller_tiles), or forward 32 of 32 where that
// makes at most two tiles a CU.  us of a forward kernel, 32 of 32 / the better of the others, bf16: 16 rows of 512 to 2048 features
// 5.7 / 7.6, 64 5.8 / 7.7, 256 (512 tiles) 6.5 / 7.7; 64 rows of 2048 to 8192 (512) 18.1 / 21.4, of 4096 to 11008 (688) 42.4 / 39.7, 96
// rows of 512 to 8192 (768) 7.4 / 8.0, 128 (1024) 11.2 / 8.3.
template <typename E> using GatedTile = MmTile<E, 256, 128, 2, 2, false, false, true, 3>;
template <typename E> using GatedHalf = MmTile<E, 128, 128, 2, 2, false, false, true, 3>;
template <typename E> using GatedFew = MmTile<E, 64, 32, 2, 1, false, false, true, 8>;
constexpr int64_t kFewTiles = 2 * 256;

template <typename T, bool WIDE, int ACT, int TERMS, typename Tl>  // TERMS: of dg and du; 0: forward
__device__ inline void gated_tile(const GatedArgs& a, LdsChar* lds) {
  using E = typename Wide<T, WIDE>::E;
  constexpr int BF = Tl::TILE_M / 2, BN = Tl::TILE_N;
  int tf, tn;
  patch_order(xcd_order(blockIdx.x, gridDim.x), a.tiles_f, a.tiles_n, 8, tf, tn);
  const int64_t n0 = (int64_t)tn * BN;
  const int f0 = tf * BF;
  typename Tl::Acc acc;
  Tl::clear(acc);
  const int fleft = a.cols - f0 < BF ? a.cols - f0 : BF;
  const int rows = (int)(a.N - n0 < BN ? a.N - n0 : BN);
  const typename Tl::Side A{a.w + f0 * a.w_ld, fleft, a.w_ld, a.w_blk, 0, a.up};
  const typename Tl::Side B{a.x + n0 * a.x_ld, rows, a.x_ld, a.x_blk, 0, 0};
  Tl::run(acc, lds, A, B, a.segs[WIDE], 0, a.ksteps);
  float f1 = 1.0f, f2 = 1.0f;
  if constexpr (__is_same(T, float)) {
    f1 = 1.0f / scale_x<T>(a.mode);
    f2 = 1.0f / scale_w<T>(a.mode);
  }
  if constexpr (TERMS == 0) {
    T* out = (T*)a.h + n0 * a.h_ld + f0;
    Tl::store_dual(lds, out, a.h_ld, rows, fleft, a.vec != 0, [&](int i, int j, int q) {
      return quad<T>([&](int e) { return act_of<ACT>(acc[i][j][4 * q + e] * f1 * f2) * (acc[i][j][4 * q + e + 8] * f1 * f2); });
    });
  } else {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
    const float sg = scale_g<T>(a.mode, 1);
    // dh goes through LDS in whole rows, 32 tokens of each wave at a time; places outside are zeros, so that dg and du
    // are zeros there.
    constexpr int PER = 16 / (int)sizeof(T), CPR = BF / PER, ROW = BF * (int)sizeof(T) + 16, NQ = 2 * Tl::MB;
    static_assert(64 * ROW <= Tl::LDS, "the staged rows of dh fit the tile's LDS");
    typedef __attribute__((__vector_size__(16))) T TV;
    typedef __attribute__((address_space(3))) TV LdsTV;
    typedef typename Quad<T>::V T4;
    typedef __attribute__((address_space(3))) T4 LdsT4;
    const T* dh = (const T*)a.dh + n0 * a.dh_ld + f0;
#pragma unroll
    for (int j = 0; j < Tl::NB; ++j) {
#pragma unroll 4
      for (int c = (int)threadIdx.x; c < 64 * CPR; c += kThreads) {
        const int row = c / CPR, f = (c - row * CPR) * PER, n = (row >> 5) * 64 + 32 * j + (row & 31);
        TV v;
        if (a.vec && n < rows && f + PER <= fleft) {
          v = *reinterpret_cast<const TV*>(dh + n * a.dh_ld + f);
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e) v[e] = n < rows && f + e < fleft ? dh[n * a.dh_ld + f + e] : (T)0.0f;
        }
        *reinterpret_cast<LdsTV*>(lds + row * ROW + f * (int)sizeof(T)) = v;
      }
      Tl::sync_lds();
      // dg and du: two terms at most as they are made; three would be more registers than the values themselves
      constexpr bool SPLIT = TERMS < 3;
      typename Quad<E>::V grads[2][SPLIT ? TERMS : 1][NQ];  // [dg, du][term]
      f32x4 values[2][SPLIT ? 1 : NQ];
      const LdsChar* at = lds + (wn * 32 + (lane & 31)) * ROW + (wm * (BF / 2) + 4 * (lane >> 5)) * (int)sizeof(T);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const T4 d = *reinterpret_cast<const LdsT4*>(at + 8 * q * (int)sizeof(T));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = q >> 1, r = 4 * (q & 1) + e;  // features 16 i + 8 (q & 1) + ...: 8 q
          const float g = acc[i][j][r] * f1 * f2, u = acc[i][j][r + 8] * f1 * f2;
          float act, slope;
          act_slope<ACT>(g, act, slope);
          const float ds = (float)d[e] * sg;
          const float v[2] = {ds * u * slope, ds * act};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if constexpr (SPLIT) {
              const Terms<E, TERMS> t(v[half]);
#pragma unroll
              for (int k = 0; k < TERMS; ++k) grads[half][k][q][e] = t.t[k];
            } else {
              values[half][q][e] = v[half];
            }
          }
        }
      }
      Tl::sync_lds();
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
          Tl::template store_operand_tokens<Tl::MB / 2>(
              lds, reinterpret_cast<E*>(a.g + half * a.half + t * a.plane) + (f0 >> 5) * (a.n_pad * 32) + n0 * 32, a.n_pad * 32, j, [&](int i, int q) {
                if constexpr (SPLIT) return grads[half][t][4 * i + q];
                else return quad<E>([&](int e) { return (float)Terms<E, TERMS>(values[half][4 * i + q][e]).t[t]; });
              });
    }
  }
}

template <typename T, int ACT, int TERMS, template <typename> class Tile>
__global__ void __launch_bounds__(Tile<T>::THREADS, Tile<T>::TILE_M == 128 ? 3 : 2) gated_kernel(GatedArgs a) {
  __shared__ char smem[Tile<typename Wide<T>::E>::LDS];  // the sizes are the same in both formats
  by_format<T>(a.mode, [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value;
    gated_tile<T, WIDE, ACT, (WIDE && TERMS > 0 ? 3 : TERMS), Tile<typename Wide<T, WIDE>::E>>(a, (LdsChar*)smem);
  });
}

__global__ void zero_kernel(uint16_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) p[i] = 0;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
int64_t es_of(int dtype) { return dtype == 0 ? 4 : 2; }
bool direct(const GatedCall& c, const void* p, int64_t ld) {
  return c.dtype != 0 && c.d % 32 == 0 && ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld * 2 * 256 < ((int64_t)1 << 32);
}

struct GatedPlan {
  int64_t n_pad, dp, x_plane, w_plane, C, g_plane;
  int planes, g_terms;
  WideShare share;
  char *x, *w, *g;
  float *dx_part, *dw_part;
  WideMode* mode;
  WidePart* parts;
  size_t bytes;
  GatedPlan(const GatedCall& c, int backward) {
    planes = planes_of(c.dtype);
    g_terms = terms_of_g(c.dtype, c.N);
    n_pad = round_up(c.N > 0 ? c.N : 1, 128);
    dp = wide_dp(c.d);
    x_plane = round_up(n_pad * dp * 2, 256);
    w_plane = round_up((int64_t)c.F * dp * 2, 256);
    char* p = (char*)c.workspace;
    size_t o = 0;
    auto take = [&](int64_t bytes) { char* q = p + o; o += (size_t)round_up(bytes, 256); return q; };
    const bool scales = c.dtype == 0 || (backward && c.dtype == 2);  // bf16 has none
    mode = scales ? (WideMode*)take(sizeof(WideMode)) : nullptr;
    parts = scales ? (WidePart*)take(kPartBytes) : nullptr;
    x = direct(c, c.x, c.x_ld) ? nullptr : take(planes * x_plane);
    w = direct(c, c.w[0], c.w_ld[0]) && direct(c, c.w[1], c.w_ld[1]) && c.w_ld[0] == c.w_ld[1] ? nullptr : take(2 * planes * w_plane);
    C = g_plane = 0;
    share = WideShare{};
    g = nullptr; dx_part = dw_part = nullptr;
    if (backward) {
      C = wide_piece(c.N, c.d, c.F, 2, c.dtype == 0 ? 3 : g_terms, c.dx != nullptr, c.dw[0] != nullptr, 2 * g_terms * 2 * n_pad, &share);
      g_plane = round_up(n_pad * C * 2, 256);
      g = take(2 * g_planes(c.dtype, c.N) * g_plane);
      if (c.dx != nullptr) dx_part = (float*)take((int64_t)share.dx_split * n_pad * dp * 4);
      if (c.dw[0] != nullptr && share.dw_split > 1) dw_part = (float*)take((int64_t)share.dw_split * 2 * C * dp * 4);
    }
    bytes = o;
  }
};

#define GATED_TRY(call) do { const hipError_t e_ = (call); if (e_ != hipSuccess) return e_; } while (0)

struct GatedOperands { const char *x, *w[2]; int64_t x_ld, x_blk, w_ld, w_blk; int x_rows; MmSegs segs[2]; };

hipError_t operands(const GatedCall& c, const GatedPlan& p, int backward, GatedOperands* o) {
  RowsCopies all = {}, copies = {};
  all.dtype = copies.dtype = c.dtype;
  all.mode = copies.mode = p.mode;
  all.add(RowsCopy{c.x, c.x_ld, c.N, c.d, p.x, p.x_plane, p.n_pad * 64, nullptr, 0, backward});
  for (int i = 0; i < 2; ++i)
    all.add(RowsCopy{c.w[i], c.w_ld[i], c.F, c.d, p.w + (p.w == nullptr ? 0 : i * p.planes * p.w_plane), p.w_plane, c.F * (int64_t)64, nullptr, 1, backward});
  if (p.x != nullptr) copies.add(all.m[0]);
  if (p.w != nullptr) { copies.add(all.m[1]); copies.add(all.m[2]); }
  if (p.mode != nullptr) {  // scales of the operands, and of dg and du
    if (backward) all.add(RowsCopy{c.dh, c.dh_ld, c.N, c.F, nullptr, 0, 0, nullptr, 2, 0});
    GATED_TRY(launch_wide_mode(all, p.parts, p.mode, 1, c.stream));
  }
  if (copies.n > 0) GATED_TRY(launch_rows_copy(copies, c.stream));
  o->x = p.x != nullptr ? p.x : (const char*)c.x;
  o->x_ld = p.x != nullptr ? 64 : c.x_ld * 2;
  o->x_blk = p.x != nullptr ? p.n_pad * 64 : 64;
  o->x_rows = (int)c.N;
  o->w[0] = p.w != nullptr ? p.w : (const char*)c.w[0];
  o->w[1] = p.w != nullptr ? p.w + p.planes * p.w_plane : (const char*)c.w[1];
  o->w_ld = p.w != nullptr ? 64 : c.w_ld[0] * 2;
  o->w_blk = p.w != nullptr ? c.F * (int64_t)64 : 64;
  o->segs[0] = o->segs[1] = MmSegs{};
  o->segs[0].n = 1;
  if (p.planes > 1) {
    o->segs[0].b[0] = p.x_plane;
    o->segs[0].a[1] = p.w_plane;
    o->segs[0].n = 3;
    o->segs[0].low = 2;
    for (int order = 2; order >= 0; --order) add_wide_segs(o->segs[1], order, 0, p.w_plane, 0, p.x_plane);
  }
  return hipSuccess;
}

GatedArgs args_of(const GatedCall& c, const GatedPlan& p, const GatedOperands& o, int64_t f0, int cols) {
  GatedArgs a = {};
  a.x = o.x; a.x_ld = o.x_ld; a.x_blk = o.x_blk; a.N = c.N; a.n_pad = p.n_pad;
  a.w = o.w[0] + f0 * o.w_ld; a.w_ld = o.w_ld; a.w_blk = o.w_blk; a.up = o.w[1] - o.w[0]; a.cols = cols;
  for (int i = 0; i < 2; ++i) a.segs[i] = o.segs[i];
  a.ksteps = (int)(p.dp / 32);
  a.mode = p.mode;
  return a;
}

template <typename T, int TERMS, template <typename> class Tile>
hipError_t launch_tiles(GatedArgs a, int act, hipStream_t s) {
  using Tl = Tile<typename Wide<T>::E>;
  a.tiles_f = (a.cols + Tl::TILE_M / 2 - 1) / (Tl::TILE_M / 2);
  a.tiles_n = (int)((a.N + Tl::TILE_N - 1) / Tl::TILE_N);
  auto* k = act == 0 ? gated_kernel<T, 0, TERMS, Tile> : gated_kernel<T, 1, TERMS, Tile>;
  hipLaunchKernelGGL(k, dim3((unsigned)((int64_t)a.tiles_f * a.tiles_n)), dim3(Tl::THREADS), 0, s, a);
  return hipGetLastError();
}

template <typename T, int TERMS>
hipError_t launch(const GatedArgs& a, int act, hipStream_t s) {
  if (TERMS == 0 && (a.cols + 31) / 32 * ((a.N + 31) / 32) <= kFewTiles) return launch_tiles<T, 0, GatedFew>(a, act, s);
  const int64_t tiles_n = (a.N + 127) / 128;
  return smaller_tiles((a.cols + 127) / 128, tiles_n, (a.cols + 63) / 64) ? launch_tiles<T, TERMS, GatedHalf>(a, act, s)
                                                                        : launch_tiles<T, TERMS, GatedTile>(a, act, s);
}

template <typename T>
hipError_t gated_fwd(const GatedCall& c) {
  if (c.N == 0) return hipSuccess;
  const GatedPlan p(c, 0);
  GatedOperands o;
  GATED_TRY(operands(c, p, 0, &o));
  GatedArgs a = args_of(c, p, o, 0, c.F);
  a.h = c.h; a.h_ld = c.F;
  a.vec = (int64_t)c.F * sizeof(T) % 16 == 0 && ((uintptr_t)c.h & 15) == 0;
  return launch<T, 0>(a, c.act, c.stream);
}

template <typename T>
hipError_t gated_bwd(const GatedCall& c) {
  if (c.N == 0) {
    for (int i = 0; i < 2; ++i)
      if (c.dw[i] != nullptr) {
        hipLaunchKernelGGL(zero_kernel, dim3(1024), dim3(kThreads), 0, c.stream, (uint16_t*)c.dw[i], (int64_t)c.F * c.d * es_of(c.dtype) / 2);
        GATED_TRY(hipGetLastError());
      }
    return hipSuccess;
  }
  const GatedPlan p(c, 1);
  GatedOperands o;
  GATED_TRY(operands(c, p, 1, &o));
  for (int64_t f0 = 0; f0 < c.F; f0 += p.C) {
    const int cols = (int)(c.F - f0 < p.C ? c.F - f0 : p.C);
    GatedArgs a = args_of(c, p, o, f0, cols);
    a.dh = (const T*)c.dh + f0; a.dh_ld = c.dh_ld;
    a.vec = c.dh_ld * sizeof(T) % 16 == 0 && ((uintptr_t)c.dh & 15) == 0;
    a.g = p.g; a.plane = p.g_plane; a.half = g_planes(c.dtype, c.N) * p.g_plane;
    GATED_TRY((p.g_terms == 2 ? launch<T, 2>(a, c.act, c.stream) : launch<T, __is_same(T, float) ? 2 : 1>(a, c.act, c.stream)));
    WideProducts q = {};
    q.dtype = c.dtype; q.gated = 1; q.N = c.N; q.n_pad = p.n_pad; q.d = c.d; q.dp = p.dp; q.halves = 2; q.cols = cols; q.C = p.C;
    q.x = o.x; q.x_ld = o.x_ld; q.x_blk = o.x_blk; q.x_plane = p.x_plane; q.x_rows = o.x_rows;
    for (int i = 0; i < 2; ++i) {
      q.w[i] = o.w[i] + f0 * o.w_ld;
      q.dw[i] = c.dw[i] == nullptr ? nullptr : (char*)c.dw[i] + f0 * c.d * es_of(c.dtype);
    }
    q.w_ld = o.w_ld; q.w_blk = o.w_blk; q.w_plane = p.w_plane; q.w_rows = (int)(c.F - f0);
    q.g = p.g; q.g_plane = p.g_plane; q.g_half = g_planes(c.dtype, c.N) * p.g_plane; q.g_terms = p.g_terms;
    q.dx_part = p.dx_part; q.dx_add = f0 > 0; q.dw_part = p.dw_part;
    q.share = p.share; q.mode = p.mode; q.unit.mode = 3; q.use_live = 0;
    GATED_TRY(launch_wide_products(q, c.stream));
  }
  if (c.dx != nullptr) {
    const WideFinish f{c.dtype, 1, c.N, p.n_pad, c.d, p.dp, p.share.dx_split, p.dx_part, nullptr, p.mode, GradUnit{nullptr, 1.0f, 3}, nullptr, c.dx};
    GATED_TRY(launch_wide_finish(f, c.stream));
  }
  return hipSuccess;
}

}  // namespace

size_t gated_workspace_bytes(const GatedCall& c, int backward) { return GatedPlan(c, backward).bytes; }

hipError_t launch_gated_fwd(const GatedCall& c) {
  return c.dtype == 0 ? gated_fwd<float>(c) : c.dtype == 1 ? gated_fwd<bf16>(c) : gated_fwd<f16>(c);
}
hipError_t launch_gated_bwd(const GatedCall& c) {
  return c.dtype == 0 ? gated_bwd<float>(c) : c.dtype == 1 ? gated_bwd<bf16>(c) : gated_bwd<f16>(c);
}

}  // namespace msa

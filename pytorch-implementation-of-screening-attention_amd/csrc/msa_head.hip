// Losses of rows against a vocabulary without its logits: softmax cross entropy and the divergence from a teacher's
// largest logits.  With z2_nv = log2(e) x_n . W_v / T and lse2_n = log2 sum_v 2^z2_nv:
//   cross entropy  L_n = ln2 (lse2_n - z2_n,y)
//   distillation   L_n = T^2 (sum_k p_k ln p_k - ln2 sum_k p_k (z2_n,id(k) - lse2_n)),  p = softmax of the row's entries
//   both           dL_n/dz_nv = T (2^(z2_nv - lse2_n) - sum_{k: id(k) = v} p_k)        (z: logits before 1/T)
// Forward: one product over all of the vocabulary whose tiles leave each row's maximum and sum; a row's own logits are
// K dot products in the same order.  Backward, in pieces of the vocabulary: the product again, now with lse2 known, gives the piece's
// gradient G in the operand type (up to 1 GB, fp32 1.5 GB, or 256 columns, whichever is more); then dx += G W and dW = G^T x (msa_wide.hip).
// Rows that do not count are taken out before the products, but for a few rows' scores, which leave them unused
// (x_direct): their x may hold anything.
// The products bound it: 8192 rows of 512 by 50257 bf16, a training pass 1800 us = logits 400 to 480 (870 to 1020 TFLOP/s),
// G 580 to 600 (its 823 MB store beside the product), both products 970 to 1030 (820 to 870), all else 75.  Their matrix units are
// busy 53, 41 and 49% of the cycles, at 1.7 to 2.0 GHz that the card's power allows; the rest are waits for copies and at
// the barrier of every 32 k, and G's store.
#include "msa_wide.h"

#include <float.h>

namespace msa {
namespace {

constexpr int kThreads = 256;
constexpr int kHeadMaxK = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What the backward pass needs: mode, pos[N] (row of the operand, -1: does not count), lse[N rows of the operand]: the
// largest of x_n . W_v, and log2 of the sum of 2^z2 over its own; t[N][K]: 2^(z2 - lse2) - p of the targets (p summed over
// equal ids).
struct HeadState {
  WideMode* mode;
  int* pos;
  float2* lse;
  float* t;
  size_t bytes;
  HeadState(void* p, int64_t N, int K) {
    char* c = (char*)p;
    size_t o = (size_t)round_up(sizeof(WideMode), 256);
    mode = (WideMode*)c;
    pos = (int*)(c + o); o += (size_t)round_up(N * 4, 256);
    lse = (float2*)(c + o); o += (size_t)round_up(round_up(N, 128) * 8, 256);
    t = (float*)(c + o); o += (size_t)round_up(N * K * 4, 256);
    bytes = o;
  }
};

// ---------------------------------------------------------------------------
// Which rows count
// ---------------------------------------------------------------------------
// One block: pos[n] = how many rows before n count, or -1.  A wave takes up to 64 groups of 64 neighbouring rows at a time
// and lane i keeps which of group i count; 65536 rows are one round.  32768 rows: 42 us with a thread to 32 neighbours, 26
// with reads of whole lines.
template <typename Fn>
__device__ inline int number_rows(int64_t N, int* pos, Fn counts) {
  __shared__ int sums[16];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (int)(N >= 65536 ? 64 : (N + 1023) / 1024);
  int total = 0;
  for (int64_t base = 0; base < N; base += (int64_t)per * 1024) {
    const int64_t from = base + (int64_t)wave * per * 64 + lane;
    unsigned long long bits = 0;
#pragma unroll 8
    for (int i = 0; i < per; ++i) {
      const int64_t n = from + i * 64;
      const bool is = counts(n < N ? n : N - 1) && n < N;
      const unsigned long long b = __ballot(is);
      bits = lane == i ? b : bits;
    }
    const int c = __popcll(bits);
    int incl = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int at = total + incl - c;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) at += sums[w];
      total += sums[w];
    }
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll 8
    for (int i = 0; i < per; ++i) {
      const int64_t n = from + i * 64;
      const unsigned long long b = __shfl(bits, i);
      const int first = __shfl(at, i);
      if (n < N) pos[n] = (b >> lane) & 1 ? first + __popcll(b & below) : -1;
    }
  }
  return total;
}

__global__ void __launch_bounds__(1024) plan_kernel(const int64_t* ids, int64_t ids_ld, int64_t ignore,
                                                    const uint8_t* live, int64_t N, int* pos, WideMode* mode) {
  const int total = live != nullptr ? number_rows(N, pos, [&](int64_t n) { return live[n] != 0; })
                                    : number_rows(N, pos, [&](int64_t n) { return ids[n * ids_ld] != ignore; });
  if (threadIdx.x == 0) *mode = WideMode{total, 0, 1.0f, 1.0f, 1.0f};
}

// A teacher's record of a row: entries with an id >= 0 and a logit above -inf; p = their softmax at 1/T.  A wave per
// row.  tp[n][k] = (p, p summed over the row's entries of the same id), p = -1: no entry; ent[n] = sum p ln p.
// NaN logits, or +inf, give NaN.
template <typename L>
__global__ void __launch_bounds__(kThreads) teacher_kernel(const L* logits, int64_t lld, const int64_t* ids,
                                                           int64_t ids_ld, int64_t N, int K, float inv_t, float2* tp,
                                                           float* ent, uint8_t* live) {
  constexpr int R = kHeadMaxK / 64;
  __shared__ int64_t sid[4][kHeadMaxK];
  __shared__ float sp[4][kHeadMaxK];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * 4 + wave;
  if (n < N) {
    float t[R];
    int64_t id[R];
    float mx = -INFINITY;
    bool any = false;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int k = q * 64 + lane;
      id[q] = k < K ? ids[n * ids_ld + k] : -1;
      const float raw = id[q] >= 0 ? to_f(logits[n * lld + k]) : -INFINITY;
      t[q] = fabsf(raw) < INFINITY ? fminf(fmaxf(raw * inv_t, -FLT_MAX), FLT_MAX) : raw;  // a finite logit stays an entry
      any = any || !(t[q] == -INFINITY);
      mx = fmaxf(mx, t[q]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    any = __ballot(any) != 0ull;
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < R; ++q) sum += t[q] == -INFINITY ? 0.0f : exp2f((t[q] - mx) * kLog2e);
    sum = wave_sum(sum);
    const float ls = logf(sum);
    float h = 0.0f;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int k = q * 64 + lane;
      const float lp = t[q] - mx - ls, p = t[q] == -INFINITY ? 0.0f : expf(lp);
      h += p > 0.0f ? p * lp : p;  // 0 ln 0 = 0; NaN stays
      t[q] = t[q] == -INFINITY ? -1.0f : p;
      sid[wave][k] = id[q];
      sp[wave][k] = p;
    }
    h = wave_sum(h);
    wave_lds_sync();
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int k = q * 64 + lane;
      if (q * 64 >= K) break;
      float all = 0.0f;
      for (int o = 0; o < K; ++o) all += sid[wave][o] == id[q] ? sp[wave][o] : 0.0f;
      if (k < K) tp[n * K + k] = float2{t[q], all};
    }
    if (lane == 0) {
      ent[n] = h;
      live[n] = any ? 1 : 0;
    }
  }
}

// ---------------------------------------------------------------------------
// The product's maxima and sums
// ---------------------------------------------------------------------------
struct StatsArgs {
  const char* x; int64_t x_ld, x_blk; int64_t rows;  // readable rows
  const char* w; int64_t w_ld, w_blk; int64_t V;
  MmSegs segs[2];                   // of the narrow and the wide format
  int ksteps, tiles_v, tiles_n;
  float to_log2;  // log2(e) / T
  const WideMode* mode;             // null: the rows as they are
  float2* part; int64_t part_ld;  // [tiles_v][part_ld]
};

// Logits as the product leaves them, a, times f > 0 are z2.  Statistics keep a row's largest a itself and a sum over
// 2^(f (a - max)), and G takes a - max too, so that the largest one's term is 1 whatever its size.  One fma with f max rounded
// would be off by up to half a step of it: 2^(1/32) at z2 = 2^20, past any number at 2^31.  It would save 5 us of
// 1780 (ce_train_8k_bf16: stats 4, G 1).

// Features from `left` on become v: only the last tile along the vocabulary pays for the comparisons.
template <typename Tl>
__device__ inline void mask_features(typename Tl::Acc& acc, int left, int wm, int lane, float v) {
#pragma unroll
  for (int i = 0; i < Tl::MB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool out = Tl::m_of(wm, lane, i, r >> 2) + (r & 3) >= left;
#pragma unroll
      for (int j = 0; j < Tl::NB; ++j) acc[i][j][r] = out ? v : acc[i][j][r];
    }
}

// 256 tokens of the vocabulary by 128 rows, or 64 by 32 for up to 32 rows, whose time is the weight's stream: small tiles in all
// CUs with seven stages ahead.  Only up to three of them a CU, which LDS holds at once: a fourth comes late, and large tiles
// leave fewer partial sums.  us of 16 scores, small / large, bf16, d = 512: V 8003 12.3 / 17.7, 24000 13.1 / 17.9, 40000 17.8 / 20.3,
// 50257 22.3 / 21.1, 100000 30.0 / 29.0; d = 1024: 40000 25.5 / 29.2, 50257 33.3 / 30.0; fp32, d = 512: 40000 85.0 / 88.7, 50257 105.1 / 98.7.
template <typename E> using HeadTile = MmTile<E, 256, 128, 2, 2, false, false, false, 3>;
template <typename E> using HeadFew = MmTile<E, 64, 32, 2, 1, false, false, false, 8>;
constexpr int kFew = 32, kFewTiles = 3 * 256;

template <typename T, bool WIDE, typename Tl>
__device__ inline void stats_tile(const StatsArgs& a, LdsChar* lds, float2 (*red)[Tl::TILE_N]) {
  constexpr int BM = Tl::TILE_M, BN = Tl::TILE_N, WM = Tl::WAVES_M;
  int tv, tn;
  patch_order(xcd_order(blockIdx.x, gridDim.x), a.tiles_v, a.tiles_n, 8, tv, tn);
  const int64_t v0 = (int64_t)tv * BM, n0 = (int64_t)tn * BN;
  const int64_t rows = a.mode != nullptr ? a.mode->live : a.rows;
  if (n0 >= rows) return;
  typename Tl::Acc acc;
  Tl::clear(acc);
  const int vleft = (int)(a.V - v0 < BM ? a.V - v0 : BM);
  const int readable = (int)(a.rows - n0 < BN ? a.rows - n0 : BN);
  const typename Tl::Side A{a.w + v0 * a.w_ld, vleft, a.w_ld, a.w_blk, 0, 0};
  const typename Tl::Side B{a.x + n0 * a.x_ld, readable, a.x_ld, a.x_blk, 0, 0};
  Tl::run(acc, lds, A, B, a.segs[WIDE], 0, a.ksteps);
  float f = a.to_log2;
  if constexpr (__is_same(T, float)) f = f / scale_x<T>(a.mode) / scale_w<T>(a.mode);
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, wm = wave % WM, wn = wave / WM;
  if (vleft < BM) mask_features<Tl>(acc, vleft, wm, lane, -INFINITY);
#pragma unroll
  for (int j = 0; j < Tl::NB; ++j) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < Tl::MB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[i][j][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float top = mx == -INFINITY ? 0.0f : mx;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < Tl::MB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f((acc[i][j][r] - top) * f);
    s += __shfl_xor(s, 32);
    if (lane < 32) red[wm][Tl::n_of(wn, lane, j)] = float2{mx, s};
  }
  __syncthreads();
  if ((int)threadIdx.x < BN && (int)threadIdx.x < readable) {
    const float2 p = red[0][threadIdx.x], q = red[1][threadIdx.x];
    static_assert(WM == 2, "two waves share a row's features");
    const float m = fmaxf(p.x, q.x), at = m == -INFINITY ? 0.0f : m;
    a.part[(int64_t)tv * a.part_ld + n0 + threadIdx.x] =
        float2{m, p.y * __builtin_amdgcn_exp2f((p.x - at) * f) + q.y * __builtin_amdgcn_exp2f((q.x - at) * f)};
  }
}

template <typename T, template <typename> class Tile>
__global__ void __launch_bounds__(Tile<T>::THREADS, 2) stats_kernel(StatsArgs a) {
  using Any = Tile<typename Wide<T>::E>;  // the sizes are the same in both formats
  __shared__ char smem[Any::LDS];
  __shared__ float2 red[Any::WAVES_M][Any::TILE_N];
  by_format<T>(a.mode, [&](auto wide) {
    stats_tile<T, decltype(wide)::value, Tile<typename Wide<T, decltype(wide)::value>::E>>(a, (LdsChar*)smem, red);
  });
}

// ---------------------------------------------------------------------------
// A row's targets' logits, its sum over the tiles and its loss.  A block takes up to 8 rows: its waves form 32 targets'
// logits at a time, its threads share the tiles, then each thread has a target.  Few rows are spread over more blocks.
//
// Logits are formed as the product formed them, by the same MFMA in the same order, so that a target's is bitwise the one in
// its row's sum: away = lse2 - z2 is then log2 of a sum that has 1 in it, and neither that nor 1 - q hides behind the logits'
// own rounding.  (By another order they are off by 1e-5 at logits of 120: losses below that come out negative and their
// gradients of either sign.)  32 targets and their rows are A and B; of the 32 x 32 results the diagonal counts.
// Bound by the latency of what it gathers: 8192 rows of 64 targets at d = 256 (537 MB) 61 us, 8192 rows of one at 512 21 us.  A
// lone pair is one wave's, 8 steps in flight instead of 4 (16 scores: a call 23.1 -> 22.4 us with the tiles' loads ahead of it);
// with more pairs a CU holds one block of those instead of three (8192 rows 35 us).
// ---------------------------------------------------------------------------
constexpr int kRows = 8;  // of a block, at most
struct RowsArgs {
  const char* x; int64_t x_ld, x_blk;  // operands, as in StatsArgs
  const char* w; int64_t w_ld, w_blk;
  MmSegs segs[2];
  int ksteps;
  const int64_t* ids; int64_t ids_ld;
  const float2* tp;  // null: cross entropy
  const float* ent;
  const float2* part; int64_t part_ld; int tiles;
  int64_t N, V, ignore; int K, rows;
  float temperature;
  const int* pos;  // null: every row whose id is not `ignore`, in its own place
  const WideMode* mode;
  float2* lse; float* t; float* loss;  // lse, t: null where no gradient follows
};

// The products of 32 pairs of rows, U steps of 32 k in flight, a lane holding its pair's (that of lane & 31, in one of the two lanes).
template <typename E, int U>
__device__ inline float pair_products(const char* a, const char* b, int64_t a_blk, int64_t b_blk, const MmSegs& segs, int steps) {
  using M = Mma<E>;
  const int n = (int)threadIdx.x & 31, half = ((int)threadIdx.x >> 5) & 1;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (int seg = 0; seg < segs.n; ++seg) {
    if (segs.low != 0 && seg == segs.low) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] *= kLowTerm;
    }
    const char* pa = a + segs.a[seg] + half * 16;
    const char* pb = b + segs.b[seg] + half * 16;
    for (int s = 0; s < steps; s += U) {
      typename M::frag fa[2 * U], fb[2 * U];
#pragma unroll
      for (int u = 0; u < 2 * U; ++u) {
        if (s + u / 2 < steps) {
          fa[u] = M::load(reinterpret_cast<const E*>(pa + (u / 2) * a_blk + (u & 1) * 32));
          fb[u] = M::load(reinterpret_cast<const E*>(pb + (u / 2) * b_blk + (u & 1) * 32));
        } else {
          fa[u] = fb[u] = M::zero();
        }
      }
#pragma unroll
      for (int u = 0; u < 2 * U; ++u) acc = M::mma_ng(fa[u], fb[u], acc);
      guard_run(fa, acc);
      guard_keep(fb);
      pa += U * a_blk;
      pb += U * b_blk;
    }
  }
  float z = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) z = 8 * (r >> 2) + 4 * half + (r & 3) == n ? acc[r] : z;
  return z;
}

template <typename T, int U>
__global__ void __launch_bounds__(kThreads) rows_kernel(RowsArgs a) {
  __shared__ float2 red[kThreads];
  __shared__ float2 stat[kRows];  // the row's largest logit and log2 of its sum
  __shared__ int place[kRows];    // the row's place in the operand, -1: it does not count
  __shared__ float terms[kRows][kHeadMaxK];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int64_t first = (int64_t)blockIdx.x * a.rows;
  const float to_log2 = kLog2e / a.temperature;
  float f = to_log2, unscale = 1.0f;  // of the product's own numbers, and to x . W
  if constexpr (__is_same(T, float)) {
    f = f / scale_x<T>(a.mode) / scale_w<T>(a.mode);
    unscale = 1.0f / scale_x<T>(a.mode) / scale_w<T>(a.mode);
  }
  if (tid < kRows) {
    int at = -1;
    if (tid < a.rows && first + tid < a.N)
      at = a.pos != nullptr ? a.pos[first + tid] : a.ids[(first + tid) * a.ids_ld] == a.ignore ? -1 : (int)(first + tid);
    place[tid] = at;
  }
  __syncthreads();
  const int r_of = tid & (a.rows - 1), g = tid / a.rows, groups = kThreads / a.rows;  // rows is a power of two
  const int at_of = place[r_of];
  float2 p[4];
  auto load = [&](int t) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      p[q] = at_of >= 0 && t + groups * q < a.tiles ? a.part[(int64_t)(t + groups * q) * a.part_ld + at_of] : float2{-INFINITY, 0.0f};
  };
  load(g);  // all there are where rows are few, on their way beside the targets'
  by_format<T>(a.mode, [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value;
    for (int e0 = (3 - (tid >> 6)) * 32; e0 < a.rows * a.K; e0 += 128) {
      const int e = e0 + (lane & 31), r = e / a.K, k = e - r * a.K;
      int at = 0;
      int64_t id = 0;
      bool is = false;
      if (e < a.rows * a.K && place[r] >= 0) {
        const int64_t v = a.ids[(first + r) * a.ids_ld + k];
        is = v >= 0 && v < a.V;
        if (is) { id = v; at = place[r]; }
      }
      if (__ballot(is) == 0ull) continue;  // a pair that is none takes rows that are there
      const float z = pair_products<typename Wide<T, WIDE>::E, U>(a.w + id * a.w_ld, a.x + (int64_t)at * a.x_ld, a.w_blk, a.x_blk, a.segs[WIDE], a.ksteps);
      if (is && (lane >> 5) == ((lane >> 2) & 1)) terms[r][k] = z;
    }
  });
  {
    float m = -INFINITY, s = 0.0f;
    auto add = [&](float2 p) {
      const float mn = fmaxf(m, p.x), b = mn == -INFINITY ? 0.0f : mn;
      s = s * __builtin_amdgcn_exp2f((m - b) * f) + p.y * __builtin_amdgcn_exp2f((p.x - b) * f);
      m = mn;
    };
    for (int t = g; t < a.tiles; t += groups * 4) {
      if (t > g) load(t);
#pragma unroll
      for (int q = 0; q < 4; ++q) add(p[q]);
    }
    red[tid] = float2{m, s};
    __syncthreads();
    for (int o = kThreads / 2; o >= a.rows; o >>= 1) {
      if (tid < o) {
        add(red[tid + o]);
        red[tid] = float2{m, s};
      }
      __syncthreads();
    }
    if (tid < a.rows) stat[tid] = float2{m, log2f(s)};
    __syncthreads();
  }
  for (int e = tid; e < a.rows * a.K; e += kThreads) {
    const int r = e / a.K, k = e - r * a.K;
    if (place[r] < 0) continue;
    const int64_t n = first + r, id = a.ids[n * a.ids_ld + k];
    const float2 p = a.tp == nullptr ? float2{1.0f, 1.0f} : a.tp[n * a.K + k];
    float t = 0.0f, term = 0.0f;
    if (id >= 0 && id < a.V) {
      float away = fmaf(stat[r].x - terms[r][k], f, stat[r].y);  // lse2 - z2
      away = away < 0.0f ? 0.0f : away;  // a rounding of the sum; NaN stays
      t = __builtin_amdgcn_exp2f(-away) - p.y;
      term = p.x > 0.0f || !(p.x == p.x) ? p.x * away : 0.0f;
    } else if (a.tp == nullptr || (id >= 0 && !(p.x < 0.0f))) {
      t = term = NAN;  // an entry outside the vocabulary
    }
    terms[r][k] = term;
    if (a.t != nullptr) a.t[n * a.K + k] = t;
  }
  __syncthreads();
  {
    const int r = tid >> 5, l = tid & 31;
    const int64_t n = first + r;
    if (r < a.rows && n < a.N) {
      const int at = place[r];
      float away = 0.0f;
      if (at >= 0)
        for (int k = l; k < a.K; k += 32) away += terms[r][k];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) away += __shfl_xor(away, o);
      if (l == 0) {
        float loss = kLn2 * away;
        if (a.tp != nullptr && at >= 0) loss = a.temperature * a.temperature * (loss + a.ent[n]);
        a.loss[n] = at >= 0 ? loss : 0.0f;
        // a target outside the vocabulary makes the row NaN, its gradient too
        if (at >= 0 && a.lse != nullptr) a.lse[at] = float2{stat[r].x * unscale, away == away ? stat[r].y : NAN};
      }
    }
  }
}

// One block: the mean or the sum of the rows' losses, in 64 bits.  (The last block of rows_kernel could do it; but making
// each block's rows visible to it writes back its L2: 160 -> 390 us for 8192 rows of 64 targets.)
__global__ void __launch_bounds__(1024) total_kernel(const float* rows, int64_t N, const WideMode* mode, int mean, float* out) {
  __shared__ double sums[16];
  double s = 0.0;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < N; n += 1024) s += (double)rows[n];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += sums[w];
    out[0] = (float)(mean ? s / (double)mode->live : s);
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// Coefficients of the rows of the operand where each row's loss has a gradient of its own, as g_n / cmax with a power of
// two cmax, at least the largest finite |g_n|; zero behind the last row up to the next multiple of 128.  One block.  (A mean
// or a sum has one coefficient for all: G is formed for 1 and so rounded from the probabilities themselves.)  fp32: rows of G
// are as uneven as the coefficients, and past 2^kEvenCoef the pass takes the wide format, whichever the forward pass took.
constexpr int kEvenCoef = 20;
__global__ void __launch_bounds__(1024) coef_kernel(const float* dloss, float factor, int64_t N, int64_t n_pad, const int* pos,
                                                    const WideMode* fwd, WideMode* mode, float* cmax, float* coef) {
  const int tid = (int)threadIdx.x;
  const int live = fwd->live;
  __shared__ float red[16], least[16];
  float mx = 0.0f, mn = INFINITY;
  for (int64_t n = tid; n < N; n += 1024) {
    const float g = pos[n] >= 0 ? fabsf(dloss[n] * factor) : 0.0f;
    if (g < INFINITY) mx = fmaxf(mx, g);
    if (g > 0.0f) mn = fminf(mn, g);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, o));
    mn = fminf(mn, __shfl_xor(mn, o));
  }
  if ((tid & 63) == 0) { red[tid >> 6] = mx; least[tid >> 6] = mn; }
  __syncthreads();
  for (int w = 0; w < 16; ++w) {
    mx = fmaxf(mx, red[w]);
    mn = fminf(mn, least[w]);
  }
  const float inv = pow2_to(mx, 0);  // mx inv in [0.5, 1)
  if (tid == 0) {
    *cmax = 1.0f / inv;
    const bool wide = fwd->wide || mn < mx * (1.0f / (1 << kEvenCoef));
    *mode = WideMode{live, wide ? 1 : 0, wide ? 1.0f : fwd->sx, wide ? 1.0f : fwd->sw, wide ? 1.0f : fwd->sg};
  }
  for (int64_t n = tid; n < N; n += 1024)
    if (pos[n] >= 0) coef[pos[n]] = dloss[n] * factor * inv;
  for (int64_t i = live + tid; i < n_pad; i += 1024) coef[i] = 0.0f;
}

struct GradArgs {
  const char* x; int64_t n_pad;
  const char* w; int64_t w_ld, w_blk;  // the piece's first row
  int cols;                     // its rows
  MmSegs segs[2];               // of the narrow and the wide format
  int ksteps, tiles_v, tiles_n;
  float to_log2;
  const WideMode* mode;
  const float2* lse; const float* coef;
  char* g; int64_t plane;
};

// G of one tile: c_n 2^(z2 - lse2), without the targets, which scatter_kernel puts in their place.
template <typename T, bool WIDE, int TERMS>
__device__ inline void grad_tile(const GradArgs& a, LdsChar* lds) {
  using E = typename Wide<T, WIDE>::E;
  using Tl = HeadTile<E>;
  int tv, tn;
  patch_order(xcd_order(blockIdx.x, gridDim.x), a.tiles_v, a.tiles_n, 8, tv, tn);
  const int64_t v0 = (int64_t)tv * 256, n0 = (int64_t)tn * 128;
  const int64_t live = a.mode->live;
  if (n0 >= live) return;
  typename Tl::Acc acc;
  Tl::clear(acc);
  const int vleft = (int)(a.cols - v0 < 256 ? a.cols - v0 : 256);
  const int64_t blk = a.n_pad * 32;
  E* out = reinterpret_cast<E*>(a.g) + (v0 >> 5) * blk + n0 * 32;
  const typename Tl::Side A{a.w + v0 * a.w_ld, vleft, a.w_ld, a.w_blk, 0, 0};
  const typename Tl::Side B{a.x + n0 * 64, (int)(a.n_pad - n0 < 128 ? a.n_pad - n0 : 128), 64, a.n_pad * 64, 0, 0};
  Tl::run(acc, lds, A, B, a.segs[WIDE], 0, a.ksteps);
  const float f = a.to_log2 / scale_x<T>(a.mode) / scale_w<T>(a.mode), lg = __is_same(E, bf16) ? 0.0f : 15.0f;  // log2 of scale_g
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
  if (vleft < 256) mask_features<Tl>(acc, vleft, wm, lane, -INFINITY);
#pragma unroll
  for (int j = 0; j < Tl::NB; ++j) {
    const int64_t n = n0 + Tl::n_of(wn, lane, j);
    const bool ok = n < live;
    // a row behind the last one has an operand of zeros, lse of infinity and so a gradient of zeros; the power of two sg
    // goes into the exponent
    const float2 lse = ok ? a.lse[n] : float2{0.0f, INFINITY};
    const float top = lse.x * scale_x<T>(a.mode) * scale_w<T>(a.mode), l = lse.y - lg;
#pragma unroll
    for (int i = 0; i < Tl::MB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r] - top, f, -l));
    if (a.coef != nullptr) {
      const float c = ok ? a.coef[n] : 0.0f;
#pragma unroll
      for (int i = 0; i < Tl::MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] *= c;
    }
  }
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    if (t > 0) Tl::renew(acc);
    Tl::store_operand(lds, reinterpret_cast<E*>(reinterpret_cast<char*>(out) + t * a.plane), blk, [&](int i, int j, int g) {
      return quad<E>([&](int e) { return (float)Terms<E, TERMS>(acc[i][j][4 * g + e]).t[t]; });
    });
  }
}

template <typename T, int TERMS>
__global__ void __launch_bounds__(kThreads, 2) grad_kernel(GradArgs a) {
  __shared__ char smem[HeadTile<typename Wide<T>::E>::LDS];
  by_format<T>(a.mode, [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value;
    grad_tile<T, WIDE, WIDE ? Wide<T, WIDE>::P : TERMS>(a, (LdsChar*)smem);
  });
}

// The targets' entries of a piece's G.  Entries of equal ids write equal values.
template <typename T>
__global__ void __launch_bounds__(kThreads) scatter_kernel(const int64_t* ids, int64_t ids_ld, int64_t N, int K, const int* pos,
                                                           const float* t, const float* coef, const WideMode* mode, int64_t v0,
                                                           int cols, char* g, int64_t n_pad, int64_t plane, int terms) {
  const int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t n = e / K;
  if (n >= N) return;
  const int at = pos[n];
  const int64_t v = ids[n * ids_ld + (e - n * K)] - v0;
  if (at < 0 || v < 0 || v >= cols) return;
  const float x = (coef != nullptr ? t[e] * coef[at] : t[e]) * scale_g<T>(mode, 0);
  char* const p = g + ((v >> 5) * (n_pad * 32) + (int64_t)at * 32 + (v & 31)) * 2;
  by_format<T>(mode, [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value;
    using E = typename Wide<T, WIDE>::E;
    if constexpr (WIDE) {
      const Terms<E, 3> w(x);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<E*>(p + k * plane) = w.t[k];
    } else {
      const Terms<E, 2> w(x);
      *reinterpret_cast<E*>(p) = w.t[0];
      if (terms == 2) *reinterpret_cast<E*>(p + plane) = w.t[1];
    }
  });
}

__global__ void zero_kernel(uint16_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) p[i] = 0;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
int64_t es_of(int dtype) { return dtype == 0 ? 4 : 2; }
bool w_direct(const HeadCall& c) {
  return c.dtype != 0 && c.d % 32 == 0 && ((uintptr_t)c.w & 15) == 0 && c.w_ld % 8 == 0 && c.w_ld * 2 * 256 < ((int64_t)1 << 32);
}
// Scores of a few rows without a gradient: the rows are operands as they are, and none is taken out.  16 rows of 512 by 50257
// bf16: 28.0 us with the plan and the copy, 21.6 without.  But rows that do not count are then multiplied as well; us with /
// without: 512 rows 49.6 / 43.2, of which 40% do not count 43.1 / 42.6; 1024 rows 76.5 / 70.6 and 53.5 / 69.3.
constexpr int64_t kDirectRows = 512;
bool x_direct(const HeadCall& c) {
  return c.state == nullptr && c.teacher == nullptr && c.reduction == 0 && c.N <= kDirectRows && w_direct(c) &&
         ((uintptr_t)c.x & 15) == 0 && c.x_ld % 8 == 0 && c.x_ld * 2 * 256 < ((int64_t)1 << 32);
}

struct HeadPlan {
  int64_t n_pad, dp, x_plane, w_plane, C, g_plane;
  int planes, g_terms, tiles_n, tiles_v;
  WideShare share;
  bool distill, few, direct;  // direct: x is used as it is
  WideMode* mode;             // backward, a coefficient a row: the format that they need
  char *x, *w, *g, *state = nullptr;
  float2 *part, *tp;
  WidePart* parts;
  float *ent, *rows, *coef, *cmax, *dx_part, *dw_part;
  uint8_t* live;
  size_t bytes;
  HeadPlan(const HeadCall& c, int backward) {
    distill = c.teacher != nullptr;
    planes = planes_of(c.dtype);
    g_terms = terms_of_g(c.dtype, c.N);
    n_pad = round_up(c.N > 0 ? c.N : 1, 128);
    dp = wide_dp(c.d);
    x_plane = round_up(n_pad * dp * 2, 256);
    w_plane = round_up(c.V * dp * 2, 256);
    tiles_n = (int)(n_pad / 128);
    few = c.N <= kFew && (c.V + 63) / 64 <= kFewTiles;
    tiles_v = (int)(few ? (c.V + 63) / 64 : (c.V + 255) / 256);
    char* p = (char*)c.workspace;
    size_t o = 0;
    auto take = [&](int64_t bytes) { char* q = p + o; o += (size_t)round_up(bytes, 256); return q; };
    direct = !backward && x_direct(c);
    x = direct ? nullptr : take(planes * x_plane);
    w = w_direct(c) ? nullptr : take(planes * w_plane);
    C = g_plane = 0;
    share = WideShare{};
    mode = nullptr; parts = nullptr; part = tp = nullptr; ent = rows = coef = cmax = dx_part = dw_part = nullptr; live = nullptr; g = nullptr;
    if (!backward) {
      part = (float2*)take((int64_t)tiles_v * n_pad * 8);
      state = c.state == nullptr && !direct ? take((int64_t)HeadState(nullptr, c.N, c.K).bytes) : (char*)c.state;
      if (c.dtype == 0) parts = (WidePart*)take(kPartBytes);
      if (c.reduction != 0) rows = (float*)take(c.N * 4);
      if (distill) {
        tp = (float2*)take(c.N * c.K * 8);
        ent = (float*)take(c.N * 4);
        live = (uint8_t*)take(c.N);
      }
    } else {
      C = wide_piece(c.N, c.d, c.V, 1, c.dtype == 0 ? 3 : g_terms, c.dx != nullptr, c.dw != nullptr, g_terms * 2 * n_pad, &share);
      g_plane = round_up(n_pad * C * 2, 256);
      g = take(g_planes(c.dtype, c.N) * g_plane);
      if (c.reduction == 0) {
        coef = (float*)take(n_pad * 4);
        cmax = (float*)take(4);
        mode = (WideMode*)take(sizeof(WideMode));
      }
      if (c.dx != nullptr) dx_part = (float*)take((int64_t)share.dx_split * n_pad * dp * 4);
      if (c.dw != nullptr && share.dw_split > 1) dw_part = (float*)take((int64_t)share.dw_split * C * dp * 4);
    }
    bytes = o;
  }
  void logits(MmSegs (&s)[2]) const {
    s[0] = s[1] = MmSegs{};
    s[0].n = 1;
    if (planes > 1) {
      s[0].b[0] = x_plane;
      s[0].a[1] = w_plane;
      s[0].n = 3;
      s[0].low = 2;
      for (int order = 2; order >= 0; --order) add_wide_segs(s[1], order, 0, w_plane, 0, x_plane);
    }
  }
};

#define HEAD_TRY(call) do { const hipError_t e_ = (call); if (e_ != hipSuccess) return e_; } while (0)

// hidden's counting rows and the weight as operands; the forward pass finds fp32's scales and format for both passes
hipError_t operands(const HeadCall& c, const HeadPlan& p, const HeadState& st, const WideMode* mode, bool find) {
  RowsCopies all = {};
  all.dtype = c.dtype;
  all.mode = mode;
  all.add(RowsCopy{c.x, c.x_ld, c.N, c.d, p.x, p.x_plane, p.n_pad * 64, st.pos, 0, 0});
  if (p.w != nullptr) all.add(RowsCopy{c.w, c.w_ld, c.V, c.d, p.w, p.w_plane, c.V * 64, nullptr, 1, 0});
  if (c.dtype == 0 && find) HEAD_TRY(launch_wide_mode(all, p.parts, st.mode, 0, c.stream));
  return launch_rows_copy(all, c.stream);
}

template <typename T>
hipError_t head_fwd(const HeadCall& c) {
  const HeadPlan p(c, 0);
  const HeadState st(p.state, c.N, c.K);
  const unsigned row_blocks = (unsigned)((c.N + 3) / 4);
  const float inv_t = 1.0f / c.temperature;
  if (p.distill && c.N > 0) {
    if (c.teacher_dtype == 0)
      hipLaunchKernelGGL(teacher_kernel<float>, dim3(row_blocks), dim3(kThreads), 0, c.stream, (const float*)c.teacher, c.teacher_ld, c.ids, c.ids_ld, c.N, c.K, inv_t, p.tp, p.ent, p.live);
    else if (c.teacher_dtype == 1)
      hipLaunchKernelGGL(teacher_kernel<bf16>, dim3(row_blocks), dim3(kThreads), 0, c.stream, (const bf16*)c.teacher, c.teacher_ld, c.ids, c.ids_ld, c.N, c.K, inv_t, p.tp, p.ent, p.live);
    else
      hipLaunchKernelGGL(teacher_kernel<f16>, dim3(row_blocks), dim3(kThreads), 0, c.stream, (const f16*)c.teacher, c.teacher_ld, c.ids, c.ids_ld, c.N, c.K, inv_t, p.tp, p.ent, p.live);
    HEAD_TRY(hipGetLastError());
  }
  const bool direct = p.direct;
  if (!direct) {
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, c.stream, c.ids, c.ids_ld, c.ignore_index, p.live, c.N, st.pos, st.mode);
    HEAD_TRY(hipGetLastError());
  }
  if (c.N > 0) {
    if (!direct) HEAD_TRY(operands(c, p, st, st.mode, true));
    StatsArgs a;
    a.x = direct ? (const char*)c.x : p.x; a.x_ld = direct ? c.x_ld * 2 : 64; a.x_blk = direct ? 64 : p.n_pad * 64; a.rows = direct ? c.N : p.n_pad;
    a.w = p.w != nullptr ? p.w : (const char*)c.w; a.w_ld = p.w != nullptr ? 64 : c.w_ld * 2; a.w_blk = p.w != nullptr ? c.V * 64 : 64; a.V = c.V;
    p.logits(a.segs); a.ksteps = (int)(p.dp / 32); a.tiles_v = p.tiles_v; a.tiles_n = p.few ? 1 : p.tiles_n;
    a.to_log2 = kLog2e / c.temperature; a.mode = direct ? nullptr : st.mode; a.part = p.part; a.part_ld = p.n_pad;
    using E = typename Wide<T>::E;
    const unsigned blocks = (unsigned)((int64_t)a.tiles_v * a.tiles_n);
    if (p.few) hipLaunchKernelGGL((stats_kernel<T, HeadFew>), dim3(blocks), dim3(HeadFew<E>::THREADS), 0, c.stream, a);
    else hipLaunchKernelGGL((stats_kernel<T, HeadTile>), dim3(blocks), dim3(HeadTile<E>::THREADS), 0, c.stream, a);
    HEAD_TRY(hipGetLastError());
    RowsArgs r;
    r.x = a.x; r.x_ld = a.x_ld; r.x_blk = a.x_blk; r.w = a.w; r.w_ld = a.w_ld; r.w_blk = a.w_blk; r.ksteps = a.ksteps;
    for (int i = 0; i < 2; ++i) r.segs[i] = a.segs[i];
    r.ids = c.ids; r.ids_ld = c.ids_ld; r.tp = p.tp; r.ent = p.ent;
    r.part = p.part; r.part_ld = p.n_pad; r.tiles = p.tiles_v; r.N = c.N; r.V = c.V; r.ignore = c.ignore_index; r.K = c.K;
    r.rows = c.N > 2048 ? 8 : c.N > 1024 ? 4 : c.N > 512 ? 2 : 1;
    r.temperature = c.temperature; r.pos = direct ? nullptr : st.pos; r.mode = direct ? nullptr : st.mode; r.lse = direct ? nullptr : st.lse; r.t = direct ? nullptr : st.t;
    r.loss = c.reduction == 0 ? c.loss : p.rows;
    hipLaunchKernelGGL((r.rows * r.K > 1 ? rows_kernel<T, 4> : rows_kernel<T, 8>), dim3((unsigned)((c.N + r.rows - 1) / r.rows)), dim3(kThreads), 0, c.stream, r);
    HEAD_TRY(hipGetLastError());
  }
  if (c.reduction != 0) {
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, c.stream, p.rows, c.N, st.mode, c.reduction == 1, c.loss);
    HEAD_TRY(hipGetLastError());
  }
  return hipSuccess;
}

template <typename T>
hipError_t head_bwd(const HeadCall& c) {
  const HeadPlan p(c, 1);
  const HeadState st(c.state, c.N, c.K);
  if (c.N == 0) {
    if (c.dw != nullptr)
      hipLaunchKernelGGL(zero_kernel, dim3(1024), dim3(kThreads), 0, c.stream, (uint16_t*)c.dw, c.V * c.d * es_of(c.dtype) / 2);
    return hipGetLastError();
  }
  const float factor = p.distill ? c.temperature : 1.0f;  // T^2 of the loss, 1/T of z
  const GradUnit unit{c.dloss, factor, c.reduction};
  const WideMode* const mode = c.reduction == 0 ? p.mode : st.mode;
  if (c.reduction == 0) {
    hipLaunchKernelGGL(coef_kernel, dim3(1), dim3(1024), 0, c.stream, c.dloss, factor, c.N, p.n_pad, st.pos, st.mode, p.mode, p.cmax, p.coef);
    HEAD_TRY(hipGetLastError());
  }
  HEAD_TRY(operands(c, p, st, mode, false));
  const char* w = p.w != nullptr ? p.w : (const char*)c.w;
  const int64_t w_ld = p.w != nullptr ? 64 : c.w_ld * 2, w_blk = p.w != nullptr ? c.V * 64 : 64;
  for (int64_t v0 = 0; v0 < c.V; v0 += p.C) {
    const int cols = (int)(c.V - v0 < p.C ? c.V - v0 : p.C);
    GradArgs a;
    a.x = p.x; a.n_pad = p.n_pad; a.w = w + v0 * w_ld; a.w_ld = w_ld; a.w_blk = w_blk; a.cols = cols;
    p.logits(a.segs); a.ksteps = (int)(p.dp / 32); a.tiles_v = (int)(round_up(cols, 256) / 256); a.tiles_n = p.tiles_n;
    a.to_log2 = kLog2e / c.temperature; a.mode = mode; a.lse = st.lse; a.coef = p.coef; a.g = p.g; a.plane = p.g_plane;
    auto* grad = p.g_terms == 2 ? grad_kernel<T, 2> : grad_kernel<T, __is_same(T, float) ? 2 : 1>;
    hipLaunchKernelGGL(grad, dim3((unsigned)((int64_t)a.tiles_v * a.tiles_n)), dim3(kThreads), 0, c.stream, a);
    HEAD_TRY(hipGetLastError());
    hipLaunchKernelGGL(scatter_kernel<T>, dim3((unsigned)((c.N * c.K + kThreads - 1) / kThreads)), dim3(kThreads), 0, c.stream,
                       c.ids, c.ids_ld, c.N, c.K, st.pos, st.t, p.coef, mode, v0, cols, p.g, p.n_pad, p.g_plane, p.g_terms);
    HEAD_TRY(hipGetLastError());
    WideProducts q = {};
    q.dtype = c.dtype; q.gated = 0; q.N = c.N; q.n_pad = p.n_pad; q.d = c.d; q.dp = p.dp; q.halves = 1; q.cols = cols;
    q.C = p.C;
    q.x = p.x; q.x_ld = 64; q.x_blk = p.n_pad * 64; q.x_plane = p.x_plane; q.x_rows = (int)p.n_pad;
    q.w[0] = w + v0 * w_ld; q.w_ld = w_ld; q.w_blk = w_blk; q.w_plane = p.w_plane; q.w_rows = (int)(c.V - v0);
    q.g = p.g; q.g_plane = p.g_plane; q.g_half = 0; q.g_terms = p.g_terms;
    q.dx_part = p.dx_part; q.dx_add = v0 > 0;
    q.dw[0] = c.dw == nullptr ? nullptr : (char*)c.dw + v0 * c.d * es_of(c.dtype); q.dw_part = p.dw_part;
    q.share = p.share; q.mode = mode; q.unit = unit; q.cmax = p.cmax; q.use_live = 1;
    HEAD_TRY(launch_wide_products(q, c.stream));
  }
  if (c.dx != nullptr) {
    const WideFinish f{c.dtype, 0, c.N, p.n_pad, c.d, p.dp, p.share.dx_split, p.dx_part, st.pos, mode, unit, p.cmax, c.dx};
    HEAD_TRY(launch_wide_finish(f, c.stream));
  }
  return hipSuccess;
}

}  // namespace

size_t head_state_bytes(int64_t N, int K) { return HeadState(nullptr, N, K).bytes; }
size_t head_workspace_bytes(const HeadCall& c, int backward) { return HeadPlan(c, backward).bytes; }

hipError_t launch_head_fwd(const HeadCall& c) {
  return c.dtype == 0 ? head_fwd<float>(c) : c.dtype == 1 ? head_fwd<bf16>(c) : head_fwd<f16>(c);
}
hipError_t launch_head_bwd(const HeadCall& c) {
  return c.dtype == 0 ? head_bwd<float>(c) : c.dtype == 1 ? head_bwd<bf16>(c) : head_bwd<f16>(c);
}

}  // namespace msa

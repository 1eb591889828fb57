// Verification of drafted tokens against the target model's rows (gfx950).
//
// Node 0 of a sequence's tree is its last committed token; target row i is the
// target's distribution after node i.  From node 0 the walk takes, at each
// node, the first child in index order that is accepted:
//   greedy  x is the row's largest entry (the first of equal ones)
//   tree    u p' <= p: u_i (1 - sum of the refused siblings' p) < p(x_i), where a
//           token that an earlier sibling had counts as 0 (it was refused)
//   chain   u_i q(x_i) < p(x_i), q the row that the token was drawn from
// and where none is, one token more: the row's largest entry, or with u_0 from
// p without the refused children, from max(p - q, 0), or, past a chain's last
// node or before one without a token, from p: the first v with weight and cumulated weight > u_0 total.  The
// tokens so produced are distributed as the target's own.
// All sums and comparisons are in 64 bits: probabilities of fp32 or fewer bits
// are exact there and so is u q, and the borders between tokens move by 1e-16.
//
// What bounds it: latency.  The walk needs M gathered entries (3.8 us with the
// launch), then one row (two for a chain), which a block of 1024 threads per
// sequence reads once for 16 segment sums (5 us at V = 50257, 9 at 128000) and
// whose chosen sixteenth it reads a second time, in order (3 us).  Greedy reads
// all M rows, a block per 8192 entries (8 x 64 rows of 50257 bf16: 14.7 us, 3.5
// TB/s), then walks (3.8 us).
#include "msa_device.h"
#include "msa_internal.h"

namespace msa {

constexpr int kPart = 8192;  // entries of a block of the greedy pass
constexpr int kVerifyThreads = 1024, kVerifyWaves = kVerifyThreads / 64;

// VEC consecutive entries of a row as fp32, from an address of any alignment
// of the type (global loads need no more).
template <typename T> struct RowLoad;
template <> struct RowLoad<float> {
  static constexpr int N = 4;
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct RowLoad<bf16> {
  static constexpr int N = 8;
  typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct RowLoad<f16> {
  static constexpr int N = 8;
  typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <typename T>
__device__ inline void load_row(const T* p, int64_t v, int64_t V, float (&x)[RowLoad<T>::N], float past) {
  constexpr int N = RowLoad<T>::N;
  if (v + N <= V) {
    const auto y = *reinterpret_cast<const typename RowLoad<T>::vec*>(p + v);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (float)y[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = v + e < V ? to_f(p[v + e]) : past;
  }
}

// Larger key: larger value, NaN above all (as torch's argmax has it), then the
// lower index.
__device__ inline unsigned long long arg_key(float x, uint32_t v) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
  const uint32_t k = x != x ? 0xffffffffu : (b & 0x80000000u) != 0u ? ~b : b | 0x80000000u;
  return ((unsigned long long)k << 32) | (0xffffffffu - v);
}
__device__ inline unsigned long long shfl_xor64(unsigned long long x, int o) {
  return ((unsigned long long)(uint32_t)__shfl_xor((int)(x >> 32), o) << 32) | (uint32_t)__shfl_xor((int)x, o);
}
__device__ inline double shfl_up_d(double x, int o) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x);
  return __longlong_as_double((long long)(((unsigned long long)(uint32_t)__shfl_up((int)(b >> 32), o) << 32) |
                                          (uint32_t)__shfl_up((int)b, o)));
}
__device__ inline double shfl_d(double x, int l) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x);
  return __longlong_as_double((long long)(((unsigned long long)(uint32_t)__shfl((int)(b >> 32), l) << 32) |
                                          (uint32_t)__shfl((int)b, l)));
}

// The largest entry of part blockIdx.y (kPart entries) of row blockIdx.x = b M +
// i.  A thread holds its entries in registers: their maximum first (NaN noted
// apart), and once the block's is known, its place in the threads that have it.
template <typename T>
__global__ __launch_bounds__(256) void argmax_kernel(VerifyCall a) {
  constexpr int N = RowLoad<T>::N, U = kPart / (256 * N);
  __shared__ unsigned long long red[4];
  const int b = blockIdx.x / a.M, i = blockIdx.x % a.M;
  const T* row = (const T*)a.target + b * a.t_sb + i * a.t_sn;
  const int64_t v0 = (int64_t)blockIdx.y * kPart + threadIdx.x * N;
  float x[U][N];
  if ((int64_t)(blockIdx.y + 1) * kPart <= a.V) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const auto y = *reinterpret_cast<const typename RowLoad<T>::vec*>(row + v0 + u * 256 * N);
#pragma unroll
      for (int e = 0; e < N; ++e) x[u][e] = (float)y[e];
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) load_row(row, v0 + u * 256 * N, a.V, x[u], -INFINITY);
  }
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      top = fmaxf(top, x[u][e]);
      nan = nan || x[u][e] != x[u][e];
    }
  float m = nan ? NAN : top;
  // the wave's, then the first place of it in the wave
  bool wnan = __ballot(nan) != 0ull;
  float wtop = top;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) wtop = fmaxf(wtop, __shfl_xor(wtop, o));
  uint32_t at = 0xffffffffu;
  if (wnan ? nan : m == wtop) {
#pragma unroll
    for (int u = U - 1; u >= 0; --u)
#pragma unroll
      for (int e = N - 1; e >= 0; --e)
        if (wnan ? x[u][e] != x[u][e] : x[u][e] == wtop) at = (uint32_t)(v0 + u * 256 * N + e);
    if (at >= a.V) at = 0xffffffffu;  // behind the row (all of its entries are -inf)
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)at, o);
    at = y < at ? y : at;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = at == 0xffffffffu ? 0ull : arg_key(wnan ? NAN : wtop, at);
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long best = red[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) best = red[w] > best ? red[w] : best;
    a.best[(int64_t)blockIdx.x * gridDim.y + blockIdx.y] = best;
  }
}

// A sequence's nodes, one per lane.
struct Nodes {
  int parent;     // -1: node 0, or not part of the tree (never reached)
  int64_t token;
  bool valid;     // a token of the vocabulary
  __device__ Nodes(const VerifyCall& a, int b, int lane) {
    const bool in = lane < a.M;
    token = in ? a.tokens[(int64_t)b * a.M + lane] : -1;
    valid = token >= 0 && token < a.V;
    const int64_t p = a.parents == nullptr ? lane - 1 : (in ? a.parents[b * a.par_sb + lane] : -1);
    parent = in && p >= 0 && p < lane ? (int)p : -1;
  }
  // The nodes before this one under the same parent (nodes without one: none),
  // by the bits of the parents.
  __device__ unsigned long long before(int lane) const {
    unsigned long long m = __ballot(parent >= 0);
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      const bool bit = ((parent >> k) & 1) != 0;
      const unsigned long long on = __ballot(bit);
      m &= bit ? on : ~on;
    }
    return parent >= 0 ? m & ((1ull << lane) - 1ull) : 0ull;
  }
};
__device__ inline int64_t shfl_i64(int64_t x, int l) {
  return ((int64_t)__shfl((int)(x >> 32), l) << 32) | (uint32_t)__shfl((int)x, l);
}

// The way down from node 0 over nodes taken (at most one child of each), into
// path (-1 behind it) and count.  Returns the last node.  Wave-wide.
__device__ inline int walk(const VerifyCall& a, int b, int lane, const Nodes& n, bool taken) {
  int node = 0, len = 1, mine = lane == 0 ? 0 : -1;
  for (;;) {
    const unsigned long long next = __ballot(taken && n.parent == node);
    if (next == 0ull) break;
    node = (int)__builtin_ctzll(next);  // a later node than its parent: the walk ends
    if (lane == len) mine = node;
    ++len;
  }
  if (lane < a.M) a.path[(int64_t)b * a.M + lane] = mine;
  if (lane == 0) a.count[b] = len;
  return node;
}

// Greedy: the rows' largest entries are in a.best, `parts` per row.
__global__ __launch_bounds__(64) void greedy_walk_kernel(VerifyCall a, int parts) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const Nodes n(a, b, lane);
  unsigned long long best = 0ull;
  if (lane < a.M)
#pragma unroll 8
    for (int s = 0; s < parts; ++s) {
      const unsigned long long k = a.best[((int64_t)b * a.M + lane) * parts + s];
      best = k > best ? k : best;
    }
  const int top = (int)(0xffffffffu - (uint32_t)best);  // V <= 2^31
  const int want = __shfl(top, n.parent < 0 ? 0 : n.parent);
  bool taken = n.parent >= 0 && n.token == want;
  if ((__ballot(taken) & n.before(lane)) != 0ull) taken = false;  // the first of the siblings that have the token
  const int last = walk(a, b, lane, n, taken);
  const int tok = __shfl(top, last);
  if (lane == 0) a.token[b] = tok;
}

// Sampled: block per sequence.
template <typename T, bool kChain>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyCall a) {
  constexpr int N = RowLoad<T>::N;
  __shared__ double seg[kVerifyWaves];
  __shared__ int64_t gone[64];          // tokens refused at the last node
  __shared__ uint32_t bins[128];        // which of 4096 stretches of the row hold one
  __shared__ int last_s, gone_s;
  __shared__ unsigned long long first_s, tail_s;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const double u0 = (double)a.uniforms[(int64_t)b * a.M];
  int shift = 3;  // a stretch holds whole loads
  while ((a.V >> shift) > 4095) ++shift;
  if (t < 128) bins[t] = 0u;
  if (t == 0) {
    first_s = ~0ull;
    tail_s = 0ull;
  }
  __syncthreads();
  if (wave == 0) {
    const Nodes n(a, b, lane);
    const float u = lane < a.M ? a.uniforms[(int64_t)b * a.M + lane] : 0.0f;
    const bool asked = n.parent >= 0 && n.valid;
    const int up = asked ? n.parent : 0;
    double p = asked ? (double)to_f(((const T*)a.target + b * a.t_sb + (int64_t)up * a.t_sn)[n.token]) : 0.0;
    bool taken;
    const bool on = asked && (!kChain || n.parent == lane - 1);  // a draft that the walk may ask
    if constexpr (kChain) {
      const double q = on ? (double)to_f(((const T*)a.draft + b * a.d_sb + (int64_t)up * a.d_sn)[n.token]) : 0.0;
      taken = on && (double)u * q < p;
    } else {
      if (!(p > 0.0)) p = 0.0;
      const unsigned long long before = asked ? n.before(lane) : 0ull;
      // a token that an earlier sibling had counts once
      for (unsigned long long m = before; __ballot(m != 0ull) != 0ull; m &= m - 1ull) {
        const int64_t tok = shfl_i64(n.token, m != 0ull ? (int)__builtin_ctzll(m) : lane);
        if (m != 0ull && tok == n.token) p = 0.0;
      }
      double left = 1.0;
      for (unsigned long long m = before; __ballot(m != 0ull) != 0ull; m &= m - 1ull) {
        const double share = shfl_d(p, m != 0ull ? (int)__builtin_ctzll(m) : lane);
        if (m != 0ull) left -= share;
      }
      taken = asked && (double)u * left < p;
      if ((__ballot(taken) & before) != 0ull) taken = false;
    }
    const int last = walk(a, b, lane, n, taken);
    // the children of the last node, none of them taken; a chain whose next node
    // is missing or holds no token of the vocabulary has refused nothing there
    const unsigned long long out = __ballot(on && n.parent == last);
    if (!kChain && ((out >> lane) & 1ull) != 0ull) {
      gone[__builtin_popcountll(out & ((1ull << lane) - 1ull))] = n.token;
      const uint32_t bin = (uint32_t)(n.token >> shift);
      atomicOr(&bins[bin >> 5], 1u << (bin & 31u));
    }
    if (lane == 0) {
      last_s = last;
      gone_s = __builtin_popcountll(out);
    }
  }
  __syncthreads();
  const int last = last_s, ngone = gone_s;
  const T* prow = (const T*)a.target + b * a.t_sb + (int64_t)last * a.t_sn;
  const T* qrow = kChain && ngone > 0 ? (const T*)a.draft + b * a.d_sb + (int64_t)last * a.d_sn : nullptr;
  bool plain = false;  // the second time, if nothing is left: p itself

  typedef typename RowLoad<T>::vec vec;
  // weights of entries v .. v + N - 1 (v a multiple of N) with probabilities p
  // (and the draft's q)
  auto weigh = [&](int64_t v, const float (&p)[N], const float (&q)[N], double (&x)[N]) {
    if (kChain && qrow != nullptr && !plain) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double d = (double)p[e] - (double)q[e];
        x[e] = d > 0.0 ? d : 0.0;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (double)fmaxf(p[e], 0.0f);  // a NaN counts as 0
    if (kChain || plain) return;
    const uint32_t bin = (uint32_t)(v >> shift);
    if (((bins[bin >> 5] >> (bin & 31u)) & 1u) != 0u)
      for (int j = 0; j < ngone; ++j) {
        const int64_t g = gone[j];
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (v + e == g) x[e] = 0.0;
      }
  };
  auto weights = [&](int64_t v, double (&x)[N]) {  // the row ends at V
    float p[N], q[N];
    load_row(prow, v, a.V, p, 0.0f);
    if (kChain && qrow != nullptr) load_row(qrow, v, a.V, q, 0.0f);
    weigh(v, p, q, x);
  };

  // sums of the row's sixteenths, one a wave
  const int64_t len = ((a.V + kVerifyWaves - 1) / kVerifyWaves + N - 1) / N * N;
  double total = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    plain = pass == 1;
    const int64_t lo = len * wave, hi = lo + len < a.V ? lo + len : a.V;
    double s = 0.0;
    constexpr int U = 32 / N;  // loads in flight
    for (int64_t v0 = lo + lane * N; v0 < hi; v0 += U * 64 * N) {
      vec p[U], q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t v = v0 + u * 64 * N;
        p[u] = q[u] = vec(0);
        if (v + N <= hi) {
          p[u] = *reinterpret_cast<const vec*>(prow + v);
          if (kChain && qrow != nullptr) q[u] = *reinterpret_cast<const vec*>(qrow + v);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float pf[N], qf[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          pf[e] = (float)p[u][e];
          qf[e] = (float)q[u][e];
        }
        double x[N];
        weigh(v0 + u * 64 * N, pf, qf, x);
#pragma unroll
        for (int e = 0; e < N; ++e) s += x[e];
      }
    }
    const int64_t rest = lo + (hi - lo) / N * N;  // the row's last entries, fewer than a load
    if (lane == 0 && rest < hi) {
      double x[N];
      weights(rest, x);
#pragma unroll
      for (int e = 0; e < N; ++e) s += x[e];
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long k = shfl_xor64((unsigned long long)__double_as_longlong(s), o);
      s += __longlong_as_double((long long)k);
    }
    __syncthreads();
    if (lane == 0) seg[wave] = s;
    __syncthreads();
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kVerifyWaves; ++w) total += seg[w];
    if (total > 0.0) break;
  }
  const double want = u0 * total;
  // the first sixteenth whose sums pass `want`, else the last with any weight
  int at = -1;
  double base = 0.0, run = 0.0;
  for (int w = 0; w < kVerifyWaves; ++w) {
    if (seg[w] > 0.0) {
      if (at < 0 || !(base + seg[at] > want)) {
        at = w;
        base = run;
      }
    }
    run += seg[w];
  }
  if (at < 0) {  // no weight anywhere
    if (t == 0) a.token[b] = 0;
    return;
  }
  // its entries in order: thread t has `each` of them from t each on
  const int64_t lo = len * at, hi = lo + len < a.V ? lo + len : a.V;
  const int64_t each = ((len + kVerifyThreads - 1) / kVerifyThreads + N - 1) / N * N;
  const int64_t v0 = lo + t * each, v1 = v0 + each < hi ? v0 + each : hi;
  double s = 0.0;
  for (int64_t v = v0; v < v1; v += N) {
    double x[N];
    weights(v, x);
#pragma unroll
    for (int e = 0; e < N; ++e) s += v + e < v1 ? x[e] : 0.0;
  }
  double incl = s;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = shfl_up_d(incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();  // seg has been read
  if (lane == 63) seg[wave] = incl;
  __syncthreads();
  double sum = base + (incl - s);
  for (int w = 0; w < wave; ++w) sum += seg[w];
  unsigned long long first = ~0ull, tail = 0ull;
  for (int64_t v = v0; v < v1; v += N) {
    double x[N];
    weights(v, x);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (v + e < v1 && x[e] > 0.0) {
        sum += x[e];
        if (sum > want && first == ~0ull) first = (unsigned long long)(v + e);
        tail = (unsigned long long)(v + e) + 1ull;
      }
  }
  // entries grow with the lanes: the wave's first and last
  const unsigned long long some = __ballot(first != ~0ull), rest = __ballot(tail != 0ull);
  if (some != 0ull && lane == (int)__builtin_ctzll(some)) atomicMin(&first_s, first);
  if (rest != 0ull && lane == 63 - (int)__builtin_clzll(rest)) atomicMax(&tail_s, tail);
  __syncthreads();
  if (t == 0) a.token[b] = first_s != ~0ull ? (int64_t)first_s : (int64_t)tail_s - 1;
}

// Parts of a row in the greedy pass.
int verify_parts(int64_t V) { return (int)((V + kPart - 1) / kPart); }

template <typename T>
static hipError_t launch_verify_t(const VerifyCall& c) {
  if (c.uniforms == nullptr) {
    const int parts = verify_parts(c.V);
    hipLaunchKernelGGL((argmax_kernel<T>), dim3((unsigned)(c.B * c.M), (unsigned)parts), dim3(256), 0, c.stream, c);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(greedy_walk_kernel, dim3((unsigned)c.B), dim3(64), 0, c.stream, c, parts);
  } else if (c.draft != nullptr) {
    hipLaunchKernelGGL((verify_kernel<T, true>), dim3((unsigned)c.B), dim3(kVerifyThreads), 0, c.stream, c);
  } else {
    hipLaunchKernelGGL((verify_kernel<T, false>), dim3((unsigned)c.B), dim3(kVerifyThreads), 0, c.stream, c);
  }
  return hipGetLastError();
}

hipError_t launch_verify(const VerifyCall& c) {
  if (c.dtype == 1) return launch_verify_t<bf16>(c);
  if (c.dtype == 2) return launch_verify_t<f16>(c);
  return launch_verify_t<float>(c);
}

}  // namespace msa

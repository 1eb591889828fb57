// Screening attention of a tree of drafted tokens over a key/value cache
// (gfx950): N <= 64 nodes per sequence, over caches of the input type or of
// 8-bit codes with a scale per row.  N = 1 is the decode of one token.
//
// Sequence b's cache holds its committed tokens at positions [0, n) and the
// nodes' own rows at n, n + 1, ...; node i stands at position n + depth_i and
// sees the committed keys of its window and, of the drafted rows, its own and
// its ancestors':
//   s = q^.k^,  a = max(1 - r(1 - s), 0),  m = (cos(pi d/w) + 1)/2 for 0 <= d < w
//   y = TanhNorm(sum a^2 m v^)
// There is no softmax, so partial sums over any split of the keys just add.
//
// One wave takes 32 nodes (the columns of a product) and walks 32-key units of
// the window: S = K Q^T on the matrix cores, a vote on the threshold, and only
// for a unit with a live pair the weights, V (through LDS, transposed on the
// way out) and h^T += V^T P^T.  Every key row is thus read once for 32 nodes;
// the nodes' operand and the sums stay in registers.
//
// Operands: rows of the input type enter as they are, 1/|x| multiplies the
// fp32 results.  Codes enter as fp16, which holds every code of both types
// exactly; the nodes' rows are scaled to fp16's range by a power of two (an
// fp32 row as the sum of two fp16 rows, 22 bits).  Pair weights are rounded to
// two terms of the operand's type (16 or 22 bits), in fp16 after a power of two
// that keeps small weights clear of its subnormals.
//
// What bounds it: long windows of few nodes the cache's bytes (one token of 16
// sequences over 94K int8 positions on average, 819 MB: 140 us, 5.9 TB/s); many
// nodes or live units the vector instructions of a unit (about 570 for 64 nodes of
// bf16, 340 for the 16-column form: 56 and 37 to 41 us, half to two thirds of the
// issue slots); short windows the latency of the call (12 us at 9 units a head, of
// which the launch and the tree take 4 and a unit's way through a wave 2 to 3).
#include "../../include/msa.h"
#include "msa_device.h"
#include "msa_internal.h"

namespace msa {

constexpr int kTreeMax = 64;   // nodes of a tree: one lane each
static_assert(kTreeMax == MSA_TREE_MAX);
constexpr int kTreeWaves = 4;  // waves of a block
// Fewest units of a block, so that a block's sums stay small beside its keys (16
// instead of 8: 21 nodes over 5001 e4m3 rows of D = 128 24 -> 30 us, 40 over 6000
// fp32 of D = 32 27 -> 39; 4: no gain).
constexpr int kTreeMinUnits = 8;
// Heads of at most kTreeSmall units are a block each, with no sums to join: at 9
// units one block 12.8 us, two 18.5; at 22 units 14.0 and 14.5; at 41 units 22.0
// and 17.4.  A batch that fills the card twice with heads of at most kTreeLong
// units likewise (256 x 8 heads of 38 units bf16: 130 us, shared 159; of windows
// 2 .. 1500 int8 84, shared 82).
constexpr int kTreeSmall = 24, kTreeLong = 64;

// Waves per SIMD that the kernel's registers are budgeted for, by the bytes of
// the stored row.  Operands of 8-bit rows are fp16, so <int8 or fp8, 32, 1, 2>
// spill 12 and 37 registers at 3 and the D = 128 ones 3 to 6; most 2-byte and 8-bit
// instances of one tile need fewer than they are given, and one or two more of
// their waves fit.
constexpr int tree_occupancy(int row_bytes, int parts) {
  return row_bytes * parts <= 64 ? 3 : row_bytes <= 256 ? 2 : 1;
}
constexpr int tree_occupancy16(int row_bytes, int parts) {  // the same of tree16_kernel
  return row_bytes * parts <= 128 ? 3 : 2;
}

// How a cache row of type C enters the products.
template <typename C> struct TreeRow {
  typedef C comp;  // operand type
  static constexpr bool kCodes = false;
};
template <> struct TreeRow<int8_t> { typedef f16 comp; static constexpr bool kCodes = true; };
template <> struct TreeRow<fp8> { typedef f16 comp; static constexpr bool kCodes = true; };

// Power of two on the pair weights (fp16 operands only): a^2 m <= 1 times the
// row factor, at most 2 for fp16 rows scaled to [1/2, 1), at most 1/64 for codes.
template <typename C> constexpr float kWeightUp = 1.0f;
template <> constexpr float kWeightUp<f16> = 16384.0f;
template <> constexpr float kWeightUp<int8_t> = 2097152.0f;
template <> constexpr float kWeightUp<fp8> = 2097152.0f;

typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4;
typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;
typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2;

// Four codes as fp16.  int8: the code + 128 in the low bits of 1024 is the
// fp16 number 1152 + code; the subtraction is exact.
__device__ inline void decode_f16(uint32_t c, int8_t, f16* o) {
  const uint32_t u = c ^ 0x80808080u;
  const f16x2 off = {(f16)1152.0f, (f16)1152.0f};
  const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
  const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
  o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
}
__device__ inline void decode_f16(uint32_t c, fp8, f16* o) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  o[0] = (f16)a[0]; o[1] = (f16)a[1]; o[2] = (f16)b[0]; o[3] = (f16)b[1];
}
template <typename C>
__device__ inline f16x8 decode8(uint32_t c0, uint32_t c1) {
  f16 o[8];
  decode_f16(c0, C{}, o);
  decode_f16(c1, C{}, o + 4);
  f16x8 f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = o[e];
  return f;
}

// Sum of squares of the int8 codes in N words.
template <int N>
__device__ inline int code_dot(const u32x4& c) {
  int s = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) s = __builtin_amdgcn_sdot4((int)c[e], (int)c[e], s, false);
  return s;
}

// Waits that keep a run's A/B fragments and its result's registers apart from
// later writes (guard_run, for any number of fragments).
template <typename F, int N>
__device__ inline void guard_all(const F (&f)[N], const f32x16& c) {
  if constexpr (__is_same(F, f32x4)) {
    const int x = __builtin_amdgcn_readfirstlane(__float_as_int(c[15]));
#pragma unroll
    for (int k = 0; k < N; ++k) asm volatile("" ::"v"(f[k]), "s"(x));
  } else {
    asm volatile(MSA_NOP16 ::"v"(c[15]));
#pragma unroll
    for (int k = 0; k < N; ++k) asm volatile("" ::"v"(f[k]));
  }
}

// The key operand of a unit: lane l holds row perm_row(l % 32), slots in the
// column order col() below.
template <typename C, int D>
struct KeyRows {
  using comp = typename TreeRow<C>::comp;
  using M = Mma<comp>;
  using frag = typename M::frag;
  static constexpr bool kCodes = TreeRow<C>::kCodes;
  static constexpr int NKS = D / M::KS;
  static constexpr int LB = kCodes && D == 16 ? 8 : 16;            // bytes of a load
  static constexpr int NL = D * (int)sizeof(C) / (2 * LB);         // loads of a lane
  u32x4 raw[NL];
  float scale;

  // Column of slot e of fragment ks in a lane of half `half`.
  __device__ static constexpr int col(int ks, int half) {
    if constexpr (!kCodes) return M::KS * ks + M::PER * half;
    else if constexpr (D == 16) return 8 * half;
    else return 32 * (ks / 2) + 16 * half + 8 * (ks & 1);
  }
  // `off`: the lane's row and half in bytes from the wave-uniform address
  // `rows`, `soff` its scale's.
  __device__ inline void load(const char* rows, uint32_t off, const char* scales, uint32_t soff) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const char* p = rows + off + 2 * i * LB;
      if constexpr (LB == 8) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        raw[i] = u32x4{x[0], x[1], 0u, 0u};
      } else {
        raw[i] = *reinterpret_cast<const u32x4*>(p);
      }
    }
    if constexpr (kCodes) scale = *reinterpret_cast<const float*>(scales + soff);
  }
  __device__ inline void frags(frag (&f)[NKS]) const {
    if constexpr (!kCodes) {
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) f[ks] = __builtin_bit_cast(frag, raw[ks]);
    } else {
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        f[ks] = decode8<C>(raw[D == 16 ? 0 : ks / 2][2 * (ks & 1)], raw[D == 16 ? 0 : ks / 2][2 * (ks & 1) + 1]);
    }
  }
  // 1/max(|k|, eps) of the row, times the code's scale.  A row that is not
  // finite gives 0 or NaN: its pairs are not live.
  __device__ inline float factor(const frag (&f)[NKS], float eps, float inv_eps) const {
    if constexpr (__is_same(C, int8_t)) {
      int ss = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) ss += code_dot<LB / 4>(raw[i]);
      return code_factor(half_sum((float)ss), scale, inv_eps);
    } else if constexpr (kCodes) {
      return code_factor(half_sum(row_dot<comp>(f, f)), scale, inv_eps);
    } else {
      return inv_len_of<C>(half_sum(row_dot<comp>(f, f)), eps);
    }
  }
  // min(1/|c|, scale/eps): the factor that takes a row of codes c with this
  // scale to its unit row (0 for a row of zeros, NaN for one that is not finite).
  __device__ static inline float code_factor(float ss, float scale, float inv_eps) {
    const float f = fminf(inv_len_of<float>(ss, 1e-30f), scale * inv_eps);
    return scale == scale ? f : scale;
  }
};

// The nodes' operand: lane l holds node row l % 32 in the key rows' column
// order; PARTS terms whose sum is the row (scaled for codes).
template <typename C, int D, int PARTS>
struct NodeRows {
  using K = KeyRows<C, D>;
  using frag = typename K::frag;
  frag f[PARTS][K::NKS];
  float inv;  // 1/max(|q|, eps), over the scaling
  template <typename T>
  __device__ inline void load(const T* row, bool ok, float eps, int half) {
    constexpr int PER = K::M::PER, VEC = 16 / (int)sizeof(T);  // PER is a multiple of 4, VEC 4 or 8
    constexpr int W = PER < VEC ? PER : VEC;
    float x[K::NKS][PER];
    float ss = 0.0f, mx = 0.0f;
#pragma unroll
    for (int ks = 0; ks < K::NKS; ++ks)
#pragma unroll
      for (int e0 = 0; e0 < PER; e0 += W) {
        typedef __attribute__((__vector_size__(W * sizeof(T)))) T vec;
        const vec v = *reinterpret_cast<const vec*>(row + K::col(ks, half) + e0);
#pragma unroll
        for (int e = 0; e < W; ++e) x[ks][e0 + e] = ok ? to_f(v[e]) : 0.0f;
      }
#pragma unroll
    for (int ks = 0; ks < K::NKS; ++ks)
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        ss = fmaf(x[ks][e], x[ks][e], ss);
        mx = fmaxf(mx, fabsf(x[ks][e]));
      }
    const float p = TreeRow<C>::kCodes ? row_pow2(half_max(mx)) : 1.0f;
    inv = inv_len_of<float>(half_sum(ss), eps) / p;
#pragma unroll
    for (int ks = 0; ks < K::NKS; ++ks)
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        float rest = x[ks][e] * p;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const auto part = from_f<typename K::comp>(rest);
          f[i][ks][e] = part;
          rest -= to_f(part);
        }
      }
  }
};

// V of a unit on its way to LDS: coalesced 16-byte loads (a row's CPR lanes are
// neighbours), then the operand rows in UnitTile's layout and each row's factor.
template <typename C, int D>
struct ValueRows {
  using comp = typename TreeRow<C>::comp;
  static constexpr bool kCodes = TreeRow<C>::kCodes;
  static constexpr int DP = D < 32 ? 32 : D;
  using Tile = UnitTile<comp, DP>;
  static constexpr int CPR = D * (int)sizeof(C) / 16;
  static constexpr int NV = (kUnit * CPR + 63) / 64;
  u32x4 raw[NV];
  float scale[kCodes ? NV : 1];

  static constexpr int RPI = CPR > 2 ? 64 / CPR : kUnit;  // rows of a load (CPR 1: the upper lanes repeat them)

  // `rows`: wave-uniform address of the unit's first row, rows `st` bytes apart,
  // `lim` the last of them that exists (later ones read it); the scales alike.
  __device__ inline void load(const char* rows, uint32_t st, const char* scales, uint32_t sst, int lim, int lane) {
    const int r0 = (lane / CPR) & (kUnit - 1);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      int r = r0 + i * RPI;
      if (lim < kUnit - 1) r = r < lim ? r : lim;
      raw[i] = *reinterpret_cast<const u32x4*>(rows + (uint32_t)r * st + 16 * (lane % CPR));
      if constexpr (kCodes) scale[i] = *reinterpret_cast<const float*>(scales + (uint32_t)r * sst);
    }
  }
  // A row that is not finite is staged as zeros; its factor is NaN, so that a
  // live pair still sees it and a masked one does not; then the result is true.
  // (A finite row whose length overflows has factor 0.)  The factors are times
  // kWeightUp.
  __device__ inline bool stage(char* tile, float* fac, float eps, float inv_eps, int lane) const {
    typedef typename Mma<comp>::frag vec;  // 16 bytes of an operand row
    constexpr int N = 16 / (int)sizeof(comp);
    constexpr int W = kCodes ? 2 : 1;      // operand chunks of a load
    const int r0 = (lane / CPR) & (kUnit - 1), ch = W * (lane % CPR);
    // lds_swz is linear over the row's bits, and r0 < RPI: the rows of load i
    // differ from r0's place by constants
    uint32_t at[W];
#pragma unroll
    for (int u = 0; u < W; ++u) at[u] = (uint32_t)(r0 * Tile::ROWB + (((ch + u) ^ Tile::swz(r0)) << 4));
    bool odd = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      vec x[W];
      if constexpr (kCodes) {
        x[0] = decode8<C>(raw[i][0], raw[i][1]);
        x[W - 1] = decode8<C>(raw[i][2], raw[i][3]);
      } else {
        x[0] = __builtin_bit_cast(vec, raw[i]);
      }
      float ss = 0.0f;
      if constexpr (__is_same(C, int8_t)) ss = (float)code_dot<4>(raw[i]);
      else
#pragma unroll
      for (int u = 0; u < W; ++u) {
        if constexpr (sizeof(comp) == 2) ss = frag_dot(x[u], x[u], ss);
        else
#pragma unroll
          for (int e = 0; e < N; ++e) ss = fmaf(x[u][e], x[u][e], ss);
      }
      ss = group_sum<CPR>(ss);
      bool finite = ss < INFINITY;
      if constexpr (kCodes) finite = finite && scale[i] == scale[i];
      float f;
      if constexpr (kCodes) f = KeyRows<C, D>::code_factor(ss, scale[i], inv_eps);
      else f = inv_len_of<C>(ss, eps);
      if (__ballot(!finite) != 0ull) {
        float bad = 0.0f;  // an element (or its scale) that is not finite, and not only the squares' sum
        if constexpr (kCodes) bad = scale[i] == scale[i] ? 0.0f : 1.0f;
#pragma unroll
        for (int u = 0; u < W; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (!(fabsf(to_f(x[u][e])) < INFINITY)) bad = 1.0f;
        bad = group_sum<CPR>(bad);
        odd = true;
        if (!finite) {
          f = bad > 0.0f ? __uint_as_float(0x7fc00000u) : 0.0f;
#pragma unroll
          for (int u = 0; u < W; ++u) x[u] = Mma<comp>::zero();
        }
      }
      if constexpr (kCodes) {
        // cache_write's rows reach the type's largest code, so |codes| >= 127 and the
        // factor is at most 1/127; rows of smaller codes (an e4m3 code is 2^-9 at
        // least) are scaled up to a length of 64
        const bool small = ss < 16129.0f;
        if (__ballot(small) != 0ull && small) {
          const float up = ss > 0.0f ? Pow2Split::recip(__uint_as_float(__float_as_uint(sqrtf(ss)) & 0x7f800000u)) * 64.0f : 1.0f;
#pragma unroll
          for (int u = 0; u < W; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) x[u][e] *= (f16)up;
          f = ss > 0.0f ? f / up : 0.0f;
        }
      }
      if constexpr (__is_same(C, f16)) {  // |v| to [1/2, 1) by a power of two, the rest in the factor
        if (finite) {
          const Pow2Split sp(f);
#pragma unroll
          for (int e = 0; e < N; ++e) x[0][e] = (f16)(to_f(x[0][e]) * sp.c1 * sp.c2);
          f = sp.w;
        }
      }
      const bool mine = kUnit * CPR >= 64 || lane < kUnit * CPR;
      if (mine) {
#pragma unroll
        for (int u = 0; u < W; ++u)
          *reinterpret_cast<vec*>(tile + (at[u] ^ (uint32_t)(Tile::swz((i * RPI) & (kUnit - 1)) << 4)) + i * RPI * Tile::ROWB) = x[u];
        if (lane % CPR == 0) fac[r0 + i * RPI] = f * kWeightUp<C>;
      }
    }
    return odd;
  }
};

// The values of unit u of a window whose rows (of `st` bytes) and scales start
// at `rows` and `scales` and end with row `last`.
template <typename C, int D>
__device__ inline void load_values_at(ValueRows<C, D>& val, const char* rows, int64_t st, const char* scales,
                                      int64_t scale_st, int u, int last, int lane) {
  val.load(rows + (int64_t)u * kUnit * st, (uint32_t)st, scales + (int64_t)u * kUnit * scale_st * 4,
           (uint32_t)(scale_st * 4), last - u * kUnit, lane);
}

// Where a C block's registers (rows = tcol-ordered columns) go: groups of
// consecutive columns of one row.
template <typename COMP, typename OUT, int D, typename Fn>
__device__ inline void store_row(OUT* row, int half, Fn fn) {
  constexpr int NDH = (D + 31) / 32;
  if constexpr (sizeof(COMP) == 2) {
#pragma unroll
    for (int dblk = 0; dblk < NDH; ++dblk)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int d0 = 32 * dblk + 16 * g + 8 * half;
        if (d0 < D) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = fn(dblk, 8 * g + e);
          store8(row + d0, v);
        }
      }
  } else {
#pragma unroll
    for (int dblk = 0; dblk < NDH; ++dblk)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d0 = 32 * dblk + 8 * g + 4 * half;
        if (d0 < D) store4(row + d0, fn(dblk, 4 * g), fn(dblk, 4 * g + 1), fn(dblk, 4 * g + 2), fn(dblk, 4 * g + 3));
      }
  }
}
template <typename COMP, int D, typename Fn>
__device__ inline void store_row_as(void* y, int64_t off, int dtype, int half, Fn fn) {
  if (dtype == 1) store_row<COMP, bf16, D>((bf16*)y + off, half, fn);
  else if (dtype == 2) store_row<COMP, f16, D>((f16*)y + off, half, fn);
  else store_row<COMP, float, D>((float*)y + off, half, fn);
}

__device__ inline int wave_max(int x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_xor(x, o);
    x = y > x ? y : x;
  }
  return x;
}

// What a wave knows of the tree: each lane's node, its depth and the bitmap of
// the nodes on its way up (itself among them).  A parent that is no earlier
// node makes the node a root.
struct Tree {
  int depth;
  unsigned long long above;
  __device__ Tree(const int64_t* parents, int N, int lane) {
    if (parents == nullptr) {  // a chain
      depth = lane;
      above = ~0ull >> (63 - lane);
      return;
    }
    int64_t p64 = lane < N ? parents[lane] : -1;
    int p = p64 >= 0 && p64 < lane ? (int)p64 : -1;
    above = 1ull << lane;
    depth = p >= 0 ? 1 : 0;
    // each step doubles the way that `above` covers: p is the first node past it
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      const int at = p < 0 ? lane : p;
      const unsigned long long up =
          ((unsigned long long)(uint32_t)__shfl((int)(above >> 32), at) << 32) | (uint32_t)__shfl((int)above, at);
      const int d = __shfl(depth, at), q = __shfl(p, at);
      if (p >= 0) {
        above |= up;
        depth += d;
        p = q;
      }
    }
  }
};

// Committed length of sequence b; head h's key units: keys lo, lo + 1, ..., n +
// N - 1 in units of 32 (none for an empty window).
struct TreeSpan {
  int n;
  __device__ TreeSpan(const TreeCall& a, int b) {
    int64_t x = a.lengths[(int64_t)b * a.len_step];
    x = x > a.cap - a.N ? a.cap - a.N : x;
    n = x < 0 ? 0 : (int)x;
  }
  __device__ int lo(int wc) const { return n - wc + 1 < 0 ? 0 : n - wc + 1; }
  __device__ int units(const TreeCall& a, int wc) const {
    return wc == 0 ? 0 : (n + a.N - lo(wc) + kUnit - 1) / kUnit;
  }
};

// How the blocks of a sequence share its heads' units: head h's are cut into
// pieces of `per`, the heads' pieces numbered one after the other, a block
// each; `per` is the least (in steps of about an eighth) for which the blocks
// suffice.  Windows differ by orders of magnitude between heads, and blocks per
// head would leave most of the card to the widest.  Wave-uniform.
struct TreeMap {
  int per;
  __device__ static int units_of(const TreeCall& a, const TreeSpan& sp, int h) {
    return h < a.H ? sp.units(a, head_params(a.r, a.w, h, true).wc) : 0;
  }
  __device__ static int sum(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return x;
  }
  __device__ TreeMap(const TreeCall& a, const TreeSpan& sp, int lane) {
    const int first = units_of(a, sp, lane);
    int all = sum(first);
    for (int h = 64; h < a.H; h += 64) all += sum(units_of(a, sp, h + lane));
    per = (all + a.blocks - 1) / a.blocks;
    per = per < kTreeMinUnits ? kTreeMinUnits : per;
    for (;; per += per / 8 + 1) {  // ends: one piece a head fits
      int pieces = sum((first + per - 1) / per);
      for (int h = 64; h < a.H; h += 64) pieces += sum((units_of(a, sp, h + lane) + per - 1) / per);
      if (pieces <= a.blocks) return;
    }
  }
  // The head of piece i, or -1; its first piece.
  __device__ int head_of(const TreeCall& a, const TreeSpan& sp, int lane, int i, int& piece0) const {
    int carry = 0;
    for (int h = 0; h < a.H; h += 64) {
      const int c = (units_of(a, sp, h + lane) + per - 1) / per;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o);
        if (lane >= o) incl += y;
      }
      incl += carry;
      const unsigned long long past = __ballot(incl > i);
      if (past != 0ull) {
        const int l = (int)__builtin_ctzll(past);
        piece0 = __shfl(incl - c, l);
        return h + l;
      }
      carry = __shfl(incl, 63);
    }
    return -1;
  }
  // Every head's first piece and how many it has, for the sums' reduction (one
  // wave of a sequence's first block).
  __device__ void write(const TreeCall& a, const TreeSpan& sp, int lane, int2* table) const {
    int carry = 0;
    for (int h = 0; h < a.H; h += 64) {
      const int c = (units_of(a, sp, h + lane) + per - 1) / per;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o);
        if (lane >= o) incl += y;
      }
      incl += carry;
      if (h + lane < a.H) table[h + lane] = make_int2(incl - c, c);
      carry = __shfl(incl, 63);
    }
  }
};

// Block (x, y): piece x of sequence y, or all of head x.  The waves of a node
// tile take every WPT-th unit of it.
template <typename C, int D, int PARTS, int T>
__global__ __launch_bounds__(64 * kTreeWaves, tree_occupancy(D * (int)sizeof(C), PARTS * T)) void tree_kernel(TreeCall a) {
  using K = KeyRows<C, D>;
  using V = ValueRows<C, D>;
  using comp = typename K::comp;
  using frag = typename K::frag;
  using M = Mma<comp>;
  using Tile = typename V::Tile;
  constexpr int NDH = Tile::NDH, NC = Tile::NC;
  constexpr bool kTwo = sizeof(comp) == 2;
  constexpr int kRed = kUnit * V::DP * 4;   // a wave's sums of a node tile
  constexpr int kLds = kTreeWaves * (Tile::BYTES > T * kRed / 2 ? Tile::BYTES : T * kRed / 2);
  __shared__ __align__(16) char lds[kLds];
  __shared__ __align__(16) float kfac[kTreeWaves][kUnit], vfac[kTreeWaves][kUnit], mtab[kTreeWaves][128];
  __shared__ int dtab[kTreeWaves][kTreeMax];

  const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  // T = 1: the block's waves share its node tiles, wpt of them to each
  const int tiles = T == 2 ? 1 : (a.N + 31) / 32, wpt = kTreeWaves / tiles, tile = wave / wpt, kw = wave % wpt;
  const TreeSpan sp(a, b);
  int h = blockIdx.x, u0 = 0, per = 0;
  if (a.blocks != a.H) {
    const TreeMap map(a, sp, lane);
    int piece0 = 0;
    if (blockIdx.x == 0 && wave == 0) map.write(a, sp, lane, a.table + (int64_t)b * a.H);
    h = map.head_of(a, sp, lane, blockIdx.x, piece0);
    if (h < 0) return;
    per = map.per;
    u0 = ((int)blockIdx.x - piece0) * per;
  }
  const HeadParams hp = head_params(a.r, a.w, h, true);
  const int units = sp.units(a, hp.wc), lo_key = sp.lo(hp.wc);
  if (per == 0) per = units;
  const int u1 = u0 + per < units ? u0 + per : units;

  const int64_t kst = a.ks.st * (int64_t)sizeof(C), vst = a.vs.st * (int64_t)sizeof(C);
  const char* kb = (const char*)a.kc + (b * a.ks.sb + h * a.ks.sh) * (int64_t)sizeof(C) + lo_key * kst;
  const char* vb = (const char*)a.vc + (b * a.vs.sb + h * a.vs.sh) * (int64_t)sizeof(C) + lo_key * vst;
  const char* ksc = (const char*)(a.kscale + b * a.kss.sb + h * a.kss.sh + lo_key * a.kss.st);
  const char* vsc = (const char*)(a.vscale + b * a.vss.sb + h * a.vss.sh + lo_key * a.vss.st);
  const int last = sp.n + a.N - 1 - lo_key;  // last key row, from the window's first
  auto load_keys = [&](K& key, int u) {
    int r = perm_row(l32);
    const int lim = last - u * kUnit;
    if (lim < kUnit - 1) r = r < lim ? r : lim;
    key.load(kb + (int64_t)u * kUnit * kst, (uint32_t)r * (uint32_t)kst + half * K::LB,
             ksc + (int64_t)u * kUnit * a.kss.st * 4, (uint32_t)r * (uint32_t)(a.kss.st * 4));
  };
  // Keys are in flight a unit ahead; values are asked for once the vote has
  // found a live pair and arrive behind its weights.  (Asked for with the keys
  // where the last unit was live, they cost registers: 4 x 64 nodes over 30K bf16
  // 106 instead of 70 us, chain of 8 over 16K int8 53 instead of 50.)
  K key_next;
  if (u0 + kw < u1) load_keys(key_next, u0 + kw);

  const Tree tree(a.parents == nullptr ? nullptr : a.parents + b * a.par_sb, a.N, lane);
  dtab[wave][lane] = tree.depth;
  int node[T], depth[T];
  unsigned long long above[T];
  NodeRows<C, D, PARTS> q[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    node[t] = 32 * (T == 2 ? t : tile) + l32;
    depth[t] = __shfl(tree.depth, node[t]);
    above[t] = ((unsigned long long)(uint32_t)__shfl((int)(tree.above >> 32), node[t]) << 32) |
               (uint32_t)__shfl((int)tree.above, node[t]);
    const bool ok = node[t] < a.N;
    const int64_t off = b * a.q_sb + (int64_t)(ok ? node[t] : 0) * a.q_sn + h * a.q_sh;
    if (a.q_dtype == 1) q[t].load((const bf16*)a.q + off, ok, a.eps, half);
    else if (a.q_dtype == 2) q[t].load((const f16*)a.q + off, ok, a.eps, half);
    else q[t].load((const float*)a.q + off, ok, a.eps, half);
  }

  char* vt = lds + wave * Tile::BYTES;
  if constexpr (D < V::DP) {  // the columns past D
#pragma unroll
    for (int i = 0; i < Tile::BYTES / 1024; ++i)
      *reinterpret_cast<u32x4*>(vt + i * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
  }
  const uint32_t cbase = Tile::col_base(lane);
  f32x16 acc[T][NDH];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int d = 0; d < NDH; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][d][r] = 0.0f;

  const int depth_max = a.parents == nullptr ? a.N - 1 : wave_max(tree.depth);
  for (int u = u0 + kw; u < u1; u += wpt) {
    const int k0 = lo_key + u * kUnit;  // position of the unit's first row (a drafted row: n + its node)
    const K key = key_next;
    if (u + wpt < u1) load_keys(key_next, u + wpt);
    frag kf[K::NKS];
    key.frags(kf);
    const float f = key.factor(kf, a.eps, a.inv_eps);
    if (half == 0) kfac[wave][perm_row(l32)] = f;
    f32x16 s[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      s[t] = unit_product<comp, K::NKS>(kf, q[t].f[0]);
      if constexpr (PARTS == 2) {
        const f32x16 s2 = unit_product<comp, K::NKS>(kf, q[t].f[1]);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] += s2[r];
      }
    }
    guard_all(kf, s[T - 1]);
    wave_lds_sync();
    float x[16];
    read_row_scales(kfac[wave], half, x);
    bool vote = false;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] *= x[r];
        top = fmaxf(top, s[t][r]);
      }
      vote = vote || top * q[t].inv > hp.thr;
    }
    if (__ballot(vote) == 0ull) continue;
    V val;
    load_values_at<C, D>(val, vb, vst, vsc, a.vss.st, u, last, lane);

    // a^2 m of every pair: register r is key row 16 (r/8) + 8 half + r%8 (the
    // clamp takes a NaN to 0)
    float any = 0.0f;
    if (k0 + kUnit <= sp.n) {
      // committed keys: m from a table over depth - row (entry e: distance n - k0 - 31 + e)
      const int dmin = sp.n - k0 - 31;
      for (int e = lane; e < 32 + depth_max; e += 64)
        mtab[wave][e] = in_window(dmin + e, hp) ? mask_fast(dmin + e, hp.w, hp.iw) : 0.0f;
      wave_lds_sync();
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float* mt = mtab[wave] + (depth[t] + 8 - 8 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float av = __builtin_amdgcn_fmed3f(fmaf(-hp.r, fmaf(-s[t][r], q[t].inv, 1.0f), 1.0f), 0.0f, 1.0f);
          s[t][r] = av * av * mt[23 - 16 * (r >> 3) - (r & 7)];
          any = fmaxf(any, s[t][r]);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 16 * (r >> 3) + 8 * half + (r & 7), j = k0 + row - sp.n;  // j >= 0: drafted
          const bool draft = j >= 0;
          const int dd = depth[t] - (draft ? dtab[wave][j & (kTreeMax - 1)] : j);
          const bool seen = draft ? j < a.N && ((above[t] >> (j & 63)) & 1ull) != 0ull : true;
          const float av = __builtin_amdgcn_fmed3f(fmaf(-hp.r, fmaf(-s[t][r], q[t].inv, 1.0f), 1.0f), 0.0f, 1.0f);
          s[t][r] = seen && in_window(dd, hp) ? av * av * mask_fast(dd, hp.w, hp.iw) : 0.0f;
          any = fmaxf(any, s[t][r]);
        }
    }
    if (__ballot(any > 0.0f) == 0ull) continue;

    const bool odd = val.stage(vt, vfac[wave], a.eps, a.inv_eps, lane);
    wave_lds_sync();
    read_row_scales(vfac[wave], half, x);
    frag hi[T][NC], lo[T][kTwo ? NC : 1];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (odd) {  // a NaN factor reaches live pairs only
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = s[t][r] > 0.0f ? s[t][r] * x[r] : 0.0f;
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] *= x[r];
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        hi[t][c] = M::pack(s[t], M::PER * c);
        // one rounding for both uses below: formed anew from the factors it may be
        // rounded once instead of twice, and the second term would not be its rest
        asm volatile("" : "+v"(hi[t][c]));
      }
      if constexpr (kTwo) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
          for (int e = 0; e < M::PER; ++e) s[t][M::PER * c + e] -= M::get(hi[t][c], e);
          lo[t][c] = M::pack(s[t], M::PER * c);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < NDH; ++d) {
      frag vf[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) vf[c] = Tile::col_frag(vt, cbase, d, c);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t][d] = M::mma_ng(vf[c], hi[t][c], acc[t][d]);
      if constexpr (kTwo) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int t = 0; t < T; ++t) acc[t][d] = M::mma_ng(vf[c], lo[t][c], acc[t][d]);
      }
#pragma unroll
      for (int t = 0; t < T; ++t) guard_all(vf, acc[t][d]);
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      guard_all(hi[t], acc[t][NDH - 1]);
      if constexpr (kTwo) guard_all(lo[t], acc[t][NDH - 1]);
    }
  }

  // the waves of a tile, the upper half of them into the lower, until one has all
  for (int step = wpt / 2; step >= 1; step /= 2) {
    char* red = lds + (tile * step + kw % step) * (T * kRed) + lane * 16;
    __syncthreads();
    if (kw >= step && kw < 2 * step) {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int d = 0; d < NDH; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(red + ((t * NDH + d) * 4 + g) * 1024) =
                f32x4{acc[t][d][4 * g], acc[t][d][4 * g + 1], acc[t][d][4 * g + 2], acc[t][d][4 * g + 3]};
    }
    __syncthreads();
    if (kw < step) {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int d = 0; d < NDH; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(red + ((t * NDH + d) * 4 + g) * 1024);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][d][4 * g + e] += y[e];
          }
    }
  }
  if (kw != 0) return;
  constexpr float down = 1.0f / kWeightUp<C>;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    if (node[t] >= a.N) continue;  // lanes l and l + 32 share a node
    if (a.blocks != a.H) {
      float* p = a.part + (((int64_t)b * a.blocks + blockIdx.x) * a.N + node[t]) * D;
      store_row<comp, float, D>(p, half, [&](int d, int r) { return acc[t][d][r] * down; });
      continue;
    }
    float ss = 0.0f;
#pragma unroll
    for (int d = 0; d < NDH; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[t][d][r] *= down;
        ss = fmaf(acc[t][d][r], acc[t][d][r], ss);
      }
    const float nc = fmaxf(sqrtf(half_sum(ss)), a.eps), fy = tanhf(nc) / nc;
    store_row_as<comp, D>(a.y, (((int64_t)b * a.N + node[t]) * a.H + h) * D, a.q_dtype, half,
                          [&](int d, int r) { return acc[t][d][r] * fy; });
  }
}

// ---------------------------------------------------------------------------
// Trees of at most 16 nodes: the same walk on the 16x16x32 product, whose block
// of 16 columns halves the per-pair work (and the sums' registers) that 32
// columns would spend on absent nodes.  2-byte operands only.
//
//   Operands: lane l supplies row (A) / column (B) l%16 and the 8 contraction
//   slots of group l/16.  C block: lane l, register r -> row 4 (l/16) + r, column
//   l%16.
// A unit's keys are two row blocks t; block row m holds unit row 8 (m/4) + 4 t +
// m%4, so that a lane's registers (t, r) are unit rows 8 (l/16) + 4 t + r: the
// eight slots it supplies to the value product.  The value columns of block d
// likewise: row m holds column 32 (d/2) + 8 (m/4) + 4 (d%2) + m%4, and a lane's
// registers of two blocks are 8 consecutive columns.
// ---------------------------------------------------------------------------
template <typename T> struct Mma16;
template <> struct Mma16<bf16> {
  __device__ static inline f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma16<f16> {
  __device__ static inline f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <typename F, int N>
__device__ inline void guard_all16(const F (&f)[N], const f32x4& c) {
  asm volatile(MSA_NOP16 ::"v"(c[3]));
#pragma unroll
  for (int k = 0; k < N; ++k) asm volatile("" ::"v"(f[k]));
}
// Sum over the four lanes l%16 + 16 i.
__device__ inline float quarter_sum(float x) { return half_sum(x + __shfl_xor(x, 16)); }
__device__ inline float quarter_max(float x) { return half_max(fmaxf(x, __shfl_xor(x, 16))); }

template <typename C, int D>
struct KeyRows16 {
  using comp = typename TreeRow<C>::comp;
  typedef typename Mma<comp>::frag frag;
  static constexpr bool kCodes = TreeRow<C>::kCodes;
  static constexpr int NKS = D < 32 ? 1 : D / 32;
  static constexpr int LB = kCodes && D <= 32 ? 8 : 16;                      // bytes of a load
  static constexpr int NL = D < 32 ? 1 : D * (int)sizeof(C) / (4 * LB);      // loads of a lane and block
  static constexpr bool kHalf = D < 32;                                      // groups 2, 3 hold no columns
  u32x4 raw[2][NL];
  float scale[2];

  __device__ static inline int row(int t, int lane) { return 8 * ((lane & 15) >> 2) + 4 * t + (lane & 3); }
  __device__ static constexpr int col(int ks, int g) {
    if constexpr (kCodes && D >= 64) return 64 * (ks / 2) + 16 * g + 8 * (ks & 1);
    else return 32 * ks + 8 * (kHalf ? g & 1 : g);
  }
  // `off[t]`: block t's row of this lane and its group's first bytes.
  __device__ inline void load(const char* rows, const uint32_t (&off)[2], const char* scales, const uint32_t (&soff)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const char* p = rows + off[t] + 4 * i * LB;
        if constexpr (LB == 8) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p);
          raw[t][i] = u32x4{x[0], x[1], 0u, 0u};
        } else {
          raw[t][i] = *reinterpret_cast<const u32x4*>(p);
        }
      }
      if constexpr (kCodes) scale[t] = *reinterpret_cast<const float*>(scales + soff[t]);
    }
  }
  __device__ inline void frags(int t, int lane, frag (&f)[NKS]) const {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      if constexpr (!kCodes) f[ks] = __builtin_bit_cast(frag, raw[t][ks]);
      else if constexpr (D >= 64) f[ks] = decode8<C>(raw[t][ks / 2][2 * (ks & 1)], raw[t][ks / 2][2 * (ks & 1) + 1]);
      else f[ks] = decode8<C>(raw[t][0][0], raw[t][0][1]);
      if (kHalf && lane >= 32) f[ks] = Mma<comp>::zero();
    }
  }
  __device__ inline float factor(int t, const frag (&f)[NKS], float eps, float inv_eps) const {
    float ss = 0.0f;
    if constexpr (__is_same(C, int8_t)) {
      int si = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) si += code_dot<LB / 4>(raw[t][i]);
      ss = kHalf && (threadIdx.x & 32) != 0 ? 0.0f : (float)si;
    } else {
      ss = row_dot<comp>(f, f);
    }
    ss = quarter_sum(ss);
    if constexpr (kCodes) return KeyRows<C, D>::code_factor(ss, scale[t], inv_eps);
    else return inv_len_of<C>(ss, eps);
  }
};

template <typename C, int D, int PARTS>
struct NodeRows16 {
  using K = KeyRows16<C, D>;
  typename K::frag f[PARTS][K::NKS];
  float inv;
  template <typename T>
  __device__ inline void load(const T* row, bool ok, float eps, int g) {
    constexpr int VEC = 16 / (int)sizeof(T);
    float x[K::NKS][8];
    float ss = 0.0f, mx = 0.0f;
    ok = ok && !(K::kHalf && g >= 2);
#pragma unroll
    for (int ks = 0; ks < K::NKS; ++ks)
#pragma unroll
      for (int e0 = 0; e0 < 8; e0 += VEC) {
        typedef __attribute__((__vector_size__(16))) T vec;
        const vec v = *reinterpret_cast<const vec*>(row + K::col(ks, g) + e0);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[ks][e0 + e] = ok ? to_f(v[e]) : 0.0f;
      }
#pragma unroll
    for (int ks = 0; ks < K::NKS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(x[ks][e], x[ks][e], ss);
        mx = fmaxf(mx, fabsf(x[ks][e]));
      }
    const float p = TreeRow<C>::kCodes ? row_pow2(quarter_max(mx)) : 1.0f;
    inv = inv_len_of<float>(quarter_sum(ss), eps) / p;
#pragma unroll
    for (int ks = 0; ks < K::NKS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float rest = x[ks][e] * p;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const auto part = from_f<typename K::comp>(rest);
          f[i][ks][e] = part;
          rest -= to_f(part);
        }
      }
  }
};

template <typename C, int D, int PARTS>
__global__ __launch_bounds__(64 * kTreeWaves, tree_occupancy16(D * (int)sizeof(C), PARTS)) void tree16_kernel(TreeCall a) {
  using K = KeyRows16<C, D>;
  using V = ValueRows<C, D>;
  using comp = typename K::comp;
  using frag = typename K::frag;
  using Tile = typename V::Tile;
  constexpr int NDT = V::DP / 16;
  constexpr int kRed = NDT * 1024;
  constexpr int kLds = kTreeWaves * (Tile::BYTES > kRed / 2 ? Tile::BYTES : kRed / 2);
  __shared__ __align__(16) char lds[kLds];
  __shared__ __align__(16) float kfac[kTreeWaves][kUnit], vfac[kTreeWaves][kUnit], mtab[kTreeWaves][64];
  __shared__ int dtab[kTreeWaves][kTreeMax];

  const int lane = threadIdx.x & 63, g = lane >> 4, node = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  const TreeSpan sp(a, b);
  int h = blockIdx.x, u0 = 0, per = 0;
  if (a.blocks != a.H) {
    const TreeMap map(a, sp, lane);
    int piece0 = 0;
    if (blockIdx.x == 0 && wave == 0) map.write(a, sp, lane, a.table + (int64_t)b * a.H);
    h = map.head_of(a, sp, lane, blockIdx.x, piece0);
    if (h < 0) return;
    per = map.per;
    u0 = ((int)blockIdx.x - piece0) * per;
  }
  const HeadParams hp = head_params(a.r, a.w, h, true);
  const int units = sp.units(a, hp.wc), lo_key = sp.lo(hp.wc);
  if (per == 0) per = units;
  const int u1 = u0 + per < units ? u0 + per : units;

  const int64_t kst = a.ks.st * (int64_t)sizeof(C), vst = a.vs.st * (int64_t)sizeof(C);
  const char* kb = (const char*)a.kc + (b * a.ks.sb + h * a.ks.sh) * (int64_t)sizeof(C) + lo_key * kst;
  const char* vb = (const char*)a.vc + (b * a.vs.sb + h * a.vs.sh) * (int64_t)sizeof(C) + lo_key * vst;
  const char* ksc = (const char*)(a.kscale + b * a.kss.sb + h * a.kss.sh + lo_key * a.kss.st);
  const char* vsc = (const char*)(a.vscale + b * a.vss.sb + h * a.vss.sh + lo_key * a.vss.st);
  const int last = sp.n + a.N - 1 - lo_key;  // last key row, from the window's first
  auto load_keys = [&](K& key, int u) {
    const int lim = last - u * kUnit;
    uint32_t off[2], soff[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int r = K::row(t, lane);
      if (lim < kUnit - 1) r = r < lim ? r : lim;
      off[t] = (uint32_t)r * (uint32_t)kst + (K::kHalf ? g & 1 : g) * K::LB;
      soff[t] = (uint32_t)r * (uint32_t)(a.kss.st * 4);
    }
    key.load(kb + (int64_t)u * kUnit * kst, off, ksc + (int64_t)u * kUnit * a.kss.st * 4, soff);
  };
  K key_next;
  if (u0 + wave < u1) load_keys(key_next, u0 + wave);

  const Tree tree(a.parents == nullptr ? nullptr : a.parents + b * a.par_sb, a.N, lane);
  dtab[wave][lane] = tree.depth;
  const int depth = __shfl(tree.depth, node);
  const uint32_t above = (uint32_t)__shfl((int)tree.above, node);
  NodeRows16<C, D, PARTS> q;
  {
    const bool ok = node < a.N;
    const int64_t off = b * a.q_sb + (int64_t)(ok ? node : 0) * a.q_sn + h * a.q_sh;
    if (a.q_dtype == 1) q.load((const bf16*)a.q + off, ok, a.eps, g);
    else if (a.q_dtype == 2) q.load((const f16*)a.q + off, ok, a.eps, g);
    else q.load((const float*)a.q + off, ok, a.eps, g);
  }
  char* vt = lds + wave * Tile::BYTES;
  if constexpr (D < V::DP) {  // the columns past D
#pragma unroll
    for (int i = 0; i < Tile::BYTES / 1024; ++i)
      *reinterpret_cast<u32x4*>(vt + i * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
  }
  // value column operands: a 16-lane group transposes 4 rows x 16 columns; lane
  // 4 k + q gives row k's columns 8 q + 4 (d%2) .. of block d
  const int cr = 8 * g + ((lane & 15) >> 2), cq = lane & 3;
  const uint32_t cbase = (uint32_t)(cr * Tile::ROWB + ((cq ^ Tile::swz(cr)) << 4));
  auto value_frag = [&](int d) {
    typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
    typedef __attribute__((__vector_size__(8 * sizeof(short)))) short s16x8;
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* p = vt + (cbase ^ (uint32_t)((Tile::swz(4 * j) ^ (4 * (d >> 1))) << 4)) + 4 * j * Tile::ROWB + 8 * (d & 1);
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)const_cast<char*>(p));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * j + e] = x[e];
    }
    return __builtin_bit_cast(frag, v);
  };
  f32x4 acc[NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int depth_max = a.parents == nullptr ? a.N - 1 : wave_max(tree.depth);

  for (int u = u0 + wave; u < u1; u += kTreeWaves) {
    const int k0 = lo_key + u * kUnit;
    const K key = key_next;
    if (u + kTreeWaves < u1) load_keys(key_next, u + kTreeWaves);
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      frag kf[K::NKS];
      key.frags(t, lane, kf);
      const float f = key.factor(t, kf, a.eps, a.inv_eps);
      if (g == 0) kfac[wave][K::row(t, lane)] = f;
      f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = PARTS - 1; i >= 0; --i)
#pragma unroll
        for (int ks = 0; ks < K::NKS; ++ks) c = Mma16<comp>::mma(kf[ks], q.f[i][ks], c);
      guard_all16(kf, c);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * t + r] = c[r];
    }
    wave_lds_sync();
    float x[8];
    auto read8 = [&](const float* p) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(p + 8 * g + 4 * t);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[4 * t + r] = v[r];
      }
    };
    read8(kfac[wave]);
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      s[r] *= x[r];
      top = fmaxf(top, s[r]);
    }
    if (__ballot(top * q.inv > hp.thr) == 0ull) continue;
    V val;
    load_values_at<C, D>(val, vb, vst, vsc, a.vss.st, u, last, lane);

    float any = 0.0f;
    if (k0 + kUnit <= sp.n) {
      const int dmin = sp.n - k0 - 31, e = lane;  // entries 0 .. 31 + 15
      if (e < 32 + depth_max) mtab[wave][e] = in_window(dmin + e, hp) ? mask_fast(dmin + e, hp.w, hp.iw) : 0.0f;
      wave_lds_sync();
      const float* mt = mtab[wave] + (depth + 24 - 8 * g);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float av = __builtin_amdgcn_fmed3f(fmaf(-hp.r, fmaf(-s[r], q.inv, 1.0f), 1.0f), 0.0f, 1.0f);
        s[r] = av * av * mt[7 - r];
        any = fmaxf(any, s[r]);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int j = k0 + 8 * g + r - sp.n;  // j >= 0: drafted
        const bool draft = j >= 0;
        const int dd = depth - (draft ? dtab[wave][j & (kTreeMax - 1)] : j);
        const bool seen = draft ? j < a.N && ((above >> (j & 31)) & 1u) != 0u : true;
        const float av = __builtin_amdgcn_fmed3f(fmaf(-hp.r, fmaf(-s[r], q.inv, 1.0f), 1.0f), 0.0f, 1.0f);
        s[r] = seen && in_window(dd, hp) ? av * av * mask_fast(dd, hp.w, hp.iw) : 0.0f;
        any = fmaxf(any, s[r]);
      }
    }
    if (__ballot(any > 0.0f) == 0ull) continue;

    const bool odd = val.stage(vt, vfac[wave], a.eps, a.inv_eps, lane);
    wave_lds_sync();
    read8(vfac[wave]);
    if (odd) {  // a NaN factor reaches live pairs only
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = s[r] > 0.0f ? s[r] * x[r] : 0.0f;
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] *= x[r];
    }
    frag w[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[0][e] = from_f<comp>(s[e]);
    asm volatile("" : "+v"(w[0]));  // one rounding for both its uses (tree_kernel)
#pragma unroll
    for (int e = 0; e < 8; ++e) w[1][e] = from_f<comp>(s[e] - to_f(w[0][e]));
    frag vf[NDT];
#pragma unroll
    for (int d = 0; d < NDT; ++d) vf[d] = value_frag(d);
#pragma unroll
    for (int d = 0; d < NDT; ++d) acc[d] = Mma16<comp>::mma(vf[d], w[0], acc[d]);
#pragma unroll
    for (int d = 0; d < NDT; ++d) acc[d] = Mma16<comp>::mma(vf[d], w[1], acc[d]);
    guard_all16(vf, acc[NDT - 1]);
    guard_all16(w, acc[NDT - 1]);
  }

  // the waves' sums, the upper half of them into the lower, until one has all
  for (int step = kTreeWaves / 2; step >= 1; step /= 2) {
    char* red = lds + (wave % step) * kRed + lane * 16;
    __syncthreads();
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int d = 0; d < NDT; ++d) *reinterpret_cast<f32x4*>(red + d * 1024) = acc[d];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(red + d * 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[d][e] += y[e];
      }
    }
  }
  if (wave != 0) return;
  constexpr float down = 1.0f / kWeightUp<C>;
  float fy = down;
  if (a.blocks == a.H) {
    float ss = 0.0f;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) ss = fmaf(acc[d][r] * down, acc[d][r] * down, ss);
    const float nc = fmaxf(sqrtf(quarter_sum(ss)), a.eps);
    fy = down * (tanhf(nc) / nc);
  }
  if (node >= a.N) return;
  auto store = [&](auto* row) {
#pragma unroll
    for (int j = 0; j < NDT / 2; ++j) {
      const int d0 = 32 * j + 8 * g;
      if (d0 < D) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = acc[2 * j][r] * fy;
          v[4 + r] = acc[2 * j + 1][r] * fy;
        }
        store8(row + d0, v);
      }
    }
  };
  if (a.blocks != a.H) {
    store(a.part + (((int64_t)b * a.blocks + blockIdx.x) * a.N + node) * D);
    return;
  }
  const int64_t at = (((int64_t)b * a.N + node) * a.H + h) * D;
  if (a.q_dtype == 1) store((bf16*)a.y + at);
  else if (a.q_dtype == 2) store((f16*)a.y + at);
  else store((float*)a.y + at);
}

// Sum of a node's block sums and TanhNorm: a wave per node, D/4 lanes for a
// block's sums and 256/D blocks at a time.
template <int D>
__global__ __launch_bounds__(256) void tree_reduce_kernel(TreeCall a) {
  constexpr int L = D / 4, G = 64 / L;
  const int lane = threadIdx.x & 63, node = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int b = blockIdx.y / a.H, h = blockIdx.y % a.H;
  if (node >= a.N) return;
  const int2 at_pieces = a.table[blockIdx.y];  // first piece of the head, and how many
  const int used = at_pieces.y;
  const float* p = a.part + (((int64_t)b * a.blocks + at_pieces.x) * a.N + node) * D + 4 * (lane % L);
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int c = lane / L; c < used; c += G) x += *reinterpret_cast<const f32x4*>(p + (int64_t)c * a.N * D);
#pragma unroll
  for (int o = L; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o);
  const float ss = group_sum<L>(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
  const float nc = fmaxf(sqrtf(ss), a.eps), fy = tanhf(nc) / nc;
  if (lane >= L) return;
  const int64_t at = (((int64_t)b * a.N + node) * a.H + h) * D + 4 * lane;
  if (a.q_dtype == 1) store4((bf16*)a.y + at, x[0] * fy, x[1] * fy, x[2] * fy, x[3] * fy);
  else if (a.q_dtype == 2) store4((f16*)a.y + at, x[0] * fy, x[1] * fy, x[2] * fy, x[3] * fy);
  else store4((float*)a.y + at, x[0] * fy, x[1] * fy, x[2] * fy, x[3] * fy);
}

// Whether a wave takes all of more than 32 nodes: its registers hold two tiles'
// operands and sums for rows of at most 64 values in 2-byte operands.  A wave a
// tile converts, votes on and stages every unit twice: 4 x 64 nodes over 30K bf16
// 88 us, together 75; before training 48, together 42.
bool tree_both(int N, int D, bool f32) { return N > 32 && D <= 64 && !f32; }
// Whether a tree takes the 16-column form: 8 nodes over 16K int8 49 -> 46 us, fp32
// queries 53 -> 45 (D = 128: 85 -> 71), one node at windows 2 .. 256 10.1 -> 8.6,
// 16 nodes over 8K bf16 of D = 128 61 -> 59; one node over 100K int8, which its
// bytes bound, the same.  (The transposed reads of natural column blocks, 16 d +
// 0 .. 15, spread over twice the banks and were no faster.)
bool tree_few(int N, bool f32_operands) { return N <= 16 && !f32_operands; }
// Blocks of a sequence: as many as run at one time on the card's 256 CUs by the
// waves budgeted above (more fit of some instances) share its heads' keys; one a head (H) where heads are short, or the batch alone
// fills the card several times over with heads that are not long.
int tree_blocks(int B, int H, int N, int D, int q_dtype, int cache_dtype, int span) {
  const int64_t units = ((int64_t)span + N + kUnit - 1) / kUnit;
  const bool codes = cache_dtype == kInt8 || cache_dtype == kFp8;
  const int row = D * (codes ? 1 : cache_dtype == 0 ? 4 : 2);
  const bool f32 = codes ? q_dtype == 0 : cache_dtype == 0;
  const int parts = codes && q_dtype == 0 ? 2 : 1;
  const int slots = 256 * (tree_few(N, !codes && f32) ? tree_occupancy16(row, parts)
                                                      : tree_occupancy(row, tree_both(N, D, f32) ? 2 : parts));
  if (units <= kTreeSmall || ((int64_t)B * H >= 2 * slots && units <= kTreeLong)) return H;
  const int each = slots / B;
  return each < 2 * H ? 2 * H : each;
}

template <typename C, int D, int PARTS, int T>
static hipError_t launch_tree_t(const TreeCall& c) {
  const dim3 grid((unsigned)c.blocks, (unsigned)c.B), block(64 * kTreeWaves);
  if constexpr (T == 0) hipLaunchKernelGGL((tree16_kernel<C, D, PARTS>), grid, block, 0, c.stream, c);
  else hipLaunchKernelGGL((tree_kernel<C, D, PARTS, T>), grid, block, 0, c.stream, c);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || c.blocks == c.H) return e;
  hipLaunchKernelGGL((tree_reduce_kernel<D>), dim3((unsigned)((c.N + 3) / 4), (unsigned)(c.B * c.H)), dim3(256), 0, c.stream, c);
  return hipGetLastError();
}
template <typename C, int D, int PARTS>
static hipError_t launch_tree_n(const TreeCall& c) {
  constexpr bool f32 = PARTS == 2 || __is_same(C, float);
  if constexpr (!__is_same(C, float))
    if (tree_few(c.N, false)) return launch_tree_t<C, D, PARTS, 0>(c);
  if constexpr (D <= 64 && !f32)
    if (tree_both(c.N, D, f32)) return launch_tree_t<C, D, PARTS, 2>(c);
  return launch_tree_t<C, D, PARTS, 1>(c);
}
template <typename C, int PARTS>
static hipError_t launch_tree_d(const TreeCall& c) {
  switch (c.D) {
    case 16: return launch_tree_n<C, 16, PARTS>(c);
    case 32: return launch_tree_n<C, 32, PARTS>(c);
    case 64: return launch_tree_n<C, 64, PARTS>(c);
    default: return launch_tree_n<C, 128, PARTS>(c);
  }
}
hipError_t launch_tree(const TreeCall& c) {
  // an fp32 query over codes is two fp16 rows
  if (c.cache_dtype == kInt8) return c.q_dtype == 0 ? launch_tree_d<int8_t, 2>(c) : launch_tree_d<int8_t, 1>(c);
  if (c.cache_dtype == kFp8) return c.q_dtype == 0 ? launch_tree_d<fp8, 2>(c) : launch_tree_d<fp8, 1>(c);
  if (c.cache_dtype == 1) return launch_tree_d<bf16, 1>(c);
  if (c.cache_dtype == 2) return launch_tree_d<f16, 1>(c);
  return launch_tree_d<float, 1>(c);
}

}  // namespace msa

// Key/value cache rows: written in the model's type or as 8-bit codes with one
// scale per row, and read back (gfx950).
//
// A quantised row x of D values is kept as D codes and the fp32 scale A/TOP,
// A = max|x| and TOP the type's largest code (127; 448 for e4m3).  A code is the
// nearest one to TOP x / A, ties to the even one, exactly (codes_of).  So
// the codes depend on nothing but the row: a row written twice, or moved, has
// the same codes.  A row of zeros has scale 0; a row that holds an infinity or
// a NaN has scale NaN and codes 0, and reads back as NaN.
//
// Both kernels are bound by their bytes (a row in its type and its D + 4 bytes
// of code and scale); D/VEC lanes share a row (16 bytes of it each), so the row
// is read once, its maximum is a lane-group reduction and nothing is staged.
// 4 x 8192 x 8 rows of k and v, D = 64 bf16 to int8: written in 23 us (4.4 TB/s),
// read back in 18 (5.7 TB/s; a large copy reaches 4.95).
// The rows of a block are consecutive positions of one head, whose codes are
// contiguous in head-major storage.
#include "msa_device.h"
#include "msa_internal.h"

namespace msa {

// 16 bytes of a row in its type.
template <typename T> struct RowVec;
template <> struct RowVec<bf16> { typedef bf16x8 type; static constexpr int N = 8; };
template <> struct RowVec<f16> { typedef f16x8 type; static constexpr int N = 8; };
template <> struct RowVec<float> { typedef f32x4 type; static constexpr int N = 4; };

// The largest x of aligned groups of G lanes (non-negative integers).
template <int G>
__device__ inline uint32_t group_max_u32(uint32_t x) {
#pragma unroll
  for (int o = 1; o < G; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, o);
    x = y > x ? y : x;
  }
  return x;
}

template <typename C> struct CodeTop { static constexpr float v = 1.0f; };
template <> struct CodeTop<int8_t> { static constexpr float v = 127.0f; };
template <> struct CodeTop<fp8> { static constexpr float v = 448.0f; };

// The code of x in a row of largest magnitude `top`, by 64 bits.
template <typename C>
__device__ inline uint32_t exact_code(float x, float top) {
  const double d = (double)CodeTop<C>::v * (double)x / (double)top;
  if constexpr (__is_same(C, int8_t)) {
    return (uint32_t)(int)rint(d) & 0xffu;
  } else {
    // rounded to odd on the way to fp32, so that the second rounding sees on
    // which side of a border the quotient lies
    float f = (float)d;
    if ((double)f != d) {
      uint32_t b = __float_as_uint(f);
      if (fabs((double)f) > fabs(d)) b -= 1u;
      f = __uint_as_float(b | 1u);
    }
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false) & 0xffu;
  }
}

// The codes nearest to x f, four to a word.  int8 rounds in the addition of
// 1.5 2^23 (the sum's low byte is the code).
__device__ inline uint32_t codes4(const float* x, float f, int8_t) {
  constexpr float magic = 12582912.0f;
  const uint32_t a = __float_as_uint(fmaf(x[0], f, magic)), b = __float_as_uint(fmaf(x[1], f, magic));
  const uint32_t c = __float_as_uint(fmaf(x[2], f, magic)), d = __float_as_uint(fmaf(x[3], f, magic));
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                               0x05040100u);
}
__device__ inline uint32_t codes4(const float* x, float f, fp8) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * f, x[1] * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * f, x[3] * f, lo, true);
}

// Codes of N values of a row of largest magnitude `top`, of type T.
//
// The quotient TOP x / top lies between x inv (1 - 2^-21) and x inv (1 + 2^-21),
// inv = TOP/top in fp32; where both ends have one code, it is the quotient's.
// Else fp32 rows take 64 bits.  2-byte rows have X 2^i and P 2^j for x and top
// with X, P < 2^11, and TOP = N 2^n (N = 127 or 7): a quotient that is not on a
// border M 2^m (M < 2^8, or 2^5) is at least 1/(M P) or 1/(N X) > 2^-19 of it
// away, so the fp32 quotient, rounded once, decides.
//
// int8 codes of 2-byte rows need only the upper end: 2^-21 crosses no border,
// and of those hit exactly, 63.5 (x = top/2, in every sixth row of 64 values)
// goes up to the even 64.  Others, (n + 1/2) P = 127 X 2^k, need a P that 127
// divides: such rows take the quotient.
template <typename T, typename C, int N>
__device__ inline void codes_of(const float (&x)[N], float top, uint32_t (&code)[N / 4]) {
  const float inv = CodeTop<C>::v / top;
  constexpr float e = 4.76837158203125e-7f;  // 2^-21
  const float lo = fmaf(-e, inv, inv), hi = fmaf(e, inv, inv);
  bool differ = false;
#pragma unroll
  for (int w = 0; w < N / 4; ++w) code[w] = codes4(x + 4 * w, hi, C{});
  if constexpr (sizeof(T) == 2 && __is_same(C, int8_t)) {
    differ = ((__float_as_uint(top) & 0x7fffffu) | 0x800000u) % 127u == 0u;
  } else {
#pragma unroll
    for (int w = 0; w < N / 4; ++w) differ = differ || code[w] != codes4(x + 4 * w, lo, C{});
  }
  if (!differ) return;
#pragma unroll
  for (int w = 0; w < N / 4; ++w) {
    if constexpr (sizeof(T) == 2) {
      float q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = CodeTop<C>::v * x[4 * w + k] / top;
      code[w] = codes4(q, 1.0f, C{});
    } else {
      code[w] = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) code[w] |= exact_code<C>(x[4 * w + k], top) << (8 * k);
    }
  }
}

// Values of four codes.
__device__ inline void decode4(uint32_t c, float (&v)[4], int8_t) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)(int8_t)(c >> (8 * e));
}
__device__ inline void decode4(uint32_t c, float (&v)[4], fp8) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
}

// Cache position of row t of sequence b, or -1 if it lies outside the cache.
__device__ inline int cache_position(const CacheCall& a, int b, int t) {
  int64_t s = a.start != nullptr ? a.start[(int64_t)b * a.start_step] : a.start0;
  if (s < -(int64_t)a.T || s >= (int64_t)a.cap) return -1;
  s += t;
  return s >= 0 && s < a.cap ? (int)s : -1;
}

// Block (x, y): rows x 256/LPR, ... of head y = b H + h, of k and of v: their
// loads are in flight together and the positions are found once.  (Blocks over
// several heads of the same positions, so that each reads whole lines of a
// stacked projection, were no faster.)
template <typename T, typename C, int D>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheCall a) {
  using vec = typename RowVec<T>::type;
  constexpr int VEC = RowVec<T>::N, LPR = D / VEC;
  const int b = blockIdx.y / a.H, h = blockIdx.y % a.H;
  const int t = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, d0 = (threadIdx.x % LPR) * VEC;
  int64_t src = t;
  int pos = -1;
  if (t < a.T && (a.count == nullptr || t < a.count[b])) {
    if (a.rows != nullptr) src = a.rows[(int64_t)b * a.T + t];
    if (src >= 0 && src < a.Tx) pos = cache_position(a, b, t);
  }
  vec x[2];
#pragma unroll
  for (int z = 0; z < 2; ++z) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[z][e] = from_f<T>(0.0f);
    const Strides3 xs = a.xs[z];
    if (pos >= 0) x[z] = *reinterpret_cast<const vec*>((const T*)a.x[z] + b * xs.sb + src * xs.st + h * xs.sh + d0);
  }
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const Strides3 cs = a.cs[z], ss = a.ss[z];
    char* row = (char*)a.c[z] + (b * cs.sb + (int64_t)pos * cs.st + h * cs.sh + d0) * (int64_t)sizeof(C);
    if constexpr (sizeof(C) > 1) {
      if (pos >= 0) *reinterpret_cast<vec*>(row) = x[z];
    } else {
      uint32_t m = 0u;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t y = __float_as_uint(to_f(x[z][e])) & 0x7fffffffu;
        m = y > m ? y : m;
      }
      m = group_max_u32<LPR>(m);  // a NaN's magnitude is above an infinity's
      if (pos < 0) continue;
      const bool finite = m < 0x7f800000u;
      const float top = __uint_as_float(m);
      uint32_t code[VEC / 4] = {};
      if (finite && m != 0u) {
        // below 2^-118 TOP/top may leave fp32's range: scaled by a power of two
        const float up = m < 0x04800000u ? 1.0633823966279327e37f : 1.0f;  // 2^123
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = to_f(x[z][e]) * up;
        codes_of<T, C, VEC>(f, top * up, code);
      }
      if constexpr (VEC == 8) *reinterpret_cast<uint2*>(row) = make_uint2(code[0], code[1]);
      else *reinterpret_cast<uint32_t*>(row) = code[0];
      if (d0 == 0)
        a.s[z][b * ss.sb + (int64_t)pos * ss.st + h * ss.sh] = finite ? top / CodeTop<C>::v : __uint_as_float(0x7fc00000u);
    }
  }
}

// The same block shape; rows outside the cache read as zeros.
template <typename T, typename C, int D>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheCall a) {
  using vec = typename RowVec<T>::type;
  constexpr int VEC = RowVec<T>::N, LPR = D / VEC;
  const int b = blockIdx.y / a.H, h = blockIdx.y % a.H;
  const int t = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, d0 = (threadIdx.x % LPR) * VEC;
  if (t >= a.T) return;
  const int pos = cache_position(a, b, t);
  vec x[2];
  uint32_t code[2][VEC / 4];
  float sc[2] = {0.0f, 0.0f};
#pragma unroll
  for (int z = 0; z < 2; ++z) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[z][e] = from_f<T>(0.0f);
    const Strides3 cs = a.cs[z], ss = a.ss[z];
    const char* row = (const char*)a.c[z] + (b * cs.sb + (int64_t)pos * cs.st + h * cs.sh + d0) * (int64_t)sizeof(C);
    if (pos >= 0) {
      if constexpr (sizeof(C) > 1) {
        x[z] = *reinterpret_cast<const vec*>(row);
      } else {
#pragma unroll
        for (int w = 0; w < VEC / 4; ++w) code[z][w] = reinterpret_cast<const uint32_t*>(row)[w];
        sc[z] = a.s[z][b * ss.sb + (int64_t)pos * ss.st + h * ss.sh];
      }
    }
  }
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    if constexpr (sizeof(C) == 1) {
      if (pos >= 0) {
#pragma unroll
        for (int w = 0; w < VEC / 4; ++w) {
          float v[4];
          decode4(code[z][w], v, C{});
#pragma unroll
          for (int e = 0; e < 4; ++e) x[z][4 * w + e] = from_f<T>(v[e] * sc[z]);
        }
      }
    }
    const Strides3 xs = a.xs[z];
    *reinterpret_cast<vec*>((T*)const_cast<void*>(a.x[z]) + b * xs.sb + (int64_t)t * xs.st + h * xs.sh + d0) = x[z];
  }
}

template <typename T, typename C, int D>
static hipError_t launch_cache_t(const CacheCall& c) {
  constexpr int rows = 256 / (D / RowVec<T>::N);
  const dim3 grid((unsigned)((c.T + rows - 1) / rows), (unsigned)(c.B * c.H));
  if (c.read) hipLaunchKernelGGL((cache_read_kernel<T, C, D>), grid, dim3(256), 0, c.stream, c);
  else hipLaunchKernelGGL((cache_write_kernel<T, C, D>), grid, dim3(256), 0, c.stream, c);
  return hipGetLastError();
}

template <typename T, typename C>
static hipError_t launch_cache_d(const CacheCall& c) {
  switch (c.D) {
    case 16: return launch_cache_t<T, C, 16>(c);
    case 32: return launch_cache_t<T, C, 32>(c);
    case 64: return launch_cache_t<T, C, 64>(c);
    default: return launch_cache_t<T, C, 128>(c);
  }
}

template <typename T>
static hipError_t launch_cache_c(const CacheCall& c) {
  if (c.cache_dtype == kInt8) return launch_cache_d<T, int8_t>(c);
  if (c.cache_dtype == kFp8) return launch_cache_d<T, fp8>(c);
  return launch_cache_d<T, T>(c);
}

hipError_t launch_cache(const CacheCall& c) {
  if (c.dtype == 1) return launch_cache_c<bf16>(c);
  if (c.dtype == 2) return launch_cache_c<f16>(c);
  return launch_cache_c<float>(c);
}

}  // namespace msa

// Host-side internal interface between the C ABI (msa_capi.hip) and the
// kernel translation units.  Everything here is validated before use.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace msa {

// Padded head dimension the kernels are instantiated for.
inline int padded_dim(int D) { return D <= 32 ? 32 : (D <= 64 ? 64 : 128); }
inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline int ntiles(int64_t T) { return (int)((T + 63) / 64); }

struct Geometry {
  int B, H, Tq, Tk, D, DP, dtype, causal;
  int nqt, nkt;
  int nku_words;  // words per row of the live-unit bitmap (2*nkt 32-key units)
  int64_t Tq_pad, Tk_pad;
  size_t esize;  // bytes per element of dtype
};

struct Strides3 { int64_t sb, st, sh; };

// Forward workspace: khat [b*h][Tk_pad][DP], unit-normalised K rows (zero for
// padded and masked keys) that the forward stages through LDS.
size_t fwd_ws_bytes(const Geometry& g);

// Backward workspace: per-query-unit partial sums of dr, dw ([2][b*h][2*nqt]
// fp32), then dh ([b*h][Tq_pad][DP] in the input type) and 1/|q|
// ([b*h][Tq_pad] fp32) that dq_kernel hands to dkdv_kernel.
size_t bwd_ws_bytes(const Geometry& g);

// Attention dropout on alpha*m: pair (b, h, i, j) is kept iff the top 32 bits
// of its hash reach `thresh`, and kept pairs are scaled by `scale` = 1/(1-p).
struct Dropout {
  uint64_t seed;
  uint32_t thresh;
  float scale;
  int on;  // p > 0
};

// Dropout factor of pair (b*H+h, i, j): 0 or d.scale.  The SplitMix64
// finaliser (Steele, Lea and Flood, "Fast splittable pseudorandom number
// generators", OOPSLA 2014) of seed + key * 0x9E3779B97F4A7C15, key =
// bh << 44 | i << 22 | j (bh < 2^16, i, j < 2^22), decides: kept iff its top
// 32 bits reach d.thresh.
__device__ inline float dropout_factor(const Dropout& d, int bh, int i, int j) {
  const uint64_t key = ((uint64_t)(uint32_t)bh << 44) | ((uint64_t)(uint32_t)i << 22) | (uint64_t)(uint32_t)j;
  uint64_t z = d.seed + key * 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z ^= z >> 31;
  return (uint32_t)(z >> 32) >= d.thresh ? d.scale : 0.0f;
}

struct FwdCall {
  Geometry g;
  const void* q; Strides3 qs;
  const void* k; Strides3 ks;
  const void* v; Strides3 vs;
  const float* r; const float* w; const uint8_t* kpm;
  float eps;
  Dropout drop;
  void* y; float* hnorm; uint32_t* bits;
  void* khat;
  hipStream_t stream;
};
hipError_t launch_fwd(const FwdCall& c);

struct BwdCall {
  Geometry g;
  const void* q; Strides3 qs;
  const void* k; Strides3 ks;
  const void* v; Strides3 vs;
  const float* r; const float* w; const uint8_t* kpm;
  float eps;
  Dropout drop;
  const void* y; const float* hnorm; const void* dy;
  const uint32_t* bits;
  void* workspace;
  void* dq; void* dk; void* dv; float* dr; float* dw;
  hipStream_t stream;
};
hipError_t launch_bwd(const BwdCall& c);

struct DecodeCall {
  int B, H, D, DP, dtype, len;
  const void* q; int64_t q_sb, q_sh;
  const void* kc; Strides3 ks;
  const void* vc; Strides3 vs;
  const float* r; const float* w; float eps;
  void* y; float* part;
  int blocks;  // grid size of the partial-sum kernel (any value >= 1 gives the same result)
  int single;  // 1: one block per head walks its chunks (no partials); same result
  const int64_t* last_pos;  // device position of the newest key, or null (len is the length)
  int cap;                  // cache capacity (bounds the device length)
  hipStream_t stream;
};
int decode_chunk_keys();
// Chunks of a head's window at most, ceil(max_len / chunk): the decode
// workspace holds B*H of them, D floats each.
int decode_max_chunks(int max_len);
hipError_t launch_decode(const DecodeCall& c);

// Types of cache rows beside the input types 0..2 (msa.h's msa_dtype).
constexpr int kInt8 = 3, kFp8 = 4;

// Rows of a cache written or read back; index 0 is k, 1 is v.
struct CacheCall {
  const void* x[2]; Strides3 xs[2];  // the rows in the model's type: read by a write, written by a read
  void* c[2]; Strides3 cs[2];        // the cache
  float* s[2]; Strides3 ss[2];       // its scales (quantised caches)
  const int64_t* rows;               // (B, T) which row of x each written row is, or null: row t
  const int64_t* count;              // (B) rows written of each sequence, or null: T
  const int64_t* start; int start_step;  // first position of each sequence (step 0: of all), or null: start0
  int64_t start0;
  int B, T, Tx, H, D, cap, dtype, cache_dtype, read;
  hipStream_t stream;
};
hipError_t launch_cache(const CacheCall& c);

// Screening attention of a tree of N nodes per sequence over a cache.
struct TreeCall {
  int B, H, N, D, q_dtype, cache_dtype, cap;
  const void* q; int64_t q_sb, q_sn, q_sh;
  const void* kc; Strides3 ks;
  const void* vc; Strides3 vs;
  const float* kscale; Strides3 kss;  // 8-bit caches
  const float* vscale; Strides3 vss;
  const int64_t* lengths; int len_step;       // committed positions, one (step 0) or per sequence
  const int64_t* parents; int64_t par_sb;     // parents of a sequence's nodes, or null: a chain
  const float* r; const float* w; float eps, inv_eps;
  int2* table;  // [b][h] first piece and number of pieces of the head, where blocks != H
  float* part;  // [b][block][node][D] sums, where blocks != H
  void* y;
  int blocks;   // blocks that share a sequence's keys; H: a block per head
  hipStream_t stream;
};
int tree_blocks(int B, int H, int N, int D, int q_dtype, int cache_dtype, int span);
hipError_t launch_tree(const TreeCall& c);

// Drafted tokens against the target's rows.
struct VerifyCall {
  int B, M, dtype;
  int64_t V;
  const void* target; int64_t t_sb, t_sn;  // (B, M, V)
  const void* draft; int64_t d_sb, d_sn;   // (B, M - 1, V), or null
  const int64_t* tokens;                   // (B, M)
  const int64_t* parents; int64_t par_sb;  // or null: a chain
  const float* uniforms;                   // (B, M), or null: greedy
  int64_t* path; int64_t* count; int64_t* token;
  unsigned long long* best;                // greedy: [b*M + i][part] keys
  hipStream_t stream;
};
int verify_parts(int64_t V);
hipError_t launch_verify(const VerifyCall& c);

// Losses of rows against a vocabulary, straight from the rows: z = hidden weight^T / temperature, cross entropy
// (teacher null, K = 1) or the divergence from a teacher's K largest logits.
struct HeadCall {
  int64_t N, V; int d, K, dtype, teacher_dtype, reduction;  // reduction 0: a loss per row, 1: their mean, 2: their sum
  float temperature;
  int64_t ignore_index;
  const void* x; int64_t x_ld;
  const void* w; int64_t w_ld;
  const int64_t* ids; int64_t ids_ld;
  const void* teacher; int64_t teacher_ld;
  void* state;
  float* loss;
  const float* dloss;
  void* dx; void* dw;
  void* workspace;
  hipStream_t stream;
};
size_t head_state_bytes(int64_t N, int K);
size_t head_workspace_bytes(const HeadCall& c, int backward);
hipError_t launch_head_fwd(const HeadCall& c);
hipError_t launch_head_bwd(const HeadCall& c);

// h = act(x w[0]^T) * (x w[1]^T) and its gradients.
struct GatedCall {
  int64_t N; int d, F, dtype, act;  // act 0: silu, 1: gelu (erf)
  const void* x; int64_t x_ld;
  const void* w[2]; int64_t w_ld[2];
  void* h;
  const void* dh; int64_t dh_ld;
  void* dx; void* dw[2];
  void* workspace;
  hipStream_t stream;
};
size_t gated_workspace_bytes(const GatedCall& c, int backward);
hipError_t launch_gated_fwd(const GatedCall& c);
hipError_t launch_gated_bwd(const GatedCall& c);

// Waves that share a row (32-query or 32-key unit) in the live, dq and dK/dV
// passes: launches with few rows split each row's units, so that about 2048
// waves (2-byte types) or 4096 (fp32, whose rows take several times as long)
// are in flight.  us of the three passes with 1 / 2 / 4 waves, about 5% of the
// pairs live, T = 512 and T = 1280 .. 2048 (a wave's fixed part weighs more in
// short rows, so the best split lies lower there):
//                 512 rows                 1024                     2048
//   bf16 D=64     72/52/43    229/141/93   80/62/71    240/152/121  90/95/127   258/191/221
//   bf16 D=128    102/76/86   334/207/163  114/113/161 356/242/284  164/204/311 394/414/538
//   fp32 D=64     246/154/135 912/510/319  258/210/257 941/559/548  337/381/480 1017/943/1067
//   fp32 D=128    508/307/292 1854/987/616 591/455/558 2054/1121/1122  829/864/1084 2395/2107/2232
// (3072 rows of fp32: D=64 487/555/716 and 1356/1397/1575.)
template <typename T>
inline int split_waves(int64_t rows) {
  const int64_t most = sizeof(T) == 2 ? 2048 : 4096;
  return rows * 4 <= most ? 4 : (rows * 2 <= most ? 2 : 1);
}

// Optional event pairs around one kernel's launches (msa_timer_arm).
void timer_begin(int kernel, hipStream_t s);
void timer_end(int kernel, hipStream_t s);

hipError_t launch_selftest(const float* a16, const float* b16, float* out16,
                           const float* a2, const float* b2, float* out2,
                           hipStream_t stream);

}  // namespace msa

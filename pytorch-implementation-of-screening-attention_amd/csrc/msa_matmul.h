// Matrix products on gfx950 for the kernels whose work is a product with a fused epilogue (the vocabulary head's
// losses, the gated feed-forward): a block computes one tile C[m][n] = sum_k A[m][k] B[n][k] of 16-bit operands in
// fp32 registers, the caller's epilogue does the rest.
//
// Feature rows (weights, or the columns of an output) are the m side and tokens the n side, so that a lane holds
// many features of few tokens: sums over a token's features need no shuffles, and four registers are four
// neighbours of an output row.
//
// Each operand lies in memory with either its k contiguous (rows of A or B) or its m or n contiguous (k rows), and
// is staged in that order; MFMA fragments come by ds_read_b128 or, transposed, by ds_read_b64_tr_b16.
#pragma once

#include "msa_device.h"

namespace msa {

constexpr int kMmK = 32;      // k of a stage
constexpr int kMmSegs = 12;   // products that one tile adds up

// A sum over up to kMmSegs operand pairs of the same shape (byte offsets to A and B).  fp32 operands enter as two
// fp16 terms, x s = h + 2^-11 l with a power of two s: three products h l + l h, then 2^-11 of their sum, then h h; or as
// three bf16 terms, x = h + m + l: h l + l h + m m, then h m + m h, then h h (what is left out is 2^-26 of x).
struct MmSegs {
  int64_t a[kMmSegs], b[kMmSegs];
  int n, low;  // products; the first `low` are of order 2^-11 (0: none)
};
constexpr float kLowTerm = 1.0f / 2048.0f;

// Starts the copy of 16 bytes a lane from base (uniform) + off to LDS at `to` (uniform) + 16 lane.  Written out because
// the compiler waits for every copy in flight before it reads any of the array that one goes to, which would undo the
// stages; the loop waits for the stage that it reads (MmTile::arrive).  M0 takes a wait state before its use.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // M0 is reserved: the clobber still tells the compiler that it changed
__device__ inline void mm_copy(const char* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// Four neighbours of an output row.
template <typename O> struct Quad { typedef __attribute__((__vector_size__(4 * sizeof(O)))) O V; };
template <typename O, typename Fn>
__device__ inline typename Quad<O>::V quad(Fn fn) {
  typename Quad<O>::V v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from_f<O>(fn(e));
  return v;
}

// E: operand type.  BM x BN: the block's tile; WM x WN waves share it.  AMN, BMN: the operand's m or n is
// contiguous.  DUAL: A is two matrices, whose rows alternate by 16 (m = 32 i + j: row 16 i + j of the first for j < 16, row
// 16 i + j - 16 of the second above): registers r and r + 8 of a lane are the same row of both, r < 8.  NST: stages.
template <typename E, int BM, int BN, int WM, int WN, bool AMN, bool BMN, bool DUAL, int NST>
struct MmTile {
  using M = Mma<E>;
  using frag = typename M::frag;
  static constexpr int NT = 64 * WM * WN;                    // threads
  static constexpr int MB = BM / WM / 32, NB = BN / WN / 32;  // 32x32 blocks of a wave
  static constexpr int ABYTES = BM * kMmK * 2, BBYTES = BN * kMmK * 2, STAGE = ABYTES + BBYTES;
  static constexpr int TILE_M = BM, TILE_N = BN, THREADS = NT, WAVES_M = WM;
  static constexpr int STAGED = 32 * WN * (BM * 4 + 16);  // store_tokens of fp32
  static constexpr int LDS = NST * STAGE > STAGED ? NST * STAGE : STAGED;
  static constexpr int NWAVES = WM * WN;
  static constexpr int AI = ABYTES / 1024 / NWAVES, BI = BBYTES / 1024 / NWAVES;  // copies of 1 KiB a wave issues
  static_assert(AI * NWAVES * 1024 == ABYTES && BI * NWAVES * 1024 == BBYTES, "a stage is whole copies of every wave");
  static_assert(MB <= 4 && NB <= 4, "blocks are found by two address bits");
  static_assert(!DUAL || (!AMN && NWAVES % 2 == 0), "a wave's copies are one matrix's");

  typedef f32x16 Acc[MB][NB];

  // Places of 16-byte chunks are XOR-swizzled so that reads are free of bank conflicts whether the LDS serves 128 or 256
  // bytes a cycle.  K-contiguous rows R of 4 chunks: by (b1 ^ b3, b2) of R, one-to-one on rows 0, 2, 4, 6 (which
  // share a half of 128 bytes) and on 0, 4, 8, 12 (a quarter of 256).  k rows of the other order: a transposed read
  // takes 4 neighbours k at 2 chunks (128 bytes) or 4 (256): by bits 1 to 3 (k1, k0, k1).  (With half of the banks at
  // a time in mind only, half of all LDS cycles were conflicts.)
  __device__ static constexpr int swz_row(int R) { return (((R >> 1) ^ (R >> 3)) & 1) | (((R >> 2) & 1) << 1); }
  __device__ static constexpr int swz_k(int k) { return ((k & 2) * 5) | ((k & 1) << 2); }

  // One operand's copies.  K-contiguous: rows of 64 bytes, a copy is 16 rows.  Otherwise: k rows of W columns.
  template <bool MN, int W, int NI, bool ALT>
  struct Loader {
    uint32_t off[NI];
    uint32_t ld;   // bytes from row to row
    int rows, r0;  // MN: k rows of the matrix (later ones read the last), the lane's row of copy 0
    static constexpr int CPR = W / 8;            // MN: chunks of a row
    static constexpr int RPI = 64 / CPR;         // MN: rows of a copy (W <= 512)
    // first: the tile's first row (K-contiguous) or column (MN); count: rows or columns of the matrix from there on.
    // ALT: count of each of the two matrices.
    __device__ inline void init(int64_t stride_bytes, int64_t blk, int count, int wave, int lane, int krows) {
      ld = (uint32_t)stride_bytes;
      rows = krows;
      if constexpr (!MN) {
        const int lr = lane >> 2, chunk = (lane & 3) ^ swz_row(lr);
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int g = j * NWAVES + wave;  // a copy's 16 rows
          int r = (ALT ? g >> 1 : g) * 16 + lr;
          r = r < count ? r : count - 1;
          off[j] = (uint32_t)r * ld + (uint32_t)chunk * 16u;
        }
      } else {
        static_assert(64 % CPR == 0, "a copy is whole rows");
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int p = (j * NWAVES + wave) * 64 + lane, k = p / CPR;
          int col = ((p % CPR) ^ swz_k(k)) * 8;
          col = col < count ? col : count - 8;  // count is a multiple of 8
          off[j] = (uint32_t)k * ld + (uint32_t)(col >> 5) * (uint32_t)blk + (uint32_t)(col & 31) * 2u;
        }
        r0 = wave * RPI + lane / CPR;
      }
    }
    // Starts the copies of the stage whose k begins at k0; base points to (first row, k0) or (k0, first column).
    __device__ inline void issue(const char* base, int64_t alt, LdsChar* lds, int wave, int k0) const {
      // k rows behind the last one read it again (their other operand is zero); all of this is block-uniform
      const bool cut = MN && k0 + kMmK > rows;
      int last = 0;
      if (cut) {
        const int from = k0 < rows ? k0 : rows - 1;
        base -= (int64_t)(k0 - from) * ld;
        last = rows - 1 - from;
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        uint32_t o = off[j];
        if constexpr (MN) {
          if (cut) {
            const int k = r0 + j * NWAVES * RPI;
            if (k > last) o -= (uint32_t)(k - last) * ld;
          }
        }
        const char* b = ALT && (wave & 1) ? base + alt : base;
        mm_copy(b, o, (uint32_t)(uintptr_t)lds + (uint32_t)((j * NWAVES + wave) * 1024));
      }
    }
  };

  // The lane's fragment address in a staged operand: block i of 32 rows or columns from `first`, half c of the k.
  template <bool MN, int W>
  struct Reader {
    uint32_t at;
    __device__ inline void init(int first, int lane) {
      const int half = lane >> 5;
      if constexpr (!MN) {
        const int R = lane & 31;
        at = (uint32_t)((first + R) * 64 + ((half ^ swz_row(R)) << 4));
      } else {
        const int kk = (lane & 15) >> 2, q = lane & 3, gg = (lane >> 4) & 1;
        at = (uint32_t)((8 * half + kk) * (W * 2) + (((first / 8 + 2 * gg + (q >> 1)) ^ swz_k(kk)) << 4) + 8 * (q & 1));
      }
    }
    __device__ inline frag read(const LdsChar* tile, int i, int c) const {
      if constexpr (!MN) {
        return *reinterpret_cast<const __attribute__((address_space(3))) frag*>(tile + (at ^ (uint32_t)(c << 5)) + i * 2048);
      } else {
        typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
        typedef __attribute__((__vector_size__(8 * sizeof(short)))) short s16x8;
        s16x8 v;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const LdsChar* p = tile + (at ^ (uint32_t)(i << 6)) + (16 * c + 4 * j) * (W * 2);  // `first` is a multiple of 32 times the wave's blocks, which are at most 4
          const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)const_cast<LdsChar*>(p));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * j + e] = x[e];
        }
        return __builtin_bit_cast(frag, v);
      }
    }
  };

  // The tile's operands: where (first row or column, k = 0) lies, rows or columns there are from it on, bytes from
  // row to row and from 32 columns to the next 32, k rows (MN).  Rows as they are in a tensor: blk = 64.  Operands that a
  // kernel writes lie in blocks of 32 columns, row behind row (ld = 64): a stage is then whole kilobytes, where 64 bytes of
  // a long row are half a cache line and a request of its own.
  struct Side {
    const char* p;
    int count;
    int64_t ld, blk;
    int krows;
    int64_t alt;  // DUAL: to the second matrix
  };

  // acc += the tile's product over k in [k0, k0 + 32 steps).  Every thread of the block calls it with the same
  // arguments.  lds: LDS bytes of the block's own, free on entry; on return every wave is past its last read.
  __device__ static inline void run(Acc& acc, LdsChar* lds, const Side& A, const Side& B, const MmSegs& segs, int k0,
                                    int steps) {
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    Loader<AMN, BM, AI, DUAL> la;
    Loader<BMN, BN, BI, false> lb;
    la.init(A.ld, A.blk, A.count, wave, lane, A.krows);
    lb.init(B.ld, B.blk, B.count, wave, lane, B.krows);
    Reader<AMN, BM> ra;
    Reader<BMN, BN> rb;
    ra.init(wm * (BM / WM), lane);
    rb.init(wn * (BN / WN), lane);
    const int64_t astep = AMN ? A.ld * kMmK : A.blk, bstep = BMN ? B.ld * kMmK : B.blk;
    const char* const a0 = A.p + astep * (k0 / kMmK);
    const char* const b0 = B.p + bstep * (k0 / kMmK);

    const int total = steps * segs.n;
    int iseg = 0, istep = 0;  // the next stage to copy
    const char* ia = a0 + segs.a[0];
    const char* ib = b0 + segs.b[0];
    auto issue = [&](int slot) {
      LdsChar* s = lds + slot * STAGE;
      la.issue(ia, A.alt, s, wave, k0 + istep * kMmK);
      lb.issue(ib, 0, s + ABYTES, wave, k0 + istep * kMmK);
      ia += astep;
      ib += bstep;
      if (++istep == steps) {
        istep = 0;
        if (++iseg < segs.n) {
          ia = a0 + segs.a[iseg];
          ib = b0 + segs.b[iseg];
        }
      }
    };
    int filled = 0;
#pragma unroll
    for (int u = 0; u < NST; ++u)
      if (u < total) { issue(u); ++filled; }
    const int low = steps * segs.low;
    frag a[2][MB], b[2][NB];
    auto fetch = [&](int slot, auto C) {  // fragments of half C of a landed stage
      constexpr int c = decltype(C)::value;
      const LdsChar* at = lds + slot * STAGE;
#pragma unroll
      for (int i = 0; i < MB; ++i) a[c][i] = ra.read(at, i, c);
#pragma unroll
      for (int j = 0; j < NB; ++j) b[c][j] = rb.read(at + ABYTES, j, c);
    };
    auto multiply = [&](auto C) {
      constexpr int c = decltype(C)::value;
      // MB * NB independent sums: an accumulator comes again only after all the others, so no MFMA waits for the
      // one before it and none reads its operands late (see the source-operand guard in msa_device.h)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = M::mma_ng(a[c][i], b[c][j], acc[i][j]);
      if constexpr (MB * NB < 4) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) asm volatile(MSA_NOP16 : "+v"(a[c][i]), "+v"(b[c][j]));
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    typedef std::integral_constant<int, 0> First;
    typedef std::integral_constant<int, 1> Second;
    if (filled == NST) arrive<(NST - 1) * (AI + BI)>();
    else arrive<0>();
    fetch(0, First());
    fetch(0, Second());
    auto scale_low = [&]() {
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] *= kLowTerm;
    };
    int slot = 0;  // of stage t
    for (int t = 0; t < total - 1; ++t) {
      if (low != 0 && t == low) scale_low();
      multiply(First());
      // Between the halves: stage t + 1 has landed once only the younger ones are outstanding, and every wave holds the
      // fragments of stage t, so its slot takes the next copy.
      if (filled - t >= NST) arrive<(NST - 2) * (AI + BI)>();
      else arrive<0>();
      if (filled < total) { issue(slot); ++filled; }
      slot = slot + 1 == NST ? 0 : slot + 1;
      fetch(slot, First());
      __builtin_amdgcn_sched_barrier(0);
      multiply(Second());
      fetch(slot, Second());
      __builtin_amdgcn_sched_barrier(0);
    }
    if (low != 0 && total - 1 == low) scale_low();
    multiply(First());
    multiply(Second());
    arrive<0>();
  }

  // The block's barrier for LDS alone: __syncthreads would also wait for the wave's stores to memory.
  __device__ static inline void sync_lds() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // The block's barrier, with this wave's LDS reads done and at most N of its copies outstanding.
  template <int N>
  __device__ static inline void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // Operand rows for a later product, in blocks of 32 columns (Side): dst is the tile's first row in its first block, blk
  // elements from block to block; the tile's rows and columns are all there.
  template <typename Fn>
  __device__ static inline void store_operand(LdsChar* lds, E* dst, int64_t blk, Fn fn) {
#pragma unroll
    for (int j = 0; j < NB; ++j) store_operand_tokens<MB>(lds, dst, blk, j, [&](int i, int g) { return fn(i, j, g); });
  }
  template <int MS, typename Fn>
  __device__ static inline void store_operand_tokens(LdsChar* lds, E* dst, int64_t blk, int j, Fn fn) {
    constexpr int W = 32 * MS * WM, R = 32 * WN, ROW = W * 2 + 16;
    stage_tokens<E, MS>(lds, j, fn);
    const int tid = (int)threadIdx.x;
#pragma unroll 4
    for (int u = tid; u < R * W / 8; u += NT) {
      const int c4 = u & 3, r = (u >> 2) % R, b = (u >> 2) / R, n = (r >> 5) * (BN / WN) + 32 * j + (r & 31);
      typedef __attribute__((__vector_size__(16))) E EV;
      const EV v = *reinterpret_cast<const __attribute__((address_space(3))) EV*>(lds + r * ROW + b * 64 + c4 * 16);
      *reinterpret_cast<EV*>(dst + b * blk + (int64_t)n * 32 + c4 * 8) = v;
    }
    sync_lds();
  }
  // Registers of the blocks (., j) as rows of 32 tokens of each wave in LDS.
  template <typename O, int MS, typename Fn>
  __device__ static inline void stage_tokens(LdsChar* lds, int j, Fn fn) {
    constexpr int QUADS = DUAL && MB == 1 ? 2 : 4, W = 8 * QUADS * MS * WM;  // a lone DUAL block is 16 features
    constexpr int ROW = W * (int)sizeof(O) + 16;
    static_assert(32 * WN * ROW <= LDS, "the staged rows fit the tile's LDS");
    typedef __attribute__((address_space(3))) typename Quad<O>::V LdsQuad;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wn = wave / WM;
    LdsChar* to = lds + (wn * 32 + (lane & 31)) * ROW + (wm * 8 * QUADS * MS + 4 * (lane >> 5)) * (int)sizeof(O);
#pragma unroll
    for (int i = 0; i < MS; ++i)
#pragma unroll
      for (int g = 0; g < QUADS; ++g) {
        const typename Quad<O>::V v = fn(i, g);
        *reinterpret_cast<LdsQuad*>(to + (32 * i + 8 * g) * (int)sizeof(O)) = v;
      }
    sync_lds();
  }

  // A DUAL tile's rows of an output: fn(i, j, g) of registers 4 g .. 4 g + 3 and 8 more, g < 2.
  template <typename O, typename Fn>
  __device__ static inline void store_dual(LdsChar* lds, O* dst, int64_t ld, int rows, int cols, bool vec, Fn fn) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
      store_tokens<O, false, (MB + 1) / 2>(lds, dst, ld, rows, cols, vec, j, [&](int i, int g) { return fn(2 * i + (g >> 1), j, g & 1); });
  }

  // Writes rows of an output: dst[n ld + m .. + 3] = fn(i, j, g) of registers 4 g .. 4 g + 3 of blocks (i, j), i < MS, for
  // n < rows and m < cols; ADD: added to what is there (O float).  A wave's MS blocks are neighbours (MS = MB: the tile itself).  vec:
  // dst and ld allow 16-byte accesses.  The values go through the block's LDS (free on entry and on return), 32
  // tokens of each wave at a time, so that a wave writes whole rows.
  template <typename O, bool ADD, int MS = MB, typename Fn>
  __device__ static inline void store_rows(LdsChar* lds, O* dst, int64_t ld, int rows, int cols, bool vec, Fn fn) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
      store_tokens<O, ADD, MS>(lds, dst, ld, rows, cols, vec, j, [&](int i, int g) { return fn(i, j, g); });
  }
  // The part of it for the tokens of blocks (., j).
  template <typename O, bool ADD, int MS, typename Fn>
  __device__ static inline void store_tokens(LdsChar* lds, O* dst, int64_t ld, int rows, int cols, bool vec, int j, Fn fn) {
    constexpr int QUADS = DUAL && MB == 1 ? 2 : 4, W = 8 * QUADS * MS * WM;
    constexpr int ROW = W * (int)sizeof(O) + 16, PER = 16 / (int)sizeof(O), CPR = W / PER, R = 32 * WN;
    stage_tokens<O, MS>(lds, j, fn);
    const int tid = (int)threadIdx.x;
#pragma unroll 4
    for (int u = tid; u < R * CPR; u += NT) {
      const int r = u / CPR, c = (u - r * CPR) * PER, n = (r >> 5) * (BN / WN) + 32 * j + (r & 31);
      if (n < rows && c < cols) {
        typedef __attribute__((__vector_size__(16))) O OV;
        OV v = *reinterpret_cast<const __attribute__((address_space(3))) OV*>(lds + r * ROW + c * (int)sizeof(O));
        O* p = dst + (int64_t)n * ld + c;
        if (vec && c + PER <= cols) {
          if constexpr (ADD) v += *reinterpret_cast<const OV*>(p);
          *reinterpret_cast<OV*>(p) = v;
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (c + e < cols) p[e] = ADD ? (O)((float)p[e] + (float)v[e]) : v[e];
        }
      }
    }
    sync_lds();
  }

  // Hides the values from the compiler, which would otherwise keep what it formed from them for a second use.
  __device__ static inline void renew(Acc& acc) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) asm volatile("" : "+v"(acc[i][j]));
  }

  __device__ static inline void clear(Acc& acc) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  }

  // Place of a lane's registers in the tile: register 4 g + e of block (i, j) is C[m(i, g) + e][n(j)].
  __device__ static inline int m_of(int wm, int lane, int i, int g) { return wm * (BM / WM) + 32 * i + 8 * g + 4 * (lane >> 5); }
  __device__ static inline int n_of(int wn, int lane, int j) { return wn * (BN / WN) + 32 * j + (lane & 31); }
};

// Whether a grid of tiles of 256 by 128 (two a CU at a time) is better cut into twice as many of 128 by 128: those take
// about 12% longer for the same work, but the CU with most of them may have less of it.
inline bool smaller_tiles(int64_t tiles_m, int64_t tiles_n, int64_t small_m) {
  return (small_m * tiles_n + 255) / 256 * 112 < (tiles_m * tiles_n + 255) / 256 * 200;
}

// Blocks of a grid go to the eight XCDs in turn, each with an L2 of its own: block id -> position in an order whose
// consecutive eighths are an XCD's.
__device__ inline int64_t xcd_order(int64_t id, int64_t total) {
  const int64_t x = id & 7, i = id >> 3, q = total >> 3, r = total & 7;
  return x * q + (x < r ? x : r) + i;
}

// Tile (tm, tn) at position t of an order that walks patches of G m-tiles by all n-tiles, m first: the tiles in flight
// on an XCD then share few rows of both operands.
__device__ inline void patch_order(int64_t t, int tiles_m, int tiles_n, int G, int& tm, int& tn) {
  const int64_t per = (int64_t)G * tiles_n;
  const int g = (int)(t / per), in = (int)(t - g * per);
  const int w = tiles_m - g * G < G ? tiles_m - g * G : G;
  tn = in / w;
  tm = g * G + (in - tn * w);
}

}  // namespace msa

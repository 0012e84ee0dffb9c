// Matrix products on the matrix cores (gfx950), for the fused kernels of r3d_loss.hip.
//
// C[m][n] = sum_k A(m,k) B(n,k) in tiles of BM x BN x 64, every wave FM x FN blocks of v_mfma_f32_32x32x16.  How an operand lies:
//   Rows    A[m][k], k contiguous
//   Cols    A[k][m], m contiguous
//   Pieces  in pieces of 8 values, piece-major: value (r, c) at ((c / 8) * rows + r) * 8 + c % 8 -- what a product that is an
//           operand of the next one is stored as, because 32 lanes then write (and read) 512 contiguous bytes.  PiecesRows: m = r,
//           k = c; PiecesCols: k = r, m = c.
// Operands go to LDS as they lie, by direct-to-LDS loads of 16 bytes a lane; where k is not the contiguous axis the fragment is
// turned on the way out of LDS (ds_read_b64_tr_b16: 16 lanes read 4 k-rows of 16 columns, lane i gets column i).  LDS takes the
// lanes of a load in one line, so the swizzle that spreads a fragment over the banks is applied to the global address.
#pragma once

#include <hip/hip_runtime.h>

namespace r3d {

constexpr int kTileK = 64;
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Tile and waves.  A wave's share of 128 x 64 reads 0.75 of the 128 bytes a clock that LDS gives while the matrix cores are
// busy, one of 64 x 64 all of them; a tile of 256 x 256 takes 32 bytes a clock and CU out of L2, one of 128 x 128 64.
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, threads = 64 * WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int a_elems = BM * kTileK, b_elems = BN * kTileK, buffer = a_elems + b_elems;
};
using Big = Shape<256, 256, 2, 4>;
using Small = Shape<128, 128, 2, 2>;

enum class Lies { Rows, Cols, PiecesRows, PiecesCols };

template <class T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// One operand.  ld: elements between rows, or rows of a piece-major one; plane: between the planes of a split one; idx: rows by number.
struct Operand {
  const void *p;
  int64_t ld, plane;
  const int32_t *idx;
};

typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ void load_lds16(const void *g, void *lds_wave_base) {
  __builtin_amdgcn_global_load_lds((global_void *)g, (lds_void *)lds_wave_base, 16, 0, 0);
}

// A thread's part of an operand tile of R rows (or columns) x 64 k: `per` pieces of 16 bytes, piece number i * threads + thread.
template <class T, Lies L, int R, int kThreads>
struct Loader {
  static constexpr int per = R * kTileK / 8 / kThreads;
  const T *at[per];      // Rows, Pieces: where the thread's pieces of the current tile begin
  int64_t row[per];      // Cols: rows of the next k-block, looked up one block ahead
  int col;

  // first: first row (Rows, PiecesRows) or column of the tile; limit: how many there are.  What lies behind is read from the last
  // one, any finite or infinite values: its results are not used.
  __device__ __forceinline__ void tile(const Operand &o, int64_t first, int64_t limit) {
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int c = i * kThreads + threadIdx.x;
      if constexpr (L == Lies::Rows) {
        const int r = c >> 3;
        int64_t n = first + r;
        n = n < limit ? n : limit - 1;
        if (o.idx) n = o.idx[n];
        at[i] = static_cast<const T *>(o.p) + n * o.ld + (((c & 7) ^ ((r >> 1) & 7)) << 3);
      } else if constexpr (L == Lies::PiecesRows) {
        const int r = c % R, q = c / R;      // LDS: [8 pieces of k][R rows]
        int64_t n = first + r;
        n = n < limit ? n : limit - 1;
        at[i] = static_cast<const T *>(o.p) + (q * o.ld + n) * 8;
      } else if constexpr (L == Lies::PiecesCols) {
        const int k = c & 63, q = c >> 6;    // LDS: [R / 8 pieces of m][64 k], k in fours at k ^ 4 (q & 3)
        int64_t p = first / 8 + q;
        p = p < limit / 8 ? p : limit / 8 - 1;
        at[i] = static_cast<const T *>(o.p) + (p * o.ld + (k ^ ((q & 3) << 2))) * 8;
      }
    }
    if constexpr (L == Lies::Cols) {
      const int c = threadIdx.x, k = c / (R / 8);      // (the pieces of a thread differ by multiples of 4 rows)
      const int64_t m = first + (((c % (R / 8)) ^ ((k & 3) << 2)) << 3);
      col = (int)(m + 8 <= limit ? m : limit - 8);
    }
  }
  // Cols: the rows of k-block kb.
  __device__ __forceinline__ void look(const Operand &o, int64_t kb, int64_t rows) {
    if constexpr (L == Lies::Cols) {
#pragma unroll
      for (int i = 0; i < per; ++i) {
        int64_t r = kb * kTileK + (i * kThreads + threadIdx.x) / (R / 8);
        r = r < rows ? r : rows - 1;
        row[i] = o.idx ? o.idx[r] : r;
      }
    }
  }
  __device__ __forceinline__ void issue(const Operand &o, T *lds, int64_t kb, int64_t plane) const {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < per; ++i) {
      T *to = lds + (i * kThreads + wave * 64) * 8;
      if constexpr (L == Lies::Rows) load_lds16(at[i] + plane + kb * kTileK, to);
      else if constexpr (L == Lies::PiecesRows) load_lds16(at[i] + plane + kb * 8 * o.ld * 8, to);
      else if constexpr (L == Lies::PiecesCols) load_lds16(at[i] + plane + kb * kTileK * 8, to);
      else load_lds16(static_cast<const T *>(o.p) + plane + row[i] * o.ld + col, to);
    }
  }
};

// Fragment of the 32 rows (columns) from r0, k-step kk of 16: lane holds row lane & 31, k = (lane >> 5) * 8 + 0..7.
template <class T, Lies L, int R>
__device__ __forceinline__ typename Mma<T>::v8 fragment(const T *lds, int r0, int kk) {
  const int lane = threadIdx.x & 63;
  if constexpr (L == Lies::Rows || L == Lies::PiecesRows) {
    const int r = r0 + (lane & 31), q = kk * 2 + (lane >> 5);
    const T *at = L == Lies::Rows ? lds + r * kTileK + ((q ^ ((r >> 1) & 7)) << 3) : lds + (q * R + r) * 8;
    return *reinterpret_cast<const typename Mma<T>::v8 *>(at);
  } else {
    typedef short s4 __attribute__((ext_vector_type(4)));
    const int group = lane >> 4, p = lane & 15;
    const int c = r0 + (group & 1) * 16 + (p & 3) * 4, k = kk * 16 + (group >> 1) * 8 + (p >> 2), q = c >> 3;
    const T *lo_at, *hi_at;
    if constexpr (L == Lies::Cols) {
      lo_at = lds + k * R + ((q ^ ((k & 3) << 2)) << 3) + (c & 7);
      hi_at = lo_at + 4 * R;
    } else {
      lo_at = lds + (q * 64 + (k ^ ((q & 3) << 2))) * 8 + (c & 7);
      hi_at = lds + (q * 64 + ((k + 4) ^ ((q & 3) << 2))) * 8 + (c & 7);
    }
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)lo_at);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)hi_at);
    return __builtin_bit_cast(typename Mma<T>::v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

template <class T>
__device__ __forceinline__ float sum8(typename Mma<T>::v8 v, float s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s += (float)v[i];
  return s;
}

// (plane of A, plane of B) of the products of two operands in three planes of 8 bits each: what is left out is below 2^-24.
constexpr int kPairs = 6;
__device__ constexpr int kPlaneA[kPairs] = {0, 0, 1, 1, 0, 2}, kPlaneB[kPairs] = {0, 1, 0, 1, 2, 0};

// A stream of k-blocks through two LDS buffers: the next block is on its way while the current one is multiplied.
template <class T, class S, Lies LA, Lies LB>
struct Stream {
  Operand a, b;
  Loader<T, LA, S::BM, S::threads> la;
  Loader<T, LB, S::BN, S::threads> lb;
  int64_t rows_a, rows_b;      // rows of Cols operands
  int64_t kb, kb0, kb1;
  int pair, pairs, buf;

  __device__ __forceinline__ void range(int64_t first, int64_t end, int planes) {
    kb0 = first;
    kb1 = end;
    pairs = planes == 3 ? kPairs : 1;
    buf = 0;
    rewind();
  }
  __device__ __forceinline__ void rewind() {
    kb = kb0;
    pair = 0;
    la.look(a, kb, rows_a);
    lb.look(b, kb, rows_b);
  }
  __device__ __forceinline__ void issue(T *lds, int to) {
    la.issue(a, lds + to * S::buffer, kb, kPlaneA[pair] * a.plane);
    lb.issue(b, lds + to * S::buffer + S::a_elems, kb, kPlaneB[pair] * b.plane);
    if (++kb == kb1) {
      kb = kb0;
      ++pair;
    }
    la.look(a, kb, rows_a);
    lb.look(b, kb, rows_b);
  }
  // acc += all k-blocks of the tile whose first block is in the current buffer; `next()` is called while the last block is
  // multiplied and says whether there is another tile, whose loaders it has set.  kSums: row_sum += sums over k of A,
  // where `sums`.
  template <bool kSums, class Next>
  __device__ __forceinline__ void run(T *lds, f32x16 (&acc)[S::FM][S::FN], float (&row_sum)[S::FM], bool sums, Next &&next) {
    const int wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
    const int64_t steps = (kb1 - kb0) * pairs;
    int at_pair = 0;
    int64_t pair_end = kb1 - kb0;
    for (int64_t s = 0; s < steps; ++s) {
      if (s == pair_end) {
        ++at_pair;
        pair_end += kb1 - kb0;
      }
      if (s + 1 < steps) {
        issue(lds, buf ^ 1);
      } else if (next()) {
        rewind();
        issue(lds, buf ^ 1);
      }
      const T *pa = lds + buf * S::buffer, *pb = pa + S::a_elems;
      typename Mma<T>::v8 fa[2][S::FM], fb[2][S::FN];
      auto read = [&](int kk, int into) {
#pragma unroll
        for (int i = 0; i < S::FM; ++i) fa[into][i] = fragment<T, LA, S::BM>(pa, (wm * S::FM + i) * 32, kk);
#pragma unroll
        for (int j = 0; j < S::FN; ++j) fb[into][j] = fragment<T, LB, S::BN>(pb, (wn * S::FN + j) * 32, kk);
      };
      read(0, 0);
#pragma unroll
      for (int kk = 0; kk < kTileK / 16; ++kk) {
        if (kk + 1 < kTileK / 16) read(kk + 1, (kk + 1) & 1);
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
          for (int j = 0; j < S::FN; ++j) acc[i][j] = Mma<T>::mma(fa[kk & 1][i], fb[kk & 1][j], acc[i][j]);
        if (kSums && sums && kPlaneB[at_pair] == 0) {      // (every plane of A once)
#pragma unroll
          for (int i = 0; i < S::FM; ++i) row_sum[i] = sum8<T>(fa[kk & 1][i], row_sum[i]);
        }
      }
      __syncthreads();
      buf ^= 1;
    }
  }
};

template <int FM, int FN>
__device__ __forceinline__ void clear(f32x16 (&acc)[FM][FN]) {
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
}

// Row of C in a 32 x 32 block that register j of a lane holds (its column is lane & 31).
__device__ __forceinline__ int mma_row(int j) { return (j & 3) + 8 * (j >> 2) + 4 * ((threadIdx.x & 63) >> 5); }

// Work number of a block such that neighbours in number are on one XCD (blocks go round the eight) and share its L2.
__device__ __forceinline__ int64_t xcd_order(int64_t block, int64_t blocks) {
  const int64_t each = blocks / 8, rest = blocks % 8, x = block % 8, at = block / 8;
  return x * each + (x < rest ? x : rest) + at;
}

}  // namespace r3d

// Matrix products on the matrix cores (gfx950), for the fused kernels of r3d_loss.hip.
//
// C[m][n] = sum_k A(m,k) B(n,k) in tiles of 128 x 128 x 64: four waves, each 64 x 64 as 2 x 2 of v_mfma_f32_32x32x16.
// An operand lies in memory with k contiguous ("rows": A[m][k]) or with m contiguous ("columns": A[k][m]); both go to LDS as
// they lie, by direct-to-LDS loads of 16 bytes a lane, and the second kind is turned on the way out of LDS
// (ds_read_b64_tr_b16: 16 lanes read 4 k-rows of 16 columns, lane i gets column i).  LDS takes the lanes of a load in one line,
// so the bank swizzle is applied to the global address: chunk c of row r stands at c ^ swizzle(r).
#pragma once

#include <hip/hip_runtime.h>

namespace r3d {

constexpr int kTileM = 128, kTileN = 128, kTileK = 64, kMmaThreads = 256;
constexpr int kOperandElems = kTileM * kTileK;      // 16 KB of LDS per operand and buffer

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// One operand.  rows x ld elements, `plane` elements between the planes of a split one, rows taken through idx where given.
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

// "Rows" operand: the four rows of the tile a thread loads from, as pointers to their first element.
template <class T>
struct RowLoader {
  const T *row[4];
  __device__ __forceinline__ void tile(const Operand &o, int64_t first, int64_t rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 32 + (threadIdx.x >> 3);
      int64_t at = first + r;
      at = at < rows ? at : rows - 1;      // rows behind the last one: any finite values, their results are not used
      if (o.idx) at = o.idx[at];
      row[i] = static_cast<const T *>(o.p) + at * o.ld + (((threadIdx.x & 7) ^ ((r >> 1) & 7)) << 3);
    }
  }
  __device__ __forceinline__ void issue(T *lds, int64_t offset) const {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i) load_lds16(row[i] + offset, lds + (i * 256 + wave * 64) * 8);
  }
};

// "Columns" operand: tile [64 k][128 m]; the rows of the next k-block are looked up one block ahead.
template <class T>
struct ColLoader {
  int64_t at[4];
  int col;
  __device__ __forceinline__ void look(const Operand &o, int64_t k0, int64_t rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int64_t r = k0 + i * 16 + (threadIdx.x >> 4);
      r = r < rows ? r : rows - 1;
      at[i] = o.idx ? o.idx[r] : r;
    }
  }
  __device__ __forceinline__ void tile(int64_t first, int64_t cols) {
    const int k = threadIdx.x >> 4;      // (i * 16 does not change k & 3)
    int64_t c = first + (((threadIdx.x & 15) ^ ((k & 3) << 2)) << 3);
    col = (int)(c + 8 <= cols ? c : cols - 8);
  }
  __device__ __forceinline__ void issue(const Operand &o, T *lds, int64_t offset) const {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i) load_lds16(static_cast<const T *>(o.p) + offset + at[i] * o.ld + col, lds + (i * 256 + wave * 64) * 8);
  }
};

template <class T>
__device__ __forceinline__ typename Mma<T>::v8 read_rows(const T *lds, int row0, int kk) {
  const int lane = threadIdx.x & 63, r = row0 + (lane & 31), c = kk * 2 + (lane >> 5);
  return *reinterpret_cast<const typename Mma<T>::v8 *>(lds + r * kTileK + ((c ^ ((r >> 1) & 7)) << 3));
}

template <class T>
__device__ __forceinline__ typename Mma<T>::v8 read_cols(const T *lds, int col0, int kk) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef short s8 __attribute__((ext_vector_type(8)));
  const int lane = threadIdx.x & 63, group = lane >> 4, p = lane & 15;
  const int col = col0 + (group & 1) * 16 + (p & 3) * 4, k = kk * 16 + (group >> 1) * 8 + (p >> 2);
  const T *at = lds + k * kTileM + (((col >> 3) ^ ((k & 3) << 2)) << 3) + (col & 7);
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at);
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(at + 4 * kTileM));
  const s8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(typename Mma<T>::v8, both);
}

// One k-block of 64 of the wave's 64 x 64: wave (wm, wn) of 2 x 2.
template <class T, bool kACols, bool kBCols>
__device__ __forceinline__ void mma_block(const T *a, const T *b, int wm, int wn, f32x16 (&acc)[2][2]) {
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    typename Mma<T>::v8 fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = kACols ? read_cols(a, wm * 64 + i * 32, kk) : read_rows(a, wm * 64 + i * 32, kk);
      fb[i] = kBCols ? read_cols(b, wn * 64 + i * 32, kk) : read_rows(b, wn * 64 + i * 32, kk);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = Mma<T>::mma(fa[i], fb[j], acc[i][j]);
  }
}

// Row of C in a 32 x 32 block that register j of a lane holds (its column is lane & 31).
__device__ __forceinline__ int mma_row(int j) { return (j & 3) + 8 * (j >> 2) + 4 * ((threadIdx.x & 63) >> 5); }

}  // namespace r3d

// Matrix products on the matrix cores (gfx950), for the fused kernels of r3d_loss.hip.
//
// C[m][n] = sum_k A(m,k) B(n,k) in tiles of BM x BN x 32, every wave FM x FN blocks of v_mfma_f32_32x32x16.  How an operand lies:
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

constexpr int kTileK = 32;      // k of a block: what one barrier is for
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Tile and waves.  A wave's share of 128 x 64 reads 0.75 of the 128 bytes a clock that LDS gives while the matrix cores are
// busy, one of 64 x 64 all of them; a tile of 256 x 256 takes 32 bytes a clock and CU out of L2, one of 128 x 128 64.
// ahead: blocks on their way to LDS beside the one that is multiplied (a block takes 0.4 us, HBM up to 1).  256 x 128 with two
// workgroups a CU, the one's products beside the other's exponentials, was no faster (1.56 ms against 1.47, 8192 x 161280 x 512).
template <int BM_, int BN_, int WM_, int WN_, int ahead_, int per_cu_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, threads = 64 * WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int a_elems = BM * kTileK, b_elems = BN * kTileK, buffer = a_elems + b_elems;
  static constexpr int ahead = ahead_, buffers = ahead + 1, per_cu = per_cu_;
};
using Big = Shape<256, 256, 2, 4, 3, 1>;
using Small = Shape<128, 128, 2, 2, 3, 2>;

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

typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes a lane from `g` to LDS, lanes in one line from the wave's base `to`.  Written out, because the compiler waits for all
// of the builtin's loads before every ds_read_b64_tr_b16 that follows, whichever buffer it reads; nothing but LDS is written, and
// wait_loads() stands between a load and the reads of what it brought.  (One wait state between m0 and its use.)
__device__ __forceinline__ void load_lds16(const void *g, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(g) : "m0", "memory");
}

// A thread's part of an operand tile of R rows (or columns) x kTileK: `per` pieces of 16 bytes, piece number i * threads + thread,
// from pointers that move from k-block to k-block.
template <class T, Lies L, int R, int kThreads>
struct Loader {
  static constexpr int per = R * kTileK / 8 / kThreads;
  static constexpr int row_lanes = R / 8;      // Cols: lanes to a row
  const T *at[per];
  int col;      // Cols: first column of the thread's pieces

  // The tile's first k-block.  first: first row (Rows, PiecesRows) or column of the tile; limit: how many there are.  What lies
  // behind is read from the last one, whatever it holds: its results are not used.
  __device__ __forceinline__ void tile(const Operand &o, int64_t first, int64_t limit) {
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int c = i * kThreads + threadIdx.x;
      if constexpr (L == Lies::Rows) {
        const int r = c >> 2;
        int64_t n = first + r;
        n = n < limit ? n : limit - 1;
        if (o.idx) n = o.idx[n];
        at[i] = static_cast<const T *>(o.p) + n * o.ld + (((c & 3) ^ ((r >> 2) & 3)) << 3);
      } else if constexpr (L == Lies::PiecesRows) {
        const int r = c % R, q = c / R;      // LDS: [4 pieces of k][R rows]
        int64_t n = first + r;
        n = n < limit ? n : limit - 1;
        at[i] = static_cast<const T *>(o.p) + (q * o.ld + n) * 8;
      } else if constexpr (L == Lies::PiecesCols) {
        const int k = c & 31, q = c >> 5;    // LDS: [R / 8 pieces of m][32 k], k in fours at k ^ 4 (q & 3)
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
  // Elements from one k-block to the next.
  static __device__ __forceinline__ int64_t step(const Operand &o) {
    return L == Lies::Rows ? kTileK : L == Lies::PiecesRows ? (kTileK / 8) * o.ld * 8 : L == Lies::PiecesCols ? kTileK * 8 : kTileK * o.ld;
  }
  __device__ __forceinline__ void move(int64_t elements) {
#pragma unroll
    for (int i = 0; i < per; ++i) at[i] += elements;
  }
  // Cols: row of the k-block that piece i is of.
  static __device__ __forceinline__ int row_of(int i) { return (i * kThreads + (int)threadIdx.x) / row_lanes; }
  // Cols: k-block kb, by row numbers (`numbers`: the block's, in LDS) or in order.
  __device__ __forceinline__ void to_block(const Operand &o, int kb, int rows, int64_t plane, const int32_t *numbers) {
    if constexpr (L == Lies::Cols) {
      const T *base = static_cast<const T *>(o.p) + plane;
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const int row = numbers ? numbers[row_of(i)] : min(kb * kTileK + row_of(i), rows - 1);
        at[i] = base + ((uint64_t)(uint32_t)row * (uint32_t)o.ld + (uint32_t)col);
      }
    }
  }
  __device__ __forceinline__ void issue(unsigned to) const {
#pragma unroll
    for (int i = 0; i < per; ++i) load_lds16(at[i], to + i * kThreads * 16);
  }
};

// Eight k of a lane's column, from two rows of fours (each lane's address: its row's, see above).
template <class T>
__device__ __forceinline__ typename Mma<T>::v8 turned(const T *lo_at, const T *hi_at) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)lo_at);
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)hi_at);
  return __builtin_bit_cast(typename Mma<T>::v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Fragment of the 32 rows (columns) from r0, k-step kk of 16: lane holds row lane & 31, k = (lane >> 5) * 8 + 0..7.
template <class T, Lies L, int R>
__device__ __forceinline__ typename Mma<T>::v8 fragment(const T *lds, int r0, int kk) {
  const int lane = threadIdx.x & 63;
  if constexpr (L == Lies::Rows || L == Lies::PiecesRows) {
    const int r = r0 + (lane & 31), q = kk * 2 + (lane >> 5);
    const T *at = L == Lies::Rows ? lds + r * kTileK + ((q ^ ((r >> 2) & 3)) << 3) : lds + (q * R + r) * 8;
    return *reinterpret_cast<const typename Mma<T>::v8 *>(at);
  } else {
    const int group = lane >> 4, p = lane & 15;
    const int c = r0 + (group & 1) * 16 + (p & 3) * 4, k = kk * 16 + (group >> 1) * 8 + (p >> 2), q = c >> 3;
    const T *lo_at, *hi_at;
    if constexpr (L == Lies::Cols) {
      lo_at = lds + k * R + ((q ^ ((k & 3) << 2)) << 3) + (c & 7);
      hi_at = lo_at + 4 * R;
    } else {
      lo_at = lds + (q * kTileK + (k ^ ((q & 3) << 2))) * 8 + (c & 7);
      hi_at = lds + (q * kTileK + ((k + 4) ^ ((q & 3) << 2))) * 8 + (c & 7);
    }
    return turned<T>(lo_at, hi_at);
  }
}

// (plane of A, plane of B) of the products of two operands in three planes of 8 bits each: what is left out is below 2^-24.  (Heads
// that stand in LDS; a stream takes them plane by plane.)
constexpr int kPairs = 6;
__device__ constexpr int kPlaneA[kPairs] = {0, 0, 1, 1, 0, 2}, kPlaneB[kPairs] = {0, 1, 0, 1, 2, 0};

// Waits until at most `left` of the wave's loads are on their way, then for the other waves.
template <int left>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(left) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A stream of k-blocks through LDS buffers: S::ahead blocks are on their way while one is multiplied.  One barrier a
// block: behind it the block is there for all waves, and all of them are done with the one before, whose buffer the next load
// takes.  The stream goes on over the tiles of a workgroup (`more`): their loads do not wait for a tile's end.
// kGather: the rows of a Cols operand B are taken by their numbers, b.idx.  Those of a block come to LDS S::ahead blocks before its
// own loads, with the loads of that earlier block (every wave for itself): looked up when they are wanted, by vector or by
// scalar loads, they hold up every step (dW of 119999 x 260 x 256: 73 us by scalar loads a step, 139 a step ahead).
// kPlanes = 3: operands of three planes; a block comes plane by plane, plane 0 stays in registers for the products of the other two
// (13 777 points x 20 244 classes x 512, all products: 6.5 ms, with two planes loaded for each product 7.5).
template <class T, class S, Lies LA, Lies LB, int kPlanes, bool kGather = false>
struct Stream {
  Operand a, b;
  Loader<T, LA, S::BM, S::threads> la;
  Loader<T, LB, S::BN, S::threads> lb;
  static constexpr int loads = Loader<T, LA, S::BM, S::threads>::per + Loader<T, LB, S::BN, S::threads>::per + (kGather ? 1 : 0);
  static constexpr int number_words = kGather ? 64 * S::buffers * (S::threads / 64) : 1;      // LDS that `numbers` has
  int rows_b;                  // rows of a Cols operand
  int kb, kb0, kb1, plane;     // the next to load
  int get, put;                // buffers: the next to multiply, the next to fill
  int number_kb, number_plane; // the next whose numbers are fetched
  bool dry;                    // nothing left to load
  unsigned base;               // LDS address of the wave's part of buffer 0
  int32_t *numbers;            // [S::buffers][64] of this wave: slot put holds those of the next block to load

  // The numbers of the block after those that have them (they go round within a tile; clamped behind the last row) to slot `slot`.
  __device__ __forceinline__ void fetch_numbers(int slot) {
    const int row = number_kb * kTileK + (threadIdx.x & 31);
    const int32_t *from = b.idx + (row < rows_b ? row : rows_b - 1);
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_void *)(numbers + slot * 64));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "m0", "memory");
    if (++number_plane < kPlanes) return;
    number_plane = 0;
    if (++number_kb == kb1) number_kb = kb0;
  }

  // k-blocks [first, end) of every tile (at least one); the loaders hold the first tile.
  template <class More>
  __device__ __forceinline__ void begin(T *lds, int first, int end, More &&more, int32_t *number_lds = nullptr) {
    kb = kb0 = number_kb = first;
    kb1 = end;
    get = put = plane = number_plane = 0;
    dry = false;
    base = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_void *)lds + (threadIdx.x >> 6) * 1024);
    la.move(first * la.step(a));
    if constexpr (kGather) {
      numbers = number_lds + (threadIdx.x >> 6) * 64 * S::buffers;
#pragma unroll
      for (int i = 0; i < S::ahead; ++i) fetch_numbers(i);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else if constexpr (LB == Lies::Cols) {
      lb.to_block(b, kb, rows_b, 0, nullptr);
    } else {
      lb.move(first * lb.step(b));
    }
#pragma unroll
    for (int i = 0; i < S::ahead; ++i) issue(more);
  }
  // The next block on its way; at the end of a tile `more()` sets A's loader for the next one and says whether there is one.
  // Without one the last block is loaded again: the count of loads on their way stays what wait_loads() takes it for.
  template <class More>
  __device__ __forceinline__ void issue(More &&more) {
    if constexpr (kGather) {
      lb.to_block(b, kb, rows_b, plane * b.plane, numbers + put * 64);
      fetch_numbers((put + S::ahead) % S::buffers);      // (the slot that was read S::buffers - S::ahead blocks ago)
    }
    const unsigned to = base + put * (S::buffer * (unsigned)sizeof(T));
    la.issue(to);
    lb.issue(to + S::a_elems * (unsigned)sizeof(T));
    put = (put + 1) % S::buffers;
    if (dry) return;
    if (kPlanes > 1 && ++plane < kPlanes) {
      la.move(a.plane);
      if constexpr (!kGather) lb.move(b.plane);
      return;
    }
    plane = 0;
    const int64_t back_a = (kPlanes - 1) * a.plane, back_b = (kPlanes - 1) * b.plane;
    if (++kb < kb1) {
      la.move(la.step(a) - back_a);
      if constexpr (!kGather) {
        if (LB == Lies::Cols && (kb + 1) * kTileK > rows_b) lb.to_block(b, kb, rows_b, 0, nullptr);
        else lb.move(lb.step(b) - back_b);
      }
      return;
    }
    if (!more()) {
      dry = true;
      kb = kb1 - 1;
      plane = kPlanes - 1;
      return;
    }
    kb = kb0;
    la.move(kb0 * la.step(a));
    if constexpr (!kGather) {
      if constexpr (LB == Lies::Cols) lb.to_block(b, kb, rows_b, 0, nullptr);
      else lb.move((kb0 + 1 - kb1) * lb.step(b) - back_b);
    }
  }
  // acc += all k-blocks of a tile whose rows from `rows` on are not there: a wave leaves out its blocks of 32 behind them.
  // (Waves w and w + 4 of the large shape share a SIMD and have different halves of the rows: what one leaves out the other gains.)
  template <class More>
  __device__ __forceinline__ void run(T *lds, f32x16 (&acc)[S::FM][S::FN], More &&more, int64_t rows) {
    const int64_t mine = (rows + 31) / 32 - (int)(threadIdx.x >> 6) / S::WN * S::FM;
    const int blocks = __builtin_amdgcn_readfirstlane((int)(mine < 0 ? 0 : mine < S::FM ? mine : S::FM));
    if (blocks == S::FM) run_blocks<true>(lds, acc, more, S::FM);
    else run_blocks<false>(lds, acc, more, blocks);
  }
  typedef typename Mma<T>::v8 v8;
  template <bool kAll>
  __device__ __forceinline__ void read(const T *lds, int kk, v8 (&fa)[S::FM], v8 (&fb)[S::FN], int blocks) const {
    const int wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
    const T *pa = lds + get * S::buffer, *pb = pa + S::a_elems;
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
      if (kAll || i < blocks) fa[i] = fragment<T, LA, S::BM>(pa, (wm * S::FM + i) * 32, kk);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) fb[j] = fragment<T, LB, S::BN>(pb, (wn * S::FN + j) * 32, kk);
  }
  template <bool kAll>
  static __device__ __forceinline__ void multiply(const v8 (&fa)[S::FM], const v8 (&fb)[S::FN], f32x16 (&acc)[S::FM][S::FN], int blocks) {
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
      if (kAll || i < blocks)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = Mma<T>::mma(fa[i], fb[j], acc[i][j]);
  }
  // A fragment is read one k-step before it is multiplied, over the blocks' borders too: the reads after a barrier would else hold
  // up the matrix cores of all waves at once.
  template <bool kAll, class More>
  __device__ __forceinline__ void run_blocks(T *lds, f32x16 (&acc)[S::FM][S::FN], More &&more, int blocks) {
    static_assert(kTileK == 32, "two k-steps a block");
    const int steps = kb1 - kb0;
    v8 fa[2][S::FM], fb[2][S::FN];
    auto next = [&] { get = (get + 1) % S::buffers; };
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    if constexpr (kPlanes == 1) {
      wait_loads<(S::ahead - 1) * loads>();
      read<kAll>(lds, 0, fa[0], fb[0], blocks);
      for (int s = 0; s < steps; ++s) {
        read<kAll>(lds, 1, fa[1], fb[1], blocks);
        fence();
        multiply<kAll>(fa[0], fb[0], acc, blocks);
        fence();
        // the next block is there, and all waves are done with the one before this one: its buffer is filled
        wait_loads<(S::ahead - 2) * loads>();
        issue(more);
        next();
        if (s + 1 < steps) read<kAll>(lds, 0, fa[0], fb[0], blocks);
        fence();
        multiply<kAll>(fa[1], fb[1], acc, blocks);
        fence();
      }
    } else {
      // the products of planes 00, 01 10 11, 02 20; behind a barrier the buffer of the plane before is filled, so its reads are
      // waited for (their first product stands between)
      auto turn = [&] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_loads<(S::ahead - 1) * loads>();
      };
      v8 fa0[2][S::FM], fb0[2][S::FN];
      for (int s = 0; s < steps; ++s) {
        turn();
        read<kAll>(lds, 0, fa0[0], fb0[0], blocks);
        if (s) multiply<kAll>(fa[1], fb0[1], acc, blocks);      // (20 of the block before)
        read<kAll>(lds, 1, fa0[1], fb0[1], blocks);
        issue(more);
        next();
        fence();
        multiply<kAll>(fa0[0], fb0[0], acc, blocks);
        turn();
        read<kAll>(lds, 0, fa[0], fb[0], blocks);
        issue(more);
        fence();
        multiply<kAll>(fa0[1], fb0[1], acc, blocks);
        fence();
        read<kAll>(lds, 1, fa[1], fb[1], blocks);
        next();
        fence();
        multiply<kAll>(fa0[0], fb[0], acc, blocks);
        multiply<kAll>(fa[0], fb0[0], acc, blocks);
        multiply<kAll>(fa[0], fb[0], acc, blocks);
        multiply<kAll>(fa0[1], fb[1], acc, blocks);
        multiply<kAll>(fa[1], fb0[1], acc, blocks);
        turn();
        read<kAll>(lds, 0, fa[0], fb[0], blocks);
        issue(more);
        fence();
        multiply<kAll>(fa[1], fb[1], acc, blocks);
        fence();
        read<kAll>(lds, 1, fa[1], fb[1], blocks);
        next();
        fence();
        multiply<kAll>(fa0[0], fb[0], acc, blocks);
        multiply<kAll>(fa[0], fb0[0], acc, blocks);
        multiply<kAll>(fa0[1], fb[1], acc, blocks);
      }
      multiply<kAll>(fa[1], fb0[1], acc, blocks);
    }
  }
  // Before LDS is used for anything else, and before the workgroup ends: nothing on its way to it.
  __device__ __forceinline__ void end() { wait_loads<0>(); }
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

// The sums over the 32 columns of a block whose register r holds v[r]: lane l < 8 of every 16 gets that of the row block_sum_row(l).
// A swap of 16 lanes and an addition make one register of two, then four rotated additions a register.
__device__ __forceinline__ float block_sum(const float (&v)[16]) {
  float mine = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v[k]), __builtin_bit_cast(unsigned, v[k + 8]), false, false);
    const unsigned lo = s[0], hi = s[1];      // (a cast of an element itself takes element 0)
    float t = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
    t += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, t), 0x128, 0xf, 0xf, false));      // row_ror:8
    t += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, t), 0x124, 0xf, 0xf, false));
    t += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, t), 0x122, 0xf, 0xf, false));
    t += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, t), 0x121, 0xf, 0xf, false));
    mine = (threadIdx.x & 15) == k ? t : mine;
  }
  return mine;
}
__device__ __forceinline__ int block_sum_row() { return mma_row((threadIdx.x & 7) + 8 * ((threadIdx.x >> 4) & 1)); }

// Work number of a block such that neighbours in number are on one XCD (blocks go round the eight) and share its L2.
__device__ __forceinline__ int64_t xcd_order(int64_t block, int64_t blocks) {
  const int64_t each = blocks / 8, rest = blocks % 8, x = block % 8, at = block / 8;
  return x * each + (x < rest ? x : rest) + at;
}

}  // namespace r3d

// The gradients of a linear head with few features and many classes (gfx950): logits are made again for dx and once more for dW,
// and their gradients never leave the registers.
//
// With at most 128 features a logit costs less to make than its gradient to store and read back: dl in memory is 6 bytes a logit
// over both products (1.3 ps at 4.7 TB/s), making it again 2 x 128 operations (0.2 ps at 1.4 PFLOP/s).  One kernel, three calls:
//   statistics: a wave keeps 32 or 64 points (their features as fragments) and meets all classes, the maximum and sum running;
//   dx: the same, with dx as the sums of a second product;
//   dW: it keeps as many classes and meets all points.
// What is met comes through LDS, 64 rows a time, two buffers, one barrier.  C of the first product (rows: what is met; columns:
// what is kept, one a lane) is, as it stands, the operand of the second one, whose k are the rows in the order in which the lanes
// have them: kept^T += met^T dl.  db is the sum of a lane's dl, before it is rounded.
//
// Bound by the vector unit: 417 824 points x 3114 classes x 64 fp16 take 425 / 475 / 585 us (643 where weights differ), 770 to 1200 cycles of a SIMD for every
// 32 x 32 logits, of which 16 exponentials take 256, their arguments, products and roundings some 300, the matrix cores 128 or 256
// beside them.  Two waves a SIMD (a wave's exponentials beside the other's products) is what the registers allow.
#include "r3d_loss.hpp"

namespace {
using namespace r3d;

constexpr int kThreads = 256, kRows = 64;

// kDP: features, padded; kSB: blocks of 32 rows that a wave keeps (points, for dW classes).
template <class V, class T, int kPlanes, int kDP, int kSB, Narrow kWhat>
__global__ __launch_bounds__(kThreads, 2) void k_ce_narrow(NarrowArgs a) {
  typedef typename Mma<T>::v8 v8;
  typedef T t4 __attribute__((ext_vector_type(4)));
  constexpr bool kPoints = kWhat != Narrow::Dw, kLse = kWhat == Narrow::Lse;
  constexpr int kPitch = kDP + 8, kPlane = kRows * kPitch, kCols = kDP / 8, kPer = kRows * kCols / kThreads, kPairCount = kPlanes == 3 ? kPairs : 1;
  __shared__ __attribute__((aligned(16))) T lds[2][kPlanes * kPlane];
  // bias of a class; or a point's base, its share (over the sum of its parts: its weight, or 1 where weights differ) and its weight
  __shared__ __attribute__((aligned(16))) float s_a[2][kRows], s_share[2][kRows], s_weight[2][kRows];
  __shared__ __attribute__((aligned(16))) int s_tgt[2][kRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, low = lane & 31, group = lane >> 4, sub = lane & 15;
  const int nc = a.counted->n, kept_n = kPoints ? nc : (int)a.v, met_n = kPoints ? (int)a.v : nc;
  const int64_t id = xcd_order(blockIdx.x, gridDim.x);
  const int split = (int)(id / a.tiles), kept0 = (int)(id - (int64_t)split * a.tiles) * (kThreads / 64 * 32 * kSB) + wave * 32 * kSB;
  if (kept0 - wave * 32 * kSB >= kept_n) return;
  const int chunks = (int)(((int64_t)met_n + kRows - 1) / kRows);
  const int c0 = (int)((int64_t)chunks * split / a.splits), c1 = (int)((int64_t)chunks * (split + 1) / a.splits);

  v8 own[kSB][kDP / 16][kPlanes];
  float own_a[kSB], own_sum[kSB], own_share[kSB];      // a point's base, sum and share; a class's bias
  int own_tgt[kSB];                       // a point's class
  int64_t own_row[kSB];
#pragma unroll
  for (int s = 0; s < kSB; ++s) {
    const int at = kept0 + s * 32 + low, in = at < kept_n ? at : kept_n - 1;
    own_row[s] = kPoints ? a.kept.idx[in] : in;
    const T *p = static_cast<const T *>(a.kept.p) + own_row[s] * a.kept.ld + half * 8;
#pragma unroll
    for (int k = 0; k < kDP / 16; ++k)
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl) own[s][k][pl] = *reinterpret_cast<const v8 *>(p + pl * a.kept.plane + k * 16);
    own_a[s] = kLse ? 0.0f : kPoints ? (at < kept_n ? a.base[at] : INFINITY) : a.bias2[at];
    own_sum[s] = kPoints && !kLse && at < kept_n ? a.sum[at] : 1.0f;
    own_share[s] = kPoints && !kLse && at < kept_n ? a.weight[at] * a.held / own_sum[s] : 0.0f;
    own_tgt[s] = kPoints && at < kept_n ? a.tgt[at] : -1;
  }
  f32x16 sums[kLse ? 1 : kDP / 32][kSB];
  float db[kSB], top[kSB], sum[kSB];
  if constexpr (!kLse) clear(sums);
#pragma unroll
  for (int s = 0; s < kSB; ++s) {
    db[s] = sum[s] = 0.0f;
    top[s] = -INFINITY;
  }

  // what is met: numbers two chunks ahead, rows one
  v8 reg[kPlanes][kPer];
  int64_t number[kPer];
  float next_p = 0.0f, next_q = 1.0f;      // wave 0: a class's bias, or a point's base and class; wave 1: a point's weight and sum
  auto numbers = [&](int c) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int r = c * kRows + (i * kThreads + (int)threadIdx.x) / kCols;
      r = r < met_n ? r : met_n - 1;      // (behind the last class: probability 0 by its bias; behind the last point: weight 0)
      number[i] = kPoints ? r : a.met.idx[r];
    }
  };
  auto fetch = [&](int c) {
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        reg[pl][i] = *reinterpret_cast<const v8 *>(static_cast<const T *>(a.met.p) + pl * a.met.plane + number[i] * a.met.ld + ((int)threadIdx.x % kCols) * 8);
    const int r = c * kRows + lane;
    if (wave == 0) {
      next_p = kPoints ? a.bias2[r] : r < nc ? a.base[r] : INFINITY;
      if constexpr (!kPoints) next_q = __builtin_bit_cast(float, r < nc ? a.tgt[r] : -1);
    } else if (!kPoints && wave == 1) {
      next_p = r < nc ? a.weight[r] * a.held : 0.0f;
      next_q = r < nc ? a.sum[r] : 1.0f;
    }
  };
  if (c0 < c1) {
    numbers(c0);
    fetch(c0);
    numbers(c0 + 1 < c1 ? c0 + 1 : c0);
  }
  for (int c = c0; c < c1; ++c) {
    const int buf = c & 1;
    T *met = lds[buf];
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = i * kThreads + threadIdx.x;
        *reinterpret_cast<v8 *>(met + pl * kPlane + at / kCols * kPitch + at % kCols * 8) = reg[pl][i];
      }
    if (wave == 0) {
      s_a[buf][lane] = next_p;
      if constexpr (!kPoints) s_tgt[buf][lane] = __builtin_bit_cast(int, next_q);
    } else if (!kPoints && wave == 1) {
      s_share[buf][lane] = (a.each ? 1.0f : next_p) / next_q;
      s_weight[buf][lane] = next_p;
    }
    __syncthreads();      // (whoever still multiplies reads the other buffer)
    if (c + 1 < c1) {
      fetch(c + 1);
      numbers(c + 2 < c1 ? c + 2 : c + 1);
    }
#pragma unroll
    for (int vb = 0; vb < kRows / 32; ++vb) {
      f32x16 acc[kSB];
#pragma unroll
      for (int s = 0; s < kSB; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[s][r] = 0.0f;
      const T *rows = met + (vb * 32 + low) * kPitch + half * 8;
#pragma unroll
      for (int pr = 0; pr < kPairCount; ++pr)
#pragma unroll
        for (int k = 0; k < kDP / 16; ++k) {
          // (classes by kPlaneA, points by kPlaneB, whichever are met: the logits of all three calls are the same bits)
          const v8 f = *reinterpret_cast<const v8 *>(rows + (kPoints ? kPlaneA : kPlaneB)[pr] * kPlane + k * 16);
#pragma unroll
          for (int s = 0; s < kSB; ++s) acc[s] = Mma<T>::mma(f, own[s][k][(kPoints ? kPlaneB : kPlaneA)[pr]], acc[s]);
        }
      float ma[16], mw[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        ma[r] = s_a[buf][vb * 32 + mma_row(r)];
        if constexpr (!kPoints) mw[r] = s_share[buf][vb * 32 + mma_row(r)];
      }
      if constexpr (kLse) {
#pragma unroll
        for (int s = 0; s < kSB; ++s) {
          float t[16], now = top[s];
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            t[r] = logit2(acc[s][r], ma[r]);
            now = fmaxf(now, t[r]);
          }
          const float base = base_of(now);
          sum[s] *= part_of(top[s], base);
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[s] += part_of(t[r], base);
          top[s] = now;
          const int d = own_tgt[s] - (c * kRows + vb * 32);
          if (__any(d >= 0 && d < 32)) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (d == mma_row(r)) a.hit[kept0 + s * 32 + low] = t[r];
          }
        }
        continue;
      }
      t4 q[kSB][4][kPlanes];
#pragma unroll
      for (int s = 0; s < kSB; ++s) {
        float p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r)
          p[r] = kPoints ? part_of(logit2(acc[s][r], ma[r]), own_a[s]) : part_of(logit2(acc[s][r], own_a[s]), ma[r]);
        if constexpr (kPoints) {
          const int d = own_tgt[s] - (c * kRows + vb * 32);
          if (__any(d >= 0 && d < 32)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] -= d == mma_row(r) ? own_sum[s] : 0.0f;
          }
        } else {
          // one weight for all: it is in the share already; else it is multiplied in behind the target's 1 (looked up there, row by
          // row, weights cost registers that a wave does not have: 99 us became 143, 200 000 x 1000 x 64 bf16)
          const int first = kept0 + s * 32, d = s_tgt[buf][vb * 32 + low] - first;
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] *= mw[r];
          if (__any(d >= 0 && d < 32)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] -= s_tgt[buf][vb * 32 + mma_row(r)] - first == low ? (a.each ? 1.0f : a.held) : 0.0f;
          }
          if (a.each) {
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] *= s_weight[buf][vb * 32 + mma_row(r)];
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float w = kPoints ? p[r] * own_share[s] : p[r];
          if constexpr (!kPoints) db[s] += w;
          if constexpr (kPlanes == 3) {
            T h, m, l;
            split3(w, h, m, l);
            q[s][r >> 2][0][r & 3] = h;
            q[s][r >> 2][1][r & 3] = m;
            q[s][r >> 2][2][r & 3] = l;
          } else {
            q[s][r >> 2][0][r & 3] = (T)w;
          }
        }
      }
      const T *wt = met + (vb * 32 + 4 * half + (sub >> 2)) * kPitch + (group & 1) * 16 + (sub & 3) * 4;
#pragma unroll
      for (int pr = 0; pr < kPairCount; ++pr)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int f = 0; f < kDP / 32; ++f) {
            const T *at = wt + kPlaneA[pr] * kPlane + 16 * k * kPitch + f * 32;
            const v8 m = turned<T>(at, at + 8 * kPitch);
#pragma unroll
            for (int s = 0; s < kSB; ++s)
              sums[f][s] = Mma<T>::mma(m, __builtin_shufflevector(q[s][2 * k][kPlaneB[pr]], q[s][2 * k + 1][kPlaneB[pr]], 0, 1, 2, 3, 4, 5, 6, 7), sums[f][s]);
          }
    }
  }

  if constexpr (kLse) {
    // a logit that is NaN leaves the maximum as it was and the sum NaN
#pragma unroll
    for (int s = 0; s < kSB; ++s) {
      const float ot = __shfl_xor(top[s], 32), os = __shfl_xor(sum[s], 32), now = fmaxf(top[s], ot), base = base_of(now);
      const int at = kept0 + s * 32 + low;
      if (half == 0 && at < kept_n) {
        a.part_m[split * a.split_stride + at] = now;
        a.part_l[split * a.split_stride + at] = sum[s] * part_of(top[s], base) + os * part_of(ot, base);
      }
    }
    return;
  }
  const float scale = a.final_out ? *a.scale * a.unheld : 1.0f;
#pragma unroll
  for (int s = 0; s < kSB; ++s) {
    const int at = kept0 + s * 32 + low;
    if (!kPoints && a.sums) {
      const float sum = db[s] + __shfl_xor(db[s], 32);
      if (half == 0 && at < kept_n) a.sums[split * a.sums_stride + at] = sum;
    }
    if (at >= kept_n || (!a.final_out && !a.out)) continue;
#pragma unroll
    for (int f = 0; f < kDP / 32; ++f)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int col = f * 32 + 8 * h + 4 * half;
        if (!a.final_out) {
          typedef float f4 __attribute__((ext_vector_type(4)));
          const f4 o = {sums[f][s][4 * h], sums[f][s][4 * h + 1], sums[f][s][4 * h + 2], sums[f][s][4 * h + 3]};
          *reinterpret_cast<f4 *>(a.out + split * a.split_stride + (int64_t)at * kDP + col) = o;
          continue;
        }
        V *out = static_cast<V *>(a.final_out) + own_row[s] * a.d + col;
        typedef V v4 __attribute__((ext_vector_type(4)));
        const v4 o = {(V)(sums[f][s][4 * h] * scale), (V)(sums[f][s][4 * h + 1] * scale), (V)(sums[f][s][4 * h + 2] * scale), (V)(sums[f][s][4 * h + 3] * scale)};
        if (a.vector_out && col + 4 <= a.d) {
          *reinterpret_cast<v4 *>(out) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < a.d) out[e] = o[e];
        }
      }
  }
}

// What fits the registers of two waves a SIMD.
constexpr int blocks_kept(Narrow what, int planes, int dp) {
  return what == Narrow::Lse ? (planes == 1 || dp == 64 ? 2 : 1) : planes == 1 && dp == 64 ? 2 : 1;
}

template <class V, class T, int kPlanes, int kDP, Narrow kWhat>
void launch(const NarrowArgs &a, hipStream_t st) {
  hipLaunchKernelGGL((k_ce_narrow<V, T, kPlanes, kDP, blocks_kept(kWhat, kPlanes, kDP), kWhat>), dim3((unsigned)(a.tiles * a.splits)), dim3(kThreads), 0, st, a);
}
template <class V, class T, int kPlanes, int kDP>
void launch(Narrow what, const NarrowArgs &a, hipStream_t st) {
  if (what == Narrow::Lse) launch<V, T, kPlanes, kDP, Narrow::Lse>(a, st);
  else if (what == Narrow::Dx) launch<V, T, kPlanes, kDP, Narrow::Dx>(a, st);
  else launch<V, T, kPlanes, kDP, Narrow::Dw>(a, st);
}
template <class V, class T, int kPlanes>
void launch(Narrow what, const NarrowArgs &a, int dp, hipStream_t st) {
  if (dp == 64) launch<V, T, kPlanes, 64>(what, a, st);
  else launch<V, T, kPlanes, 128>(what, a, st);
}
}  // namespace

namespace r3d {
int narrow_rows(Narrow what, int planes, int dp) { return kThreads / 64 * 32 * blocks_kept(what, planes, dp); }

void narrow(Narrow what, const NarrowArgs &a, int type, int dp, hipStream_t st) {
  if (type == R3D_T_F32) launch<float, __bf16, 3>(what, a, dp, st);
  else if (type == R3D_T_BF16) launch<__bf16, __bf16, 1>(what, a, dp, st);
  else launch<_Float16, _Float16, 1>(what, a, dp, st);
}
}  // namespace r3d

// Softmax cross entropy of a linear head, in pieces of the classes, without keeping the logits (gfx950).
//
//   l = x W^T + b,  loss_n = log sum_v exp l_nv - l_n,target;   dl = g_n (softmax(l) - onehot),  dx = dl W,  dW = dl^T x,  db = sum_n dl.
//
// This file: any sizes, and heads of up to 288 classes that stand in LDS; r3d_loss_few.hip: few classes and not many features;
// r3d_loss_narrow.hip: at most 128 features.  few_plan() and plan() choose.
//
// Forward: one product x W^T whose tiles end in a running maximum and sum per point (base 2), joined over the waves and over
// the splits of the classes.  Backward: for one piece of the classes at a time the logits once more, their gradient rounded to
// 16 bits into the workspace, and the two products with it.  Points whose target is ignored are left out at the start: the
// others are numbered in a line (stable, by prefix sums) and everything runs over that line, so they cost nothing and whatever
// their features hold (padding is rarely initialised) reaches no sum.
//
// Sums are in 32 bits (matrix cores, softmax statistics, gradients over points and classes), the mean's sum over points in 64.
// Rounded to fewer: dl, to the inputs' 16-bit type -- the matrix cores' operand; half a step of a term each, at random, beside
// half a step of the rounded result (dx of one point with few classes that matter: 2.5e-3 from 64 bits where 32-bit dl gives 1.7e-3, bfloat16).
// Two planes of dl would double the products that follow.  float16 has no room for a probability of 1e-6, so dl is held times 2^15 (|dl| <= 1) and
// the caller's weights of the points relative to the largest.  float32 operands are split into three bfloat16 planes (8 bits
// each, all 24) and multiplied as the six products that reach beyond 2^-24: 2.5 PFLOP/s of bfloat16 in six are more than the
// 0.16 of float32.
#include "r3d_host.hpp"
#include "r3d_loss.hpp"

#include <cmath>

namespace {
using namespace r3d;

// ---- which points count, and the operands --------------------------------------------------------------------------------
constexpr int kStartThreads = 1024, kStartRows = 4 * kStartThreads;
constexpr int kOneGroup = 16384;      // points one workgroup numbers by itself (in 10 us; two launches over many take 8)

// A side of the products: rows padded to whole k-blocks, split into planes where the type is wider.
struct PackArgs {
  const void *src;
  void *dst;
  int64_t ld, rows, width, ld_out, plane;      // width: of the source; ld_out a multiple of 64
  int32_t vector;                              // rows begin at multiples of 16 bytes
  int32_t blocks;
};

struct StartArgs {
  const void *target, *bias;
  int64_t n, v, ignore;
  int32_t wide_target, mean;
  int32_t *part, *idx, *place, *tgt;      // idx: point of a number, place: number of a point or -1, tgt: its class or -1 (not a class)
  Counted *counted;
  float *bias2;                           // in units of log 2, -inf behind the last class: those count for nothing anywhere
  int64_t v_pad;
  int32_t groups, bias_blocks;
  PackArgs pack[2];
};

__device__ __forceinline__ int64_t target_of(const StartArgs &a, int64_t i) {
  return a.wide_target ? static_cast<const int64_t *>(a.target)[i] : static_cast<const int32_t *>(a.target)[i];
}

// Numbers the points [first, first + kStartRows) that count from `at` on; returns the next number.  s: 16 words.
__device__ __forceinline__ int number_rows(const StartArgs &a, int64_t first, int at, int *s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t mine0 = first + threadIdx.x * 4;
  int64_t t[4];
  int mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t[j] = mine0 + j < a.n ? target_of(a, mine0 + j) : a.ignore;
    mine += t[j] != a.ignore;
  }
  int run = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  if (lane == 63) s[wave] = run;
  __syncthreads();
  int to = at + run - mine, end = at;
#pragma unroll
  for (int w = 0; w < kStartThreads / 64; ++w) {
    to += w < wave ? s[w] : 0;
    end += s[w];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (mine0 + j >= a.n) break;
    const bool counts = t[j] != a.ignore;
    a.place[mine0 + j] = counts ? to : -1;
    if (counts) {
      a.idx[to] = (int32_t)(mine0 + j);
      a.tgt[to++] = t[j] >= 0 && t[j] < a.v ? (int32_t)t[j] : -1;
    }
  }
  return end;
}

__device__ __forceinline__ void put_counted(const StartArgs &a, int n) {
  a.counted->n = n;
  a.counted->share = !a.mean ? 1.0f : n ? 1.0f / (float)n : 0.0f;
  a.counted->ticket = 0;
}

template <class T>
struct alignas(16) Piece {
  T v[8];
};

// A thread makes a piece of 8 values of a row.
template <class S, class T, int kPlanes>
__device__ __forceinline__ void pack_rows(const PackArgs &a, int block) {
  const unsigned each = (unsigned)(a.ld_out / 8);
  const int64_t all = a.rows * each;
  for (int64_t i = (int64_t)block * kStartThreads + threadIdx.x; i < all; i += (int64_t)a.blocks * kStartThreads) {
    const int64_t r = all <= UINT32_MAX ? (unsigned)i / each : i / each;
    const int64_t c = (i - r * each) * 8;
    const S *src = static_cast<const S *>(a.src) + r * a.ld + c;
    S v[8];
    if (c + 8 <= a.width && a.vector) {
      typedef S s4 __attribute__((ext_vector_type(16 / sizeof(S))));
#pragma unroll
      for (int k = 0; k < (int)sizeof(S) / 2; ++k) {
        const s4 w = reinterpret_cast<const s4 *>(src)[k];
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(S); ++e) v[k * (16 / sizeof(S)) + e] = w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < a.width ? src[e] : (S)0.0f;
    }
    Piece<T> out[kPlanes];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kPlanes == 3) split3(v[e], out[0].v[e], out[1].v[e], out[2].v[e]);
      else out[0].v[e] = v[e];
    }
#pragma unroll
    for (int k = 0; k < kPlanes; ++k) *reinterpret_cast<Piece<T> *>(static_cast<T *>(a.dst) + k * a.plane + r * a.ld_out + c) = out[k];
  }
}

// Everything the products need, in one launch: the points that count numbered (or, where they are many, counted by groups), the
// bias, the operands packed.
template <class S, class T, int kPlanes>
__global__ __launch_bounds__(kStartThreads) void k_ce_start(StartArgs a) {
  __shared__ int s[kStartThreads / 64];
  int block = blockIdx.x;
  if (block < a.groups) {
    if (a.n <= kOneGroup) {
      int at = 0;
      for (int64_t first = 0; first < a.n; first += kStartRows) at = number_rows(a, first, at, s);
      if (threadIdx.x == 0) put_counted(a, at);
      return;
    }
    int c = 0;
    const int64_t first = (int64_t)block * kStartRows + threadIdx.x * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) c += first + j < a.n && target_of(a, first + j) != a.ignore;
#pragma unroll
    for (int d = 32; d; d >>= 1) c += __shfl_xor(c, d);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
      c = 0;
      for (int w = 0; w < kStartThreads / 64; ++w) c += s[w];
      a.part[block] = c;
    }
    return;
  }
  block -= a.groups;
  if (block < a.bias_blocks) {
    const int64_t i = (int64_t)block * kStartThreads + threadIdx.x;
    if (i < a.v_pad) a.bias2[i] = i >= a.v ? -INFINITY : a.bias ? (float)static_cast<const S *>(a.bias)[i] * kLog2e : 0.0f;
    return;
  }
  block -= a.bias_blocks;
  if (block < a.pack[0].blocks) pack_rows<S, T, kPlanes>(a.pack[0], block);
  else pack_rows<S, T, kPlanes>(a.pack[1], block - a.pack[0].blocks);
}

__global__ __launch_bounds__(kStartThreads) void k_ce_index(StartArgs a) {
  __shared__ int s[kStartThreads / 64], s_before[kStartThreads / 64], s_all[kStartThreads / 64];
  int before = 0, all = 0;
  for (int b = threadIdx.x; b < a.groups; b += kStartThreads) {
    const int v = a.part[b];
    all += v;
    before += b < (int)blockIdx.x ? v : 0;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    before += __shfl_xor(before, d);
    all += __shfl_xor(all, d);
  }
  if ((threadIdx.x & 63) == 0) {
    s_before[threadIdx.x >> 6] = before;
    s_all[threadIdx.x >> 6] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < kStartThreads / 64; ++w) {
    before += s_before[w];
    all += s_all[w];
  }
  number_rows(a, (int64_t)blockIdx.x * kStartRows, before, s);
  if (blockIdx.x == 0 && threadIdx.x == 0) put_counted(a, all);
}

// ---- products --------------------------------------------------------------------------------------------------------------
struct Product {
  Operand a, b;
};

// Tiles in groups of 8 in n, so that the workgroups that run at a time share their rows of both operands.
__device__ __forceinline__ void tile_of(int64_t id, int64_t mtiles, int64_t ntiles, int64_t &mt, int64_t &nt) {
  const int64_t group = id / (8 * mtiles), first = group * 8, wide = ntiles - first < 8 ? ntiles - first : 8, in = id - group * 8 * mtiles;
  mt = in / wide;
  nt = first + in - mt * wide;
}

struct LseArgs {
  Product p;      // a: W [V], b: x [points]
  int64_t v, kb, ntiles;
  int32_t vtiles, splits;
  const float *bias2;
  const int32_t *tgt;
  const Counted *counted;
  float *part_m, *part_l, *hit;
  int64_t n_pad;
};

// Maximum and sum of 2^(logit * log2 e - maximum) over a split of the classes for the points of a tile.  The classes are the rows of C, so
// a lane holds 16 FM classes of each of its FN points: the statistics of a tile stay in its registers, lanes and waves are
// joined once at the end.  8192 points x 161 280 classes x 512 bf16: 1.5 ms, 0.9 PFLOP/s of the 1.41 that a large library product
// reaches here: a tile's exponentials (16 384 cycles of products, some 8000 of the vector unit) find no products to stand beside.
template <class T, class S, int kPlanes>
__global__ __launch_bounds__(S::threads, 2) void k_ce_lse(LseArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[S::buffers * S::buffer];
  const int nc = a.counted->n;
  const int64_t id = xcd_order(blockIdx.x, gridDim.x);
  const int split = (int)(id / a.ntiles);
  const int64_t n0 = (id - split * a.ntiles) * S::BN;
  if (n0 >= nc) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  float m[S::FN], l[S::FN];
  int tgt[S::FN];
#pragma unroll
  for (int j = 0; j < S::FN; ++j) {
    const int64_t col = n0 + (wn * S::FN + j) * 32 + (lane & 31);
    m[j] = -INFINITY;
    l[j] = 0.0f;
    tgt[j] = col < nc ? a.tgt[col] : -1;
  }
  const int vt0 = (int)((int64_t)a.vtiles * split / a.splits), vt1 = (int)((int64_t)a.vtiles * (split + 1) / a.splits);
  Stream<T, S, Lies::Rows, Lies::Rows, kPlanes> st;
  st.a = a.p.a;
  st.b = a.p.b;
  st.rows_b = 0;
  st.lb.tile(st.b, n0, nc);
  st.la.tile(st.a, (int64_t)vt0 * S::BM, a.v);
  int ahead = vt0;      // the tile that is being loaded
  auto more = [&] {
    if (++ahead >= vt1) return false;
    st.la.tile(st.a, (int64_t)ahead * S::BM, a.v);
    return true;
  };
  if (vt1 > vt0) st.begin(lds, 0, (int)a.kb, more);
  for (int vt = vt0; vt < vt1; ++vt) {
    f32x16 acc[S::FM][S::FN];
    clear(acc);
    st.run(lds, acc, more, a.v - (int64_t)vt * S::BM);
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
      const int vb = vt * S::BM + (wm * S::FM + i) * 32;
      float b[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) b[r] = a.bias2[vb + mma_row(r)];
#pragma unroll
      for (int j = 0; j < S::FN; ++j) {
        float t[16], top = m[j];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          t[r] = logit2(acc[i][j][r], b[r]);
          top = fmaxf(top, t[r]);
        }
        const float base = base_of(top);
        float sum = l[j] * part_of(m[j], base);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += part_of(t[r], base);
        m[j] = top;
        l[j] = sum;
        const int d = tgt[j] - vb;
        if (__any(d >= 0 && d < 32)) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (d == mma_row(r)) a.hit[n0 + (wn * S::FN + j) * 32 + (lane & 31)] = t[r];
        }
      }
    }
  }
  st.end();
  // a logit that is NaN leaves the maximum as it was and the sum NaN
  float *s_m = reinterpret_cast<float *>(lds), *s_l = s_m + S::WM * S::BN;
#pragma unroll
  for (int j = 0; j < S::FN; ++j) {
    const float om = __shfl_xor(m[j], 32), ol = __shfl_xor(l[j], 32), top = fmaxf(m[j], om), base = base_of(top);
    const float sum = l[j] * part_of(m[j], base) + ol * part_of(om, base);
    if (lane < 32) {
      const int at = wm * S::BN + (wn * S::FN + j) * 32 + lane;
      s_m[at] = top;
      s_l[at] = sum;
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < S::BN; c += S::threads) {
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < S::WM; ++w) top = fmaxf(top, s_m[w * S::BN + c]);
    const float base = base_of(top);
#pragma unroll
    for (int w = 0; w < S::WM; ++w) sum += s_l[w * S::BN + c] * part_of(s_m[w * S::BN + c], base);
    a.part_m[split * a.n_pad + n0 + c] = top;
    a.part_l[split * a.n_pad + n0 + c] = sum;
  }
}

struct JoinArgs {
  const float *part_m, *part_l, *hit;
  const int32_t *tgt, *place;
  Counted *counted;
  float *base, *sum, *each, *loss;
  double *sums;
  int64_t n, n_pad;
  int32_t splits, mean, points;      // points: of a workgroup
};

constexpr int kJoinThreads = 1024, kJoinSlices = 16;

__device__ __forceinline__ double group_sum(double d, double *s) {
#pragma unroll
  for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = d;
  __syncthreads();
  d = 0.0;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 64; ++w) d += s[w];
  return d;
}

// The splits joined; the loss of every point (each), or their sum: every workgroup leaves that of its points, the last one adds them
// up, always in the same order.  Over the points as the caller numbers them.  Few points have many splits: a workgroup takes 64 of
// them then and 16 threads share the splits of each (24 points x 38 322 classes, 300 splits: 140 us with one thread a point, 11 so;
// 8192 points of 8 splits: 10 and 22, every workgroup raises the one counter that tells which is the last).
int join_points(int splits) { return splits >= 16 ? kJoinThreads / kJoinSlices : kJoinThreads; }

__global__ __launch_bounds__(kJoinThreads) void k_ce_join(JoinArgs a) {
  __shared__ double s[kJoinThreads / 64];
  __shared__ int s_last;
  __shared__ float s_top[kJoinThreads], s_sum[kJoinThreads];
  const int points = a.points, slices = kJoinThreads / points, p = (int)threadIdx.x % points, slice = (int)threadIdx.x / points;
  double losses = 0.0;
  for (int64_t block = blockIdx.x; block * points < a.n; block += gridDim.x) {
    const int64_t i = block * points + p;
    const int at = i < a.n ? a.place[i] : -1;
    float top = -INFINITY, sum = 0.0f;
    if (at >= 0) {
#pragma unroll 4
      for (int k = slice; k < a.splits; k += slices) top = fmaxf(top, a.part_m[k * a.n_pad + at]);
      const float base = base_of(top);
#pragma unroll 4
      for (int k = slice; k < a.splits; k += slices) sum += a.part_l[k * a.n_pad + at] * part_of(a.part_m[k * a.n_pad + at], base);
    }
    if (slices > 1) {
      __syncthreads();
      s_top[threadIdx.x] = top;
      s_sum[threadIdx.x] = sum;
      __syncthreads();
      sum = 0.0f;
      for (int k = 0; k < slices; ++k) top = fmaxf(top, s_top[k * points + p]);
      const float base = base_of(top);
      for (int k = 0; k < slices; ++k) sum += s_sum[k * points + p] * part_of(s_top[k * points + p], base);
    }
    float loss = 0.0f;
    if (at >= 0 && slice == 0) {
      const bool fine = a.tgt[at] >= 0;      // a target that is no class: NaN, and so are its gradients
      a.base[at] = fine ? base_of(top) : NAN;
      a.sum[at] = sum;
      loss = fine ? point_loss(top, sum, a.hit[at]) : NAN;
    }
    losses += loss;
    if (a.each && i < a.n && slice == 0) a.each[i] = loss;
  }
  if (a.each) return;
  const double mine = group_sum(losses, s);
  if (threadIdx.x == 0) {
    a.sums[blockIdx.x] = mine;
    __threadfence();
    s_last = atomicAdd(&a.counted->ticket, 1) == (int)gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  double d = 0.0;
  for (int64_t b = threadIdx.x; b < gridDim.x; b += kJoinThreads) d += __hip_atomic_load(&a.sums[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  d = group_sum(d, s);
  if (threadIdx.x == 0) {
    const int c = a.counted->n;
    *a.loss = (float)(a.mean && c ? d / c : d);
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
// The factor that is taken out of dl: the one weight of a sum or a mean; for float16 the largest weight of single points.
__global__ __launch_bounds__(256) void k_ce_top(const float *grad, int64_t n, const int32_t *place, float *part) {
  __shared__ float s[4];
  float top = 0.0f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    if (place[i] >= 0 && fabsf(grad[i]) < INFINITY) top = fmaxf(top, fabsf(grad[i]));      // (what is no number or infinite is left out)
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

struct WeightArgs {
  const float *grad, *part;
  int32_t each, parts;
  const int32_t *idx, *place;
  const Counted *counted;
  float *scale;       // [1] the factor taken out of dl
  float *weight;      // of every point in the line, at most 1 where a factor is taken out; 0 up to n_pad
  int64_t n, n_pad, d;
  void *dx;           // rows of the points that do not count become zeros here, where nothing else writes them
};

template <class V>
__global__ __launch_bounds__(256) void k_ce_weight(WeightArgs a) {
  const int nc = a.counted->n;
  float scale;
  if (a.each) {
    scale = 0.0f;
    for (int b = threadIdx.x & 63; b < a.parts; b += 64) scale = fmaxf(scale, a.part[b]);
#pragma unroll
    for (int d = 32; d; d >>= 1) scale = fmaxf(scale, __shfl_xor(scale, d));
    if (!(scale > 0.0f)) scale = 1.0f;      // nothing to take out
  } else {
    scale = nc ? a.grad[0] * a.counted->share : 0.0f;      // (of no point: 0, whatever comes in)
  }
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < a.n_pad) a.weight[i] = i >= nc ? 0.0f : a.each ? a.grad[a.idx[i]] / scale : 1.0f;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.scale = scale;
  if (!a.dx) return;
  // a wave's 64 points: those that do not count one after the other
  const int64_t first = (int64_t)blockIdx.x * 256 + (threadIdx.x & ~63);
  uint64_t out = __ballot(i < a.n && a.place[i < a.n ? i : 0] < 0);
  V *dx = static_cast<V *>(a.dx);
  while (out) {
    const int64_t row = first + __builtin_ctzll(out);
    out &= out - 1;
    for (int64_t c = threadIdx.x & 63; c < a.d; c += 64) dx[row * a.d + c] = (V)0.0f;
  }
}

struct DlArgs {
  Product p;
  int64_t v, kb, ntiles;
  int64_t piece0, dl_plane, n_pad;      // first class of the piece
  int32_t vtiles, width;                // width: classes of the piece, a multiple of 64
  float held;                           // 2^15 for float16
  const float *bias2, *base, *sum, *weight;
  const int32_t *tgt;
  const Counted *counted;
  void *dl;        // [planes][width / 8][n_pad][8]
  float *sums;     // [tiles of points][piece]: db of a tile's points, before dl is rounded; or null
  int64_t piece;
};

// dl of a piece of the classes.  A lane holds 4 neighbouring classes of a point and its partner 32 lanes on the next 4: a swap
// makes pieces of 8, and 32 lanes write 512 contiguous bytes.  The same head: 2.1 ms, 2.6 GB written; what it takes beyond
// k_ce_lse is a workgroup's first loads and the stores.  (A workgroup that goes on to the next tile: 2.0, but 1 % more at 30 000 x 20 000 x 256.)
template <class T, class S, int kPlanes>
__global__ __launch_bounds__(S::threads, 2) void k_ce_dl(DlArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[S::buffers * S::buffer];
  const int nc = a.counted->n;
  int64_t vt, nt;
  tile_of(xcd_order(blockIdx.x, gridDim.x), a.vtiles, a.ntiles, vt, nt);
  const int64_t n0 = nt * S::BN;
  if (n0 >= nc) {
    for (int c = threadIdx.x; a.sums && c < S::BM && vt * S::BM + c < a.width; c += S::threads) a.sums[nt * a.piece + vt * S::BM + c] = 0.0f;
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  f32x16 acc[S::FM][S::FN];
  clear(acc);
  {
    Stream<T, S, Lies::Rows, Lies::Rows, kPlanes> st;
    st.a = a.p.a;
    st.b = a.p.b;
    st.rows_b = 0;
    st.la.tile(st.a, a.piece0 + vt * S::BM, a.v);
    st.lb.tile(st.b, n0, nc);
    auto more = [] { return false; };
    st.begin(lds, 0, (int)a.kb, more);
    st.run(lds, acc, more, (a.v - a.piece0 < a.width ? a.v - a.piece0 : a.width) - vt * S::BM);
    st.end();
  }
  T *dl = static_cast<T *>(a.dl);
  float *s_sum = reinterpret_cast<float *>(lds);      // [WN][BM]
  int64_t col[S::FN];
  int tgt[S::FN];
  float base[S::FN], sum[S::FN], share[S::FN];      // share: the weight over the sum of the parts
#pragma unroll
  for (int j = 0; j < S::FN; ++j) {
    col[j] = n0 + (wn * S::FN + j) * 32 + (lane & 31);
    const bool in = col[j] < nc;
    tgt[j] = in ? a.tgt[col[j]] : -1;
    base[j] = in ? a.base[col[j]] : 0.0f;
    sum[j] = in ? a.sum[col[j]] : 1.0f;
    share[j] = in ? a.weight[col[j]] * a.held / sum[j] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
    const int local = (int)vt * S::BM + (wm * S::FM + i) * 32;
    if (local >= a.width) continue;
    const int64_t vb = a.piece0 + local;
    float b[16], sums[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      b[r] = a.bias2[vb + mma_row(r)];
      sums[r] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int64_t d = tgt[j] - vb;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = part_of(logit2(acc[i][j][r], b[r]), base[j]);
      if (__any(d >= 0 && d < 32)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] -= d == mma_row(r) ? sum[j] : 0.0f;
      }
      typedef T t4 __attribute__((ext_vector_type(4)));
      typedef unsigned u2 __attribute__((ext_vector_type(2)));
      typedef unsigned u4 __attribute__((ext_vector_type(4)));
      t4 q[4][kPlanes];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float w = col[j] < nc ? p[r] * share[j] : 0.0f;
        sums[r] += w;
        if constexpr (kPlanes == 3) {
          T h, mm, l;
          split3(w, h, mm, l);
          q[r >> 2][0][r & 3] = h;
          q[r >> 2][1][r & 3] = mm;
          q[r >> 2][2][r & 3] = l;
        } else {
          q[r >> 2][0][r & 3] = (T)w;
        }
      }
#pragma unroll
      for (int k = 0; k < kPlanes; ++k)
#pragma unroll
        for (int h = 0; h < 4; h += 2) {
          const u2 even = __builtin_bit_cast(u2, q[h][k]), odd = __builtin_bit_cast(u2, q[h + 1][k]);
          const auto s0 = __builtin_amdgcn_permlane32_swap(even[0], odd[0], false, false);
          const auto s1 = __builtin_amdgcn_permlane32_swap(even[1], odd[1], false, false);
          const u4 out = {s0[0], s1[0], s0[1], s1[1]};
          const int64_t piece = local / 8 + h + (lane >> 5);
          *reinterpret_cast<u4 *>(dl + k * a.dl_plane + (piece * a.n_pad + col[j]) * 8) = out;
        }
    }
    if (a.sums) {
      const float mine = block_sum(sums);
      if ((lane & 15) < 8) s_sum[wn * S::BM + (wm * S::FM + i) * 32 + block_sum_row()] = mine;
    }
  }
  if (!a.sums) return;
  __syncthreads();
  for (int c = threadIdx.x; c < S::BM; c += S::threads) {
    const int local = (int)vt * S::BM + c;
    if (local >= a.width) break;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < S::WN; ++w) sum += s_sum[w * S::BM + c];
    a.sums[nt * a.piece + local] = sum;
  }
}

struct OutArgs {
  Product p;
  int64_t m, n, kb;                      // m: rows of the result, n: columns that are written
  int64_t limit_a, limit_b, rows_b;      // columns of the operands, rows of b
  int32_t points;                        // 0: m and the rest as given; 1: m is the points that count; 2: k is
  int32_t first, most;                   // 2: of those, `most` from number `first` on
  int32_t mtiles, ntiles, splits, add;
  const Counted *counted;
  float *out;                            // [splits][m_pad][ld], or null:
  int64_t ld, split_stride;
  void *final_out;                       // the result itself, rows through idx where given
  const int32_t *idx;
  const float *scale;
  float unheld;
};

// The products with dl: dx = dl W and dW = dl^T x, into 32-bit sums in the workspace or, where nothing is left to add, to the
// result.  The same head: 1.36 and 1.44 ms, 1.0 PFLOP/s; a block of 32 k costs LDS as many cycles as the matrix cores, 1024.
template <class V, class T, class S, Lies LA>
__global__ __launch_bounds__(S::threads, 2) void k_ce_out(OutArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[S::buffers * S::buffer];
  const int nc = a.points == 2 ? min(max(a.counted->n - a.first, 0), a.most) : a.counted->n;
  const int64_t id = xcd_order(blockIdx.x, gridDim.x), tiles = (int64_t)a.mtiles * a.ntiles;
  const int split = (int)(id / tiles);
  int64_t mt, nt;
  tile_of(id - split * tiles, a.mtiles, a.ntiles, mt, nt);
  const int64_t m0 = mt * S::BM, n0 = nt * S::BN;
  const int64_t m = a.points == 1 ? nc : a.m, kb = a.points == 2 ? (nc + kTileK - 1) / kTileK : a.kb;
  if (m0 >= m) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  f32x16 acc[S::FM][S::FN];
  clear(acc);
  const int64_t kb0 = kb * split / a.splits, kb1 = kb * (split + 1) / a.splits;
  constexpr bool kGather = LA == Lies::PiecesCols;      // x by the points' numbers
  constexpr int kPlanes = sizeof(V) == 4 ? 3 : 1;
  __shared__ int32_t numbers[Stream<T, S, LA, Lies::Cols, kPlanes, kGather>::number_words];
  if (kb1 > kb0) {
    Stream<T, S, LA, Lies::Cols, kPlanes, kGather> st;
    st.a = a.p.a;
    st.b = a.p.b;
    st.rows_b = (int)(a.points == 2 ? nc : a.rows_b);
    st.la.tile(st.a, m0, a.points == 1 ? nc : a.limit_a);
    st.lb.tile(st.b, n0, a.limit_b);
    auto more = [] { return false; };
    st.begin(lds, (int)kb0, (int)kb1, more, numbers);
    st.run(lds, acc, more, m - m0);
    st.end();
  }
  const float scale = a.final_out ? *a.scale * a.unheld : 1.0f;
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int64_t n = n0 + (wn * S::FN + j) * 32 + (lane & 31), row0 = m0 + (wm * S::FM + i) * 32;
      if (n >= a.n) continue;
      if (a.final_out) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t row = row0 + mma_row(r);
          if (row < m) static_cast<V *>(a.final_out)[(a.idx ? a.idx[row] : row) * a.ld + n] = (V)(acc[i][j][r] * scale);
        }
      } else {
        float *at = a.out + split * a.split_stride + row0 * a.ld + n;
        if (a.add) {      // (all loads before the first store: one at a time they are 128 latencies)
          float old[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) old[r] = row0 + mma_row(r) < m ? at[mma_row(r) * a.ld] : 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] += old[r];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (row0 + mma_row(r) < m) at[mma_row(r) * a.ld] = acc[i][j][r];
      }
    }
  }
}

struct Finish {
  const float *acc;
  int64_t ld, split_stride, rows, width;      // ld a multiple of 4
  int32_t splits, vector;                     // vector: four values of the result can be stored at once
  const int32_t *place;
  void *out;
};
struct FinishArgs {
  Finish of[3];
  const float *scale;
  float unheld;      // 2^-15 for float16
};

// Splits joined, the factor put back, one rounding; gridDim.y results.  A thread makes four neighbouring values; where there are
// many splits the four waves of a workgroup share them.
template <class V>
__global__ __launch_bounds__(256) void k_ce_finish(FinishArgs all) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  struct alignas(4 * sizeof(V)) Out {
    V v[4];
  };
  __shared__ f4 s[4][64];
  const Finish a = all.of[blockIdx.y];
  const float scale = *all.scale * all.unheld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slices = a.splits >= 8 ? 4 : 1;
  const unsigned each = (unsigned)((a.width + 3) / 4);
  const int64_t count = a.rows * each, step = (int64_t)gridDim.x * (256 / slices);
  for (int64_t i0 = (int64_t)blockIdx.x * (256 / slices); i0 < count; i0 += step) {
    const int64_t i = i0 + (slices == 4 ? lane : (int)threadIdx.x);
    const int64_t r = count <= UINT32_MAX ? (unsigned)i / each : i / each;
    const int64_t c = (i - r * each) * 4;
    const int64_t at = i >= count ? -1 : a.place ? a.place[r] : r;
    f4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at >= 0) {
      const float *from = a.acc + at * a.ld + c;
#pragma unroll 8
      for (int k = slices == 4 ? wave : 0; k < a.splits; k += slices) {
        const f4 v = *reinterpret_cast<const f4 *>(from + k * a.split_stride);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
      }
    }
    if (slices == 4) {
      s[wave][lane] = sum;
      __syncthreads();
      const f4 t[4] = {s[0][lane], s[1][lane], s[2][lane], s[3][lane]};
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = t[0][e] + t[1][e] + t[2][e] + t[3][e];
      __syncthreads();
      if (wave) continue;
    }
    if (i >= count) continue;
    Out out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out.v[e] = (V)(at >= 0 ? sum[e] * scale : 0.0f);
    V *to = static_cast<V *>(a.out) + r * a.width + c;
    if (a.vector) {
      *reinterpret_cast<Out *>(to) = out;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.width) to[e] = out.v[e];
    }
  }
}

// ---- a head that fits LDS ------------------------------------------------------------------------------------------------------
// Up to 288 classes of the 16-bit types: the head stands in LDS once a workgroup, and a wave goes its way alone, 32 points a
// time, without a barrier.  Their features come from memory as the fragments that the product takes (two lanes share a row: 32
// bytes each time, the rest of the cache line with the next k-steps), all classes' logits are in its registers, and in the
// backward pass dx = dl W is multiplied from there: the classes of a k-step are taken in the order in which the lanes have them.
// 119 999 x 260 x 256 fp16: 28 us forward (HBM 13; LDS 7 at 128 bytes a clock: every wave reads the head, 147 KB for 32 points), 71
// backward (HBM 42: x, dl and dx; LDS 14 at that rate), then dW 43 from dl.  Neither bounds it: a wave has 1.8 tiles, one after the other,
// behind a head that has to come first, and two waves a SIMD.  In tiles of r3d_mfma.hpp the whole step took 300, so 213 then.
// Beyond 64 features its points are cut where dl of all of them is more than it may hold (plan()).
constexpr int kHeadThreads = 512, kHeadBlocks = 9;

struct HeadArgs {
  Operand w, x;
  int64_t v, d;
  int32_t dp;
  const float *bias2;
  const int32_t *tgt, *idx;          // (these, and the points' other arrays, from number `first` on)
  const Counted *counted;
  int32_t first, most;               // the points of this launch: of those that count, `most` from number `first` on
  float *part_m, *part_l, *hit;      // forward
  // backward
  const float *base, *sum, *weight, *scale;
  float held, unheld;
  void *dl, *dx;                     // dl: pieces of 8 classes, or null
  float *sums;                       // [workgroups][classes padded to 32]: db of its points, or null
  int64_t n_pad;
  int32_t vector_out;
};

template <class T, int kVB, bool kGrad>
__global__ __launch_bounds__(kHeadThreads, 2) void k_ce_head(HeadArgs a) {
  typedef typename Mma<T>::v8 v8;
  typedef T t4 __attribute__((ext_vector_type(4)));
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int pitch = a.dp + 8;      // an odd number of 16 bytes: rows begin on different banks
  T *ws = reinterpret_cast<T *>(smem);
  float *bias2 = reinterpret_cast<float *>(ws + kVB * 32 * pitch);
  const int lane = threadIdx.x & 63, half = lane >> 5, low = lane & 31, group = lane >> 4, sub = lane & 15;
  const int nc = min(max(a.counted->n - a.first, 0), a.most), cols = a.dp / 8;
  if ((int)blockIdx.x * 32 >= nc) {
    if (kGrad && a.sums)
      for (int c = threadIdx.x; c < kVB * 32; c += kHeadThreads) a.sums[(int64_t)blockIdx.x * kVB * 32 + c] = 0.0f;
    return;
  }
  for (int i0 = threadIdx.x; i0 < kVB * 32 * cols; i0 += 6 * kHeadThreads) {      // (six loads on their way: 147 KB are 18 a thread)
    v8 v[6];
    int to[6];
#pragma unroll
    for (int e = 0; e < 6; ++e) {
      const int i = i0 + e * kHeadThreads, r = (unsigned)i / (unsigned)cols, c = (i - r * cols) * 8;
      to[e] = r < kVB * 32 ? r * pitch + c : -1;
      const int from = r < a.v ? r : (int)a.v - 1;      // (classes behind the last one: probability 0 by their bias)
      v[e] = *reinterpret_cast<const v8 *>(static_cast<const T *>(a.w.p) + from * a.w.ld + c);
    }
#pragma unroll
    for (int e = 0; e < 6; ++e)
      if (to[e] >= 0) *reinterpret_cast<v8 *>(ws + to[e]) = v[e];
  }
  for (int i = threadIdx.x; i < kVB * 32; i += kHeadThreads) bias2[i] = a.bias2[i];
  float *sums = bias2 + kVB * 32;      // [waves][classes] db of a wave's points, before dl is rounded (in registers they spill)
  if constexpr (kGrad)
    for (int i = threadIdx.x; i < kHeadThreads / 64 * kVB * 32; i += kHeadThreads) sums[i] = 0.0f;
  __syncthreads();
  float *mine = sums + (threadIdx.x >> 6) * kVB * 32 + block_sum_row();
  const float out_scale = kGrad && a.dx ? *a.scale * a.unheld : 1.0f;
  // neighbouring tiles go to different workgroups, so that a few tiles are a few workgroups' too
  for (int64_t tile = blockIdx.x + (int64_t)gridDim.x * (threadIdx.x >> 6); tile * 32 < nc; tile += (int64_t)gridDim.x * (kHeadThreads / 64)) {
    const int64_t point = tile * 32 + low;
    const bool in = point < nc;
    const int64_t row = a.idx[in ? point : nc - 1];
    const T *x = static_cast<const T *>(a.x.p) + row * a.x.ld + half * 8;
    f32x16 acc[kVB];
#pragma unroll
    for (int v = 0; v < kVB; ++v)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[v][r] = 0.0f;
    v8 f[2][4];
    auto features = [&](int k, int into) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[into][e] = *reinterpret_cast<const v8 *>(x + k + e * 16);
    };
    // the head's fragments three products ahead (left alone, the compiler reads one, waits, multiplies)
    auto multiply = [&](int k, int of) {
      const T *w = ws + low * pitch + half * 8 + k;
      v8 fa[4];
      auto read = [&](int i) { fa[i & 3] = *reinterpret_cast<const v8 *>(w + (i % kVB) * 32 * pitch + (i / kVB) * 16); };
#pragma unroll
      for (int i = 0; i < 3; ++i) read(i);
#pragma unroll
      for (int i = 0; i < 4 * kVB; ++i) {
        if (i + 3 < 4 * kVB) read(i + 3);
        acc[i % kVB] = Mma<T>::mma(fa[i & 3], f[of][i / kVB], acc[i % kVB]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    features(0, 0);
    int k = 0;
    for (; k + 128 <= a.dp; k += 128) {      // (dp is a multiple of 64)
      features(k + 64, 1);
      multiply(k, 0);
      if (k + 128 < a.dp) features(k + 128, 0);
      multiply(k + 64, 1);
    }
    if (k < a.dp) multiply(k, 0);
    const int t = in ? a.tgt[point] : -1;
    if constexpr (!kGrad) {
      float top = -INFINITY, sum = 0.0f, hit = -INFINITY;
#pragma unroll
      for (int v = 0; v < kVB; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          acc[v][r] = logit2(acc[v][r], bias2[v * 32 + mma_row(r)]);
          top = fmaxf(top, acc[v][r]);
          hit = t == v * 32 + mma_row(r) ? acc[v][r] : hit;
        }
      if (t >= 0 && (t >> 2 & 1) == half) a.hit[point] = hit;      // (the lane that holds the target's class)
      top = fmaxf(top, __shfl_xor(top, 32));
      const float base = base_of(top);
#pragma unroll
      for (int v = 0; v < kVB; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += part_of(acc[v][r], base);
      sum += __shfl_xor(sum, 32);
      if (in && half == 0) {
        a.part_m[point] = top;
        a.part_l[point] = sum;
      }
    } else {
      typedef unsigned u2 __attribute__((ext_vector_type(2)));
      typedef unsigned u4 __attribute__((ext_vector_type(4)));
      const float base = in ? a.base[point] : 0.0f, sum = in ? a.sum[point] : 1.0f, share = in ? a.weight[point] * a.held / sum : 0.0f;
      t4 q[kVB][4];
#pragma unroll
      for (int v = 0; v < kVB; ++v) {
        float w[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float p = part_of(logit2(acc[v][r], bias2[v * 32 + mma_row(r)]), base);
          p -= t == v * 32 + mma_row(r) ? sum : 0.0f;
          w[r] = in ? p * share : 0.0f;
          q[v][r >> 2][r & 3] = (T)w[r];
        }
        if (a.sums) {
          const float s = block_sum(w);
          if ((lane & 15) < 8) mine[v * 32] += s;
        }
        __builtin_amdgcn_sched_barrier(0);      // (a block at a time: all blocks' addresses and biases at once spill; of nine blocks 25 registers still do)
      }
      if (a.dl) {
#pragma unroll
        for (int v = 0; v < kVB; ++v)
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const u2 even = __builtin_bit_cast(u2, q[v][h]), odd = __builtin_bit_cast(u2, q[v][h + 1]);
            const auto s0 = __builtin_amdgcn_permlane32_swap(even[0], odd[0], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(even[1], odd[1], false, false);
            const u4 out = {s0[0], s1[0], s0[1], s1[1]};
            *reinterpret_cast<u4 *>(static_cast<T *>(a.dl) + ((int64_t)(v * 4 + h + half) * a.n_pad + point) * 8) = out;
          }
      }
      if (a.dx) {
        const T *wt = ws + (4 * half + (sub >> 2)) * pitch + (group & 1) * 16 + (sub & 3) * 4;
        T *out = static_cast<T *>(a.dx) + row * a.d;
        for (int f0 = 0; f0 < a.d; f0 += 32) {
          f32x16 g;
#pragma unroll
          for (int r = 0; r < 16; ++r) g[r] = 0.0f;
#pragma unroll
          for (int v = 0; v < kVB; ++v) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
              g = Mma<T>::mma(turned<T>(wt + (v * 32 + 16 * s) * pitch + f0, wt + (v * 32 + 16 * s + 8) * pitch + f0),
                              __builtin_shufflevector(q[v][2 * s], q[v][2 * s + 1], 0, 1, 2, 3, 4, 5, 6, 7), g);
            if (v % 3 == 2) __builtin_amdgcn_sched_barrier(0);
          }
          if (!in) continue;
          if (a.vector_out && f0 + 32 <= a.d) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const t4 o = {(T)(g[4 * h] * out_scale), (T)(g[4 * h + 1] * out_scale), (T)(g[4 * h + 2] * out_scale), (T)(g[4 * h + 3] * out_scale)};
              *reinterpret_cast<t4 *>(out + f0 + 8 * h + 4 * half) = o;
            }
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (f0 + mma_row(r) < a.d) out[f0 + mma_row(r)] = (T)(g[r] * out_scale);
          }
        }
      }
    }
  }
  if constexpr (kGrad) {
    if (!a.sums) return;
    __syncthreads();
    for (int c = threadIdx.x; c < kVB * 32; c += kHeadThreads) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kHeadThreads / 64; ++w) sum += sums[w * kVB * 32 + c];
      a.sums[(int64_t)blockIdx.x * kVB * 32 + c] = sum;
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// What a piece's dl may take.  8192 points x 161280 classes x 512: 8.4 ms with 64 MB, 6.6 with 256, 6.3 with 512 and with all 2.6 GB.
constexpr int64_t kPieceBytes = 512ll << 20;
constexpr int kCus = 256, kHeadLds = 160 * 1024;
constexpr int kPadK = 64;      // a head in LDS and few features: padded to whole cache lines; pieces of the classes

int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t tiles_of(int64_t m, int64_t n, int64_t bm, int64_t bn) { return (up(m, bm) / bm) * (up(n, bn) / bn); }

// Parts in which the long axis of a product is cut: enough workgroups for the chip (two of the small shape a CU: dW of 119 999 x
// 260 x 256 takes 58 us with one, 45 with two), and no last round that leaves most of it idle.
int cut(int64_t tiles, int64_t slots, int64_t most) {
  int64_t best = 1;
  double best_share = 0.0;
  for (int k = 0; k <= 4; ++k) {      // one part, and what fills one to four rounds
    int64_t s = k ? k * slots / tiles : 1;
    s = s > most ? most : s > 1024 ? 1024 : s;
    if (s < 1) s = 1;
    const int64_t all = tiles * s, rounds = (all + slots - 1) / slots;
    const double share = (double)all / (double)(rounds * slots);
    if (share > best_share * 1.05) {
      best = s;
      best_share = share;
    }
  }
  return (int)best;
}

// Parts in which the rows that meet are cut (r3d_loss_narrow.hip): rounds of workgroups times 2.5 us for every 64 rows of a part
// (417 824 points x 3114 classes x 64: 2.3), and what parts cost that have to be added, written and read at 4.7 TB/s.
int narrow_splits(int64_t kept, int64_t rows, int64_t slots, int64_t met, int64_t bytes) {
  const int64_t tiles = (kept + rows - 1) / rows, chunks = (met + 63) / 64;
  int64_t best = 1;
  double best_us = 0.0;
  for (int k = 0; k < 4; ++k) {
    int64_t s = k ? k * slots / tiles : 1;
    s = s < 1 ? 1 : s > chunks ? chunks : s;
    const double us = (double)((tiles * s + slots - 1) / slots * ((chunks + s - 1) / s)) * 2.5 + (s > 1 ? (double)(s * kept * bytes) * 2.0 / 4.7e6 : 0.0);
    if (k == 0 || us < best_us) {
      best = s;
      best_us = us;
    }
  }
  return (int)best;
}

// A product's tiles: the large ones where their rounds take less time than those of the small ones.  A large tile is four times the
// work; the small one loses a fifth to LDS (each number that it holds is multiplied half as often).  A large tile with rows behind
// the last one takes its loads, 0.3 of it, and the blocks of 32 that are there.  70 657 points x 152 classes x 586 fp32, logits: 183
// us in large tiles, 214 in small; 35 061 x 260 x 256 fp32, dx: 80 and 69.
bool large_tiles(int64_t m, int64_t n, int64_t most_splits) {
  auto rounds = [&](int64_t tiles) {
    const int64_t s = cut(tiles, kCus, most_splits);
    return (double)((tiles * s + kCus - 1) / kCus) / (double)s;
  };
  const int64_t down = up(m, Big::BM) / Big::BM;
  const double full = (double)(m / Big::BM) + (m % Big::BM ? 0.3 + 0.7 * (double)up(m % Big::BM, 32) / Big::BM : 0.0);
  return rounds(tiles_of(m, n, Big::BM, Big::BN)) * 4 * full / (double)down <= rounds(tiles_of(m, n, Small::BM, Small::BN)) * 1.2;
}

struct Plan {
  bool direct;      // the operands are multiplied where they lie
  int planes, type_bytes;
  int64_t dp, n_pad, v_pad, piece;
  bool lse_big, dl_big, dx_big, dw_big;
  bool narrow;      // dl stays in registers (r3d_loss_narrow.hip)
  int lse_splits, dx_splits, dw_splits, db_parts, top_parts, groups;
  int head;                     // blocks of 32 classes of a head that fits LDS, or 0
  int64_t head_points, head_ranges, dl_rows;      // its points whose dl is held at a time; rows of dl
  size_t head_lds;
  bool dx_final, dw_final;      // nothing to add: straight into the result
  // kept from the forward to the backward pass
  Counted *counted;
  int32_t *idx, *place, *tgt;
  float *base, *sum, *bias2;
  void *xp, *wp;
  size_t state_bytes;
  // workspace
  int32_t *part;
  float *part_m, *part_l, *hit;
  double *sums;
  float *top, *scale, *weight, *accx, *accw, *accb;
  void *dl;
  size_t bytes;
};

int64_t head_groups(int64_t points) { return up(points, 32) / 32 < kCus ? up(points, 32) / 32 : kCus; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

Plan plan(const r3d_linear_ce_t &d, bool backward, void *workspace) {
  Plan p{};
  p.planes = d.type == R3D_T_F32 ? 3 : 1;
  p.type_bytes = d.type == R3D_T_F32 ? 4 : 2;
  p.dp = up(d.d, kPadK);
  p.n_pad = up(d.n, Big::BN);
  p.v_pad = up(d.v, Big::BM);
  p.head_lds = (size_t)up(d.v, 32) * ((p.dp + 8) * 2 + 4 + kHeadThreads / 64 * 4);
  p.head = p.planes == 1 && d.v <= kHeadBlocks * 32 && p.head_lds <= (size_t)kHeadLds ? (int)(up(d.v, 32) / 32) : 0;
  // Few features: logits are made again rather than their gradients stored.  Stored / made again, us, forward and backward: bf16
  // 417 824 x 3114 x 9 4350 / 1400, 200 000 x 1000 x 64 630 / 350, 20 000 x 20 000 x 128 1050 / 690, 2000 x 161 280 x 128 920 / 600;
  // fp32 199 334 x 878 x 10 2010 / 610, 5000 x 5000 x 128 330 / 240.  A head in LDS with 128 features stores: 100 000 x 150 x 128
  // 106 / 117, 126 403 x 260 x 128 160 / 157; with 64 it does not: 270 597 x 260 x 64 237 / 214, 200 000 x 150 x 64 142 / 143.
  p.narrow = p.dp <= 128 && !(p.head && p.dp > 64);
  if (!p.head && !p.narrow) p.dp = up(d.d, kTileK);      // (13 421 x 80 469 x 139 bf16: padded to 160 3370 us, to 192 3500)
  p.direct = p.planes == 1 && d.d == p.dp && d.ld_x % 8 == 0 && d.ld_w % 8 == 0 && aligned16(d.x) && aligned16(d.w);
  const int64_t slots = p.planes == 3 && p.dp > 64 ? kCus : 2 * kCus;      // workgroups of r3d_loss_narrow.hip that the chip holds
  p.groups = d.n <= kOneGroup ? 1 : (int)((d.n + kStartRows - 1) / kStartRows);
  Carver k(d.state);
  p.counted = k.take<Counted>(1);
  p.idx = k.take<int32_t>(d.n);
  p.place = k.take<int32_t>(d.n);
  p.tgt = k.take<int32_t>(d.n);
  p.base = k.take<float>(d.n);
  p.sum = k.take<float>(d.n);
  p.bias2 = k.take<float>(p.v_pad);
  if (!p.direct) {
    p.xp = k.take<uint16_t>((size_t)p.planes * d.n * p.dp);
    p.wp = k.take<uint16_t>((size_t)p.planes * d.v * p.dp);
  }
  p.state_bytes = k.off;
  Carver c(workspace);
  if (!backward) {
    p.lse_big = p.planes == 1 && large_tiles(d.v, d.n, up(d.v, Big::BM) / Big::BM);
    const int64_t bm = p.lse_big ? Big::BM : Small::BM, bn = p.lse_big ? Big::BN : Small::BN;
    const int64_t of_points = p.narrow ? narrow_rows(Narrow::Lse, p.planes, (int)p.dp) : 0;
    p.lse_splits = p.head ? 1 : p.narrow ? narrow_splits(d.n, of_points, slots, d.v, 8) : cut(up(d.n, bn) / bn, kCus * (p.lse_big ? Big::per_cu : Small::per_cu), up(d.v, bm) / bm);
    p.part = c.take<int32_t>(p.groups);
    p.part_m = c.take<float>((size_t)p.lse_splits * p.n_pad);
    p.part_l = c.take<float>((size_t)p.lse_splits * p.n_pad);
    p.hit = c.take<float>(p.n_pad);
    p.sums = c.take<double>(kCus);
  } else {
    const int64_t v64 = up(d.v, kPadK);
    p.top_parts = (int)(d.n < 256 * 256 ? (d.n + 255) / 256 : 256);
    p.top = c.take<float>(p.top_parts);
    p.scale = c.take<float>(1);
    p.weight = c.take<float>(p.n_pad);
    if (p.narrow) {
      const int64_t of_points = narrow_rows(Narrow::Dx, p.planes, (int)p.dp), of_classes = narrow_rows(Narrow::Dw, p.planes, (int)p.dp);
      p.piece = v64;
      p.dx_splits = narrow_splits(d.n, of_points, slots, d.v, p.dp * 4);
      p.dw_splits = p.db_parts = narrow_splits(d.v, of_classes, slots, d.n, p.dp * 4);
      p.dx_final = p.dx_splits == 1;
      p.dw_final = p.dw_splits == 1;
      if (!p.dx_final && d.dx) p.accx = c.take<float>((size_t)p.dx_splits * p.n_pad * p.dp);
      if (!p.dw_final && d.dw) p.accw = c.take<float>((size_t)p.dw_splits * v64 * p.dp);
      if (d.db) p.accb = c.take<float>((size_t)p.db_parts * v64);
      p.bytes = c.off;
      return p;
    }
    int64_t piece = d.piece > 0 ? up(d.piece, kPadK) : kPieceBytes / (p.n_pad * 2 * p.planes) / Big::BM * Big::BM;
    if (piece < Small::BM) piece = Small::BM;
    p.piece = piece < v64 ? piece : v64;
    if (d.piece == 0) p.piece = up((v64 + (v64 + p.piece - 1) / p.piece - 1) / ((v64 + p.piece - 1) / p.piece), Big::BM);      // pieces of one size
    if (p.piece > v64 || p.head) p.piece = v64;
    // A head in LDS takes all classes at a time, so it is its points that are cut where dl is too much, into what a piece takes.
    p.dl_rows = p.head_points = p.n_pad;
    if (p.head && d.dw) {
      const int64_t bytes = d.piece > 0 && d.piece < d.v ? p.n_pad * up(d.piece, kPadK) * 2 : kPieceBytes;
      const int64_t rows = bytes / (v64 * 2) / Big::BN * Big::BN;
      p.dl_rows = p.head_points = rows < Big::BN ? Big::BN : rows < p.n_pad ? rows : p.n_pad;
    }
    p.head_ranges = (d.n + p.head_points - 1) / p.head_points;
    p.dl_big = p.planes == 1 && large_tiles(p.piece, d.n, 1);
    const int64_t kx = p.piece / 256, kw = p.dl_rows / 256;
    p.dx_big = p.planes == 1 && large_tiles(d.n, p.dp, kx);
    p.dw_big = p.planes == 1 && large_tiles(p.piece, p.dp, kw);
    auto tiles = [&](int64_t m, int64_t n, bool big) { return big ? tiles_of(m, n, Big::BM, Big::BN) : tiles_of(m, n, Small::BM, Small::BN); };
    p.dx_splits = cut(tiles(d.n, p.dp, p.dx_big), kCus * (p.dx_big ? Big::per_cu : Small::per_cu), kx);
    p.dw_splits = cut(tiles(p.piece, p.dp, p.dw_big), kCus * (p.dw_big ? Big::per_cu : Small::per_cu), kw);
    p.dx_final = p.head || (p.dx_splits == 1 && p.piece >= d.v);
    p.dw_final = p.dw_splits == 1 && p.head_ranges == 1;
    p.dl = c.take<uint16_t>(p.head && !d.dw ? 0 : (size_t)p.planes * p.dl_rows * p.piece);
    if (!p.dx_final) p.accx = c.take<float>((size_t)p.dx_splits * p.n_pad * p.dp);
    p.accw = c.take<float>((size_t)(p.dw_final || !d.dw ? 0 : p.dw_splits) * p.piece * p.dp);
    // db: a part for every tile of points (the tiles of dl) or every workgroup of a head in LDS
    p.db_parts = p.head ? (int)(p.head_ranges * head_groups(d.n < p.head_points ? d.n : p.head_points)) : (int)(up(d.n, p.dl_big ? Big::BN : Small::BN) / (p.dl_big ? Big::BN : Small::BN));
    p.accb = c.take<float>((size_t)p.db_parts * p.piece);
  }
  p.bytes = c.off;
  return p;
}

int check(const r3d_linear_ce_t *d) {
  if (!d) return fail(R3D_E_ARG, "linear_ce: null descriptor");
  if (d->n <= 0 || d->v <= 0 || d->d <= 0 || d->n > INT32_MAX - 1024 || d->v > INT32_MAX - 1024 || d->d > (1 << 20) || d->ld_x < d->d || d->ld_w < d->d ||
      d->ld_x > INT32_MAX || d->ld_w > INT32_MAX || d->piece < 0)
    return fail(R3D_E_ARG, "linear_ce: bad size");
  if (d->type != R3D_T_F32 && d->type != R3D_T_BF16 && d->type != R3D_T_F16) return fail(R3D_E_ARG, "linear_ce: type");
  if (d->target_type != R3D_T_I32 && d->target_type != R3D_T_I64) return fail(R3D_E_ARG, "linear_ce: type of the targets");
  if (d->reduction != R3D_CE_NONE && d->reduction != R3D_CE_SUM && d->reduction != R3D_CE_MEAN) return fail(R3D_E_ARG, "linear_ce: reduction");
  return R3D_OK;
}

// What the kernels take for granted of the addresses that a call brings.
int check_aligned(const r3d_linear_ce_t &d, const void *workspace) {
  const size_t size = d.type == R3D_T_F32 ? 4 : 2;
  if (!aligned(d.state, 16) || !aligned(workspace, 16)) return fail(R3D_E_ARG, "linear_ce: state and workspace must be 16-byte aligned");
  if (!aligned(d.x, size) || !aligned(d.w, size) || !aligned(d.bias, size) || !aligned(d.dx, size) || !aligned(d.dw, size) || !aligned(d.db, size) ||
      !aligned(d.target, d.target_type == R3D_T_I64 ? 8 : 4) || !aligned(d.loss, 4) || !aligned(d.grad, 4))
    return fail(R3D_E_ARG, "linear_ce: an array is not aligned to its type");
  return R3D_OK;
}

// The operands as the products take them: in place, or as the forward pass has packed them.
void operands(const r3d_linear_ce_t &d, const Plan &p, Operand &x, Operand &w) {
  x = p.direct ? Operand{d.x, d.ld_x, 0, p.idx} : Operand{p.xp, p.dp, d.n * p.dp, p.idx};
  w = p.direct ? Operand{d.w, d.ld_w, 0, nullptr} : Operand{p.wp, p.dp, d.v * p.dp, nullptr};
}

PackArgs pack_args(const Plan &p, const void *src, void *dst, int64_t ld, int64_t rows, int64_t width) {
  const bool vector = aligned16(src) && ld * p.type_bytes % 16 == 0;
  return PackArgs{src, dst, ld, rows, width, p.dp, rows * p.dp, vector, blocks_for(rows * p.dp / 8, kStartThreads * 2, 1024)};
}

// Three planes take the small tiles alone: plane 0 beside the others' fragments and the sums of a large one are more than 256
// registers, and six products for three planes' loads are enough for the matrix cores (6 x 512 cycles of them a k-block and CU,
// 2300 of LDS).
template <int kPlanes, class F>
void with_shape(bool big, F &&f) {
  if constexpr (kPlanes == 1) {
    if (big) return f(Big{});
  }
  f(Small{});
}

template <class T, class S, int kPlanes>
void lse(LseArgs a, const Plan &p, int64_t n, int64_t v, hipStream_t st) {
  a.ntiles = up(n, S::BN) / S::BN;
  a.vtiles = (int)(up(v, S::BM) / S::BM);
  hipLaunchKernelGGL((k_ce_lse<T, S, kPlanes>), dim3((unsigned)(a.ntiles * p.lse_splits)), dim3(S::threads), 0, st, a);
}

void join(const r3d_linear_ce_t &d, const Plan &p, hipStream_t st) {
  JoinArgs ja{p.part_m, p.part_l, p.hit, p.tgt, p.place, p.counted, p.base, p.sum, d.reduction == R3D_CE_NONE ? d.loss : nullptr, d.loss, p.sums, d.n, p.n_pad,
              p.lse_splits, d.reduction == R3D_CE_MEAN};
  ja.points = join_points(p.lse_splits);
  // a sum: a workgroup a CU, each raises the one counter (270 597 points: 39 us with one for every 256 points, 13 so)
  hipLaunchKernelGGL(k_ce_join, dim3(blocks_for(d.n, ja.points, d.reduction == R3D_CE_NONE ? INT32_MAX : kCus)), dim3(kJoinThreads), 0, st, ja);
}

HeadArgs head_args(const r3d_linear_ce_t &d, const Plan &p) {
  HeadArgs a{};
  operands(d, p, a.x, a.w);
  a.v = d.v;
  a.d = d.d;
  a.dp = (int)p.dp;
  a.bias2 = p.bias2;
  a.tgt = p.tgt;
  a.idx = p.idx;
  a.counted = p.counted;
  a.most = (int32_t)d.n;
  a.part_m = p.part_m;
  a.part_l = p.part_l;
  a.hit = p.hit;
  a.base = p.base;
  a.sum = p.sum;
  a.weight = p.weight;
  a.scale = p.scale;
  a.dl = p.dl;
  a.dx = d.dx;
  a.n_pad = p.n_pad;
  a.vector_out = d.d % 4 == 0 && aligned16(d.dx);
  return a;
}

template <class T, bool kGrad>
int head(const HeadArgs &a, const Plan &p, int64_t points, hipStream_t st) {
  auto run = [&](auto *kernel) {
    if (p.head_lds > 64 * 1024)
      R3D_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.head_lds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)head_groups(points)), dim3(kHeadThreads), p.head_lds, st, a);
    return R3D_OK;
  };
  switch (p.head) {
    case 1: return run(&k_ce_head<T, 1, kGrad>);
    case 2: return run(&k_ce_head<T, 2, kGrad>);
    case 3: return run(&k_ce_head<T, 3, kGrad>);
    case 4: return run(&k_ce_head<T, 4, kGrad>);
    case 5: return run(&k_ce_head<T, 5, kGrad>);
    case 6: return run(&k_ce_head<T, 6, kGrad>);
    case 7: return run(&k_ce_head<T, 7, kGrad>);
    case 8: return run(&k_ce_head<T, 8, kGrad>);
    default: return run(&k_ce_head<T, 9, kGrad>);
  }
}

template <class S, class T, int kPlanes>
int forward(const r3d_linear_ce_t &d, const Plan &p, hipStream_t st) {
  const bool mean = d.reduction == R3D_CE_MEAN;
  StartArgs sa{};
  sa.target = d.target;
  sa.bias = d.bias;
  sa.n = d.n;
  sa.v = d.v;
  sa.ignore = d.ignore_index;
  sa.wide_target = d.target_type == R3D_T_I64;
  sa.mean = mean;
  sa.part = p.part;
  sa.idx = p.idx;
  sa.place = p.place;
  sa.tgt = p.tgt;
  sa.counted = p.counted;
  sa.bias2 = p.bias2;
  sa.v_pad = p.v_pad;
  sa.groups = p.groups;
  sa.bias_blocks = blocks_for(p.v_pad, kStartThreads, 1 << 30);
  if (!p.direct) {
    sa.pack[0] = pack_args(p, d.w, p.wp, d.ld_w, d.v, d.d);
    sa.pack[1] = pack_args(p, d.x, p.xp, d.ld_x, d.n, d.d);
  }
  hipLaunchKernelGGL((k_ce_start<S, T, kPlanes>), dim3(sa.groups + sa.bias_blocks + sa.pack[0].blocks + sa.pack[1].blocks), dim3(kStartThreads), 0, st, sa);
  if (p.groups > 1) hipLaunchKernelGGL(k_ce_index, dim3(p.groups), dim3(kStartThreads), 0, st, sa);
  if (p.head) {
    if constexpr (kPlanes == 1) {
      const int rc = head<T, false>(head_args(d, p), p, d.n, st);
      if (rc != R3D_OK) return rc;
    }
    join(d, p, st);
    return R3D_OK;
  }
  if (p.narrow) {
    NarrowArgs na{};
    operands(d, p, na.kept, na.met);
    const int64_t of_points = narrow_rows(Narrow::Lse, kPlanes, (int)p.dp);
    na.v = d.v;
    na.bias2 = p.bias2;
    na.tgt = p.tgt;
    na.counted = p.counted;
    na.tiles = (int)((d.n + of_points - 1) / of_points);
    na.splits = p.lse_splits;
    na.split_stride = p.n_pad;
    na.part_m = p.part_m;
    na.part_l = p.part_l;
    na.hit = p.hit;
    narrow(Narrow::Lse, na, d.type, (int)p.dp, st);
    join(d, p, st);
    return R3D_OK;
  }
  LseArgs la{};
  operands(d, p, la.p.b, la.p.a);
  la.v = d.v;
  la.kb = p.dp / kTileK;
  la.splits = p.lse_splits;
  la.bias2 = p.bias2;
  la.tgt = p.tgt;
  la.counted = p.counted;
  la.part_m = p.part_m;
  la.part_l = p.part_l;
  la.hit = p.hit;
  la.n_pad = p.n_pad;
  with_shape<kPlanes>(p.lse_big, [&](auto shape) { lse<T, decltype(shape), kPlanes>(la, p, d.n, d.v, st); });
  join(d, p, st);
  return R3D_OK;
}

template <class T, class S, int kPlanes>
void dl_piece(DlArgs a, int64_t n, hipStream_t st) {
  a.ntiles = up(n, S::BN) / S::BN;
  a.vtiles = (int)(up(a.width, S::BM) / S::BM);
  hipLaunchKernelGGL((k_ce_dl<T, S, kPlanes>), dim3((unsigned)(a.ntiles * a.vtiles)), dim3(S::threads), 0, st, a);
}

template <class V, class T, class S, Lies LA>
void out_product(OutArgs a, int64_t m, int64_t n, hipStream_t st) {
  a.mtiles = (int)(up(m, S::BM) / S::BM);
  a.ntiles = (int)(up(n, S::BN) / S::BN);
  hipLaunchKernelGGL((k_ce_out<V, T, S, LA>), dim3((unsigned)((int64_t)a.mtiles * a.ntiles * a.splits)), dim3(S::threads), 0, st, a);
}

template <class V>
Finish finish_of(const float *acc, int64_t ld, int64_t split_stride, int64_t rows, int64_t width, int splits, const int32_t *place, void *out) {
  const bool vector = width % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(V)) == 0;
  return Finish{acc, ld, split_stride, rows, width, splits, vector, place, out};
}

template <class V>
void finish(const Finish *of, int n, const Plan &p, float unheld, hipStream_t st) {
  FinishArgs a{};
  a.scale = p.scale;
  a.unheld = unheld;
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    a.of[i] = of[i];
    const int64_t threads = of[i].rows * ((of[i].width + 3) / 4) * (of[i].splits >= 8 ? 4 : 1);
    if (threads > most) most = threads;
  }
  if (n) hipLaunchKernelGGL(k_ce_finish<V>, dim3(blocks_for(most, 256, 8192), n), dim3(256), 0, st, a);
}

// A head in LDS: head_points of the points at a time, dx from the kernel itself, dW added up over them.
template <class S, class T>
int backward_head(const r3d_linear_ce_t &d, const Plan &p, Operand x, float held, hipStream_t st) {
  const int64_t each = d.n < p.head_points ? d.n : p.head_points, classes = up(d.v, 32);
  const Operand dl{p.dl, p.dl_rows, 0, nullptr};
  const float unheld = 1.0f / held;
  for (int64_t first = 0; first < d.n; first += each) {
    HeadArgs ha = head_args(d, p);
    ha.first = (int32_t)first;
    ha.most = (int32_t)(d.n - first < each ? d.n - first : each);
    ha.idx += first;
    ha.tgt += first;
    ha.base += first;
    ha.sum += first;
    ha.weight += first;
    ha.held = held;
    ha.unheld = unheld;
    ha.n_pad = p.dl_rows;
    if (!d.dw) ha.dl = nullptr;
    ha.sums = d.db ? p.accb + first / each * head_groups(each) * classes : nullptr;
    const int rc = head<T, true>(ha, p, each, st);
    if (rc != R3D_OK) return rc;
    if (!d.dw) continue;
    OutArgs oa{};
    oa.p = Product{dl, x};
    oa.p.b.idx += first;
    oa.m = p.dw_final ? d.v : p.piece;
    oa.n = p.dw_final ? d.d : p.dp;
    oa.limit_a = p.piece;
    oa.limit_b = p.dp;
    oa.points = 2;
    oa.first = ha.first;
    oa.most = ha.most;
    oa.splits = p.dw_splits;
    oa.add = first > 0;
    oa.counted = p.counted;
    oa.out = p.accw;
    oa.ld = p.dw_final ? d.d : p.dp;
    oa.split_stride = p.piece * p.dp;
    oa.final_out = p.dw_final ? d.dw : nullptr;
    oa.scale = p.scale;
    oa.unheld = unheld;
    with_shape<1>(p.dw_big, [&](auto shape) { out_product<S, T, decltype(shape), Lies::PiecesCols>(oa, p.piece, p.dp, st); });
  }
  Finish of[2];
  int n_of = 0;
  if (d.dw && !p.dw_final) of[n_of++] = finish_of<S>(p.accw, p.dp, p.piece * p.dp, d.v, d.d, p.dw_splits, nullptr, d.dw);
  if (d.db) of[n_of++] = finish_of<S>(p.accb, classes, classes, 1, d.v, p.db_parts, nullptr, d.db);
  finish<S>(of, n_of, p, unheld, st);
  return R3D_OK;
}

template <class S, class T, int kPlanes>
int backward(const r3d_linear_ce_t &d, const Plan &p, hipStream_t st) {
  const bool each = d.reduction == R3D_CE_NONE;
  const int parts = each && d.type == R3D_T_F16 ? p.top_parts : 0;
  if (parts) hipLaunchKernelGGL(k_ce_top, dim3(parts), dim3(256), 0, st, d.grad, d.n, p.place, p.top);
  hipLaunchKernelGGL(k_ce_weight<S>, dim3((unsigned)(p.n_pad / 256)), dim3(256), 0, st,
                     WeightArgs{d.grad, p.top, each ? 1 : 0, parts, p.idx, p.place, p.counted, p.scale, p.weight, d.n, p.n_pad, d.d,
                                p.dx_final ? d.dx : nullptr});
  Operand x, w;
  operands(d, p, x, w);
  const float held = d.type == R3D_T_F16 ? 32768.0f : 1.0f, unheld = 1.0f / held;
  if (p.narrow) {
    Finish of[3];
    int n_of = 0;
    NarrowArgs na{};
    na.v = d.v;
    na.bias2 = p.bias2;
    na.base = p.base;
    na.sum = p.sum;
    na.weight = p.weight;
    na.tgt = p.tgt;
    na.counted = p.counted;
    na.held = held;
    na.each = each;
    na.d = d.d;
    na.scale = p.scale;
    na.unheld = unheld;
    const int64_t of_points = narrow_rows(Narrow::Dx, kPlanes, (int)p.dp), of_classes = narrow_rows(Narrow::Dw, kPlanes, (int)p.dp);
    auto vector = [&](const void *out) { return d.d % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(S)) == 0; };
    if (d.dx) {
      na.kept = x;
      na.met = w;
      na.tiles = (int)((d.n + of_points - 1) / of_points);
      na.splits = p.dx_splits;
      na.out = p.accx;
      na.split_stride = p.n_pad * p.dp;
      na.final_out = p.dx_final ? d.dx : nullptr;
      na.vector_out = vector(d.dx);
      narrow(Narrow::Dx, na, d.type, (int)p.dp, st);
      if (!p.dx_final) of[n_of++] = finish_of<S>(p.accx, p.dp, p.n_pad * p.dp, d.n, d.d, p.dx_splits, p.place, d.dx);
    }
    if (d.dw || d.db) {
      na.kept = w;
      na.met = x;
      na.tiles = (int)((d.v + of_classes - 1) / of_classes);
      na.splits = p.dw_splits;
      na.out = p.accw;
      na.split_stride = p.piece * p.dp;
      na.final_out = p.dw_final ? d.dw : nullptr;
      na.vector_out = vector(d.dw);
      na.sums = p.accb;
      na.sums_stride = p.piece;
      narrow(Narrow::Dw, na, d.type, (int)p.dp, st);
      if (!p.dw_final && d.dw) of[n_of++] = finish_of<S>(p.accw, p.dp, p.piece * p.dp, d.v, d.d, p.dw_splits, nullptr, d.dw);
      if (d.db) of[n_of++] = finish_of<S>(p.accb, p.piece, p.piece, 1, d.v, p.db_parts, nullptr, d.db);
    }
    finish<S>(of, n_of, p, unheld, st);
    return R3D_OK;
  }
  if constexpr (kPlanes == 1) {
    if (p.head) return backward_head<S, T>(d, p, x, held, st);
  }
  for (int64_t v0 = 0; v0 < d.v; v0 += p.piece) {
    const int64_t real_v = p.piece < d.v - v0 ? p.piece : d.v - v0, width = up(real_v, kPadK);
    Finish of[3];
    int n_of = 0;
    DlArgs da{};
    da.p = Product{w, x};
    da.v = d.v;
    da.kb = p.dp / kTileK;
    da.piece0 = v0;
    da.dl_plane = p.n_pad * p.piece;
    da.n_pad = p.n_pad;
    da.width = (int)width;
    da.held = held;
    da.bias2 = p.bias2;
    da.base = p.base;
    da.sum = p.sum;
    da.weight = p.weight;
    da.tgt = p.tgt;
    da.counted = p.counted;
    da.dl = p.dl;
    da.sums = d.db ? p.accb : nullptr;
    da.piece = p.piece;
    with_shape<kPlanes>(p.dl_big, [&](auto shape) { dl_piece<T, decltype(shape), kPlanes>(da, d.n, st); });
    const Operand dl{p.dl, p.n_pad, p.n_pad * p.piece, nullptr};
    if (d.dx) {
      Operand wv = w;      // the rows of this piece
      wv.p = static_cast<const char *>(w.p) + v0 * w.ld * 2;
      OutArgs oa{};
      oa.p = Product{dl, wv};
      oa.n = p.dx_final ? d.d : p.dp;
      oa.kb = width / kTileK;
      oa.limit_b = p.dp;
      oa.rows_b = real_v;
      oa.points = 1;
      oa.splits = p.dx_splits;
      oa.add = v0 > 0;
      oa.counted = p.counted;
      oa.out = p.accx;
      oa.ld = p.dx_final ? d.d : p.dp;
      oa.split_stride = p.n_pad * p.dp;
      oa.final_out = p.dx_final ? d.dx : nullptr;
      oa.idx = p.idx;
      oa.scale = p.scale;
      oa.unheld = unheld;
      with_shape<kPlanes>(p.dx_big, [&](auto shape) { out_product<S, T, decltype(shape), Lies::PiecesRows>(oa, d.n, p.dp, st); });
      if (!p.dx_final && v0 + p.piece >= d.v) of[n_of++] = finish_of<S>(p.accx, p.dp, p.n_pad * p.dp, d.n, d.d, p.dx_splits, p.place, d.dx);
    }
    if (d.dw) {
      const bool straight = p.dw_final;
      OutArgs oa{};
      oa.p = Product{dl, x};
      oa.m = straight ? real_v : width;
      oa.n = straight ? d.d : p.dp;
      oa.limit_a = width;
      oa.limit_b = p.dp;
      oa.points = 2;
      oa.most = (int32_t)d.n;
      oa.splits = p.dw_splits;
      oa.counted = p.counted;
      oa.out = p.accw;
      oa.ld = straight ? d.d : p.dp;
      oa.split_stride = p.piece * p.dp;
      oa.final_out = straight ? static_cast<char *>(d.dw) + v0 * d.d * p.type_bytes : nullptr;
      oa.scale = p.scale;
      oa.unheld = unheld;
      with_shape<kPlanes>(p.dw_big, [&](auto shape) { out_product<S, T, decltype(shape), Lies::PiecesCols>(oa, width, p.dp, st); });
      if (!straight)
        of[n_of++] = finish_of<S>(p.accw, p.dp, p.piece * p.dp, real_v, d.d, p.dw_splits, nullptr, static_cast<char *>(d.dw) + v0 * d.d * p.type_bytes);
    }
    if (d.db) of[n_of++] = finish_of<S>(p.accb, p.piece, p.piece, 1, real_v, p.db_parts, nullptr, static_cast<char *>(d.db) + v0 * p.type_bytes);
    finish<S>(of, n_of, p, unheld, st);
  }
  return R3D_OK;
}
}  // namespace

extern "C" size_t r3d_linear_ce_bytes(const r3d_linear_ce_t *d, int32_t which) {
  if (check(d) != R3D_OK || which < R3D_CE_BYTES_STATE || which > R3D_CE_BYTES_BACKWARD) return 0;
  if (few_takes(*d)) return few_bytes(*d, which);
  const Plan p = plan(*d, which == R3D_CE_BYTES_BACKWARD, nullptr);
  return which == R3D_CE_BYTES_STATE ? p.state_bytes : p.bytes;
}

extern "C" int r3d_linear_ce_forward(const r3d_linear_ce_t *d, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check(d);
  if (rc != R3D_OK) return rc;
  if (!d->x || !d->w || !d->target || !d->state || !d->loss || !workspace) return fail(R3D_E_ARG, "linear_ce_forward: null pointer");
  rc = check_aligned(*d, workspace);
  if (rc != R3D_OK) return rc;
  if (workspace_bytes < r3d_linear_ce_bytes(d, R3D_CE_BYTES_FORWARD)) return fail(R3D_E_WORKSPACE, "linear_ce_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (few_takes(*d)) {
    rc = few_forward(*d, workspace, st);
  } else {
    const Plan p = plan(*d, false, workspace);
    rc = d->type == R3D_T_F32 ? forward<float, __bf16, 3>(*d, p, st) : d->type == R3D_T_BF16 ? forward<__bf16, __bf16, 1>(*d, p, st) : forward<_Float16, _Float16, 1>(*d, p, st);
  }
  if (rc != R3D_OK) return rc;
  R3D_LAUNCHED("linear_ce forward kernels");
  return R3D_OK;
}

extern "C" int r3d_linear_ce_backward(const r3d_linear_ce_t *d, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check(d);
  if (rc != R3D_OK) return rc;
  if (!d->x || !d->w || !d->target || !d->state || !d->grad || !workspace) return fail(R3D_E_ARG, "linear_ce_backward: null pointer");
  rc = check_aligned(*d, workspace);
  if (rc != R3D_OK) return rc;
  if (workspace_bytes < r3d_linear_ce_bytes(d, R3D_CE_BYTES_BACKWARD)) return fail(R3D_E_WORKSPACE, "linear_ce_backward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (few_takes(*d)) {
    rc = few_backward(*d, workspace, st);
  } else {
    const Plan p = plan(*d, true, workspace);
    rc = d->type == R3D_T_F32 ? backward<float, __bf16, 3>(*d, p, st) : d->type == R3D_T_BF16 ? backward<__bf16, __bf16, 1>(*d, p, st) : backward<_Float16, _Float16, 1>(*d, p, st);
  }
  if (rc != R3D_OK) return rc;
  R3D_LAUNCHED("linear_ce backward kernels");
  return R3D_OK;
}

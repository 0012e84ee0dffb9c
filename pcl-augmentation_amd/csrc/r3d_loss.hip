// Softmax cross entropy of a linear head, in pieces of the classes, without keeping the logits (gfx950).
//
//   l = x W^T + b,  loss_n = log sum_v exp l_nv - l_n,target;   dl = g_n (softmax(l) - onehot),  dx = dl W,  dW = dl^T x,  db = sum_n dl.
//
// Forward: one product x W^T whose tiles end in a running maximum and sum per point (base 2), joined over the waves and over
// the splits of the classes.  Backward: for one piece of the classes at a time the logits once more, their gradient rounded to
// 16 bits into the workspace, and the two products with it.  Points whose target is ignored are left out at the start: the
// others are numbered in a line (stable, by prefix sums) and everything runs over that line, so they cost nothing and whatever
// their features hold (padding is rarely initialised) reaches no sum.
//
// Sums are in 32 bits (matrix cores, softmax statistics, gradients over points and classes), the mean's sum over points in 64.
// Rounded to fewer: dl, to the inputs' 16-bit type -- the matrix cores' operand; half a step of a term each, at random, beside
// half a step of the rounded result.  float16 has no room for a probability of 1e-6, so dl is held times 2^15 (|dl| <= 1) and
// the caller's weights of the points relative to the largest.  float32 operands are split into three bfloat16 planes (8 bits
// each, all 24) and multiplied as the six products that reach beyond 2^-24: 2.5 PFLOP/s of bfloat16 in six are more than the
// 0.16 of float32.
#include "r3d_host.hpp"
#include "r3d_loss.hpp"

#include <cmath>

namespace {
using namespace r3d;

template <class T>
__device__ __forceinline__ float wide(T v) { return (float)v; }

// ---- which points count -------------------------------------------------------------------------------------------------
constexpr int kCountRows = 1024;

struct IndexArgs {
  const void *target;
  int64_t n, v, ignore;
  int32_t wide_target, mean;
  int32_t *part, *idx, *place, *tgt;      // idx: point of a number, place: number of a point or -1, tgt: its class or -1 (not a class)
  Counted *counted;
};

__device__ __forceinline__ int64_t target_of(const IndexArgs &a, int64_t i) {
  return a.wide_target ? static_cast<const int64_t *>(a.target)[i] : static_cast<const int32_t *>(a.target)[i];
}

__global__ __launch_bounds__(256) void k_ce_count(IndexArgs a) {
  __shared__ int s[4];
  int c = 0;
  const int64_t first = (int64_t)blockIdx.x * kCountRows + threadIdx.x * 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) c += first + j < a.n && target_of(a, first + j) != a.ignore;
#pragma unroll
  for (int d = 32; d; d >>= 1) c += __shfl_xor(c, d);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) a.part[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}

__global__ __launch_bounds__(256) void k_ce_index(IndexArgs a) {
  __shared__ int s[4], s_before[4], s_all[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int before = 0, all = 0;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 256) {
    const int v = a.part[b];
    all += v;
    before += b < (int)blockIdx.x ? v : 0;
  }
  const int64_t first = (int64_t)blockIdx.x * kCountRows + threadIdx.x * 4;
  int64_t t[4];
  int mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t[j] = first + j < a.n ? target_of(a, first + j) : a.ignore;
    mine += t[j] != a.ignore;
  }
  int run = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    before += __shfl_xor(before, d);
    all += __shfl_xor(all, d);
  }
  if (lane == 63) s[wave] = run;
  if (lane == 0) {
    s_before[wave] = before;
    s_all[wave] = all;
  }
  __syncthreads();
  int at = run - mine + s_before[0] + s_before[1] + s_before[2] + s_before[3];
  for (int w = 0; w < wave; ++w) at += s[w];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (first + j >= a.n) break;
    const bool counts = t[j] != a.ignore;
    a.place[first + j] = counts ? at : -1;
    if (counts) {
      a.idx[at] = (int32_t)(first + j);
      a.tgt[at++] = t[j] >= 0 && t[j] < a.v ? (int32_t)t[j] : -1;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const int n = s_all[0] + s_all[1] + s_all[2] + s_all[3];
    a.counted->n = n;
    a.counted->share = !a.mean ? 1.0f : n ? 1.0f / (float)n : 0.0f;
  }
}

// ---- operands: rows of whole k-blocks, split into planes where the type is wider -------------------------------------------
struct PackArgs {
  const void *src;
  void *dst;
  int64_t ld, rows, width, ld_out, plane;      // width: of the source; ld_out a multiple of 64
  const int32_t *idx;
  const Counted *counted;      // rows: how many of them, where given
  int32_t vector;              // rows begin at multiples of 16 bytes
};

template <class T>
struct alignas(16) Piece {
  T v[8];
};

// A thread makes a piece of 8 values of a row.
template <class S, class T, int kPlanes>
__global__ __launch_bounds__(256) void k_ce_pack(PackArgs a) {
  const int64_t rows = a.counted ? a.counted->n : a.rows;
  const unsigned each = (unsigned)(a.ld_out / 8);
  const int64_t all = rows * each;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = all <= UINT32_MAX ? (unsigned)i / each : i / each;
    const int64_t c = (i - r * each) * 8;
    const S *src = static_cast<const S *>(a.src) + (a.idx ? a.idx[r] : r) * a.ld + c;
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

// The bias in units of log 2, -inf behind the last class: those count for nothing anywhere.
template <class S>
__global__ __launch_bounds__(256) void k_ce_bias(const S *bias, float *out, int64_t v, int64_t v_all) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < v_all) out[i] = i >= v ? -INFINITY : bias ? wide(bias[i]) * kLog2e : 0.0f;
}

// ---- products --------------------------------------------------------------------------------------------------------------
struct Product {
  Operand a, b;
  int32_t planes;
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

// Maximum and sum of 2^(logit * log2 e) over a split of the classes for the points of a tile.  The classes are the rows of C, so
// a lane holds 16 FM classes of each of its FN points: the statistics of a tile stay in its registers, lanes and waves are
// joined once at the end.
template <class T, class S>
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
  Stream<T, S, Lies::Rows, Lies::Rows> st;
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
  if (vt1 > vt0) st.begin(lds, 0, (int)a.kb, a.p.planes, more);
  for (int vt = vt0; vt < vt1; ++vt) {
    f32x16 acc[S::FM][S::FN];
    float none[S::FM];
    clear(acc);
    st.template run<false>(lds, acc, none, false, more);
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
          t[r] = __builtin_fmaf(acc[i][j][r], kLog2e, b[r]);
          top = fmaxf(top, t[r]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = l[j] * __builtin_amdgcn_exp2f(m[j] - base);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(t[r] - base);
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
    const float om = __shfl_xor(m[j], 32), ol = __shfl_xor(l[j], 32), top = fmaxf(m[j], om), base = top == -INFINITY ? 0.0f : top;
    const float sum = l[j] * __builtin_amdgcn_exp2f(m[j] - base) + ol * __builtin_amdgcn_exp2f(om - base);
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
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < S::WM; ++w) sum += s_l[w * S::BN + c] * __builtin_amdgcn_exp2f(s_m[w * S::BN + c] - base);
    a.part_m[split * a.n_pad + n0 + c] = top;
    a.part_l[split * a.n_pad + n0 + c] = sum;
  }
}

struct CombineArgs {
  const float *part_m, *part_l, *hit;
  const int32_t *tgt, *place;
  const Counted *counted;
  float *lse2, *each, *loss;
  double *sums;
  int64_t n, n_pad;
  int32_t splits;
};

// The splits joined; the loss of every point (each) or the sums of 256 of them.  Over the points as the caller numbers them.
__global__ __launch_bounds__(256) void k_ce_join(CombineArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int at = i < a.n ? a.place[i] : -1;
  float loss = 0.0f;
  if (at >= 0) {
    float top = -INFINITY, sum = 0.0f;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_m[s * a.n_pad + at]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int s = 0; s < a.splits; ++s) sum += a.part_l[s * a.n_pad + at] * __builtin_amdgcn_exp2f(a.part_m[s * a.n_pad + at] - base);
    const bool fine = a.tgt[at] >= 0;      // a target that is no class: NaN, and so are its gradients
    const float lse2 = fine ? top + __builtin_amdgcn_logf(sum) : NAN;
    a.lse2[at] = lse2;
    loss = fine ? (lse2 - a.hit[at]) * kLn2 : NAN;
  }
  if (a.each) {
    if (i < a.n) a.each[i] = loss;
    return;
  }
  __shared__ double s[4];
  double d = loss;
#pragma unroll
  for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = d;
  __syncthreads();
  if (threadIdx.x == 0) a.sums[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}

__global__ __launch_bounds__(256) void k_ce_mean(const double *sums, int64_t n, const Counted *counted, int32_t mean, float *loss) {
  __shared__ double s[4];
  double d = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) d += sums[i];
#pragma unroll
  for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    d = s[0] + s[1] + s[2] + s[3];
    const int c = counted->n;
    *loss = (float)(mean && c ? d / c : d);
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
// The factor that is taken out of dl: the one weight of a sum or a mean; for float16 the largest weight of single points.
__global__ __launch_bounds__(256) void k_ce_top(const float *grad, int64_t n, const int32_t *place, float *part) {
  __shared__ float s[4];
  float top = 0.0f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    if (place[i] >= 0) top = fmaxf(top, fabsf(grad[i]));      // (fmaxf passes over NaN)
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

struct WeightArgs {
  const float *grad, *part;
  int32_t each, parts;
  const int32_t *idx;
  const Counted *counted;
  float *scale;       // [1] the factor taken out of dl
  float *weight;      // of every point in the line, at most 1; 0 up to n_pad
  int64_t n_pad;
};

__global__ __launch_bounds__(256) void k_ce_weight(WeightArgs a) {
  const int nc = a.counted->n;
  float scale;
  if (a.each) {
    scale = 0.0f;
    for (int b = threadIdx.x & 63; b < a.parts; b += 64) scale = fmaxf(scale, a.part[b]);
#pragma unroll
    for (int d = 32; d; d >>= 1) scale = fmaxf(scale, __shfl_xor(scale, d));
    if (!(scale > 0.0f) || scale == INFINITY) scale = 1.0f;      // nothing to take out
  } else {
    scale = a.grad[0] * a.counted->share;
  }
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < a.n_pad) a.weight[i] = i >= nc ? 0.0f : a.each ? a.grad[a.idx[i]] / scale : 1.0f;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.scale = scale;
}

struct DlArgs {
  Product p;
  int64_t v, kb, ntiles;
  int64_t piece0, dl_plane, n_pad;      // first class of the piece
  int32_t vtiles, width;                // width: classes of the piece, a multiple of 64
  float held;                           // 2^15 for float16
  const float *bias2, *lse2, *weight;
  const int32_t *tgt;
  const Counted *counted;
  void *dl;        // [planes][width / 8][n_pad][8]
};

// dl of a piece of the classes.  A lane holds 4 neighbouring classes of a point and its partner 32 lanes on the next 4: a swap
// makes pieces of 8, and 32 lanes write 512 contiguous bytes.
template <class T, class S, int kPlanes>
__global__ __launch_bounds__(S::threads, 2) void k_ce_dl(DlArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[S::buffers * S::buffer];
  const int nc = a.counted->n;
  int64_t vt, nt;
  tile_of(xcd_order(blockIdx.x, gridDim.x), a.vtiles, a.ntiles, vt, nt);
  const int64_t n0 = nt * S::BN;
  if (n0 >= nc) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  f32x16 acc[S::FM][S::FN];
  float none[S::FM];
  clear(acc);
  {
    Stream<T, S, Lies::Rows, Lies::Rows> st;
    st.a = a.p.a;
    st.b = a.p.b;
    st.rows_b = 0;
    st.la.tile(st.a, a.piece0 + vt * S::BM, a.v);
    st.lb.tile(st.b, n0, nc);
    auto more = [] { return false; };
    st.begin(lds, 0, (int)a.kb, a.p.planes, more);
    st.template run<false>(lds, acc, none, false, more);
    st.end();
  }
  T *dl = static_cast<T *>(a.dl);
#pragma unroll
  for (int j = 0; j < S::FN; ++j) {
    const int64_t col = n0 + (wn * S::FN + j) * 32 + (lane & 31);
    const bool in = col < nc;
    const int tgt = in ? a.tgt[col] : -1;
    const float lse2 = in ? a.lse2[col] : 0.0f, weight = in ? a.weight[col] * a.held : 0.0f;
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
      const int local = (int)vt * S::BM + (wm * S::FM + i) * 32;
      if (local >= a.width) continue;
      const int64_t vb = a.piece0 + local;
      const int64_t d = tgt - vb;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, a.bias2[vb + mma_row(r)]) - lse2);
      if (__any(d >= 0 && d < 32)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] -= d == mma_row(r) ? 1.0f : 0.0f;
      }
      typedef T t4 __attribute__((ext_vector_type(4)));
      typedef unsigned u2 __attribute__((ext_vector_type(2)));
      typedef unsigned u4 __attribute__((ext_vector_type(4)));
      t4 q[4][kPlanes];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float w = in ? p[r] * weight : 0.0f;
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
          *reinterpret_cast<u4 *>(dl + k * a.dl_plane + (piece * a.n_pad + col) * 8) = out;
        }
    }
  }
}

struct OutArgs {
  Product p;
  int64_t m, n, kb;                      // m: rows of the result, n: columns that are written
  int64_t limit_a, limit_b, rows_b;      // columns of the operands, rows of b
  int32_t points;                        // 0: m and the rest as given; 1: m is the points that count; 2: k is
  int32_t mtiles, ntiles, splits, add;
  const Counted *counted;
  float *out;                            // [splits][m_pad][ld], or null:
  int64_t ld, split_stride;
  void *final_out;                       // the result itself, rows through idx where given
  const int32_t *idx;
  const float *scale;
  float unheld;
  float *row_sum;                        // [splits][sum_stride]: sums over k of A, or null
  int64_t sum_stride;
};

// The products with dl: dx = dl W and dW = dl^T x (with db, the sums of dl's columns, which pass by), into 32-bit sums in the
// workspace or, where nothing is left to add, to the result.
template <class V, class T, class S, Lies LA>
__global__ __launch_bounds__(S::threads, 2) void k_ce_out(OutArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[S::buffers * S::buffer];
  const int nc = a.counted->n;
  const int64_t id = xcd_order(blockIdx.x, gridDim.x), tiles = (int64_t)a.mtiles * a.ntiles;
  const int split = (int)(id / tiles);
  int64_t mt, nt;
  tile_of(id - split * tiles, a.mtiles, a.ntiles, mt, nt);
  const int64_t m0 = mt * S::BM, n0 = nt * S::BN;
  const int64_t m = a.points == 1 ? nc : a.m, kb = a.points == 2 ? (nc + kTileK - 1) / kTileK : a.kb;
  if (m0 >= m) return;
  constexpr bool kSums = LA == Lies::PiecesCols;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  const bool sums = kSums && a.row_sum && nt == 0 && wn == 0;
  f32x16 acc[S::FM][S::FN];
  float row_sum[S::FM];
  clear(acc);
#pragma unroll
  for (int i = 0; i < S::FM; ++i) row_sum[i] = 0.0f;
  const int64_t kb0 = kb * split / a.splits, kb1 = kb * (split + 1) / a.splits;
  if (kb1 > kb0) {
    Stream<T, S, LA, Lies::Cols> st;
    st.a = a.p.a;
    st.b = a.p.b;
    st.rows_b = (int)(a.points == 2 ? nc : a.rows_b);
    st.la.tile(st.a, m0, a.points == 1 ? nc : a.limit_a);
    st.lb.tile(st.b, n0, a.limit_b);
    auto more = [] { return false; };
    st.begin(lds, (int)kb0, (int)kb1, a.p.planes, more);
    st.template run<kSums>(lds, acc, row_sum, sums, more);
    st.end();
  }
  const float scale = a.final_out ? *a.scale * a.unheld : 1.0f;
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
    if (kSums && sums) {
      const float s = row_sum[i] + __shfl_xor(row_sum[i], 32);
      const int64_t row = m0 + (wm * S::FM + i) * 32 + lane;
      if (lane < 32 && row < m) a.row_sum[split * a.sum_stride + row] = s;
    }
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

// Rows of the points that do not count.
template <class V>
__global__ __launch_bounds__(256) void k_ce_zero(V *dx, int64_t n, int64_t d, const int32_t *place) {
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += (int64_t)gridDim.x * 4)
    if (place[r] < 0)
      for (int64_t c = threadIdx.x & 63; c < d; c += 64) dx[r * d + c] = (V)0.0f;
}

struct FinishArgs {
  const float *acc;
  int64_t ld, split_stride, rows, width, ld_out;
  int32_t splits;
  float unheld;      // 2^-15 for float16
  const int32_t *place;
  const float *scale;
  void *out;
};

// Splits joined, the factor put back, one rounding.  A thread makes kVec neighbouring values.
template <class V, int kVec>
__global__ __launch_bounds__(256) void k_ce_finish(FinishArgs a) {
  typedef float fv __attribute__((ext_vector_type(kVec)));
  struct alignas(kVec * sizeof(V)) Out {
    V v[kVec];
  };
  const float scale = *a.scale * a.unheld;
  const unsigned each = (unsigned)(a.width / kVec);
  const int64_t all = a.rows * each;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = all <= UINT32_MAX ? (unsigned)i / each : i / each;
    const int64_t c = (i - r * each) * kVec, at = a.place ? a.place[r] : r;
    float sum[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[e] = 0.0f;
    if (at >= 0) {
      const float *from = a.acc + at * a.ld + c;
#pragma unroll 8
      for (int s = 0; s < a.splits; ++s) {
        if constexpr (kVec == 1) {
          sum[0] += from[s * a.split_stride];
        } else {
          const fv v = *reinterpret_cast<const fv *>(from + s * a.split_stride);
#pragma unroll
          for (int e = 0; e < kVec; ++e) sum[e] += v[e];
        }
      }
    }
    Out out;
#pragma unroll
    for (int e = 0; e < kVec; ++e) out.v[e] = (V)(at >= 0 ? sum[e] * scale : 0.0f);
    *reinterpret_cast<Out *>(static_cast<V *>(a.out) + r * a.ld_out + c) = out;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// What a piece's dl may take.  8192 points x 161280 classes x 512: 8.8 ms with 64 MB, 7.1 with 256, 6.7 with 512, 6.4 with all 2.6 GB.
constexpr int64_t kPieceBytes = 512ll << 20;
constexpr int kCus = 256;
constexpr int kPadK = 64;      // operands are padded to whole cache lines along k

int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t tiles_of(int64_t m, int64_t n, int64_t bm, int64_t bn) { return (up(m, bm) / bm) * (up(n, bn) / bn); }

// Parts in which the long axis of a product is cut: enough workgroups for the chip, and no last round that leaves most of it
// idle; at least four k-blocks each.
int cut(int64_t tiles, int64_t slots, int64_t most) {
  if (most < 1) most = 1;
  int best = 1;
  double best_share = 0.0;
  for (int64_t s = 1; s <= most && s <= 1024; ++s) {
    const int64_t all = tiles * s, rounds = (all + slots - 1) / slots;
    const double share = (double)all / (double)(rounds * slots);
    if (share > best_share * 1.05) {
      best = (int)s;
      best_share = share;
    }
    if (all >= 4 * slots) break;
  }
  return best;
}

// A product's tiles: large ones where they fill the chip and waste no more than a quarter over small ones at the edges.
bool large_tiles(int64_t m, int64_t n, int64_t most_splits) {
  const int64_t big = tiles_of(m, n, Big::BM, Big::BN), small = tiles_of(m, n, Small::BM, Small::BN);
  return big * most_splits >= kCus && big * 4 * 4 <= small * 5;
}

struct Plan {
  bool direct;      // the operands are multiplied where they lie
  int planes, type_bytes;
  int64_t dp, n_pad, v_pad, piece;
  bool lse_big, dl_big, dx_big, dw_big;
  int lse_splits, dx_splits, dw_splits, top_parts, groups;
  bool dx_final, dw_final;      // nothing to add: straight into the result
  // workspace
  int32_t *part;
  void *xp, *wp;
  float *bias2, *part_m, *part_l, *hit;
  double *sums;
  float *top, *scale, *weight, *accx, *accw, *accb;
  void *dl;
  size_t bytes;
};

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

Plan plan(const r3d_linear_ce_t &d, bool backward, void *workspace) {
  Plan p{};
  p.planes = d.type == R3D_T_F32 ? 3 : 1;
  p.type_bytes = d.type == R3D_T_F32 ? 4 : 2;
  p.direct = p.planes == 1 && d.d % kPadK == 0 && d.ld_x % 8 == 0 && d.ld_w % 8 == 0 && aligned16(d.x) && aligned16(d.w);
  p.dp = up(d.d, kPadK);
  p.n_pad = up(d.n, Big::BN);
  p.v_pad = up(d.v, Big::BM);
  p.groups = (int)((d.n + kCountRows - 1) / kCountRows);
  Carver c(workspace);
  p.bias2 = c.take<float>(p.v_pad);
  if (!p.direct) {
    p.xp = c.take<uint16_t>((size_t)p.planes * p.n_pad * p.dp);
    p.wp = c.take<uint16_t>((size_t)p.planes * p.v_pad * p.dp);
  }
  if (!backward) {
    p.lse_big = large_tiles(d.v, d.n, 1);
    const int64_t bm = p.lse_big ? Big::BM : Small::BM, bn = p.lse_big ? Big::BN : Small::BN;
    p.lse_splits = cut(up(d.n, bn) / bn, kCus * (p.lse_big ? Big::per_cu : Small::per_cu), up(d.v, bm) / bm);
    p.part = c.take<int32_t>(p.groups);
    p.part_m = c.take<float>((size_t)p.lse_splits * p.n_pad);
    p.part_l = c.take<float>((size_t)p.lse_splits * p.n_pad);
    p.hit = c.take<float>(p.n_pad);
    p.sums = c.take<double>((d.n + 255) / 256);
  } else {
    const int64_t v64 = up(d.v, kPadK);
    int64_t piece = d.piece > 0 ? up(d.piece, kPadK) : kPieceBytes / (p.n_pad * 2 * p.planes) / Big::BM * Big::BM;
    if (piece < Small::BM) piece = Small::BM;
    p.piece = piece < v64 ? piece : v64;
    if (d.piece == 0) p.piece = up((v64 + (v64 + p.piece - 1) / p.piece - 1) / ((v64 + p.piece - 1) / p.piece), Big::BM);      // pieces of one size
    if (p.piece > v64) p.piece = v64;
    p.dl_big = large_tiles(p.piece, d.n, 1);
    const int64_t kx = p.piece / 256, kw = p.n_pad / 256;
    p.dx_big = large_tiles(d.n, p.dp, kx);
    p.dw_big = large_tiles(p.piece, p.dp, kw);
    auto tiles = [&](int64_t m, int64_t n, bool big) { return big ? tiles_of(m, n, Big::BM, Big::BN) : tiles_of(m, n, Small::BM, Small::BN); };
    p.dx_splits = cut(tiles(d.n, p.dp, p.dx_big), kCus * (p.dx_big ? Big::per_cu : Small::per_cu), kx);
    p.dw_splits = cut(tiles(p.piece, p.dp, p.dw_big), kCus * (p.dw_big ? Big::per_cu : Small::per_cu), kw);
    p.dx_final = p.dx_splits == 1 && p.piece >= d.v;
    p.dw_final = p.dw_splits == 1;
    p.top_parts = (int)(d.n < 256 * 256 ? (d.n + 255) / 256 : 256);
    p.top = c.take<float>(p.top_parts);
    p.scale = c.take<float>(1);
    p.weight = c.take<float>(p.n_pad);
    p.dl = c.take<uint16_t>((size_t)p.planes * p.n_pad * p.piece);
    if (!p.dx_final) p.accx = c.take<float>((size_t)p.dx_splits * p.n_pad * p.dp);
    p.accw = c.take<float>((size_t)(p.dw_final && d.dw ? 0 : p.dw_splits) * p.piece * p.dp);
    p.accb = c.take<float>((size_t)p.dw_splits * p.piece);
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

template <class S, class T, int kPlanes>
void pack(const PackArgs &a, int64_t rows, hipStream_t st) {
  hipLaunchKernelGGL((k_ce_pack<S, T, kPlanes>), dim3(blocks_for(rows * a.ld_out, 2048, 8192)), dim3(256), 0, st, a);
}

// The operands as the products take them: in place, or packed into the workspace.
template <class S, class T, int kPlanes>
void operands(const r3d_linear_ce_t &d, const Plan &p, const Counted *counted, hipStream_t st, Operand &x, Operand &w) {
  hipLaunchKernelGGL(k_ce_bias<S>, dim3(blocks_for(p.v_pad, 256, 1 << 30)), dim3(256), 0, st, static_cast<const S *>(d.bias), p.bias2, d.v, p.v_pad);
  if (p.direct) {
    x = Operand{d.x, d.ld_x, 0, d.idx};
    w = Operand{d.w, d.ld_w, 0, nullptr};
    return;
  }
  const int size = (int)sizeof(S);
  pack<S, T, kPlanes>(PackArgs{d.x, p.xp, d.ld_x, d.n, d.d, p.dp, p.n_pad * p.dp, d.idx, counted, aligned16(d.x) && d.ld_x * size % 16 == 0}, d.n, st);
  pack<S, T, kPlanes>(PackArgs{d.w, p.wp, d.ld_w, d.v, d.d, p.dp, p.v_pad * p.dp, nullptr, nullptr, aligned16(d.w) && d.ld_w * size % 16 == 0}, d.v, st);
  x = Operand{p.xp, p.dp, p.n_pad * p.dp, nullptr};
  w = Operand{p.wp, p.dp, p.v_pad * p.dp, nullptr};
}

template <class T, class S>
void lse(LseArgs a, const Plan &p, int64_t n, int64_t v, hipStream_t st) {
  a.ntiles = up(n, S::BN) / S::BN;
  a.vtiles = (int)(up(v, S::BM) / S::BM);
  hipLaunchKernelGGL((k_ce_lse<T, S>), dim3((unsigned)(a.ntiles * p.lse_splits)), dim3(S::threads), 0, st, a);
}

template <class S, class T, int kPlanes>
void forward(const r3d_linear_ce_t &d, const Plan &p, hipStream_t st) {
  Counted *counted = static_cast<Counted *>(d.counted);
  IndexArgs ia{d.target, d.n, d.v, d.ignore_index, d.target_type == R3D_T_I64, d.reduction == R3D_CE_MEAN, p.part, d.idx, d.place, d.tgt, counted};
  hipLaunchKernelGGL(k_ce_count, dim3(p.groups), dim3(256), 0, st, ia);
  hipLaunchKernelGGL(k_ce_index, dim3(p.groups), dim3(256), 0, st, ia);
  LseArgs la{};
  operands<S, T, kPlanes>(d, p, counted, st, la.p.b, la.p.a);
  la.p.planes = kPlanes;
  la.v = d.v;
  la.kb = p.dp / kTileK;
  la.splits = p.lse_splits;
  la.bias2 = p.bias2;
  la.tgt = d.tgt;
  la.counted = counted;
  la.part_m = p.part_m;
  la.part_l = p.part_l;
  la.hit = p.hit;
  la.n_pad = p.n_pad;
  if (p.lse_big) lse<T, Big>(la, p, d.n, d.v, st);
  else lse<T, Small>(la, p, d.n, d.v, st);
  CombineArgs ca{p.part_m, p.part_l, p.hit, d.tgt, d.place, counted, d.lse2, d.reduction == R3D_CE_NONE ? d.loss : nullptr, d.loss, p.sums, d.n, p.n_pad,
                 p.lse_splits};
  const int blocks = (int)((d.n + 255) / 256);
  hipLaunchKernelGGL(k_ce_join, dim3(blocks), dim3(256), 0, st, ca);
  if (d.reduction != R3D_CE_NONE)
    hipLaunchKernelGGL(k_ce_mean, dim3(1), dim3(256), 0, st, p.sums, (int64_t)blocks, counted, d.reduction == R3D_CE_MEAN ? 1 : 0, d.loss);
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
void finish(const FinishArgs &a, hipStream_t st) {
  const bool four = a.width % 4 == 0 && a.ld % 4 == 0 && a.ld_out % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(V))) == 0;
  const int64_t threads = a.rows * a.width / (four ? 4 : 1);
  if (four) hipLaunchKernelGGL((k_ce_finish<V, 4>), dim3(blocks_for(threads, 256, 8192)), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_ce_finish<V, 1>), dim3(blocks_for(threads, 256, 8192)), dim3(256), 0, st, a);
}

template <class S, class T, int kPlanes>
void backward(const r3d_linear_ce_t &d, const Plan &p, hipStream_t st) {
  const Counted *counted = static_cast<const Counted *>(d.counted);
  const bool each = d.reduction == R3D_CE_NONE;
  const int parts = each && d.type == R3D_T_F16 ? p.top_parts : 0;
  if (parts) hipLaunchKernelGGL(k_ce_top, dim3(parts), dim3(256), 0, st, d.grad, d.n, d.place, p.top);
  hipLaunchKernelGGL(k_ce_weight, dim3(blocks_for(p.n_pad, 256, 1 << 30)), dim3(256), 0, st,
                     WeightArgs{d.grad, p.top, each ? 1 : 0, parts, d.idx, counted, p.scale, p.weight, p.n_pad});
  Operand x, w;
  operands<S, T, kPlanes>(d, p, counted, st, x, w);
  const float held = d.type == R3D_T_F16 ? 32768.0f : 1.0f, unheld = 1.0f / held;
  for (int64_t v0 = 0; v0 < d.v; v0 += p.piece) {
    const int64_t real_v = p.piece < d.v - v0 ? p.piece : d.v - v0, width = up(real_v, kPadK);
    DlArgs da{};
    da.p = Product{w, x, kPlanes};
    da.v = d.v;
    da.kb = p.dp / kTileK;
    da.piece0 = v0;
    da.dl_plane = p.n_pad * p.piece;
    da.n_pad = p.n_pad;
    da.width = (int)width;
    da.held = held;
    da.bias2 = p.bias2;
    da.lse2 = d.lse2;
    da.weight = p.weight;
    da.tgt = d.tgt;
    da.counted = counted;
    da.dl = p.dl;
    if (p.dl_big) dl_piece<T, Big, kPlanes>(da, d.n, st);
    else dl_piece<T, Small, kPlanes>(da, d.n, st);
    const Operand dl{p.dl, p.n_pad, p.n_pad * p.piece, nullptr};
    if (d.dx) {
      Operand wv = w;      // the rows of this piece
      wv.p = static_cast<const char *>(w.p) + v0 * w.ld * 2;
      OutArgs oa{};
      oa.p = Product{dl, wv, kPlanes};
      oa.n = p.dx_final ? d.d : p.dp;
      oa.kb = width / kTileK;
      oa.limit_b = p.dp;
      oa.rows_b = real_v;
      oa.points = 1;
      oa.splits = p.dx_splits;
      oa.add = v0 > 0;
      oa.counted = counted;
      oa.out = p.accx;
      oa.ld = p.dx_final ? d.d : p.dp;
      oa.split_stride = p.n_pad * p.dp;
      oa.final_out = p.dx_final ? d.dx : nullptr;
      oa.idx = d.idx;
      oa.scale = p.scale;
      oa.unheld = unheld;
      if (p.dx_big) out_product<S, T, Big, Lies::PiecesRows>(oa, d.n, p.dp, st);
      else out_product<S, T, Small, Lies::PiecesRows>(oa, d.n, p.dp, st);
    }
    if (d.dw || d.db) {
      const bool straight = p.dw_final && d.dw;
      OutArgs oa{};
      oa.p = Product{dl, x, kPlanes};
      oa.m = straight ? real_v : width;
      oa.n = straight ? d.d : p.dp;
      oa.limit_a = width;
      oa.limit_b = p.dp;
      oa.points = 2;
      oa.splits = p.dw_splits;
      oa.counted = counted;
      oa.out = p.accw;
      oa.ld = straight ? d.d : p.dp;
      oa.split_stride = p.piece * p.dp;
      oa.final_out = straight ? static_cast<char *>(d.dw) + v0 * d.d * p.type_bytes : nullptr;
      oa.scale = p.scale;
      oa.unheld = unheld;
      oa.row_sum = d.db ? p.accb : nullptr;
      oa.sum_stride = p.piece;
      if (p.dw_big) out_product<S, T, Big, Lies::PiecesCols>(oa, width, p.dp, st);
      else out_product<S, T, Small, Lies::PiecesCols>(oa, width, p.dp, st);
      if (d.dw && !straight)
        finish<S>(FinishArgs{p.accw, p.dp, p.piece * p.dp, real_v, d.d, d.d, p.dw_splits, unheld, nullptr, p.scale,
                             static_cast<char *>(d.dw) + v0 * d.d * p.type_bytes}, st);
      if (d.db)
        finish<S>(FinishArgs{p.accb, 1, p.piece, real_v, 1, 1, p.dw_splits, unheld, nullptr, p.scale, static_cast<char *>(d.db) + v0 * p.type_bytes}, st);
    }
  }
  if (d.dx && p.dx_final)
    hipLaunchKernelGGL(k_ce_zero<S>, dim3(blocks_for(d.n, 4, 2048)), dim3(256), 0, st, static_cast<S *>(d.dx), d.n, d.d, d.place);
  else if (d.dx)
    finish<S>(FinishArgs{p.accx, p.dp, p.n_pad * p.dp, d.n, d.d, d.d, p.dx_splits, unheld, d.place, p.scale, d.dx}, st);
}
}  // namespace

extern "C" size_t r3d_linear_ce_workspace_bytes(const r3d_linear_ce_t *d, int32_t backward_pass) {
  if (check(d) != R3D_OK) return 0;
  const size_t few = few_bytes(*d, backward_pass != 0);
  return few ? few : plan(*d, backward_pass != 0, nullptr).bytes;
}

extern "C" int r3d_linear_ce_forward(const r3d_linear_ce_t *d, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check(d);
  if (rc != R3D_OK) return rc;
  if (!d->x || !d->w || !d->target || !d->idx || !d->place || !d->tgt || !d->lse2 || !d->counted || !d->loss || !workspace)
    return fail(R3D_E_ARG, "linear_ce_forward: null pointer");
  if (workspace_bytes < r3d_linear_ce_workspace_bytes(d, 0)) return fail(R3D_E_WORKSPACE, "linear_ce_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (few_bytes(*d, false)) {
    rc = few_forward(*d, workspace, st);
    if (rc != R3D_OK) return rc;
    R3D_LAUNCHED("linear_ce forward kernels, few classes");
    return R3D_OK;
  }
  const Plan p = plan(*d, false, workspace);
  if (d->type == R3D_T_F32) forward<float, __bf16, 3>(*d, p, st);
  else if (d->type == R3D_T_BF16) forward<__bf16, __bf16, 1>(*d, p, st);
  else forward<_Float16, _Float16, 1>(*d, p, st);
  R3D_LAUNCHED("linear_ce forward kernels");
  return R3D_OK;
}

extern "C" int r3d_linear_ce_backward(const r3d_linear_ce_t *d, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check(d);
  if (rc != R3D_OK) return rc;
  if (!d->x || !d->w || !d->idx || !d->place || !d->tgt || !d->lse2 || !d->counted || !d->grad || !workspace)
    return fail(R3D_E_ARG, "linear_ce_backward: null pointer");
  if (workspace_bytes < r3d_linear_ce_workspace_bytes(d, 1)) return fail(R3D_E_WORKSPACE, "linear_ce_backward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (few_bytes(*d, true)) {
    rc = few_backward(*d, workspace, st);
    if (rc != R3D_OK) return rc;
    R3D_LAUNCHED("linear_ce backward kernels, few classes");
    return R3D_OK;
  }
  const Plan p = plan(*d, true, workspace);
  if (d->type == R3D_T_F32) backward<float, __bf16, 3>(*d, p, st);
  else if (d->type == R3D_T_BF16) backward<__bf16, __bf16, 1>(*d, p, st);
  else backward<_Float16, _Float16, 1>(*d, p, st);
  R3D_LAUNCHED("linear_ce backward kernels");
  return R3D_OK;
}

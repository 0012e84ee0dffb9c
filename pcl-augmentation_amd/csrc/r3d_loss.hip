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
#include "r3d_mfma.hpp"

#include <cmath>

namespace {
using namespace r3d;

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kPairs = 6;      // (plane of A, plane of B) of a split product, largest last dropped: m*l, l*l < 2^-24
__device__ constexpr int kPlaneA[kPairs] = {0, 0, 1, 1, 0, 2}, kPlaneB[kPairs] = {0, 1, 0, 1, 2, 0};

struct Counted {      // the points that count, on the device
  int32_t n;          // how many
  float share;        // 1 / n for a mean (0 where none counts), 1 else
  float pad[2];
};

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
};

__device__ __forceinline__ __bf16 toward_zero(float v) {      // (rounding up the largest floats would give infinities)
  return __builtin_bit_cast(__bf16, (unsigned short)(__builtin_bit_cast(unsigned, v) >> 16));
}
__device__ __forceinline__ void split3(float v, __bf16 &h, __bf16 &m, __bf16 &l) {
  h = toward_zero(v);
  const float r = v - (float)h;
  m = toward_zero(r);
  l = (__bf16)(r - (float)m);
}

template <class S, class T, int kPlanes>
__global__ __launch_bounds__(256) void k_ce_pack(PackArgs a) {
  const int64_t rows = a.counted ? a.counted->n : a.rows, all = rows * a.ld_out;
  const S *src = static_cast<const S *>(a.src);
  T *dst = static_cast<T *>(a.dst);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / a.ld_out, c = i - r * a.ld_out;
    const S v = c < a.width ? src[(a.idx ? a.idx[r] : r) * a.ld + c] : (S)0.0f;
    if constexpr (kPlanes == 3) split3(v, dst[i], dst[i + a.plane], dst[i + 2 * a.plane]);
    else dst[i] = v;
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

// acc += the k-blocks [kb0, kb1) of one 128 x 128 tile.  Ends with a barrier: LDS is free.
template <class T, bool kACols, bool kBCols>
__device__ __forceinline__ void product_tile(const Product &p, int64_t m0, int64_t n0, int64_t rows_a, int64_t rows_b, int64_t cols_a,
                                             int64_t cols_b, int64_t kb0, int64_t kb1, T *lds, f32x16 (&acc)[2][2]) {
  const int wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  const int pairs = p.planes == 3 ? kPairs : 1;
  const int64_t n_kb = kb1 - kb0, steps = n_kb * pairs;
  if (steps <= 0) return;
  RowLoader<T> ra, rb;
  ColLoader<T> ca, cb;
  if constexpr (kACols) ca.tile(m0, cols_a); else ra.tile(p.a, m0, rows_a);
  if constexpr (kBCols) cb.tile(n0, cols_b); else rb.tile(p.b, n0, rows_b);
  int64_t kb = kb0;
  int pair = 0;
  if constexpr (kACols) ca.look(p.a, kb * kTileK, rows_a);
  if constexpr (kBCols) cb.look(p.b, kb * kTileK, rows_b);
  auto issue = [&](int buf) {
    T *la = lds + buf * 2 * kOperandElems, *lb = la + kOperandElems;
    const int64_t oa = (int64_t)kPlaneA[pair] * p.a.plane, ob = (int64_t)kPlaneB[pair] * p.b.plane;
    if constexpr (kACols) ca.issue(p.a, la, oa); else ra.issue(la, oa + kb * kTileK);
    if constexpr (kBCols) cb.issue(p.b, lb, ob); else rb.issue(lb, ob + kb * kTileK);
    if (++kb == kb1) {
      kb = kb0;
      ++pair;
    }
    if constexpr (kACols) ca.look(p.a, kb * kTileK, rows_a);
    if constexpr (kBCols) cb.look(p.b, kb * kTileK, rows_b);
  };
  issue(0);
  __syncthreads();
  for (int64_t s = 0; s < steps; ++s) {
    const int buf = (int)(s & 1);
    if (s + 1 < steps) issue(buf ^ 1);
    const T *la = lds + buf * 2 * kOperandElems;
    mma_block<T, kACols, kBCols>(la, la + kOperandElems, wm, wn, acc);
    __syncthreads();
  }
}

__device__ __forceinline__ void clear(f32x16 (&acc)[2][2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
}

struct LseArgs {
  Product p;      // a: W [V], b: x [points]
  int64_t v, kb, n_rows_x;      // n_rows_x: rows of x's storage
  int32_t vtiles, splits, packed;
  const float *bias2;
  const int32_t *tgt;
  const Counted *counted;
  float *part_m, *part_l, *hit;
  int64_t n_pad;
};

// Maximum and sum of 2^(logit * log2 e) over a split of the classes for 128 points.  The classes are the rows of C, so a lane
// holds 32 classes of each of its two points: the statistics of a tile stay in its registers, lanes and waves are joined once
// at the end.
template <class T>
__global__ __launch_bounds__(kMmaThreads, 2) void k_ce_lse(LseArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[4 * kOperandElems];
  const int nc = a.counted->n;
  const int64_t n0 = (int64_t)(blockIdx.x / a.splits) * kTileN;
  const int split = blockIdx.x % a.splits;
  if (n0 >= nc) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  int64_t col[2];
  int tgt[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    col[j] = n0 + wn * 64 + j * 32 + (lane & 31);
    tgt[j] = col[j] < nc ? a.tgt[col[j]] : -1;
  }
  const int vt0 = (int)((int64_t)a.vtiles * split / a.splits), vt1 = (int)((int64_t)a.vtiles * (split + 1) / a.splits);
  for (int vt = vt0; vt < vt1; ++vt) {
    f32x16 acc[2][2];
    clear(acc);
    product_tile<T, false, false>(a.p, (int64_t)vt * kTileM, n0, a.v, nc, 0, 0, 0, a.kb, lds, acc);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int vb = vt * kTileM + wm * 64 + i * 32;
      float b[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) b[r] = a.bias2[vb + mma_row(r)];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
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
            if (d == mma_row(r)) a.hit[col[j]] = t[r];
        }
      }
    }
  }
  // a logit that is NaN leaves the maximum as it was and the sum NaN
  float *s_m = reinterpret_cast<float *>(lds), *s_l = s_m + 2 * kTileN;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float om = __shfl_xor(m[j], 32), ol = __shfl_xor(l[j], 32), top = fmaxf(m[j], om), base = top == -INFINITY ? 0.0f : top;
    const float sum = l[j] * __builtin_amdgcn_exp2f(m[j] - base) + ol * __builtin_amdgcn_exp2f(om - base);
    if (lane < 32) {
      const int at = wm * kTileN + wn * 64 + j * 32 + lane;
      s_m[at] = top;
      s_l[at] = sum;
    }
  }
  __syncthreads();
  if (threadIdx.x < kTileN) {
    const float m0 = s_m[threadIdx.x], m1 = s_m[kTileN + threadIdx.x], top = fmaxf(m0, m1), base = top == -INFINITY ? 0.0f : top;
    const int64_t at = split * a.n_pad + n0 + threadIdx.x;
    a.part_m[at] = top;
    a.part_l[at] = s_l[threadIdx.x] * __builtin_amdgcn_exp2f(m0 - base) + s_l[kTileN + threadIdx.x] * __builtin_amdgcn_exp2f(m1 - base);
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
// The factor that is taken out of dl: the one weight of a sum or a mean, the largest weight of single points.
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
  int64_t v, kb;
  int64_t piece0, piece, dl_plane;      // first class of the piece, its width in the workspace (a multiple of 128)
  int32_t vtiles;
  float held;      // 2^15 for float16
  const float *bias2, *lse2, *weight;
  const int32_t *tgt;
  const Counted *counted;
  void *dl;        // [planes][points][piece]
};

template <class T, int kPlanes>
__global__ __launch_bounds__(kMmaThreads, 2) void k_ce_dl(DlArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[4 * kOperandElems];
  const int nc = a.counted->n;
  const int64_t n0 = (int64_t)(blockIdx.x / a.vtiles) * kTileN;
  const int vt = blockIdx.x % a.vtiles;
  if (n0 >= nc) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  f32x16 acc[2][2];
  clear(acc);
  product_tile<T, false, false>(a.p, a.piece0 + (int64_t)vt * kTileM, n0, a.v, nc, 0, 0, 0, a.kb, lds, acc);
  T *dl = static_cast<T *>(a.dl);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t col = n0 + wn * 64 + j * 32 + (lane & 31);
    const bool in = col < nc;
    const int tgt = in ? a.tgt[col] : -1;
    const float lse2 = in ? a.lse2[col] : 0.0f, weight = a.weight[col] * a.held;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int local = vt * kTileM + wm * 64 + i * 32;
      const int64_t vb = a.piece0 + local;
      const int64_t d = tgt - vb;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, a.bias2[vb + mma_row(r)]) - lse2);
      if (__any(d >= 0 && d < 32)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] -= d == mma_row(r) ? 1.0f : 0.0f;
      }
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 q[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = in ? p[r + e] * weight : 0.0f;
          if constexpr (kPlanes == 3) {
            T h, mm, l;
            split3(w, h, mm, l);
            q[0][e] = h;
            q[1][e] = mm;
            q[2][e] = l;
          } else {
            q[0][e] = (T)w;
          }
        }
#pragma unroll
        for (int k = 0; k < kPlanes; ++k) *reinterpret_cast<t4 *>(dl + k * a.dl_plane + col * a.piece + local + mma_row(r)) = q[k];
      }
    }
  }
}

struct OutArgs {
  Product p;
  int64_t m, n, k_rows_a, k_rows_b;      // k_rows: storage rows of a "columns" operand
  int64_t cols_a, cols_b, kb;
  int32_t m_counted, k_counted;          // the dimension is the points: take it from the device
  int32_t mtiles, ntiles, splits, add;
  const Counted *counted;
  float *out;                            // [splits][m_pad][ld]
  int64_t ld, split_stride;
  float *row_sum;                        // [splits][m_pad]: sums over k of A, or null
};

template <class T>
__device__ __forceinline__ float sum8(typename Mma<T>::v8 v, float s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s += (float)v[i];
  return s;
}

// The products with dl: dx = dl W (A rows, B columns) and dW = dl^T x (both columns), in 32 bits into the workspace.
template <class T, bool kACols>
__global__ __launch_bounds__(kMmaThreads, 2) void k_ce_out(OutArgs a) {
  __shared__ __attribute__((aligned(128))) T lds[4 * kOperandElems];
  const int nc = a.counted->n;
  const int tiles = a.mtiles * a.ntiles, tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int64_t m0 = (int64_t)(tile / a.ntiles) * kTileM, n0 = (int64_t)(tile % a.ntiles) * kTileN;
  const int64_t m = a.m_counted ? nc : a.m, kb = a.k_counted ? (nc + kTileK - 1) / kTileK : a.kb;
  if (m0 >= m) return;
  const int64_t kb0 = kb * split / a.splits, kb1 = kb * (split + 1) / a.splits;
  f32x16 acc[2][2];
  clear(acc);
  product_tile<T, kACols, true>(a.p, m0, n0, kACols ? a.k_rows_a : m, a.k_counted ? nc : a.k_rows_b, a.cols_a, a.cols_b, kb0, kb1, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t n = n0 + wn * 64 + j * 32 + (lane & 31);
      if (n >= a.n) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t row = m0 + wm * 64 + i * 32 + mma_row(r);
        float *at = a.out + split * a.split_stride + row * a.ld + n;
        if (row < m) *at = a.add ? *at + acc[i][j][r] : acc[i][j][r];
      }
    }
}

// db: the columns of dl summed over the points, a thread per class and slice of the points.
template <class T, int kPlanes>
__global__ __launch_bounds__(256) void k_ce_db(const T *dl, int64_t piece, int64_t plane, const Counted *counted, int32_t slices, float *out) {
  const int nc = counted->n;
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= piece) return;
  const int64_t lo = (int64_t)nc * blockIdx.y / slices, hi = (int64_t)nc * (blockIdx.y + 1) / slices;
  float sum = 0.0f;
  for (int64_t n = lo; n < hi; ++n)
#pragma unroll
    for (int k = 0; k < kPlanes; ++k) sum += (float)dl[k * plane + n * piece + c];
  out[blockIdx.y * piece + c] = sum;
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

// Splits joined, the factor put back, one rounding.
template <class S>
__global__ __launch_bounds__(256) void k_ce_finish(FinishArgs a) {
  const float scale = *a.scale * a.unheld;
  const int64_t all = a.rows * a.width;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / a.width, c = i - r * a.width, at = a.place ? a.place[r] : r;
    float sum = 0.0f;
    if (at >= 0) {
      for (int s = 0; s < a.splits; ++s) sum += a.acc[s * a.split_stride + at * a.ld + c];
      sum *= scale;
    }
    static_cast<S *>(a.out)[r * a.ld_out + c] = (S)sum;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
constexpr int64_t kPieceBytes = 256ll << 20;      // what a piece's dl may take: the last-level cache's size

int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Plan {
  bool direct;      // the operands are multiplied where they lie
  int planes, type_bytes;
  int64_t dp, n_pad, v_pad, piece;
  int lse_splits, dx_splits, dw_splits, db_slices, top_parts, groups;
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
  p.direct = p.planes == 1 && d.d % kTileK == 0 && d.ld_x % 8 == 0 && d.ld_w % 8 == 0 && aligned16(d.x) && aligned16(d.w);
  p.dp = up(d.d, kTileK);
  p.n_pad = up(d.n, kTileN);
  p.v_pad = up(d.v, kTileM);
  p.groups = (int)((d.n + kCountRows - 1) / kCountRows);
  const int64_t ntiles = p.n_pad / kTileN, vtiles = p.v_pad / kTileM;
  auto splits = [](int64_t tiles, int64_t most) {      // about two workgroups a CU
    int64_t s = (512 + tiles - 1) / tiles;
    return (int)(s < 1 ? 1 : s > most ? (most < 1 ? 1 : most) : s);
  };
  Carver c(workspace);
  p.bias2 = c.take<float>(p.v_pad);
  if (!p.direct) {
    p.xp = c.take<uint16_t>((size_t)p.planes * p.n_pad * p.dp);
    p.wp = c.take<uint16_t>((size_t)p.planes * p.v_pad * p.dp);
  }
  if (!backward) {
    p.lse_splits = splits(ntiles, vtiles);
    p.part = c.take<int32_t>(p.groups);
    p.part_m = c.take<float>((size_t)p.lse_splits * p.n_pad);
    p.part_l = c.take<float>((size_t)p.lse_splits * p.n_pad);
    p.hit = c.take<float>(p.n_pad);
    p.sums = c.take<double>((d.n + 255) / 256);
  } else {
    int64_t piece = d.piece > 0 ? up(d.piece, kTileM) : kPieceBytes / (p.n_pad * 2 * p.planes) / kTileM * kTileM;
    if (piece < kTileM) piece = kTileM;
    p.piece = piece < p.v_pad ? piece : p.v_pad;
    const int64_t dtiles = (p.dp + kTileN - 1) / kTileN;
    p.dx_splits = splits(ntiles * dtiles, p.piece / kTileK / 4);
    p.dw_splits = splits(p.piece / kTileM * dtiles, p.n_pad / kTileK / 4);
    p.db_slices = splits((p.piece + 255) / 256, (d.n + 63) / 64);
    p.top_parts = (int)(d.n < 256 * 256 ? (d.n + 255) / 256 : 256);
    p.top = c.take<float>(p.top_parts);
    p.scale = c.take<float>(1);
    p.weight = c.take<float>(p.n_pad);
    p.dl = c.take<uint16_t>((size_t)p.planes * p.n_pad * p.piece);
    p.accx = c.take<float>((size_t)p.dx_splits * p.n_pad * p.dp);
    p.accw = c.take<float>((size_t)p.dw_splits * p.piece * p.dp);
    p.accb = c.take<float>((size_t)p.db_slices * p.piece);
  }
  p.bytes = c.off;
  return p;
}

int check(const r3d_linear_ce_t *d) {
  if (!d) return fail(R3D_E_ARG, "linear_ce: null descriptor");
  if (d->n <= 0 || d->v <= 0 || d->d <= 0 || d->n > INT32_MAX - 1024 || d->v > INT32_MAX - 1024 || d->d > (1 << 20) || d->ld_x < d->d || d->ld_w < d->d ||
      d->piece < 0)
    return fail(R3D_E_ARG, "linear_ce: bad size");
  if (d->type != R3D_T_F32 && d->type != R3D_T_BF16 && d->type != R3D_T_F16) return fail(R3D_E_ARG, "linear_ce: type");
  if (d->target_type != R3D_T_I32 && d->target_type != R3D_T_I64) return fail(R3D_E_ARG, "linear_ce: type of the targets");
  if (d->reduction != R3D_CE_NONE && d->reduction != R3D_CE_SUM && d->reduction != R3D_CE_MEAN) return fail(R3D_E_ARG, "linear_ce: reduction");
  return R3D_OK;
}

template <class S, class T, int kPlanes>
void pack(const PackArgs &a, int64_t rows, hipStream_t st) {
  hipLaunchKernelGGL((k_ce_pack<S, T, kPlanes>), dim3(blocks_for(rows * a.ld_out, 1024, 8192)), dim3(256), 0, st, a);
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
  pack<S, T, kPlanes>(PackArgs{d.x, p.xp, d.ld_x, d.n, d.d, p.dp, p.n_pad * p.dp, d.idx, counted}, d.n, st);
  pack<S, T, kPlanes>(PackArgs{d.w, p.wp, d.ld_w, d.v, d.d, p.dp, p.v_pad * p.dp, nullptr, nullptr}, d.v, st);
  x = Operand{p.xp, p.dp, p.n_pad * p.dp, nullptr};
  w = Operand{p.wp, p.dp, p.v_pad * p.dp, nullptr};
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
  la.vtiles = (int)(p.v_pad / kTileM);
  la.splits = p.lse_splits;
  la.bias2 = p.bias2;
  la.tgt = d.tgt;
  la.counted = counted;
  la.part_m = p.part_m;
  la.part_l = p.part_l;
  la.hit = p.hit;
  la.n_pad = p.n_pad;
  hipLaunchKernelGGL(k_ce_lse<T>, dim3((unsigned)(p.n_pad / kTileN * p.lse_splits)), dim3(kMmaThreads), 0, st, la);
  CombineArgs ca{p.part_m, p.part_l, p.hit, d.tgt, d.place, counted, d.lse2, d.reduction == R3D_CE_NONE ? d.loss : nullptr, d.loss, p.sums, d.n, p.n_pad,
                 p.lse_splits};
  const int blocks = (int)((d.n + 255) / 256);
  hipLaunchKernelGGL(k_ce_join, dim3(blocks), dim3(256), 0, st, ca);
  if (d.reduction != R3D_CE_NONE)
    hipLaunchKernelGGL(k_ce_mean, dim3(1), dim3(256), 0, st, p.sums, (int64_t)blocks, counted, d.reduction == R3D_CE_MEAN ? 1 : 0, d.loss);
}

template <class S, class T, int kPlanes>
void backward(const r3d_linear_ce_t &d, const Plan &p, hipStream_t st) {
  const Counted *counted = static_cast<const Counted *>(d.counted);
  const bool each = d.reduction == R3D_CE_NONE;
  if (each) hipLaunchKernelGGL(k_ce_top, dim3(p.top_parts), dim3(256), 0, st, d.grad, d.n, d.place, p.top);
  hipLaunchKernelGGL(k_ce_weight, dim3(blocks_for(p.n_pad, 256, 1 << 30)), dim3(256), 0, st,
                     WeightArgs{d.grad, p.top, each ? 1 : 0, p.top_parts, d.idx, counted, p.scale, p.weight, p.n_pad});
  Operand x, w;
  operands<S, T, kPlanes>(d, p, counted, st, x, w);
  const float held = d.type == R3D_T_F16 ? 32768.0f : 1.0f;
  const int64_t dtiles = (p.dp + kTileN - 1) / kTileN;
  for (int64_t v0 = 0; v0 < p.v_pad; v0 += p.piece) {
    const int64_t wide_v = p.piece < p.v_pad - v0 ? p.piece : p.v_pad - v0;      // (a multiple of 128)
    const int64_t real_v = wide_v < d.v - v0 ? wide_v : d.v - v0;
    DlArgs da{};
    da.p = Product{w, x, kPlanes};
    da.v = d.v;
    da.kb = p.dp / kTileK;
    da.piece0 = v0;
    da.piece = p.piece;
    da.dl_plane = p.n_pad * p.piece;
    da.vtiles = (int)(wide_v / kTileM);
    da.held = held;
    da.bias2 = p.bias2;
    da.lse2 = d.lse2;
    da.weight = p.weight;
    da.tgt = d.tgt;
    da.counted = counted;
    da.dl = p.dl;
    hipLaunchKernelGGL((k_ce_dl<T, kPlanes>), dim3((unsigned)(p.n_pad / kTileN * da.vtiles)), dim3(kMmaThreads), 0, st, da);
    const Operand dl{p.dl, p.piece, p.n_pad * p.piece, nullptr};
    if (d.dx) {
      Operand wv = w;      // the rows of this piece
      wv.p = static_cast<const char *>(w.p) + v0 * w.ld * 2;
      OutArgs oa{};
      oa.p = Product{dl, wv, kPlanes};
      oa.n = p.dp;
      oa.k_rows_b = real_v;
      oa.cols_b = p.dp;
      oa.kb = wide_v / kTileK;
      oa.m_counted = 1;
      oa.mtiles = (int)(p.n_pad / kTileM);
      oa.ntiles = (int)dtiles;
      oa.splits = p.dx_splits;
      oa.add = v0 > 0;
      oa.counted = counted;
      oa.out = p.accx;
      oa.ld = p.dp;
      oa.split_stride = p.n_pad * p.dp;
      hipLaunchKernelGGL((k_ce_out<T, false>), dim3((unsigned)(oa.mtiles * dtiles * oa.splits)), dim3(kMmaThreads), 0, st, oa);
    }
    if (d.dw) {
      OutArgs oa{};
      oa.p = Product{dl, x, kPlanes};
      oa.m = wide_v;
      oa.n = p.dp;
      oa.k_rows_a = p.n_pad;
      oa.k_counted = 1;
      oa.cols_a = p.piece;
      oa.cols_b = p.dp;
      oa.mtiles = (int)(wide_v / kTileM);
      oa.ntiles = (int)dtiles;
      oa.splits = p.dw_splits;
      oa.counted = counted;
      oa.out = p.accw;
      oa.ld = p.dp;
      oa.split_stride = p.piece * p.dp;
      hipLaunchKernelGGL((k_ce_out<T, true>), dim3((unsigned)(oa.mtiles * dtiles * oa.splits)), dim3(kMmaThreads), 0, st, oa);
      FinishArgs fa{p.accw, p.dp, p.piece * p.dp, real_v, d.d, d.d, p.dw_splits, 1.0f / held, nullptr, p.scale,
                    static_cast<char *>(d.dw) + v0 * d.d * p.type_bytes};
      hipLaunchKernelGGL(k_ce_finish<S>, dim3(blocks_for(real_v * d.d, 1024, 8192)), dim3(256), 0, st, fa);
    }
    if (d.db) {
      hipLaunchKernelGGL((k_ce_db<T, kPlanes>), dim3((unsigned)((wide_v + 255) / 256), p.db_slices), dim3(256), 0, st,
                         static_cast<const T *>(p.dl), p.piece, p.n_pad * p.piece, counted, p.db_slices, p.accb);
      FinishArgs fa{p.accb, 1, p.piece, real_v, 1, 1, p.db_slices, 1.0f / held, nullptr, p.scale,
                    static_cast<char *>(d.db) + v0 * p.type_bytes};
      hipLaunchKernelGGL(k_ce_finish<S>, dim3(blocks_for(real_v, 256, 8192)), dim3(256), 0, st, fa);
    }
  }
  if (d.dx) {
    FinishArgs fa{p.accx, p.dp, p.n_pad * p.dp, d.n, d.d, d.d, p.dx_splits, 1.0f / held, d.place, p.scale, d.dx};
    hipLaunchKernelGGL(k_ce_finish<S>, dim3(blocks_for(d.n * d.d, 1024, 8192)), dim3(256), 0, st, fa);
  }
}
}  // namespace

extern "C" size_t r3d_linear_ce_workspace_bytes(const r3d_linear_ce_t *d, int32_t backward_pass) {
  if (check(d) != R3D_OK) return 0;
  return plan(*d, backward_pass != 0, nullptr).bytes;
}

extern "C" int r3d_linear_ce_forward(const r3d_linear_ce_t *d, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check(d);
  if (rc != R3D_OK) return rc;
  if (!d->x || !d->w || !d->target || !d->idx || !d->place || !d->tgt || !d->lse2 || !d->counted || !d->loss || !workspace)
    return fail(R3D_E_ARG, "linear_ce_forward: null pointer");
  const Plan p = plan(*d, false, workspace);
  if (workspace_bytes < p.bytes) return fail(R3D_E_WORKSPACE, "linear_ce_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
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
  const Plan p = plan(*d, true, workspace);
  if (workspace_bytes < p.bytes) return fail(R3D_E_WORKSPACE, "linear_ce_backward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->type == R3D_T_F32) backward<float, __bf16, 3>(*d, p, st);
  else if (d->type == R3D_T_BF16) backward<__bf16, __bf16, 1>(*d, p, st);
  else backward<_Float16, _Float16, 1>(*d, p, st);
  R3D_LAUNCHED("linear_ce backward kernels");
  return R3D_OK;
}

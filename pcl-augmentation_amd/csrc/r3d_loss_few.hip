// Softmax cross entropy of a linear head over few classes (gfx950): the labels of a point.
//
// With 20 classes the products are small and the features are everything: 480 000 points x 96 features are 92 MB to read and,
// backward, 92 MB to write.  So the features pass through once a call: a workgroup takes tiles of points, a wave 32 of them; the
// logits of a tile are one product with the head (which stays in LDS), the softmax of a point lies in the registers of two
// lanes, and in the backward pass the gradient of the features leaves from there while dW = dl^T x adds up in registers over all
// tiles of the workgroup.  The next tile's features are on their way meanwhile.  The forward pass keeps nothing: the backward
// pass makes the logits again, from features it has to read anyway.
//
// Same numbers as r3d_loss.hip: sums in 32 bits, dl rounded to the 16-bit type (three bfloat16 planes for float32), float16's dl
// held times 2^15.  Points whose target is ignored become rows of zeros on the way into LDS.
#include "r3d_host.hpp"
#include "r3d_loss.hpp"

namespace {
using namespace r3d;

constexpr int kThreads = 256, kLdsMost = 160 * 1024, kTopParts = 256;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct FewArgs {
  const void *x, *w, *bias, *target;
  int64_t ld_x, ld_w, n, ignore;
  int32_t v, d, dp, magic;      // dp: d padded to 32; magic: c / (dp / pieces of 16 bytes) = c * magic >> 20
  int32_t wide_target, vector, vector_out;
  float *each;                  // loss of every point, or null:
  double *sums;                 // sums of a workgroup's points
  int32_t *counts;
  // backward
  const float *grad, *top;      // top: [parts] largest weights of points, where they are taken out of dl
  const Counted *counted;
  int32_t grad_each, parts;
  float held, unheld;
  void *dx;
  float *part;                  // [workgroups][classes padded to 32][dp + 1]: dW, and db behind it
  int32_t want_w;
};

// The factor that is taken out of dl: the one weight of a sum or a mean; for float16 the largest weight of single points.
__device__ __forceinline__ float taken_out(const FewArgs &a) {
  if (!a.grad_each) return a.counted->n ? a.grad[0] * a.counted->share : 0.0f;      // (of no point: 0, whatever comes in)
  float top = 0.0f;
  for (int i = threadIdx.x & 63; i < a.parts; i += 64) top = fmaxf(top, a.top[i]);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  return top > 0.0f ? top : 1.0f;
}

template <class V>
__device__ __forceinline__ u32x4 load_piece(const FewArgs &a, int64_t row, int col) {
  constexpr int kEach = 16 / sizeof(V);
  u32x4 r = {0, 0, 0, 0};
  if (row >= a.n) return r;
  const V *at = static_cast<const V *>(a.x) + row * a.ld_x + col;
  if (a.vector && col + kEach <= a.d) return *reinterpret_cast<const u32x4 *>(at);
  alignas(16) V v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) v[e] = col + e < a.d ? at[e] : (V)0.0f;
  return *reinterpret_cast<const u32x4 *>(v);
}

// 16 bytes of a row into the LDS planes.
template <class V, class T, int kPlanes>
__device__ __forceinline__ void store_piece(T *to, int plane, u32x4 piece) {
  if constexpr (kPlanes == 1) {
    *reinterpret_cast<u32x4 *>(to) = piece;
  } else {
    typedef float f4 __attribute__((ext_vector_type(4)));
    typedef T t4 __attribute__((ext_vector_type(4)));
    const f4 v = __builtin_bit_cast(f4, piece);
    t4 h, m, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      T ph, pm, pl;
      split3(v[e], ph, pm, pl);
      h[e] = ph;
      m[e] = pm;
      l[e] = pl;
    }
    *reinterpret_cast<t4 *>(to) = h;
    *reinterpret_cast<t4 *>(to + plane) = m;
    *reinterpret_cast<t4 *>(to + 2 * plane) = l;
  }
}

// Waves a SIMD the registers are cut for: what the tile's LDS lets stand beside each other anyway.  480 000 x 20 x 96 bf16,
// backward: 68 us with one, 57 with three (which spill 9 vector registers and are faster all the same); 200 000 x 20 x 256: 114 with one, 69 with two.
constexpr int few_waves(int planes, int vt, int nb) { return planes == 3 ? (vt * nb == 1 ? 2 : 1) : vt * nb == 1 ? 3 : vt * nb == 2 ? 2 : 1; }

// kVT: blocks of 32 classes; kNB: blocks of 32 features of dW a wave keeps (dp <= 128 kNB); kTP: points of a tile.
template <class V, class T, int kPlanes, int kVT, int kNB, int kTP, bool kGrad>
__global__ __launch_bounds__(kThreads, few_waves(kPlanes, kVT, kNB)) void k_few(FewArgs a) {
  constexpr int kEach = 16 / sizeof(V), kPer = kTP * kNB * 128 / kEach / kThreads, kPv = kVT * 32 + 8;
  constexpr int kPairCount = kPlanes == 3 ? kPairs : 1;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int pitch = a.dp + 8;      // an odd number of 16 bytes: rows begin on different banks
  T *xs = reinterpret_cast<T *>(smem), *ws = xs + kPlanes * kTP * pitch, *dls = ws + kPlanes * kVT * 32 * pitch;
  float *bias2 = reinterpret_cast<float *>(dls + (kGrad ? kPlanes * kTP * kPv : 0));
  int *s_tgt = reinterpret_cast<int *>(bias2 + kVT * 32);      // [2][kTP]: class, -1 no class, -2 does not count
  float *s_weight = reinterpret_cast<float *>(s_tgt + 2 * kTP);  // [2][kTP]
  const int x_plane = kTP * pitch, w_plane = kVT * 32 * pitch, d_plane = kTP * kPv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, low = lane & 31, group = lane >> 4, sub = lane & 15;
  const int cols = a.dp / kEach, pieces = kTP * cols;
  const int64_t tiles = (a.n + kTP - 1) / kTP;

  // the head and the bias, once
  for (int c = threadIdx.x; c < kVT * 32 * cols; c += kThreads) {
    const int r = c / cols, col = (c - r * cols) * kEach;
    alignas(16) V v[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = r < a.v && col + e < a.d ? static_cast<const V *>(a.w)[r * a.ld_w + col + e] : (V)0.0f;
    store_piece<V, T, kPlanes>(ws + r * pitch + col, w_plane, *reinterpret_cast<const u32x4 *>(v));
  }
  for (int c = threadIdx.x; c < kVT * 32; c += kThreads)
    bias2[c] = c >= a.v ? -INFINITY : a.bias ? (float)static_cast<const V *>(a.bias)[c] * kLog2e : 0.0f;

  u32x4 reg[kPer];
  auto fetch = [&](int64_t tile) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = i * kThreads + threadIdx.x;
      if (c < pieces) {
        const int r = (int)(((unsigned)c * (unsigned)a.magic) >> 20);
        reg[i] = load_piece<V>(a, tile * kTP + r, (c - r * cols) * kEach);
      }
    }
  };
  auto target = [&](int64_t tile) {
    const int64_t i = tile * kTP + threadIdx.x;
    if (threadIdx.x >= kTP || i >= a.n) return -2;
    const int64_t t = a.wide_target ? static_cast<const int64_t *>(a.target)[i] : static_cast<const int32_t *>(a.target)[i];
    return t == a.ignore ? -2 : t >= 0 && t < a.v ? (int)t : -1;
  };
  const float scale = kGrad ? taken_out(a) : 1.0f;
  auto weight = [&](int64_t tile) {
    const int64_t i = tile * kTP + threadIdx.x;
    return kGrad && a.grad_each && threadIdx.x < kTP && i < a.n ? a.grad[i] / scale : 1.0f;
  };

  double loss_sum = 0.0;
  int count = 0;
  f32x16 acc_w[kGrad ? kVT : 1][kGrad ? kNB : 1];
  float sums[kVT];      // db of the wave's points, before dl is rounded
  if constexpr (kGrad) clear(acc_w);
#pragma unroll
  for (int v = 0; v < kVT; ++v) sums[v] = 0.0f;

  int64_t tile = blockIdx.x;
  int at = 0;
  if (tile < tiles) {
    fetch(tile);
    if (threadIdx.x < kTP) {
      s_tgt[threadIdx.x] = target(tile);
      if constexpr (kGrad) s_weight[threadIdx.x] = weight(tile);
    }
  }
  __syncthreads();
  for (; tile < tiles; tile += gridDim.x) {
    const int *tgt = s_tgt + at * kTP;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = i * kThreads + threadIdx.x;
      if (c < pieces) {
        const int r = (int)(((unsigned)c * (unsigned)a.magic) >> 20);
        const bool counts = tgt[r] != -2;
        const u32x4 zero = {0, 0, 0, 0};
        store_piece<V, T, kPlanes>(xs + r * pitch + (c - r * cols) * kEach, x_plane, counts ? reg[i] : zero);
      }
    }
    __syncthreads();
    const int64_t next = tile + gridDim.x;
    int next_tgt = -2;
    float next_weight = 1.0f;
    if (next < tiles) {
      fetch(next);
      next_tgt = target(next);
      next_weight = weight(next);
    }
    if (wave < kTP / 32) {
      f32x16 acc[kVT];
#pragma unroll
      for (int v = 0; v < kVT; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[v][r] = 0.0f;
#pragma unroll
      for (int pr = 0; pr < kPairCount; ++pr) {
        const T *wa = ws + kPlaneA[pr] * w_plane + low * pitch + half * 8, *xb = xs + kPlaneB[pr] * x_plane + (wave * 32 + low) * pitch + half * 8;
        for (int k = 0; k < a.dp; k += 16) {
          const auto fb = *reinterpret_cast<const typename Mma<T>::v8 *>(xb + k);
#pragma unroll
          for (int v = 0; v < kVT; ++v) acc[v] = Mma<T>::mma(*reinterpret_cast<const typename Mma<T>::v8 *>(wa + v * 32 * pitch + k), fb, acc[v]);
        }
      }
      // a point's classes: 16 kVT in this lane, the rest 32 lanes on
      const int t = tgt[wave * 32 + low];
      float top = -INFINITY, sum = 0.0f, hit = -INFINITY;
#pragma unroll
      for (int v = 0; v < kVT; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          acc[v][r] = logit2(acc[v][r], bias2[v * 32 + mma_row(r)]);
          top = fmaxf(top, acc[v][r]);
          hit = t == v * 32 + mma_row(r) ? acc[v][r] : hit;
        }
      top = fmaxf(top, __shfl_xor(top, 32));
      const float base = base_of(top);
#pragma unroll
      for (int v = 0; v < kVT; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += acc[v][r] = part_of(acc[v][r], base);
      sum += __shfl_xor(sum, 32);
      if constexpr (!kGrad) {
        // (only the lane that holds the target's logit has it; the other's stays -inf)
        const float other = __shfl_xor(hit, 32);
        const float mine = t >= 0 && ((t >> 2) & 1) == half ? hit : other;
        const float loss = t == -2 ? 0.0f : t == -1 ? NAN : point_loss(top, sum, mine);
        const int64_t i = tile * kTP + wave * 32 + low;
        if (half == 0) {
          if (a.each) {
            if (i < a.n) a.each[i] = loss;
          } else {
            loss_sum += loss;
          }
          count += t != -2;
        }
      } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const float share = t == -2 ? 0.0f : t == -1 ? NAN : s_weight[at * kTP + wave * 32 + low] * a.held / sum;
        t4 q[kVT][4][kPlanes];
#pragma unroll
        for (int v = 0; v < kVT; ++v) {
          float w[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float p = t == -2 ? 0.0f : (acc[v][r] - (t == v * 32 + mma_row(r) ? sum : 0.0f)) * share;
            w[r] = p;
            if constexpr (kPlanes == 3) {
              T h, m, l;
              split3(p, h, m, l);
              q[v][r >> 2][0][r & 3] = h;
              q[v][r >> 2][1][r & 3] = m;
              q[v][r >> 2][2][r & 3] = l;
            } else {
              q[v][r >> 2][0][r & 3] = (T)p;
            }
          }
          if (a.want_w) sums[v] += block_sum(w);
        }
#pragma unroll
        for (int v = 0; v < kVT; ++v)
#pragma unroll
          for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int k = 0; k < kPlanes; ++k)
              *reinterpret_cast<t4 *>(dls + k * d_plane + (wave * 32 + low) * kPv + v * 32 + 8 * h + 4 * half) = q[v][h][k];
        if (a.dx) {
          // dx = dl W: features are the rows of C.  The classes of a k-step are taken in the order in which the lanes have
          // them (fours of a lane, then of the next block of 8), from both operands alike.
          const float out_scale = t == -2 ? 0.0f : scale * a.unheld;      // (a factor that is infinite or no number makes 0 NaN)
          const int64_t i = tile * kTP + wave * 32 + low;
          V *out = static_cast<V *>(a.dx) + i * a.d;
          const T *wt = ws + (4 * half + (sub >> 2)) * pitch + (group & 1) * 16 + (sub & 3) * 4;
          for (int f0 = 0; f0 < a.dp; f0 += 32) {
            f32x16 g;
#pragma unroll
            for (int r = 0; r < 16; ++r) g[r] = 0.0f;
#pragma unroll
            for (int pr = 0; pr < kPairCount; ++pr)
#pragma unroll
              for (int v = 0; v < kVT; ++v)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                  const T *lo = wt + kPlaneA[pr] * w_plane + (v * 32 + 16 * s) * pitch + f0;
                  const auto fb = __builtin_bit_cast(typename Mma<T>::v8, __builtin_shufflevector(q[v][2 * s][kPlaneB[pr]], q[v][2 * s + 1][kPlaneB[pr]], 0, 1, 2, 3, 4, 5, 6, 7));
                  g = Mma<T>::mma(turned<T>(lo, lo + 8 * pitch), fb, g);
                }
            if (i >= a.n) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) g[r] *= out_scale;
            if (a.vector_out && f0 + 32 <= a.d) {
              if constexpr (sizeof(V) == 4) {
#pragma unroll
                for (int h = 0; h < 4; ++h)
                  *reinterpret_cast<float4 *>(out + f0 + 8 * h + 4 * half) = make_float4(g[4 * h], g[4 * h + 1], g[4 * h + 2], g[4 * h + 3]);
              } else {
                typedef V v4 __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                  const v4 o = {(V)g[4 * h], (V)g[4 * h + 1], (V)g[4 * h + 2], (V)g[4 * h + 3]};
                  *reinterpret_cast<v4 *>(out + f0 + 8 * h + 4 * half) = o;
                }
              }
            } else {
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (f0 + mma_row(r) < a.d) out[f0 + mma_row(r)] = (V)g[r];
            }
          }
        }
      }
    }
    __syncthreads();
    at ^= 1;
    if (threadIdx.x < kTP) {
      s_tgt[at * kTP + threadIdx.x] = next_tgt;
      if constexpr (kGrad) s_weight[at * kTP + threadIdx.x] = next_weight;
    }
    if constexpr (kGrad) {
      if (a.want_w) {
        // dW += dl^T x: every wave its features, all points of the tile
        const int row = (group >> 1) * 8 + (sub >> 2), col = (group & 1) * 16 + (sub & 3) * 4;
        for (int k = 0; k < kTP; k += 16)
#pragma unroll
          for (int pr = 0; pr < kPairCount; ++pr) {
            typename Mma<T>::v8 fa[kVT];
            const T *dt = dls + kPlaneA[pr] * d_plane + (k + row) * kPv + col, *xt = xs + kPlaneB[pr] * x_plane + (k + row) * pitch + col;
#pragma unroll
            for (int v = 0; v < kVT; ++v) {
              fa[v] = turned<T>(dt + v * 32, dt + v * 32 + 4 * kPv);
            }
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
              const int f0 = (wave + 4 * b) * 32;
              if (f0 < a.dp) {
                const auto fb = turned<T>(xt + f0, xt + f0 + 4 * pitch);
#pragma unroll
                for (int v = 0; v < kVT; ++v) acc_w[v][b] = Mma<T>::mma(fa[v], fb, acc_w[v][b]);
              }
            }
          }
      }
    }
    __syncthreads();
  }
  if constexpr (kGrad) {
    if (!a.want_w) return;
    float *part = a.part + (int64_t)blockIdx.x * (kVT * 32) * (a.dp + 1);
#pragma unroll
    for (int v = 0; v < kVT; ++v) {
#pragma unroll
      for (int b = 0; b < kNB; ++b) {
        const int f0 = (wave + 4 * b) * 32;
        if (f0 < a.dp)
#pragma unroll
          for (int r = 0; r < 16; ++r) part[(v * 32 + mma_row(r)) * a.dp + f0 + low] = acc_w[v][b][r];
      }
    }
    float *s_sum = reinterpret_cast<float *>(smem);      // [waves][classes] (nobody reads the tile any more)
#pragma unroll
    for (int v = 0; v < kVT; ++v)
      if ((lane & 15) < 8) s_sum[wave * kVT * 32 + v * 32 + block_sum_row()] = sums[v];
    __syncthreads();
    for (int c = threadIdx.x; c < kVT * 32; c += kThreads)
      part[kVT * 32 * a.dp + c] = s_sum[c] + s_sum[kVT * 32 + c] + s_sum[2 * kVT * 32 + c] + s_sum[3 * kVT * 32 + c];
  } else {
    __syncthreads();
    double *s_sum = reinterpret_cast<double *>(smem);
    int *s_count = reinterpret_cast<int *>(s_sum + 4);
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      loss_sum += __shfl_xor(loss_sum, d);
      count += __shfl_xor(count, d);
    }
    if (lane == 0) {
      s_sum[wave] = loss_sum;
      s_count[wave] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      a.sums[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
      a.counts[blockIdx.x] = s_count[0] + s_count[1] + s_count[2] + s_count[3];
    }
  }
}

// The workgroups' sums joined; what the backward pass needs of it.
__global__ __launch_bounds__(256) void k_few_mean(const double *sums, const int32_t *counts, int n, int reduction, float *loss, Counted *counted) {
  __shared__ double s[4];
  __shared__ int sc[4];
  double d = 0.0;
  int c = 0;
  for (int i = threadIdx.x; i < n; i += 256) {
    d += sums[i];
    c += counts[i];
  }
#pragma unroll
  for (int k = 32; k; k >>= 1) {
    d += __shfl_xor(d, k);
    c += __shfl_xor(c, k);
  }
  if ((threadIdx.x & 63) == 0) {
    s[threadIdx.x >> 6] = d;
    sc[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    d = s[0] + s[1] + s[2] + s[3];
    c = sc[0] + sc[1] + sc[2] + sc[3];
    const bool mean = reduction == R3D_CE_MEAN;
    if (reduction != R3D_CE_NONE) *loss = (float)(mean && c ? d / c : d);
    counted->n = c;
    counted->share = !mean ? 1.0f : c ? 1.0f / (float)c : 0.0f;
  }
}

// Largest weights of the points that count.
__global__ __launch_bounds__(256) void k_few_top(FewArgs a, float *top_out) {
  __shared__ float s[4];
  float top = 0.0f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = a.wide_target ? static_cast<const int64_t *>(a.target)[i] : static_cast<const int32_t *>(a.target)[i];
    if (t != a.ignore && fabsf(a.grad[i]) < INFINITY) top = fmaxf(top, fabsf(a.grad[i]));      // (what is no number or infinite is left out)
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) top_out[blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

// dW and db: the workgroups' sums joined, 64 values by sixteen slices of the workgroups a time.
template <class V>
__global__ __launch_bounds__(1024) void k_few_join(FewArgs a, int groups, int vp, V *dw, V *db) {
  __shared__ float s[16][64];
  const int v = a.v, d = a.d, dp = a.dp;
  const float scale = taken_out(a) * a.unheld;
  const int64_t stride = (int64_t)vp * (dp + 1);
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6, all = v * d + v, i = blockIdx.x * 64 + lane;
  float sum = 0.0f;
  if (i < all) {
    const float *from = a.part + (i < v * d ? (int64_t)(i / d) * dp + i % d : (int64_t)vp * dp + (i - v * d));
#pragma unroll 8
    for (int g = slice; g < groups; g += 16) sum += from[g * stride];
  }
  s[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && i < all) {
    sum = 0.0f;
#pragma unroll
    for (int g = 0; g < 16; ++g) sum += s[g][lane];
    sum *= scale;
    if (i < v * d) {
      if (dw) dw[i] = (V)sum;
    } else if (db) {
      db[i - v * d] = (V)sum;
    }
  }
}

struct FewPlan {
  int vt, nb, tp, dp, groups;
  size_t lds_forward, lds_backward;
};

// Whether the head is this file's: its classes and features beside a tile of points in LDS, dW in registers.
bool few_plan(const r3d_linear_ce_t &d, FewPlan &p) {
  const int planes = d.type == R3D_T_F32 ? 3 : 1;
  if (d.v > 128 || d.d > 256) return false;
  p.dp = (int)((d.d + 31) / 32 * 32);
  p.vt = d.v <= 32 ? 1 : d.v <= 64 ? 2 : 4;
  p.nb = p.dp <= 128 ? 1 : 2;
  // Beyond that, and for many points near it, the other kernels are faster.  200 000 points, us here / there: bf16 20 x 256 119 / 148,
  // 50 x 96 73 / 130, 100 x 96 128 / 138, but 50 x 200 211 / 186, 100 x 128 146 / 130, 100 x 256 284 / 170, 20 x 512 372 / 242; fp32 20 x 64
  // 94 / 175, 50 x 96 291 / 321, but 50 x 64 243 / 173.  4000 points: 50 x 200 42 / 49, 100 x 128 41 / 49, fp32 50 x 64 37 / 47.
  if (p.vt * p.nb > 4 || p.nb > 2 || (planes == 3 && p.vt == 4)) return false;
  if (planes == 1 ? p.vt * p.nb == 4 && p.dp > 96 && d.n > 65536 : p.vt == 2 && p.dp <= 64 && d.n > 32768) return false;
  p.tp = p.nb >= 2 || planes == 3 ? 64 : 128;      // (two workgroups a CU beat one with the longer tile: 200 000 x 20 x 256 forward 58 -> 38 us)
  const size_t pitch = p.dp + 8;
  p.lds_forward = (size_t)planes * 2 * (p.tp + p.vt * 32) * pitch + p.vt * 32 * 4 + (size_t)p.tp * 16;
  p.lds_backward = p.lds_forward + (size_t)planes * 2 * p.tp * (p.vt * 32 + 8);
  if (p.lds_backward > (size_t)kLdsMost) return false;
  const int64_t tiles = (d.n + p.tp - 1) / p.tp;
  const int per_cu = (int)(kLdsMost / p.lds_backward < 3 ? kLdsMost / p.lds_backward : 3);
  p.groups = (int)(tiles < 256 * per_cu ? tiles : 256 * per_cu);
  return true;
}

struct FewSpace {
  double *sums;
  int32_t *counts;
  float *top, *part;
  size_t bytes;
};
FewSpace few_space(const FewPlan &p, bool backward, void *workspace) {
  FewSpace s{};
  Carver c(workspace);
  if (!backward) {
    s.sums = c.take<double>(p.groups);
    s.counts = c.take<int32_t>(p.groups);
  } else {
    s.top = c.take<float>(kTopParts);
    s.part = c.take<float>((size_t)p.groups * p.vt * 32 * (p.dp + 1));
  }
  s.bytes = c.off;
  return s;
}

template <class V, class T, int kPlanes, int kVT, int kNB, int kTP, bool kGrad>
int launch(const FewArgs &a, const FewPlan &p, hipStream_t st) {
  const size_t lds = kGrad ? p.lds_backward : p.lds_forward;
  auto *kernel = &k_few<V, T, kPlanes, kVT, kNB, kTP, kGrad>;
  if (lds > 64 * 1024) R3D_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(kernel, dim3(p.groups), dim3(kThreads), lds, st, a);
  return R3D_OK;
}

template <class V, class T, int kPlanes, bool kGrad>
int dispatch(const FewArgs &a, const FewPlan &p, hipStream_t st) {
  const int key = p.vt * 10 + p.nb;
  if constexpr (kPlanes == 3) {
    switch (key) {
      case 11: return launch<V, T, 3, 1, 1, 64, kGrad>(a, p, st);
      case 12: return launch<V, T, 3, 1, 2, 64, kGrad>(a, p, st);
      case 21: return launch<V, T, 3, 2, 1, 64, kGrad>(a, p, st);
      default: return launch<V, T, 3, 2, 2, 64, kGrad>(a, p, st);
    }
  } else {
    switch (key) {
      case 11: return launch<V, T, 1, 1, 1, 128, kGrad>(a, p, st);
      case 12: return launch<V, T, 1, 1, 2, 64, kGrad>(a, p, st);
      case 21: return launch<V, T, 1, 2, 1, 128, kGrad>(a, p, st);
      case 22: return launch<V, T, 1, 2, 2, 64, kGrad>(a, p, st);
      default: return launch<V, T, 1, 4, 1, 128, kGrad>(a, p, st);
    }
  }
}

template <bool kGrad>
int by_type(const r3d_linear_ce_t &d, const FewArgs &a, const FewPlan &p, hipStream_t st) {
  if (d.type == R3D_T_F32) return dispatch<float, __bf16, 3, kGrad>(a, p, st);
  if (d.type == R3D_T_BF16) return dispatch<__bf16, __bf16, 1, kGrad>(a, p, st);
  return dispatch<_Float16, _Float16, 1, kGrad>(a, p, st);
}

FewArgs few_args(const r3d_linear_ce_t &d, const FewPlan &p) {
  FewArgs a{};
  const int size = d.type == R3D_T_F32 ? 4 : 2, cols = p.dp * size / 16;
  a.x = d.x;
  a.w = d.w;
  a.bias = d.bias;
  a.target = d.target;
  a.ld_x = d.ld_x;
  a.ld_w = d.ld_w;
  a.n = d.n;
  a.ignore = d.ignore_index;
  a.v = (int32_t)d.v;
  a.d = (int32_t)d.d;
  a.dp = p.dp;
  a.magic = ((1 << 20) + cols - 1) / cols;
  a.wide_target = d.target_type == R3D_T_I64;
  a.vector = reinterpret_cast<uintptr_t>(d.x) % 16 == 0 && d.ld_x * size % 16 == 0;
  return a;
}
}  // namespace

namespace r3d {

bool few_takes(const r3d_linear_ce_t &d) {
  FewPlan p;
  return few_plan(d, p);
}

size_t few_bytes(const r3d_linear_ce_t &d, int32_t which) {
  FewPlan p;
  few_plan(d, p);
  return which == R3D_CE_BYTES_STATE ? sizeof(Counted) : few_space(p, which == R3D_CE_BYTES_BACKWARD, nullptr).bytes;
}

int few_forward(const r3d_linear_ce_t &d, void *workspace, hipStream_t st) {
  FewPlan p;
  few_plan(d, p);
  const FewSpace s = few_space(p, false, workspace);
  FewArgs a = few_args(d, p);
  a.each = d.reduction == R3D_CE_NONE ? d.loss : nullptr;
  a.sums = s.sums;
  a.counts = s.counts;
  const int rc = by_type<false>(d, a, p, st);
  if (rc != R3D_OK) return rc;
  hipLaunchKernelGGL(k_few_mean, dim3(1), dim3(256), 0, st, s.sums, s.counts, p.groups, d.reduction, d.loss, static_cast<Counted *>(d.state));
  return R3D_OK;
}

int few_backward(const r3d_linear_ce_t &d, void *workspace, hipStream_t st) {
  FewPlan p;
  few_plan(d, p);
  const FewSpace s = few_space(p, true, workspace);
  FewArgs a = few_args(d, p);
  const bool half = d.type == R3D_T_F16;
  a.grad = d.grad;
  a.grad_each = d.reduction == R3D_CE_NONE;
  a.counted = static_cast<const Counted *>(d.state);
  a.top = s.top;
  a.parts = a.grad_each && half ? blocks_for(d.n, 256, kTopParts) : 0;
  a.held = half ? 32768.0f : 1.0f;
  a.unheld = 1.0f / a.held;
  a.dx = d.dx;
  a.part = s.part;
  a.want_w = d.dw || d.db;
  a.vector_out = reinterpret_cast<uintptr_t>(d.dx) % 16 == 0 && d.d % 4 == 0;
  if (a.parts) hipLaunchKernelGGL(k_few_top, dim3(a.parts), dim3(256), 0, st, a, s.top);
  const int rc = by_type<true>(d, a, p, st);
  if (rc != R3D_OK || !a.want_w) return rc;
  const dim3 blocks((unsigned)((d.v * d.d + d.v + 63) / 64));
  if (d.type == R3D_T_F32)
    hipLaunchKernelGGL(k_few_join<float>, blocks, dim3(1024), 0, st, a, p.groups, p.vt * 32, static_cast<float *>(d.dw), static_cast<float *>(d.db));
  else if (d.type == R3D_T_BF16)
    hipLaunchKernelGGL(k_few_join<__bf16>, blocks, dim3(1024), 0, st, a, p.groups, p.vt * 32, static_cast<__bf16 *>(d.dw), static_cast<__bf16 *>(d.db));
  else
    hipLaunchKernelGGL(k_few_join<_Float16>, blocks, dim3(1024), 0, st, a, p.groups, p.vt * 32, static_cast<_Float16 *>(d.dw), static_cast<_Float16 *>(d.db));
  return R3D_OK;
}

}  // namespace r3d

// Rotary positions with several axes (gfx950): x y z of a point, scan / row / column of a pixel.
//
// Pair i of axis a (number j of the axis' s_a pairs) is turned by  angle = pos[t][a] * base^(-j / s_a):
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin;   the backward pass is the same kernel with -sin.
// The angle is taken in turns and in double (pos * turns per unit, minus the whole turns): single precision would lose
// 1e-3 of a radian at position 1e4.  What is left is turned with single-precision sin / cos, 32-bit products, one rounding.
//
// Bound by HBM: one read and one write of q and k.  A workgroup stages a few tokens' rows in LDS with the widest loads the
// alignment allows, whatever the number of pairs is -- pairs (i, i + R) or (2i, 2i + 1) of an odd R have no alignment of
// their own --, a thread owns (token, pair) and keeps its sine and cosine over all heads, and the rows leave as they came.
// 120 000 tokens x (8 + 2) heads x 64 bf16: 68 us, 4.5 TB/s, where a copy reaches 4.7; as slices of one projection or with
// the heads in front of the tokens 70 (one element a time: 207).  400 heads a token, in parts that fit LDS: 3.2 TB/s.
#include "r3d_host.hpp"

#include <cmath>

namespace {
using namespace r3d;

constexpr int kMaxPairs = 256, kRotThreads = 256, kRotLds = 24 * 1024;

struct RotArgs {
  const void *x[2];
  void *y[2];
  int64_t token_stride[2], head_stride[2];      // of x, in elements; y is dense
  int32_t heads[2];
  int64_t tokens;
  int32_t dim, pairs, tile, half;
  int32_t flat_in[2], flat_out, unit_in[2], unit_out[2];      // flat: a tile is one piece of memory; unit: bytes of a load / store
  int32_t heads_per_group;
  float sign;
  const void *pos;
  int64_t pos_token_stride, pos_axis_stride;
  int32_t pos_type;
  double turns[kMaxPairs];      // turns per unit of position
  uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ double position(const RotArgs &a, int64_t t, int axis) {
  const int64_t i = t * a.pos_token_stride + axis * a.pos_axis_stride;
  switch (a.pos_type) {
    case R3D_T_I32: return (double)static_cast<const int32_t *>(a.pos)[i];
    case R3D_T_I64: return (double)static_cast<const int64_t *>(a.pos)[i];
    case R3D_T_F32: return (double)static_cast<const float *>(a.pos)[i];
    default: return static_cast<const double *>(a.pos)[i];
  }
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight loads of a thread are on their way before the first is put down: one at a time, the latencies add up (92 us against
// 83 for 120 000 tokens x 10 heads x 64 bf16, with 40 KB of LDS).
template <class U>
__device__ __forceinline__ void copy_flat(char *to, const char *from, int bytes) {
  const int n = bytes / (int)sizeof(U);
  for (int i0 = threadIdx.x; i0 < n; i0 += 8 * kRotThreads) {
    U v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i0 + k * kRotThreads < n) v[k] = reinterpret_cast<const U *>(from)[i0 + k * kRotThreads];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i0 + k * kRotThreads < n) reinterpret_cast<U *>(to)[i0 + k * kRotThreads] = v[k];
  }
  // what is left behind the last whole one (rows are even numbers of elements)
  const int done = n * (int)sizeof(U), left = (bytes - done) / 2;
  if ((int)threadIdx.x < left) reinterpret_cast<uint16_t *>(to + done)[threadIdx.x] = reinterpret_cast<const uint16_t *>(from + done)[threadIdx.x];
}

// Rows of `bytes` that lie apart in memory, `heads` to a token, and one after the other in LDS: a slice of a wider projection,
// heads in front of tokens, or a part of the heads.
template <class U, bool kIn>
__device__ __forceinline__ void copy_rows(char *lds, char *mem, int rows, int heads, int bytes, int64_t token_stride, int64_t head_stride) {
  const unsigned per = (unsigned)bytes / (unsigned)sizeof(U), n = rows * per;
  for (unsigned i0 = threadIdx.x; i0 < n; i0 += 8 * kRotThreads) {
    U v[8];
    char *at[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned i = i0 + k * kRotThreads, r = i / per, t = heads == 1 ? r : r / (unsigned)heads;
      at[k] = mem + t * token_stride + (r - t * heads) * head_stride + (i - r * per) * sizeof(U);
      if (i < n) v[k] = kIn ? *reinterpret_cast<const U *>(at[k]) : reinterpret_cast<const U *>(lds)[i];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned i = i0 + k * kRotThreads;
      if (i < n) *(kIn ? reinterpret_cast<U *>(lds) + i : reinterpret_cast<U *>(at[k])) = v[k];
    }
  }
}

template <class F>
__device__ __forceinline__ void with_unit(int unit, F &&f) {
  if (unit == 16) f(u32x4{});
  else if (unit == 8) f(u32x2{});
  else if (unit == 4) f(uint32_t{});
  else f(uint16_t{});
}

template <class T>
__global__ __launch_bounds__(kRotThreads) void k_rotary(RotArgs a) {
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  T *s = reinterpret_cast<T *>(s_raw);
  const int64_t t0 = (int64_t)blockIdx.x * a.tile;
  const int n = (int)min((int64_t)a.tile, a.tokens - t0);
  // the heads of this workgroup: [h0, h1) of q's and k's in one line
  const int all = a.heads[0] + a.heads[1];
  const int h0 = blockIdx.y * a.heads_per_group, h1 = min(h0 + a.heads_per_group, all);
  int at[2], from[2], count[2];
  {
    from[0] = min(h0, a.heads[0]);
    count[0] = min(h1, a.heads[0]) - from[0];
    from[1] = max(h0 - a.heads[0], 0);
    count[1] = max(h1 - a.heads[0], 0) - from[1];
    at[0] = 0;
    at[1] = (a.tile * count[0] * a.dim * (int)sizeof(T) + 15) / 16 * 16 / (int)sizeof(T);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if (count[w] <= 0) continue;
    char *to = reinterpret_cast<char *>(s + at[w]);
    const T *x = static_cast<const T *>(a.x[w]) + t0 * a.token_stride[w] + from[w] * a.head_stride[w];
    const bool line = a.head_stride[w] == a.dim;      // a token's heads in one piece
    const int row = (line ? count[w] : 1) * a.dim * (int)sizeof(T), heads = line ? 1 : count[w];
    with_unit(a.unit_in[w], [&](auto u) {
      typedef decltype(u) U;
      if (a.flat_in[w]) copy_flat<U>(to, reinterpret_cast<const char *>(x), n * row);
      else copy_rows<U, true>(to, const_cast<char *>(reinterpret_cast<const char *>(x)), n * heads, heads, row, a.token_stride[w] * (int)sizeof(T), a.head_stride[w] * (int)sizeof(T));
    });
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * a.pairs; i += kRotThreads) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    double turn = position(a, t0 + t, a.axis[p]) * a.turns[p];
    turn -= rint(turn);
    float sn, cs;
    sincospif(2.0f * (float)turn, &sn, &cs);
    sn *= a.sign;
    const int i1 = a.half ? p : 2 * p, i2 = a.half ? p + a.pairs : 2 * p + 1;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      T *row = s + at[w] + t * count[w] * a.dim;
      for (int h = 0; h < count[w]; ++h, row += a.dim) {
        const float x1 = (float)row[i1], x2 = (float)row[i2];
        row[i1] = (T)__builtin_fmaf(x1, cs, -x2 * sn);
        row[i2] = (T)__builtin_fmaf(x2, cs, x1 * sn);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if (count[w] <= 0) continue;
    char *lds = reinterpret_cast<char *>(s + at[w]);
    char *y = reinterpret_cast<char *>(static_cast<T *>(a.y[w]) + (t0 * a.heads[w] + from[w]) * a.dim);
    const int row = count[w] * a.dim * (int)sizeof(T);
    with_unit(a.unit_out[w], [&](auto u) {
      typedef decltype(u) U;
      if (a.flat_out) copy_flat<U>(y, lds, n * row);
      else copy_rows<U, false>(lds, y, n, 1, row, (int64_t)a.heads[w] * a.dim * (int)sizeof(T), 0);
    });
  }
}
}  // namespace

extern "C" int r3d_rotary(const r3d_rotary_t *d, void *stream) {
  if (!d) return fail(R3D_E_ARG, "rotary: null descriptor");
  if (d->tokens < 0 || d->tokens > (1ll << 40) || d->dim <= 0 || d->dim > 4096 || d->axes <= 0 || d->axes > R3D_ROTARY_MAX_AXES ||
      d->heads[0] < 0 || d->heads[1] < 0 || d->heads[0] > 65536 || d->heads[1] > 65536 || d->heads[0] + d->heads[1] == 0)
    return fail(R3D_E_ARG, "rotary: bad size");
  const int size = d->type == R3D_T_F32 ? 4 : d->type == R3D_T_BF16 || d->type == R3D_T_F16 ? 2 : 0;
  if (!size) return fail(R3D_E_ARG, "rotary: type");
  if (d->pos_type != R3D_T_I32 && d->pos_type != R3D_T_I64 && d->pos_type != R3D_T_F32 && d->pos_type != R3D_T_F64)
    return fail(R3D_E_ARG, "rotary: type of the positions");
  if (!(d->base > 0.0) || std::isinf(d->base)) return fail(R3D_E_ARG, "rotary: base must be positive and finite");
  RotArgs a{};
  const double octaves = std::log2(d->base);
  for (int x = 0; x < d->axes; ++x) {
    const int s = d->sections[x];
    if (s < 0 || a.pairs + s > kMaxPairs) return fail(R3D_E_ARG, "rotary: sections (at most 256 pairs)");
    for (int j = 0; j < s; ++j) {
      a.turns[a.pairs] = std::exp2(-(double)j / s * octaves) / (2.0 * M_PI);
      a.axis[a.pairs++] = (uint8_t)x;
    }
  }
  if (2 * a.pairs > d->dim) return fail(R3D_E_ARG, "rotary: more pairs than the head has");
  if (d->tokens == 0) return R3D_OK;
  if (!d->pos) return fail(R3D_E_ARG, "rotary: null positions");
  if (!aligned(d->pos, d->pos_type == R3D_T_I32 || d->pos_type == R3D_T_F32 ? 4 : 8)) return fail(R3D_E_ARG, "rotary: positions not aligned to their type");
  a.tokens = d->tokens;
  a.dim = d->dim;
  a.half = d->interleaved ? 0 : 1;
  a.sign = d->backward ? -1.0f : 1.0f;
  a.pos = d->pos;
  a.pos_type = d->pos_type;
  a.pos_token_stride = d->pos_token_stride;
  a.pos_axis_stride = d->pos_axis_stride;
  const int all = d->heads[0] + d->heads[1];
  const int64_t head_bytes = (int64_t)d->dim * size;
  // all heads of a token in LDS if they fit (32 bytes of slack for q's and k's alignment), else groups of heads
  a.heads_per_group = all * head_bytes <= kRotLds ? all : (int)(kRotLds / head_bytes);
  const int groups = (all + a.heads_per_group - 1) / a.heads_per_group;
  int64_t tile = kRotLds / (a.heads_per_group * head_bytes);
  if (tile > 256) tile = 256;
  // few tokens: smaller tiles, so that every CU gets some (four workgroups each)
  const int64_t spread = (d->tokens + 1023) / 1024;
  if (tile > spread) tile = spread;
  if (tile >= 4) tile = tile / 4 * 4;
  a.tile = (int)tile;
  for (int w = 0; w < 2; ++w) {
    a.heads[w] = d->heads[w];
    if (!d->heads[w]) continue;
    if (!d->x[w] || !d->y[w]) return fail(R3D_E_ARG, "rotary: null tensor");
    if (d->x[w] == d->y[w]) return fail(R3D_E_ARG, "rotary: an output is its input");
    a.x[w] = d->x[w];
    a.y[w] = d->y[w];
    a.token_stride[w] = d->token_stride[w];
    a.head_stride[w] = d->head_stride[w];
    // the widest load that every row begins on: of a whole tile where it is one piece of memory, else of a token or a head
    const uint64_t ts = (uint64_t)d->token_stride[w] * size, hs = (uint64_t)d->head_stride[w] * size;
    const bool line = d->heads[w] == 1 || d->head_stride[w] == d->dim;
    a.head_stride[w] = line ? d->dim : d->head_stride[w];
    a.flat_in[w] = groups == 1 && line && (d->token_stride[w] == (int64_t)d->heads[w] * d->dim || d->tokens == 1);
    const uint64_t whole = (uint64_t)tile * d->heads[w] * head_bytes, token = (uint64_t)d->heads[w] * head_bytes;
    auto unit = [](uint64_t bits) { return bits & 15 ? (int)(bits & (0 - bits)) : 16; };
    a.unit_in[w] = unit(reinterpret_cast<uintptr_t>(d->x[w]) | (a.flat_in[w] ? whole : ts | (line && groups == 1 ? token : (line ? 0 : hs) | (uint64_t)head_bytes)));
    a.unit_out[w] = unit(reinterpret_cast<uintptr_t>(d->y[w]) | (groups == 1 ? whole : (uint64_t)head_bytes));
    if (a.unit_in[w] < size || a.unit_out[w] < size) return fail(R3D_E_ARG, "rotary: a tensor is not aligned to its elements");
  }
  a.flat_out = groups == 1;
  if ((d->tokens + tile - 1) / tile > INT32_MAX || groups > 65535) return fail(R3D_E_ARG, "rotary: too many tokens or heads");
  const size_t lds = (size_t)(a.tile * a.heads_per_group * head_bytes) + 32;
  const dim3 grid((unsigned)((d->tokens + tile - 1) / tile), groups);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->type == R3D_T_F32) hipLaunchKernelGGL(k_rotary<float>, grid, dim3(kRotThreads), lds, st, a);
  else if (d->type == R3D_T_BF16) hipLaunchKernelGGL(k_rotary<__bf16>, grid, dim3(kRotThreads), lds, st, a);
  else hipLaunchKernelGGL(k_rotary<_Float16>, grid, dim3(kRotThreads), lds, st, a);
  R3D_LAUNCHED("k_rotary");
  return R3D_OK;
}

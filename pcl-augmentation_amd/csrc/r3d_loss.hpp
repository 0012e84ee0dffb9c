// What the files of the linear head's cross entropy share (r3d_loss.hip: any sizes; r3d_loss_few.hip: few classes; r3d_loss_narrow.hip:
// the gradients for few features).
#pragma once

#include "r3d_mfma.hpp"

#include "../../include/real3daug_hip.h"

namespace r3d {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// A point's softmax, in units of log 2: logits t = (x w + b) log2 e, their maximum `top` and the sum of the parts 2^(t - top).  Maximum
// and sum stay two numbers up to the loss and the gradients: the maximum plus the logarithm of the sum, in one number of 24 bits, costs
// a head that is sure of itself what it is sure of.  For the same reason every pass makes the same bits of a logit.  3000 points x
// 400 classes x 64, fp32, relative to 64 bits: at a mean loss of 0.07 dx is off by 1.9e-6 (4.3e-6 in one number), db by 7.3e-7
// (2.0e-6); at a mean loss of 6e-4 dW by 4.1e-6 (2.4e-4).
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.0f : top; }      // (every class masked: the sum is 0)
__device__ __forceinline__ float logit2(float xw, float bias2) { return __builtin_fmaf(xw, kLog2e, bias2); }
__device__ __forceinline__ float part_of(float t, float base) { return __builtin_amdgcn_exp2f(t - base); }
__device__ __forceinline__ float point_loss(float top, float sum, float hit) { return (__builtin_amdgcn_logf(sum) + (top - hit)) * kLn2; }

struct Counted {      // the points that count, on the device
  int32_t n;          // how many
  float share;        // 1 / n for a mean (0 where none counts), 1 else
  int32_t ticket;     // workgroups that have left their part of a sum
  int32_t pad;
};

__device__ __forceinline__ __bf16 toward_zero(float v) {      // (rounding up the largest floats would give infinities)
  return __builtin_bit_cast(__bf16, (unsigned short)(__builtin_bit_cast(unsigned, v) >> 16));
}
// The three planes of 8 bits of a float: v = h + m + l to 2^-25.
__device__ __forceinline__ void split3(float v, __bf16 &h, __bf16 &m, __bf16 &l) {
  h = toward_zero(v);
  const float r = v - (float)h;
  m = toward_zero(r);
  l = (__bf16)(r - (float)m);
}

// Few classes: whether a head is that, the bytes of R3D_CE_BYTES_*, the two passes.
bool few_takes(const r3d_linear_ce_t &d);
size_t few_bytes(const r3d_linear_ce_t &d, int32_t which);
int few_forward(const r3d_linear_ce_t &d, void *workspace, hipStream_t st);
int few_backward(const r3d_linear_ce_t &d, void *workspace, hipStream_t st);

// Few features (64 or 128 with the padding): the statistics of the points, dx (kept rows: points), dW and db (kept rows: classes).
enum class Narrow { Lse, Dx, Dw };
struct NarrowArgs {
  Operand kept, met;
  int64_t v;
  const float *bias2, *base, *sum, *weight;      // base, sum: a point's maximum and the sum of its parts
  const int32_t *tgt;
  const Counted *counted;
  float held;                            // 2^15 for float16
  int32_t each;                          // weights differ from point to point (else all are 1)
  int32_t tiles, splits;                 // of narrow_rows() kept rows; parts of the met ones
  float *out;                            // [splits][rows][dp] 32-bit sums, or
  int64_t split_stride;
  float *part_m, *part_l, *hit;          // statistics: [splits][split_stride], and the target's logit
  void *final_out;                       // the result: rows of d, times scale * unheld
  int64_t d;
  const float *scale;
  float unheld;
  int32_t vector_out;
  float *sums;                           // [splits][sums_stride] db, or null
  int64_t sums_stride;
};
int narrow_rows(Narrow what, int planes, int dp);
void narrow(Narrow what, const NarrowArgs &a, int type, int dp, hipStream_t st);

}  // namespace r3d

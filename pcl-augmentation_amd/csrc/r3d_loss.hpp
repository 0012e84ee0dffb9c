// What the files of the linear head's cross entropy share (r3d_loss.hip: any sizes; r3d_loss_few.hip: few classes; r3d_loss_narrow.hip:
// the gradients for few features).
#pragma once

#include "r3d_mfma.hpp"

#include "../../include/real3daug_hip.h"

namespace r3d {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

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
  const float *bias2, *lse2, *weight;
  const int32_t *tgt;
  const Counted *counted;
  float held;                            // 2^15 for float16
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

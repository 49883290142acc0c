// What the kernels of the masked attention share: the sequences, the masks and the capped scores.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "layer_ops.h"

namespace laya {

// A row's weights are 2^(s - m) against a reference m that moves only when a score passes it by more than
// 2^(kGrow + up), to up below that score. fp16's smallest number is 2^-24, so there up is 7: a weight below
// 2^-32 of the row's largest is lost, and none passes 2^15. bf16 has fp32's range: up is 0.
constexpr float kGrow = 8.f, kUpF16 = 7.f;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {  // 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp_fast(float x) {  // of infinity: 0
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows of sequence b in q and in k / v. Offsets outside the arrays, or that run backwards, are cut to
// the arrays, so nothing outside them is ever touched.
struct Sequence {
  int q0, lq, k0, lk, prefix;
};
__device__ __forceinline__ Sequence sequence(const VarlenArgs& a, int b) {
  Sequence s;
  s.q0 = min(max(a.cu_q[b], 0), a.rows_q);
  s.lq = min(max(a.cu_q[b + 1], s.q0), a.rows_q) - s.q0;
  s.k0 = min(max(a.cu_k[b], 0), a.rows_k);
  s.lk = min(max(a.cu_k[b + 1], s.k0), a.rows_k) - s.k0;
  s.prefix = a.prefix ? min(max(a.prefix[b], 0), s.lk) : 0;
  return s;
}

// Bits below n of 32.
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// Keys kg .. kg + 31 that a query at key position p sees through its window or the prefix.
__device__ __forceinline__ uint32_t window_bits(const VarlenArgs& a, const Sequence& s, int p, int kg) {
  const uint32_t w = bits_below(p + a.right + 1 - kg) & ~bits_below(p - a.left - kg);
  return (w | bits_below(s.prefix - kg)) & bits_below(s.lk - kg);
}

// tanh where |u| < kTanhSmall: the odd Taylor polynomial to u^7, off by at most 62/2835 u^8 = 3.4e-7 of
// the value; no special-function instruction.
constexpr float kTanhSmall = 0.25f;
__device__ __forceinline__ float tanh_small(float u) {
  const float z = u * u;
  return u * fmaf(z, fmaf(z, fmaf(z, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
}
// tanh u = 1 - 2 / (1 + e^(2u)) everywhere, to about 2e-7 absolutely.
__device__ __forceinline__ float tanh_any(float u) {
  return fmaf(-2.f, rcp_fast(1.f + exp2_fast(u * (2.f * kLog2e))), 1.f);
}
// v < limit ? below : other, both of which are computed (NaN takes the other): no branch.
__device__ __forceinline__ float pick_below(float v, float limit, float below, float other) {
  float r;
  asm("{\n\t.reg .pred p;\n\tsetp.lt.f32 p, %1, %2;\n\tselp.f32 %0, %3, %4, p;\n\t}"
      : "=f"(r)
      : "f"(v), "f"(limit), "f"(below), "f"(other));
  return r;
}

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, int type) {
  if (type == DT_BF16) return pack_bf16x2(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace laya

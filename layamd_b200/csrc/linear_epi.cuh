// Epilogue of the matrix product with scales, bias, activation and residual: shared by its kernels.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "layer_ops.h"

namespace laya {

// Activations in place on 8 values; the switch is uniform over the grid.
__device__ __forceinline__ void act8(float (&v)[8], int act) {
  if (act == LIN_RELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];  // NaN stays NaN
  } else if (act == LIN_GELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = gelu_as(v[j]);
  } else if (act == LIN_SILU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fdividef(v[j], 1.f + __expf(-v[j]));
  }
}

__device__ __forceinline__ uint32_t pack16_of(float lo, float hi, int type) {
  if (type == DT_BF16) return pack_bf16x2(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack16(uint32_t v, int type) {
  if (type == DT_BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// 8 consecutive columns of one row, 16 or 32 bytes (OW: the output's element size), as they lie in
// memory.
template <int OW>
struct Cols8 {
  uint4 u[OW / 2];
};

// resid[row][col .. col + 7]; zero outside M x N. Columns past N are never read.
template <int OW>
__device__ __forceinline__ void load_resid(Cols8<OW>& r, const LinearArgs& a, int row, int col) {
#pragma unroll
  for (int i = 0; i < OW / 2; ++i) r.u[i] = make_uint4(0u, 0u, 0u, 0u);
  if (!a.resid || row >= a.M || col >= a.N) return;
  const char* p = static_cast<const char*>(a.resid) + ((long long)row * a.ldr + col) * OW;
  if (a.vec_out && col + 8 <= a.N) {
#pragma unroll
    for (int i = 0; i < OW / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
    return;
  }
  uint32_t* d = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (col + j >= a.N) break;
    if constexpr (OW == 4)
      d[j] = reinterpret_cast<const uint32_t*>(p)[j];
    else
      d[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[j]) << (j & 1) * 16;
  }
}

// The scales and biases of 8 consecutive columns.
struct ColParams {
  float scale[8], bias[8];
};
__device__ __forceinline__ void load_cols(ColParams& c, const LinearArgs& a, int col) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = col + j < a.N;
    c.scale[j] = a.w_scale && in ? __ldg(a.w_scale + col + j) : 1.f;
    c.bias[j] = a.bias && in ? __ldg(a.bias + col + j) : 0.f;
  }
}

// v: the sums of row `row`, columns col .. col + 7; sa: the row's scale.
template <int OW>
__device__ __forceinline__ void emit8(float (&v)[8], const LinearArgs& a, const ColParams& c, float sa,
                                      const Cols8<OW>& r, int row, int col) {
  if (row >= a.M || col >= a.N) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = fmaf(v[j], sa * c.scale[j], c.bias[j]);
  act8(v, a.act);
  const uint32_t* d = reinterpret_cast<const uint32_t*>(&r);
  char* p = static_cast<char*>(a.out) + ((long long)row * a.ldo + col) * OW;
  if constexpr (OW == 4) {
    if (a.resid) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += __uint_as_float(d[j]);
    }
    if (a.vec_out && col + 8 <= a.N) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < a.N) reinterpret_cast<float*>(p)[j] = v[j];
  } else {
    if (a.resid) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack16(d[j], a.out_type);
        v[2 * j] += f.x;
        v[2 * j + 1] += f.y;
      }
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pack16_of(v[2 * j], v[2 * j + 1], a.out_type);
    if (a.vec_out && col + 8 <= a.N) {
      *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < a.N) reinterpret_cast<uint16_t*>(p)[j] = static_cast<uint16_t>(o[j / 2] >> (j & 1) * 16);
  }
}

}  // namespace laya

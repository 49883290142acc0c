// Matrix product for few rows (M <= 16: single tokens, a few option rows): the weight is read once and
// everything else is small, so the bound is HBM. No shared memory on the way in: a warp takes 8 (or
// 16) rows of W and a slice of K, and each thread loads 16 consecutive bytes of its W row straight into
// the registers of an mma.sync m16n8k16 operand. The instruction wants each thread's K values 2t, 2t+1,
// 2t+8, 2t+9 of a step; since a sum over K may run in any order, thread t's loaded values simply take
// those places, in A alike. The 8 warps of a block take every 8th K step of the same columns and are
// summed in warp order through shared memory. 8-bit operands are widened to fp16 in registers (exact),
// so products and sums are the same fp32 ones.
#include <cuda_fp8.h>

#include "linear_epi.cuh"

namespace laya {
namespace {

constexpr int kWarps = 8;
constexpr int kUnroll = 4;  // K steps whose loads are in flight together

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1, bool bf) {
  if (bf)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from element k on; elements past K are zero and not read. ES: element size.
template <int ES>
__device__ __forceinline__ uint4 load16(const char* row, int k, int K, bool on) {
  if (!on || k >= K) return make_uint4(0u, 0u, 0u, 0u);
  const char* p = row + (size_t)k * ES;
  if (k + 16 / ES <= K) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16 / ES; ++i)
    if (k + i < K) {
      if constexpr (ES == 2)
        w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (i & 1) * 16;
      else
        w[i / 4] |= static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(p)[i]) << (i & 3) * 8;
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Two e4m3 values as two fp16 ones.
__device__ __forceinline__ uint32_t widen(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xffffu), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One loaded step: 16-bit operands make 2 products of depth 16, 8-bit ones 4.
template <int ES>
__device__ __forceinline__ void step(float (&c)[4], const uint4& a_lo, const uint4& a_hi, const uint4& w, bool bf) {
  if constexpr (ES == 2) {
    mma16(c, a_lo.x, a_hi.x, a_lo.y, a_hi.y, w.x, w.y, bf);
    mma16(c, a_lo.z, a_hi.z, a_lo.w, a_hi.w, w.z, w.w, bf);
  } else {
    const uint32_t l[4] = {a_lo.x, a_lo.y, a_lo.z, a_lo.w}, h[4] = {a_hi.x, a_hi.y, a_hi.z, a_hi.w};
    const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mma16(c, widen(l[i]), widen(h[i]), widen(l[i] >> 16), widen(h[i] >> 16), widen(b[i]), widen(b[i] >> 16), false);
  }
}

// NC: groups of 8 columns per warp.
template <int ES, int OW, int NC>
__global__ void __launch_bounds__(32 * kWarps) linear_few_kernel(const LinearArgs a) {
  constexpr int kStep = 64 / ES;  // K values of one step (16 bytes x 4 threads)
  __shared__ float part[kWarps][16][8 * NC];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 8 * NC;
  const bool bf = a.ab_type == DT_BF16;
  const bool lo_on = g < a.M, hi_on = g + 8 < a.M;
  const char* a_lo = static_cast<const char*>(a.A) + (long long)(lo_on ? g : 0) * a.lda * ES;
  const char* a_hi = static_cast<const char*>(a.A) + (long long)(hi_on ? g + 8 : 0) * a.lda * ES;
  const char* w_row[NC];
  bool w_on[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    w_on[i] = n0 + 8 * i + g < a.N;
    w_row[i] = static_cast<const char*>(a.W) + (long long)(w_on[i] ? n0 + 8 * i + g : 0) * a.ldw * ES;
  }
  float c[NC][4];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 0.f;

  for (int k0 = warp * kStep; k0 < a.K; k0 += kWarps * kStep * kUnroll) {
    uint4 w[kUnroll][NC], l[kUnroll], h[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = k0 + u * kWarps * kStep + t * (16 / ES);
#pragma unroll
      for (int i = 0; i < NC; ++i) w[u][i] = load16<ES>(w_row[i], k, a.K, w_on[i]);
      l[u] = load16<ES>(a_lo, k, a.K, lo_on);
      h[u] = load16<ES>(a_hi, k, a.K, hi_on);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < NC; ++i) step<ES>(c[i], l[u], h[u], w[u][i], bf);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    part[warp][g][8 * i + 2 * t] = c[i][0];
    part[warp][g][8 * i + 2 * t + 1] = c[i][1];
    part[warp][g + 8][8 * i + 2 * t] = c[i][2];
    part[warp][g + 8][8 * i + 2 * t + 1] = c[i][3];
  }
  __syncthreads();
  if (threadIdx.x >= 16 * NC) return;
  const int row = threadIdx.x / NC, col = threadIdx.x % NC * 8;
  if (row >= a.M) return;
  ColParams cp;
  load_cols(cp, a, n0 + col);
  Cols8<OW> r;
  load_resid<OW>(r, a, row, n0 + col);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = part[0][row][col + j];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v[j] += part[w][row][col + j];
  }
  emit8<OW>(v, a, cp, a.a_scale ? a.a_scale[row] : 1.f, r, row, n0 + col);
}

template <int ES, int OW>
cudaError_t launch(const LinearArgs& a, int num_sms, cudaStream_t st) {
  // 16 columns per warp once that still gives every SM two blocks: A is then read half as often.
  if (a.N >= 16 * 2 * num_sms)
    return launch_pdl(linear_few_kernel<ES, OW, 2>, dim3((a.N + 15) / 16), dim3(32 * kWarps), 0, st, a);
  return launch_pdl(linear_few_kernel<ES, OW, 1>, dim3((a.N + 7) / 8), dim3(32 * kWarps), 0, st, a);
}

}  // namespace

cudaError_t linear_few_launch(const LinearArgs& a, int num_sms, cudaStream_t st) {
  if (a.M > kLinearFewRows) return cudaErrorInvalidValue;
  if (a.ab_type == DT_E4M3)
    return a.out_type == DT_F32 ? launch<1, 4>(a, num_sms, st) : launch<1, 2>(a, num_sms, st);
  return a.out_type == DT_F32 ? launch<2, 4>(a, num_sms, st) : launch<2, 2>(a, num_sms, st);
}

}  // namespace laya

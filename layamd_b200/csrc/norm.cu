// Norm of a residual sum: h = x + r, y = (h - c mean(h)) / sqrt(mean((h - c mean(h))^2) + eps) * w + b
// with c = 0 (root-mean-square norm) or 1 (LayerNorm), written in 16 or 32 bits or as e4m3 values with
// one fp32 scale per row (the largest |y| of the row maps to 448, e4m3's largest value).
//
// Bound by HBM: x, r and the stored sum are touched once, y once; a row stays in registers between its
// statistics and its output. T threads own a row (T = 32, 128 or 512), each NV pieces of 8 elements, so
// every 16-bit access is one 16-byte transaction per thread and every fp32 one two, at any alignment of
// the rows. Statistics are two-pass in fp32 (the mean first, then the squares of the differences), as the
// engine's LayerNorm computes them; h is not rounded before them, so the stored sum's rounding never
// reaches y. A row whose squares leave fp32's range is summed again, scaled by a power of two.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "layer_ops.h"

namespace laya {
namespace {

// Piece i of thread t: the row's elements 8 (i T + t) .. + 7, as they lie in memory (W: their size).
template <int W>
struct Raw8 {
  uint32_t d[2 * W];
};

// n + 4 words `s` (low word first) shifted down by o bytes (0 <= o < 16): n words of a run of bytes that
// starts o bytes into the first 16.
template <int N>
__device__ __forceinline__ void shift_down(const uint32_t (&s)[N + 4], uint32_t o, uint32_t (&d)[N]) {
  uint32_t t[N + 2];
#pragma unroll
  for (int i = 0; i < N + 2; ++i) t[i] = o & 8 ? s[i + 2] : s[i];
#pragma unroll
  for (int i = 0; i < N + 1; ++i) t[i] = o & 4 ? t[i + 1] : t[i];
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = __funnelshift_r(t[i], t[i + 1], (o & 3) * 8);
}

// The 16 bytes at p (16-byte aligned) into w; of a chunk that is not all inside [lo, hi), the elements
// of W bytes that are, and zero for the rest.
template <int W, bool ONCE>
__device__ __forceinline__ void load_chunk(uint32_t* w, const char* p, const char* lo, const char* hi) {
  if (p >= lo && p + 16 <= hi) {
    const uint4* c = reinterpret_cast<const uint4*>(p);
    const uint4 v = ONCE ? __ldcs(c) : __ldg(c);  // rows are read once: evict-first
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = 0u;
#pragma unroll
  for (int i = 0; i < 16 / W; ++i) {
    const char* q = p + i * W;
    if (q < lo || q >= hi) continue;
    if constexpr (W == 4)
      w[i] = *reinterpret_cast<const uint32_t*>(q);
    else
      w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(q)) << (i & 1) * 16;
  }
}

// One piece of a row. A row may start anywhere (a row of odd length in dense storage): memory is still
// read in aligned 16-byte chunks, each by one thread, and a thread takes the first chunk of its right
// neighbour (the warp's last thread loads it) to shift its own bytes into place. Whole warps call this.
// ALIGNED: every row starts on 16 bytes.
template <int W, int T, bool ALIGNED, bool ONCE>
__device__ __forceinline__ void load8(Raw8<W>& r, const void* row, int piece, int t, int D) {
  const char* lo = static_cast<const char*>(row);
  const char* p = lo + (size_t)(piece * T + t) * 8 * W;
  if (ALIGNED && (piece * T + t) * 8 + 8 <= D) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const uint4* c = reinterpret_cast<const uint4*>(p) + i;
      const uint4 v = ONCE ? __ldcs(c) : __ldg(c);
      r.d[4 * i] = v.x; r.d[4 * i + 1] = v.y; r.d[4 * i + 2] = v.z; r.d[4 * i + 3] = v.w;
    }
    return;
  }
  const char* hi = lo + (size_t)D * W;
  const uint32_t o = ALIGNED ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
  if (o == 0) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) load_chunk<W, ONCE>(r.d + 4 * i, p + 16 * i, lo, hi);
    return;
  }
  uint32_t s[2 * W + 4];
#pragma unroll
  for (int i = 0; i < W / 2; ++i) load_chunk<W, ONCE>(s + 4 * i, p - o + 16 * i, lo, hi);
  uint32_t last[4] = {0u, 0u, 0u, 0u};
  if ((t & 31) == 31) load_chunk<W, ONCE>(last, p - o + 8 * W, lo, hi);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t right = __shfl_down_sync(0xffffffffu, s[i], 1);
    s[2 * W + i] = (t & 31) == 31 ? last[i] : right;
  }
  shift_down<2 * W>(s, o, r.d);
}

template <int W>
__device__ __forceinline__ float value(const Raw8<W>& r, int j, int type) {
  if constexpr (W == 4) {
    return __uint_as_float(r.d[j]);
  } else {
    const uint32_t v = j & 1 ? r.d[j / 2] >> 16 : r.d[j / 2] & 0xffffu;
    return type == DT_BF16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(v)));
  }
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int type) {
  if (type == DT_BF16) return pack_bf16x2(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

template <int C>
__device__ __forceinline__ void put_chunk(const uint32_t* w, char* p) {
  if constexpr (C == 16)
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  else
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
}
// C bytes (a multiple of 4) at p, aligned to C: as one store where they are all inside [lo, hi), else
// the elements of W bytes that are.
template <int W, int C>
__device__ __forceinline__ void store_chunk(const uint32_t* w, char* p, const char* lo, const char* hi) {
  if (p >= lo && p + C <= hi) {
    put_chunk<C>(w, p);
    return;
  }
#pragma unroll
  for (int i = 0; i < C / W; ++i) {
    char* q = p + i * W;
    if (q < lo || q >= hi) continue;
    const uint32_t v = w[i * W / 4] >> (i * W % 4) * 8;
    if constexpr (W == 4)
      *reinterpret_cast<uint32_t*>(q) = v;
    else if constexpr (W == 2)
      *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(v);
    else
      *reinterpret_cast<uint8_t*>(q) = static_cast<uint8_t>(v);
  }
}

// The counterpart of load8 for 8 elements of W bytes, in chunks of C bytes (16, or 8 for e4m3): a
// thread writes the aligned chunks that end inside its bytes, the first of them with the last bytes
// of its left neighbour; the warp's first and last thread write their open ends by element.
template <int W, int T, bool ALIGNED>
__device__ __forceinline__ void store_words(const uint32_t (&d)[2 * W], void* row, int piece, int t, int D) {
  constexpr int C = W == 1 ? 8 : 16, N = 2 * W, CW = C / 4;
  char* row_lo = static_cast<char*>(row);
  char* p = row_lo + (size_t)(piece * T + t) * 8 * W;
  if (ALIGNED && (piece * T + t) * 8 + 8 <= D) {
#pragma unroll
    for (int i = 0; i < N / CW; ++i) put_chunk<C>(d + CW * i, p + C * i);
    return;
  }
  const char* hi = row_lo + (size_t)D * W;
  const uint32_t o = ALIGNED ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row_lo) & (C - 1));
  if (o == 0) {
#pragma unroll
    for (int i = 0; i < N / CW; ++i) store_chunk<W, C>(d + CW * i, p + C * i, row_lo, hi);
    return;
  }
  // s: the neighbour's last C bytes, then this thread's: the chunk at p - o starts C - o bytes into it
  uint32_t s[N + 4];
#pragma unroll
  for (int i = 0; i < CW; ++i) s[i] = __shfl_up_sync(0xffffffffu, d[N - CW + i], 1);
#pragma unroll
  for (int i = 0; i < N; ++i) s[CW + i] = d[i];
#pragma unroll
  for (int i = CW + N; i < N + 4; ++i) s[i] = 0u;
  uint32_t m[N];
  shift_down<N>(s, C - o, m);
  const char* lo = (t & 31) == 0 ? p : row_lo;  // the first thread's left neighbour is another warp's
#pragma unroll
  for (int i = 0; i < N / CW; ++i) store_chunk<W, C>(m + CW * i, p - o + C * i, lo, hi);
  if ((t & 31) == 31) {
    // the last o bytes, which no thread to the right takes along
    uint32_t e[CW + 4], n[CW];
#pragma unroll
    for (int i = 0; i < CW + 4; ++i) e[i] = i < CW ? d[N - CW + i] : 0u;
    shift_down<CW>(e, C - o, n);
    char* q = p - o + 8 * W;
    store_chunk<W, C>(n, q, row_lo, q + o < hi ? q + o : hi);
  }
}

template <int T, bool ALIGNED>
__device__ __forceinline__ void store8(const float (&v)[8], void* row, int type, int piece, int t, int D) {
  if (type == DT_F32) {
    uint32_t d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = __float_as_uint(v[j]);
    store_words<4, T, ALIGNED>(d, row, piece, t, D);
  } else if (type == DT_E4M3) {
    uint32_t d[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      d[j] = pack_e4m3x2(v[4 * j], v[4 * j + 1]) | pack_e4m3x2(v[4 * j + 2], v[4 * j + 3]) << 16;
    store_words<1, T, ALIGNED>(d, row, piece, t, D);
  } else {
    uint32_t d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = pack16(v[2 * j], v[2 * j + 1], type);
    store_words<2, T, ALIGNED>(d, row, piece, t, D);
  }
}

// Sum (or unsigned maximum) over the T threads of a row. With T > 32 every thread of the block calls
// it the same number of times; `part` holds one word per warp and call.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = warp_sum(v);
  if constexpr (T > 32) {
    const int warp = threadIdx.x >> 5, first = warp / (T / 32) * (T / 32);
    if ((threadIdx.x & 31) == 0) part[warp] = v;
    __syncthreads();
    v = part[first];
#pragma unroll
    for (int i = 1; i < T / 32; ++i) v += part[first + i];
  }
  return v;
}
template <int T>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (T > 32) {
    uint32_t* p = reinterpret_cast<uint32_t*>(part);
    const int warp = threadIdx.x >> 5, first = warp / (T / 32) * (T / 32);
    if ((threadIdx.x & 31) == 0) p[warp] = v;
    __syncthreads();
    v = p[first];
#pragma unroll
    for (int i = 1; i < T / 32; ++i) v = max(v, p[first + i]);
  }
  return v;
}

template <int T>
__host__ __device__ constexpr int block_threads() {
  return T < 256 ? 256 : T;
}

// Blocks per SM that the registers of the larger forms are held to: without it some take a few more than
// fit (16-bit rows of 16384 125 us instead of 85, unaligned ones of 8191 194 instead of 135).
template <int XW, int RW, int T, int NV, bool ALIGNED>
constexpr int min_blocks() {
  if (!ALIGNED) return NV != 2 ? 1 : T < 512 ? 3 : 2;
  return NV != 4 || XW + RW > 6 ? 1 : T < 512 ? 3 : XW == 2 ? 2 : 1;
}

// Sums that fp32 does not hold: the mean's is taken times kPart (16384 elements cannot overflow it), and
// rows whose squares leave the range are held times another power of two. Both are exact.
constexpr float kPart = 0x1p-15f, kDown = 0x1p-80f, kUp = 0x1p96f, kTiny = 0x1p-100f;
__device__ __forceinline__ bool lost(float sum) { return !(fabsf(sum) <= 3.402823466e38f); }
// Whether odd(sum) holds for this thread's row, whose sum is `own`; in blocks of several rows that meet at
// barriers (where row_sum left its partial sums in `part`), whether it holds for any of them.
template <int T, typename F>
__device__ __forceinline__ bool any_row(float own, const float* part, F odd) {
  if constexpr (T == 32 || block_threads<T>() == T) return odd(own);
  bool any = false;
#pragma unroll
  for (int r = 0; r < block_threads<T>() / T; ++r) {
    float v = part[r * (T / 32)];
#pragma unroll
    for (int i = 1; i < T / 32; ++i) v += part[r * (T / 32) + i];
    any = any || odd(v);
  }
  return any;
}

// XW / RW: sizes of x's and r's elements (RW 0: no r).
template <int XW, int RW, int T, int NV, bool ALIGNED>
__global__ void __launch_bounds__(block_threads<T>(), min_blocks<XW, RW, T, NV, ALIGNED>()) norm_kernel(const NormArgs a) {
  constexpr int kRows = block_threads<T>() / T;
  pdl_trigger();
  pdl_wait();
  __shared__ float part[4][block_threads<T>() / 32];
  const int t = threadIdx.x % T;
  const long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / T;
  const bool on = row < a.rows;
  const int D = on ? a.D : 0;  // a block's rows past the end take part in the barriers only
  const long long r0 = on ? row : 0;

  float v[NV][8];
  {
    Raw8<XW> x[NV];
    Raw8<RW ? RW : 2> r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      load8<XW, T, ALIGNED, true>(x[i], static_cast<const char*>(a.x) + r0 * a.ldx * XW, i, t, D);
    if constexpr (RW != 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        load8<RW, T, ALIGNED, true>(r[i], static_cast<const char*>(a.resid) + r0 * a.ldr * RW, i, t, D);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = value(x[i], j, a.x_type);
        if constexpr (RW != 0) v[i][j] += value(r[i], j, a.resid_type);
      }
  }
  if (a.sum && on) {
    void* row_p = static_cast<char*>(a.sum) + r0 * a.lds * (a.sum_type == DT_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<T, ALIGNED>(v[i], row_p, a.sum_type, i, t, D);
  }

  if (a.center) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(v[i][j], kPart, s);
    const float mean = row_sum<T>(s, part[0]) / (a.D * kPart);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (i * T + t) * 8 + j < D ? v[i][j] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) q = fmaf(v[i][j], v[i][j], q);
  float squares = row_sum<T>(q, part[1]);
  // (a sum that is too small matters only where eps does not cover it)
  auto odd = [&](float sum) { return lost(sum) || (a.eps < kTiny && sum < kTiny); };
  float eps = a.eps;
  if (__builtin_expect(any_row<T>(squares, part[1], odd), 0)) {
    const float f = lost(squares) ? kDown : odd(squares) ? kUp : 1.f;
    eps = eps * f * f;
    q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] *= f;
        q = fmaf(v[i][j], v[i][j], q);
      }
    squares = row_sum<T>(q, part[3]);
  }
  const float rstd = 1.f / sqrtf(squares / a.D + eps);

#pragma unroll
  for (int i = 0; i < NV; ++i) {
    Raw8<4> w, b;
    load8<4, T, ALIGNED, false>(w, a.w, i, t, D);
    if (a.b) load8<4, T, ALIGNED, false>(b, a.b, i, t, D);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = v[i][j] * rstd * value(w, j, DT_F32);
      if (a.b) v[i][j] += value(b, j, DT_F32);
    }
  }
  if (a.out_type == DT_E4M3) {
    // the largest |y| as bits: they order as the values do, with infinity and then NaN above all
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((i * T + t) * 8 + j < D) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
    // 448 is e4m3's largest value; a row of zeros (or one whose scale would be subnormal) takes the
    // smallest normal scale, so that its inverse stays finite. y / s is taken as y * (1 / s): at most
    // 1.5 units of fp32's last place from the quotient before the rounding to 4 bits.
    const float amax = __uint_as_float(row_max<T>(top, part[2]));
    const float s = amax / 448.f < 1.17549435e-38f ? 1.17549435e-38f : amax / 448.f;  // NaN stays NaN
    const float inv = 1.f / s;
    if (t == 0 && on) a.scale[row] = s;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= inv;
  }
  if (!on) return;
  const int es = a.out_type == DT_F32 ? 4 : a.out_type == DT_E4M3 ? 1 : 2;
  void* row_p = static_cast<char*>(a.out) + r0 * a.ldo * es;
#pragma unroll
  for (int i = 0; i < NV; ++i) store8<T, ALIGNED>(v[i], row_p, a.out_type, i, t, D);
}

template <int XW, int RW, bool ALIGNED>
cudaError_t launch_shape(const NormArgs& a, int T, int NV, cudaStream_t st) {
  auto go = [&](auto kernel, int threads, int rows) {
    const unsigned grid = static_cast<unsigned>((a.rows + (long long)rows - 1) / rows);
    return launch_pdl(kernel, dim3(grid), dim3(threads), 0, st, a);
  };
#define LAYA_NORM(t, nv) \
  if (T == t && NV == nv) return go(norm_kernel<XW, RW, t, nv, ALIGNED>, block_threads<t>(), block_threads<t>() / t)
  LAYA_NORM(32, 2);
  LAYA_NORM(128, 2);
  LAYA_NORM(512, 2);
  LAYA_NORM(512, 4);
  if constexpr (ALIGNED) {
    LAYA_NORM(32, 1);
    LAYA_NORM(128, 1);
    LAYA_NORM(512, 1);
    LAYA_NORM(32, 4);
    LAYA_NORM(128, 4);
  }
#undef LAYA_NORM
  return cudaErrorInvalidValue;
}

bool aligned(const void* p, long long ld, int es, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (ld * es) % bytes == 0;
}

template <int XW, int RW>
cudaError_t launch_rows(const NormArgs& a, int num_sms, cudaStream_t st) {
  bool al = aligned(a.x, a.ldx, XW, 16) && aligned(a.w, 0, 4, 16) && aligned(a.b, 0, 4, 16);
  if (RW) al = al && aligned(a.resid, a.ldr, RW, 16);
  if (a.sum) al = al && aligned(a.sum, a.lds, type_size(a.sum_type), 16);
  al = al && aligned(a.out, a.ldo, type_size(a.out_type), a.out_type == DT_E4M3 ? 8 : 16);
  // Threads per row: as few as hold the row in 4 pieces of 8 elements each (long loads in flight, one
  // warp up to 1024 elements, no barrier), but one piece each while the rows cannot fill the GPU's
  // warps, where the shorter serial chain counts. Rows at other alignments hold more registers a piece:
  // 2 pieces each.
  const int pieces = (a.D + 7) / 8;
  const bool few = static_cast<long long>(a.rows) * ((pieces + 127) / 128) < 4LL * num_sms;
  const int most = !al ? 2 : few ? 1 : 4;
  int T = 32, NV = al ? 1 : 2;
  while (T < 512 && T * most < pieces) T *= 4;
  while (T * NV < pieces) NV *= 2;
  if (NV > 4) return cudaErrorInvalidValue;
  return al ? launch_shape<XW, RW, true>(a, T, NV, st) : launch_shape<XW, RW, false>(a, T, NV, st);
}

}  // namespace

cudaError_t norm_launch(const NormArgs& a, int num_sms, cudaStream_t st) {
  const int rw = a.resid ? type_size(a.resid_type) : 0;
  if (type_size(a.x_type) == 4)
    return rw == 0   ? launch_rows<4, 0>(a, num_sms, st)
           : rw == 2 ? launch_rows<4, 2>(a, num_sms, st)
                     : launch_rows<4, 4>(a, num_sms, st);
  return rw == 0   ? launch_rows<2, 0>(a, num_sms, st)
         : rw == 2 ? launch_rows<2, 2>(a, num_sms, st)
                   : launch_rows<2, 4>(a, num_sms, st);
}

}  // namespace laya

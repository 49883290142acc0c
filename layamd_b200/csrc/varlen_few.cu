// Masked attention for few query rows (single tokens over long keys): every key and value is read once
// and nearly nothing is computed, so the bound is HBM. A CTA takes up to 16 query rows that share a key
// head (query heads of the group times query tokens) and a range of the keys. One warp streams 64-key
// chunks of K and V by TMA into a ring of 6 stages (192 KB in flight per SM: two CTAs at head dim 64,
// one at 128); the 8 others work in two groups that take the chunks in turn, 16 keys of a chunk per
// warp, on mma.sync m16n8k16 with ldmatrix from the swizzled tiles. The warps' partial rows (each
// with its own running maximum and sum) are joined through shared memory in warp order.
//
// Single tokens of 24 sequences with up to 32,768 keys (1.8 GB of K and V), capped: 356 us, 0.77 of the
// measured copy bandwidth. Operands loaded straight into registers, with no more than 64 KB in flight
// per SM, took a third longer; the softmax of the eight rows that four query heads leave empty, 15 %.
//
// The softmax is fp32; its weights are rounded to the inputs' type for the product with V (their sum is
// not), as mma.sync wants operands of one type. Masked scores are replaced. Values of keys that nobody may see are set to zero in shared memory, so
// that nothing they hold reaches a row.
#include "kernels.h"
#include "varlen.cuh"

namespace laya {
namespace {

constexpr int kWarps = 8, kKeys = 64, kStages = 6, kThreads = 32 * (kWarps + 1);
constexpr uint32_t kAtom = kKeys * 128;  // 64 rows x 64 values
// Most chunks skipped by document before one is loaded all the same (masked, it adds nothing): a skipped
// chunk takes 0.3 to 0.5 us, so that the consumers' waits stay far below their budget of a second however
// many keys lie between two of the rows' documents.
constexpr int kMostSkipped = 1 << 13;

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf) {
  if (bf)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16-byte piece `piece` of row `row` of a tile whose atoms are 64 columns (8 pieces) wide.
__device__ __forceinline__ uint32_t tile_at(uint32_t tile, int row, int piece) {
  return tile + (piece >> 3) * kAtom + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

template <int D>
struct FewSmem {
  union {
    struct {
      uint8_t k[D / 64][kAtom], v[D / 64][kAtom];
    } stage[kStages];
    float o[kWarps][16][D];  // partial rows, once every chunk has been used
  };
  alignas(8) uint64_t full[kStages], empty[kStages];
  int chunk[kStages];  // the chunk in a stage; -1: no more
  float m[kWarps][16], l[kWarps][16];
  int abort;
};
template <int D>
constexpr size_t smem_bytes() { return sizeof(FewSmem<D>) + 1024; }

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, err, code));
}

template <int D, bool MOD>
__global__ void __launch_bounds__(kThreads, D == 64 ? 2 : 1)
    varlen_few_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                      const VarlenArgs a, int* err) {
  constexpr int kQ = D / 16;  // steps of 16 dimensions
  extern __shared__ uint8_t smem_raw[];
  FewSmem<D>& S = *reinterpret_cast<FewSmem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  pdl_trigger();
  pdl_wait();
  const int G = a.Hq / a.Hkv, row_tiles = (a.max_q * G + 15) / 16;
  int u = static_cast<int>(blockIdx.x);
  const int rt = u % row_tiles;
  u /= row_tiles;
  const int hk = u % a.Hkv;  // heads next to one another in memory run together
  u /= a.Hkv;
  const int sp = u % a.splits;
  const Sequence s = sequence(a, u / a.splits);
  const int nrows = min(s.lq, a.max_q) * G;  // (token, head of the group) rows of this key head
  if (rt * 16 >= nrows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool bf = a.type == DT_BF16;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&S.full[i]), 1);
      mbar_init(smem_u32(&S.empty[i]), kWarps / 2);
    }
    S.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  volatile int* abort = &S.abort;

  // chunks that the masks can reach: the prefix's, then the window's
  const int p_first = (rt * 16) / G + s.lk - s.lq, p_last = min(rt * 16 + 15, nrows - 1) / G + s.lk - s.lq;
  const int wlo = max(0, p_first - a.left), whi = min(s.lk, p_last + a.right + 1);
  const int end_a = (s.prefix + kKeys - 1) / kKeys;
  const int beg_b = max(end_a, whi > wlo ? wlo / kKeys : 0);
  const int end_b = whi > wlo ? (whi + kKeys - 1) / kKeys : 0;
  const long long chunks = end_a + max(0, end_b - beg_b);
  const int j0 = static_cast<int>(chunks * sp / a.splits), j1 = static_cast<int>(chunks * (sp + 1) / a.splits);

  // this thread's rows: g and g + 8 of the tile
  int pos[2], head[2], qdoc[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int R = rt * 16 + g + 8 * r;
    const bool on = R < nrows;
    const int qi = on ? R / G : 0;
    head[r] = hk * G + (on ? R - qi * G : 0);
    pos[r] = qi + s.lk - s.lq;
    qdoc[r] = a.doc_q ? (on ? a.doc_q[s.q0 + qi] : -1) : 0;
  }

  if (warp == kWarps) {
    // ---------------- TMA producer
    int doc_lo = 0, doc_hi = 0;
    if (a.doc_k) {
      const int lo0 = qdoc[0] < 0 ? 0x7fffffff : qdoc[0], lo1 = qdoc[1] < 0 ? 0x7fffffff : qdoc[1];
      doc_lo = __reduce_min_sync(0xffffffffu, min(lo0, lo1));
      doc_hi = __reduce_max_sync(0xffffffffu, max(qdoc[0], qdoc[1]));
    }
    int n = 0, skipped = 0;
    bool ok = true;
    auto stage_free = [&]() {
      const int st = n % kStages;
      return n < kStages ||
             __all_sync(0xffffffffu, mbar_wait(smem_u32(&S.empty[st]), ((n / kStages) - 1) & 1, abort, err, kErrAttnLoad));
    };
    for (int j = j0; ok && j < j1; ++j) {
      const int c = j < end_a ? j : j - end_a + beg_b;
      if (a.doc_k) {  // a chunk without a key of the rows' documents is not read
        const int k = c * kKeys + lane;
        const int x = k < s.lk ? __ldg(a.doc_k + s.k0 + k) : -1, y = k + 32 < s.lk ? __ldg(a.doc_k + s.k0 + k + 32) : -1;
        const bool hit = (x >= 0 && x >= doc_lo && x <= doc_hi) || (y >= 0 && y >= doc_lo && y <= doc_hi);
        if (!__any_sync(0xffffffffu, hit) && ++skipped < kMostSkipped) continue;
        skipped = 0;
      }
      if (!stage_free()) { ok = false; break; }
      if (lane == 0) {
        const int st = n % kStages;
        const uint32_t fb = smem_u32(&S.full[st]);
        S.chunk[st] = c;
        mbar_expect_tx(fb, 2 * (D / 64) * kAtom);
#pragma unroll
        for (int d = 0; d < D / 64; ++d) {
          tma_load_3d(smem_u32(S.stage[st].k[d]), &tk, d * 64, hk, s.k0 + c * kKeys, fb);
          tma_load_3d(smem_u32(S.stage[st].v[d]), &tv, d * 64, hk, s.k0 + c * kKeys, fb);
        }
      }
      __syncwarp();
      ++n;
    }
    if (lane == 0) {  // whatever becomes of the consumers, no load is in flight when the CTA exits
      const long long t0 = clock64();
      for (int st = 0; st < kStages; ++st) {
        const int issued = (n - st + kStages - 1) / kStages;
        if (issued <= 0) continue;
        while (!mbar_try(smem_u32(&S.full[st]), (issued - 1) & 1))
          if (clock64() - t0 > kWaitBudgetCycles) { atomicCAS(err, 0, kErrGemmDrain); break; }
      }
    }
    __syncwarp();
    for (int i = 0; ok && i < 2; ++i) {  // the end, once for each group
      if (!stage_free()) { ok = false; break; }
      if (lane == 0) {
        S.chunk[n % kStages] = -1;
        mbar_arrive(smem_u32(&S.full[n % kStages]));
      }
      __syncwarp();
      ++n;
    }
    __syncthreads();
    return;
  }

  // ---------------- consumers: warp w takes keys 16 (w % 4) .. of its group's chunks
  const bool two = nrows - rt * 16 > 8;  // rows 8 .. 15 of the tile hold anything
  const int group = warp >> 2, key0 = 16 * (warp & 3);
  uint32_t q[kQ][4];
  float slope[2];
  const float cs = a.scale * kLog2e, up_by = bf ? 0.f : kUpF16;
  const float cap_in = MOD && a.cap > 0.f ? a.scale / a.cap : 0.f, cap_out = a.cap * kLog2e;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    slope[r] = MOD && a.slopes ? a.slopes[head[r]] * kLog2e : 0.f;
    const bool on = rt * 16 + g + 8 * r < nrows;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(
        static_cast<const uint16_t*>(a.q) + (long long)(s.q0 + pos[r] - s.lk + s.lq) * a.ldq + head[r] * D);
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      q[i][r] = on ? __ldg(src + 8 * i + t) : 0u;
      q[i][r + 2] = on ? __ldg(src + 8 * i + 4 + t) : 0u;
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float mr[2] = {-INFINITY, -INFINITY}, lr[2] = {0.f, 0.f};
  // ldmatrix rows of this lane: K matrices (keys 0-7, 8-15) x (dims 0-7, 8-15), V ones transposed
  const int k_row = key0 + (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
  const int v_row = key0 + (lane & 15), v_piece = lane >> 4;

  for (int n = group;; n += 2) {
    const int st = n % kStages;
    if (!warp_wait(smem_u32(&S.full[st]), (n / kStages) & 1, abort, err, kErrAttnSoftmax)) break;
    const int c = *static_cast<volatile int*>(&S.chunk[st]);
    if (c < 0) break;
    const int kb = c * kKeys + key0;
    int kid = 0;  // document of key kb + lane % 16
    if (a.doc_k) kid = kb + (lane & 15) < s.lk ? __ldg(a.doc_k + s.k0 + kb + (lane & 15)) : -1;
    const uint32_t kt = smem_u32(S.stage[st].k[0]), vt = smem_u32(S.stage[st].v[0]);
    float x[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      uint32_t b[4];
      ldmatrix4(b, tile_at(kt, k_row, 2 * i + k_piece));
      mma16(x[0], q[i], b[0], b[1], bf);
      mma16(x[1], q[i], b[2], b[3], bf);
    }
    // keys that nobody may see: their values are zero from here on
    const bool dead = kb + (lane & 15) >= s.lk || (a.doc_k && kid < 0);
    if (__any_sync(0xffffffffu, dead)) {
      if (dead) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)  // lanes l and l + 16 share a row
          *reinterpret_cast<uint4*>(S.stage[st].v[0] + (tile_at(vt, key0 + (lane & 15), 2 * i + (lane >> 4)) - vt)) =
              make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage is loaded again
      __syncwarp();
    }
    // x[i][2 r + e]: row g + 8 r, key kb + 8 i + 2 t + e
    const bool full = !a.doc_k && kb + 16 <= s.lk &&
                      ((kb >= p_last - a.left && kb + 15 <= p_first + a.right) || kb + 16 <= s.prefix);
    bool small = false;  // every score of the warp is: the general form of tanh is skipped
    if (MOD && a.cap > 0.f) {
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[i][e]));
      small = __all_sync(0xffffffffu, big * cap_in < kTanhSmall);
    }
    float top[2] = {-INFINITY, -INFINITY};
    bool up = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r == 1 && !two) break;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e) {
          const int off = 8 * i + 2 * t + (e & 1), key = kb + off;
          float v = x[i][e];
          if constexpr (MOD) {
            if (a.cap > 0.f) {  // each score's form by itself: a row's bits depend on nothing else in the tile
              const float u = v * cap_in;
              float th = tanh_small(u);
              if (!small) th = pick_below(fabsf(u), kTanhSmall, th, tanh_any(u));
              v = __fmul_rn(cap_out, th);  // (rounded before the maximum is subtracted, as the maximum is)
            } else {
              v = __fmul_rn(v, cs);
            }
            if (a.slopes) v = fmaf(-slope[r], fabsf(static_cast<float>(pos[r] - key)), v);
          } else {
            v = __fmul_rn(v, cs);
          }
          if (!full) {
            bool see = key < s.lk && ((key >= pos[r] - a.left && key <= pos[r] + a.right) || key < s.prefix);
            if (a.doc_k) {
              const int id = __shfl_sync(0xffffffffu, kid, off);
              see = see && id >= 0 && id == qdoc[r];
            }
            if (!see) v = -INFINITY;
          }
          x[i][e] = v;
        }
      top[r] = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      up = up || top[r] - mr[r] > kGrow + up_by;
    }
    // a row's reference moves when its own scores pass it
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool mine = top[r] - mr[r] > kGrow + up_by;
        const float m_new = mine ? top[r] - up_by : mr[r];
        const float alpha = mine ? exp2_fast(mr[r] - m_new) : 1.f;
        mr[r] = m_new;
        lr[r] *= alpha;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][2 * r] *= alpha;
          o[i][2 * r + 1] *= alpha;
        }
      }
    }
    uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r == 1 && !two) break;
      const float sub = mr[r] == -INFINITY ? 0.f : mr[r];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = exp2_fast(x[i][2 * r] - sub), p1 = exp2_fast(x[i][2 * r + 1] - sub);
        lr[r] += p0 + p1;
        pa[2 * i + r] = pack_pair(p0, p1, a.type);
      }
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t b[4];
      ldmatrix4_t(b, tile_at(vt, v_row, 2 * i + v_piece));
      mma16(o[2 * i], pa, b[0], b[1], bf);
      mma16(o[2 * i + 1], pa, b[2], b[3], bf);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&S.empty[st]));
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    lr[r] += __shfl_xor_sync(0xffffffffu, lr[r], 1);
    lr[r] += __shfl_xor_sync(0xffffffffu, lr[r], 2);
  }
  __syncthreads();  // every chunk has been used: the stages take the partial rows
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (t == 0) {
      S.m[warp][g + 8 * r] = mr[r];
      S.l[warp][g + 8 * r] = lr[r];
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<float2*>(&S.o[warp][g + 8 * r][8 * i + 2 * t]) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
  }
  asm volatile("bar.sync 1, 256;" ::: "memory");  // the consumers
  // 16 threads a row join the warps' partial rows
  const int row = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * (D / 16);
  const int R = rt * 16 + row;
  if (R >= nrows) return;
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, S.m[w][row]);
  float l = 0.f, v[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) v[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float f = S.m[w][row] == -INFINITY ? (S.l[w][row] == 0.f ? 0.f : 1.f) : exp2_fast(S.m[w][row] - m);
    l = fmaf(f, S.l[w][row], l);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) v[i] = fmaf(f, S.o[w][row][c0 + i], v[i]);
  }
  const float inv = l > 0.f ? 1.f / l : l;  // a row that sees nothing is 0; NaN stays NaN
  const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
  const int qi = R / G, h = hk * G + R - qi * G;
  const long long r = (long long)s.q0 + qi;
  if (a.splits == 1) {
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + r * a.ldo + h * D + c0);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dst[i] = pack_pair(v[2 * i] * inv, v[2 * i + 1] * inv, a.type);
    if (c0 == 0 && a.lse) a.lse[r * a.Hq + h] = lse2 * kLn2;
  } else {
    const long long at = ((long long)sp * a.rows_q + r) * a.Hq + h;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) a.part_o[at * D + c0 + i] = v[i] * inv;
    if (c0 == 0) a.part_l[at] = lse2;
  }
}

template <int D>
cudaError_t launch(const VarlenArgs& a, int* err, cudaStream_t st) {
  CUtensorMap tk, tv;
  auto map = [&](CUtensorMap* m, const void* base, long long ld) {
    return make_rows_map(m, base, a.type, D, static_cast<uint64_t>(a.Hkv), static_cast<uint64_t>(a.rows_k > 0 ? a.rows_k : 1), D,
                         static_cast<uint64_t>(ld), kKeys);
  };
  if (!map(&tk, a.k, a.ldk) || !map(&tv, a.v, a.ldv)) return cudaErrorInvalidValue;
  const int G = a.Hq / a.Hkv;
  const long long grid = (long long)((a.max_q * G + 15) / 16) * a.splits * a.Hkv * a.B;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  const dim3 g(static_cast<unsigned>(grid));
  return a.cap > 0.f || a.slopes
             ? launch_pdl(varlen_few_kernel<D, true>, g, dim3(kThreads), smem_bytes<D>(), st, tk, tv, a, err)
             : launch_pdl(varlen_few_kernel<D, false>, g, dim3(kThreads), smem_bytes<D>(), st, tk, tv, a, err);
}

template <int D>
cudaError_t prepare() {
  const int bytes = static_cast<int>(smem_bytes<D>());
  const cudaError_t e =
      cudaFuncSetAttribute(varlen_few_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(varlen_few_kernel<D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace

cudaError_t varlen_few_prepare_device() {
  const cudaError_t e = prepare<64>();
  return e != cudaSuccess ? e : prepare<128>();
}

// Up to 8 queries. This kernel walks the keys once for 16 rows of a group, the tile kernel once for every
// query head, in about the same time whatever its rows hold; so the queries count, not the heads that share
// a key head. This kernel and the tile kernel in us, 64 sequences of 4096 keys, head dim 128, 4 query heads
// to a key head: 4 queries 220 and 656, 8 387 and 667, 16 732 and 659; 32 heads: 4 queries 210 and 596, 8
// 384 and 596, 12 569 and 596; one head: 8 373 and 445, 16 420 and 446, 24 696 and 470. With less to do
// (8 sequences of 4096 keys, 4 heads): 4 queries 59 and 90, 8 93 and 90, 16 138 and 90; one head 8 84 and 54.
bool varlen_few_rows(int max_q) { return max_q <= 8; }

cudaError_t varlen_few_launch(const VarlenArgs& a, int* err, cudaStream_t st) {
  return a.D == 64 ? launch<64>(a, err, st) : launch<128>(a, err, st);
}

}  // namespace laya

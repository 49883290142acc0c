// Matrix product with scales, bias, activation and residual in its epilogue, on the 5th-generation
// tensor cores: out[m][n] = act(sa[m] sw[n] sum_k A[m][k] W[n][k] + bias[n]) + resid[m][n] for 16-bit
// (kind::f16) and e4m3 (kind::f8f6f4) operands of any M, N, K, both K-major, fp32 sums in tensor memory.
//
// Two kernels, chosen by the number of tiles (linear_launch):
//   pair    persistent CTA pairs, 256 x 256 tiles with the 2-SM MMA, two accumulators so that a tile's
//           epilogue (eight warps a CTA) runs under the next tile's products. For grids that fill the
//           GPU. 16384 x 8192 x 4096: fp16 834 us in single calls and 915 back to back (1.2 PFLOP/s; a
//           library product without an epilogue takes 684 and 689 on the same GPU, so power is not what
//           bounds it: W, 67 MB, is read again from L2 for every two or three row blocks), e4m3 with GELU
//           426 us (2.6 PFLOP/s), where the operands' way from L2 counts (64 KB a K block and pair); 52,287 x
//           1024 x 2624 e4m3 129 us, 152 with a bf16 residual, 179 on inputs that L2 does not hold.
//   tile    one 128 x BN tile per cluster of S CTAs (BN 64 or 128), each CTA a slice of K. The partial
//           sums go to shared memory and each CTA finishes 128 / S rows, reading the others' partials
//           through the cluster in slice order: one launch, no workspace, and the same sums in every
//           run. For grids that cannot fill the GPU, and a few rows of large weights; bound by a CTA's
//           chain of loads, products and joins.
// Both write through shared memory: a thread reads its accumulator row out of tensor memory, and the
// warp then walks the rows with 8 lanes each, so that the residual, the output, the column scales and
// biases are all touched by consecutive lanes, at any alignment and any odd N. The next residual
// piece is loaded while one is worked on.
#include <algorithm>

#include "kernels.h"
#include "linear_epi.cuh"

namespace laya {
namespace {

constexpr int kThreads = 192;  // TMA producer, MMA issuer, four epilogue warps (the pair kernel has eight)
constexpr int kSlabBytes = 128;                 // bytes of K per stage and row: one swizzle span
constexpr uint32_t kRowBlock = 128 * kSlabBytes;  // 128 rows of a stage

// Column chunks of 64 fp32 sums: 256 bytes a row, 16-byte piece j of row r at position
// (j / 2 + 8 (j % 2)) ^ (r % 8). A thread writing its row and 8 lanes reading 8 columns each of one row
// both touch every bank once per 128 bytes.
__device__ __forceinline__ int piece_at(int row, int j) { return (((j >> 1) | (j & 1) << 3) ^ (row & 7)) * 16; }

__device__ __forceinline__ void put_chunk(uint8_t* row_base, int row, const float* v) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    *reinterpret_cast<float4*>(row_base + piece_at(row, j)) =
        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
// Columns 32 half .. of the chunk.
__device__ __forceinline__ void put_half(uint8_t* row_base, int row, int half, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<float4*>(row_base + piece_at(row, 8 * half + j)) =
        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
__device__ __forceinline__ void get8(float (&v)[8], const uint8_t* row_base, int row, int c8) {
  const float4 x = *reinterpret_cast<const float4*>(row_base + piece_at(row, 2 * c8));
  const float4 y = *reinterpret_cast<const float4*>(row_base + piece_at(row, 2 * c8 + 1));
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
// The same from CTA `rank`'s shared memory, added.
__device__ __forceinline__ void add8_cluster(float (&v)[8], uint32_t row_base, int row, int c8) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(row_base + piece_at(row, 2 * c8 + h))
                 : "memory");
    v[4 * h] += x.x; v[4 * h + 1] += x.y; v[4 * h + 2] += x.z; v[4 * h + 3] += x.w;
  }
}

template <bool F8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (F8) umma_f8(d, a, b, idesc, acc);
  else umma_bf16(d, a, b, idesc, acc);
}
template <bool F8>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (F8) umma_f8_pair(d, a, b, idesc, acc);
  else umma_bf16_pair(d, a, b, idesc, acc);
}

// A bounded wait of a whole warp: all lanes get the same answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, err, code));
}

// Bounded wait, at the end of a producer, until the loads of its last round have landed.
__device__ __forceinline__ void drain_loads(uint64_t* full, int stages, uint32_t issued, uint32_t phases, int* err) {
  const long long t0 = clock64();
  for (int s = 0; s < stages; ++s) {
    if (!(issued & (1u << s))) continue;
    while (!mbar_try(smem_u32(&full[s]), (phases >> s) & 1)) {
      if (clock64() - t0 > kWaitBudgetCycles) { atomicCAS(err, 0, kErrGemmDrain); break; }
    }
  }
}

// ------------------------------------------------------------------ CTA pairs
constexpr int kPairStages = 5, kPairEpiWarps = 8, kPairThreads = 32 * (2 + kPairEpiWarps);
struct PairSmem {
  alignas(1024) uint8_t a[kPairStages][kRowBlock];
  alignas(1024) uint8_t b[kPairStages][kRowBlock];
  alignas(1024) uint8_t stg[kPairEpiWarps][32 * 256];  // per epilogue warp: 32 rows of one column chunk
  alignas(8) uint64_t full[kPairStages];
  uint64_t empty[kPairStages];
  uint64_t accf[2];
  uint64_t acce[2];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};
constexpr size_t pair_smem_bytes() { return sizeof(PairSmem) + 1024; }

template <bool F8, int OW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                       const LinearArgs p, int* err) {
  constexpr int BN = 256, kBK = F8 ? 128 : 64;
  constexpr uint32_t kStageBytes = 4 * kRowBlock;  // both CTAs' A and B halves
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  PairSmem& S = *reinterpret_cast<PairSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cid = static_cast<int>(cluster_id_x()), ncl = static_cast<int>(num_clusters_x());
  const int num_n = (p.N + BN - 1) / BN;
  const int tiles = ((p.M + 255) / 256) * num_n;
  const int nkb = (p.K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) { mbar_init(smem_u32(&S.full[s]), 1); mbar_init(smem_u32(&S.empty[s]), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(smem_u32(&S.accf[a]), 1); mbar_init(smem_u32(&S.acce[a]), 2 * kPairEpiWarps); }
    mbar_init(smem_u32(&S.drain), 1);
    S.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&ta); tma_prefetch_desc(&tb); }
  if (warp == 1) { tmem_alloc_pair(smem_u32(&S.tmem), 2 * BN); tmem_relinquish_pair(); }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  pdl_wait();
  volatile int* abort = &S.abort;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0, last_phase = 0;
      bool ok = true;
      for (int t = cid; ok && t < tiles; t += ncl) {
        const int mb = t / num_n, nb = t - (t / num_n) * num_n;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(smem_u32(&S.empty[stage]), phase ^ 1, abort, err, kErrGemmEmpty)) { ok = false; break; }
          const uint32_t fb = smem_u32(&S.full[stage]);
          if (leader) mbar_expect_tx(fb, kStageBytes);
          tma_load_3d_pair(smem_u32(S.a[stage]), &ta, kb * kBK, 0, mb * 256 + (int)rank * 128, fb);
          tma_load_3d_pair(smem_u32(S.b[stage]), &tb, kb * kBK, 0, nb * BN + (int)rank * 128, fb);
          issued |= 1u << stage;
          last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
      if (*abort && leader) drain_loads(S.full, kPairStages, issued, last_phase, err);
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      const uint32_t idesc = idesc_of(!F8 && p.ab_type == DT_BF16 ? 1u : 0u, 256, BN);
      uint32_t stage = 0, phase = 0;
      int local = 0;
      for (int t = cid; t < tiles; t += ncl, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(smem_u32(&S.acce[acc]), ((local >> 1) & 1) ^ 1, abort, err, kErrGemmAccEmpty)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        bool ok = true;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(smem_u32(&S.full[stage]), phase, abort, err, kErrGemmFull)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a0 = smem_u32(S.a[stage]), b0 = smem_u32(S.b[stage]);
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 bytes of K each
            mma_pair<F8>(d, sdesc_k128(a0 + k * 32), sdesc_k128(b0 + k * 32), idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit_pair(smem_u32(&S.empty[stage]), mapa_shared(smem_u32(&S.empty[stage]), 1));
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(&S.accf[acc]), mapa_shared(smem_u32(&S.accf[acc]), 1));
      }
      // every earlier commit has landed in both CTAs once this one has
      umma_commit_pair(smem_u32(&S.drain), mapa_shared(smem_u32(&S.drain), 1));
    }
    if (lane == 0) {
      // This wait lasts as long as the kernel: its budget starts again whenever an accumulator turns.
      long long t0 = clock64();
      bool turn = false;
      while (!mbar_try(smem_u32(&S.drain), 0)) {
        const bool now = mbar_try(smem_u32(&S.accf[0]), 0);
        if (now != turn) { turn = now; t0 = clock64(); }
        if (clock64() - t0 > kWaitBudgetCycles) { atomicCAS(err, 0, kErrGemmDrain); break; }
      }
    }
  } else {
    // Two warps per quarter of the accumulator's rows, each with every other chunk of 64 columns.
    const int q = warp & 3, side = (warp - 2) >> 2;
    uint8_t* stg = S.stg[warp - 2];
    const uint32_t acce_leader0 = mapa_shared(smem_u32(&S.acce[0]), 0);
    const uint32_t acce_leader1 = mapa_shared(smem_u32(&S.acce[1]), 0);
    const int r4 = lane >> 3, c8 = lane & 7;
    // A chunk's residual (32 rows x 64 columns a warp) is loaded as one batch when the chunk before it
    // is done, under the wait for the accumulator; single loads kept in flight step by step were slower
    // (a warp has few scoreboards, so that waiting for the oldest waits for newer ones too).
    Cols8<OW> res[8];
    struct Place {  // where this lane's first row of a chunk lies in resid
      const char* at;
      int row, col;
      bool whole;  // 8 columns in one access
    };
    const long long step_bytes = 4 * p.ldr * OW;
    auto place = [&](int t, int c) {
      const int mb = t / num_n, nb = t - mb * num_n;
      Place w;
      w.row = t < tiles ? mb * 256 + (int)rank * 128 + q * 32 + r4 : p.M;
      w.col = nb * BN + c * 64 + c8 * 8;
      w.at = static_cast<const char*>(p.resid) + (static_cast<long long>(w.row) * p.ldr + w.col) * OW;
      w.whole = p.vec_out && w.col + 8 <= p.N;
      return w;
    };
    auto fetch = [&](Cols8<OW>& r, const Place& w, int step) {
      if (w.whole) {
        if (w.row + 4 * step < p.M) {
#pragma unroll
          for (int i = 0; i < OW / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(w.at + step * step_bytes)[i];
        }
      } else {
        load_resid<OW>(r, p, w.row + 4 * step, w.col);
      }
    };
    const Place first = place(cid, side);
    if (p.resid) {
#pragma unroll
      for (int i = 0; i < 8; ++i) fetch(res[i], first, i);
    }
    int local = 0;
    for (int t = cid; t < tiles; t += ncl, ++local) {
      const int acc = local & 1;
      const int mb = t / num_n, nb = t - (t / num_n) * num_n;
      const int row0 = mb * 256 + (int)rank * 128 + q * 32;
      const float sa = p.a_scale && row0 + lane < p.M ? p.a_scale[row0 + lane] : 1.f;
      if (!warp_wait(smem_u32(&S.accf[acc]), (local >> 1) & 1, abort, err, kErrGemmAccFull)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int c = side; c < BN / 64; c += 2) {
        const int col = nb * BN + c * 64 + c8 * 8;
        ColParams cp;
        load_cols(cp, p, col);
        __syncwarp();  // the previous chunk has been read
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float v[32];
          tmem_ld32(tbase + c * 64 + 32 * half, v);
          put_half(stg + lane * 256, lane, half, v);
        }
        if (c + 2 >= BN / 64) {  // this warp's part of the accumulator is in shared memory
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acc ? acce_leader1 : acce_leader0);
        } else {
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + r4;
          float v[8];
          get8(v, stg + r * 256, r, c8);
          emit8<OW>(v, p, cp, __shfl_sync(0xffffffffu, sa, r), res[i], row0 + r, col);
        }
        if (p.resid) {
          const Place next = c + 2 < BN / 64 ? place(t, c + 2) : place(t + ncl, side);
#pragma unroll
          for (int i = 0; i < 8; ++i) fetch(res[i], next, i);
        }
      }
    }
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while its peer may still signal or read its shared memory
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN);
  }
}

// ------------------------------------------------------------------ one tile per cluster
template <int BN>
constexpr int tile_stages() { return BN == 128 ? 3 : 4; }
template <int BN>
struct TileSmem {
  // operand stages; then the partial sums of 128 rows in chunks of 64 columns (32 KB each)
  alignas(1024) uint8_t a[tile_stages<BN>()][kRowBlock];
  alignas(1024) uint8_t b[tile_stages<BN>()][BN * kSlabBytes];
  alignas(8) uint64_t full[tile_stages<BN>()];
  uint64_t empty[tile_stages<BN>()];
  uint64_t accf;
  uint32_t tmem;
  int abort;
};
template <int BN>
constexpr size_t tile_smem_bytes() { return sizeof(TileSmem<BN>) + 1024; }

template <bool F8, int OW, int BN>
__global__ void __launch_bounds__(kThreads, 2)
    linear_tile_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                       const LinearArgs p, int splits, int* err) {
  constexpr int kBK = F8 ? 128 : 64, kStages = tile_stages<BN>(), kChunks = BN / 64;
  static_assert(kStages * (kRowBlock + BN * kSlabBytes) >= kChunks * 128 * 256, "partials fit the stages");
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  using Smem = TileSmem<BN>;
  Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_n = (p.N + BN - 1) / BN;
  const int t = static_cast<int>(blockIdx.x) / splits, sp = static_cast<int>(blockIdx.x) - t * splits;
  const int mb = t / num_n, nb = t - mb * num_n;
  const int nkb = (p.K + kBK - 1) / kBK;
  const int kb0 = sp * nkb / splits, kb1 = (sp + 1) * nkb / splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(smem_u32(&S.full[s]), 1); mbar_init(smem_u32(&S.empty[s]), 1); }
    mbar_init(smem_u32(&S.accf), 1);
    S.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&ta); tma_prefetch_desc(&tb); }
  if (warp == 1) { tmem_alloc(smem_u32(&S.tmem), BN); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  pdl_wait();
  volatile int* abort = &S.abort;
  const int rows = 32 / splits;  // rows that each epilogue warp finishes: a multiple of 4
  const int q = warp & 3, r4 = lane >> 3, c8 = lane & 7;
  // The CTA finishes tile rows sp * 128 / splits .. ; warp q rows `first` .. first + rows - 1 of the tile.
  const int first = sp * (128 / splits) + q * rows;
  const int steps = kChunks * (rows / 4);  // steps of 4 rows x 64 columns, down the rows of a chunk
  Cols8<OW> res[2][4];
  auto fetch = [&](Cols8<OW> (&r)[4], int i0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = i0 + i;
      if (s >= steps) break;
      const int c = s / (rows / 4), r0 = s - c * (rows / 4);
      load_resid<OW>(r[i], p, mb * 128 + first + 4 * r0 + r4, nb * BN + c * 64 + c8 * 8);
    }
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0, last_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&S.empty[stage]), phase ^ 1, abort, err, kErrGemmEmpty)) break;
        const uint32_t fb = smem_u32(&S.full[stage]);
        mbar_expect_tx(fb, kRowBlock + BN * kSlabBytes);
        tma_load_3d(smem_u32(S.a[stage]), &ta, kb * kBK, 0, mb * 128, fb);
        tma_load_3d(smem_u32(S.b[stage]), &tb, kb * kBK, 0, nb * BN, fb);
        issued |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      if (*abort) drain_loads(S.full, kStages, issued, last_phase, err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_of(!F8 && p.ab_type == DT_BF16 ? 1u : 0u, 128, BN);
      uint32_t stage = 0, phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&S.full[stage]), phase, abort, err, kErrGemmFull)) break;
        tc_fence_after();
        const uint32_t a0 = smem_u32(S.a[stage]), b0 = smem_u32(S.b[stage]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma<F8>(tmem, sdesc_k128(a0 + k * 32), sdesc_k128(b0 + k * 32), idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        umma_commit(smem_u32(&S.empty[stage]));
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      umma_commit(smem_u32(&S.accf));
      // the products issued end before tensor memory is released, also after an abort
      const long long t0 = clock64();
      while (!mbar_try(smem_u32(&S.accf), 0)) {
        if (clock64() - t0 > kWaitBudgetCycles) { atomicCAS(err, 0, kErrGemmDrain); break; }
      }
    }
  } else {
    if (p.resid) fetch(res[0], 0);
    // all operands have been read once the accumulator is complete: the stages take the sums
    if (warp_wait(smem_u32(&S.accf), 0, abort, err, kErrGemmAccFull)) {
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        float v[64];
        tmem_ld64(tmem + c * 64 + (static_cast<uint32_t>(q * 32) << 16), v);
        put_chunk(S.a[0] + c * (128 * 256) + (q * 32 + lane) * 256, lane, v);
      }
      tc_fence_before();
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync_all();
  if (warp >= 2 && __all_sync(0xffffffffu, !*abort)) {
    const int row0 = mb * 128 + first;
    float sa = 1.f;
    if (p.a_scale && lane < rows && row0 + lane < p.M) sa = p.a_scale[row0 + lane];
    uint32_t peer[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) peer[r] = r < splits ? mapa_shared(smem_u32(S.a[0]), r) : 0u;
    ColParams cp;
    int have = -1;
#pragma unroll 1
    for (int s0 = 0; s0 < steps; s0 += 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (p.resid) fetch(res[h ^ 1], s0 + 4 * h + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int s = s0 + 4 * h + i;
          if (s >= steps) break;
          const int c = s / (rows / 4), r = 4 * (s - c * (rows / 4)) + r4;
          const int col = nb * BN + c * 64 + c8 * 8, tr = first + r;
          if (have != c) load_cols(cp, p, col);
          have = c;
          const uint32_t at = static_cast<uint32_t>(c * (128 * 256) + tr * 256);
          float v[8];
          if (splits == 1) {
            get8(v, S.a[0] + at, tr, c8);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < splits) add8_cluster(v, peer[k] + at, tr, c8);
          }
          emit8<OW>(v, p, cp, __shfl_sync(0xffffffffu, sa, r), res[h][i], mb * 128 + tr, col);
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (splits > 1) cluster_sync_all();  // no CTA leaves while a peer may still read its partial sums
  else __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

template <bool F8, int OW>
cudaError_t prepare(int* clusters) {
  cudaError_t e = cudaFuncSetAttribute(linear_tile_kernel<F8, OW, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)tile_smem_bytes<64>());
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(linear_tile_kernel<F8, OW, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)tile_smem_bytes<128>());
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(linear_pair_kernel<F8, OW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)pair_smem_bytes());
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2, 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = pair_smem_bytes();
  int n = 0;
  e = cudaOccupancyMaxActiveClusters(&n, linear_pair_kernel<F8, OW>, &cfg);
  if (e != cudaSuccess) return e;
  if (*clusters == 0 || n < *clusters) *clusters = n;
  return cudaSuccess;
}

struct Maps {
  CUtensorMap a, b;
};
bool make_maps(Maps* m, const LinearArgs& a, int box_b) {
  const uint64_t K = static_cast<uint64_t>(a.K);
  return make_rows_map(&m->a, a.A, a.ab_type, K, 1, static_cast<uint64_t>(a.M), static_cast<uint64_t>(a.lda),
                       static_cast<uint64_t>(a.lda), 128) &&
         make_rows_map(&m->b, a.W, a.ab_type, K, 1, static_cast<uint64_t>(a.N), static_cast<uint64_t>(a.ldw),
                       static_cast<uint64_t>(a.ldw), static_cast<uint32_t>(box_b));
}

template <bool F8, int OW, int BN>
cudaError_t launch_tile(const LinearArgs& a, int splits, int* err, cudaStream_t st) {
  Maps m;
  if (!make_maps(&m, a, BN)) return cudaErrorInvalidValue;
  const long long tiles = ((a.M + 127LL) / 128) * ((a.N + (long long)BN - 1) / BN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = tile_smem_bytes<BN>();
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, linear_tile_kernel<F8, OW, BN>, m.a, m.b, a, splits, err);
}

template <bool F8, int OW>
cudaError_t launch(const LinearArgs& a, int num_sms, int pairs, int* err, cudaStream_t st) {
  const long long pair_tiles = ((a.M + 255LL) / 256) * ((a.N + 255LL) / 256);
  // Pairs (if any are to be used) once their tiles fill at least half of the pairs the GPU holds; below
  // that a tile per cluster, its K cut until the CTAs fill the GPU.
  if (pairs > 0 && pair_tiles * 2 >= pairs) {
    Maps m;
    if (!make_maps(&m, a, 128)) return cudaErrorInvalidValue;
    const int ncl = static_cast<int>(std::min<long long>(pair_tiles, pairs));
    return launch_pdl(linear_pair_kernel<F8, OW>, dim3(2 * ncl), dim3(kPairThreads), pair_smem_bytes(), st, m.a, m.b, a,
                      err);
  }
  const int nkb = (a.K + (F8 ? 127 : 63)) / (F8 ? 128 : 64);
  const long long tiles128 = ((a.M + 127LL) / 128) * ((a.N + 127LL) / 128);
  const bool narrow = tiles128 * std::min(nkb, 8) < num_sms;
  const long long tiles = narrow ? ((a.M + 127LL) / 128) * ((a.N + 63LL) / 64) : tiles128;
  int splits = 1;
  while (splits < 8 && 2 * splits <= nkb && tiles * splits * 2 <= 2LL * num_sms) splits *= 2;
  return narrow ? launch_tile<F8, OW, 64>(a, splits, err, st) : launch_tile<F8, OW, 128>(a, splits, err, st);
}

}  // namespace

cudaError_t linear_prepare_device(int* pair_clusters) {
  *pair_clusters = 0;
  cudaError_t e = cudaSuccess;
  for (cudaError_t r : {prepare<false, 2>(pair_clusters), prepare<false, 4>(pair_clusters),
                        prepare<true, 2>(pair_clusters), prepare<true, 4>(pair_clusters)})
    if (r != cudaSuccess) e = r;
  return e;
}

cudaError_t linear_launch(const LinearArgs& in, int num_sms, int pair_clusters, int* err, cudaStream_t st) {
  LinearArgs a = in;
  const long long es = type_size(a.out_type);
  a.vec_out = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && (a.ldo * es) % 16 == 0 &&
              (!a.resid || ((reinterpret_cast<uintptr_t>(a.resid) & 15) == 0 && (a.ldr * es) % 16 == 0));
  // Up to 16 rows the register-fed kernel, but for a large weight the tile kernel (never pairs, which would
  // compute 256 rows) where W's rows or all of A are long. Device times in us, register-fed against tile
  // kernel (which with short A depends on where its buffers lie, hence the ranges):
  //   1 row    bf16 5248 x 1024 6.6 and 11.6, 8192 x 8192 36 and 31-46, 16384 x 16384 127 and 133-136,
  //            8192 x 28672 113 and 106-118, 5000 x 32768 116 and 75-84;
  //            e4m3 16384 x 16384 70 and 76-85, 8192 x 28672 62 and 56-65, 2048 x 65536 52 and 40-47
  //   4 rows   bf16 16384 x 8192 67 and 75-86, 16384 x 16384 128 and 94; e4m3 16384 x 16384 70 and 75-86,
  //            5000 x 32768 62 and 41
  //   8 rows   bf16 8192 x 4096 21 and 25, 32000 x 4096 63 and 83, 8192 x 8192 36 and 30, 16384 x 8192 66
  //            and 52; e4m3 19200 x 8192 44 and 62, 16384 x 16384 70 and 53
  //   16 rows  e4m3 16384 x 8192 40 and 32
  // Against the rule stand widths just above a multiple of the GPU's CTAs (9472 x 16384 bf16 70 and 84).
  const long long weight = static_cast<long long>(a.N) * a.K * type_size(a.ab_type);
  if (a.M <= kLinearFewRows) {
    const long long row = static_cast<long long>(a.K) * type_size(a.ab_type);
    const bool tile = weight >= (96LL << 20) && (row >= 56 << 10 || a.M * row >= 128 << 10);
    if (!tile) return linear_few_launch(a, num_sms, st);
    pair_clusters = 0;
  }
  if (a.ab_type == DT_E4M3)
    return a.out_type == DT_F32 ? launch<true, 4>(a, num_sms, pair_clusters, err, st)
                                : launch<true, 2>(a, num_sms, pair_clusters, err, st);
  return a.out_type == DT_F32 ? launch<false, 4>(a, num_sms, pair_clusters, err, st)
                              : launch<false, 2>(a, num_sms, pair_clusters, err, st);
}

}  // namespace laya

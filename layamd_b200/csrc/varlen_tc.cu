// Masked attention of packed sequences on the 5th-generation tensor cores (TMA + tcgen05 + TMEM), head
// dim 64 or 128, shared key heads. A work unit is 128 query rows of one sequence and head (and, with
// splits > 1, one range of the keys); it walks the 64-key chunks that its masks can reach, with the
// running maximum and sum of the softmax.
//
// Persistent, two CTAs per SM (192 threads, 256 TMEM columns each), so that one CTA's products run
// under the other's exponentials; units go round the CTAs, longest tiles first (causal rows near the
// end; by sequence where lengths differ much), heads fastest, so that the units in flight share keys in
// L2. Within a CTA the units run through one pipeline across their borders:
//   warp 0      TMA producer: finds a unit's sequence and its chunks, publishes them through a ring in
//               shared memory, loads Q (2 slots at head dim 64) and the K and V chunks into two rings
//               (4 stages at head dim 64, 2 at 128), running ahead into the next units; a K stage is
//               free when its scores are formed, a V stage when its product is
//   warp 1      MMA issuer: S = Q K^T (128 x 64 fp32, one TMEM buffer, reformed as soon as the softmax
//               warps have copied it) and O += P V (P from TMEM, V MN-major from its TMA tile)
//   warps 2..5  softmax, one query row per thread; a unit's O / l is written after the next unit's first
//               scores, when its last product has landed (O has two buffers at head dim 64; at 128 the
//               next unit's first product waits for the rows)
// Chunks are skipped whole where the window, the prefix or the documents leave nothing; a document's
// chunks are found once per unit from the key ids. Inside a chunk, groups of 32 keys that every row of
// a warp sees skip the masking. The reference maximum is raised only when it grows by more than 2^8, so
// O is rarely rescaled. What bounds it is the chain of a softmax warp's own instructions per chunk (issue
// slots 42 % busy): 850 TFLOP/s at head dim 128 (two sequences of 8192, 1288 us), 490 at 64 (16 sequences
// of 2048, 561 us). Document masks, cap / bias and type are variants of their own because every live
// register near the limit of 168 lengthens that chain (one kernel for all took a quarter longer there).
//
// The softmax is fp32; its weights are rounded to the inputs' type for the product with V (their sum is
// not), the only form in which the tensor core takes them. A row's bits depend on its own visible keys
// and on how lengths and masks cut the work, on nothing else in the tile.
//
// A masked score is replaced, so K may hold anything there. Keys that nobody may see (behind the
// sequence's end, or of a negative document) meet P = 0 in the product, and 0 * NaN would spoil the row:
// their V rows are set to zero in shared memory before the product is issued.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "varlen.cuh"

namespace laya {
namespace {

constexpr int kRows = 128, kKeys = 64, kThreads = 192;
constexpr int kDocWords = 128;  // bitmap of 4096 chunks; chunks past it are not skipped by document
constexpr uint32_t kTmemCols = 256, kTmemS = 0, kTmemO = 64, kTmemP = 192;  // P: two buffers of 32
constexpr uint32_t kAtom = kKeys * 128;                                     // 64 rows x 128 bytes
constexpr int kNoChunk = 0x7fffffff;
// References (in log2 units) from which a row's scores are scaled before the maximum is subtracted.
// Below, both are one FMA: the maximum was rounded and the product is not, so the difference may be off by
// half a unit of the maximum's last place (0.25 here), for all of the row's weights alike. Above, that would
// leave the range of P.
constexpr float kLargeMax = 4194304.f;
// No single document in a chunk, in a warp's rows. Every negative id of the caller's becomes -1 as it is
// read, so that no key can have either value.
constexpr int kMixed = -2, kMixedRows = -3;

constexpr int kRing = 3;  // units published ahead

// The chunks of a unit: [0, end_a) of the prefix and [beg_b, end_b) of the window, cut to [lo, hi).
struct Chunks {
  int end_a, beg_b, lo, hi;
  // The chunk after c; DOCS: that the bitmap `docs` has.
  template <bool DOCS>
  __device__ __forceinline__ int next(int c, const uint32_t* docs) const {
    ++c;
    if constexpr (!DOCS) {
      if (c >= end_a) c = max(c, beg_b);
      return c < hi ? c : kNoChunk;
    } else {
      for (; c < hi; ++c) {
        if (c >= end_a && c < beg_b) {
          c = beg_b;
          if (c >= hi) break;
        }
        if (c >= kDocWords * 32) return c;
        const uint32_t rest = docs[c >> 5] >> (c & 31);
        if (rest & 1) return c;
        if (rest == 0) c |= 31;  // on to the next word
      }
      return kNoChunk;
    }
  }
};

struct Unit {
  Chunks ch;
  int first;       // its first chunk, or kNoChunk
  int q_row, rows; // first query row in q, and how many
  int p0;          // key position of the first
  int k0, lk, prefix;
  int h, sp;       // h < 0: no more units
};

template <int D>
struct VarlenSmem {
  static constexpr int kStages = D == 64 ? 4 : 2, kQSlots = D == 64 ? 2 : 1;
  alignas(1024) uint8_t q[kQSlots][D / 64][kRows * 128];
  alignas(1024) uint8_t k[kStages][D / 64][kAtom];
  alignas(1024) uint8_t v[kStages][D / 64][kAtom];
  uint32_t docs[kRing][kDocWords];
  int row_doc[kRing][kRows];  // the documents of a unit's rows (-1: none); past its last row, that row's
  // per V stage: the chunk's document ids, {the one id that all its keys have or kMixed, whether it
  // holds keys that nobody may see}
  alignas(16) int ids[kStages][kKeys];
  int2 about[kStages];
  Unit units[kRing];
  alignas(8) uint64_t ufull[kRing], uempty[kRing];
  uint64_t qfull[kQSlots], qempty[kQSlots], kfull[kStages], kempty[kStages], vfull[kStages], vempty[kStages];
  uint64_t sfull, sfree, pfull[2], pfree[2], drain;
  uint64_t ofree;  // head dim 128: the one O buffer may take the next unit
  uint32_t tmem;
  int abort;
};
template <int D>
constexpr size_t smem_bytes() { return sizeof(VarlenSmem<D>) + 1024; }

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, err, code));
}

// Tile slots: sequence b owns the slots from cu_q[b] / kRows + b to the next sequence's, enough for its
// tiles wherever it starts. Offsets that run backwards may leave rows out.
__device__ __forceinline__ int first_slot(const VarlenArgs& a, int b) {
  return min(max(a.cu_q[b], 0), a.rows_q) / kRows + b;
}
// The sequence that owns `slot`; a whole warp calls it, 32 candidates a step.
__device__ __forceinline__ int slot_sequence(const VarlenArgs& a, int slot, int lane) {
  int b = 0, n = a.B;  // it is one of b .. b + n - 1
  while (n > 1) {
    const int step = (n + 31) / 32, at = lane * step;
    const uint32_t below = __ballot_sync(0xffffffffu, at < n && first_slot(a, b + at) <= slot);
    const int last = 31 - __clz(below | 1u);
    b += last * step;
    n = min(step, n - last * step);
  }
  return b;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// MOD: scores are capped or biased by distance. BF: bf16, else fp16. DOCS: with document ids.
template <int D, bool MOD, bool BF, bool DOCS>
__global__ void __launch_bounds__(kThreads, 2)
    varlen_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const VarlenArgs a, int nunits, int* err) {
  using Smem = VarlenSmem<D>;
  constexpr int kStages = Smem::kStages, kAtoms = D / 64, kQSlots = Smem::kQSlots;
  constexpr int kType = BF ? DT_BF16 : DT_F16;
  constexpr float kUp = BF ? 0.f : kUpF16;
  extern __shared__ uint8_t smem_raw[];
  Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(smem_u32(&S.ufull[i]), 1);
      mbar_init(smem_u32(&S.uempty[i]), 5);  // the MMA issuer and the four softmax warps
    }
    for (int i = 0; i < kQSlots; ++i) {
      mbar_init(smem_u32(&S.qfull[i]), 1);
      mbar_init(smem_u32(&S.qempty[i]), 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&S.kfull[i]), 1);
      mbar_init(smem_u32(&S.kempty[i]), 1);
      mbar_init(smem_u32(&S.vfull[i]), 1);
      mbar_init(smem_u32(&S.vempty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&S.pfull[i]), 4);
      mbar_init(smem_u32(&S.pfree[i]), 1);
    }
    mbar_init(smem_u32(&S.sfull), 1);
    mbar_init(smem_u32(&S.sfree), 4);
    mbar_init(smem_u32(&S.drain), 1);
    mbar_init(smem_u32(&S.ofree), 4);
    S.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&tq); tma_prefetch_desc(&tk); tma_prefetch_desc(&tv); }
  if (warp == 1) { tmem_alloc(smem_u32(&S.tmem), kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  pdl_wait();
  volatile int* abort = &S.abort;
  if (warp == 0) {
    // ---------------- producer. Counters run over all units: n chunks, nq Q tiles, nu published units.
    const int tiles = (a.max_q + kRows - 1) / kRows;
    int n = 0, nk = 0, nv = 0, nq = 0, nu = 0;
    bool ok = true;
    for (int w = static_cast<int>(blockIdx.x); ok; w += static_cast<int>(gridDim.x)) {
      // unit -> (tile, sequence, head, range), the tile slowest and last first; by slots, the last
      // sequence's last tile first
      Unit u;
      u.h = -1;
      if (w < nunits) {
        int x = w;
        u.sp = x % a.splits;
        x /= a.splits;
        const int h = x % a.Hq;
        x /= a.Hq;
        int b = x % a.B, t0 = (tiles - 1 - x / a.B) * kRows;
        if (a.slots > 0) {
          b = slot_sequence(a, a.slots - 1 - x, lane);
          t0 = (a.slots - 1 - x - first_slot(a, b)) * kRows;
        }
        const Sequence s = sequence(a, b);
        const int lq = min(s.lq, a.max_q);
        if (t0 < 0 || t0 >= lq) continue;
        u.h = h;
        u.rows = min(kRows, lq - t0);
        u.q_row = s.q0 + t0;
        u.p0 = t0 + s.lk - s.lq;
        u.k0 = s.k0;
        u.lk = s.lk;
        u.prefix = s.prefix;
        const int wlo = max(0, u.p0 - a.left), whi = min(s.lk, u.p0 + u.rows - 1 + a.right + 1);
        u.ch.end_a = (s.prefix + kKeys - 1) / kKeys;
        u.ch.beg_b = whi > wlo ? wlo / kKeys : u.ch.end_a;
        const int end_b = whi > wlo ? (whi + kKeys - 1) / kKeys : 0;
        const int lo = u.ch.end_a > 0 ? 0 : u.ch.beg_b;
        const long long all = max(0, max(u.ch.end_a, end_b) - lo);
        u.ch.lo = lo + static_cast<int>(all * u.sp / a.splits);
        u.ch.hi = lo + static_cast<int>(all * (u.sp + 1) / a.splits);
      }
      const int rs = nu % kRing;
      uint32_t* map = S.docs[rs];
      if (nu >= kRing && !warp_wait(smem_u32(&S.uempty[rs]), ((nu / kRing) - 1) & 1, abort, err, kErrAttnLoad)) break;
      if (DOCS && u.h >= 0) {
        // the rows' smallest and largest document, then the chunks that hold a key in that range
        int lo = 0x7fffffff, hi = -1;
#pragma unroll
        for (int i = 0; i < kRows; i += 32) {
          const int d = max(a.doc_q[u.q_row + min(lane + i, u.rows - 1)], -1);
          S.row_doc[rs][lane + i] = d;
          lo = min(lo, d < 0 ? 0x7fffffff : d);
          hi = max(hi, d);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        const int* ids = a.doc_k + u.k0;
        const int end = min(u.ch.hi, kDocWords * 32);
        for (int c0 = u.ch.lo & ~31; c0 < end; c0 += 32) {
          uint32_t word = 0;
          const int c1 = min(c0 + 32, end);
#pragma unroll 8
          for (int c = max(c0, u.ch.lo); c < c1; ++c) {
            const int k = c * kKeys + lane;
            const int x = k < u.lk ? ids[k] : -1, y = k + 32 < u.lk ? ids[k + 32] : -1;
            const bool hit = (x >= lo && x <= hi && x >= 0) || (y >= lo && y <= hi && y >= 0);
            if (__any_sync(0xffffffffu, hit)) word |= 1u << (c & 31);
          }
          if (lane == 0) map[c0 >> 5] = word;
        }
      }
      __syncwarp();
      int c = kNoChunk;
      if (u.h >= 0) c = u.ch.next<DOCS>(u.ch.lo - 1, map);
      u.first = c;
      if (lane == 0) {
        S.units[rs] = u;
        mbar_arrive(smem_u32(&S.ufull[rs]));
      }
      __syncwarp();
      ++nu;
      if (u.h < 0) break;
      if (c == kNoChunk) continue;
      const int hk = u.h / (a.Hq / a.Hkv);
      if (lane == 0) {
        const int qs = nq % kQSlots;
        ok = nq < kQSlots || mbar_wait(smem_u32(&S.qempty[qs]), ((nq / kQSlots) - 1) & 1, abort, err, kErrAttnLoad);
        if (ok) {
          mbar_expect_tx(smem_u32(&S.qfull[qs]), kRows * D * 2);
#pragma unroll
          for (int d = 0; d < kAtoms; ++d)
            tma_load_3d(smem_u32(S.q[qs][d]), &tq, d * 64, u.h, u.q_row, smem_u32(&S.qfull[qs]));
          ++nq;
        }
      }
      auto load_k = [&]() -> bool {  // one lane
        const int st = n % kStages;
        if (n >= kStages && !mbar_wait(smem_u32(&S.kempty[st]), ((n / kStages) - 1) & 1, abort, err, kErrAttnLoad))
          return false;
        mbar_expect_tx(smem_u32(&S.kfull[st]), kAtoms * kAtom);
#pragma unroll
        for (int d = 0; d < kAtoms; ++d)
          tma_load_3d(smem_u32(S.k[st][d]), &tk, d * 64, hk, u.k0 + c * kKeys, smem_u32(&S.kfull[st]));
        ++nk;
        return true;
      };
      auto v_free = [&]() -> bool {
        return n < kStages || mbar_wait(smem_u32(&S.vempty[n % kStages]), ((n / kStages) - 1) & 1, abort, err, kErrAttnLoad);
      };
      auto load_v = [&]() {  // one lane
        const int st = n % kStages;
        mbar_expect_tx(smem_u32(&S.vfull[st]), kAtoms * kAtom);
#pragma unroll
        for (int d = 0; d < kAtoms; ++d)
          tma_load_3d(smem_u32(S.v[st][d]), &tv, d * 64, hk, u.k0 + c * kKeys, smem_u32(&S.vfull[st]));
        ++nv;
      };
      if constexpr (!DOCS) {
        if (lane == 0) {
          for (; ok && c != kNoChunk; c = u.ch.next<false>(c, map), ++n) {
            ok = load_k() && v_free();
            if (ok) load_v();
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      } else {
        // the chunk's ids and what they have in common go along with V, a chunk ahead in registers
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
        int id[2] = {-1, -1};
        auto load_ids = [&](int chunk) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int k = chunk * kKeys + 32 * g + lane;
            id[g] = k < u.lk ? max(a.doc_k[u.k0 + k], -1) : -1;
          }
        };
        load_ids(c);
        while (ok && c != kNoChunk) {
          if (lane == 0) ok = load_k();
          ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
          if (!ok || !__all_sync(0xffffffffu, v_free())) { ok = false; break; }
          const int st = n % kStages;
          const int id0 = __shfl_sync(0xffffffffu, id[0], 0);
          const bool one = __all_sync(0xffffffffu, id[0] == id0 && id[1] == id0);
          const bool dead = __any_sync(0xffffffffu, id[0] < 0 || id[1] < 0);
          S.ids[st][lane] = id[0];
          S.ids[st][lane + 32] = id[1];
          if (lane == 0) S.about[st] = make_int2(one ? id0 : kMixed, dead ? 1 : 0);
          __syncwarp();
          if (lane == 0) load_v();
          c = u.ch.next<true>(c, map);
          ++n;
          if (c != kNoChunk) load_ids(c);
        }
      }
    }
    if (lane == 0 && *abort) {  // the loads in flight land before the CTA can exit
      const long long t = clock64();
      auto landed = [&](uint64_t* bar, int issued) {
        if (issued <= 0) return;
        while (!mbar_try(smem_u32(bar), (issued - 1) & 1))
          if (clock64() - t > kWaitBudgetCycles) { atomicCAS(err, 0, kErrGemmDrain); return; }
      };
      for (int i = 0; i < kQSlots; ++i) landed(&S.qfull[i], (nq - i + kQSlots - 1) / kQSlots);
      for (int i = 0; i < kStages; ++i) {
        landed(&S.kfull[i], (nk - i + kStages - 1) / kStages);
        landed(&S.vfull[i], (nv - i + kStages - 1) / kStages);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_of(BF ? 1u : 0u, kRows, kKeys), idesc_pv = idesc_of(BF ? 1u : 0u, kRows, 64) | (1u << 16);
      bool issued = false, ok = true;
      int n = 0, nq = 0, nu = 0;
      int pend = -1;           // chunk whose product with V is still to be issued
      bool pend_first = false; // it starts its unit's O
      int pend_unit = 0;
      uint32_t pend_o = kTmemO;
      // O += P V of the pending chunk; V's atoms of 64 columns are separate products
      auto pv = [&]() -> bool {
        const int st = pend % kStages, pb = pend & 1;
        if (!mbar_wait(smem_u32(&S.pfull[pb]), (pend >> 1) & 1, abort, err, kErrAttnMma)) return false;
        if (!mbar_wait(smem_u32(&S.vfull[st]), (pend / kStages) & 1, abort, err, kErrAttnMma)) return false;
        if (D == 128 && pend_first && !mbar_wait(smem_u32(&S.ofree), pend_unit & 1, abort, err, kErrAttnMma)) return false;
        tc_fence_after();
#pragma unroll
        for (int d = 0; d < kAtoms; ++d)
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)  // 16 keys: 8 packed columns of P
            umma_bf16_ts(tmem + pend_o + 64 * d, tmem + kTmemP + pb * 32 + kk * 8,
                         sdesc_mn128(smem_u32(S.v[st][d]) + kk * 2048), idesc_pv, (!pend_first || kk > 0) ? 1u : 0u);
        umma_commit(smem_u32(&S.pfree[pb]));
        umma_commit(smem_u32(&S.vempty[st]));
        pend = -1;
        return true;
      };
      for (;; ++nu) {
        const int rs = nu % kRing;
        if (!mbar_wait(smem_u32(&S.ufull[rs]), (nu / kRing) & 1, abort, err, kErrAttnMma)) { ok = false; break; }
        const Unit& u = S.units[rs];
        if (u.h < 0) break;
        int c = u.first;
        if (c != kNoChunk) {
          const int qs = nq % kQSlots;
          if (!mbar_wait(smem_u32(&S.qfull[qs]), (nq / kQSlots) & 1, abort, err, kErrAttnMma)) { ok = false; break; }
          for (; c != kNoChunk; ++n) {
            const int st = n % kStages;
            if (!mbar_wait(smem_u32(&S.kfull[st]), (n / kStages) & 1, abort, err, kErrAttnMma)) { ok = false; break; }
            // the softmax warps have copied the previous scores
            if (n >= 1 && !mbar_wait(smem_u32(&S.sfree), (n - 1) & 1, abort, err, kErrAttnMma)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_bf16(tmem + kTmemS, sdesc_k128(smem_u32(S.q[qs][kk / 4]) + (kk % 4) * 32),
                        sdesc_k128(smem_u32(S.k[st][kk / 4]) + (kk % 4) * 32), idesc, kk > 0 ? 1u : 0u);
            issued = true;
            umma_commit(smem_u32(&S.sfull));
            umma_commit(smem_u32(&S.kempty[st]));
            const bool is_first = c == u.first;
            c = u.ch.next<DOCS>(c, S.docs[rs]);
            if (c == kNoChunk) umma_commit(smem_u32(&S.qempty[qs]));
            if (pend >= 0 && !pv()) { ok = false; break; }
            pend = n;
            pend_first = is_first;
            pend_unit = nq;
            pend_o = kTmemO + (D == 64 ? static_cast<uint32_t>(nq & 1) * 64u : 0u);
          }
          if (!ok) break;
          ++nq;
        }
        // a unit without chunks: the softmax warps write the previous one out first
        if (c == kNoChunk && u.first == kNoChunk && pend >= 0 && !pv()) { ok = false; break; }
        mbar_arrive(smem_u32(&S.uempty[rs]));
      }
      if (ok && pend >= 0) pv();
      if (*abort && issued) {  // the products already issued finish before TMEM is released
        umma_commit(smem_u32(&S.drain));
        const long long t = clock64();
        while (!mbar_try(smem_u32(&S.drain), 0))
          if (clock64() - t > kWaitBudgetCycles) { atomicCAS(err, 0, kErrGemmDrain); break; }
      }
    }
  } else {
    // ---------------- softmax: scores stay in units of q.k until the exponential scales them
    const int qw = warp & 3, row = qw * 32 + lane;  // this thread's row; warp w owns TMEM lanes 32 (w % 4) ..
    const uint32_t tl = tmem + (static_cast<uint32_t>(qw * 32) << 16);
    const float cs = a.caps.to_log2;
    int n = 0, nq = 0, nu = 0;
    bool ok = true;

    // One thread's output row, written once its unit's last product has landed. The loop below has one
    // place that writes rows: the kernel's code size counts (instruction fetches stall the softmax).
    struct Row {
      bool on;          // a unit's row is waiting
      bool zero;        // nothing is seen: no product to wait for
      int chunk;        // its last chunk
      uint32_t o;       // its TMEM columns
      long long at;     // row in q; -1: none
      int h, sp;
      float inv, lse2;
    } wait{false, false, 0, 0, 0, 0, 0, 0.f, 0.f};
    auto flush = [&]() -> bool {
      if (!wait.on) return true;
      wait.on = false;
      if (!wait.zero) {
        if (!warp_wait(smem_u32(&S.pfree[wait.chunk & 1]), (wait.chunk >> 1) & 1, abort, err, kErrAttnSoftmax))
          return false;
        tc_fence_after();
      }
      const long long part = (static_cast<long long>(wait.sp) * a.rows_q + wait.at) * a.Hq + wait.h;
      if (wait.at >= 0) {
        if (a.splits > 1) a.part_l[part] = wait.lse2;
        else if (a.lse) a.lse[wait.at * a.Hq + wait.h] = wait.lse2 * kLn2;
      }
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        float o[32];
        __syncwarp();
        if (!wait.zero) tmem_ld32(tl + wait.o + 32 * d, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = wait.zero ? 0.f : o[i] * wait.inv;
        if (wait.at >= 0) {
          if (a.splits == 1) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + wait.at * a.ldo + wait.h * D) + 4 * d;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              dst[j] = make_uint4(pack_pair(o[8 * j], o[8 * j + 1], kType), pack_pair(o[8 * j + 2], o[8 * j + 3], kType),
                                  pack_pair(o[8 * j + 4], o[8 * j + 5], kType), pack_pair(o[8 * j + 6], o[8 * j + 7], kType));
          } else {
            float4* dst = reinterpret_cast<float4*>(a.part_o + part * D + 32 * d);
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      return true;
    };

    for (; ok; ++nu) {
      const int rs = nu % kRing;
      if (!warp_wait(smem_u32(&S.ufull[rs]), (nu / kRing) & 1, abort, err, kErrAttnSoftmax)) { ok = false; break; }
      const Unit& u = S.units[rs];
      const bool end = u.h < 0;
      const int rows = u.rows, lk = u.lk, h = u.h;
      const int p = u.p0 + row;               // this row's key position
      const int pw = u.p0 + qw * 32, pz = pw + 31;  // the warp's first and last
      const long long at = !end && row < rows ? static_cast<long long>(u.q_row) + row : -1;
      Sequence s;
      s.lk = lk;
      s.prefix = u.prefix;
      const int qdoc = DOCS ? S.row_doc[rs][row] : -1;
      const bool idle = qw * 32 >= rows;  // none of the warp's rows is one
      const float slope = MOD && a.slopes && !end ? a.slopes[h] / a.scale * a.caps.unit : 0.f;
      const uint32_t* map = S.docs[rs];
      const Chunks ch = u.ch;
      const uint32_t oc = kTmemO + (D == 64 ? static_cast<uint32_t>(nq & 1) * 64u : 0u);
      int c = end ? kNoChunk : u.first;
      const bool none_seen = c == kNoChunk;  // nothing is seen by any of its rows, or the end
      float m_used = -INFINITY;
      bool large = false;  // |m_used| >= kLargeMax
      float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
      int wdoc = kMixedRows;  // the document of all the warp's rows
      if constexpr (DOCS) {
        const int d0 = __shfl_sync(0xffffffffu, qdoc, 0);
        if (__all_sync(0xffffffffu, qdoc == d0) && d0 >= 0) wdoc = d0;
      }
      for (bool first = true;; first = false) {
        if (!none_seen) {
          const int k0 = c * kKeys, pb = n & 1, st = n % kStages;
          // per 32-key group, warp-uniform: 0 nobody sees a key, 1 some are masked, 2 all are seen
          int gk[2];
          bool dead = k0 + kKeys > lk;  // the chunk holds keys that nobody may see
          bool same = true, other = false;  // the chunk is all of the rows' document, or of another one
          if constexpr (DOCS) {
            if (!warp_wait(smem_u32(&S.vfull[st]), (n / kStages) & 1, abort, err, kErrAttnSoftmax)) { ok = false; break; }
            const int2 about = S.about[st];
            same = about.x == wdoc;
            dead = dead || about.y != 0;
            other = about.x != kMixed && wdoc != kMixedRows && !same;
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int k_lo = k0 + 32 * g, k_hi = k_lo + 31;
            const bool none = idle || other || k_lo >= lk || ((k_hi < pw - a.left || k_lo > pz + a.right) && k_lo >= s.prefix);
            const bool all = k_hi < lk && ((k_lo >= pz - a.left && k_hi <= pw + a.right) || k_hi < s.prefix);
            gk[g] = none ? 0 : all ? 2 : 1;
            if (DOCS && !same && gk[g] == 2) gk[g] = 1;
          }
          const int c_next = ch.next<DOCS>(c, map);
          if (!warp_wait(smem_u32(&S.sfull), n & 1, abort, err, kErrAttnSoftmax)) { ok = false; break; }
          tc_fence_after();
          float x[64];
          tmem_ld64(tl + kTmemS, x);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&S.sfree));  // S may take the next chunk

          if constexpr (MOD) {
            if (a.cap > 0.f) {
              float top = 0.f;
#pragma unroll
              for (int i = 0; i < 64; i += 2) top = max3(top, fabsf(x[i]), fabsf(x[i + 1]));
              // The odd polynomial of tanh_small with the cap in its coefficients, two lanes an instruction,
              // where the score is small; where it is not cap (1 - 2 / (1 + e^(2u))). Each score takes its form
              // by itself, so that a row's bits depend on nothing else in the tile; a warp whose scores are
              // all small skips the second form.
              const float2 c1 = make_float2(a.caps.k1, a.caps.k1), c2 = make_float2(a.caps.k2, a.caps.k2),
                           c3 = make_float2(a.caps.k3, a.caps.k3), one = make_float2(1.f, 1.f);
              auto small2 = [&](float2 v) {
                const float2 z = __fmul2_rn(v, v);
                return __fmul2_rn(v, __ffma2_rn(z, __ffma2_rn(z, __ffma2_rn(z, c3, c2), c1), one));
              };
              if (__all_sync(0xffffffffu, top < a.caps.all_small)) {
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                  const float2 r = small2(make_float2(x[i], x[i + 1]));
                  x[i] = r.x;
                  x[i + 1] = r.y;
                }
              } else {
                const float2 unit = make_float2(a.caps.unit, a.caps.unit),
                             ke2 = make_float2(a.caps.to_2u, a.caps.to_2u), out = make_float2(a.caps.out, a.caps.out),
                             back = make_float2(-2.f * a.caps.out, -2.f * a.caps.out);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                  const float2 v = __fmul2_rn(make_float2(x[i], x[i + 1]), unit);  // exact
                  const float2 u = __fmul2_rn(v, ke2), r = small2(v);
                  const float2 d = __fadd2_rn(make_float2(exp2_fast(u.x), exp2_fast(u.y)), one);
                  const float2 t = __ffma2_rn(make_float2(rcp_fast(d.x), rcp_fast(d.y)), back, out);
                  x[i] = pick_below(fabsf(v.x), a.caps.small, r.x, t.x);
                  x[i + 1] = pick_below(fabsf(v.y), a.caps.small, r.y, t.y);
                }
              }
            }
            if (a.slopes) {
              const float away = static_cast<float>(p - k0);
#pragma unroll
              for (int i = 0; i < 64; ++i) x[i] = fmaf(-slope, fabsf(away - static_cast<float>(i)), x[i]);
            }
          }
          float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (__builtin_expect(gk[g] == 1, 0)) {
              uint32_t see = window_bits(a, s, p, k0 + 32 * g);
              if (DOCS && !same) {
                const int doc = qdoc < 0 ? kMixedRows : qdoc;
                uint32_t mine = 0;
#pragma unroll 1
                for (int i = 28; i >= 0; i -= 4) {
                  const int4 id = *reinterpret_cast<const int4*>(&S.ids[st][32 * g + i]);
                  mine = mine << 4 | (id.x == doc ? 1u : 0u) | (id.y == doc ? 2u : 0u) | (id.z == doc ? 4u : 0u) |
                         (id.w == doc ? 8u : 0u);
                }
                see &= mine;
              }
              if (__any_sync(0xffffffffu, see != ~0u)) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(see >> i & 1)) x[32 * g + i] = -INFINITY;
              }
            }
            if (gk[g] != 0) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) mq[(i >> 1) & 3] = max3(mq[(i >> 1) & 3], x[32 * g + i], x[32 * g + i + 1]);
            }
          }
          const float mx = __fmul_rn(max3(mq[0], mq[1], fmaxf(mq[2], mq[3])), cs);
          const bool resc = mx - m_used > kGrow + kUp;
          const bool resc_o = resc && m_used != -INFINITY;  // O is exactly 0 before a row's first visible key
          float alpha = 1.f;
          float mul = cs;
          if (resc || large) {
            if (resc) {
              const float m_new = mx - kUp;
              alpha = exp2_fast(m_used - m_new);
              la.x *= alpha; la.y *= alpha; lb.x *= alpha; lb.y *= alpha;
              m_used = m_new;
              large = fabsf(m_new) >= kLargeMax;
            }
            if (large) {
              mul = 1.f;
#pragma unroll
              for (int i = 0; i < 64; ++i) x[i] = __fmul_rn(x[i], cs);  // rounded as mx is
            }
          }
          const float msub = m_used == -INFINITY ? 0.f : m_used;
          const float2 mul2 = make_float2(mul, mul), nm2 = make_float2(-msub, -msub);
          uint32_t pk[32];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (gk[g] == 0) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[16 * g + i] = 0u;
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 e = __ffma2_rn(make_float2(x[32 * g + 2 * i], x[32 * g + 2 * i + 1]), mul2, nm2);
                const float2 pp = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                if (i & 1) lb = __fadd2_rn(lb, pp); else la = __fadd2_rn(la, pp);
                pk[16 * g + i] = pack_pair(pp.x, pp.y, kType);
              }
            }
          }
          if (__builtin_expect(dead, 0)) {
            // V rows of keys that nobody may see: zero, whatever they hold (all four warps, 16 rows each)
            if (!warp_wait(smem_u32(&S.vfull[st]), (n / kStages) & 1, abort, err, kErrAttnSoftmax)) { ok = false; break; }
            const int r0 = 16 * qw + (lane >> 1);
            if (k0 + r0 >= lk || (DOCS && S.ids[st][r0] < 0)) {
#pragma unroll
              for (int d = 0; d < kAtoms; ++d) {
                uint4* z = reinterpret_cast<uint4*>(S.v[st][d] + r0 * 128 + (lane & 1) * 64);
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = make_uint4(0u, 0u, 0u, 0u);
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the tensor core reads V
          }
          // O may be rescaled once the product in flight has landed
          if (__builtin_expect(!first && __any_sync(0xffffffffu, resc_o), 0)) {
            if (!warp_wait(smem_u32(&S.pfree[(n - 1) & 1]), ((n - 1) >> 1) & 1, abort, err, kErrAttnSoftmax)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
              float o[32];
              tmem_ld32(tl + oc + 32 * d, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= alpha;
              tmem_st32(tl + oc + 32 * d, o);
            }
          }
          if (n >= 2 && !warp_wait(smem_u32(&S.pfree[pb]), ((n >> 1) - 1) & 1, abort, err, kErrAttnSoftmax)) {
            ok = false;
            break;
          }
          tc_fence_after();
          tmem_st32u(tl + kTmemP + pb * 32, pk);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&S.pfull[pb]));
          c = c_next;
          ++n;
        }
        if (first) {  // the previous unit's rows
          if (!flush()) { ok = false; break; }
          if (D == 128 && !none_seen && lane == 0) mbar_arrive(smem_u32(&S.ofree));
        }
        if (c == kNoChunk) break;
      }
      if (!ok || end) break;
      const float l = (la.x + la.y) + (lb.x + lb.y);
      // a row that sees nothing is 0; NaN stays NaN
      wait = Row{true, none_seen, n - 1, oc, at, h, u.sp, l > 0.f ? 1.f / l : l, l == 0.f ? -INFINITY : m_used + log2f(l)};
      if (!none_seen) ++nq;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&S.uempty[rs]));
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partial rows: out = sum_s 2^(lse_s - lse) o_s. One warp per query row and head.
template <int D>
__global__ void __launch_bounds__(256) varlen_join_kernel(const VarlenArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const Sequence s = sequence(a, blockIdx.y);
  const int i = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int qi = i / a.Hq, h = i - qi * a.Hq;
  if (qi >= min(s.lq, a.max_q)) return;
  const long long r = static_cast<long long>(s.q0) + qi, plane = static_cast<long long>(a.rows_q) * a.Hq;
  const long long at = r * a.Hq + h;
  const float l = lane < a.splits ? a.part_l[lane * plane + at] : -INFINITY;
  float m = l;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float w = l == -INFINITY ? 0.f : exp2_fast(l - m);  // a NaN stays one
  const float sum = warp_sum(w);
  constexpr int kPer = D / 32;
  float o[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) o[j] = 0.f;
  for (int sp = 0; sp < a.splits; ++sp) {
    const float ws = __shfl_sync(0xffffffffu, w, sp);
    if (ws == 0.f) continue;
    const float* src = a.part_o + (sp * plane + at) * D + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) o[j] = fmaf(ws, src[j], o[j]);
  }
  const float inv = sum > 0.f ? 1.f / sum : sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + r * a.ldo + h * D + lane * kPer);
#pragma unroll
  for (int j = 0; j < kPer / 2; ++j) dst[j] = pack_pair(o[2 * j] * inv, o[2 * j + 1] * inv, a.type);
  if (lane == 0 && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
}

// (tile, sequence) pairs of a call. Every tile up to max_q of every sequence, or, where a third of those or
// more are sure to be empty (one long sequence among short ones, or a max_q far above them all), the tile
// slots, of which a sequence leaves one at most. The producer warps walk what is empty, one pair in about
// 0.3 us. Tiles against slots at head dim 64, with pairs per slot: 16 causal sequences of 2048 (0.94) 314 and
// 332 us, 192 of 32 to 512 (1.2) 277 and 283; 64 causal of 32 to 2048 (1.9) 584 and 484; one of 8192 among
// 127 of 100, 64 heads (28) 1970 and 1187; 512 of 128 with max_q 65,536 (256) 4315 and 126.
struct Pairs {
  long long n;
  bool slots;
};
Pairs pairs_of(int B, int rows_q, int max_q) {
  const long long all = (max_q + (kRows - 1LL)) / kRows * B, slots = rows_q / kRows + (long long)B;
  return 2 * all > 3 * slots ? Pairs{slots, true} : Pairs{all, false};
}

// The constants of the softmax, from the caller's scale and cap.
void set_caps(VarlenArgs* a) {
  const bool cap = a->cap > 0.f;
  const float r = cap ? a->scale / a->cap : 1.f;
  const float unit = cap && (r < 0x1p-16f || r > 0x1p16f) ? std::ldexp(1.f, std::ilogb(r)) : 1.f;
  const float in = r / unit, z1 = in * in, out = cap ? a->cap / a->scale * unit : 0.f;
  a->caps = {unit,
             a->scale * kLog2e / unit,
             kTanhSmall / in,
             unit == 1.f ? kTanhSmall / in : -1.f,
             -z1 / 3.f,
             z1 * z1 * (2.f / 15.f),
             z1 * z1 * z1 * (-17.f / 315.f),
             in * (2.f * kLog2e),
             out};
}

template <int D>
cudaError_t launch(const VarlenArgs& in, int num_sms, int* err, cudaStream_t st) {
  VarlenArgs a = in;
  CUtensorMap tq, tk, tv;
  auto map = [&](CUtensorMap* m, const void* base, int heads, int rows, long long ld, int box) {
    return make_rows_map(m, base, a.type, D, static_cast<uint64_t>(heads), static_cast<uint64_t>(rows), D,
                         static_cast<uint64_t>(ld), static_cast<uint32_t>(box));
  };
  if (!map(&tq, a.q, a.Hq, a.rows_q, a.ldq, kRows) || !map(&tk, a.k, a.Hkv, std::max(1, a.rows_k), a.ldk, kKeys) ||
      !map(&tv, a.v, a.Hkv, std::max(1, a.rows_k), a.ldv, kKeys))
    return cudaErrorInvalidValue;
  set_caps(&a);
  const Pairs pairs = pairs_of(a.B, a.rows_q, a.max_q);
  a.slots = pairs.slots ? static_cast<int>(pairs.n) : 0;
  const long long units = pairs.n * a.Hq * a.splits;
  if (units > kVarlenMaxUnits) return cudaErrorInvalidValue;
  const dim3 g(static_cast<unsigned>(std::min<long long>(units, 2LL * num_sms)));
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, g, dim3(kThreads), smem_bytes<D>(), st, tq, tk, tv, a, static_cast<int>(units), err);
  };
  const int which = (a.cap > 0.f || a.slopes ? 4 : 0) + (a.type == DT_BF16 ? 2 : 0) + (a.doc_k ? 1 : 0);
  switch (which) {
    case 0: return go(varlen_tc_kernel<D, false, false, false>);
    case 1: return go(varlen_tc_kernel<D, false, false, true>);
    case 2: return go(varlen_tc_kernel<D, false, true, false>);
    case 3: return go(varlen_tc_kernel<D, false, true, true>);
    case 4: return go(varlen_tc_kernel<D, true, false, false>);
    case 5: return go(varlen_tc_kernel<D, true, false, true>);
    case 6: return go(varlen_tc_kernel<D, true, true, false>);
    default: return go(varlen_tc_kernel<D, true, true, true>);
  }
}

template <int D, bool MOD, bool BF>
cudaError_t prepare_one() {
  const int bytes = static_cast<int>(smem_bytes<D>());
  const cudaError_t e =
      cudaFuncSetAttribute(varlen_tc_kernel<D, MOD, BF, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(varlen_tc_kernel<D, MOD, BF, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <int D>
cudaError_t prepare() {
  for (cudaError_t e : {prepare_one<D, false, false>(), prepare_one<D, false, true>(), prepare_one<D, true, false>(),
                        prepare_one<D, true, true>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace

cudaError_t varlen_prepare_device() {
  for (cudaError_t e : {prepare<64>(), prepare<128>(), varlen_few_prepare_device()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

long long varlen_units(int B, int rows_q, int max_q, int Hq) { return pairs_of(B, rows_q, max_q).n * Hq; }

int varlen_splits(int B, int rows_q, int max_q, int max_k, int Hq, int Hkv, int num_sms) {
  // Enough CTAs for two per SM, each with 4 chunks (or 512 keys of the kernel for few queries) to walk.
  const bool few = varlen_few_rows(max_q);
  const long long units = few ? (long long)B * Hkv * ((max_q * (Hq / Hkv) + 15) / 16)
                              : varlen_units(B, rows_q, max_q, Hq);
  const long long most = std::max<long long>(1, max_k / (few ? 512 : 4 * kKeys));
  const long long want = units > 0 ? (few ? 6LL : 2LL) * num_sms / units : 1;
  return static_cast<int>(std::max<long long>(1, std::min<long long>({want, most, kVarlenMaxSplits})));
}

cudaError_t varlen_launch(const VarlenArgs& a, int num_sms, int* err, cudaStream_t st) {
  cudaError_t e = varlen_few_rows(a.max_q) ? varlen_few_launch(a, err, st)
                  : a.D == 64                           ? launch<64>(a, num_sms, err, st)
                                                        : launch<128>(a, num_sms, err, st);
  if (e != cudaSuccess || a.splits == 1) return e;
  const long long items = (long long)a.max_q * a.Hq;
  const dim3 g(static_cast<unsigned>((items + 7) / 8), static_cast<unsigned>(a.B));
  return a.D == 64 ? launch_pdl(varlen_join_kernel<64>, g, dim3(256), 0, st, a)
                   : launch_pdl(varlen_join_kernel<128>, g, dim3(256), 0, st, a);
}

}  // namespace laya

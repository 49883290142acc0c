// Masked attention for few query rows (single tokens over long keys): every key and value is read once
// and nearly nothing is computed, so the bound is HBM. A CTA takes up to 16 query rows that share a key
// head (query heads of the group times query tokens) and a range of the keys; its 8 warps take 16 keys
// each in turn.
//
// Operands go from memory straight into the registers of mma.sync m16n8k16. Its inner dimension may run
// in any order, so in Q K^T each thread's 16 bytes of a key row take the places of the instruction's
// K values; in P V the 8 output columns of one instruction are 8 dimensions that lie 8 apart, so that
// a thread's 16 bytes of a value row serve 8 instructions. No shared memory in the loop: the next keys
// load while the softmax and P V run, the next values while Q K^T does. The warps' partial rows (each
// with its own running maximum and sum) are joined through shared memory in warp order.
//
// Masked scores are replaced; values of keys that nobody may see are not read (zero), so that nothing
// they hold reaches a row.
#include "varlen.cuh"

namespace laya {
namespace {

constexpr int kWarps = 8, kStep = 16 * kWarps;  // keys of one round of the warps

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

template <int D>
struct FewSmem {
  float o[kWarps][16][D];
  float m[kWarps][16], l[kWarps][16];
};

template <int D, bool MOD>
__global__ void __launch_bounds__(32 * kWarps, D == 64 ? 2 : 1) varlen_few_kernel(const VarlenArgs a) {
  constexpr int kM = D / 32, kH = D / 64;
  extern __shared__ uint8_t smem_raw[];
  FewSmem<D>& S = *reinterpret_cast<FewSmem<D>*>(smem_raw);
  pdl_trigger();
  pdl_wait();
  const int G = a.Hq / a.Hkv, row_tiles = (a.max_q * G + 15) / 16;
  int u = static_cast<int>(blockIdx.x);
  const int rt = u % row_tiles;
  u /= row_tiles;
  const int sp = u % a.splits;
  u /= a.splits;
  const int hk = u % a.Hkv;
  const Sequence s = sequence(a, u / a.Hkv);
  const int nrows = min(s.lq, a.max_q) * G;  // (token, head of the group) rows of this key head
  if (rt * 16 >= nrows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool bf = a.type == DT_BF16;

  // this thread's rows: g and g + 8 of the tile
  int pos[2], head[2], qdoc[2];
  uint4 q[2][kM];
  float slope[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int R = rt * 16 + g + 8 * r;
    const bool on = R < nrows;
    const int qi = on ? R / G : 0;
    head[r] = hk * G + (on ? R - qi * G : 0);
    pos[r] = qi + s.lk - s.lq;
    qdoc[r] = a.doc_q ? (on ? a.doc_q[s.q0 + qi] : -1) : 0;
    slope[r] = MOD && a.slopes ? a.slopes[head[r]] * kLog2e : 0.f;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                      (long long)(s.q0 + qi) * a.ldq + head[r] * D);
#pragma unroll
    for (int m = 0; m < kM; ++m) q[r][m] = on ? __ldg(src + 4 * m + t) : make_uint4(0u, 0u, 0u, 0u);
  }

  // rounds of 128 keys that the masks can reach: the prefix's, then the window's
  const int p_first = (rt * 16) / G + s.lk - s.lq, p_last = min(rt * 16 + 15, nrows - 1) / G + s.lk - s.lq;
  const int wlo = max(0, p_first - a.left), whi = min(s.lk, p_last + a.right + 1);
  const int end_a = (s.prefix + kStep - 1) / kStep;
  const int beg_b = max(end_a, whi > wlo ? wlo / kStep : 0);
  const int end_b = whi > wlo ? (whi + kStep - 1) / kStep : 0;
  const long long rounds = end_a + max(0, end_b - beg_b);
  const int j0 = static_cast<int>(rounds * sp / a.splits), j1 = static_cast<int>(rounds * (sp + 1) / a.splits);
  auto key_of = [&](int j) { return (j < end_a ? j : j - end_a + beg_b) * kStep + warp * 16; };

  int doc_lo = 0, doc_hi = 0;
  if (a.doc_k) {
    const int lo0 = qdoc[0] < 0 ? 0x7fffffff : qdoc[0], lo1 = qdoc[1] < 0 ? 0x7fffffff : qdoc[1];
    doc_lo = __reduce_min_sync(0xffffffffu, min(lo0, lo1));
    doc_hi = __reduce_max_sync(0xffffffffu, max(qdoc[0], qdoc[1]));
  }
  // The rounds of the 32 from `base` on that hold a key of a document in [doc_lo, doc_hi] for this warp.
  auto active = [&](int base) -> uint32_t {
    const int j = base + lane;
    bool hit = j < j1;
    if (a.doc_k && hit) {
      const int kb = key_of(j);
      hit = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int id = kb + i < s.lk ? __ldg(a.doc_k + s.k0 + kb + i) : -1;
        hit = hit || (id >= 0 && id >= doc_lo && id <= doc_hi);
      }
    }
    return __ballot_sync(0xffffffffu, hit);
  };
  int base = j0;
  uint32_t todo = active(base);
  auto next_round = [&]() -> int {  // -1 at the end
    while (todo == 0) {
      base += 32;
      if (base >= j1) return -1;
      todo = active(base);
    }
    const int i = __ffs(todo) - 1;
    todo &= todo - 1;
    return base + i;
  };

  const char* kp = static_cast<const char*>(a.k) + ((long long)s.k0 * a.ldk + hk * D) * 2;
  const char* vp = static_cast<const char*>(a.v) + ((long long)s.k0 * a.ldv + hk * D) * 2;
  uint4 kr[2][kM], vr[4][kH];
  int kid = 0, kid_next = 0;  // document of key kb + lane % 16
  auto load_k = [&](int kb) {
    if (a.doc_k) kid_next = kb + (lane & 15) < s.lk ? __ldg(a.doc_k + s.k0 + kb + (lane & 15)) : -1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = kb + 8 * i + g;
      const uint4* src = reinterpret_cast<const uint4*>(kp + (long long)key * a.ldk * 2);
#pragma unroll
      for (int m = 0; m < kM; ++m) kr[i][m] = key < s.lk ? __ldcs(src + 4 * m + t) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto load_v = [&](int kb, int id) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int off = 2 * t + (r & 1) + 8 * (r >> 1), key = kb + off;
      bool on = key < s.lk;
      if (a.doc_k) {  // the whole warp
        const int doc = __shfl_sync(0xffffffffu, id, off);
        on = on && doc >= 0;
      }
      const uint4* src = reinterpret_cast<const uint4*>(vp + (long long)key * a.ldv * 2);
#pragma unroll
      for (int h = 0; h < kH; ++h) vr[r][h] = on ? __ldcs(src + 8 * h + g) : make_uint4(0u, 0u, 0u, 0u);
    }
  };

  const float cs = a.scale * kLog2e;
  const float cap_in = MOD && a.cap > 0.f ? a.scale / a.cap : 0.f, cap_out = a.cap * kLog2e;
  float o[kH][8][4];
#pragma unroll
  for (int h = 0; h < kH; ++h)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[h][j][e] = 0.f;
  float mr[2] = {-INFINITY, -INFINITY}, lr[2] = {0.f, 0.f};

  int j = j0 < j1 ? next_round() : -1;
  if (j >= 0) {
    load_k(key_of(j));
    kid = kid_next;
    load_v(key_of(j), kid);
  }
  while (j >= 0) {
    const int kb = key_of(j);
    float x[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        const uint4 w = kr[i][m];
        mma16(x[i], q[0][m].x, q[1][m].x, q[0][m].y, q[1][m].y, w.x, w.y, bf);
        mma16(x[i], q[0][m].z, q[1][m].z, q[0][m].w, q[1][m].w, w.z, w.w, bf);
      }
    }
    const int j_next = next_round();
    if (j_next >= 0) load_k(key_of(j_next));

    // x[i][2 r + e]: row g + 8 r, key kb + 8 i + 2 t + e
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = e >> 1, off = 8 * i + 2 * t + (e & 1), key = kb + off;
        float v = x[i][e];
        if constexpr (MOD) {
          if (a.cap > 0.f) {
            const float in = v * cap_in;
            v = cap_out * (fabsf(in) < kTanhSmall ? tanh_small(in) : tanh_any(in));
          } else {
            v *= cs;
          }
          v = fmaf(-slope[r], fabsf(static_cast<float>(pos[r] - key)), v);
        } else {
          v *= cs;
        }
        bool see = key < s.lk && ((key >= pos[r] - a.left && key <= pos[r] + a.right) || key < s.prefix);
        if (a.doc_k) {
          const int id = __shfl_sync(0xffffffffu, kid, off);
          see = see && id >= 0 && id == qdoc[r];
        }
        x[i][e] = see ? v : -INFINITY;
      }
    float top[2];
    bool up = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      up = up || top[r] > mr[r] + 8.f;
    }
    // the reference maximum moves only when some row's grows by more than 2^8
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m_new = fmaxf(mr[r], top[r]);
        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(mr[r] - m_new);
        mr[r] = m_new;
        lr[r] *= alpha;
#pragma unroll
        for (int h = 0; h < kH; ++h)
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
            o[h][jj][2 * r] *= alpha;
            o[h][jj][2 * r + 1] *= alpha;
          }
      }
    }
    uint32_t pa[2][2];  // [key group][row]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float sub = mr[r] == -INFINITY ? 0.f : mr[r];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = exp2_fast(x[i][2 * r] - sub), p1 = exp2_fast(x[i][2 * r + 1] - sub);
        lr[r] += p0 + p1;
        pa[i][r] = pack_pair(p0, p1, a.type);
      }
    }
    // column n of instruction (h, jj) is dimension 64 h + 8 n + jj
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      const uint32_t v0[4] = {vr[0][h].x, vr[0][h].y, vr[0][h].z, vr[0][h].w};
      const uint32_t v1[4] = {vr[1][h].x, vr[1][h].y, vr[1][h].z, vr[1][h].w};
      const uint32_t v2[4] = {vr[2][h].x, vr[2][h].y, vr[2][h].z, vr[2][h].w};
      const uint32_t v3[4] = {vr[3][h].x, vr[3][h].y, vr[3][h].z, vr[3][h].w};
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) {
        const uint32_t sel = jj & 1 ? 0x7632 : 0x5410;
        mma16(o[h][jj], pa[0][0], pa[0][1], pa[1][0], pa[1][1], __byte_perm(v0[jj / 2], v1[jj / 2], sel),
              __byte_perm(v2[jj / 2], v3[jj / 2], sel), bf);
      }
    }
    j = j_next;
    kid = kid_next;
    if (j >= 0) load_v(key_of(j), kid);
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    lr[r] += __shfl_xor_sync(0xffffffffu, lr[r], 1);
    lr[r] += __shfl_xor_sync(0xffffffffu, lr[r], 2);
    if (t == 0) {
      S.m[warp][g + 8 * r] = mr[r];
      S.l[warp][g + 8 * r] = lr[r];
    }
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      float4* dst = reinterpret_cast<float4*>(&S.o[warp][g + 8 * r][64 * h + 16 * t]);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          dst[2 * e + c] = make_float4(o[h][4 * c][2 * r + e], o[h][4 * c + 1][2 * r + e], o[h][4 * c + 2][2 * r + e],
                                       o[h][4 * c + 3][2 * r + e]);
    }
  }
  __syncthreads();
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
cudaError_t launch(const VarlenArgs& a, cudaStream_t st) {
  const int G = a.Hq / a.Hkv;
  const long long grid = (long long)((a.max_q * G + 15) / 16) * a.splits * a.Hkv * a.B;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  const dim3 g(static_cast<unsigned>(grid));
  auto go = [&](auto kernel) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(FewSmem<D>)));
    return e != cudaSuccess ? e : launch_pdl(kernel, g, dim3(32 * kWarps), sizeof(FewSmem<D>), st, a);
  };
  return a.cap > 0.f || a.slopes ? go(varlen_few_kernel<D, true>) : go(varlen_few_kernel<D, false>);
}

}  // namespace

// Rows that share a key head: up to four tiles of 16 are cheaper here than one of 128 per head.
bool varlen_few_rows(int max_q, int Hq, int Hkv) { return (long long)max_q * (Hq / Hkv) <= 64; }

cudaError_t varlen_few_launch(const VarlenArgs& a, cudaStream_t st) {
  return a.D == 64 ? launch<64>(a, st) : launch<128>(a, st);
}

}  // namespace laya

// C entries of the layer operators on caller-owned device memory (laya_b200_norm, laya_b200_linear,
// laya_b200_attention_varlen): the checks of their arguments, the per-device set-up and the launches.
// They are additions to the reference ABI.
//
// Every argument that can be checked on the host is checked before anything is launched; memory that
// another device, or no device, holds is refused. No entry keeps anything of a call: outputs and
// workspaces belong to the caller, so calls may overlap on any streams, and a captured call replays.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <mutex>

#include "kernels.h"
#include "laya_api.h"
#include "layer_ops.h"

namespace {
using namespace laya;

constexpr int kMaxDevices = 64;
struct Device {
  bool ready = false;
  int sms = 0;
  int pairs = 0;       // co-resident CTA pairs of the matrix product
  int* err = nullptr;  // the error word that the kernel-level entries share
};
std::mutex g_mu;
Device g_dev[kMaxDevices];

bool device_memory(const void* p, int dev) {
  cudaPointerAttributes at;
  if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev);
}

// The current device, set up, for a call on `stream` with these arrays (null ones are not given).
// Returns 0 or the entry's error code.
int begin(void* stream, int sync, std::initializer_list<const void*> arrays, Device* d) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (dev < 0 || dev >= kMaxDevices) return -4;
  for (const void* p : arrays)
    if (p && !device_memory(p, dev)) return -2;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &cap) != cudaSuccess) {
    cudaGetLastError();
    return -5;
  }
  if (cap != cudaStreamCaptureStatusNone && sync) return -2;  // a captured call cannot wait for its work
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_dev[dev].ready) {
    if (cap != cudaStreamCaptureStatusNone) return -8;  // set-up allocates: not inside a capture
    if (cudaDeviceGetAttribute(&g_dev[dev].sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -4;
    if (linear_prepare_device(&g_dev[dev].pairs) != cudaSuccess || varlen_prepare_device() != cudaSuccess) return -4;
    g_dev[dev].err = entry_error_word(dev);
    if (!g_dev[dev].err) return -4;
    g_dev[dev].ready = true;
  }
  *d = g_dev[dev];
  return 0;
}

// After the launch: its error, and with `sync` the wait and the kernel's own error code.
int finish(const char* what, cudaError_t e, void* stream, int sync, int* err) {
  if (e != cudaSuccess) {
    fprintf(stderr, "[laya] %s launch: %s\n", what, cudaGetErrorString(e));
    cudaGetLastError();
    return -5;
  }
  if (!sync) return 0;
  if (cudaStreamSynchronize(static_cast<cudaStream_t>(stream)) != cudaSuccess) return -6;
  int h = 0;
  if (cudaMemcpy(&h, err, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return -6;
  if (!h) return 0;
  cudaMemset(err, 0, sizeof(int));
  return -100 - h;
}

bool is16(int t) { return t == DT_BF16 || t == DT_F16; }
bool is_plain(int t) { return is16(t) || t == DT_F32; }
bool is_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }
// rows of `cols` elements that lie `ld` apart do not overlap (one row has no stride)
bool strides_ok(int rows, int cols, long long ld) { return rows <= 1 || ld >= cols; }
}  // namespace

extern "C" int laya_b200_norm(const void* x, int x_type, long long ldx, const void* resid, int resid_type,
                              long long ldr, void* sum, int sum_type, long long lds, const float* w, const float* b,
                              float eps, int center, void* out, int out_type, long long ldo, float* scale, int rows,
                              int D, void* stream, int sync) {
  if (rows < 0 || D < 1 || D > kNormMaxD || !is_plain(x_type) || (center != 0 && center != 1)) return -2;
  if (!(eps >= 0.f) || !std::isfinite(eps)) return -2;
  if ((resid && !is_plain(resid_type)) || (sum && !is_plain(sum_type))) return -2;
  if (!is_plain(out_type) && out_type != DT_E4M3) return -2;
  if (rows == 0) return 0;
  if (!x || !w || !out || (out_type == DT_E4M3) != (scale != nullptr)) return -2;
  if (!strides_ok(rows, D, ldx) || (resid && !strides_ok(rows, D, ldr)) || (sum && !strides_ok(rows, D, lds)) ||
      !strides_ok(rows, D, ldo))
    return -2;
  if (!is_aligned(x, type_size(x_type)) || (resid && !is_aligned(resid, type_size(resid_type))) ||
      (sum && !is_aligned(sum, type_size(sum_type))) || !is_aligned(out, type_size(out_type)) || !is_aligned(w, 4) ||
      !is_aligned(b, 4) || !is_aligned(scale, 4))
    return -2;
  Device d;
  if (int rc = begin(stream, sync, {x, resid, sum, w, b, out, scale}, &d)) return rc;
  const NormArgs a{x,      ldx,        resid,    ldr,      sum,  lds, w,      b,  out, ldo, scale,
                   x_type, resid_type, sum_type, out_type, rows, D,   center, eps};
  return finish("norm", norm_launch(a, d.sms, static_cast<cudaStream_t>(stream)), stream, sync, d.err);
}

extern "C" int laya_b200_linear(const void* A, long long lda, const void* W, long long ldw, int ab_type,
                                const float* a_scale, const float* w_scale, const float* bias, int act,
                                const void* resid, long long ldr, void* out, int out_type, long long ldo, int M, int N,
                                int K, void* stream, int sync) {
  if (M < 0 || N < 0 || K < 1 || K > kLinearMaxDim || M > kLinearMaxDim || N > kLinearMaxDim) return -2;
  if ((!is16(ab_type) && ab_type != DT_E4M3) || !is_plain(out_type) || act < LIN_NONE || act > LIN_SILU) return -2;
  if (M == 0 || N == 0) return 0;
  if (!A || !W || !out) return -2;
  const int es = type_size(ab_type), os = type_size(out_type);
  // operand rows start on 16 bytes (the tensor copies need it); one row has no stride of its own
  if (M == 1) lda = (K * (long long)es + 15) / 16 * 16 / es;
  if (N == 1) ldw = (K * (long long)es + 15) / 16 * 16 / es;
  if (lda < K || ldw < K || lda > kLinearMaxLd || ldw > kLinearMaxLd || (lda * es) % 16 != 0 || (ldw * es) % 16 != 0)
    return -2;
  if (!is_aligned(A, 16) || !is_aligned(W, 16)) return -2;
  if (!strides_ok(M, N, ldo) || (resid && !strides_ok(M, N, ldr))) return -2;
  if (!is_aligned(out, os) || !is_aligned(resid, os) || !is_aligned(a_scale, 4) || !is_aligned(w_scale, 4) ||
      !is_aligned(bias, 4))
    return -2;
  Device d;
  if (int rc = begin(stream, sync, {A, W, a_scale, w_scale, bias, resid, out}, &d)) return rc;
  const LinearArgs a{A, lda, W, ldw, a_scale, w_scale, bias, resid, ldr, out, ldo, ab_type, out_type, act, M, N, K, 0};
  return finish("linear", linear_launch(a, d.sms, d.pairs, d.err, static_cast<cudaStream_t>(stream)), stream, sync,
                d.err);
}

namespace {
// Bytes of the partial results of one key range.
long long varlen_range_bytes(long long rows_q, int Hq, int D) { return rows_q * Hq * (D + 1LL) * 4; }

// Key ranges that a call of these sizes is cut into: the call's own plan and the workspace query's.
int plan_splits(int B, int rows_q, int max_q, int max_k, int Hq, int Hkv, int sms) {
  return varlen_splits(B, rows_q, std::min(max_q, rows_q), max_k, Hq, Hkv, sms);
}

bool varlen_sizes_ok(int B, int rows_q, int max_q, int max_k, int Hq, int Hkv, int D) {
  return B >= 0 && B <= 65535 && rows_q >= 0 && rows_q <= kVarlenMaxRows && max_q >= 0 && max_q <= kVarlenMaxRows &&
         max_k >= 0 && max_k <= kVarlenMaxRows && Hkv >= 1 && Hq >= Hkv && Hq <= 1024 && Hq % Hkv == 0 &&
         (D == 64 || D == 128) && varlen_units(B, rows_q, std::min(max_q, rows_q), Hq) <= kVarlenMaxUnits;
}
}  // namespace

extern "C" long long laya_b200_attention_varlen_ws(int B, int rows_q, int max_q, int max_k, int Hq, int Hkv, int D) {
  if (!varlen_sizes_ok(B, rows_q, max_q, max_k, Hq, Hkv, D)) return -2;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  const int splits = plan_splits(B, rows_q, max_q, max_k, Hq, Hkv, sms);
  return splits > 1 ? splits * varlen_range_bytes(rows_q, Hq, D) : 0;
}

extern "C" int laya_b200_attention_varlen(const void* q, long long ldq, const void* k, long long ldk, const void* v,
                                          long long ldv, void* out, long long ldo, float* lse, int type,
                                          const int* cu_q, const int* cu_k, int B, int rows_q, int rows_k, int max_q,
                                          int max_k, int Hq, int Hkv, int D, float scale, float softcap,
                                          const float* slopes, int left, int right, const int* prefix,
                                          const int* doc_q, const int* doc_k, void* ws, long long ws_bytes,
                                          void* stream, int sync) {
  if (!varlen_sizes_ok(B, rows_q, max_q, max_k, Hq, Hkv, D) || rows_k < 0 || rows_k > kVarlenMaxRows) return -2;
  if (!is16(type) || !(scale > 0.f) || !std::isfinite(scale) || !(softcap >= 0.f) || !std::isfinite(softcap)) return -2;
  if (scale > kVarlenMaxScale || softcap > kVarlenMaxScale) return -2;
  if (softcap > 0.f && (!std::isnormal(scale / softcap) || !std::isnormal(softcap / scale))) return -2;
  if (left < -1 || right < -1 || (doc_q == nullptr) != (doc_k == nullptr) || ws_bytes < 0) return -2;
  if (B == 0 || rows_q == 0 || max_q == 0) return 0;
  if (!q || !out || !cu_q || !cu_k || (rows_k > 0 && (!k || !v))) return -2;
  const long long wq = (long long)Hq * D, wk = (long long)Hkv * D;
  if (rows_q == 1) ldq = ldo = wq;  // one row has no stride of its own
  if (rows_k <= 1) ldk = ldv = wk;
  for (long long ld : {ldq - wq, ldk - wk, ldv - wk, ldo - wq})
    if (ld < 0 || ld > kLinearMaxLd || ld % 8 != 0) return -2;  // rows start on 16 bytes
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) || !is_aligned(ws, 16) ||
      !is_aligned(lse, 4) || !is_aligned(cu_q, 4) || !is_aligned(cu_k, 4) || !is_aligned(slopes, 4) ||
      !is_aligned(prefix, 4) || !is_aligned(doc_q, 4) || !is_aligned(doc_k, 4))
    return -2;
  Device d;
  if (int rc = begin(stream, sync, {q, k, v, out, lse, cu_q, cu_k, slopes, prefix, doc_q, doc_k, ws}, &d)) return rc;
  VarlenArgs a = {};
  a.q = q;
  a.k = rows_k > 0 ? k : q;  // without keys nothing is read through the tensor maps, which need an address
  a.v = rows_k > 0 ? v : q;
  a.out = out;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldo = ldo;
  a.lse = lse;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.B = B;
  a.rows_q = rows_q;
  a.rows_k = rows_k;
  a.max_q = max_q < rows_q ? max_q : rows_q;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.type = type;
  a.scale = scale;
  a.cap = softcap;
  a.slopes = slopes;
  a.left = left < 0 || left > kVarlenMaxRows ? kVarlenMaxRows : left;
  a.right = right < 0 || right > kVarlenMaxRows ? kVarlenMaxRows : right;
  a.prefix = prefix;
  a.doc_q = doc_q;
  a.doc_k = doc_k;
  const long long range = varlen_range_bytes(rows_q, Hq, D);
  const long long fit = ws ? ws_bytes / range : 0;
  int splits = plan_splits(B, rows_q, max_q, max_k, Hq, Hkv, d.sms);
  if (fit < splits) splits = fit > 1 ? static_cast<int>(fit) : 1;
  a.splits = splits;
  a.part_o = static_cast<float*>(ws);
  a.part_l = a.part_o ? a.part_o + (long long)splits * rows_q * Hq * D : nullptr;
  return finish("attention_varlen", varlen_launch(a, d.sms, d.err, static_cast<cudaStream_t>(stream)), stream, sync, d.err);
}

// Host-side launchers of the layer operators (norm.cu, linear*.cu, varlen_*.cu): one transformer
// layer's norm, matrix product and attention on caller-owned device memory, of any size and type. They
// serve the C entries of abi_layer.cu; the engine's own pass does not use them.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace laya {

// Element types (LAYA_BF16 .. LAYA_E4M3 of the C header).
enum DataType : int { DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2, DT_E4M3 = 3 };
constexpr int type_size(int t) { return t == DT_F32 ? 4 : t == DT_E4M3 ? 1 : 2; }

// Strides (ld*) are in elements.
struct NormArgs {
  const void* x;
  long long ldx;
  const void* resid;  // or null
  long long ldr;
  void* sum;          // or null: h = x + resid in sum_type
  long long lds;
  const float* w;
  const float* b;     // or null
  void* out;
  long long ldo;
  float* scale;       // [rows], e4m3 output only
  int x_type, resid_type, sum_type, out_type;
  int rows, D, center;
  float eps;
};
constexpr int kNormMaxD = 16384;  // 512 threads x 4 pieces x 8 elements
cudaError_t norm_launch(const NormArgs& a, int num_sms, cudaStream_t st);

enum LinearAct : int { LIN_NONE = 0, LIN_RELU = 1, LIN_GELU = 2, LIN_SILU = 3 };
// out[m][n] = act(a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] + bias[n]) + resid[m][n]
struct LinearArgs {
  const void* A;
  long long lda;
  const void* W;
  long long ldw;
  const float* a_scale;  // or null: 1
  const float* w_scale;  // or null: 1
  const float* bias;     // or null
  const void* resid;     // or null; out_type
  long long ldr;
  void* out;
  long long ldo;
  int ab_type, out_type, act;
  int M, N, K;
  int vec_out;  // out and resid rows start on 16 bytes (set by the launcher)
};
cudaError_t linear_prepare_device(int* pair_clusters);
cudaError_t linear_launch(const LinearArgs& a, int num_sms, int pair_clusters, int* err, cudaStream_t st);
constexpr int kLinearMaxDim = 1 << 24;         // M, N, K: row and column arithmetic stays in 32 bits
constexpr long long kLinearMaxLd = 1LL << 32;  // the tensor maps' strides stay below 2^40 bytes
constexpr int kLinearFewRows = 16;  // most rows of the kernel for few rows
cudaError_t linear_few_launch(const LinearArgs& a, int num_sms, cudaStream_t st);

// Attention of packed sequences: s = scale q.k, capped by cap tanh(s / cap), minus slope |distance|,
// then softmax over the keys that the window, prefix and document masks leave.
struct VarlenArgs {
  const void *q, *k, *v;
  void* out;
  long long ldq, ldk, ldv, ldo;
  float* lse;          // [rows_q][Hq] or null
  const int *cu_q, *cu_k;
  int B, rows_q, rows_k, max_q;
  int Hq, Hkv, D, type;
  float scale, cap;    // cap 0: none
  const float* slopes; // [Hq] or null
  int left, right;     // kVarlenMaxRows: unbounded
  const int* prefix;   // [B] or null
  const int *doc_q, *doc_k;  // both or neither
  int splits;          // key ranges per row; above 1 the partial results go to part_*
  // Tile kernel, set by its launcher. Scores stay in units of q.k until `to_log2` scales them for the
  // exponential, capped ones in units of q.k / unit: a power of two, 1 unless a cap makes u = score / cap
  // leave the middle of fp32's range.
  struct {
    float unit, to_log2;
    float small;       // a capped score below this has u below kTanhSmall
    float all_small;   // `small` where unit is 1; else below every score
    float k1, k2, k3;  // tanh_small's coefficients for the score's square
    float to_2u, out;  // score -> 2 u log2 e; cap
  } caps;
  int slots;           // tile kernel: 0, or how many tile slots its units run over (set by its launcher)
  float* part_o;       // [splits][rows_q][Hq][D]
  float* part_l;       // [splits][rows_q][Hq], log2 units
};
constexpr int kVarlenMaxRows = 1 << 29;  // positions and window edges stay in 32 bits
constexpr float kVarlenMaxScale = 0x1p126f;  // scale and cap, times 2 log2 e, stay finite
constexpr int kVarlenMaxSplits = 32;
cudaError_t varlen_prepare_device();
// Key ranges that varlen_launch would use if the workspace allowed them. Here and below max_q is at most
// rows_q.
int varlen_splits(int B, int rows_q, int max_q, int max_k, int Hq, int Hkv, int num_sms);
// Query tiles and heads that the tile kernel runs over, empty ones included.
long long varlen_units(int B, int rows_q, int max_q, int Hq);
constexpr long long kVarlenMaxUnits = (1LL << 31) - (1 << 20);  // 32 bits, and room for one more round
cudaError_t varlen_launch(const VarlenArgs& a, int num_sms, int* err, cudaStream_t st);
bool varlen_few_rows(int max_q);
cudaError_t varlen_few_prepare_device();
cudaError_t varlen_few_launch(const VarlenArgs& a, int* err, cudaStream_t st);

// Tensor map of rows [rows][mid][cols] (strides in elements) loaded in 128-byte-wide boxes of box_rows
// rows with the 128-byte swizzle; defined beside the engine's operand maps.
bool make_rows_map(CUtensorMap* map, const void* base, int type, uint64_t cols, uint64_t mid, uint64_t rows,
                   uint64_t mid_stride, uint64_t ld, uint32_t box_rows);

}  // namespace laya

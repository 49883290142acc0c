/* C ABI of the Laya B200 engine (liblaya_b200.so).
 *
 * The first ten declarations are the reference engine's ABI, unchanged in name, signature and
 * meaning (mauimauer/layamd src/laya_api.h:5-19, implemented at src/engine.hip:543-559), so the
 * reference's ctypes server (server/laya_server.py:18-31), its parity tool (src/test_parity.cpp)
 * and its bench tool (src/bench_engine.cpp) bind to this library without change. Everything after
 * them is an addition with no counterpart in the reference.
 *
 * Threading: a handle is driven by one caller thread at a time, as in the reference
 * (docs/architecture.md:84-85). Calls are synchronous: forward returns after the results are in
 * the caller's arrays.
 */
#pragma once
#ifdef __cplusplus
extern "C" {
#endif

/* Loads `dir` (model.safetensors, encoder/config.json, rl_agent_config.json) onto the GPUs named by
 * LAYA_DEVICES (default: the current device) and sizes every buffer for LAYA_MAX_TOKENS rows.
 * Replaces src/laya_api.h:5. The reference exits the process on a load error; this library prints
 * the reason and returns NULL instead. */
void* laya_create(const char* dir);

/* B questions in one call. ids/markers are concatenated per question; markers are positions within
 * that question's sequence. logits receive sum(nmark) raw scorer logits in input order, act B*n_act
 * raw act-head logits. Returns 0, or -1 without touching the outputs when any 1<=lens[b]<=max_len,
 * 1<=nmark[b]<=255 or 0<=marker<lens[b] fails, or (an addition: the reference reads outside its
 * embedding table instead) a token id lies outside [0, vocab) or a qtype outside 0..2. Replaces
 * src/laya_api.h:8-9
 * (src/engine.hip:489-539). Also returns -2 when the GPU reported an error for this call, and -3 in
 * debug bounds mode when a pass's packing maps failed their host check (nothing was launched). */
int laya_forward_batch(void* h, int B, const int* lens, const int* ids, const int* nmark, const int* markers,
                       const int* qtypes, float* logits, float* act);

/* Single-question form; S is ignored and valid_len is the length. Input errors are ignored
 * silently, as in the reference. Replaces src/laya_api.h:10-11 (src/engine.hip:549-551). */
void laya_forward(void* h, const int* ids, int S, int valid_len, const int* markers, int K, int qtype,
                  float* logits, float* act);

int laya_n_act(void* h);       /* len(act_costs)+1 from rl_agent_config.json (src/laya_api.h:12) */
int laya_max_len(void* h);     /* max_len from rl_agent_config.json (src/laya_api.h:13) */
int laya_max_markers(void* h); /* 255 (src/laya_api.h:14) */
/* Calibration temperature of a question type (src/laya_api.h:15); 1.0 for a qtype outside the
 * configured list (the reference does not check the index). */
float laya_temperature(void* h, int qtype);
/* Per-stage device-time table printed to stdout, divided by `iters` (src/laya_api.h:16). Stages are
 * timed only while profiling is on (LAYA_PROFILE set at load, or laya_prof_enable). */
void laya_prof_report(void* h, int iters);
void laya_prof_reset(void* h); /* src/laya_api.h:17 */
/* Chooses the GEMM tile width for every (M bucket, N, K) the model can hit up front, so serving
 * never tunes on the request path (src/laya_api.h:19). */
void laya_tune_all(void* h);

/* ----------------------------------------------------------------- additions (no reference
 * counterpart) */

/* Releases every device and host resource of the handle. */
void laya_destroy(void* h);

/* laya_create with an explicit precision and device list.
 * precision 0: bf16 operands, fp32 accumulation and fp32 residual stream (production path).
 * precision 1: fp32-parity mode: every GEMM runs as three bf16 products on hi/lo splits of both
 *              operands (A_hi*W_hi + A_hi*W_lo + A_lo*W_hi) and attention runs in fp32.
 * devices: comma-separated CUDA device ordinals ("0", "0,1,2,3"); NULL or "" uses LAYA_DEVICES or
 * the current device. With several devices, each forward call shards its questions across them. */
void* laya_create_ex(const char* dir, int precision, const char* devices);

/* Number of devices (replicas) the handle runs on. */
int laya_num_devices(void* h);

/* Turns per-stage profiling on or off (CUDA events around every launch; graphs are bypassed while
 * it is on). */
void laya_prof_enable(void* h, int on);

/* Copies the accumulated time (ms) and launch count of stage `name` (e.g. "gemm_qkv"); returns 0 or
 * -1 if the stage was never timed. */
int laya_prof_get(void* h, const char* name, double* ms, long long* launches);

/* Packs a batch exactly like laya_forward_batch would (validation included) and reports the pass
 * layout without touching a GPU: n_passes, and for each pass its first question, question count and
 * packed row count (arrays of capacity `cap`). Returns the number of passes or -1 on invalid input. */
int laya_plan_passes(void* h, int B, const int* lens, const int* nmark, const int* markers, int cap,
                     int* pass_first, int* pass_count, int* pass_rows);

/* Same packing rules as laya_plan_passes for a configuration given by value, with no handle
 * (max_len, pass_tokens, max_seqs); for host-side tests. */
int laya_plan_passes_cfg(int max_len, int pass_tokens, int max_seqs, int B, const int* lens, const int* nmark,
                         const int* markers, int cap, int* pass_first, int* pass_count, int* pass_rows);

/* The engine's plan for one GEMM launch, host-only (no counterpart in the reference, which autotunes
 * per shape at start-up, src/engine.hip:293-379): *bn = 128 or 256 (one CTA per 128 x bn tile) or
 * 512 (a CTA pair per 256 x 256 tile), *splits = K slices (1 = whole K). M packed rows, the weight's
 * N x K, parity != 0 for the fp32-parity mode (three bf16 products per K block), the device's SM count
 * and co-resident CTA pairs, ln_fusable != 0 for a residual GEMM whose following bias-free LayerNorm
 * a split's reduce kernel can take over (with the default credit; LAYA_SPLIT_LN_CREDIT changes only
 * the engine's own choice). Returns 0 or -1. */
int laya_plan_gemm(int M, int N, int K, int parity, int num_sms, int pair_clusters, int ln_fusable, int* bn,
                   int* splits);

/* No counterpart in the reference. Debug bounds mode, host side and host-only: validates a batch like
 * laya_forward_batch (plus qtypes in 0..2 and ids inside the vocabulary), packs it into passes of at
 * most pass_tokens rows and max_seqs questions, fills every pass's metadata block exactly as the
 * engine uploads it (token ids, positions, row -> question map, offsets, the attention work items
 * and gathered-row maps) and checks every map against the pass and the arena. corrupt > 0 breaks map
 * number `corrupt` (1-8) of the first pass before the check, so a test can show that the check
 * catches it. Returns the number of passes checked, -1 for an invalid batch, or -100-n when check n
 * failed. The engine runs the same check on every pass when loaded with LAYA_DEBUG_BOUNDS=1 or from a
 * debug-bounds build, and then returns -3 from laya_forward_batch without launching anything. */
int laya_pack_check(int max_len, int vocab, int pad_id, int pass_tokens, int max_seqs, int B, const int* lens,
                    const int* ids, const int* nmark, const int* markers, const int* qtypes, int corrupt);

/* No counterpart in the reference. 1 when this library was built with -DLAYA_DEBUG_BOUNDS: every
 * kernel then checks the indices it reads from the packing maps (token ids, rows, work items,
 * gathered rows, marker offsets, RoPE positions) against their extents, records code 40-45 in the
 * error word and skips the access instead of reading or writing out of range (laya_forward_batch
 * then returns -2). 0 in the normal build, whose kernels carry no such checks. */
int laya_debug_bounds_build(void);

/* The replica (0..ndev-1) each of B questions goes to when a call is sharded over ndev GPUs, as
 * laya_forward_batch does it, for a model of hidden size d, GeGLU width `intermediate`, n_layers
 * encoder layers of which n_global use global attention, sliding window `window` (full width) and a
 * head FFN of 4d; host-only. Longest processing time first on each question's modelled device time
 * (its algorithmic FLOPs for length lens[b] and nmark[b] options, attention FLOPs weighted by their
 * measured cost relative to GEMM FLOPs) onto the least-loaded replica. Returns 0 or -1. */
int laya_shard_plan(int ndev, int B, const int* lens, const int* nmark, int d, int intermediate, int n_layers,
                    int n_global, int window, int* owner);

/* Benchmark support: validates, packs and uploads one batch (it must fit one pass per device) and
 * keeps it resident; laya_replay then runs the staged pass `iters` times back to back on every
 * device with the inputs already in HBM and writes the device time of the slowest device, measured
 * with CUDA events on the engine's stream, to *ms. laya_staged_results copies the last replay's
 * outputs out like laya_forward_batch. Return 0 or a negative error. */
int laya_stage(void* h, int B, const int* lens, const int* ids, const int* nmark, const int* markers,
               const int* qtypes);
int laya_replay(void* h, int iters, double* ms);
int laya_staged_results(void* h, float* logits, float* act);
/* Benchmark support (no counterpart in the reference): replays the staged pass `iters` times back
 * to back as a second graph that also records a CUDA event pair around every stage, and adds the
 * stage times of the last replay to the profile table read by laya_prof_get, so that per-stage device
 * times are taken in the same steady state as laya_replay. Return 0 or a negative error. */
int laya_replay_profiled(void* h, int iters);

/* Cumulative counters of the forward and replay calls since the last reset, summed over devices:
 * kernel launches of this library, bytes copied host->device and device->host. reset != 0 clears
 * them after reading. */
int laya_io_stats(void* h, long long* launches, long long* h2d_bytes, long long* d2h_bytes, int reset);

/* Writes the residual stream after the embedding, after every encoder layer (before the final
 * norm), after the final norm + type embedding, and after each head layer for the last forward call
 * when dumping is on: files emb.bin, enc<i>.bin, final.bin, head<i>.bin (fp32, one row per packed
 * token of pass 0, sequences back to back in input order; head<last>.bin holds the gathered rows:
 * markers of every question in order, then one CLS row per question). NULL turns dumping off. */
int laya_set_dump_dir(void* h, const char* dir);

/* Isolated encoder GEMM on caller-owned device memory (the GEMM sweep and kernel tests):
 * out = epilogue(A[planes][M][K] * W[planes][N][K]^T). epi: 0 store, 1 store with RoPE on columns
 * < rope_cols, 2 GeGLU (W interleaved in groups of bn/2, out has geglu_I columns), 3 fp32 residual
 * add into resid[M][N]. out_mode: 0 bf16, 1 bf16 hi/lo planes, 2 fp32. act: 0 none, 1 ReLU, 2 GELU.
 * bn: 128 or 256 (one CTA per 128 x bn tile) or 512 (a CTA pair per 256 x 256 tile, 2-SM MMA).
 * planes 2 selects the three-product fp32 emulation. stream may be NULL. With
 * sync != 0 the call waits for the GPU and returns -100-code if a kernel reported an error (this
 * call's, or one left unread by an earlier call with sync = 0: see laya_b200_kernel_error). */
int laya_b200_gemm(const void* A, const void* W, void* out, float* resid, const float* bias, int M, int N, int K,
                   int planes, int epi, int out_mode, int act, int bn, const float* cos_t, const float* sin_t,
                   const int* pos, int rope_cols, int geglu_I, void* stream, int sync);

/* laya_b200_gemm with the K loop split into `splits` slices (1..8, and at most one per 64-wide K
 * block: ceil(K / 64), x3 in parity mode; else -2) run by different CTAs, for small M where the
 * output tiles alone cannot fill the GPU (one-CTA tiles, bn 128 or 256). The fp32 partials
 * go to a workspace the library allocates on the device and keeps for later calls; a second kernel
 * sums them in slice order and applies the epilogue, so results do not depend on scheduling. Calls
 * that overlap on the GPU (other streams) share that workspace and must not be issued. */
int laya_b200_gemm_splitk(const void* A, const void* W, void* out, float* resid, const float* bias, int M, int N,
                          int K, int planes, int epi, int out_mode, int act, int bn, const float* cos_t,
                          const float* sin_t, const int* pos, int rope_cols, int geglu_I, int splits, void* stream,
                          int sync);

/* Isolated encoder attention on caller-owned device memory (attention tests and benchmark); replaces
 * the reference's k_flash_wmma launch (src/kernels.hip:351-356) at kernel level. qkv: bf16
 * [rows][3 * 64 * H] (q | k | v, heads of 64), sequences packed back to back with lengths lens[B]
 * (host array, sum <= rows); out: bf16 [rows][64 * H]. window 0: full attention within each
 * sequence, else |q - k| <= window. impl 0: tcgen05 kernel, 1: mma.sync kernel. Rows of qkv past the
 * sequences must hold finite values. Uses a library-owned metadata buffer per device: calls must not
 * overlap on the GPU. Returns 0, -2 bad arguments, -100-code if the kernel reported an error (sync). */
int laya_b200_attention(const void* qkv, void* out, int rows, int B, const int* lens, int H, int window, int impl,
                        void* stream, int sync);

/* No counterpart in the reference (whose engine exits on any GPU error). Exercises, on GPU `device`,
 * the bounded wait that every pipeline kernel of this library uses on its mbarriers: one thread waits
 * on a barrier phase that nothing completes, gives up after the wait budget (about 2^31 SM cycles,
 * roughly one second), records its error code in a device word and returns, so the kernel ends
 * normally and the context stays usable. The word is the one the kernel-level entry points share
 * (see laya_b200_kernel_error), and the code stays there until it is read. Writes the recorded code
 * (30) to *code, the wait's length in SM cycles to *cycles and the kernel's device time to *ms.
 * Returns 0, -2 if a CUDA call failed, or -3 without launching when that word already holds an
 * earlier, unread code. */
int laya_b200_watchdog_selftest(int device, int* code, long long* cycles, float* ms);

/* No counterpart in the reference. Kernel errors of the kernel-level entry points on GPU `device`
 * (laya_b200_gemm, laya_b200_gemm_splitk, laya_b200_gemm_splitk_noalloc, laya_b200_attention, the layer
 * operators, the watchdog self-test). A kernel whose bounded wait ran out records a code in a device
 * word (the first code wins) and ends; a call with sync != 0 reports it as -100-code, but a call with sync = 0 cannot,
 * so the word keeps the code until it is read: by the next call with sync != 0 on the same word, or by
 * this function. It waits for all work on the device, reads and clears both words (the one the
 * allocating entries share and the one in the allocation-free entry's static array) and returns the
 * first code found (GEMM 1-5, attention 16-18, self-test 30), 0 if none, -1 for a bad device
 * ordinal, -2 if a CUDA call failed. It allocates nothing. */
int laya_b200_kernel_error(int device);

/* No counterpart in the reference. laya_b200_gemm_splitk for callers that cannot allocate device
 * memory: a host whose memory manager reserves the GPU's memory up front (a serving stack with a
 * caching allocator) or a plugin host that forbids allocation in its callbacks, where a cudaMalloc
 * could fail, fragment the host's pool or stall every stream with its implicit synchronisation. Same
 * arguments and results; it calls no cudaMalloc or cudaFree. Its scratch is a fixed 16 MiB array in
 * the library's device image, held by every GPU that loads the library until the process exits:
 * splits x M x N must stay <= 4194304 fp32 partials, else the call prints why and returns -7
 * without launching. The first call on a device sets up
 * (kernel attributes and the array's device address, no allocation); make it before any stream
 * capture. Every call on a device shares the array: calls that overlap on the GPU (other streams,
 * other threads) race and must not be issued. Every slice overwrites its whole plane of partials
 * (splits may not exceed the K blocks, ceil(K / 64) x 3 in parity mode, else -2), so no call sees
 * another's partials. The error word in the array is zeroed at set-up and then kept: a code left by
 * a call with sync = 0 is reported by the next call with sync != 0 or by laya_b200_kernel_error. */
int laya_b200_gemm_splitk_noalloc(const void* A, const void* W, void* out, float* resid, const float* bias, int M,
                                  int N, int K, int planes, int epi, int out_mode, int act, int bn,
                                  const float* cos_t, const float* sin_t, const int* pos, int rope_cols,
                                  int geglu_I, int splits, void* stream, int sync);

/* ----------------------------------------------------------------- layer operators
 * A transformer layer's norm, matrix product and attention on caller-owned device memory (additions,
 * no counterpart in the reference). They share these rules. Pointers name memory of the current
 * device; a pointer that no device or another device owns is refused (-2). Element types are
 * LAYA_BF16, LAYA_F16, LAYA_F32 and LAYA_E4M3 (8 bits: 4 exponent and 3 mantissa bits, largest value
 * 448). ld* are distances between rows in elements; rows must not overlap. Outputs are written inside
 * their rows and columns only. Every call launches on `stream` (NULL: the default stream), keeps
 * nothing of a call and may overlap other calls; it can be captured into a graph once any layer
 * operator has run on the device outside a capture (else -8), with sync 0. sync != 0 waits for the
 * GPU. Returns 0, -1 no device, -2 an argument is refused (nothing was launched), -4 set-up failed,
 * -5 a launch failed, -6 the GPU reported an error, -8 as above, -100-code when a kernel gave up
 * (sync; see laya_b200_kernel_error). */
enum { LAYA_BF16 = 0, LAYA_F16 = 1, LAYA_F32 = 2, LAYA_E4M3 = 3 };

/* Norm of a residual sum, per row of D elements (1 <= D <= 16384):
 *   h = x + resid;  z = h - center * mean(h);  y = z / sqrt(mean(z^2) + eps) * w + b
 * center 0: root-mean-square norm, 1: LayerNorm. resid (or NULL) and x are LAYA_BF16 / F16 / F32, w
 * and b (or NULL) fp32. sum (or NULL) receives h in sum_type; it may be x or resid itself (the same
 * pointer, type and stride); out overlaps no input. y is computed from h in fp32, before h is rounded
 * to sum_type, for any h whose z stays in fp32's range (and any eps, 0 included). out_type LAYA_BF16 /
 * F16 / F32: out = y. LAYA_E4M3: scale[row] = max(max|y| / 448, 2^-126) and out = y * (1 / scale[row]),
 * rounded to nearest even; scale is given exactly with this type. A row with a NaN has NaN in its scale.
 * rows 0 does nothing. */
int laya_b200_norm(const void* x, int x_type, long long ldx, const void* resid, int resid_type, long long ldr,
                   void* sum, int sum_type, long long lds, const float* w, const float* b, float eps, int center,
                   void* out, int out_type, long long ldo, float* scale, int rows, int D, void* stream, int sync);

/* Matrix product with everything after it in one pass:
 *   out[m][n] = act(a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] + bias[n]) + resid[m][n]
 * A [M][K] and W [N][K] both LAYA_BF16, LAYA_F16 or LAYA_E4M3 (ab_type), sums in fp32; a_scale [M],
 * w_scale [N] (with any ab_type; 1 where NULL) and bias [N] (or NULL) fp32. act 0 none, 1 ReLU, 2 GELU
 * (erf, to 1e-6 absolutely), 3 SiLU. out_type LAYA_BF16 / F16 / F32 is also resid's; resid (or NULL) may
 * be out itself (the same pointer and stride); out overlaps no other input. Any M, N, K up to 2^24 (K >=
 * 1; M or N 0 does nothing). Rows of A and W start on 16 bytes: their addresses and strides in bytes are
 * multiples of 16, so rows of torch.nn.Linear's dense weight fit where K elements are a multiple of 16
 * bytes, and have to be copied to padded storage where not (one row alone may have any stride); what
 * storage holds past column K is not used. out, resid and the vectors may have any alignment of their
 * type. The sums' order depends only on the sizes and types. */
int laya_b200_linear(const void* A, long long lda, const void* W, long long ldw, int ab_type, const float* a_scale,
                     const float* w_scale, const float* bias, int act, const void* resid, long long ldr, void* out,
                     int out_type, long long ldo, int M, int N, int K, void* stream, int sync);

/* Attention of packed sequences with masks, distance bias and capped scores. Sequence b has query rows
 * cu_q[b] .. cu_q[b + 1] - 1 of q [rows_q][Hq][D] and key rows cu_k[b] .. cu_k[b + 1] - 1 of k and v
 * [rows_k][Hkv][D] (device arrays of B + 1 offsets, B <= 65535); query head h uses key head h / (Hq / Hkv).
 * Query i of lq sits at key position p = i + lk - lq: at lq = lk on its own key, with fewer queries than
 * keys on the last ones. For key j:
 *   s = scale * q_i . k_j;  softcap > 0: s = softcap * tanh(s / softcap);  slopes: s -= slopes[h] * |p - j|
 *   seen: (p - left <= j <= p + right, or j < prefix[b])  and  doc_q[i] == doc_k[j] >= 0
 *   out_i = sum_j softmax(s)_j v_j over the keys seen, lse[i][h] = log sum_j exp(s)
 * left, right -1: unbounded (right 0 is causal); slopes [Hq] fp32, prefix [B], doc_q [rows_q] and doc_k
 * [rows_k] (both or neither) are device arrays or NULL; lse [rows_q][Hq] fp32 or NULL. A row that sees
 * nothing gets 0 and lse -infinity. q, k, v, out are LAYA_BF16 or LAYA_F16, D is 64 or 128; their rows
 * start on 16 bytes (they may be columns of one projection's rows; one row alone may have any stride).
 * scale is positive, scale and softcap are at most 2^126, and with a cap scale / softcap and its inverse
 * are normal fp32 numbers; slopes[h] / scale times the longest distance stays in fp32's range. out may not overlap the inputs. Scores and sums are fp32, capped scores to
 * within 4e-7 of the cap; the weights are rounded to the inputs' type for the product with v.
 * max_q is at least every lq (later rows of a longer sequence are left as they are), and may lie far
 * above them; max_k only guides how the work is cut. What needs 2^31 or more units of work (query heads
 * times the smaller of B * max_q / 128 and B + rows_q / 128, about) is refused. Offsets outside the arrays
 * are cut to them; behind offsets that run backwards rows may stay unwritten. Rows of no sequence are
 * not written. Keys behind a sequence's end or of a negative document (any negative number) may hold
 * anything; other values are finite, or a NaN can reach rows whose masks hide it. ws: workspace for
 * calls with few rows over many keys, 16-byte aligned, laya_b200_attention_varlen_ws bytes for the same
 * sizes (NULL or fewer bytes: the keys are cut into fewer ranges, with rounding differences); two calls
 * in flight need two. bf16 self-attention with D 64, Hq = Hkv and a symmetric window or none runs 10 to
 * 40 % faster through laya_b200_attention, whose lengths are a host array. */
int laya_b200_attention_varlen(const void* q, long long ldq, const void* k, long long ldk, const void* v,
                               long long ldv, void* out, long long ldo, float* lse, int type, const int* cu_q,
                               const int* cu_k, int B, int rows_q, int rows_k, int max_q, int max_k, int Hq, int Hkv,
                               int D, float scale, float softcap, const float* slopes, int left, int right,
                               const int* prefix, const int* doc_q, const int* doc_k, void* ws, long long ws_bytes,
                               void* stream, int sync);
/* Workspace bytes for a call of these sizes on the current device (0: none), -1 no device, -2 refused. */
long long laya_b200_attention_varlen_ws(int B, int rows_q, int max_q, int max_k, int Hq, int Hkv, int D);

#ifdef __cplusplus
}
#endif

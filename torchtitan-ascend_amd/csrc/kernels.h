// Host-side launchers of the device kernels (internal to libttamd_moe.so).
// All sizes have been validated by the C ABI layer before these are called.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "probe.h"

namespace ttamd {

// routing.hip
size_t route_workspace_bytes(int64_t M, int E);
// Bytes of the per-chunk histogram the route kernels read and write.
size_t route_hist_bytes(int64_t M, int E);
// Histogram geometry: chunks of route_chunk_labels() flat labels, the
// histogram stored bucket-major, hist[b * num_chunks + chunk].
int route_num_chunks(int64_t M);
int route_chunk_labels();
// The rank pass folds the histogram scan in (one launch) for histograms of
// at most 32768 entries.
bool route_fused_scan(int64_t M, int E);
// Scan + rank from an accumulated histogram: counts, offsets, the stable
// order; optionally adds the counts to tokens_per_expert and builds the
// forward GEMMs' tile table (tiles of at most plan_max_rows rows) in `plan`
// (gemm workspace layout).
hipError_t launch_route_from_hist(const void* labels, bool is64, int M, int E, const float* scores,
                                  int* counts, int* offsets, int* sorted_idx, int* inverse,
                                  float* sorted_scores, int* hist, float* tokens_per_expert,
                                  void* plan, int plan_max_rows, hipStream_t stream);
hipError_t launch_route(const void* labels, bool is64, int M, int E, const float* scores,
                        int* counts, int* offsets, int* sorted_idx, int* inverse,
                        float* sorted_scores, void* ws, hipStream_t stream);
// The library-owned route workspace of the device that runs `stream` (the
// current device for a null stream): its size, and its device address
// (looked up once per device, then cached).
size_t route_scratch_bytes();
hipError_t route_scratch(hipStream_t stream, void** ptr);
hipError_t launch_gather_rows(const void* in, const int* src, const float* scale,
                              bool scale_by_src, int n_in, int n_src_max, int rows, int hidden,
                              int div, void* out, hipStream_t stream);
hipError_t launch_invert_perm(const int* sorted, int M, int* inv, hipStream_t stream);
hipError_t launch_dispatch_rows(const void* in, const int* inverse, const float* scores, int T, int K,
                                int hidden, void* out, hipStream_t stream);
hipError_t launch_combine(const void* in, const int* inverse, const float* probs, int T,
                          int topk, int hidden, void* out, hipStream_t stream);
hipError_t launch_rowdot(const void* a, const void* b, const int* bidx, int bdiv,
                         bool out_by_bidx, int rows, int n_b, int n_out, int hidden, float* out,
                         hipStream_t stream);
hipError_t launch_group_labels(const int* counts_group, int G, int E_loc, int rows, int* labels,
                               hipStream_t stream);
hipError_t launch_router_topk(const float* logits, const float* bias, int T, int E, int K,
                              int score_func, int renorm, float renorm_eps, float route_scale,
                              float* top_scores, int64_t* top_idx, hipStream_t stream);

// Group-limited selection (router_group.hip): experts in `groups` equal runs,
// `kept` of them eligible, a group's value the sum of its two largest
// selection values (top2) or its largest.
struct RouterGroups {
  int groups, kept, top2;
};

// router.hip
size_t router_workspace_bytes(int64_t T, int E, int64_t D);
hipError_t launch_router_fused(const void* x, const void* w, const float* bias, int T, int E, int D, int K,
                               int score_func, int renorm, float renorm_eps, float route_scale,
                               float* top_scores, int64_t* top_idx, void* logits, void* ws,
                               hipStream_t stream, const RouterGroups* groups = nullptr);
// The same router, also accumulating the route histogram of the picks into
// `hist` ((E + 1) * route_num_chunks(T * K) ints, cleared by the gate GEMM
// kernel first), ready for launch_route_from_hist.
hipError_t launch_router_hist(const void* x, const void* w, const float* bias, int T, int E, int D, int K,
                              int score_func, int renorm, float renorm_eps, float route_scale,
                              float* top_scores, int64_t* top_idx, void* logits, void* ws, int* hist,
                              hipStream_t stream, const RouterGroups* groups = nullptr);

// Group-limited selection (router_group.hip).
hipError_t launch_router_topk_grouped(const void* logits, bool bf16, const float* bias, int T, int E, int K,
                                      const RouterGroups& g, int score_func, int renorm, float renorm_eps,
                                      float route_scale, float* top_scores, int64_t* top_idx, hipStream_t stream);
// The same on the gate GEMM's partial logits [S][T][E] (E <= 256).
hipError_t launch_group_topk_partials(const float* part, int S, const float* bias, int T, int E, int K,
                                      const RouterGroups& g, int score_func, int renorm, float renorm_eps,
                                      float route_scale, float* top_scores, int64_t* top_idx, void* logits, int* hist,
                                      int nchunks, int chunk, hipStream_t stream);
// d(top_scores) [T, K] -> d(logits) [T, E] in the logits' type.
hipError_t launch_router_topk_backward(const float* grad, const int64_t* idx, const void* logits, bool bf16, int T,
                                       int E, int K, int score_func, int renorm, float renorm_eps, float route_scale,
                                       void* grad_logits, hipStream_t stream);

// Router backward: d(top_scores) -> d(logits) -> dx (bf16 [T, D], nullable)
// and dW_r ([E, D], fp32 or bf16, nullable).
size_t router_backward_workspace_bytes(int64_t T, int E, int64_t D);
hipError_t launch_router_backward(const float* grad, const int64_t* idx, const void* logits, const void* x,
                                  const void* w, int T, int E, int D, int K, int score_func, int renorm,
                                  float renorm_eps, float route_scale, void* dx, void* dw, bool dw_fp32,
                                  void* ws, hipStream_t stream);

// block_norm.hip: f = K-way sum of branch rows; p = rmsnorm(f) * post;
// u = residual + scale * act(gate) * p; n = rmsnorm(u) * pre.
struct NormArgs {
  int T, D, K;
  const uint16_t* rows;   // bf16 [T * K, D], or null: u is the residual
  const int* inverse;     // [T * K] row of slot t K + k, or null
  const float* probs;     // [T * K], or null
  const void* residual;   // [T, D] of the stream's type, or null
  const void* post;       // [D], or null: p = f
  const void* gate;       // [T], [D] or [T, D] by gate_kind
  const void* pre;        // [D], or null: no n
  int gate_kind;          // 0 none, 1 per token, 2 per channel, 3 per element
  int sigmoid;            // act: sigmoid, else the gate itself
  int stream32, post32, gate32, pre32;  // fp32 instead of bf16
  float scale, eps;
  void* u;                // [T, D] of the stream's type, or null
  void* n;                // bf16 [T, D]
  float* rstd;            // [2, T]: r_f, r_u; or null
};
hipError_t launch_norm_forward(const NormArgs& a, hipStream_t stream);
struct NormBwdArgs {
  NormArgs fwd;           // K = 1; rstd read; u, n unused
  const void* du;         // [T, D] of the stream's type, or null: zero
  const void* dn;         // bf16 [T, D], or null (no pre)
  void *dbranch, *dresidual, *dpost, *dgate, *dpre;  // each nullable
  float* part;
};
size_t norm_backward_workspace_bytes(int64_t T, int64_t D);
hipError_t launch_norm_backward(const NormBwdArgs& a, hipStream_t stream);

// gemm.hip
int gemm_max_qtiles(int M, int E);
size_t gemm_workspace_bytes(int64_t M, int E);
size_t gemm_plan_bytes(int64_t M, int E);
// Largest token tile of the bf16 forward / dgrad GEMMs (tile plans are built for it).
int gemm_fwd_tile_rows();
void gemm_tiles(const int* counts, int E, int64_t weight_rows, int k, bool fp8, int* tile_rows, int* tile_cols,
                int* pieces);
// The next forward grouped-GEMM launch records these events around its main
// kernel on its stream, then the probe disarms (nullptr, nullptr: disarm).
void gemm_probe_arm(hipEvent_t start, hipEvent_t end);
// The next n_launches kernel launches of the library take the event pairs
// (events[2 i], events[2 i + 1]) as their start and end stamps (n_launches
// <= kProbeMaxChain; 0 disarms).
void probe_chain_arm(const hipEvent_t* events, int n_launches);
hipError_t launch_grouped_mm(const void* x, const void* w, const int* offs, int M, int E, int N,
                             int K, void* out, void* ws, hipStream_t stream);
hipError_t launch_grouped_mm_swiglu(const void* x, const void* w13, const int* offs, int M,
                                    int E, int H, int D, float limit, void* a_out, void* h_out,
                                    void* ws, hipStream_t stream);
hipError_t launch_grouped_mm_swiglu_gather(const void* tokens, int n_tokens, const int* src_index,
                                           int src_div, const void* w13, const int* offs, int M, int E,
                                           int H, int D, float limit, void* a_out, void* h_out, void* ws,
                                           hipStream_t stream);
hipError_t launch_grouped_mm_unpermute(const void* act, const void* w2, const int* offs, int M,
                                       int E, int D, int H, const float* row_scale,
                                       const int* dest, int n_dest, void* out, void* ws,
                                       hipStream_t stream);
hipError_t launch_shared_expert_add(const void* x, int T, int D, int H, const void* w13s, const void* w2s,
                                   const float* gate_logits, float limit, void* a_scratch, void* out,
                                   void* ws, hipStream_t stream);
// The expert stage of the inference forward: (gather [+ score] ->) w13 +
// SwiGLU -> w2 + score + scatter (-> K-way sum), both GEMMs on one tile
// table (`plan`, or one built into the workspace when plan is null).  rows:
// `out` takes the weighted rows in flat-slot order, without the K-way sum.
size_t moe_experts_forward_workspace_bytes(int64_t T, int64_t D, int64_t H, int E, int K, bool permute_first,
                                           bool rows = false);
hipError_t launch_moe_experts_forward(const void* tokens, int T, int D, int H, int E, int K,
                                      const int* sorted_idx, const int* offs, const float* sorted_scores,
                                      bool score_before, float limit, const void* w13, const void* w2,
                                      void* out, void* plan, void* ws, hipStream_t stream, bool rows = false);
hipError_t launch_grouped_mm_dgrad(const void* dy, const void* w, const int* offs, int M, int E,
                                   int N, int K, void* dx, void* ws, hipStream_t stream);
// The same without the tail split: plan is gemm_plan_bytes(M, E) bytes.
hipError_t launch_grouped_mm_dgrad_unsplit(const void* dy, const void* w, const int* offs, int M, int E, int N,
                                           int K, void* dx, void* plan, hipStream_t stream);
hipError_t launch_grouped_mm_dgrad_swiglu(const void* dy, const void* w2, const void* h,
                                          const int* offs, int M, int E, int D, int H,
                                          float limit, void* dh, void* a_out, void* ws,
                                          hipStream_t stream);
// ws: NULL (no tail split) or gemm_workspace_bytes(M, E) bytes (the
// leftover tiles' partial sums and arrival counters).
// x_rows (nullable, [M + 64], every entry a row of x): reduction row m reads x
// row x_rows[m].
hipError_t launch_grouped_mm_wgrad(const void* dy, const void* x, const int* offs, int M, int E,
                                   int N, int K, void* dw, bool fp32, void* ws, hipStream_t stream,
                                   const int* x_rows = nullptr);

// 8-bit activation checkpoints (checkpoint.hip): e4m3 codes [R, C], exponent
// bytes [R, ceil(C / 128)].
hipError_t launch_pack_rows(const void* in, int64_t R, int C, void* codes, void* exps, hipStream_t stream);
// out row j = row src_index[j] / src_div of n_src (nullable -> j), times
// row_scale[j] (nullable).  ids_out[j] (nullable) = the clamped row of
// ids_index[j], j < n_ids, and row 0 in the 64 entries after them.
hipError_t launch_unpack_rows(const void* codes, const void* exps, int n_src, const int* src_index, int src_div,
                              const float* row_scale, int64_t R, int C, void* out, const int* ids_index, int* ids_out,
                              int n_ids, hipStream_t stream);
hipError_t launch_grouped_mm_dgrad_swiglu_packed(const void* dy, const void* w2, const void* codes, const void* exps,
                                                 const int* offs, int M, int E, int D, int H, float limit, void* dh,
                                                 void* a_out, void* ws, hipStream_t stream);
size_t wgrad_packed_workspace_bytes(int64_t rows, int64_t M, int E, int64_t K);
hipError_t launch_grouped_mm_wgrad_packed(const void* dy, const void* codes, const void* exps, int n_src,
                                          const int* src_index, int src_div, const float* row_scale, const int* offs,
                                          int M, int E, int N, int K, void* dw, bool fp32, void* ws,
                                          hipStream_t stream);

// 4-bit weights (fp4.hip): tiles of 16 rows x 128 columns.
hipError_t launch_pack_fp4(const void* in, bool f32, int64_t E, int N, int K, void* codes, void* exps,
                           hipStream_t stream);
hipError_t launch_unpack_fp4(const void* codes, const void* exps, int64_t E, int N, int K, void* out,
                             hipStream_t stream);

// The layer for a few tokens (decode.hip), products with 4-bit weights (fp4_mm.hip).
constexpr int kDecodeMaxTokens = 64;
constexpr int kDecodeMaxTopk = 16;
size_t router_decode_workspace_bytes(int64_t T, int E);
struct RouterDecode {
  const void *x, *w_router;
  const void* w_gate;  // nullable: gate[t] = sigmoid of the token's product with it
  const float* bias;
  RouterGroups groups;
  int score_func, renorm;
  float eps, scale;
  float* top_scores;
  int64_t* top_idx;
  float* gate;
  void* logits;        // router_decode_workspace_bytes
};
hipError_t launch_router_decode(const RouterDecode& r, int T, int E, int D, int K, hipStream_t stream);
struct ExpertsDecode {
  int T, D, H, E, K, Hs;
  const void* x;
  const void* idx;
  int is64, before, fp4;
  const float* scores;
  float limit;
  const void *w13, *w2, *s13, *s2;
  const uint8_t *e13, *e2, *es13, *es2;  // exponents of 4-bit weights
  const float* gate;
  void* out;
};
size_t experts_decode_workspace_bytes(int64_t T, int64_t D, int64_t H, int K, int64_t Hs);
// router (nullable): its picks are made first (c.idx, c.scores and c.gate are its outputs).
hipError_t launch_experts_decode(const ExpertsDecode& c, const RouterDecode* router, void* ws, hipStream_t stream);
hipError_t launch_grouped_mm_fp4(const void* x, const void* codes, const void* exps, const int* offs, const void* bias,
                                 bool bias32, int M, int E, int N, int K, void* out, hipStream_t stream);

// fp8 e4m3 path (quant.hip, gemm_fp8.hip via gemm.hip)
hipError_t launch_quantize_rows(const void* in, const int* src_index, int src_div, const float* row_mul,
                                int n_in, int R, int K, void* q_out, float* scale_t, hipStream_t stream);
hipError_t launch_quantize_blocks(const void* w, int E, int N, int K, void* q_out, float* scale,
                                  hipStream_t stream);
hipError_t launch_grouped_mm_fp8(const void* xq, const float* sx, const void* wq, const float* sw,
                                 const int* offs, int M, int E, int N, int K, void* out, void* ws,
                                 hipStream_t stream);
hipError_t launch_grouped_mm_fp8_swiglu(const void* xq, const float* sx, const void* w13q,
                                        const float* s13, const int* offs, int M, int E, int H, int D,
                                        float limit, void* a_out, void* h_out, void* ws,
                                        hipStream_t stream);
hipError_t launch_grouped_mm_fp8_unpermute(const void* aq, const float* sa, const void* w2q,
                                           const float* s2, const int* offs, int M, int E, int D, int H,
                                           const float* row_scale, const int* dest, int n_dest,
                                           void* out, void* ws, hipStream_t stream);

}  // namespace ttamd

// Internal launcher interface between the HIP kernel translation units and the C-ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mtp {

typedef uint16_t bf16_t;

// MI355X has 256 compute units in 8 XCDs; launch geometry is a pure function of the problem
// shape so that results do not depend on the device a call lands on.
constexpr int kNumCU = 256;

// Row pitch of the backward's bf16 gradient-tile buffer is chunk + kGPitchPad elements: a pitch
// that is a multiple of a large power of two (chunk is a multiple of 256) makes the 256 rows of
// one operand tile fall on the same memory channels.
constexpr int kGPitchPad = 64;

struct LceHead {
  int q4;                 // 0: dense bf16 [V][D]; 1: 4-bit affine, group size 64
  const bf16_t* w;        // dense weight
  const bf16_t* wt;       // optional transposed (4-bit: dequantized) weight [D][lce_head_t_ld(V)], or null
  const uint32_t* wq;     // packed nibbles [V][D/8]
  const bf16_t* sc;       // scales [V][D/64]
  const bf16_t* bi;       // biases [V][D/64]
};

int lce_fwd_nsplit(long N, long V);
long lce_head_t_ld(long V);

// A staged 4-bit chunk (backward without the cached transposed copy) also holds its dequantized rows
// [chunk][D] bf16, after the transposed chunk [D][lce_head_t_ld(chunk)] (element offset below), so the
// chunk's gradient tiles are a dense product.
#ifndef MTP_Q4_STAGE_ROWS
#define MTP_Q4_STAGE_ROWS 1
#endif
constexpr bool kQ4StageRows = MTP_Q4_STAGE_ROWS != 0;
inline long lce_stage_rows_offset(long D, long chunk) { return (D * lce_head_t_ld(chunk) + 127) / 128 * 128; }
// Parts of the backward's dH contraction over `ktiles` 256-wide vocab tiles for a block of `rows`
// rows (1 = one workgroup per output tile), and the fp32 part tiles that takes (0 when 1).
int lce_dh_ksplit(long rows, long D, long ktiles);
size_t lce_dh_parts_bytes(long rows, long D, long ktiles);

hipError_t launch_lce_head_transpose(const LceHead& h, int V, int D, bf16_t* Wt, hipStream_t stream,
                                     bf16_t* rows_out = nullptr);

// Vocab rows of the forward's largest split (N rows, V vocab), and of its largest run when it
// stages runs of whole splits into `stage_rows` rows.
long lce_fwd_stage_rows_max(long N, long V);
long lce_fwd_stage_rows_used(long N, long V, long stage_rows);

// stage (optional, 4-bit head with D % 64 == 0): a buffer of stage_rows >= lce_fwd_stage_rows_max rows
// of D bf16 into which runs of vocab splits are dequantized before a dense product over them (the
// same partials as the in-register dequantization).
hipError_t launch_lce_fwd(const LceHead& h, const bf16_t* H, const int64_t* targets, int N, int D, int V,
                          long long ignore_index, float* nll, float* lse, float* tgt, float* ws,
                          bf16_t* stage, long stage_rows, hipStream_t stream);

// Token scoring (score_kernels.hip) takes the forward's tiles with more of their statistics. A forward's STAT is a sum of:
enum { kStatScaled = 1, kStatEntropy = 2, kStatGroups = 4, kStatList = 8, kStatKeep = 16 };
constexpr int kGroup = 128;  // consecutive logits whose maximum a forward keeps
// Logits to put away of each row: ascending columns (kNoColumn past the last) to their places in z, and out of the statistics; with an entropy one
// column a row (k = 1), which stays in them.
constexpr int kNoColumn = 0x7fffffff;
struct ScoreList {
  const int* column;  // [N][k], or null
  float* z;           // [N][k]
  int k;
};
struct ScoreStats {
  float scale2;        // log2(e) / temperature: the partials are of x = z scale2
  float *m, *s;        // [lce_fwd_nsplit][N] maximum of x, sum of 2^(x - m)
  float* u;            // the same of 2^(x - m) (x - m), or null
  float* gmax;         // [N][ldg] the maximum z of each group of kGroup (ldg: an even number of them), or null (with u)
  int ldg;
  float* z;            // [N][ldz] the logits, or null (with u); ldz a multiple of kGroup
  long ldz;
  ScoreList list;
};
hipError_t launch_lce_stats(const LceHead& h, const bf16_t* H, int N, int D, int V, const ScoreStats& st, bf16_t* stage,
                            long stage_rows, hipStream_t stream);

// The gradient of a loss of softmax(z / temperature) by the logits z that is p (alpha + beta z) but for k columns a row.
// Rows with neither factor get zeros, whatever their hidden state holds.
struct AffineRows {
  const float *alpha, *beta;  // [N]; beta may be null (0)
  float scale2;               // log2(e) / temperature
};
struct AffineGrad {
  AffineRows rows;
  const int* columns;    // [N][k], no column twice in a row; < 0: none
  const float* value;    // [N][k] the gradient there
  int k;
  const float* z;        // [N][ldz] the logits that a forward kept, or null: they are formed again
  long ldz;
  const void* clean;     // for dW: the hidden states with the rows that get zeros cleared (bf16; fp32 in the fp32 backward)
  // With z, bf16: fp32 [2 N][D], or null. A gradient then is two bf16 numbers, its rounding and what that leaves, in rows t and N + t of
  // G (and clean holds the hidden states twice): the products' rows up to a tile cost nothing (steps of 5 to 75 tokens take the same time),
  // and dH is off by its own rounding alone: 5 x 64 x 997, lists of 4: 1.7e-3 of the norm, with one number 2.6e-3.
  float* halves;
};

// affine: that gradient in the place of the loss's (targets, dnll unused).
hipError_t launch_lce_bwd(const LceHead& h, const bf16_t* H, const int64_t* targets, const float* lse,
                          const float* dnll, int N, int D, int V, long long ignore_index, int chunk, int row_block,
                          bf16_t* dH, bf16_t* dW, bf16_t* Gbuf, float* acc32, float* parts, bf16_t* stage,
                          hipStream_t stream, const AffineGrad* affine = nullptr);

hipError_t launch_lce_mean(const float* nll, const int64_t* targets, long n, long long ignore_index, float* mean,
                           float* count, hipStream_t stream);
hipError_t launch_lce_mean_bwd(const float* d_mean, const float* count, long n, float* d_nll, hipStream_t stream);

struct AttnShape {
  int b, hq, hkv, s, dh;
  float scale;
  int causal;  // 1: key j visible to query i iff j <= i (and, packed, same segment); 0: every key
};

// Splits of each key block's work in the head_dim-128 dK/dV kernel (1 = none), and the backward
// workspace: D plus the fp32 dK/dV partials when either mode splits.
int attn_dkv_nsplit(int b, int hq, int hkv, int s, int dh, int causal);
size_t attn_bwd_workspace(int b, int hq, int hkv, int s, int dh);

hipError_t launch_attn_fwd(const AttnShape& sh, const bf16_t* q, const bf16_t* k, const bf16_t* v,
                           const int32_t* seg_id, const int32_t* seg_start, bf16_t* o, float* lse,
                           hipStream_t stream);

hipError_t launch_attn_bwd(const AttnShape& sh, const bf16_t* q, const bf16_t* k, const bf16_t* v,
                           const bf16_t* o, const float* lse, const bf16_t* d_o, const int32_t* seg_id,
                           const int32_t* seg_start, bf16_t* dq, bf16_t* dk, bf16_t* dv, float* dvec,
                           hipStream_t stream);

// Sum of the fp32 partials of a split dK/dV pass; plane: elements of dK.
hipError_t launch_attn_dkv_reduce(const float* part, int ns, long plane, bf16_t* dk, bf16_t* dv, hipStream_t stream);

// Scores and masks beyond the plain ones (attn_scored.hip): cap > 0: cap tanh(x / cap) in the place of a
// scaled score x; slopes [hq]: minus slope |i - j|; start and end [b][s]: key j visible to query i iff
// start[i] <= j < end[i] (both given or neither; AttnShape.causal is then 0).
struct AttnScore {
  float cap;
  const float* slopes;
  const int32_t* start;
  const int32_t* end;
};
size_t attn_scored_bwd_workspace(int b, int hq, int hkv, int s, int dh);
size_t attn_scored_fwd_workspace(int b, int hq, int hkv, int s, int dh);  // less: unsplit
size_t attn_scored_plan(int b, int hq, int hkv, int s, int dh);  // bytes; 0: no use for one
hipError_t launch_attn_scored_fwd(const AttnShape& sh, const AttnScore& sc, const bf16_t* q, const bf16_t* k,
                                  const bf16_t* v, bf16_t* o, int8_t* o_low, int32_t* plan, float* lse,
                                  void* workspace, size_t bytes, hipStream_t stream);
hipError_t launch_attn_scored_bwd(const AttnShape& sh, const AttnScore& sc, const bf16_t* q, const bf16_t* k,
                                  const bf16_t* v, const bf16_t* o, const int8_t* o_low, const int32_t* plan,
                                  const float* lse, const bf16_t* d_o, bf16_t* dq, bf16_t* dk, bf16_t* dv, void* workspace,
                                  hipStream_t stream);
// Workspaces of the fp32 passes; less than that (the backward: at least D) runs what lacks room unsplit.
size_t attn32_scored_fwd_workspace(int b, int hq, int hkv, int s, int dh);
size_t attn32_scored_bwd_workspace(int b, int hq, int hkv, int s, int dh);
hipError_t launch_attn32_scored_fwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k,
                                    const float* v, float* o, float* lse, void* workspace, size_t bytes, hipStream_t stream);
hipError_t launch_attn32_scored_bwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k,
                                    const float* v, const float* o, const float* lse, const float* d_o, float* dq,
                                    float* dk, float* dv, void* workspace, size_t bytes, hipStream_t stream);

// fp32 inputs (f32_kernels.hip): fp32 MFMA products, fp32 outputs and gradients.
struct LceHead32 {
  int q4;                 // 0: dense fp32 [V][D]; 1: 4-bit affine, group size 64, fp32 scales/biases
  const float* w;
  const uint32_t* wq;
  const float* sc;        // [V][D/64]
  const float* bi;
};
int lce32_fwd_nsplit(long N, long V);
int lce32_dh_parts(long N, long D, long kcols, int* per);
hipError_t launch_lce32_fwd(const LceHead32& h, const float* H, const int64_t* targets, int N, int D, int V,
                            long long ignore_index, float* nll, float* lse, float* tgt, float* ws, hipStream_t stream);
// Gbuf: fp32 [N][chunk + 4]; dH fp32 [N][D]; dW (optional, dense head) fp32 [V][D].
hipError_t launch_lce32_bwd(const LceHead32& h, const float* H, const int64_t* targets, const float* lse,
                            const float* dnll, int N, int D, int V, long long ignore_index, int chunk, float* dH,
                            float* dW, float* Gbuf, hipStream_t stream, const AffineGrad* affine = nullptr);
hipError_t launch_lce32_stats(const LceHead32& h, const float* H, int N, int D, int V, const ScoreStats& st,
                              hipStream_t stream);  // [lce32_fwd_nsplit][N]
hipError_t launch_attn32_fwd(const AttnShape& sh, const float* q, const float* k, const float* v,
                             const int32_t* seg_start, float* o, float* lse, hipStream_t stream);
hipError_t launch_attn32_dkv_reduce(const float* part, int ns, long plane, float* dk, float* dv, hipStream_t stream);
// Splits of the fp32 dK/dV pass (1: none), and the backward's workspace with them: D, then the partials.
int attn32_dkv_splits(int b, int hq, int hkv, int s, int dh);
size_t attn32_bwd_workspace(int b, int hq, int hkv, int s, int dh, int nsplit);
// dvec: the workspace, D = rowsum(dO * O) fp32 [b][hq][s] first (formed by the dQ pass for the dK/dV pass).
hipError_t launch_attn32_bwd(const AttnShape& sh, const float* q, const float* k, const float* v, const float* o,
                             const float* lse, const float* d_o, const int32_t* seg_start, float* dq, float* dk,
                             float* dv, float* dvec, int nsplit, hipStream_t stream);

// Token scoring and distillation (score_kernels.hip). The logits of groups of kGroup that single tokens want are formed
// again: an entry is a token (x) and the place of its group in rows (y); a tile is up to kGroup entries of one group.
struct GatherTile {
  int group, first, count, unused;
};
struct GatherPlan {
  const int2* entries;
  const GatherTile* tiles;  // [max_tiles], with count 0 past the last
  int max_tiles;
  float* rows;              // [entries][kGroup]
};
hipError_t launch_dequant32(const LceHead32& h, long V, long D, float* out, hipStream_t stream);  // [V][D]
hipError_t launch_lce_gather(const LceHead& h, const bf16_t* H, int D, int V, const GatherPlan& p, hipStream_t stream);
hipError_t launch_lce32_gather(const LceHead32& h, const float* H, int D, int V, const GatherPlan& p, hipStream_t stream);

constexpr long kScoreRows = 16384;   // tokens of one pass of a forward: more are taken in blocks
constexpr int kScoreTop = 128;       // most alternatives, and longest teacher's list
constexpr long kScoreVocab = 1 << 21;
constexpr long kScoreDims = 1 << 22; // hidden dims from which a tile's rows (256 of bf16, 128 of fp32) pass its 31-bit offsets: bf16 is
                                     // refused there, fp32 takes the core that has none
constexpr long kFewTokens = 128;     // tokens up to which a bf16 forward keeps its logits
constexpr long kFewTokens32 = 64;    // an fp32 one (hidden dims that are multiples of 4)
constexpr long kKeptBytes = 256L << 20;  // of logits that a forward with alternatives may keep
constexpr double kTailFloor = 1e-6;  // least mass that the outcomes outside a list count as

// One head of either type; w32 where the hidden states are fp32.
struct ScoreHead {
  int f32;
  LceHead h;
  LceHead32 h32;
  const void* hidden;
};
struct ScoreShape {
  long n, d, v;
  float inv_t, c2;   // 1 / temperature; log2(e) / temperature, rounded once: softmax(z / temperature) is that of 2^(z c2) everywhere
  int stage;         // 4-bit: dequantize the whole head into the workspace first
};
// logits, in a forward's outputs: [n][logits_ld(v)], which then keeps them there for its backward, or null.
inline long logits_ld(long v) { return (v + kGroup - 1) / kGroup * kGroup; }
struct LogprobsOut {
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_ids;
  float *lse, *tgt, *logits;
};
size_t logprobs_fwd_workspace(const ScoreShape& sh, int f32, int q4, int top, int keep);
hipError_t launch_logprobs_fwd(const ScoreHead& h, const ScoreShape& sh, const int64_t* targets, long long ignore_index,
                               int top, const LogprobsOut& out, void* ws, hipStream_t stream);
enum { kDistillForward = 0, kDistillReverse = 1, kDistillJsd = 2 };
struct DistillLoss {
  int k, kind, renormalize, reduction;
  double beta, inv_t;
};
struct DistillOut {
  float *loss, *scale;        // scale [1]: what a row's gradient is multiplied with, 1 / rows that count for a mean
  float *lse, *rest, *coef;   // [n], [n], [n][k]
  int* columns;               // [n][k]
  float* logits;
};
size_t distill_fwd_workspace(const ScoreShape& sh, int f32, int q4, int k, int keep);
hipError_t launch_distill_fwd(const ScoreHead& h, const ScoreShape& sh, const int64_t* ids, const float* teacher,
                              const uint8_t* mask, const DistillLoss& p, const DistillOut& out, void* ws, hipStream_t stream);
// What the backwards hand to launch_lce_bwd / launch_lce32_bwd: alpha, beta, columns, value (k = 1).
hipError_t launch_logprobs_coef(const float* d_logprobs, const float* d_entropy, const int64_t* targets, long long ignore_index,
                                const float* lse, const float* entropy, const float* tgt, long n, long v, float inv_t,
                                float* alpha, float* beta, int* columns, float* value, hipStream_t stream);
// Gradient tiles from kept logits, columns [v_begin, v_begin + cols) (zeros from vlim on; cols a multiple of 8, fp32: of 4).
hipError_t launch_affine_tiles(const AffineGrad& a, const float* lse, long n, int v_begin, int vlim, int cols, long ldg, bf16_t* g,
                               hipStream_t stream);
// dH = the sum of its halves.
hipError_t launch_join_halves(const float* halves, long count, bf16_t* dH, hipStream_t stream);
hipError_t launch_affine_tiles(const AffineGrad& a, const float* lse, long n, int v_begin, int vlim, int cols, long ldg, float* g,
                               hipStream_t stream);
hipError_t launch_distill_coef(const float* d_loss, int per_row, const float* scale, const float* rest, const float* coef,
                               long n, int k, float* alpha, float* value, hipStream_t stream);
// Hidden states with the rows whose factors are both 0 cleared; row_bytes a multiple of 4.
hipError_t launch_clean_rows(const void* hidden, const float* alpha, const float* beta, long n, long row_bytes, int copies, void* out,
                             hipStream_t stream);

// Preference and policy losses (preference_kernels.hip).
enum { kPrefSigmoid = 0, kPrefHinge = 1, kPrefIpo = 2 };
enum { kReduceNone = 0, kReduceMean = 1, kReduceSum = 2, kReduceSequences = 3 };
struct PrefLoss {
  int kind, reduction;
  double beta, smoothing;
};
struct PolicyLoss {
  int reduction;      // none: per token; mean over the tokens; sequences: mean of each sequence's mean
  int has_ref, adv_per_token;
  double log_low, log_high;   // log(1 - clip_low), log(1 + clip_high)
  float edge_low, edge_high;  // 1 - clip_low, 1 + clip_high
  float kl_coef;
};
size_t pref_workspace(long pairs, long n);
size_t policy_workspace(long rows, long n);
// reduction none: loss [pairs], else [1]; reward, coef [2 pairs]. offsets [2 pairs + 1], or null: rows of n / (2 pairs).
hipError_t launch_pref_fwd(const float* nll, const float* ref, const uint8_t* mask, const int64_t* offsets, long pairs, long n,
                           const PrefLoss& p, float* loss, float* reward, float* coef, void* ws, hipStream_t stream);
hipError_t launch_pref_bwd(const float* d_loss, const float* coef, const uint8_t* mask, const int64_t* offsets, long pairs,
                           long n, int per_pair, float* d_nll, hipStream_t stream);
// reduction none: loss [n], else [1]; stats [2], weight [rows].
hipError_t launch_policy_fwd(const float* nll, const float* old, const float* ref, const float* adv, const uint8_t* mask,
                             const int64_t* offsets, long rows, long n, const PolicyLoss& p, float* loss, float* stats,
                             float* weight, void* ws, hipStream_t stream);
hipError_t launch_policy_bwd(const float* d_loss, const float* nll, const float* old, const float* ref, const float* adv,
                             const uint8_t* mask, const int64_t* offsets, long rows, long n, const PolicyLoss& p,
                             const float* weight, float* d_nll, hipStream_t stream);

}  // namespace mtp

// C-ABI entry points: argument validation, workspace planning and launch.
// Every function validates shapes, alignment and workspace before any launch and reports a
// negative MTP_ERR_* code with a thread-local message; nothing here allocates device memory or
// synchronizes the host.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <mutex>

#include "../../include/mtp_hip.h"
#include "mtp_launch.hpp"

// Scratch of mtp_lce_fwd_noalloc: the forward's per-(vocab split, token) partial maxima and sums,
// held in a file-scope device array so that entry point allocates nothing. Each GPU the library
// runs on holds its own copy until the process ends. The host may not pass the array's name to a
// kernel (in host code it is a stand-in, not a device address): its device address, per device, is
// looked up once with hipGetSymbolAddress and used everywhere host code needs the array.
static constexpr size_t kNoAllocScratchBytes = size_t(4) << 20;
static __device__ __align__(256) float scratch[kNoAllocScratchBytes / sizeof(float)];

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return MTP_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 1;
constexpr int64_t kMaxLossTokens = (int64_t(1) << 31) - 2048;  // a whole workgroup's tokens end below 2^31
constexpr int64_t kTile = 256;

size_t lce_fwd_ws(int64_t n, int64_t v) {
  return (size_t)2 * (size_t)mtp::lce_fwd_nsplit(n, v) * (size_t)n * sizeof(float);
}

int check_lce_common(const void* hidden, const void* w, const uint32_t* w_q, const void* scales,
                     const void* biases, const int64_t* targets, int64_t n, int64_t d, int64_t v,
                     int32_t head_kind) {
  if (n < 1 || d < 1 || v < 1) return fail(MTP_ERR_INPUT, "n, d, v must be >= 1 (got n=%lld d=%lld v=%lld)", (long long)n, (long long)d, (long long)v);
  if (n > kMaxDim || d > kMaxDim || v > kMaxDim) return fail(MTP_ERR_INPUT, "n, d, v must each be < 2^31");
  if (!hidden || !targets) return fail(MTP_ERR_INPUT, "hidden and targets must be non-null");
  if (!aligned16(hidden)) return fail(MTP_ERR_UNSUPPORTED, "hidden must be 16-byte aligned");
  if (head_kind == MTP_HEAD_DENSE || head_kind == MTP_HEAD_DENSE_STAGED) {
    if (!w) return fail(MTP_ERR_INPUT, "dense head: w must be non-null");
    if (!aligned16(w)) return fail(MTP_ERR_UNSUPPORTED, "dense head: w must be 16-byte aligned");
    if (d % 8 != 0) return fail(MTP_ERR_UNSUPPORTED, "kernel impl requires d %% 8 == 0 for a dense head (got d=%lld); use impl='chunked'", (long long)d);
    if (head_kind == MTP_HEAD_DENSE_STAGED && d % 64 != 0)
      return fail(MTP_ERR_UNSUPPORTED, "MTP_HEAD_DENSE_STAGED requires d %% 64 == 0 (got d=%lld)", (long long)d);
  } else if (head_kind == MTP_HEAD_Q4 || head_kind == MTP_HEAD_Q4_STAGED) {
    if (!w_q || !scales || !biases) return fail(MTP_ERR_INPUT, "quantized head: w_q, scales and biases must be non-null");
    if (!aligned16(w_q)) return fail(MTP_ERR_UNSUPPORTED, "quantized head: w_q must be 16-byte aligned");
    if (d % 64 != 0) return fail(MTP_ERR_UNSUPPORTED, "kernel impl requires the quantized head's hidden dim to be a multiple of 64 (got d=%lld); use impl='chunked'", (long long)d);
  } else {
    return fail(MTP_ERR_UNSUPPORTED, "unknown head_kind %d", (int)head_kind);
  }
  return MTP_OK;
}

mtp::LceHead make_head(const void* w, const uint32_t* w_q, const void* scales, const void* biases, int32_t head_kind) {
  mtp::LceHead h;
  h.q4 = head_kind == MTP_HEAD_Q4 || head_kind == MTP_HEAD_Q4_STAGED;
  h.w = static_cast<const mtp::bf16_t*>(w);
  h.wt = nullptr;
  h.wq = w_q;
  h.sc = static_cast<const mtp::bf16_t*>(scales);
  h.bi = static_cast<const mtp::bf16_t*>(biases);
  return h;
}

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

int check_attn(const void* q, const void* k, const void* v, int64_t b, int64_t hq, int64_t hkv, int64_t s,
               int64_t dh, int32_t causal, const int32_t* seg_id, const int32_t* seg_start) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1) return fail(MTP_ERR_INPUT, "b, hq, hkv, s must be >= 1");
  if (hq % hkv != 0) return fail(MTP_ERR_INPUT, "Hq=%lld must be a multiple of Hkv=%lld for GQA grouping", (long long)hq, (long long)hkv);
  if (b * hq * s > kMaxDim || s > (int64_t(1) << 24)) return fail(MTP_ERR_INPUT, "b*hq*s must be < 2^31 and s < 2^24");
  if (dh != 64 && dh != 96 && dh != 128) return fail(MTP_ERR_UNSUPPORTED, "kernel impl only supports head_dim in (64, 96, 128) (got %lld); use impl='reference'", (long long)dh);
  if (causal != 0 && causal != 1) return fail(MTP_ERR_INPUT, "causal must be 0 or 1 (got %d)", (int)causal);
  if ((seg_id == nullptr) != (seg_start == nullptr)) return fail(MTP_ERR_INPUT, "seg_id and seg_start must be both given or both null");
  if (seg_id && !causal) return fail(MTP_ERR_UNSUPPORTED, "segments (packed attention) require causal=1; packing composes on top of the causal triangle");
  if (!q || !k || !v) return fail(MTP_ERR_INPUT, "q, k, v must be non-null");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return fail(MTP_ERR_UNSUPPORTED, "q, k, v must be 16-byte aligned");
  return MTP_OK;
}

int check_scored(const void* q, const void* k, const void* v, int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh,
                 float scale, int32_t causal, float softcap, const float* slopes, const int32_t* span_start,
                 const int32_t* span_end) {
  const int rc = check_attn(q, k, v, b, hq, hkv, s, dh, causal, nullptr, nullptr);
  if (rc) return rc;
  // Distances exact in fp32, and the byte count of a row's keys within 32 bits.
  if (s >= (int64_t(1) << 23)) return fail(MTP_ERR_INPUT, "s must be < 2^23 with softcap, slopes or spans (got %lld)", (long long)s);
  if (!(scale > 0.f) || !(scale < HUGE_VALF)) return fail(MTP_ERR_INPUT, "scale must be positive and finite (got %g)", (double)scale);
  if (!(softcap >= 0.f) || !(softcap < HUGE_VALF)) return fail(MTP_ERR_INPUT, "softcap must be finite and >= 0, 0 for none (got %g)", (double)softcap);
  if (softcap != 0.f && !(softcap >= 1e-3f && softcap <= 1e3f)) return fail(MTP_ERR_UNSUPPORTED, "kernel impl serves a softcap in [1e-3, 1e3] (got %g); use impl='reference'", (double)softcap);
  if ((span_start == nullptr) != (span_end == nullptr)) return fail(MTP_ERR_INPUT, "span_start and span_end must be both given or both null");
  if (span_start && causal) return fail(MTP_ERR_INPUT, "spans are the whole mask: causal must be 0 with them");
  if (!span_start && !slopes && softcap == 0.f) return fail(MTP_ERR_INPUT, "no softcap, slopes or spans given: use mtp_attn_fwd / mtp_attn_bwd");
  return MTP_OK;
}

// Rows and tokens of a preference or policy loss.
int check_rows(int64_t rows, int64_t n, const int64_t* offsets) {
  if (rows < 1 || n < 1) return fail(MTP_ERR_INPUT, "the loss needs at least one sequence and one token (got %lld sequences, %lld tokens)", (long long)rows, (long long)n);
  if (rows > (int64_t(1) << 24) || n > kMaxLossTokens) return fail(MTP_ERR_INPUT, "at most 2^24 sequences and 2^31 - 2048 tokens");
  if (!offsets && n % rows) return fail(MTP_ERR_INPUT, "without offsets the %lld tokens must be %lld rows of one length", (long long)n, (long long)rows);
  return MTP_OK;
}

int policy_params(mtp::PolicyLoss* p, const float* ref_nll, int32_t adv_per_token, double clip_low, double clip_high,
                  double kl_coef, int32_t reduction) {
  if (!(clip_low >= 0.0 && clip_low <= 1.0)) return fail(MTP_ERR_INPUT, "clip_low must be in [0, 1] (got %g)", clip_low);
  if (!(clip_high >= 0.0 && clip_high < HUGE_VAL)) return fail(MTP_ERR_INPUT, "clip_high must be finite and >= 0 (got %g)", clip_high);
  if (!(kl_coef >= 0.0 && kl_coef < HUGE_VAL)) return fail(MTP_ERR_INPUT, "kl_coef must be finite and >= 0 (got %g)", kl_coef);
  if (kl_coef != 0.0 && !ref_nll) return fail(MTP_ERR_INPUT, "kl_coef needs ref_nll");
  if (reduction != MTP_REDUCE_NONE && reduction != MTP_REDUCE_MEAN && reduction != MTP_REDUCE_SEQUENCES)
    return fail(MTP_ERR_INPUT, "unknown reduction %d of a policy loss", (int)reduction);
  *p = mtp::PolicyLoss{reduction, ref_nll != nullptr, adv_per_token != 0, log1p(-clip_low), log1p(clip_high),
                       (float)(1.0 - clip_low), (float)(1.0 + clip_high), (float)kl_coef};
  return MTP_OK;
}

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};

// The address of `scratch` on the device that runs `stream` (the current device for the null
// stream), looked up on the first call on that device with that device current. The launch goes to
// `stream`, so the scratch must be that device's copy whatever device the calling thread has current.
int scratch_for_stream(hipStream_t stream, void** out) {
  int cur = -1;
  hipError_t e = hipGetDevice(&cur);
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "hipGetDevice failed: %s", hipGetErrorString(e));
  int dev = cur;
  if (stream) {
    hipDevice_t sd = -1;
    e = hipStreamGetDevice(stream, &sd);
    if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "hipStreamGetDevice failed: %s", hipGetErrorString(e));
    dev = sd;
  }
  if (dev < 0 || dev >= kMaxDevices) return fail(MTP_ERR_RUNTIME, "device index %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    if (dev != cur && (e = hipSetDevice(dev)) != hipSuccess)
      return fail(MTP_ERR_RUNTIME, "hipSetDevice(%d) failed: %s", dev, hipGetErrorString(e));
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    const hipError_t er = dev != cur ? hipSetDevice(cur) : hipSuccess;
    if (e != hipSuccess || !p)
      return fail(MTP_ERR_RUNTIME, "hipGetSymbolAddress(scratch) failed on device %d: %s", dev, hipGetErrorString(e));
    if (er != hipSuccess) return fail(MTP_ERR_RUNTIME, "hipSetDevice(%d) failed: %s", cur, hipGetErrorString(er));
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return MTP_OK;
}

}  // namespace

extern "C" {

const char* mtp_last_error(void) { return g_err; }

int mtp_abi_version(void) { return MTP_ABI_VERSION; }

// MTP_HEAD_Q4_STAGED forward (d % 64 == 0): the partials, then (256-byte aligned) the staging buffer
// for runs of vocab splits dequantized to bf16 rows of d.
static bool fwd_staged(int32_t head_kind, int64_t d) { return head_kind == MTP_HEAD_Q4_STAGED && d % 64 == 0; }
static size_t lce_fwd_stage_offset(int64_t n, int64_t v) { return (lce_fwd_ws(n, v) + 255) / 256 * 256; }

size_t mtp_lce_fwd_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind) {
  if (n < 1 || v < 1 || d < 1) return 0;
  if (fwd_staged(head_kind, d))
    return lce_fwd_stage_offset(n, v) + (size_t)mtp::lce_fwd_stage_rows_max((long)n, (long)v) * (size_t)d * 2;
  return lce_fwd_ws(n, v);
}

size_t mtp_lce_fwd_stage_workspace_bytes(int64_t n, int64_t d, int64_t v, size_t budget_bytes) {
  if (n < 1 || v < 1 || d < 1 || d % 64 != 0) return 0;
  const size_t off = lce_fwd_stage_offset(n, v);
  long cap = budget_bytes > off ? (long)((budget_bytes - off) / ((size_t)d * 2)) : 0;
  const long least = mtp::lce_fwd_stage_rows_max((long)n, (long)v);
  if (cap < least) cap = least;
  // The largest run of whole splits the launcher forms with `cap` rows.
  return off + (size_t)mtp::lce_fwd_stage_rows_used((long)n, (long)v, cap) * (size_t)d * 2;
}

int mtp_lce_fwd(const void* hidden, const void* w, const uint32_t* w_q, const void* scales, const void* biases,
                const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                float* nll, float* lse, float* tgt, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_lce_common(hidden, w, w_q, scales, biases, targets, n, d, v, head_kind);
  if (rc) return rc;
  if (!nll || !lse || !tgt) return fail(MTP_ERR_INPUT, "nll, lse, tgt outputs must be non-null");
  const size_t need = mtp_lce_fwd_workspace_bytes(n, d, v, head_kind);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "lce forward needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  mtp::bf16_t* stage = nullptr;
  long stage_rows = 0;
  if (fwd_staged(head_kind, d)) {   // as many vocab rows as the workspace holds past the partials
    if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
    stage = reinterpret_cast<mtp::bf16_t*>(static_cast<char*>(workspace) + lce_fwd_stage_offset(n, v));
    stage_rows = (long)((workspace_bytes - lce_fwd_stage_offset(n, v)) / ((size_t)d * 2));
  }
  hipError_t e = mtp::launch_lce_fwd(make_head(w, w_q, scales, biases, head_kind), static_cast<const mtp::bf16_t*>(hidden),
                                     targets, (int)n, (int)d, (int)v, (long long)ignore_index, nll, lse, tgt,
                                     static_cast<float*>(workspace), stage, stage_rows, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "lce forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

size_t mtp_lce_fwd_noalloc_max_workspace_bytes(void) { return kNoAllocScratchBytes; }

int mtp_lce_fwd_noalloc(const void* hidden, const void* w, const uint32_t* w_q, const void* scales,
                        const void* biases, const int64_t* targets, int64_t n, int64_t d, int64_t v,
                        int32_t head_kind, int64_t ignore_index, float* nll, float* lse, float* tgt, void* stream) {
  int rc = check_lce_common(hidden, w, w_q, scales, biases, targets, n, d, v, head_kind);
  if (rc) return rc;
  if (!nll || !lse || !tgt) return fail(MTP_ERR_INPUT, "nll, lse, tgt outputs must be non-null");
  const size_t need = lce_fwd_ws(n, v);
  if (need > kNoAllocScratchBytes)
    return fail(MTP_ERR_WORKSPACE, "mtp_lce_fwd_noalloc: n=%lld, v=%lld needs %zu bytes of scratch, above its fixed "
                "%zu; use mtp_lce_fwd with a caller workspace", (long long)n, (long long)v, need, kNoAllocScratchBytes);
  void* ws = nullptr;
  rc = scratch_for_stream(static_cast<hipStream_t>(stream), &ws);
  if (rc) return rc;
  // Every partial the forward reads is written by the same launch before it is read (one entry
  // per vocab split and token), so the scratch needs no clearing between calls.
  hipError_t e = mtp::launch_lce_fwd(make_head(w, w_q, scales, biases, head_kind), static_cast<const mtp::bf16_t*>(hidden),
                                     targets, (int)n, (int)d, (int)v, (long long)ignore_index, nll, lse, tgt,
                                     static_cast<float*>(ws), nullptr, 0, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "lce forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int64_t mtp_lce_bwd_row_block(int64_t n, int64_t d, int64_t v, size_t budget_bytes) {
  if (n < 1 || d < 1 || v < 1) return 0;
  const int64_t vpad = round_up(v, kTile);
  const size_t row_bytes = (size_t)(vpad + mtp::kGPitchPad) * 2;  // one row of gradient tiles
  if ((size_t)n * row_bytes <= budget_bytes) return n;
  // Split the rows in 2 or 4 blocks while each block's whole-vocab G fits the budget and its dH
  // product keeps at least one 256 x 256 output tile per CU.
  for (int64_t parts = 2; parts <= 4; parts *= 2) {
    const int64_t rows = round_up((n + parts - 1) / parts, kTile);
    if ((rows / kTile) * ((d + kTile - 1) / kTile) < mtp::kNumCU) break;
    if ((size_t)rows * row_bytes <= budget_bytes) return rows;
  }
  // Otherwise the vocab is chunked, with an fp32 dH read-modify-write per chunk. Past 4 chunks,
  // 8 or 16 smaller row blocks whose dH products split their contraction (lce_dh_ksplit) instead
  // measured faster (N = 30720, D = 2048, 7 chunks: 50.0 against 52.1 ms); at 3 chunks the chunked
  // plan was (N = 12288, D = 4096: 34.7 ms against 35.4 for 4 blocks and 36.4 for 8).
  const int64_t chunk = mtp_lce_bwd_chunk(n, d, v, budget_bytes);
  if ((v + chunk - 1) / chunk > 4) {
    for (int64_t parts = 8; parts <= 16; parts *= 2) {
      const int64_t rows = round_up((n + parts - 1) / parts, kTile);
      if ((size_t)rows * row_bytes <= budget_bytes) return rows;
    }
  }
  return n;
}

int64_t mtp_lce_bwd_chunk(int64_t n, int64_t d, int64_t v, size_t budget_bytes) {
  if (n < 1 || d < 1 || v < 1) return 0;
  const int64_t vpad = round_up(v, kTile);
  // All n rows in one block: one chunk if the whole padded vocab fits the budget; otherwise the
  // budget also carries the fp32 dH accumulator. Gradient-tile rows are chunk + kGPitchPad
  // elements apart.
  if ((size_t)n * (size_t)(vpad + mtp::kGPitchPad) * 2 <= budget_bytes) return vpad;
  const size_t acc = (size_t)n * (size_t)d * 4;
  const size_t rest = budget_bytes > acc ? budget_bytes - acc : 0;
  int64_t c = ((int64_t)(rest / ((size_t)n * 2)) - mtp::kGPitchPad) / kTile * kTile;
  if (c < kTile) c = kTile;
  if (c > vpad) c = vpad;
  return c;
}

// Bytes of the fp32 part tiles of a split dH product: the most any (row block, vocab chunk) of the
// backward takes (the last row block and the last chunk may be shorter and split otherwise).
static size_t lce_dh_parts_max(int64_t n, int64_t d, int64_t v, int64_t chunk, int64_t row_block) {
  const int64_t last_rows = n - (n - 1) / row_block * row_block;
  const int64_t last_tiles = (v - (v - 1) / chunk * chunk + kTile - 1) / kTile;
  size_t most = 0;
  for (int64_t rows : {row_block, last_rows})
    for (int64_t kt : {chunk / kTile, last_tiles}) {
      const size_t b = mtp::lce_dh_parts_bytes((long)rows, (long)d, (long)kt);
      if (b > most) most = b;
    }
  return most;
}

// Gradient tiles [row_block][chunk + kGPitchPad] bf16, then the fp32 dH accumulator
// [row_block][d] when the vocab takes more than one chunk, then the split dH's fp32 part tiles.
static size_t lce_bwd_acc_offset(int64_t chunk, int64_t row_block) {
  return (size_t)row_block * (size_t)(chunk + mtp::kGPitchPad) * 2;
}
static size_t lce_bwd_parts_offset(int64_t d, int64_t v, int64_t chunk, int64_t row_block) {
  const int64_t nchunks = (v + chunk - 1) / chunk;
  return lce_bwd_acc_offset(chunk, row_block) + (nchunks > 1 ? (size_t)row_block * (size_t)d * 4 : 0);
}

static bool staged_kind(int32_t head_kind) { return head_kind == MTP_HEAD_Q4_STAGED || head_kind == MTP_HEAD_DENSE_STAGED; }

// The staging buffer of the MTP_HEAD_*_STAGED kinds: one chunk of the head, transposed (a 4-bit head
// dequantized), [d][lce_head_t_ld(chunk)] bf16, after the part tiles (256-byte aligned); for a 4-bit
// head the chunk's dequantized rows [chunk][d] bf16 follow (mtp::lce_stage_rows_offset).
static size_t lce_bwd_stage_offset(int64_t n, int64_t d, int64_t v, int64_t chunk, int64_t row_block) {
  return (lce_bwd_parts_offset(d, v, chunk, row_block) + lce_dh_parts_max(n, d, v, chunk, row_block) + 255) / 256 * 256;
}
static bool stage_rows(int32_t head_kind) { return head_kind == MTP_HEAD_Q4_STAGED && mtp::kQ4StageRows; }
static size_t lce_bwd_stage_bytes(int64_t d, int64_t chunk, int32_t head_kind) {
  if (stage_rows(head_kind)) return ((size_t)mtp::lce_stage_rows_offset((long)d, (long)chunk) + (size_t)chunk * (size_t)d) * 2;
  return (size_t)d * (size_t)mtp::lce_head_t_ld((long)chunk) * 2;
}

size_t mtp_lce_bwd_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t chunk,
                                   int64_t row_block) {
  if (n < 1 || d < 1 || v < 1 || chunk < kTile || chunk % kTile) return 0;
  if (chunk > round_up(v, kTile)) chunk = round_up(v, kTile);
  if (row_block < 1 || row_block > n) row_block = n;
  if (staged_kind(head_kind))
    return lce_bwd_stage_offset(n, d, v, chunk, row_block) + lce_bwd_stage_bytes(d, chunk, head_kind);
  return lce_bwd_parts_offset(d, v, chunk, row_block) + lce_dh_parts_max(n, d, v, chunk, row_block);
}

int64_t mtp_lce_bwd_stage_chunk(int64_t n, int64_t d, int64_t v, int32_t head_kind, size_t budget_bytes) {
  if (n < 1 || d < 1 || v < 1 || !staged_kind(head_kind)) return 0;
  const int64_t vpad = round_up(v, kTile);
  // All n rows in one block. Per vocab column the gradient tiles take 2 n bytes and the staged head
  // chunk 2 d (4 d with a 4-bit chunk's dequantized rows); one chunk if the whole padded vocab fits,
  // otherwise the budget also carries the fp32 dH accumulator.
  const size_t per_col = (size_t)2 * (size_t)(n + d) + (stage_rows(head_kind) ? (size_t)2 * (size_t)d : 0);
  if (per_col * (size_t)(vpad + mtp::kGPitchPad) <= budget_bytes) return vpad;
  const size_t acc = (size_t)n * (size_t)d * 4;
  const size_t rest = budget_bytes > acc ? budget_bytes - acc : 0;
  int64_t c = ((int64_t)(rest / per_col) - mtp::kGPitchPad) / kTile * kTile;
  if (c < kTile) c = kTile;
  if (c > vpad) c = vpad;
  return c;
}

int64_t mtp_lce_head_t_ld(int64_t v) { return v < 1 ? 0 : (int64_t)mtp::lce_head_t_ld((long)v); }

int mtp_lce_head_transpose(const void* w, const uint32_t* w_q, const void* scales, const void* biases, int64_t v,
                           int64_t d, int32_t head_kind, void* w_t, void* stream) {
  if (v < 1 || d < 1 || v > kMaxDim || d > kMaxDim) return fail(MTP_ERR_INPUT, "v, d must be in [1, 2^31) (got v=%lld d=%lld)", (long long)v, (long long)d);
  if (!w_t) return fail(MTP_ERR_INPUT, "w_t must be non-null");
  if (!aligned16(w_t)) return fail(MTP_ERR_UNSUPPORTED, "w_t must be 16-byte aligned");
  if (head_kind == MTP_HEAD_DENSE) {
    if (!w) return fail(MTP_ERR_INPUT, "dense head: w must be non-null");
    if (!aligned16(w)) return fail(MTP_ERR_UNSUPPORTED, "dense head: w must be 16-byte aligned");
    if (d % 8 != 0) return fail(MTP_ERR_UNSUPPORTED, "head transpose requires d %% 8 == 0 (got d=%lld)", (long long)d);
  } else if (head_kind == MTP_HEAD_Q4) {
    if (!w_q || !scales || !biases) return fail(MTP_ERR_INPUT, "quantized head: w_q, scales and biases must be non-null");
    if (d % 64 != 0) return fail(MTP_ERR_UNSUPPORTED, "quantized head transpose requires d %% 64 == 0 (got d=%lld)", (long long)d);
  } else {
    return fail(MTP_ERR_UNSUPPORTED, "unknown head_kind %d", (int)head_kind);
  }
  hipError_t e = mtp::launch_lce_head_transpose(make_head(w, w_q, scales, biases, head_kind), (int)v, (int)d,
                                                static_cast<mtp::bf16_t*>(w_t), static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "head transpose launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_lce_bwd(const void* hidden, const void* w, const void* w_t, const uint32_t* w_q, const void* scales,
                const void* biases, const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind,
                int64_t ignore_index, const float* lse, const float* d_nll, void* d_hidden, void* d_w, int64_t chunk,
                int64_t row_block, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_lce_common(hidden, w, w_q, scales, biases, targets, n, d, v, head_kind);
  if (rc) return rc;
  if (w_t && !aligned16(w_t)) return fail(MTP_ERR_UNSUPPORTED, "w_t must be 16-byte aligned");
  if (!lse || !d_nll || !d_hidden) return fail(MTP_ERR_INPUT, "lse, d_nll and d_hidden must be non-null");
  if (!aligned16(d_hidden) || (d_w && !aligned16(d_w)))
    return fail(MTP_ERR_UNSUPPORTED, "d_hidden and d_w must be 16-byte aligned");
  if (d_w && head_kind != MTP_HEAD_DENSE && head_kind != MTP_HEAD_DENSE_STAGED)
    return fail(MTP_ERR_UNSUPPORTED, "a quantized head is frozen: d_w must be null");
  if (w_t && staged_kind(head_kind))
    return fail(MTP_ERR_INPUT, "the staged head kinds transpose the head chunk-wise: w_t must be null");
  if (chunk < kTile || chunk % kTile) return fail(MTP_ERR_INPUT, "chunk must be a positive multiple of 256 (got %lld)", (long long)chunk);
  if (chunk > round_up(v, kTile)) chunk = round_up(v, kTile);
  if (row_block == 0 || row_block > n) row_block = n;
  if (row_block < n && (row_block < 0 || row_block % kTile))
    return fail(MTP_ERR_INPUT, "row_block must be 0, >= n, or a positive multiple of 256 (got %lld)", (long long)row_block);
  if (d_w && row_block < n)
    return fail(MTP_ERR_INPUT, "a trainable head (d_w) sums over every row: row_block must cover all n=%lld rows", (long long)n);
  const size_t need = mtp_lce_bwd_workspace_bytes(n, d, v, head_kind, chunk, row_block);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "lce backward needs a workspace of %zu bytes at chunk=%lld, row_block=%lld (got %zu)", need, (long long)chunk, (long long)row_block, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  mtp::bf16_t* gbuf = static_cast<mtp::bf16_t*>(workspace);
  float* acc32 = reinterpret_cast<float*>(static_cast<char*>(workspace) + lce_bwd_acc_offset(chunk, row_block));
  float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + lce_bwd_parts_offset(d, v, chunk, row_block));
  mtp::bf16_t* stage = staged_kind(head_kind)
                           ? reinterpret_cast<mtp::bf16_t*>(static_cast<char*>(workspace) +
                                                            lce_bwd_stage_offset(n, d, v, chunk, row_block))
                           : nullptr;
  mtp::LceHead head = make_head(w, w_q, scales, biases, head_kind);
  head.wt = static_cast<const mtp::bf16_t*>(w_t);
  hipError_t e = mtp::launch_lce_bwd(head, static_cast<const mtp::bf16_t*>(hidden),
                                     targets, lse, d_nll, (int)n, (int)d, (int)v, (long long)ignore_index, (int)chunk,
                                     (int)row_block,
                                     static_cast<mtp::bf16_t*>(d_hidden), static_cast<mtp::bf16_t*>(d_w), gbuf, acc32,
                                     parts, stage, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "lce backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_lce_mean(const float* nll, const int64_t* targets, int64_t n, int64_t ignore_index, float* mean, float* count,
                 void* stream) {
  if (n < 1 || n > kMaxDim) return fail(MTP_ERR_INPUT, "n must be in [1, 2^31) (got n=%lld)", (long long)n);
  if (!nll || !targets || !mean || !count) return fail(MTP_ERR_INPUT, "nll, targets, mean and count must be non-null");
  hipError_t e = mtp::launch_lce_mean(nll, targets, (long)n, (long long)ignore_index, mean, count, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "lce mean launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_lce_mean_bwd(const float* d_mean, const float* count, int64_t n, float* d_nll, void* stream) {
  if (n < 1 || n > kMaxDim) return fail(MTP_ERR_INPUT, "n must be in [1, 2^31) (got n=%lld)", (long long)n);
  if (!d_mean || !count || !d_nll) return fail(MTP_ERR_INPUT, "d_mean, count and d_nll must be non-null");
  hipError_t e = mtp::launch_lce_mean_bwd(d_mean, count, (long)n, d_nll, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "lce mean backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_attn_fwd(const void* q, const void* k, const void* v, int64_t b, int64_t hq, int64_t hkv, int64_t s,
                 int64_t dh, float scale, int32_t causal, const int32_t* seg_id, const int32_t* seg_start, void* o,
                 float* lse, void* stream) {
  int rc = check_attn(q, k, v, b, hq, hkv, s, dh, causal, seg_id, seg_start);
  if (rc) return rc;
  if (!o || !lse) return fail(MTP_ERR_INPUT, "o and lse must be non-null");
  if (!aligned16(o)) return fail(MTP_ERR_UNSUPPORTED, "o must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  hipError_t e = mtp::launch_attn_fwd(sh, static_cast<const mtp::bf16_t*>(q), static_cast<const mtp::bf16_t*>(k),
                                      static_cast<const mtp::bf16_t*>(v), seg_id, seg_start,
                                      static_cast<mtp::bf16_t*>(o), lse, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "attention forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

size_t mtp_attn_bwd_workspace_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn_bwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
}

int mtp_attn_bwd_dkv_splits(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh, int32_t causal) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn_dkv_nsplit((int)b, (int)hq, (int)hkv, (int)s, (int)dh, causal ? 1 : 0);
}

int mtp_attn_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* d_o,
                 int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh, float scale, int32_t causal,
                 const int32_t* seg_id, const int32_t* seg_start, void* d_q, void* d_k, void* d_v, void* workspace,
                 size_t workspace_bytes, void* stream) {
  int rc = check_attn(q, k, v, b, hq, hkv, s, dh, causal, seg_id, seg_start);
  if (rc) return rc;
  if (!o || !lse || !d_o || !d_q || !d_k || !d_v) return fail(MTP_ERR_INPUT, "o, lse, d_o, d_q, d_k, d_v must be non-null");
  if (!aligned16(o) || !aligned16(d_o) || !aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v))
    return fail(MTP_ERR_UNSUPPORTED, "o, d_o, d_q, d_k, d_v must be 16-byte aligned");
  const size_t need = mtp_attn_bwd_workspace_bytes(b, hq, hkv, s, dh);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "attention backward needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  hipError_t e = mtp::launch_attn_bwd(sh, static_cast<const mtp::bf16_t*>(q), static_cast<const mtp::bf16_t*>(k),
                                      static_cast<const mtp::bf16_t*>(v), static_cast<const mtp::bf16_t*>(o), lse,
                                      static_cast<const mtp::bf16_t*>(d_o), seg_id, seg_start,
                                      static_cast<mtp::bf16_t*>(d_q), static_cast<mtp::bf16_t*>(d_k),
                                      static_cast<mtp::bf16_t*>(d_v), static_cast<float*>(workspace),
                                      static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "attention backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

// ---------------------------------------------------------------------------------------------
// fp32 inputs
// ---------------------------------------------------------------------------------------------

static int check_lce32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales,
                       const float* biases, const int64_t* targets, int64_t n, int64_t d, int64_t v,
                       int32_t head_kind) {
  if (n < 1 || d < 1 || v < 1) return fail(MTP_ERR_INPUT, "n, d, v must be >= 1 (got n=%lld d=%lld v=%lld)", (long long)n, (long long)d, (long long)v);
  if (n > kMaxDim || d > kMaxDim || v > kMaxDim || n * d > (int64_t(1) << 40)) return fail(MTP_ERR_INPUT, "n, d, v must each be < 2^31");
  if (!hidden || !targets) return fail(MTP_ERR_INPUT, "hidden and targets must be non-null");
  if (!aligned16(hidden)) return fail(MTP_ERR_UNSUPPORTED, "hidden must be 16-byte aligned");
  if (head_kind == MTP_HEAD_DENSE) {
    if (!w) return fail(MTP_ERR_INPUT, "dense head: w must be non-null");
    if (!aligned16(w)) return fail(MTP_ERR_UNSUPPORTED, "dense head: w must be 16-byte aligned");
  } else if (head_kind == MTP_HEAD_Q4) {
    if (!w_q || !scales || !biases) return fail(MTP_ERR_INPUT, "quantized head: w_q, scales and biases must be non-null");
    if (d % 64 != 0) return fail(MTP_ERR_UNSUPPORTED, "kernel impl requires the quantized head's hidden dim to be a multiple of 64 (got d=%lld); use impl='chunked'", (long long)d);
  } else {
    return fail(MTP_ERR_UNSUPPORTED, "unknown head_kind %d", (int)head_kind);
  }
  return MTP_OK;
}

static mtp::LceHead32 make_head32(const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                                  int32_t head_kind) {
  return mtp::LceHead32{head_kind == MTP_HEAD_Q4, w, w_q, scales, biases};
}

size_t mtp_lce_fwd_f32_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind) {
  (void)d;
  (void)head_kind;
  if (n < 1 || v < 1) return 0;
  return (size_t)2 * (size_t)mtp::lce32_fwd_nsplit((long)n, (long)v) * (size_t)n * sizeof(float);
}

int mtp_lce_fwd_f32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                    const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                    float* nll, float* lse, float* tgt, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_lce32(hidden, w, w_q, scales, biases, targets, n, d, v, head_kind);
  if (rc) return rc;
  if (!nll || !lse || !tgt) return fail(MTP_ERR_INPUT, "nll, lse, tgt outputs must be non-null");
  const size_t need = mtp_lce_fwd_f32_workspace_bytes(n, d, v, head_kind);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "fp32 lce forward needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  hipError_t e = mtp::launch_lce32_fwd(make_head32(w, w_q, scales, biases, head_kind), hidden, targets, (int)n, (int)d,
                                       (int)v, (long long)ignore_index, nll, lse, tgt, static_cast<float*>(workspace),
                                       static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "fp32 lce forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int64_t mtp_lce_bwd_f32_chunk(int64_t n, int64_t d, int64_t v, size_t budget_bytes) {
  (void)d;
  if (n < 1 || v < 1) return 0;
  const int64_t vpad = round_up(v, 128);
  int64_t c = ((int64_t)(budget_bytes / ((size_t)n * 4)) - 4) / 128 * 128;
  if (c < 128) c = 128;
  return c > vpad ? vpad : c;
}

size_t mtp_lce_bwd_f32_workspace_bytes(int64_t n, int64_t d, int64_t v, int64_t chunk) {
  if (n < 1 || v < 1 || chunk < 128 || chunk % 128) return 0;
  if (chunk > round_up(v, 128)) chunk = round_up(v, 128);
  const int np = mtp::lce32_dh_parts((long)n, (long)d, (long)(chunk < v ? chunk : v), nullptr);
  return (size_t)n * (size_t)(chunk + 4) * sizeof(float) + (np > 1 ? (size_t)np * (size_t)n * (size_t)d * sizeof(float) : 0);
}

int mtp_lce_bwd_f32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                    const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                    const float* lse, const float* d_nll, float* d_hidden, float* d_w, int64_t chunk, void* workspace,
                    size_t workspace_bytes, void* stream) {
  int rc = check_lce32(hidden, w, w_q, scales, biases, targets, n, d, v, head_kind);
  if (rc) return rc;
  if (!lse || !d_nll || !d_hidden) return fail(MTP_ERR_INPUT, "lse, d_nll and d_hidden must be non-null");
  if (d_w && head_kind != MTP_HEAD_DENSE) return fail(MTP_ERR_UNSUPPORTED, "a quantized head is frozen: d_w must be null");
  if (chunk < 128 || chunk % 128) return fail(MTP_ERR_INPUT, "chunk must be a positive multiple of 128 (got %lld)", (long long)chunk);
  if (chunk > round_up(v, 128)) chunk = round_up(v, 128);
  const size_t need = mtp_lce_bwd_f32_workspace_bytes(n, d, v, chunk);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "fp32 lce backward needs a workspace of %zu bytes at chunk=%lld (got %zu)", need, (long long)chunk, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  hipError_t e = mtp::launch_lce32_bwd(make_head32(w, w_q, scales, biases, head_kind), hidden, targets, lse, d_nll, (int)n,
                                       (int)d, (int)v, (long long)ignore_index, (int)chunk, d_hidden, d_w,
                                       static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "fp32 lce backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_attn_fwd_f32(const float* q, const float* k, const float* v, int64_t b, int64_t hq, int64_t hkv, int64_t s,
                     int64_t dh, float scale, int32_t causal, const int32_t* seg_id, const int32_t* seg_start, float* o,
                     float* lse, void* stream) {
  int rc = check_attn(q, k, v, b, hq, hkv, s, dh, causal, seg_id, seg_start);
  if (rc) return rc;
  if (!o || !lse) return fail(MTP_ERR_INPUT, "o and lse must be non-null");
  if (!aligned16(o)) return fail(MTP_ERR_UNSUPPORTED, "o must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  hipError_t e = mtp::launch_attn32_fwd(sh, q, k, v, seg_start, o, lse, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "fp32 attention forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

size_t mtp_attn_bwd_f32_workspace_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  const int ns = mtp::attn32_dkv_splits((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
  return mtp::attn32_bwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh, ns);
}

int mtp_attn_bwd_f32(const float* q, const float* k, const float* v, const float* o, const float* lse, const float* d_o,
                     int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh, float scale, int32_t causal,
                     const int32_t* seg_id, const int32_t* seg_start, float* d_q, float* d_k, float* d_v,
                     void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_attn(q, k, v, b, hq, hkv, s, dh, causal, seg_id, seg_start);
  if (rc) return rc;
  if (!o || !lse || !d_o || !d_q || !d_k || !d_v) return fail(MTP_ERR_INPUT, "o, lse, d_o, d_q, d_k, d_v must be non-null");
  if (!aligned16(o) || !aligned16(d_o) || !aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v))
    return fail(MTP_ERR_UNSUPPORTED, "o, d_o, d_q, d_k, d_v must be 16-byte aligned");
  // D is all it needs; a workspace without room for the split's partials runs the dK/dV pass unsplit.
  const size_t need = mtp::attn32_bwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh, 1);
  const bool split = workspace_bytes >= mtp_attn_bwd_f32_workspace_bytes(b, hq, hkv, s, dh);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "fp32 attention backward needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  const int ns = split ? mtp::attn32_dkv_splits(sh.b, sh.hq, sh.hkv, sh.s, sh.dh) : 1;
  hipError_t e = mtp::launch_attn32_bwd(sh, q, k, v, o, lse, d_o, seg_start, d_q, d_k, d_v,
                                        static_cast<float*>(workspace), ns, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "fp32 attention backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

// ---------------------------------------------------------------------------------------------
// Attention with capped scores, a bias by distance and key spans
// ---------------------------------------------------------------------------------------------

int mtp_attn_scored_fwd(const void* q, const void* k, const void* v, int64_t b, int64_t hq, int64_t hkv, int64_t s,
                        int64_t dh, float scale, int32_t causal, float softcap, const float* slopes,
                        const int32_t* span_start, const int32_t* span_end, void* o, int8_t* o_low, int32_t* plan,
                        float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_scored(q, k, v, b, hq, hkv, s, dh, scale, causal, softcap, slopes, span_start, span_end);
  if (rc) return rc;
  if (!o || !lse) return fail(MTP_ERR_INPUT, "o and lse must be non-null");
  if (!aligned16(o) || !aligned16(o_low) || !aligned16(plan) || !aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "o, o_low, plan and workspace must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  mtp::AttnScore sc{softcap, slopes, span_start, span_end};
  hipError_t e = mtp::launch_attn_scored_fwd(sh, sc, static_cast<const mtp::bf16_t*>(q), static_cast<const mtp::bf16_t*>(k),
                                             static_cast<const mtp::bf16_t*>(v), static_cast<mtp::bf16_t*>(o), o_low, plan, lse,
                                             workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "scored attention forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_attn_scored_fwd_f32(const float* q, const float* k, const float* v, int64_t b, int64_t hq, int64_t hkv, int64_t s,
                            int64_t dh, float scale, int32_t causal, float softcap, const float* slopes,
                            const int32_t* span_start, const int32_t* span_end, float* o, float* lse, void* workspace,
                            size_t workspace_bytes, void* stream) {
  int rc = check_scored(q, k, v, b, hq, hkv, s, dh, scale, causal, softcap, slopes, span_start, span_end);
  if (rc) return rc;
  if (!o || !lse) return fail(MTP_ERR_INPUT, "o and lse must be non-null");
  if (!aligned16(o)) return fail(MTP_ERR_UNSUPPORTED, "o must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  mtp::AttnScore sc{softcap, slopes, span_start, span_end};
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  hipError_t e = mtp::launch_attn32_scored_fwd(sh, sc, q, k, v, o, lse, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "fp32 scored attention forward launch failed: %s", hipGetErrorString(e));
  return ok();
}

size_t mtp_attn_scored_fwd_f32_workspace_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn32_scored_fwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
}

size_t mtp_attn_scored_bwd_f32_workspace_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn32_scored_bwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
}

size_t mtp_attn_scored_fwd_workspace_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn_scored_fwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
}

size_t mtp_attn_scored_plan_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn_scored_plan((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
}

size_t mtp_attn_scored_bwd_workspace_bytes(int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh) {
  if (b < 1 || hq < 1 || hkv < 1 || s < 1 || hq % hkv || b * hq * s > kMaxDim) return 0;
  return mtp::attn_scored_bwd_workspace((int)b, (int)hq, (int)hkv, (int)s, (int)dh);
}

int mtp_attn_scored_bwd(const void* q, const void* k, const void* v, const void* o, const int8_t* o_low,
                        const int32_t* plan, const float* lse, const void* d_o, int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh, float scale, int32_t causal,
                        float softcap, const float* slopes, const int32_t* span_start, const int32_t* span_end, void* d_q,
                        void* d_k, void* d_v, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_scored(q, k, v, b, hq, hkv, s, dh, scale, causal, softcap, slopes, span_start, span_end);
  if (rc) return rc;
  if (!o || !o_low || !lse || !d_o || !d_q || !d_k || !d_v) return fail(MTP_ERR_INPUT, "o, o_low, lse, d_o, d_q, d_k, d_v must be non-null");
  if (!aligned16(o) || !aligned16(o_low) || !aligned16(plan) || !aligned16(d_o) || !aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v))
    return fail(MTP_ERR_UNSUPPORTED, "o, o_low, plan, d_o, d_q, d_k, d_v must be 16-byte aligned");
  const size_t need = mtp_attn_scored_bwd_workspace_bytes(b, hq, hkv, s, dh);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "scored attention backward needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  mtp::AttnScore sc{softcap, slopes, span_start, span_end};
  hipError_t e = mtp::launch_attn_scored_bwd(sh, sc, static_cast<const mtp::bf16_t*>(q), static_cast<const mtp::bf16_t*>(k),
                                             static_cast<const mtp::bf16_t*>(v), static_cast<const mtp::bf16_t*>(o), o_low, plan, lse,
                                             static_cast<const mtp::bf16_t*>(d_o), static_cast<mtp::bf16_t*>(d_q),
                                             static_cast<mtp::bf16_t*>(d_k), static_cast<mtp::bf16_t*>(d_v), workspace,
                                             static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "scored attention backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_attn_scored_bwd_f32(const float* q, const float* k, const float* v, const float* o, const float* lse,
                            const float* d_o, int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t dh, float scale,
                            int32_t causal, float softcap, const float* slopes, const int32_t* span_start,
                            const int32_t* span_end, float* d_q, float* d_k, float* d_v, void* workspace,
                            size_t workspace_bytes, void* stream) {
  int rc = check_scored(q, k, v, b, hq, hkv, s, dh, scale, causal, softcap, slopes, span_start, span_end);
  if (rc) return rc;
  if (!o || !lse || !d_o || !d_q || !d_k || !d_v) return fail(MTP_ERR_INPUT, "o, lse, d_o, d_q, d_k, d_v must be non-null");
  if (!aligned16(o) || !aligned16(d_o) || !aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v))
    return fail(MTP_ERR_UNSUPPORTED, "o, d_o, d_q, d_k, d_v must be 16-byte aligned");
  // D is all it needs; a pass without room for its partials runs unsplit.
  const size_t need = (size_t)b * hq * s * sizeof(float);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "fp32 scored attention backward needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  mtp::AttnShape sh{(int)b, (int)hq, (int)hkv, (int)s, (int)dh, scale, (int)causal};
  mtp::AttnScore sc{softcap, slopes, span_start, span_end};
  hipError_t e = mtp::launch_attn32_scored_bwd(sh, sc, q, k, v, o, lse, d_o, d_q, d_k, d_v, workspace, workspace_bytes,
                                               static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "fp32 scored attention backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

// ---------------------------------------------------------------------------------------------
// Preference and policy losses
// ---------------------------------------------------------------------------------------------

size_t mtp_pref_workspace_bytes(int64_t pairs, int64_t n) {
  return pairs < 1 || pairs > (int64_t(1) << 23) || n < 1 || n > kMaxLossTokens ? 0 : mtp::pref_workspace((long)pairs, (long)n);
}

int mtp_pref_fwd(const float* nll, const float* ref_nll, const uint8_t* mask, const int64_t* offsets, int64_t pairs, int64_t n,
                 int32_t kind, double beta, double label_smoothing, int32_t reduction, float* loss, float* rewards,
                 float* coef, void* workspace, size_t workspace_bytes, void* stream) {
  if (pairs < 1) return fail(MTP_ERR_INPUT, "pairs must be >= 1 (got %lld)", (long long)pairs);
  int rc = check_rows(pairs > (int64_t(1) << 24) ? pairs : 2 * pairs, n, offsets);
  if (rc) return rc;
  if (!nll || !ref_nll || !loss || !rewards || !coef) return fail(MTP_ERR_INPUT, "nll, ref_nll, loss, rewards and coef must be non-null");
  if (kind < MTP_PREF_SIGMOID || kind > MTP_PREF_IPO) return fail(MTP_ERR_INPUT, "unknown kind %d of a preference loss", (int)kind);
  if (!(beta > 0.0 && beta < HUGE_VAL)) return fail(MTP_ERR_INPUT, "beta must be positive and finite (got %g)", beta);
  if (!(label_smoothing >= 0.0 && label_smoothing < 0.5)) return fail(MTP_ERR_INPUT, "label_smoothing must be in [0, 0.5) (got %g)", label_smoothing);
  if (label_smoothing != 0.0 && kind != MTP_PREF_SIGMOID) return fail(MTP_ERR_INPUT, "label_smoothing belongs to the sigmoid loss");
  if (reduction != MTP_REDUCE_NONE && reduction != MTP_REDUCE_MEAN && reduction != MTP_REDUCE_SUM)
    return fail(MTP_ERR_INPUT, "unknown reduction %d of a preference loss", (int)reduction);
  const size_t need = mtp_pref_workspace_bytes(pairs, n);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "the preference loss needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  hipError_t e = mtp::launch_pref_fwd(nll, ref_nll, mask, offsets, (long)pairs, (long)n,
                                      mtp::PrefLoss{kind, reduction, beta, label_smoothing}, loss, rewards, coef, workspace,
                                      static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "preference loss launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_pref_bwd(const float* d_loss, const float* coef, const uint8_t* mask, const int64_t* offsets, int64_t pairs, int64_t n,
                 int32_t reduction, float* d_nll, void* stream) {
  if (pairs < 1) return fail(MTP_ERR_INPUT, "pairs must be >= 1 (got %lld)", (long long)pairs);
  int rc = check_rows(pairs > (int64_t(1) << 24) ? pairs : 2 * pairs, n, offsets);
  if (rc) return rc;
  if (!d_loss || !coef || !d_nll) return fail(MTP_ERR_INPUT, "d_loss, coef and d_nll must be non-null");
  hipError_t e = mtp::launch_pref_bwd(d_loss, coef, mask, offsets, (long)pairs, (long)n, reduction == MTP_REDUCE_NONE, d_nll,
                                      static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "preference loss backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

size_t mtp_policy_workspace_bytes(int64_t rows, int64_t n) {
  return rows < 1 || rows > (int64_t(1) << 24) || n < 1 || n > kMaxLossTokens ? 0 : mtp::policy_workspace((long)rows, (long)n);
}

int mtp_policy_fwd(const float* nll, const float* old_nll, const float* ref_nll, const float* advantages,
                   int32_t adv_per_token, const uint8_t* mask, const int64_t* offsets, int64_t rows, int64_t n,
                   double clip_low, double clip_high, double kl_coef, int32_t reduction, float* loss, float* stats,
                   float* weight, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_rows(rows, n, offsets);
  if (rc) return rc;
  if (!nll || !old_nll || !advantages || !loss || !stats || !weight)
    return fail(MTP_ERR_INPUT, "nll, old_nll, advantages, loss, stats and weight must be non-null");
  mtp::PolicyLoss p;
  rc = policy_params(&p, ref_nll, adv_per_token, clip_low, clip_high, kl_coef, reduction);
  if (rc) return rc;
  const size_t need = mtp_policy_workspace_bytes(rows, n);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "the policy loss needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  hipError_t e = mtp::launch_policy_fwd(nll, old_nll, ref_nll, advantages, mask, offsets, (long)rows, (long)n, p, loss, stats,
                                        weight, workspace, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "policy loss launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_policy_bwd(const float* d_loss, const float* nll, const float* old_nll, const float* ref_nll, const float* advantages,
                   int32_t adv_per_token, const uint8_t* mask, const int64_t* offsets, int64_t rows, int64_t n,
                   double clip_low, double clip_high, double kl_coef, int32_t reduction, const float* weight, float* d_nll,
                   void* stream) {
  int rc = check_rows(rows, n, offsets);
  if (rc) return rc;
  if (!d_loss || !nll || !old_nll || !advantages || !weight || !d_nll)
    return fail(MTP_ERR_INPUT, "d_loss, nll, old_nll, advantages, weight and d_nll must be non-null");
  mtp::PolicyLoss p;
  rc = policy_params(&p, ref_nll, adv_per_token, clip_low, clip_high, kl_coef, reduction);
  if (rc) return rc;
  hipError_t e = mtp::launch_policy_bwd(d_loss, nll, old_nll, ref_nll, advantages, mask, offsets, (long)rows, (long)n, p, weight,
                                        d_nll, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "policy loss backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

// ---------------------------------------------------------------------------------------------
// Token scoring and distillation
// ---------------------------------------------------------------------------------------------

static int check_score(int f32, int64_t d, int64_t v, double temperature) {
  if (!f32 && d >= mtp::kScoreDims) return fail(MTP_ERR_UNSUPPORTED, "token scoring and distillation serve fewer than 2^22 bf16 hidden dims (got d=%lld); use impl='reference'", (long long)d);
  if (v > mtp::kScoreVocab) return fail(MTP_ERR_UNSUPPORTED, "token scoring and distillation serve a vocabulary of at most 2^21 (got v=%lld); use impl='reference'", (long long)v);
  if (!(temperature >= 1e-3 && temperature <= 1e3)) return fail(MTP_ERR_INPUT, "temperature must be in [1e-3, 1e3] (got %g)", temperature);
  return MTP_OK;
}

static int check_list(int32_t k) {
  if (k < 1 || k > MTP_SCORE_MAX) return fail(MTP_ERR_UNSUPPORTED, "a teacher's list has 1 to %d slots (got k=%d); use impl='reference'", MTP_SCORE_MAX, (int)k);
  return MTP_OK;
}

static bool q4_kind(int32_t head_kind) { return head_kind == MTP_HEAD_Q4 || head_kind == MTP_HEAD_Q4_STAGED; }

static mtp::ScoreHead score_head(int f32, const void* hidden, const void* w, const uint32_t* w_q, const void* scales,
                                 const void* biases, int32_t head_kind) {
  mtp::ScoreHead h{};
  h.f32 = f32;
  h.hidden = hidden;
  if (f32)
    h.h32 = make_head32(static_cast<const float*>(w), w_q, static_cast<const float*>(scales), static_cast<const float*>(biases),
                        q4_kind(head_kind) ? MTP_HEAD_Q4 : head_kind);
  else
    h.h = make_head(w, w_q, scales, biases, head_kind);
  return h;
}

// check_lce_common / check_lce32 without a target of each token.
static int check_score_head(int f32, const void* hidden, const void* w, const uint32_t* w_q, const void* scales,
                            const void* biases, int64_t n, int64_t d, int64_t v, int32_t head_kind) {
  static const int64_t any = 0;
  if (f32)  // (staged: this section's alone)
    return check_lce32(static_cast<const float*>(hidden), static_cast<const float*>(w), w_q, static_cast<const float*>(scales),
                       static_cast<const float*>(biases), &any, n, d, v, head_kind == MTP_HEAD_Q4_STAGED ? MTP_HEAD_Q4 : head_kind);
  return check_lce_common(hidden, w, w_q, scales, biases, &any, n, d, v, head_kind);
}

static float log2e_over(double temperature) { return (float)(1.4426950408889634 / temperature); }
static mtp::ScoreShape score_shape(int64_t n, int64_t d, int64_t v, double temperature, int32_t head_kind) {
  return mtp::ScoreShape{(long)n, (long)d, (long)v, (float)(1.0 / temperature), log2e_over(temperature), head_kind == MTP_HEAD_Q4_STAGED};
}

static bool score_sizes(int64_t n, int64_t d, int64_t v) {
  return n >= 1 && d >= 1 && v >= 1 && n <= kMaxDim && d <= kMaxDim && v <= mtp::kScoreVocab;
}

int64_t mtp_score_logits_ld(int64_t v) { return v < 1 ? 0 : (int64_t)mtp::logits_ld((long)v); }

static size_t logprobs_fwd_ws(int f32, int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t top, int keep) {
  if (!score_sizes(n, d, v) || top < 0 || top > MTP_SCORE_MAX) return 0;
  return mtp::logprobs_fwd_workspace(score_shape(n, d, v, 1.0, head_kind), f32, q4_kind(head_kind), top, keep != 0);
}
size_t mtp_logprobs_fwd_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t top, int32_t keep) {
  return logprobs_fwd_ws(0, n, d, v, head_kind, top, keep);
}
size_t mtp_logprobs_fwd_f32_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t top, int32_t keep) {
  return logprobs_fwd_ws(1, n, d, v, head_kind, top, keep);
}

static int logprobs_fwd(int f32, const void* hidden, const void* w, const uint32_t* w_q, const void* scales, const void* biases,
                        const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                        int32_t top, double temperature, const mtp::LogprobsOut& out, void* workspace,
                        size_t workspace_bytes, void* stream) {
  int rc = check_score_head(f32, hidden, w, w_q, scales, biases, n, d, v, head_kind);
  if (rc) return rc;
  rc = check_score(f32, d, v, temperature);
  if (rc) return rc;
  if (top < 0 || top > v) return fail(MTP_ERR_INPUT, "top must be in [0, v=%lld] (got %d)", (long long)v, (int)top);
  if (top > MTP_SCORE_MAX) return fail(MTP_ERR_UNSUPPORTED, "at most %d alternatives (got top=%d); use impl='reference'", MTP_SCORE_MAX, (int)top);
  if (!out.entropy || !out.lse || (targets && (!out.logprobs || !out.tgt)) || (top && (!out.top_logprobs || !out.top_ids)))
    return fail(MTP_ERR_INPUT, "entropy and lse, with targets logprobs and tgt, with top top_logprobs and top_ids must be non-null");
  if (!aligned16(out.logits)) return fail(MTP_ERR_UNSUPPORTED, "logits must be 16-byte aligned");
  const size_t need = logprobs_fwd_ws(f32, n, d, v, head_kind, top, out.logits != nullptr);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "token scoring needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  const hipError_t e = mtp::launch_logprobs_fwd(score_head(f32, hidden, w, w_q, scales, biases, head_kind),
                                                score_shape(n, d, v, temperature, head_kind), targets, (long long)ignore_index,
                                                (int)top, out, workspace, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "token scoring launch failed: %s", hipGetErrorString(e));
  return ok();
}

int mtp_logprobs_fwd(const void* hidden, const void* w, const uint32_t* w_q, const void* scales, const void* biases,
                     const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                     int32_t top, double temperature, float* logprobs, float* entropy, float* top_logprobs,
                     int64_t* top_ids, float* lse, float* tgt, float* logits, void* workspace, size_t workspace_bytes,
                     void* stream) {
  return logprobs_fwd(0, hidden, w, w_q, scales, biases, targets, n, d, v, head_kind, ignore_index, top, temperature,
                      mtp::LogprobsOut{logprobs, entropy, top_logprobs, top_ids, lse, tgt, logits}, workspace, workspace_bytes, stream);
}
int mtp_logprobs_fwd_f32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                         const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                         int32_t top, double temperature, float* logprobs, float* entropy, float* top_logprobs,
                         int64_t* top_ids, float* lse, float* tgt, float* logits, void* workspace, size_t workspace_bytes,
                     void* stream) {
  return logprobs_fwd(1, hidden, w, w_q, scales, biases, targets, n, d, v, head_kind, ignore_index, top, temperature,
                      mtp::LogprobsOut{logprobs, entropy, top_logprobs, top_ids, lse, tgt, logits}, workspace, workspace_bytes, stream);
}

// Rows of G in the bf16 backward: two a token where that fills a row tile at most (AffineGrad's halves).
static int64_t score_g_rows(int64_t n) { return 2 * n <= kTile ? 2 * n : n; }
// After the loss's workspace (of score_g_rows rows): alpha [n], beta [n], the columns [n] of scoring, the values [n][k], the halves, the
// cleared hidden states, or an fp32 4-bit head's rows (staged bytes). g_rows: of G.
struct ScoreBwd {
  size_t alpha, beta, columns, value, halves, clean, bytes;
};
static ScoreBwd score_bwd_parts(size_t lce, int64_t n, int64_t g_rows, int64_t d, int32_t k, int32_t trainable, size_t elem, size_t staged) {
  auto pad = [](size_t x) { return (x + 255) / 256 * 256; };
  ScoreBwd p;
  p.alpha = pad(lce);
  p.beta = p.alpha + pad((size_t)n * 4);
  p.columns = p.beta + pad((size_t)n * 4);
  p.value = p.columns + pad((size_t)n * 4);
  p.halves = p.value + pad((size_t)n * k * 4);
  p.clean = p.halves + (g_rows > n ? pad((size_t)g_rows * d * 4) : 0);
  p.bytes = p.clean + (trainable ? (size_t)g_rows * d * elem : staged);
  return p;
}
size_t mtp_score_bwd_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t chunk, int64_t row_block,
                                     int32_t k, int32_t trainable) {
  const int64_t rows = score_g_rows(n);
  const size_t lce = mtp_lce_bwd_workspace_bytes(rows, d, v, head_kind, chunk, rows > n ? rows : row_block);
  return !lce || k < 1 || k > MTP_SCORE_MAX ? 0 : score_bwd_parts(lce, n, rows, d, k, trainable, 2, 0).bytes;
}
static size_t staged32_bytes(int64_t d, int64_t v, int32_t head_kind) { return head_kind == MTP_HEAD_Q4_STAGED ? (size_t)v * d * 4 : 0; }
size_t mtp_score_bwd_f32_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t chunk, int32_t k, int32_t trainable) {
  const size_t lce = mtp_lce_bwd_f32_workspace_bytes(n, d, v, chunk);
  return !lce || k < 1 || k > MTP_SCORE_MAX ? 0 : score_bwd_parts(lce, n, n, d, k, trainable, 4, staged32_bytes(d, v, head_kind)).bytes;
}

}  // extern "C"

// The shared backward: `factors` launches what fills alpha, beta (or none), columns and value.
template <class FACTORS>
static int score_bwd(int f32, const void* hidden, const void* w, const void* w_t, const uint32_t* w_q, const void* scales,
                     const void* biases, int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, double temperature,
                     const float* lse, const int32_t* columns, const float* logits, void* d_hidden, void* d_w, int64_t chunk,
                     int64_t row_block, void* workspace, size_t workspace_bytes, hipStream_t stream, const FACTORS& factors) {
  int rc = check_score_head(f32, hidden, w, w_q, scales, biases, n, d, v, head_kind);
  if (rc) return rc;
  rc = check_score(f32, d, v, temperature);
  if (rc) return rc;
  if (!lse || !d_hidden) return fail(MTP_ERR_INPUT, "lse and d_hidden must be non-null");
  if (!aligned16(d_hidden) || !aligned16(d_w) || !aligned16(w_t) || !aligned16(logits))
    return fail(MTP_ERR_UNSUPPORTED, "d_hidden, d_w, w_t and logits must be 16-byte aligned");
  if (d_w && q4_kind(head_kind)) return fail(MTP_ERR_UNSUPPORTED, "a quantized head is frozen: d_w must be null");
  if (w_t && (f32 || staged_kind(head_kind))) return fail(MTP_ERR_INPUT, "fp32 and the staged head kinds take no w_t");
  const int64_t tile = f32 ? 128 : kTile;
  if (chunk < tile || chunk % tile) return fail(MTP_ERR_INPUT, "chunk must be a positive multiple of %lld (got %lld)", (long long)tile, (long long)chunk);
  if (chunk > round_up(v, tile)) chunk = round_up(v, tile);
  if (row_block == 0 || row_block > n) row_block = n;
  if (row_block < n && (f32 || row_block < 0 || row_block % kTile))
    return fail(MTP_ERR_INPUT, "row_block must be 0, >= n, or (bf16) a positive multiple of 256 (got %lld)", (long long)row_block);
  if (d_w && row_block < n) return fail(MTP_ERR_INPUT, "a trainable head (d_w) sums over every row: row_block must cover all n=%lld rows", (long long)n);
  const int64_t g_rows = f32 ? n : score_g_rows(n);
  if (g_rows > n) row_block = g_rows;  // (all rows in one block)
  const size_t lce = f32 ? mtp_lce_bwd_f32_workspace_bytes(n, d, v, chunk) : mtp_lce_bwd_workspace_bytes(g_rows, d, v, head_kind, chunk, row_block);
  const ScoreBwd parts = score_bwd_parts(lce, n, g_rows, d, k, d_w != nullptr, f32 ? 4 : 2, f32 ? staged32_bytes(d, v, head_kind) : 0);
  if (!workspace || workspace_bytes < parts.bytes)
    return fail(MTP_ERR_WORKSPACE, "the backward needs a workspace of %zu bytes at chunk=%lld, row_block=%lld (got %zu)", parts.bytes, (long long)chunk, (long long)row_block, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  float* alpha = reinterpret_cast<float*>(ws + parts.alpha);
  float* beta = reinterpret_cast<float*>(ws + parts.beta);
  int* own_columns = reinterpret_cast<int*>(ws + parts.columns);
  float* value = reinterpret_cast<float*>(ws + parts.value);
  float* halves = logits && g_rows > n ? reinterpret_cast<float*>(ws + parts.halves) : nullptr;
  bool has_beta = false;
  hipError_t e = factors(alpha, beta, own_columns, value, &has_beta);
  if (e == hipSuccess && d_w)
    e = mtp::launch_clean_rows(hidden, alpha, has_beta ? beta : nullptr, (long)n, (long)d * (f32 ? 4 : 2), halves ? 2 : 1, ws + parts.clean, stream);
  if (e == hipSuccess) {
    const mtp::AffineGrad grad{{alpha, has_beta ? beta : nullptr, log2e_over(temperature)}, columns ? columns : own_columns, value, (int)k, logits, mtp::logits_ld((long)v), ws + parts.clean, halves};
    if (f32) {
      mtp::LceHead32 head = score_head(1, hidden, w, w_q, scales, biases, head_kind).h32;
      if (head_kind == MTP_HEAD_Q4_STAGED) {
        float* rows = reinterpret_cast<float*>(ws + parts.clean);
        e = mtp::launch_dequant32(head, (long)v, (long)d, rows, stream);
        if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "backward launch failed: %s", hipGetErrorString(e));
        head = mtp::LceHead32{0, rows, nullptr, nullptr, nullptr};
      }
      e = mtp::launch_lce32_bwd(head, static_cast<const float*>(hidden), nullptr, lse, nullptr, (int)n, (int)d, (int)v, 0, (int)chunk, static_cast<float*>(d_hidden),
                                static_cast<float*>(d_w), static_cast<float*>(workspace), stream, &grad);
    } else {
      mtp::LceHead head = make_head(w, w_q, scales, biases, head_kind);
      head.wt = static_cast<const mtp::bf16_t*>(w_t);
      mtp::bf16_t* stage = staged_kind(head_kind) ? reinterpret_cast<mtp::bf16_t*>(ws + lce_bwd_stage_offset(g_rows, d, v, chunk, row_block)) : nullptr;
      e = mtp::launch_lce_bwd(head, static_cast<const mtp::bf16_t*>(hidden), nullptr, lse, nullptr, (int)n, (int)d, (int)v, 0,
                              (int)chunk, (int)row_block, static_cast<mtp::bf16_t*>(d_hidden), static_cast<mtp::bf16_t*>(d_w),
                              static_cast<mtp::bf16_t*>(workspace),
                              reinterpret_cast<float*>(ws + lce_bwd_acc_offset(chunk, row_block)),
                              reinterpret_cast<float*>(ws + lce_bwd_parts_offset(d, v, chunk, row_block)), stage, stream, &grad);
    }
  }
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "backward launch failed: %s", hipGetErrorString(e));
  return ok();
}

extern "C" {

static int logprobs_bwd(int f32, const void* hidden, const void* w, const void* w_t, const uint32_t* w_q, const void* scales,
                        const void* biases, const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind,
                        int64_t ignore_index, double temperature, const float* lse, const float* entropy, const float* tgt,
                        const float* logits, const float* d_logprobs, const float* d_entropy, void* d_hidden, void* d_w, int64_t chunk,
                        int64_t row_block, void* workspace, size_t workspace_bytes, void* stream) {
  if (!entropy || (targets && !tgt)) return fail(MTP_ERR_INPUT, "entropy, and with targets tgt, must be non-null");
  if (d_logprobs && !targets) return fail(MTP_ERR_INPUT, "d_logprobs needs targets");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return score_bwd(f32, hidden, w, w_t, w_q, scales, biases, n, d, v, head_kind, 1, temperature, lse, nullptr, logits, d_hidden, d_w, chunk,
                   row_block, workspace, workspace_bytes, st, [&](float* alpha, float* beta, int* columns, float* value, bool* has_beta) {
                     *has_beta = d_entropy != nullptr;
                     return mtp::launch_logprobs_coef(d_logprobs, d_entropy, targets, (long long)ignore_index, lse, entropy, tgt,
                                                      (long)n, (long)v, (float)(1.0 / temperature), alpha, beta, columns, value, st);
                   });
}
int mtp_logprobs_bwd(const void* hidden, const void* w, const void* w_t, const uint32_t* w_q, const void* scales,
                     const void* biases, const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind,
                     int64_t ignore_index, double temperature, const float* lse, const float* entropy, const float* tgt,
                     const float* logits, const float* d_logprobs, const float* d_entropy, void* d_hidden, void* d_w, int64_t chunk,
                     int64_t row_block, void* workspace, size_t workspace_bytes, void* stream) {
  return logprobs_bwd(0, hidden, w, w_t, w_q, scales, biases, targets, n, d, v, head_kind, ignore_index, temperature, lse, entropy,
                      tgt, logits, d_logprobs, d_entropy, d_hidden, d_w, chunk, row_block, workspace, workspace_bytes, stream);
}
int mtp_logprobs_bwd_f32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                         const int64_t* targets, int64_t n, int64_t d, int64_t v, int32_t head_kind, int64_t ignore_index,
                         double temperature, const float* lse, const float* entropy, const float* tgt, const float* logits,
                         const float* d_logprobs, const float* d_entropy, float* d_hidden, float* d_w, int64_t chunk, void* workspace,
                         size_t workspace_bytes, void* stream) {
  return logprobs_bwd(1, hidden, w, nullptr, w_q, scales, biases, targets, n, d, v, head_kind, ignore_index, temperature, lse, entropy,
                      tgt, logits, d_logprobs, d_entropy, d_hidden, d_w, chunk, 0, workspace, workspace_bytes, stream);
}

static size_t distill_fwd_ws(int f32, int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, int keep) {
  if (!score_sizes(n, d, v) || k < 1 || k > MTP_SCORE_MAX) return 0;
  return mtp::distill_fwd_workspace(score_shape(n, d, v, 1.0, head_kind), f32, q4_kind(head_kind), k, keep != 0);
}
size_t mtp_distill_fwd_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, int32_t keep) {
  return distill_fwd_ws(0, n, d, v, head_kind, k, keep);
}
size_t mtp_distill_fwd_f32_workspace_bytes(int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, int32_t keep) {
  return distill_fwd_ws(1, n, d, v, head_kind, k, keep);
}

static int check_reduction(int32_t reduction) {
  if (reduction != MTP_REDUCE_NONE && reduction != MTP_REDUCE_MEAN && reduction != MTP_REDUCE_SUM)
    return fail(MTP_ERR_INPUT, "unknown reduction %d of a distillation loss", (int)reduction);
  return MTP_OK;
}

static int distill_fwd(int f32, const void* hidden, const void* w, const uint32_t* w_q, const void* scales, const void* biases,
                       const int64_t* ids, const float* teacher, const uint8_t* mask, int64_t n, int64_t d, int64_t v,
                       int32_t head_kind, int32_t k, int32_t kind, double beta, double temperature, int32_t renormalize,
                       int32_t reduction, const mtp::DistillOut& out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_score_head(f32, hidden, w, w_q, scales, biases, n, d, v, head_kind);
  if (rc) return rc;
  if ((rc = check_score(f32, d, v, temperature)) || (rc = check_list(k)) || (rc = check_reduction(reduction))) return rc;
  if (kind < MTP_DISTILL_FORWARD || kind > MTP_DISTILL_JSD) return fail(MTP_ERR_INPUT, "unknown kind %d of a distillation loss", (int)kind);
  if (kind == MTP_DISTILL_JSD && !(beta > 0.0 && beta < 1.0)) return fail(MTP_ERR_INPUT, "beta must be in (0, 1) (got %g)", beta);
  if (kind == MTP_DISTILL_REVERSE && renormalize) return fail(MTP_ERR_INPUT, "a renormalized teacher gives nothing to what its list leaves out: the reverse divergence is infinite");
  if (!ids || !teacher) return fail(MTP_ERR_INPUT, "ids and teacher must be non-null");
  if (!out.loss || !out.lse || !out.rest || !out.coef || !out.columns || (reduction != MTP_REDUCE_NONE && !out.scale))
    return fail(MTP_ERR_INPUT, "loss, scale, lse, rest, coef and columns must be non-null");
  if (!aligned16(out.logits)) return fail(MTP_ERR_UNSUPPORTED, "logits must be 16-byte aligned");
  const size_t need = distill_fwd_ws(f32, n, d, v, head_kind, k, out.logits != nullptr);
  if (!workspace || workspace_bytes < need)
    return fail(MTP_ERR_WORKSPACE, "distillation needs a workspace of %zu bytes (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned16(workspace)) return fail(MTP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
  const hipError_t e = mtp::launch_distill_fwd(score_head(f32, hidden, w, w_q, scales, biases, head_kind),
                                               score_shape(n, d, v, temperature, head_kind), ids, teacher, mask,
                                               mtp::DistillLoss{(int)k, kind, renormalize != 0, reduction, beta, 1.0 / temperature}, out, workspace,
                                               static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return fail(MTP_ERR_RUNTIME, "distillation launch failed: %s", hipGetErrorString(e));
  return ok();
}
int mtp_distill_fwd(const void* hidden, const void* w, const uint32_t* w_q, const void* scales, const void* biases,
                    const int64_t* ids, const float* teacher, const uint8_t* mask, int64_t n, int64_t d, int64_t v,
                    int32_t head_kind, int32_t k, int32_t kind, double beta, double temperature, int32_t renormalize,
                    int32_t reduction, float* loss, float* scale, float* lse, float* rest, float* coef, int32_t* columns,
                    float* logits, void* workspace, size_t workspace_bytes, void* stream) {
  return distill_fwd(0, hidden, w, w_q, scales, biases, ids, teacher, mask, n, d, v, head_kind, k, kind, beta, temperature, renormalize,
                     reduction, mtp::DistillOut{loss, scale, lse, rest, coef, columns, logits}, workspace, workspace_bytes, stream);
}
int mtp_distill_fwd_f32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                        const int64_t* ids, const float* teacher, const uint8_t* mask, int64_t n, int64_t d, int64_t v,
                        int32_t head_kind, int32_t k, int32_t kind, double beta, double temperature, int32_t renormalize,
                        int32_t reduction, float* loss, float* scale, float* lse, float* rest, float* coef, int32_t* columns,
                        float* logits, void* workspace, size_t workspace_bytes, void* stream) {
  return distill_fwd(1, hidden, w, w_q, scales, biases, ids, teacher, mask, n, d, v, head_kind, k, kind, beta, temperature, renormalize,
                     reduction, mtp::DistillOut{loss, scale, lse, rest, coef, columns, logits}, workspace, workspace_bytes, stream);
}

static int distill_bwd(int f32, const void* hidden, const void* w, const void* w_t, const uint32_t* w_q, const void* scales,
                       const void* biases, int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, double temperature,
                       int32_t reduction, const float* d_loss, const float* scale, const float* lse, const float* rest,
                       const float* coef, const int32_t* columns, const float* logits, void* d_hidden, void* d_w, int64_t chunk,
                       int64_t row_block, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_list(k)) || (rc = check_reduction(reduction))) return rc;
  if (!d_loss || !rest || !coef || !columns || (reduction != MTP_REDUCE_NONE && !scale))
    return fail(MTP_ERR_INPUT, "d_loss, scale, rest, coef and columns must be non-null");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return score_bwd(f32, hidden, w, w_t, w_q, scales, biases, n, d, v, head_kind, k, temperature, lse, columns, logits, d_hidden, d_w, chunk,
                   row_block, workspace, workspace_bytes, st, [&](float* alpha, float*, int*, float* value, bool*) {
                     return mtp::launch_distill_coef(d_loss, reduction == MTP_REDUCE_NONE, scale, rest, coef, (long)n, (int)k, alpha, value, st);
                   });
}
int mtp_distill_bwd(const void* hidden, const void* w, const void* w_t, const uint32_t* w_q, const void* scales,
                    const void* biases, int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, double temperature,
                    int32_t reduction, const float* d_loss, const float* scale, const float* lse, const float* rest,
                    const float* coef, const int32_t* columns, const float* logits, void* d_hidden, void* d_w, int64_t chunk,
                    int64_t row_block, void* workspace, size_t workspace_bytes, void* stream) {
  return distill_bwd(0, hidden, w, w_t, w_q, scales, biases, n, d, v, head_kind, k, temperature, reduction, d_loss, scale, lse, rest, coef,
                     columns, logits, d_hidden, d_w, chunk, row_block, workspace, workspace_bytes, stream);
}
int mtp_distill_bwd_f32(const float* hidden, const float* w, const uint32_t* w_q, const float* scales, const float* biases,
                        int64_t n, int64_t d, int64_t v, int32_t head_kind, int32_t k, double temperature, int32_t reduction,
                        const float* d_loss, const float* scale, const float* lse, const float* rest, const float* coef,
                        const int32_t* columns, const float* logits, float* d_hidden, float* d_w, int64_t chunk, void* workspace,
                        size_t workspace_bytes, void* stream) {
  return distill_bwd(1, hidden, w, nullptr, w_q, scales, biases, n, d, v, head_kind, k, temperature, reduction, d_loss, scale, lse, rest,
                     coef, columns, logits, d_hidden, d_w, chunk, 0, workspace, workspace_bytes, stream);
}

}  // extern "C"

// Preference and policy losses over the per-token losses of linear_cross_entropy (nll = -log pi, fp32).
//
// Tokens belong to sequences: rows of a [rows][T] batch, or the ranges [offsets[r], offsets[r + 1]) of a flat run of
// tokens (each clamped into it, so that any offsets stay in bounds). A mask, where given, says which tokens count; what
// the others hold is not used, NaN included.
//
// Preference loss: sequence p is the chosen and sequence pairs + p the rejected answer of pair p.
//   g_r = sum_t (ref_t - nll_t), the log ratio of policy to reference (ipo: its mean over the tokens), reward_r = beta g_r,
//   d_p = reward_p - reward_{pairs + p}
//   sigmoid: (1 - e) softplus(-d) + e softplus(d); hinge: max(0, 1 - d); ipo: (d / beta - 1 / (2 beta))^2
// A token's gradient is its sequence's factor coef_r, whatever the token: the forward leaves coef, the backward spreads it.
//
// Policy loss: with s_t = old_t - nll_t (the ratio is e^s), A the advantage of the token or its sequence, d_t = nll_t - ref_t:
//   loss_t = -min(e^s A, clip(e^s, 1 - low, 1 + high) A) + kl_coef (e^d - d - 1)
//   d loss_t / d nll_t = [not clipped] e^s A + kl_coef (e^d - 1)
// clipped: A > 0 and e^s > 1 + high, or A < 0 and e^s < 1 - low.
//
// Both are bound by their launches until some hundred thousand tokens, then by reading 8 to 17 bytes a token. Sums are in
// 64 bits: a log ratio is the small difference of long sums. Every sequence is cut into `chunks` equal parts, a workgroup
// each, whose partial sums one workgroup joins in order, so a result does not depend on scheduling.
#include "mtp_common.hpp"
#include "mtp_launch.hpp"

namespace mtp {

namespace {
constexpr int kPrefThreads = 256;
constexpr int kJoinThreads = 1024;

struct Span {
  long begin, end;
};
__device__ __forceinline__ Span sequence_of(const int64_t* offsets, long rows, long n, long r) {
  if (!offsets) {
    const long t = n / rows;
    return Span{r * t, (r + 1) * t};
  }
  long a = offsets[r], b = offsets[r + 1];
  a = a < 0 ? 0 : a < n ? a : n;
  b = b < a ? a : b < n ? b : n;
  return Span{a, b};
}
__device__ __forceinline__ Span part_of(const Span& s, int c, int chunks) {
  const long len = s.end - s.begin;
  return Span{s.begin + len * c / chunks, s.begin + len * (c + 1) / chunks};
}

// Sum over the workgroup's threads, in every thread: within a wave by halves, then the waves in order.
template <int THREADS, class T>
__device__ __forceinline__ T block_sum(T x) {
  __shared__ T part[THREADS / 64];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  __syncthreads();  // the last use of part is over
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  T s = part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s += part[w];
  return s;
}

struct PrefPart {
  double gap;
  long count;
};

__global__ __launch_bounds__(kPrefThreads) void pref_sums_kernel(const float* __restrict__ nll, const float* __restrict__ ref,
                                                                 const uint8_t* __restrict__ mask,
                                                                 const int64_t* __restrict__ offsets, long rows, long n,
                                                                 int chunks, PrefPart* __restrict__ part) {
  const long r = blockIdx.x / chunks;
  const Span s = part_of(sequence_of(offsets, rows, n, r), blockIdx.x % chunks, chunks);
  double gap = 0;
  int count = 0;
  for (long t = s.begin + threadIdx.x; t < s.end; t += kPrefThreads) {
    if (mask && !mask[t]) continue;
    gap += (double)ref[t] - (double)nll[t];
    ++count;
  }
  gap = block_sum<kPrefThreads>(gap);
  count = block_sum<kPrefThreads>(count);
  if (threadIdx.x == 0) part[blockIdx.x] = PrefPart{gap, count};
}

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// Joins the parts of each sequence; loss [pairs] (reduction none) or [1], reward and coef [2 pairs].
__global__ __launch_bounds__(kJoinThreads) void pref_join_kernel(const PrefPart* __restrict__ part, long pairs, int chunks,
                                                                 PrefLoss p, float* __restrict__ loss,
                                                                 float* __restrict__ reward, float* __restrict__ coef) {
  auto sum = [&](long r, double& weight) {
    double gap = 0;
    long count = 0;
    for (int c = 0; c < chunks; ++c) {
      gap += part[r * chunks + c].gap;
      count += part[r * chunks + c].count;
    }
    weight = p.kind == kPrefIpo ? 1.0 / (double)(count > 1 ? count : 1) : 1.0;
    return gap * weight * p.beta;
  };
  const double share = p.reduction == kReduceMean ? 1.0 / (double)pairs : 1.0;
  double total = 0;
  for (long i = threadIdx.x; i < pairs; i += kJoinThreads) {
    double wc, wr;
    const double chosen = sum(i, wc), rejected = sum(pairs + i, wr), d = chosen - rejected;
    double l, slope;
    if (p.kind == kPrefSigmoid) {
      l = (1.0 - p.smoothing) * softplus(-d) + p.smoothing * softplus(d);
      slope = p.smoothing - 1.0 / (1.0 + exp(d));
    } else if (p.kind == kPrefHinge) {
      l = d < 1.0 ? 1.0 - d : d >= 1.0 ? 0.0 : d;  // NaN stays
      slope = d < 1.0 ? -1.0 : d >= 1.0 ? 0.0 : d;
    } else {
      const double h = d / p.beta - 0.5 / p.beta;
      l = h * h;
      slope = 2.0 * h / p.beta;
    }
    reward[i] = (float)chosen;
    reward[pairs + i] = (float)rejected;
    coef[i] = (float)(-slope * p.beta * wc * share);
    coef[pairs + i] = (float)(slope * p.beta * wr * share);
    if (p.reduction == kReduceNone) loss[i] = (float)l;
    total += l;
  }
  if (p.reduction == kReduceNone) return;
  total = block_sum<kJoinThreads>(total);
  if (threadIdx.x == 0) loss[0] = (float)(total * share);
}

// The gradient of tokens of no sequence: before the first offset (row 0's workgroups) and behind the last.
__device__ __forceinline__ void zero_outside(const int64_t* offsets, long rows, long n, long r, const Span& s, int c, float* out) {
  if (!offsets || c != 0) return;
  if (r == 0)
    for (long t = threadIdx.x; t < s.begin; t += kPrefThreads) out[t] = 0.f;
  if (r == rows - 1)
    for (long t = s.end + threadIdx.x; t < n; t += kPrefThreads) out[t] = 0.f;
}

__global__ __launch_bounds__(kPrefThreads) void pref_bwd_kernel(const float* __restrict__ d_loss, const float* __restrict__ coef,
                                                                const uint8_t* __restrict__ mask,
                                                                const int64_t* __restrict__ offsets, long pairs, long n,
                                                                int chunks, int per_pair, float* __restrict__ d_nll) {
  const long rows = 2 * pairs, r = blockIdx.x / chunks;
  const Span whole = sequence_of(offsets, rows, n, r), s = part_of(whole, blockIdx.x % chunks, chunks);
  const float g = coef[r] * d_loss[per_pair ? r % pairs : 0];
  for (long t = s.begin + threadIdx.x; t < s.end; t += kPrefThreads) d_nll[t] = (!mask || mask[t]) ? g : 0.f;
  zero_outside(offsets, rows, n, r, whole, blockIdx.x % chunks, d_nll);
}

// e^d - d - 1 without the cancellation near 0: its series there.
__device__ __forceinline__ float kl_of(float d) {
  if (fabsf(d) < 0.5f) {
    // d^2 / 2 (1 + d / 3 (1 + d / 4 (1 + ...))), up to d^9 / 10!: 2^-26 of the sum at 0.5.
    float p = 1.f;
#pragma unroll
    for (int k = 10; k >= 3; --k) p = __builtin_fmaf(d * (1.f / (float)k), p, 1.f);
    return 0.5f * d * d * p;
  }
  return expm1f(d) - d;
}

struct PolicyToken {
  float loss, slope, kl;
  bool clipped;
};
__device__ __forceinline__ PolicyToken policy_token(const PolicyLoss& p, float nll, float old, float ref, float adv) {
  PolicyToken k;
  // Which side of its border a ratio is on is told in 64 bits, where the difference of two floats is exact: a token's
  // gradient is all or nothing there.
  const double s = (double)old - (double)nll;
  const float ratio = expf((float)s);
  k.clipped = adv > 0.f ? s > p.log_high : adv < 0.f ? s < p.log_low : false;
  k.loss = -(k.clipped ? (adv > 0.f ? p.edge_high : p.edge_low) : ratio) * adv;
  k.slope = k.clipped ? 0.f : ratio * adv;
  k.kl = 0.f;
  if (p.has_ref) {
    const float d = nll - ref;
    k.kl = kl_of(d);
    if (p.kl_coef != 0.f) {  // 0: the KL is reported alone, and may be infinite
      k.loss += p.kl_coef * k.kl;
      k.slope += p.kl_coef * expm1f(d);
    }
  }
  return k;
}

struct PolicyPart {
  double loss, kl;
  long count, clipped;
};

__global__ __launch_bounds__(kPrefThreads) void policy_sums_kernel(const float* __restrict__ nll, const float* __restrict__ old,
                                                                   const float* __restrict__ ref, const float* __restrict__ adv,
                                                                   const uint8_t* __restrict__ mask,
                                                                   const int64_t* __restrict__ offsets, long rows, long n,
                                                                   int chunks, PolicyLoss p, PolicyPart* __restrict__ part,
                                                                   float* __restrict__ loss) {
  const long r = blockIdx.x / chunks;
  const Span whole = sequence_of(offsets, rows, n, r), s = part_of(whole, blockIdx.x % chunks, chunks);
  const float a_row = p.adv_per_token ? 0.f : adv[r];
  double sum = 0, kl = 0;
  int count = 0, clipped = 0;
  for (long t = s.begin + threadIdx.x; t < s.end; t += kPrefThreads) {
    float l = 0.f;
    if (!mask || mask[t]) {
      const PolicyToken k = policy_token(p, nll[t], old[t], p.has_ref ? ref[t] : 0.f, p.adv_per_token ? adv[t] : a_row);
      l = k.loss;
      sum += k.loss;
      kl += k.kl;
      ++count;
      clipped += k.clipped;
    }
    if (p.reduction == kReduceNone) loss[t] = l;
  }
  sum = block_sum<kPrefThreads>(sum);
  kl = block_sum<kPrefThreads>(kl);
  count = block_sum<kPrefThreads>(count);
  clipped = block_sum<kPrefThreads>(clipped);
  if (threadIdx.x == 0) part[blockIdx.x] = PolicyPart{sum, kl, count, clipped};
  if (p.reduction == kReduceNone) zero_outside(offsets, rows, n, r, whole, blockIdx.x % chunks, loss);
}

// Joins the parts: stats = (mean KL, share of clipped tokens), weight [rows] the factor of a sequence's tokens in the
// loss, and the loss unless it is per token.
__global__ __launch_bounds__(kJoinThreads) void policy_join_kernel(const PolicyPart* __restrict__ part, long rows, int chunks,
                                                                   PolicyLoss p, float* __restrict__ loss,
                                                                   float* __restrict__ stats, float* __restrict__ weight) {
  double sum = 0, kl = 0, means = 0;
  long count = 0, clipped = 0, filled = 0;
  for (long r = threadIdx.x; r < rows; r += kJoinThreads) {
    double s = 0;
    long n = 0;
    for (int c = 0; c < chunks; ++c) {
      const PolicyPart& x = part[r * chunks + c];
      s += x.loss;
      n += x.count;
      kl += x.kl;
      clipped += x.clipped;
    }
    sum += s;
    count += n;
    filled += n > 0;
    if (n > 0) means += s / (double)n;
  }
  sum = block_sum<kJoinThreads>(sum);
  kl = block_sum<kJoinThreads>(kl);
  means = block_sum<kJoinThreads>(means);
  count = block_sum<kJoinThreads>(count);
  clipped = block_sum<kJoinThreads>(clipped);
  filled = block_sum<kJoinThreads>(filled);
  const double tokens = (double)(count > 1 ? count : 1), seqs = (double)(filled > 1 ? filled : 1);
  if (threadIdx.x == 0) {
    stats[0] = (float)(kl / tokens);
    stats[1] = (float)((double)clipped / tokens);
    if (p.reduction == kReduceMean) loss[0] = (float)(sum / tokens);
    if (p.reduction == kReduceSequences) loss[0] = (float)(means / seqs);
  }
  for (long r = threadIdx.x; r < rows; r += kJoinThreads) {
    double w = 1.0;
    if (p.reduction == kReduceMean) w = 1.0 / tokens;
    if (p.reduction == kReduceSequences) {
      long n = 0;
      for (int c = 0; c < chunks; ++c) n += part[r * chunks + c].count;
      w = 1.0 / ((double)(n > 1 ? n : 1) * seqs);
    }
    weight[r] = (float)w;
  }
}

__global__ __launch_bounds__(kPrefThreads) void policy_bwd_kernel(const float* __restrict__ d_loss, const float* __restrict__ nll,
                                                                  const float* __restrict__ old, const float* __restrict__ ref,
                                                                  const float* __restrict__ adv,
                                                                  const uint8_t* __restrict__ mask,
                                                                  const int64_t* __restrict__ offsets, long rows, long n,
                                                                  int chunks, PolicyLoss p, const float* __restrict__ weight,
                                                                  float* __restrict__ d_nll) {
  const long r = blockIdx.x / chunks;
  const Span whole = sequence_of(offsets, rows, n, r), s = part_of(whole, blockIdx.x % chunks, chunks);
  const float a_row = p.adv_per_token ? 0.f : adv[r];
  const float w = p.reduction == kReduceNone ? 1.f : weight[r] * d_loss[0];
  for (long t = s.begin + threadIdx.x; t < s.end; t += kPrefThreads) {
    float g = 0.f;
    if (!mask || mask[t]) {
      g = policy_token(p, nll[t], old[t], p.has_ref ? ref[t] : 0.f, p.adv_per_token ? adv[t] : a_row).slope * w;
      if (p.reduction == kReduceNone) g *= d_loss[t];
    }
    d_nll[t] = g;
  }
  zero_outside(offsets, rows, n, r, whole, blockIdx.x % chunks, d_nll);
}

// Parts of a sequence: about 4096 tokens each on average, at most 64.
int chunks_of(long rows, long n) {
  const long c = (n / rows + 4095) / 4096;
  return c < 1 ? 1 : c > 64 ? 64 : (int)c;
}
}  // namespace

size_t pref_workspace(long pairs, long n) { return (size_t)(2 * pairs) * chunks_of(2 * pairs, n) * sizeof(PrefPart); }
size_t policy_workspace(long rows, long n) { return (size_t)rows * chunks_of(rows, n) * sizeof(PolicyPart); }

hipError_t launch_pref_fwd(const float* nll, const float* ref, const uint8_t* mask, const int64_t* offsets, long pairs, long n,
                           const PrefLoss& p, float* loss, float* reward, float* coef, void* ws, hipStream_t st) {
  const int chunks = chunks_of(2 * pairs, n);
  PrefPart* part = static_cast<PrefPart*>(ws);
  hipLaunchKernelGGL(pref_sums_kernel, dim3((unsigned)(2 * pairs * chunks)), dim3(kPrefThreads), 0, st, nll, ref, mask, offsets,
                     2 * pairs, n, chunks, part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pref_join_kernel, dim3(1), dim3(kJoinThreads), 0, st, part, pairs, chunks, p, loss, reward, coef);
  return hipGetLastError();
}

hipError_t launch_pref_bwd(const float* d_loss, const float* coef, const uint8_t* mask, const int64_t* offsets, long pairs,
                           long n, int per_pair, float* d_nll, hipStream_t st) {
  const int chunks = chunks_of(2 * pairs, n);
  hipLaunchKernelGGL(pref_bwd_kernel, dim3((unsigned)(2 * pairs * chunks)), dim3(kPrefThreads), 0, st, d_loss, coef, mask,
                     offsets, pairs, n, chunks, per_pair, d_nll);
  return hipGetLastError();
}

hipError_t launch_policy_fwd(const float* nll, const float* old, const float* ref, const float* adv, const uint8_t* mask,
                             const int64_t* offsets, long rows, long n, const PolicyLoss& p, float* loss, float* stats,
                             float* weight, void* ws, hipStream_t st) {
  const int chunks = chunks_of(rows, n);
  PolicyPart* part = static_cast<PolicyPart*>(ws);
  hipLaunchKernelGGL(policy_sums_kernel, dim3((unsigned)(rows * chunks)), dim3(kPrefThreads), 0, st, nll, old, ref, adv, mask,
                     offsets, rows, n, chunks, p, part, loss);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(policy_join_kernel, dim3(1), dim3(kJoinThreads), 0, st, part, rows, chunks, p, loss, stats, weight);
  return hipGetLastError();
}

hipError_t launch_policy_bwd(const float* d_loss, const float* nll, const float* old, const float* ref, const float* adv,
                             const uint8_t* mask, const int64_t* offsets, long rows, long n, const PolicyLoss& p,
                             const float* weight, float* d_nll, hipStream_t st) {
  const int chunks = chunks_of(rows, n);
  hipLaunchKernelGGL(policy_bwd_kernel, dim3((unsigned)(rows * chunks)), dim3(kPrefThreads), 0, st, d_loss, nll, old, ref, adv,
                     mask, offsets, rows, n, chunks, p, weight, d_nll);
  return hipGetLastError();
}

}  // namespace mtp

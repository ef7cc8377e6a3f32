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
// Both read 8 to 17 bytes a token and are bound by launches and latency up to some hundred thousand tokens. So each wave
// takes 512 consecutive tokens, whatever sequences they belong to (sequences dealt to workgroups made the longest of a
// ragged batch the whole time), and has all its loads in flight at once: eight tokens a lane. For every sequence r that
// wave w touches it leaves one part at slot w + r; as w and r never decrease along the tokens no two parts share a slot,
// so nwaves + rows slots hold them. A join, one workgroup, adds each sequence's parts in a fixed order. Sums are in 64 bits,
// since a log ratio is the small difference of long sums, and no result depends on scheduling. Small batches take one
// launch of one workgroup that does both, the parts in LDS (one_launch).
//
// Measured, 512 packed sequences of 2048 tokens, four tensors read (16.8 MB): policy forward 9.3 us (1.8 TB/s), join 8.1,
// backward 8.7 (21 MB: 2.4 TB/s; a large copy reaches 4.9); 16 x 1024 padded tokens: preference forward and join 8.0 us in
// one launch (7.7 in two and the gap between them), backward 3.4. The host takes 60 us for
// such a step, so that what is left here does not show.
#include "mtp_common.hpp"
#include "mtp_launch.hpp"

namespace mtp {

namespace {
constexpr int kLaneTokens = 8, kWaveTokens = 64 * kLaneTokens;
constexpr int kThreads = 256;        // a workgroup of the large grid
constexpr int kJoinThreads = 1024;   // the join's, and that of the one-launch form
// Bounds of the one-launch form: tokens of a preference and of a policy loss with up to kFewRows sequences, and with up to
// kOneRows.
constexpr int kPrefTokens = 16384, kPolicyTokens = 8192, kFewRows = 64, kRowTokens = 4096, kOneRows = 512;
constexpr int kOneParts = kRowTokens / kWaveTokens + kOneRows;
static_assert(kPrefTokens / kWaveTokens + kFewRows <= kOneParts && kPolicyTokens <= kPrefTokens);

struct Seqs {
  const int64_t* offsets;
  int rows, n, t;  // t: tokens of a row, without offsets
  __device__ __forceinline__ int clamp(long x) const { return x < 0 ? 0 : x < n ? (int)x : n; }
  __device__ __forceinline__ int begin(int r) const { return offsets ? clamp(offsets[r]) : r * t; }
  __device__ __forceinline__ int end(int r) const { return offsets ? clamp(offsets[r + 1]) : (r + 1) * t; }
  // The first sequence that ends past token s (rows if none), the same in every lane: a search by 64 probes at a time.
  __device__ __forceinline__ int first(int s) const {
    if (!offsets) return s / t;
    int lo = 0, hi = rows;
    while (lo < hi) {
      const int step = (hi - lo + 63) / 64, probe = lo + ((int)(threadIdx.x & 63) + 1) * step - 1;
      const uint64_t past = __builtin_amdgcn_ballot_w64(probe >= hi || offsets[probe + 1] > s);
      if (past == 0) return hi;
      lo += __builtin_ctzll(past) * step;
      hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return lo;
  }
};

// A lane's tokens of wave-tile w are w kWaveTokens + token(k) for k = 0 .. 7: two runs of four.
__device__ __forceinline__ int token(int k) { return 256 * (k >> 2) + 4 * (int)(threadIdx.x & 63) + (k & 3); }

// The lane's eight values of src (tokens from n on: not read). VEC: src is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const float* __restrict__ src, int s, int n, float (&x)[kLaneTokens]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = s + token(4 * h);
    if (VEC && t + 3 < n) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(src + t);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * h + j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * h + j] = t + j < n ? src[t + j] : 0.f;
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* __restrict__ dst, int s, int n, const float (&x)[kLaneTokens]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = s + token(4 * h);
    if (VEC && t + 3 < n) {
      *reinterpret_cast<f32x4*>(dst + t) = f32x4{x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t + j < n) dst[t + j] = x[4 * h + j];
    }
  }
}
// Bit k: token k counts (VEC: mask is 4-byte aligned).
template <bool VEC>
__device__ __forceinline__ uint32_t keep8(const uint8_t* __restrict__ mask, int s, int n) {
  if (!mask) return 0xff;
  uint32_t keep = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = s + token(4 * h);
    if (VEC && t + 3 < n) {
      const uint32_t m = *reinterpret_cast<const uint32_t*>(mask + t);
#pragma unroll
      for (int j = 0; j < 4; ++j) keep |= ((m >> (8 * j)) & 0xffu) ? 1u << (4 * h + j) : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) keep |= (t + j < n && mask[t + j]) ? 1u << (4 * h + j) : 0u;
    }
  }
  return keep;
}
// f(r, part) for every sequence r of tile w, in order: bit k of `part` tells whether token k is one of it.
template <class F>
__device__ __forceinline__ void each_sequence(const Seqs& q, int w, F&& f) {
  const int s = w * kWaveTokens, e = s + kWaveTokens < q.n ? s + kWaveTokens : q.n;
  for (int r = q.first(s); r < q.rows; ++r) {
    const int a = q.begin(r), b = q.end(r);
    if (a >= e) break;
    uint32_t part = 0;
#pragma unroll
    for (int k = 0; k < kLaneTokens; ++k) {
      const int t = s + token(k);
      part |= (t >= a && t < b) ? 1u << k : 0u;  // b <= n
    }
    f(r, part);
  }
}

// x of another lane of the same 16, by the DPP control CTRL: lanes 1 or 2 away, or mirrored within 8 or 16.
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;
template <int CTRL, class T>
__device__ __forceinline__ T dpp(T x) {
  static_assert(sizeof(T) % 4 == 0);
  struct Words {
    int w[sizeof(T) / 4];
  };
  Words v = __builtin_bit_cast(Words, x);
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) v.w[i] = __builtin_amdgcn_update_dpp(0, v.w[i], CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(T, v);
}
template <class T>
__device__ __forceinline__ T read_lane(T x, int lane) {
  struct Words {
    int w[sizeof(T) / 4];
  };
  Words v = __builtin_bit_cast(Words, x);
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) v.w[i] = __builtin_amdgcn_readlane(v.w[i], lane);
  return __builtin_bit_cast(T, v);
}
// Sum over each 16 lanes, in all of them; a quarter of the time of exchanges through LDS.
template <class T>
__device__ __forceinline__ T row_add(T x) {
  x += dpp<kXor1>(x);
  x += dpp<kXor2>(x);
  x += dpp<kMirror8>(x);
  return x + dpp<kMirror16>(x);
}
template <class T>
__device__ __forceinline__ T wave_add(T x) {
  x = row_add(x);
  return ((read_lane(x, 0) + read_lane(x, 16)) + read_lane(x, 32)) + read_lane(x, 48);
}
// Sum over the join's threads, in every thread.
template <class T>
__device__ __forceinline__ T block_add(T x) {
  static_assert(kJoinThreads == 16 * 64);
  __shared__ T part[16];
  x = wave_add(x);
  __syncthreads();  // the last use of part is over
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  return row_add(part[threadIdx.x % 16]);
}

// The join gives every item (a pair, a sequence) a group of lanes, as many as there are threads for (a power of two, 64 at
// most), and a lane of the group every group-th part.
__device__ __forceinline__ int join_group(int items) {
  int g = 64;
  while (g > 1 && g * items > kJoinThreads) g >>= 1;
  return g;
}
template <class T>
__device__ __forceinline__ T group_add(T x, int group) {
  if (group >= 2) x += dpp<kXor1>(x);
  if (group >= 4) x += dpp<kXor2>(x);
  if (group >= 8) x += dpp<kMirror8>(x);
  if (group >= 16) x += dpp<kMirror16>(x);
  if (group >= 32) x += __shfl_xor(x, 16, 64);
  if (group >= 64) x += __shfl_xor(x, 32, 64);
  return x;
}
// Tiles [first, last] with a part of sequence r; none for an empty one.
__device__ __forceinline__ void tiles_of(const Seqs& q, int r, int& first, int& last) {
  const int a = q.begin(r), b = q.end(r);
  first = a / kWaveTokens;
  last = b > a ? (b - 1) / kWaveTokens : first - 1;
}

struct PrefPart {
  double gap;
  long count;
};

template <bool VEC>
__device__ __forceinline__ void pref_tile(const float* __restrict__ nll, const float* __restrict__ ref,
                                          const uint8_t* __restrict__ mask, const Seqs& q, int w, PrefPart* part) {
  const int s = w * kWaveTokens;
  float x[kLaneTokens], y[kLaneTokens];
  load8<VEC>(nll, s, q.n, x);
  load8<VEC>(ref, s, q.n, y);
  const uint32_t keep = keep8<VEC>(mask, s, q.n);
  each_sequence(q, w, [&](int r, uint32_t mine) {
    mine &= keep;
    double gap = 0;
#pragma unroll
    for (int k = 0; k < kLaneTokens; ++k)
      if ((mine >> k) & 1) gap += (double)y[k] - (double)x[k];
    gap = wave_add(gap);
    const int count = wave_add(__builtin_popcount(mine));
    if ((threadIdx.x & 63) == 0) part[w + r] = PrefPart{gap, count};
  });
}

// softplus and the logistic of a difference that is already exact to 2^-53: fp32 results need no more than fp32 functions.
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

__device__ __forceinline__ void pref_join(const PrefPart* part, const Seqs& q, const PrefLoss& p, float* __restrict__ loss,
                                          float* __restrict__ reward, float* __restrict__ coef) {
  const int pairs = q.rows / 2, group = join_group(pairs), lane = threadIdx.x % group;
  auto sum = [&](int r, double& weight) {
    int first, last;
    tiles_of(q, r, first, last);
    double gap = 0;
    long count = 0;
    for (int w = first + lane; w <= last; w += group) {
      gap += part[w + r].gap;
      count += part[w + r].count;
    }
    gap = group_add(gap, group);
    count = group_add(count, group);
    weight = p.kind == kPrefIpo ? 1.0 / (double)(count > 1 ? count : 1) : 1.0;
    return gap * weight * p.beta;
  };
  const double share = p.reduction == kReduceMean ? 1.0 / (double)pairs : 1.0;
  double total = 0;
  for (int i0 = 0; i0 < pairs; i0 += kJoinThreads / group) {  // whole groups stay together for group_add
    const int i = i0 + (int)threadIdx.x / group;
    const bool live = i < pairs;
    double wc, wr;
    const double chosen = sum(live ? i : 0, wc), rejected = sum(pairs + (live ? i : 0), wr), d = chosen - rejected;
    if (!live || lane != 0) continue;
    double l, slope;
    if (p.kind == kPrefSigmoid) {
      const float x = (float)d;
      l = (1.0 - p.smoothing) * softplus(-x);
      if (p.smoothing != 0.0) l += p.smoothing * softplus(x);  // 0 of an infinite one is 0
      slope = p.smoothing - 1.f / (1.f + expf(x));
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
  total = block_add(total);
  if (threadIdx.x == 0) loss[0] = (float)(total * share);
}

// Tiles [first, ntiles) by steps of `step` of a wave, or (ONE) all tiles by one workgroup and the join behind them.
template <bool VEC, bool ONE>
__global__ __launch_bounds__(ONE ? kJoinThreads : kThreads) void pref_fwd_kernel(
    const float* __restrict__ nll, const float* __restrict__ ref, const uint8_t* __restrict__ mask, Seqs q, PrefLoss p,
    PrefPart* ws, float* __restrict__ loss, float* __restrict__ reward, float* __restrict__ coef) {
  __shared__ PrefPart lds[ONE ? kOneParts : 1];
  PrefPart* part = ONE ? lds : ws;
  constexpr int kWaves = (ONE ? kJoinThreads : kThreads) / 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ntiles = (q.n + kWaveTokens - 1) / kWaveTokens;
  for (int w = ONE ? wave : (int)blockIdx.x * kWaves + wave; w < ntiles; w += ONE ? kWaves : ntiles)
    pref_tile<VEC>(nll, ref, mask, q, w, part);
  if constexpr (ONE) {
    __syncthreads();
    pref_join(part, q, p, loss, reward, coef);
  }
}
__global__ __launch_bounds__(kJoinThreads) void pref_join_kernel(const PrefPart* __restrict__ part, Seqs q, PrefLoss p,
                                                                 float* __restrict__ loss, float* __restrict__ reward,
                                                                 float* __restrict__ coef) {
  pref_join(part, q, p, loss, reward, coef);
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void pref_bwd_kernel(const float* __restrict__ d_loss, const float* __restrict__ coef,
                                                            const uint8_t* __restrict__ mask, Seqs q, int per_pair,
                                                            float* __restrict__ d_nll) {
  const int w = (int)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = w * kWaveTokens;
  if (s >= q.n) return;
  const uint32_t keep = keep8<VEC>(mask, s, q.n);
  const int pairs = q.rows / 2;
  float g[kLaneTokens] = {};  // tokens of no sequence: 0
  each_sequence(q, w, [&](int r, uint32_t mine) {
    mine &= keep;
    const float c = coef[r] * d_loss[per_pair ? (r < pairs ? r : r - pairs) : 0];
#pragma unroll
    for (int k = 0; k < kLaneTokens; ++k) g[k] = ((mine >> k) & 1) ? c : g[k];
  });
  store8<VEC>(d_nll, s, q.n, g);
}

// e^d - d - 1 without the cancellation near 0: its series there.
__device__ __forceinline__ float kl_of(float d, float em1) {
  if (fabsf(d) < 0.5f) {
    // d^2 / 2 (1 + d / 3 (1 + d / 4 (1 + ...))), up to d^10 / 10!: what follows is 2^-33 of the sum at 0.5.
    float p = 1.f;
#pragma unroll
    for (int k = 10; k >= 3; --k) p = __builtin_fmaf(d * (1.f / (float)k), p, 1.f);
    return 0.5f * d * d * p;
  }
  return em1 - d;
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
  // An advantage of 0 leaves nothing of a ratio that overflows either.
  const bool flat = k.clipped || adv == 0.f;
  k.loss = -(flat ? (adv > 0.f ? p.edge_high : p.edge_low) : ratio) * adv;
  k.slope = flat ? 0.f : ratio * adv;
  k.kl = 0.f;
  if (p.has_ref) {
    const float d = nll - ref, em1 = expm1f(d);
    k.kl = kl_of(d, em1);
    if (p.kl_coef != 0.f) {  // 0: the KL is reported alone, and may be infinite
      k.loss += p.kl_coef * k.kl;
      k.slope += p.kl_coef * em1;
    }
  }
  return k;
}

struct PolicyPart {
  double loss, kl;
  int count, clipped;
};

// The tokens of a tile in registers.
template <bool VEC>
struct PolicyTile {
  float x[kLaneTokens], o[kLaneTokens], r[kLaneTokens], a[kLaneTokens];
  uint32_t keep;
  __device__ __forceinline__ void load(const float* __restrict__ nll, const float* __restrict__ old, const float* __restrict__ ref,
                                       const float* __restrict__ adv, const uint8_t* __restrict__ mask, const PolicyLoss& p, int s,
                                       int n) {
    load8<VEC>(nll, s, n, x);
    load8<VEC>(old, s, n, o);
#pragma unroll
    for (int k = 0; k < kLaneTokens; ++k) r[k] = a[k] = 0.f;
    if (p.has_ref) load8<VEC>(ref, s, n, r);
    if (p.adv_per_token) load8<VEC>(adv, s, n, a);
    keep = keep8<VEC>(mask, s, n);
  }
};

template <bool VEC>
__device__ __forceinline__ void policy_tile(const float* __restrict__ nll, const float* __restrict__ old,
                                            const float* __restrict__ ref, const float* __restrict__ adv,
                                            const uint8_t* __restrict__ mask, const Seqs& q, const PolicyLoss& p, int w,
                                            PolicyPart* part, float* __restrict__ loss) {
  const int s = w * kWaveTokens;
  PolicyTile<VEC> t;
  t.load(nll, old, ref, adv, mask, p, s, q.n);
  float each[kLaneTokens] = {};
  each_sequence(q, w, [&](int r, uint32_t mine) {
    mine &= t.keep;
    const float a_row = p.adv_per_token ? 0.f : adv[r];
    double sum = 0, kl = 0;
    int count = 0;  // and, from bit 16 on, the clipped ones
#pragma unroll
    for (int k = 0; k < kLaneTokens; ++k)
      if ((mine >> k) & 1) {
        const PolicyToken y = policy_token(p, t.x[k], t.o[k], t.r[k], p.adv_per_token ? t.a[k] : a_row);
        sum += y.loss;
        kl += y.kl;
        count += y.clipped ? 0x10001 : 1;
        each[k] = y.loss;
      }
    sum = wave_add(sum);
    if (p.has_ref) kl = wave_add(kl);
    count = wave_add(count);
    if ((threadIdx.x & 63) == 0) part[w + r] = PolicyPart{sum, kl, count & 0xffff, count >> 16};
  });
  if (p.reduction == kReduceNone) store8<VEC>(loss, s, q.n, each);
}

// stats = (mean KL, share of clipped tokens), weight [rows] the factor of a sequence's tokens in the loss, and the loss
// unless it is per token.
__device__ __forceinline__ void policy_join(const PolicyPart* part, const Seqs& q, const PolicyLoss& p,
                                            float* __restrict__ loss, float* __restrict__ stats, float* __restrict__ weight) {
  const int group = join_group(q.rows), lane = threadIdx.x % group;
  double sum = 0, kl = 0, means = 0;
  long count = 0, clipped = 0;
  int filled = 0;
  for (int r0 = 0; r0 < q.rows; r0 += kJoinThreads / group) {
    const int r = r0 + (int)threadIdx.x / group;
    double s = 0;
    long n = 0;
    if (r < q.rows) {
      int first, last;
      tiles_of(q, r, first, last);
      for (int w = first + lane; w <= last; w += group) {
        const PolicyPart x = part[w + r];
        s += x.loss;
        n += x.count;
        kl += x.kl;
        clipped += x.clipped;
      }
    }
    sum += s;
    count += n;
    if (p.reduction == kReduceSequences) {
      s = group_add(s, group);
      n = group_add(n, group);
      if (lane == 0 && r < q.rows) {
        if (n > 0) {
          means += s / (double)n;
          ++filled;
        }
        weight[r] = (float)(n > 1 ? n : 1);  // below: its reciprocal over the sequences
      }
    }
  }
  kl = block_add(kl);
  count = block_add(count);
  clipped = block_add(clipped);
  const double tokens = (double)(count > 1 ? count : 1);
  double seqs = 1;
  if (p.reduction == kReduceMean) sum = block_add(sum);
  if (p.reduction == kReduceSequences) {
    means = block_add(means);
    filled = block_add(filled);
    seqs = (double)(filled > 1 ? filled : 1);
  }
  if (threadIdx.x == 0) {
    stats[0] = (float)(kl / tokens);
    stats[1] = (float)((double)clipped / tokens);
    if (p.reduction == kReduceMean) loss[0] = (float)(sum / tokens);
    if (p.reduction == kReduceSequences) loss[0] = (float)(means / seqs);
  }
  // (block_add's barriers lie between the weights' two steps)
  for (int r = threadIdx.x; r < q.rows; r += kJoinThreads)
    weight[r] = p.reduction == kReduceMean ? (float)(1.0 / tokens) : p.reduction == kReduceNone ? 1.f
                                           : (float)(1.0 / ((double)weight[r] * seqs));
}

template <bool VEC, bool ONE>
__global__ __launch_bounds__(ONE ? kJoinThreads : kThreads) void policy_fwd_kernel(
    const float* __restrict__ nll, const float* __restrict__ old, const float* __restrict__ ref, const float* __restrict__ adv,
    const uint8_t* __restrict__ mask, Seqs q, PolicyLoss p, PolicyPart* ws, float* __restrict__ loss,
    float* __restrict__ stats, float* weight) {
  __shared__ PolicyPart lds[ONE ? kOneParts : 1];
  PolicyPart* part = ONE ? lds : ws;
  constexpr int kWaves = (ONE ? kJoinThreads : kThreads) / 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ntiles = (q.n + kWaveTokens - 1) / kWaveTokens;
  for (int w = ONE ? wave : (int)blockIdx.x * kWaves + wave; w < ntiles; w += ONE ? kWaves : ntiles)
    policy_tile<VEC>(nll, old, ref, adv, mask, q, p, w, part, loss);
  if constexpr (ONE) {
    __syncthreads();
    policy_join(part, q, p, loss, stats, weight);
  }
}
__global__ __launch_bounds__(kJoinThreads) void policy_join_kernel(const PolicyPart* __restrict__ part, Seqs q, PolicyLoss p,
                                                                   float* __restrict__ loss, float* __restrict__ stats,
                                                                   float* weight) {
  policy_join(part, q, p, loss, stats, weight);
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void policy_bwd_kernel(const float* __restrict__ d_loss, const float* __restrict__ nll,
                                                              const float* __restrict__ old, const float* __restrict__ ref,
                                                              const float* __restrict__ adv, const uint8_t* __restrict__ mask,
                                                              Seqs q, PolicyLoss p, const float* __restrict__ weight,
                                                              float* __restrict__ d_nll) {
  const int w = (int)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = w * kWaveTokens;
  if (s >= q.n) return;
  PolicyTile<VEC> t;
  t.load(nll, old, ref, adv, mask, p, s, q.n);
  float up[kLaneTokens], g[kLaneTokens] = {};
  const bool each = p.reduction == kReduceNone;
  if (each) load8<VEC>(d_loss, s, q.n, up);
  const float one = each ? 1.f : d_loss[0];
  each_sequence(q, w, [&](int r, uint32_t mine) {
    mine &= t.keep;
    const float a_row = p.adv_per_token ? 0.f : adv[r], f = each ? 1.f : weight[r] * one;
#pragma unroll
    for (int k = 0; k < kLaneTokens; ++k)
      if ((mine >> k) & 1)
        g[k] = policy_token(p, t.x[k], t.o[k], t.r[k], p.adv_per_token ? t.a[k] : a_row).slope * (each ? up[k] : f);
  });
  store8<VEC>(d_nll, s, q.n, g);
}

int tiles(long n) { return (int)((n + kWaveTokens - 1) / kWaveTokens); }
dim3 tile_grid(long n) { return dim3((unsigned)((tiles(n) + kThreads / 64 - 1) / (kThreads / 64))); }
Seqs seqs(const int64_t* offsets, long rows, long n) { return Seqs{offsets, (int)rows, (int)n, offsets ? 0 : (int)(n / rows)}; }
bool aligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
}  // namespace

size_t pref_workspace(long pairs, long n) { return (size_t)(tiles(n) + 2 * pairs) * sizeof(PrefPart); }
size_t policy_workspace(long rows, long n) { return (size_t)(tiles(n) + rows) * sizeof(PolicyPart); }

// One workgroup for a whole loss: a launch less (4 us and more of host time, 4 of GPU time for the join), but its 16 waves
// alone form the parts, of which there are as many as tiles and sequences. us in one launch | in two, without the gap between
// them: 16 sequences, preference 6.1 | 7.1 at 8192 tokens, 7.9 | 7.7 at 16384, 12 | 8.5 at 32768; policy 10.2 | 9.1,
// 16.1 | 9.3, 28 | 10.1. 64 sequences of 16384 in all: 10.0 | 9.2, 18.5 | 10.2 (policy, 8192: 14.2 | 11.9). 512: preference
// 38 | 36 at 4096, 31 | 22 at 8192, policy 71 | 68, 54 | 40.
static bool one_launch(long rows, long n, long tokens) { return n <= (rows <= kFewRows ? tokens : kRowTokens) && rows <= kOneRows; }

hipError_t launch_pref_fwd(const float* nll, const float* ref, const uint8_t* mask, const int64_t* offsets, long pairs, long n,
                           const PrefLoss& p, float* loss, float* reward, float* coef, void* ws, hipStream_t st) {
  PrefPart* part = static_cast<PrefPart*>(ws);
  const Seqs q = seqs(offsets, 2 * pairs, n);
  const bool vec = aligned(nll, 16) && aligned(ref, 16) && aligned(mask, 4);
  if (one_launch(2 * pairs, n, kPrefTokens)) {
    auto k = vec ? pref_fwd_kernel<true, true> : pref_fwd_kernel<false, true>;
    hipLaunchKernelGGL(k, dim3(1), dim3(kJoinThreads), 0, st, nll, ref, mask, q, p, part, loss, reward, coef);
    return hipGetLastError();
  }
  auto k = vec ? pref_fwd_kernel<true, false> : pref_fwd_kernel<false, false>;
  hipLaunchKernelGGL(k, tile_grid(n), dim3(kThreads), 0, st, nll, ref, mask, q, p, part, loss, reward, coef);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pref_join_kernel, dim3(1), dim3(kJoinThreads), 0, st, part, q, p, loss, reward, coef);
  return hipGetLastError();
}

hipError_t launch_pref_bwd(const float* d_loss, const float* coef, const uint8_t* mask, const int64_t* offsets, long pairs,
                           long n, int per_pair, float* d_nll, hipStream_t st) {
  auto k = aligned(d_nll, 16) && aligned(mask, 4) ? pref_bwd_kernel<true> : pref_bwd_kernel<false>;
  hipLaunchKernelGGL(k, tile_grid(n), dim3(kThreads), 0, st, d_loss, coef, mask, seqs(offsets, 2 * pairs, n), per_pair, d_nll);
  return hipGetLastError();
}

hipError_t launch_policy_fwd(const float* nll, const float* old, const float* ref, const float* adv, const uint8_t* mask,
                             const int64_t* offsets, long rows, long n, const PolicyLoss& p, float* loss, float* stats,
                             float* weight, void* ws, hipStream_t st) {
  PolicyPart* part = static_cast<PolicyPart*>(ws);
  const Seqs q = seqs(offsets, rows, n);
  const bool vec = aligned(nll, 16) && aligned(old, 16) && aligned(ref, 16) && (!p.adv_per_token || aligned(adv, 16)) &&
                   aligned(mask, 4) && (p.reduction != kReduceNone || aligned(loss, 16));
  if (one_launch(rows, n, kPolicyTokens)) {
    auto k = vec ? policy_fwd_kernel<true, true> : policy_fwd_kernel<false, true>;
    hipLaunchKernelGGL(k, dim3(1), dim3(kJoinThreads), 0, st, nll, old, ref, adv, mask, q, p, part, loss, stats, weight);
    return hipGetLastError();
  }
  auto k = vec ? policy_fwd_kernel<true, false> : policy_fwd_kernel<false, false>;
  hipLaunchKernelGGL(k, tile_grid(n), dim3(kThreads), 0, st, nll, old, ref, adv, mask, q, p, part, loss, stats, weight);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(policy_join_kernel, dim3(1), dim3(kJoinThreads), 0, st, part, q, p, loss, stats, weight);
  return hipGetLastError();
}

hipError_t launch_policy_bwd(const float* d_loss, const float* nll, const float* old, const float* ref, const float* adv,
                             const uint8_t* mask, const int64_t* offsets, long rows, long n, const PolicyLoss& p,
                             const float* weight, float* d_nll, hipStream_t st) {
  const bool vec = aligned(nll, 16) && aligned(old, 16) && aligned(ref, 16) && (!p.adv_per_token || aligned(adv, 16)) &&
                   aligned(mask, 4) && aligned(d_nll, 16) && (p.reduction != kReduceNone || aligned(d_loss, 16));
  auto k = vec ? policy_bwd_kernel<true> : policy_bwd_kernel<false>;
  hipLaunchKernelGGL(k, tile_grid(n), dim3(kThreads), 0, st, d_loss, nll, old, ref, adv, mask, seqs(offsets, rows, n), p, weight,
                     d_nll);
  return hipGetLastError();
}

}  // namespace mtp

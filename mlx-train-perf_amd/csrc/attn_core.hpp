// Flash attention forward and backward for gfx950 (GQA; causal, packed segments or key spans; capped
// scores and a bias by distance): the kernels, instantiated by attn_kernels.hip (plain and packed) and
// attn_scored.hip (spans, caps and biases).
//
// Semantics follow the reference oracles: O = softmax(scale * Q K^T + mask) V with an fp32 softmax,
// L = row logsumexp of the masked scaled scores (attention/reference.py:42-116); the backward uses
// the FlashAttention equations D = rowsum(dO * O), P = exp(S - L), dV = P^T dO, dP = dO V^T,
// dS = P * (dP - D), dQ = scale dS K, dK = scale dS^T Q, with dK and dV summed over the query-head
// group of each kv head (attention/api.py:126-194). Query head h reads kv head h / (Hq / Hkv).
// Packed mode: key j is visible to query i iff seg_id[i] == seg_id[j] and j <= i
// (attention/segments.py:22-29); seg_start (non-decreasing, gapless layout) only bounds loops.
// Span mode: key j is visible to query i iff start[i] <= j < end[i], both non-decreasing along a row, so
// the queries that see key j are a range too (col_begin, col_end). A query may see nothing: O = 0.
// Scores: with x = scale q.k, the softmax is over cap tanh(x / cap) - slope |i - j| (either part may be
// missing); dS then has the factor 1 - tanh^2, and the bias has no gradient.
//
// Rounded to bf16: the probabilities and dS, as the MFMA takes them (their sums, the softmax and D are fp32), and the
// outputs; with spans, caps and biases, what such a rounding does to D is kept out of dS (o_low, lr in attn_kv_kernel, HALF
// in the dK/dV kernel), which leaves errors of 2.0e-3 of the norm in O, 2.3e-3 in dV and 2.4e-3 to 3.0e-3 in dQ and dK.
//
// Bound by the SIMDs' issue, matrix and vector instructions together: with a cap the matrix pipe is busy for 0.44 to 0.55
// of the time (8192 positions, 32/8 heads, head_dim 128: forward 637 us, dQ 828, dK/dV 1166; without a cap 515, 690 and
// 1010), as a score costs an exponential and a reciprocal more. With slopes alone the products begin from the bias and the
// forward and dQ take the plain kernels' times (4 x 16 heads x 2048 x 64: 59 and 68 us); dK/dV 101, 3% more (kUp).
//
// Kernel structure (all MFMA 32x32x16 bf16, fp32 accumulate):
//   attn_kv_kernel<DH, MASK, DQ, MOD> (forward, and the dQ pass, which also forms D): a wave owns 32
//                 queries of one head; a workgroup holds up to 4 heads of one GQA group so every
//                 K/V tile staged in LDS (copied global -> LDS, two stages) feeds 128 query rows.
//                 Scores are computed transposed (keys x queries) so each lane owns one query
//                 column: the online softmax is lane-local plus one exchange with lane^32, and the
//                 probability (or dS) tile feeds the next product directly from registers.
//   attn_bwd_dkv_ab_kernel<DH, MASK, MOD>: 8 waves per 128-key block, operand-split P waves and dS
//                 waves (below); dK^T and dV^T accumulate in registers (no atomics).
#pragma once
#include <type_traits>

#include "mtp_common.hpp"
#include "mtp_launch.hpp"

namespace mtp {


constexpr int kKT = 64;  // positions (keys or queries) per LDS tile
// Online softmax: the running maximum (log2 domain) is raised, and O and l rescaled, only when a
// tile's maximum exceeds it by more than this, so unnormalized probabilities stay <= 2^8.
constexpr float kRescaleLog2 = 8.f;

// Scores in the log2 domain, cap2 tanh(x / cap) - slope2 |i - j|, formed in the place of the raw products s (the
// registers have no room for a second array) so that the last step is the plain score's one multiply-add,
// score = v mul + add, with mul > 0, and a maximum of v is one of the scores:
//   raw: v = -1 / (1 + e^(2x/cap)) with a cap, as tanh(t) = 1 - 2 / (1 + e^2t): mul = 2 cap2, add = cap2; else v = s,
//     mul = scale2. Both ends of the cap are exact; between them v is off by about 2^-22, 2e-5 of a score at a cap of 50
//     and 4e-4 at 1000, the largest allowed: below the step of the bf16 probability formed from it.
//   slant: v -= slope2 / mul |rel - c| for the element at distance |rel - c|, c a constant and rel the lane's and tile's.
//     Where all of a wave's tile lies on one side of its positions that is a term in c, the rest (rel) in add: one
//     multiply-add, or none where the product began from the term (ramp, a cap aside) instead of from 0.
//   A row's biases, and with them its L, count from the highest of them, that of the key at distance top (top_distance):
//     -slope2 (|rel - c| - top), the difference a whole number. Where the slope is below 0, or spans hide the keys nearby, a
//     bias of slope2 |rel - c| has no digits left for what tells the row's keys apart (slope -4, distances of 60000: P off by
//     1%; slope -300: by a factor).
//   bend(v): -v - v^2 = (1 - tanh^2) / 4, the cap's derivative, negated and without its 4, which the gradients' last
//     multiplier has (-4 scale).
// A hidden pair has v = hidden<BWD>(): its score is -inf or so low that its probability is 0; in the backward it stays
// finite under a cap, so that probability times bend is 0 as well.
template <int MOD>
struct Score {
  static constexpr bool kCap = MOD & kModCap, kSlope = MOD & kModSlope;
  float in2, mul, add, slope2, ratio;
  __device__ __forceinline__ Score(float scale_log2, float cap)
      : in2(kCap ? scalar(2.f * scale_log2 / cap) : 0.f), mul(kCap ? scalar(2.f * cap * kLog2e) : scale_log2),
        add(kCap ? scalar(cap * kLog2e) : 0.f), slope2(0.f), ratio(0.f) {}
  // (the same in every lane: kept in scalar registers, as the vector ones are full)
  __device__ __forceinline__ void set_slope(float slope) {
    slope2 = scalar(slope * kLog2e);
    ratio = scalar(slope2 / mul);
  }
  static __device__ __forceinline__ float scalar(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
  }
  template <bool BWD>
  static __device__ __forceinline__ float hidden() { return BWD && kCap ? -1e15f : -__builtin_huge_valf(); }
  __device__ __forceinline__ float raw(float s) const { return kCap ? __builtin_amdgcn_rcpf(-1.f - fast_exp2(s * in2)) : s; }
  static __device__ __forceinline__ constexpr float at(int half, int r) { return (float)(32 * half + 8 * (r >> 2) + (r & 3)); }
  // SIGN ratio c: what a product begins from (`none`: 0).
  template <int SIGN>
  __device__ __forceinline__ void set_ramp(f32x16 (&ramp)[2], bool none = false) const {
    const float step = none ? 0.f : SIGN * ratio;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) ramp[h][r] = step * at(h, r);
  }
  // Queries in lanes. side: 1 where rel >= c (no key behind its query) for every pair of the wave's tile that is not hidden,
  // -1 where rel <= c, 0 where neither: such a tile keeps the usual term (a ramp's, rel >= c) and corrects it.
  template <bool RAMP>
  __device__ __forceinline__ void slant(f32x16& v, int half, int side, float rel) const {
    if constexpr (RAMP) {
      if (side == -1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = __builtin_fmaf(-2 * ratio, at(half, r), v[r]);
      }
    } else {
      const float k = side == -1 ? -ratio : ratio;
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = __builtin_fmaf(k, at(half, r), v[r]);
    }
    if (side == 0) {  // -|d| = -d + 2 min(d, 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = __builtin_fmaf(2.f * ratio, fminf(rel - at(half, r), 0.f), v[r]);
    }
  }
  // add of such a tile.
  __device__ __forceinline__ float slant_add(int side, float rel, float top) const {
    return __builtin_fmaf(-slope2, (side == -1 ? -rel : rel) - top, add);
  }
  // Keys in lanes: k times c and, where keys lie on both sides, the correction (the usual term is that of rel <= c).
  __device__ __forceinline__ void lean(f32x16 (&v)[2], float k, bool both, float rel) const {
    if (k != 0.f) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) v[h][r] = __builtin_fmaf(k * ratio, at(h, r), v[h][r]);
    }
    if (both) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) v[h][r] = __builtin_fmaf(2.f * ratio, fminf(at(h, r) - rel, 0.f), v[h][r]);
    }
  }
  static __device__ __forceinline__ float bend(float v) { return __builtin_fmaf(v, v, v); }
};


// Compiler-visible waits: an inline-asm s_waitcnt is opaque to the compiler's own wait insertion,
// which then keeps earlier loads outstanding and waits for them again later (and for every copy
// in flight with them).
__device__ __forceinline__ void vm_wait0() { __builtin_amdgcn_s_waitcnt(0x0F70); }    // vmcnt(0)
__device__ __forceinline__ void lgkm_wait0() { __builtin_amdgcn_s_waitcnt(0xC07F); }  // lgkmcnt(0)

__device__ __forceinline__ uint32_t lds_addr(const char* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// ds_read_b64_tr_b16 (gfx950 LDS transpose read) of LDS byte address a + OFF, as inline asm. The
// builtin form is treated by the compiler's wait insertion as a possible reader of every LDS DMA
// in flight, so each tile would wait for the copies of the tile after next before its transposed
// product; the asm form is invisible to it, and callers wait for the results (slab_wait) before use.
template <int OFF>
__device__ __forceinline__ u32x2 tr16_asm(uint32_t a) {
  u32x2 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF));
  return r;
}
__device__ __forceinline__ bf16x8 tr_pair(u32x2 lo, u32x2 hi) {
  return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
}
// Waits until at most N LDS reads are outstanding and marks one slab's NDB fragments as produced here.
template <int N, int NDB = 4>
__device__ __forceinline__ void slab_wait(bf16x8 (&f)[4]) {
  static_assert(N >= 0 && N <= 15, "lgkmcnt is a 4-bit field");
  if constexpr (NDB == 4) {
    asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]) : "n"(N));
  } else if constexpr (NDB == 3) {
    asm volatile("s_waitcnt lgkmcnt(%3)" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]) : "n"(N));
  } else {
    static_assert(NDB == 2, "head_dim 64, 96 or 128");
    asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(f[0]), "+v"(f[1]) : "n"(N));
  }
}
// max(x of lane l, x of lane l ^ 32): the two lane halves hold the two key halves of one query
// column. v_permlane32_swap exchanges the upper half of one register with the lower half of the
// other; started from two copies of x, each register then holds one half twice. A VALU operation,
// so unlike a ds_bpermute exchange it does not wait behind LDS reads in flight. The s_nops cover
// the VALU-write / permlane-read hazard, which the compiler does not see inside inline asm.
__device__ __forceinline__ float max_xhalf(float x) {
  float y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}
// x of lane l plus x of lane l ^ 32 (see max_xhalf).
__device__ __forceinline__ float sum_xhalf(float x) {
  float y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
  return x + y;
}

// One LDS-DMA load: 16 bytes per lane from src + voff (lanes past `bytes` read zeros) to dst, a
// wave-uniform LDS address.
__device__ __forceinline__ void lds_copy16(const bf16_t* src, int bytes, char* dst, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(src), (short)0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0, 0);
}
// The same with 4 bytes per lane (lane i writes dst + 4 i).
__device__ __forceinline__ void lds_copy4(const float* src, int bytes, char* dst, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), (short)0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 4, voff, 0, 0, 0);
}

// Transposed fragments f[KS][db] of slab KS (rows 16 KS.. of a swizzled tile of ROWB-byte rows):
// head_dim block db < NDB (32 columns) in the MFMA accumulator-row order (4 hf + 0..3,
// 4 hf + 8..11), from the LDS addresses a0/a1[db] of reads 0 and 1 (16-row slab 0). Asm reads:
// slab_wait before use.
template <int KS, int NDB = 4, int ROWB = 256>
__device__ __forceinline__ void tr_slab(const uint32_t (&a0)[4], const uint32_t (&a1)[4], bf16x8 (&f)[4][4]) {
  constexpr int off = KS * 16 * ROWB;
#pragma unroll
  for (int db = 0; db < NDB; ++db) f[KS][db] = tr_pair(tr16_asm<off>(a0[db]), tr16_asm<off>(a1[db]));
}

__device__ __forceinline__ int heads_per_wg(int G) { return (G % 4 == 0) ? 4 : ((G % 2 == 0) ? 2 : 1); }

namespace kvdma {
// LDS layout of a 64-position K/V tile for head_dim DH: rows of kRowB bytes, 16-byte chunk c of row r
// at slot c ^ sw(r). head_dim 64 packs a row into 128 B; 96 and 128 use 256 B rows (96 leaves chunks
// 12-15 empty: their copies read nothing and write zeros). Both swizzles keep every row-fragment
// read (ds_read_b128, 16 rows at one chunk per 16 lanes) and every transposed read
// (ds_read_b64_tr_b16, 4 rows x 2 chunks per 16 lanes) on distinct banks, and repeat every 16 rows.
template <int DH>
struct Lay {
  static constexpr int kRowB = DH == 64 ? 128 : 256;
  static constexpr int kChunks = kRowB / 16;
  static constexpr int kTile = kKT * kRowB;
  static constexpr int kStage = 2 * kTile;  // K, V
  static __device__ __forceinline__ int sw(int r) {
    if constexpr (DH == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
};

// Per-lane constants: row-fragment swizzle and the transposed-read offsets tro[t] of read t (0, 1)
// of head_dim block 0 within a 16-row slab (block db adds db << 6 by XOR: 4 db only touches chunk
// bits 2 and up of the swizzled 16-byte chunk index).
template <int DH>
struct Lanes {
  int sw_r;
  int tro[2];
  __device__ __forceinline__ void init() {
    using L = Lay<DH>;
    const int lane = threadIdx.x & 63;
    const int hf = lane >> 5, col = lane & 31;
    sw_r = L::sw(col & 15);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int rl = 4 * hf + 8 * t + ((lane & 15) >> 2);
      const int c0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      tro[t] = rl * L::kRowB + ((c0 ^ L::sw(rl)) << 4) + 8 * (lane & 1);
    }
  }
};
}  // namespace kvdma

// The 8 bits of x below those of its bf16, `top` its bits, as a byte (attn_kv_kernel's o_low).
__device__ __forceinline__ uint32_t below_bf16(float x, uint32_t top) {
  const int rest = (__builtin_bit_cast(int, x) - (int)top + 0x80) >> 8;  // in [-128, 128]
  return (uint32_t)(rest < 127 ? rest : 127) & 0xff;
}

// First index i in [lo, hi) with a[i] > x (hi if none); a is non-decreasing.
__device__ __forceinline__ int first_above(const int32_t* a, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The queries [begin, end) that see keys x to y: as start and end do not decrease along a row, those from the first with
// end > x to the first with start > y. The two searches run side by side: each is a chain of dependent loads, a quarter
// of a microsecond a link.
__device__ __forceinline__ void queries_of(const int32_t* start, const int32_t* end, int S, int x, int y, int& qb, int& qe) {
  int lo0 = 0, hi0 = S, lo1 = 0, hi1 = S;
  while (lo0 < hi0 || lo1 < hi1) {
    const int m0 = (lo0 + hi0) >> 1, m1 = (lo1 + hi1) >> 1;
    const int v0 = end[m0 < S ? m0 : S - 1], v1 = start[m1 < S ? m1 : S - 1];
    if (lo0 < hi0) {
      if (v0 > x) hi0 = m0;
      else lo0 = m0 + 1;
    }
    if (lo1 < hi1) {
      if (v1 > y) hi1 = m1;
      else lo1 = m1 + 1;
    }
  }
  qb = lo0;
  qe = lo1;
}

// Counting sort of the work items 0 .. n - 1 of one workgroup of 1024 threads by cost(i) < kSchedBuckets,
// highest first: order[r] is the item of rank r. Items of one cost land in any order.
constexpr int kSchedBuckets = 2048;
// Right shift that brings a tile count of at most ceil(S / 64) + 1 below kSchedBuckets.
__device__ __forceinline__ int sched_shift(int S) {
  int shift = 0;
  while (((S + 63) / 64 + 2) >> shift >= kSchedBuckets) ++shift;
  return shift;
}
template <class Cost>
__device__ __forceinline__ void sched_sort(int n, Cost cost, int32_t* order) {
  __shared__ int cnt[kSchedBuckets];
  __shared__ int wsum[16];
  const int t = threadIdx.x;
  for (int j = t; j < kSchedBuckets; j += 1024) cnt[j] = 0;
  __syncthreads();
  for (int i = t; i < n; i += 1024) atomicAdd(&cnt[cost(i)], 1);
  __syncthreads();
  // First rank of each bucket, buckets in descending cost: thread t sums buckets (descending
  // position) 2t and 2t + 1, then an exclusive scan over the 1024 threads.
  const int ja = kSchedBuckets - 1 - 2 * t, jb = ja - 1;
  const int ca = cnt[ja], cb = cnt[jb];
  int x = ca + cb;
  const int lane = t & 63, wv = t >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) wsum[wv] = x;
  __syncthreads();
  int before = 0;
  for (int u = 0; u < wv; ++u) before += wsum[u];
  const int excl = before + x - (ca + cb);
  __syncthreads();
  cnt[ja] = excl;
  cnt[jb] = excl + ca;
  __syncthreads();
  for (int i = t; i < n; i += 1024) order[atomicAdd(&cnt[cost(i)], 1)] = i;
}

// ------------------------------------------------------------------------------------------
// Backward dK, dV (head_dim 64, 96, 128), operand-split: 8 waves per 128-key workgroup, two per SIMD.
// Waves 0-3 ("P waves") own 32 keys each and hold K: S = Q K^T, P = exp2(S scale log2 e - L log2 e)
// (hidden pairs 0), P handed to the partner wave through LDS, dV^T += dO^T P. Waves 4-7 ("dS waves")
// own the same keys and hold V: dP = dO V^T, dS = P (dP - D) with the partner's P, dK^T += Q^T dS.
// Each wave keeps one operand (32 registers) and one accumulator set (64), so a SIMD runs one wave
// of each kind. The two are skewed by half a tile: between two barriers the P wave finishes tile t
// (dV) and starts tile t+1 (S, P), the dS wave finishes tile t (dS, dK) and starts tile t+1 (dP),
// so each has 32 products with its probability or dS arithmetic between them, and the SIMD
// overlaps the arithmetic of one with the products of the other. Q and dO tiles are copied
// global -> LDS in the K/V tile layout of the forward (kvdma: same swizzle and fragment reads) into
// a ring of three stages, the copy of tile t+3 issued when tile t's stage is released; P goes
// through a ring of three LDS buffers. The loop is unrolled by three so every stage is named
// statically.
// ------------------------------------------------------------------------------------------
namespace dkvab {
// Q, dO, and of the 64 queries L, D and, with slopes, the top (Score).
template <int DH, int MOD>
constexpr int kStage = 2 * kvdma::Lay<DH>::kTile + ((MOD & kModSlope) ? 3 : 2) * 256;
constexpr int kPBytes = kKT * 32 * 2;           // P of one key group (64 queries x 32 keys, bf16)
constexpr int kPBuf = 4 * kPBytes;              // P of the workgroup's four key groups
}  // namespace dkvab

template <int DH, int MASK, int MOD = kModNone>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void attn_bwd_dkv_ab_kernel(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
                               const bf16_t* __restrict__ d_o, const float* __restrict__ lse,
                               const float* __restrict__ dvec, const int32_t* __restrict__ seg_end,
                               bf16_t* __restrict__ dk, bf16_t* __restrict__ dv, int B, int Hq, int Hkv, int S,
                               float scale_log2, float scale, int causal, int nsplit,
                               float* __restrict__ part, const int32_t* __restrict__ order,
                               const int32_t* __restrict__ col_begin, float cap, const float* __restrict__ slopes) {
  // seg_end: the end of each position's segment (packed), or of the queries that see it (span), whose first
  // is col_begin.
  constexpr bool PACKED = MASK != kMaskPlain, SPAN = MASK == kMaskSpan, CAP = MOD & kModCap;
  using L = kvdma::Lay<DH>;
  constexpr int kRowB = L::kRowB, kTile = L::kTile;
  auto sw = [](int r) { return L::sw(r); };
  constexpr int kDK = DH / 16, kDB = DH / 32;
  __shared__ __attribute__((aligned(1024))) char st0[dkvab::kStage<DH, MOD>];
  __shared__ __attribute__((aligned(1024))) char st1[dkvab::kStage<DH, MOD>];
  __shared__ __attribute__((aligned(1024))) char st2[dkvab::kStage<DH, MOD>];
  __shared__ __attribute__((aligned(1024))) char pb0[dkvab::kPBuf];
  __shared__ __attribute__((aligned(1024))) char pb1[dkvab::kPBuf];
  __shared__ __attribute__((aligned(1024))) char pb2[dkvab::kPBuf];

  const int G = Hq / Hkv;
  const int nkv = B * Hkv;
  // Block g: split g % nsplit of key block (g / nsplit) / nkv of kv head (g / nsplit) % nkv; the
  // earliest keys (most work under the causal mask) first. Packed, with a work order: item
  // order[g / (nsplit Hkv)] (batch row item / nkb, key block item % nkb), heaviest first, with its
  // Hkv heads and splits consecutive.
  const int g = blockIdx.x;
  const int split = g % nsplit;
  int bidx, kvh, ktile;
  if (PACKED && order != nullptr) {
    const int nkb = (S + 127) / 128;
    int item = order[g / (nsplit * Hkv)];
    item = item < 0 ? 0 : (item < B * nkb ? item : B * nkb - 1);  // in range whatever the order holds
    bidx = item / nkb;
    ktile = item % nkb;
    kvh = (g / nsplit) % Hkv;
  } else {
    const int kvi = (g / nsplit) % nkv;
    ktile = (g / nsplit) / nkv;
    bidx = kvi / Hkv;
    kvh = kvi % Hkv;
  }
  const int k0 = ktile * 128;

  const int tid = threadIdx.x;
  const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = w & 3;             // key group: keys k0 + 32 grp .. + 31
  const bool pwave = w < 4;          // P wave (K, dV) or dS wave (V, dK)
  const int hf = lane >> 5, col = lane & 31;
  const int kw0 = k0 + 32 * grp;
  const int kj = kw0 + col;
  const bool kvalid = kj < S;

  const long krow = (long)(bidx * Hkv + kvh) * S;
  const int32_t* send = PACKED ? seg_end + (long)bidx * S : nullptr;

  // This wave's operand of the first product: K (P wave) or V (dS wave) rows of its keys.
  bf16x8 opf[kDK];
  {
    const bf16_t* src = (pwave ? k : v) + krow * DH;
#pragma unroll
    for (int ks = 0; ks < kDK; ++ks)
      opf[ks] = kvalid ? as_bf16x8(*reinterpret_cast<const u32x4*>(src + (long)kj * DH + 16 * ks + 8 * hf)) : as_bf16x8(zero4());
  }

  const int32_t* cbeg = SPAN ? col_begin + (long)bidx * S : nullptr;
  const int q_begin = SPAN ? (__builtin_amdgcn_readfirstlane(cbeg[k0]) / kKT) * kKT
                           : causal ? (k0 / kKT) * kKT : 0;  // non-causal: every query
  int q_end = S;
  if (PACKED) {
    const int klast = (k0 + 127 < S) ? k0 + 127 : S - 1;
    q_end = __builtin_amdgcn_readfirstlane(send[klast]);
  }
  // Queries q with kj <= q < my_lim see key kj (packed: my_lim is the end of kj's segment, at most
  // q_end since seg_end is non-decreasing); w_lim is the wave's smallest limit, its first key's.
  int my_lim = S, w_lim = S;
  if (PACKED) {
    my_lim = kvalid ? send[kj] : S;
    w_lim = __builtin_amdgcn_readfirstlane(my_lim);
  }
  int my_beg = 0, w_beg = 0;  // span: the first query that sees kj; the wave's largest, its last key's
  if (SPAN) {
    my_beg = kvalid ? cbeg[kj] : S;
    w_beg = kw0 < S ? __builtin_amdgcn_readfirstlane(cbeg[kw0 + 31 < S ? kw0 + 31 : S - 1]) : 0;
  }
  Score<MOD> score(scale_log2, cap);
  const int ntq = (q_end > q_begin) ? (q_end - q_begin + kKT - 1) / kKT : 0;
  const int niter = G * ntq;
  // This workgroup's share of the key block's (head, query tile) items: [it0, it0 + nloc).
  const int it0 = (int)((long)niter * split / nsplit);
  const int nloc = (int)((long)niter * (split + 1) / nsplit) - it0;

  f32x16 acc[kDB];  // dV^T (P wave) or dK^T (dS wave)
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;

  // Copy lanes: a tile of each operand is kNp 1 KiB pieces, piece p holding rows kRpp p .. + kRpp - 1;
  // P wave w copies pieces w + 8 m and (for its dS partner) w + 4 + 8 m, m < kNp / 8. A lane's source
  // is the logical chunk its LDS slot holds (chunks past head_dim point beyond the buffer and read
  // zeros).
  constexpr int kNp = kTile / 1024, kM = kNp / 8;
  constexpr int kLpr = L::kChunks, kRpp = 64 / kLpr;  // lanes per LDS row, rows per piece
  constexpr int kCopies = 4 * kM;                      // per operand pair and tile, per P wave: Q, dO
  uint32_t coff[kM];
#pragma unroll
  for (int m = 0; m < kM; ++m) {
    const int row = kRpp * (8 * m + w) + lane / kLpr;
    const int c = (lane % kLpr) ^ sw(row);
    coff[m] = 16 * c < 2 * DH ? (uint32_t)(row * 2 * DH + 16 * c) : 0x7ffffff0u;
  }
  int ro[kDK];
#pragma unroll
  for (int ks = 0; ks < kDK; ++ks) ro[ks] = col * kRowB + (((2 * ks + hf) ^ sw(col & 15)) << 4);
  int tro[2][kDB];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int rl = 4 * hf + 8 * t + ((lane & 15) >> 2);
    const int swt = sw(rl);
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      const int c = 4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      tro[t][db] = rl * kRowB + ((c ^ swt) << 4) + 8 * (lane & 1);
    }
  }
  // With a cap (or slopes' ramp at head_dim 96, slopes and spans at 128) P's two copies leave no room for these 16 offsets:
  // each is then formed at its use from the first of its kind (2 ks touches chunk bits 1-3, 4 db bits 2-3, of an
  // XOR-swizzled chunk index).
  constexpr bool kForm = CAP || (MOD == kModSlope && (DH == 96 || (SPAN && DH == 128)));
  auto row_off = [&](int base, int ks) __attribute__((always_inline)) { return kForm ? base ^ (ks << 5) : ro[ks]; };
  auto tr_off = [&](int base, int t, int db) __attribute__((always_inline)) { return kForm ? base ^ (db << 6) : tro[t][db]; };
  // The P wave reads Q rows and dO^T; the dS wave dO rows and Q^T.
  const int row_src = pwave ? 0 : kTile;
  const int tr_src = pwave ? kTile : 0;
  const int pmine = grp * dkvab::kPBytes;

  // Copies of tile `it` into stage `st`: this wave's load j (0-1 Q rows, 2-3 dO rows); zero bytes,
  // no memory access (zeros into a free stage), when not `live`.
  // The per-query scalars L and D of the tile's 64 queries go beside it (waves 0 and 4, one 4-byte
  // load each), and with slopes, where they are read, the dQ pass' tops (wave 1).
  constexpr bool SLOPE = MOD & kModSlope, TOPS = SLOPE && (SPAN || CAP);
  struct CopySrc {
    const bf16_t* qs;
    const bf16_t* ds;
    const float* scal;
    int bytes, sbytes;
  };
  auto copy_src = [&](int it, bool live) __attribute__((always_inline)) {
    const int itc = live ? it0 + it : 0;
    const int hh = itc / ntq, tq = itc % ntq;
    const long qrow = (long)(bidx * Hq + kvh * G + hh) * S;
    const int q0 = q_begin + tq * kKT;
    const int rows = live ? ((S - q0 < kKT) ? S - q0 : kKT) : 0;
    return CopySrc{q + (qrow + q0) * DH, d_o + (qrow + q0) * DH, (TOPS && w == 1 ? dvec + 2L * B * Hq * S : w < 4 ? lse : dvec) + qrow + q0, rows * 2 * DH, rows * 4};
  };
  // The P waves copy for their dS partners too (the dS waves are the longer role): load j of a P wave
  // covers Q (j < 2 kM) or dO rows, piece 8 m + w (m = j % kM) or that of wave w + 4 (j / kM odd),
  // whose rows lie 4 kRpp on with the same swizzle (it repeats every 16 rows).
  auto issue_one = [&](const CopySrc& c, char* st, int j) __attribute__((always_inline)) {
    const int m = j % kM, part = (j / kM) & 1;
    const bool qop = j < 2 * kM;
    lds_copy16(qop ? c.qs : c.ds, c.bytes, st + (qop ? 0 : kTile) + 1024 * (8 * m + w + 4 * part),
               coff[m] + (part ? (uint32_t)(4 * kRpp * 2 * DH) : 0u));
  };
  auto issue_scal = [&](const CopySrc& c, char* st) __attribute__((always_inline)) {
    if (grp == 0 || (TOPS && w == 1))
      lds_copy4(c.scal, c.sbytes, st + 2 * kTile + (TOPS && w == 1 ? 512 : pwave ? 0 : 256), (uint32_t)(4 * lane));
  };

  // Start of tile `it` (stage `st`): the first product of both halves into a1; the P wave then
  // forms P (hidden pairs 0) and writes it to `pb`.
  f32x16 a1[2];
  // With slopes alone the P wave's products begin from the bias' ramp of the head at hand, where it fits the registers, and
  // with spans, where tops are not all 0, from the biases themselves, formed one by one.
  constexpr bool kRamp = MOD == kModSlope && DH <= 96;
  f32x16 ramp[2];
  int ramp_head = -1;
  // HALF: the P wave hands its partner P (with a cap P (1 - tanh^2)), which dS is formed from, in fp16, and keeps P in bf16
  // in registers for its own second product: bf16 there made dK's error 2.9e-3 of its norm instead of 2.4e-3. P is formed
  // 2^15 times as large, so that fp16 holds it to the last bit down to 2^-29; the last multipliers of dV and dK take the
  // factor back.
  constexpr bool HALF = SPAN || MOD != kModNone;
  constexpr float kUp = HALF ? 15.f : 0.f, kDown = HALF ? 0x1p-15f : 1.f;
  bf16x8 pown[HALF ? 2 : 1][2];
  auto start = [&](int it, const char* st, char* pb, const CopySrc& cx, char* sx) __attribute__((always_inline)) {
    const float* tops = reinterpret_cast<const float*>(st + 2 * kTile + 512);
    bool far = false;  // slopes and spans: some query of the tile has its top at another distance than 0
    {
      // Row fragments read two k16 steps ahead of their products.
      bf16x8 rf[3][2];
      int rbase = ro[0];
      if constexpr (kForm) asm volatile("" : "+v"(rbase));
      auto rd = [&](int ks) {
#pragma unroll
        for (int h = 0; h < 2; ++h) rf[ks % 3][h] = as_bf16x8(lds_read16(st + row_src, 32 * h * kRowB + row_off(rbase, ks)));
      };
      const float mine = SPAN && MOD == kModSlope && pwave ? tops[lane] : 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) a1[h][r] = 0.f;
      issue_scal(cx, sx);
      rd(0);
      rd(1);
      if constexpr (SLOPE) {
        const int hh = (it0 + it) / ntq;
        if (pwave && (!kRamp || hh != ramp_head)) {
          ramp_head = hh;
          score.set_slope(slopes ? slopes[kvh * G + hh] : 0.f);
          if constexpr (kRamp) score.template set_ramp<-1>(ramp, !SPAN && score.slope2 < 0.f);
        }
        if constexpr (SPAN && MOD == kModSlope) far = pwave && __builtin_amdgcn_ballot_w64(mine != 0.f) != 0;
      }
#pragma unroll
      for (int ks = 0; ks < kDK; ++ks) {
        if (ks + 2 < kDK) rd(ks + 2);
        // (the first products in branches of their own: one behind them would copy what they begin from)
        auto product = [&](auto&& from) __attribute__((always_inline)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) a1[h] = mfma32(rf[ks % 3][h], opf[ks], from(h));
        };
        if (SPAN && MOD == kModSlope && ks == 0 && far) {
          const float rel = (float)(kj - (q_begin + ((it0 + it) % ntq) * kKT) - 4 * hf);
          product([&](int h) {
            f32x16 x;
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
              const f32x4 t4 = *reinterpret_cast<const f32x4*>(tops + 32 * h + 8 * rq + 4 * hf);
#pragma unroll
              for (int u = 0; u < 4; ++u) x[4 * rq + u] = -score.ratio * (__builtin_fabsf(rel - (float)(32 * h + 8 * rq + u)) - t4[u]);
            }
            return x;
          });
        } else if (kRamp && ks == 0 && pwave) {
          product([&](int h) { return ramp[h]; });
        } else {
          product([&](int h) { return a1[h]; });
        }
        // The copy loads of the tile after next, spread over the k16 steps of the P waves, between
        // products that wait: a copy load holds its wave at issue while the CU's load path serves
        // others.
        if (pwave) {
#pragma unroll
          for (int j = kCopies * ks / kDK; j < kCopies * (ks + 1) / kDK; ++j) issue_one(cx, sx, j);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (pwave) {
      const int q0 = q_begin + ((it0 + it) % ntq) * kKT;
      // Query row 32 h + 8 rq + 4 hf + u is visible to key kj iff thr <= c < lim, c = 32 h + 8 rq + u.
      const int thr = kvalid ? (SPAN ? my_beg - q0 - 4 * hf : causal ? kj - q0 - 4 * hf : -(1 << 20)) : (1 << 20);
      const int lim = my_lim - q0 - 4 * hf;
      const bool need_mask = (causal && q0 < kw0 + 31) || (q0 + kKT > S) || (PACKED && q0 + kKT > w_lim) || (SPAN && q0 < w_beg);
      // With a cap and slopes bend needs v as raw left it, so that the bias comes after (mixed).
      constexpr bool kMixed = MOD == kModBoth;
      float add = score.add + kUp;
      const float rel = (float)(kj - q0 - 4 * hf);
      if constexpr (MOD != kModNone) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r) a1[h][r] = score.raw(a1[h][r]);
        if constexpr (MOD == kModSlope) {
          if (!far) {
            // |i - j| - top, i the query: i - j or, on the other side, j - i. Without spans and for a slope below 0 top is i, or
            // without the causal mask S - 1 - i where that is more (a tile's first half then has that correction: mid).
            const int side = (causal || q0 >= kw0 + 31) ? -1 : q0 + kKT - 1 <= kw0 ? 1 : 0, i0 = q0 + 4 * hf;
            const bool neg = !SPAN && score.slope2 < 0.f, back = !causal && 2 * (q0 + kKT - 1) <= S - 1;
            const bool mid = neg && !back && !causal && 2 * q0 < S - 1;
            const int k = (side == 1 ? 1 : -1) + (neg ? back ? -1 : 1 : kRamp ? 1 : 0);  // how often c is in -(|i - j| - top)
            score.lean(a1, (float)k, side == 0, rel);
            if (mid) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                  a1[h][r] = __builtin_fmaf(score.ratio, fmaxf((float)(S - 1 - 2 * i0) - 2.f * Score<MOD>::at(h, r), 0.f), a1[h][r]);
            }
            add = __builtin_fmaf(-score.slope2, (side == 1 ? rel : -rel) - (neg ? (float)(back ? S - 1 - i0 : i0) : 0.f), add);
          }
        }
      }
      if (need_mask) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int c = 32 * h + 8 * (r >> 2) + (r & 3);
            a1[h][r] = (c >= thr && c < lim) ? a1[h][r] : Score<MOD>::template hidden<true>();
          }
      }
      const float* ls = reinterpret_cast<const float*>(st + 2 * kTile);
      std::conditional_t<HALF, f16x8, bf16x8> pf[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(ls + 32 * h + 8 * rq + 4 * hf);
          f32x4 t4;
          if constexpr (kMixed) {
            if constexpr (DH == 128) __builtin_amdgcn_sched_barrier(0);  // (the reads of later ones would spill)
            t4 = *reinterpret_cast<const f32x4*>(tops + 32 * h + 8 * rq + 4 * hf);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int r = 4 * rq + u;
            if constexpr (!HALF) {
              pf[h][r >> 3][r & 7] = (__bf16)fast_exp2(__builtin_fmaf(a1[h][r], scale_log2, -l4[u] * kLog2e));
            } else {
              // What is added to a query's scores, but for slopes alone, is one number, which the dQ pass left in the place of L
              // (8192 positions, 32/8 heads, head_dim 128, cap 50: 1177 against 1190 us).
              float y = __builtin_fmaf(a1[h][r], score.mul, MOD == kModSlope ? __builtin_fmaf(-kLog2e, l4[u], add) : l4[u]);
              if constexpr (kMixed) {
                const float d = __builtin_fabsf(rel - (float)(32 * h + 8 * rq + u));
                y = __builtin_fmaf(-score.slope2, d - t4[u], y);
              }
              // P is at most 1, but y is the difference of two numbers of the scores' size: from 2^22 on its rounding alone is
              // 1, and 2^16 is past fp16; from 2^29 on 2^y may leave fp32. (A cap keeps scores below 2^12. NaN stays. 3% of the pass
              // at 4 x 16 heads, 2048 positions, head_dim 64, slopes.)
              if constexpr (!CAP) y = __builtin_elementwise_minimum(y, kUp);
              const float p = fast_exp2(y);
              pown[h][r >> 3][r & 7] = (__bf16)p;
              pf[h][r >> 3][r & 7] = (_Float16)(CAP ? p * Score<MOD>::bend(a1[h][r]) : p);
            }
          }
        }
      // Chunk j of every lane is one contiguous KiB of this key group's P.
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<u32x4*>(pb + pmine + 1024 * j + 16 * lane) = __builtin_bit_cast(u32x4, pf[j >> 1][j & 1]);
    }
  };
  // Finish of tile `it` (stage `st`, P in `pb`): the second products, acc += X^T B over the tile's 64
  // queries (X = dO for the P wave, Q for the dS wave, read transposed; B = P, or dS formed from the
  // partner's P and this wave's dP).
  // The transposed reads of the first two 16-query slabs are issued first, in flight while P is read
  // (and dS formed); each slab's products wait for its reads (lgkmcnt counts LDS reads in issue
  // order) while the slab after next is read.
  auto finish = [&](const char* st, const char* pb, const bf16x8 (&pold)[HALF ? 2 : 1][2]) __attribute__((always_inline)) {
    uint32_t ta0[4], ta1[4];
    {
      const uint32_t b = lds_addr(st + tr_src);
      int t0 = tro[0][0], t1 = tro[1][0];
      if constexpr (kForm) asm volatile("" : "+v"(t0), "+v"(t1));
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        ta0[db] = b + tr_off(t0, 0, db);
        ta1[db] = b + tr_off(t1, 1, db);
      }
    }
    bf16x8 tf[4][4];
    tr_slab<0, kDB, kRowB>(ta0, ta1, tf);
    tr_slab<1, kDB, kRowB>(ta0, ta1, tf);
    bf16x8 bo[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (HALF && pwave) bo[h][j] = pold[HALF ? h : 0][j];
        else bo[h][j] = as_bf16x8(*reinterpret_cast<const u32x4*>(pb + pmine + 1024 * (2 * h + j) + 16 * lane));
      }
    if (!pwave) {
      // dS = P (dP - D).
      const float* ds_ = reinterpret_cast<const float*>(st + 2 * kTile) + 64;
      bf16x8 ds;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(ds_ + 32 * h + 8 * rq + 4 * hf);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int r = 4 * rq + u;
            if constexpr (HALF) {
              const float p = (float)__builtin_bit_cast(f16x8, bo[h][r >> 3])[r & 7];
              ds[r & 7] = (__bf16)__builtin_fmaf(p, a1[h][r] - d4[u], 0.f);  // (a conversion less than a product)
              if ((r & 7) == 7) bo[h][r >> 3] = ds;
            } else {
              bo[h][r >> 3][r & 7] = (__bf16)((float)bo[h][r >> 3][r & 7] * (a1[h][r] - d4[u]));
            }
          }
        }
    }
    slab_wait<2 * kDB, kDB>(tf[0]);
#pragma unroll
    for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[0][db], bo[0][0], acc[db]);
    tr_slab<2, kDB, kRowB>(ta0, ta1, tf);
    slab_wait<2 * kDB, kDB>(tf[1]);
#pragma unroll
    for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[1][db], bo[0][1], acc[db]);
    tr_slab<3, kDB, kRowB>(ta0, ta1, tf);
    slab_wait<2 * kDB, kDB>(tf[2]);
#pragma unroll
    for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[2][db], bo[1][0], acc[db]);
    slab_wait<0, kDB>(tf[3]);
#pragma unroll
    for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[3][db], bo[1][1], acc[db]);
  };
  // Waits for this wave's LDS reads and copies, then the workgroup barrier.
  auto sync = [&]() {
    lgkm_wait0();
    vm_wait0();
    asm volatile("s_barrier" ::: "memory");
  };

  // Tile t runs on stage t % 3 and P buffer t % 3.
  // At the start of step t, tile t+1 sits in stage (t+1) % 3 and stage (t+2) % 3 is free (tile t-1
  // was finished in step t-1): step t copies tile t+2 into it, spread over the products of
  // start(t+1), and the sync that ends the step waits for those copies.
  if (nloc > 0) {
    if (pwave) {
      const CopySrc c0 = copy_src(0, true);
#pragma unroll
      for (int j = 0; j < kCopies; ++j) issue_one(c0, st0, j);
    }
    issue_scal(copy_src(0, true), st0);
    sync();
#pragma unroll
    for (int ks = 0; ks < kDK; ++ks) asm volatile("" : "+v"(opf[ks]));
    start(0, st0, pb0, copy_src(1, nloc > 1), st1);
    sync();
  }
  // Step t: the dS wave finishes tile t (with its dP, still in a1) and then starts tile t+1; the P
  // wave starts tile t+1 first (its S products, the copies of tile t+2 into stage sx, P into pn)
  // and then finishes tile t (its own P of tile t comes back from LDS), so its products fall where
  // the dS wave forms dS and runs dP. Then the barrier. The roles run separate copies of the loop. The last
  // tile is finished outside it: run as a step it would start a tile that does not exist, and padding
  // the count to the unroll of three added up to two more, against the 2 or 3 tiles that a workgroup of
  // a short sequence has (dK/dV of B = 4, S = 509, 16/8 heads, head_dim 64: 26.9 -> 20.2 us; packed
  // S = 16384, head_dim 128: 536 -> 524 us). Up to two steps run with the stages in variables.
  auto run = [&](auto pw) __attribute__((always_inline)) {
    constexpr bool PW = decltype(pw)::value;
    auto step = [&](int t, const char* sc, const char* pc, const char* sn, char* pn, char* sx) __attribute__((always_inline)) {
      if constexpr (PW) {
        bf16x8 pold[HALF ? 2 : 1][2];
        if constexpr (HALF) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) pold[h][j] = pown[h][j];
        }
        start(t + 1, sn, pn, copy_src(t + 2, t + 2 < nloc), sx);
        finish(sc, pc, pold);
      } else {
        finish(sc, pc, pown);
        start(t + 1, sn, pn, copy_src(t + 2, t + 2 < nloc), sx);
      }
      sync();
    };
    int t = 0;
    for (; t + 3 < nloc; t += 3) {
      step(t, st0, pb0, st1, pb1, st2);
      step(t + 1, st1, pb1, st2, pb2, st0);
      step(t + 2, st2, pb2, st0, pb0, st1);
    }
    char *sa = st0, *sb = st1, *sc = st2, *pa = pb0, *pb = pb1, *pc = pb2;
    for (; t + 1 < nloc; ++t) {
      step(t, sa, pa, sb, pb, sc);
      char *s = sa, *p = pa;
      sa = sb, sb = sc, sc = s;
      pa = pb, pb = pc, pc = p;
    }
    finish(sa, pa, pown);
  };
  if (nloc > 0) {
    if (pwave) run(std::true_type{});
    else run(std::false_type{});
  }

  if (kvalid) {
    const float mul = kDown * (pwave ? 1.f : CAP ? -4.f * scale : scale);  // (Score::bend)
    if (nsplit == 1) {
      bf16_t* o = (pwave ? dv : dk) + (krow + kj) * DH;
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const int d = 32 * db + 8 * rq + 4 * hf;
          *reinterpret_cast<u32x2*>(o + d) = u32x2{pack_bf16x2(acc[db][4 * rq] * mul, acc[db][4 * rq + 1] * mul),
                                                   pack_bf16x2(acc[db][4 * rq + 2] * mul, acc[db][4 * rq + 3] * mul)};
        }
    } else {
      // fp32 partial of this split: part[split][dk | dv][b][kv head][key][d], summed by
      // attn_dkv_reduce_kernel.
      const long plane = (long)B * Hkv * S * DH;
      float* o = part + (2L * split + (pwave ? 1 : 0)) * plane + (krow + kj) * DH;
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const int d = 32 * db + 8 * rq + 4 * hf;
          *reinterpret_cast<f32x4*>(o + d) = f32x4{acc[db][4 * rq] * mul, acc[db][4 * rq + 1] * mul,
                                                   acc[db][4 * rq + 2] * mul, acc[db][4 * rq + 3] * mul};
        }
    }
  }
}

// ------------------------------------------------------------------------------------------
// Forward and dQ, DMA-fed, for head_dim 64, 96 and 128 (query-row owners; no atomics). Each 64-key K
// and V tile is copied global -> LDS (rows past S read as zeros) in a swizzled row layout (kvdma
// below); S^T = K Q^T and dP^T = V dO^T read row fragments, O^T += V^T P^T and dQ^T += K^T dS^T
// read transposed fragments of the same tiles. Two LDS stages, one barrier per key tile.
// ------------------------------------------------------------------------------------------

// Waves a SIMD: at head_dim 64 a forward with spans, a cap or slopes fits three (without the bias' ramp), whose exponentials
// and products overlap more than two waves': 2 x 32/8 x 4096 causal with a cap 250 us against 262, 4 x 16/16 x 2048 with
// slopes, not causal, 122 against 135, causal 72 against 75; a round of workgroups or two (2 x 16 x 1024) 25.6 against 25.2.
// The dQ pass would spill.
template <int DH, int MASK, bool DQ, int MOD>
constexpr int kv_waves() { return DH == 64 && !DQ && (MASK == kMaskSpan || MOD != kModNone) ? 3 : 2; }
template <int DH, int MASK, bool DQ, int MOD = kModNone, bool FIXED = false, bool SPLIT = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kv_waves<DH, MASK, DQ, MOD>(), kv_waves<DH, MASK, DQ, MOD>())))
void attn_kv_kernel(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
                    const bf16_t* __restrict__ d_o, const bf16_t* __restrict__ o_in, const float* __restrict__ lse_in,
                    float* __restrict__ dvec, const int32_t* __restrict__ span_end,
                    const int32_t* __restrict__ seg_start, bf16_t* __restrict__ out, float* __restrict__ lse_out,
                    int B, int Hq, int Hkv, int S, float scale_log2, float scale, int causal,
                    const int32_t* __restrict__ order, float cap, const float* __restrict__ slopes,
                    int8_t* __restrict__ o_low, int32_t* __restrict__ col_begin, int32_t* __restrict__ col_end, int nsplit,
                    float* __restrict__ part) {
  // seg_start: the first key that each query sees (packed: its segment's start; span: its span's).
  // o_low (spans, caps and biases): the 8 bits of O below bf16's, written by the forward where given, read with O for
  // D = rowsum(dO o O). dS = P (dP - D) is a difference that all but cancels where one probability is nearly 1, and
  // D of the rounded O was the largest part of dQ's and dK's error there (3.6e-3 of the norm against 2.4e-3: 4 x 16 heads,
  // 2048 positions, slopes). A value x is its bf16 plus o_low in units of 2^8 of its bits' value, whatever the exponent.
  // SPLIT (spans, caps and biases; a variant of its own, as its walk cost the others 2.5%): workgroup `split` of a query
  // block takes every nsplit-th key tile of its walk from tile `split` on, and writes its dQ, or its O before the division,
  // to part[split] ([b][hq][s][dh]; the forward's maximum and sums [split][b][hq][s][4] behind all of them):
  // attn_scored.hip joins them.
  constexpr bool PACKED = MASK != kMaskPlain, SPAN = MASK == kMaskSpan, CAP = MOD & kModCap;
  using L = kvdma::Lay<DH>;
  constexpr int kRowB = L::kRowB, kTile = L::kTile, kStage = L::kStage;
  auto sw = [](int r) { return L::sw(r); };
  constexpr int kDK = DH / 16, kDB = DH / 32;
  __shared__ __attribute__((aligned(1024))) char lds0[kStage];
  __shared__ __attribute__((aligned(1024))) char lds1[kStage];

  const int G = Hq / Hkv;
  const int hpw = heads_per_wg(G);
  constexpr int NW = 4;
  const int P = 32 * (NW / hpw);
  const int npb = (S + P - 1) / P;
  const int hgb = Hq / hpw;
  const int nhg = B * hgb;
  constexpr bool SCORED = SPAN || MOD != kModNone;
  static_assert(!SPLIT || SCORED);
  const int ns = SPLIT ? nsplit : 1, split = SPLIT ? (int)blockIdx.x % ns : 0;
  const int g = SPLIT ? (int)blockIdx.x / ns : blockIdx.x;
  // Heaviest query blocks first: the latest under the causal mask; packed, with a work order, item
  // order[g / hgb] (batch row item / npb, query block item % npb), its head groups consecutive.
  int pb, bidx, h0;
  if (PACKED && order != nullptr) {
    int item = order[g / hgb];
    item = item < 0 ? 0 : (item < B * npb ? item : B * npb - 1);  // in range whatever the order holds
    bidx = item / npb;
    pb = item % npb;
    h0 = (g % hgb) * hpw;
  } else {
    const int hg = g % nhg;
    pb = npb - 1 - g / nhg;
    bidx = hg / hgb;
    h0 = (hg % hgb) * hpw;
  }
  const int kvh = h0 / G;

  const int tid = threadIdx.x;
  // The wave index is read as a scalar so that every per-wave bound below (and the decisions built
  // on them) is a scalar branch, not a per-lane select.
  const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, col = lane & 31;
  const int head = h0 + (w % hpw);
  const int qw0 = pb * P + 32 * (w / hpw);
  const int qi = qw0 + col;
  const bool qvalid = qi < S;
  const bool wave_has = qw0 < S;
  const int wq_last = wave_has ? ((qw0 + 31 < S) ? qw0 + 31 : S - 1) : 0;

  const long qrow = (long)(bidx * Hq + head) * S;
  const bf16_t* kh = k + (long)(bidx * Hkv + kvh) * S * DH;
  const bf16_t* vh = v + (long)(bidx * Hkv + kvh) * S * DH;
  const int32_t* snd = SPAN ? span_end + (long)bidx * S : nullptr;
  const int32_t* sst = PACKED ? seg_start + (long)bidx * S : nullptr;

  // A span backward without work orders: the queries that see each key, for the dK/dV pass (attn_scored.hip), each by the
  // workgroup of the first heads whose queries stand where the key does.
  if constexpr (SPAN && DQ) {
    if (col_begin != nullptr && h0 == 0 && split == 0 && tid < P && pb * P + tid < S) {
      int qb, qe;
      queries_of(sst, snd, S, pb * P + tid, pb * P + tid, qb, qe);
      col_begin[(long)bidx * S + pb * P + tid] = qb;
      col_end[(long)bidx * S + pb * P + tid] = qe;
    }
  }

  bf16x8 qf[kDK], df[DQ ? kDK : 1], of[DQ ? kDK : 1];
  u32x2 low[DQ && SCORED ? kDK : 1];
#pragma unroll
  for (int ks = 0; ks < kDK; ++ks)
    qf[ks] = qvalid ? as_bf16x8(*reinterpret_cast<const u32x4*>(q + (qrow + qi) * DH + 16 * ks + 8 * hf)) : as_bf16x8(zero4());
  float l2q = 0.f, dq_row = 0.f;
  if constexpr (DQ) {
#pragma unroll
    for (int ks = 0; ks < kDK; ++ks)
      df[ks] = qvalid ? as_bf16x8(*reinterpret_cast<const u32x4*>(d_o + (qrow + qi) * DH + 16 * ks + 8 * hf)) : as_bf16x8(zero4());
    l2q = qvalid ? lse_in[qrow + qi] * kLog2e : 0.f;
#pragma unroll
    for (int ks = 0; ks < kDK; ++ks)
      of[ks] = qvalid ? as_bf16x8(*reinterpret_cast<const u32x4*>(o_in + (qrow + qi) * DH + 16 * ks + 8 * hf)) : as_bf16x8(zero4());
    if constexpr (SCORED) {
#pragma unroll
      for (int ks = 0; ks < kDK; ++ks)
        low[ks] = qvalid ? *reinterpret_cast<const u32x2*>(o_low + (qrow + qi) * DH + 16 * ks + 8 * hf) : u32x2{0, 0};
    }
  }

  const int wg_q0 = pb * P;
  auto in_row = [&](int x) { return x < 0 ? 0 : x < S ? x : S; };  // spans, in range whatever they hold
  const int wg_q1 = SPAN ? in_row(__builtin_amdgcn_readfirstlane(snd[(wg_q0 + P < S ? wg_q0 + P : S) - 1]))
                         : (causal && wg_q0 + P < S) ? wg_q0 + P : S;  // non-causal: every key
  int kv_begin = 0;
  if (SPAN) kv_begin = (in_row(__builtin_amdgcn_readfirstlane(sst[wg_q0])) / kKT) * kKT;
  else if (PACKED) kv_begin = (sst[wg_q0] / kKT) * kKT;
  const int nwalk = (SPAN && wg_q1 <= kv_begin) ? 0 : (wg_q1 - kv_begin + kKT - 1) / kKT;
  const int ntiles = !SPLIT ? nwalk : nwalk > split ? (nwalk - split + ns - 1) / ns : 0;  // this workgroup's

  // Packed: with contiguous, gapless segments, key j shares query i's segment and j <= i iff
  // seg_start[i] <= j <= i, so the mask is a range test on this lane's seg_start.
  int my_sst = 0, w_sst_first = 0, w_sst_last = 0;
  if (PACKED) {
    my_sst = qvalid ? sst[qi] : S;
    w_sst_first = __builtin_amdgcn_readfirstlane(wave_has ? sst[qw0] : 0);
    w_sst_last = __builtin_amdgcn_readfirstlane(wave_has ? sst[wq_last] : 0);
  }
  // Span: the end of this lane's, and the smallest and largest of the wave's (its first and last query's).
  int my_end = S, w_end_first = S, w_end_last = S;
  if (SPAN) {
    my_end = qvalid ? in_row(snd[qi]) : 0;
    w_end_first = in_row(__builtin_amdgcn_readfirstlane(wave_has ? snd[qw0] : 0));
    w_end_last = in_row(__builtin_amdgcn_readfirstlane(wave_has ? snd[wq_last] : 0));
  }
  Score<MOD> score(scale_log2, cap);
  float top = 0.f;
  if constexpr (MOD & kModSlope) {
    score.set_slope(slopes ? slopes[head] : 0.f);
    top = top_distance(score.slope2, qi, SPAN ? in_row(my_sst) : 0, SPAN ? my_end : causal ? qi + 1 : S);
  }
  // The side of its queries that a tile's keys lie on (Score::slant).
  auto side_of = [&](int kv0) { return (causal || kv0 + kKT - 1 <= qw0) ? 1 : kv0 >= qw0 + 31 ? -1 : 0; };

  // Slopes alone: the products K Q^T begin from the bias' ramp where it fits the registers (kv_waves).
  constexpr bool kRamp = MOD == kModSlope && (DQ ? DH <= 96 : DH == 96 || (DH == 128 && !(SPAN && SPLIT)));
  f32x16 ramp[2];
  if constexpr (kRamp) score.template set_ramp<1>(ramp);

  // Forward with a fixed maximum (FIXED): under a cap of at most kFixedCap no score exceeds the cap, as biases count from
  // the row's highest, and of every row that sees anything some score is at least its negative. So probabilities are
  // formed against 0: at most 2^80, summed over a row and times a value below 2^24 still in fp32's range, and their sum is
  // at least 2^-80. That saves the running maximum, its exchange and every rescale.
  static_assert(!FIXED || (!DQ && CAP));
  float m = FIXED ? 0.f : kNegInf, l = 0.f;
  // Spans, caps and biases: O is divided by the sum of the bf16 probabilities that it was formed from, L is of the exact
  // sum. The probabilities' roundings then shift O, and D with it, only by what dP differs between keys, which is what dS is
  // made of: with the exact sum dQ's and dK's error grew to 5.9e-3 of the norm in rows of 2 to 8 keys, and is 3.0e-3 at most.
  float lr = 0.f;
  auto add_rounded = [&](const bf16x8& p) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) lr = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[j], p[j + 1]}, bf16x2{(__bf16)1.f, (__bf16)1.f}, lr, false);
  };
  f32x16 acc[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;

  kvdma::Lanes<DH> ln;
  ln.init();
  // Row-fragment offset of rows 32 kb + col, k16 step ks: 32 kb kRowB + (kbase ^ (ks << 5)) (the
  // chunk index 2 ks + hf is XOR-swizzled with the row's pattern and 2 ks touches chunk bits 1-3
  // only). Transposed-read offsets: tro[t][db] = tro[t][0] ^ (db << 6) (4 db touches chunk bits 2-3
  // only). The bases pass through an empty asm in each tile, so the XORs are recomputed at each use
  // instead of 32 offsets per lane (two stages) being held in registers across the loop.
  const int kbase = col * kRowB + ((hf ^ ln.sw_r) << 4);
  const int tbase0 = ln.tro[0], tbase1 = ln.tro[1];
  // Copies of tile t into stage st: this wave's load j (0 .. kLd-1 K rows, kLd .. 2 kLd-1 V rows);
  // each wave copies kLd 1 KiB pieces of each tile, piece NW jj + w holding rows kRpp (NW jj + w)
  // .. + kRpp - 1. A lane's source is the logical chunk its LDS slot holds (chunks past head_dim
  // point beyond the buffer and read zeros). The copies of the next tile are issued during the
  // current one, spread over the k16 steps of its first product: a copy load holds its wave at
  // issue while the CU's load path (~64 B/clk) serves the other waves' copies, and issued between
  // products that wait overlaps MFMA work. Past the last tile the loads get an empty buffer range
  // (no memory access; zeros into a stage nobody reads), so no branch splits the product loop.
  constexpr int kLd = kTile / 1024 / NW;
  constexpr int kLpr = L::kChunks, kRpp = 64 / kLpr;  // lanes per LDS row, rows per 1 KiB piece
  uint32_t coff[kLd];
#pragma unroll
  for (int jj = 0; jj < kLd; ++jj) {
    const int row = kRpp * (NW * jj + w) + lane / kLpr;
    const int c = (lane % kLpr) ^ sw(row);
    coff[jj] = 16 * c < 2 * DH ? (uint32_t)(row * 2 * DH + 16 * c) : 0x7ffffff0u;
  }
  // Slopes without a fixed maximum: the tile of the queries' own keys first, then down from it and on from the end. Their
  // bias is the highest there; walking up to it raised the maximum, and rescaled O, at every tile of a steep head (16
  // heads of 4 x 2048 x 64: 79.6 us against the plain forward's 59.7).
  constexpr bool kNearFirst = !DQ && (MOD & kModSlope) && !FIXED;
  const int near = kNearFirst ? (wg_q0 / kKT * kKT <= kv_begin ? 0 : (wg_q0 / kKT * kKT - kv_begin) / kKT) : 0;
  auto tile_at = [&](int t) {
    if constexpr (SPLIT) t = split + t * ns;
    if constexpr (!kNearFirst) return kv_begin + t * kKT;
    int i = (near < nwalk ? near : nwalk - 1) - t;
    if (i < 0) i += nwalk;
    return kv_begin + i * kKT;
  };
  auto issue_one = [&](int t, char* st, int j) __attribute__((always_inline)) {
    const bool ok = t < ntiles;
    const int kv0 = tile_at(t);
    const int jj = j % kLd;
    lds_copy16((j < kLd ? kh : vh) + (ok ? (long)kv0 * DH : 0), ok ? (S - kv0) * 2 * DH : 0,
               st + (j < kLd ? 0 : kTile) + 1024 * (NW * jj + w), coff[jj]);
  };
  // Copies j of tile t+1 issued in k16 step i of the first product: an even share of the 2 kLd.
  auto issue_step = [&](int t, char* nxt, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = (2 * kLd) * i / kDK; j < (2 * kLd) * (i + 1) / kDK; ++j) issue_one(t + 1, nxt, j);
  };

#pragma unroll
  for (int j = 0; j < 2 * kLd; ++j) issue_one(0, lds0, j);
  vm_wait0();
  lgkm_wait0();
  asm volatile("s_barrier" ::: "memory");
  // The kernel-start Q (and dO) fragment loads are complete here: tell the compiler.
#pragma unroll
  for (int ks = 0; ks < kDK; ++ks) asm volatile("" : "+v"(qf[ks]));
  if constexpr (DQ) {
    // D = rowsum(dO o O) of this lane's query (each lane holds half of the dO and O rows, lane
    // l ^ 32 the other half), written out for the dK/dV pass. The O loads were issued with the dO
    // loads, ahead of the first tile's copies, so their latency overlaps those.
    float dp = 0.f;
#pragma unroll
    for (int ks = 0; ks < kDK; ++ks) {
      asm volatile("" : "+v"(df[ks]), "+v"(of[ks]));
      if constexpr (SCORED) asm volatile("" : "+v"(low[ks]));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x = (float)of[ks][j];
        if constexpr (SCORED)
          x = __builtin_bit_cast(float, __builtin_bit_cast(int, x) + (((int)(low[ks][j >> 2] << (24 - 8 * (j & 3))) >> 24) << 8));
        dp = __builtin_fmaf((float)df[ks][j], x, dp);
      }
    }
    dq_row = sum_xhalf(dp);
    if (qvalid && hf == 0 && split == 0) {
      dvec[qrow + qi] = dq_row;
      if constexpr (SCORED && MOD != kModSlope) dvec[(long)B * Hq * S + qrow + qi] = score.add + 15.f - l2q;  // (kUp there)
      if constexpr ((MOD & kModSlope) && (SPAN || CAP)) dvec[2L * B * Hq * S + qrow + qi] = top;
    }
  }

  // dQ pass, tile t from stage cur; the copies of tile t+1 go to stage nxt (free since the barrier
  // that ended tile t-1).
  auto body = [&](int t, const char* cur, char* nxt) __attribute__((always_inline)) {
    const int kv0 = tile_at(t);
    const bool skip = !wave_has || (causal && kv0 > wq_last) || (PACKED && kv0 + kKT - 1 < w_sst_first) ||
                      (SPAN && kv0 >= w_end_last);
    const char* kt = cur;
    const char* vt = cur + kTile;
    int kb_ = kbase, t0_ = tbase0, t1_ = tbase1;
    asm volatile("" : "+v"(kb_), "+v"(t0_), "+v"(t1_));
    auto taddr = [&](const char* tile, uint32_t (&a0)[4], uint32_t (&a1)[4]) __attribute__((always_inline)) {
      const uint32_t b = lds_addr(tile);
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        a0[db] = b + (uint32_t)(t0_ ^ (db << 6));
        a1[db] = b + (uint32_t)(t1_ ^ (db << 6));
      }
    };
    // S^T = K Q^T and dP^T = V dO^T: row fragments one k16 step ahead, the two 32-key accumulator
    // chains interleaved.
    f32x16 sacc[2], pacc[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sacc[kb][r] = kRamp ? ramp[kb][r] : 0.f;
        pacc[kb][r] = 0.f;
      }
    constexpr int RA = 1;
    bf16x8 rk[RA + 1][2], rv[RA + 1][2];
    auto rd = [&](int ks) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        rk[ks % (RA + 1)][kb] = as_bf16x8(lds_read16(kt, 32 * kb * kRowB + (kb_ ^ (ks << 5))));
        rv[ks % (RA + 1)][kb] = as_bf16x8(lds_read16(vt, 32 * kb * kRowB + (kb_ ^ (ks << 5))));
      }
    };
#pragma unroll
    for (int ks = 0; ks < RA; ++ks) rd(ks);
#pragma unroll
    for (int ks = 0; ks < kDK; ++ks) {
      if (ks + RA < kDK) rd(ks + RA);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        sacc[kb] = mfma32(rk[ks % (RA + 1)][kb], qf[ks], sacc[kb]);
        pacc[kb] = mfma32(rv[ks % (RA + 1)][kb], df[ks], pacc[kb]);
      }
      issue_step(t, nxt, ks);
      // Keep each k16 step's reads, products and copy load together (the scheduler would
      // otherwise bunch the copies and hoist the transposed reads into this loop).
      __builtin_amdgcn_sched_barrier(0);
    }
    // The products above run for every wave, as they carry the copies; the rest only for a wave
    // with keys of this tile to attend to (the others meet them at the barrier either way).
    if (!skip) {
      // Transposed fragments of K (the dQ^T products' operand), read after dS, when the score
      // registers are free.
      bf16x8 tf[4][4];
      // Key kv0 + 4 hf + c (c = 32 kb + 8 (r >> 2) + (r & 3)) is visible to this lane's query iff
      // c <= thr (causal and tail bounds) and, packed, c >= lo (at or after the row's segment
      // start). Only tiles that cross the wave's diagonal, the sequence end or (packed) a segment
      // start are masked (scores of hidden keys set to -inf, so their probabilities are 0); the
      // test is per wave, a scalar branch.
      const bool need_mask = (causal && kv0 + kKT - 1 > qw0) || (kv0 + kKT > S) || (PACKED && kv0 < w_sst_last) ||
                             (SPAN && kv0 + kKT > w_end_first);
      const int thr = qvalid ? ((SPAN ? my_end - 1 : causal && qi < S - 1 ? qi : S - 1) - kv0 - 4 * hf) : -1;
      const int lo = my_sst - kv0 - 4 * hf;
      auto visible = [&](int kb, int r) {
        const int c = 32 * kb + 8 * (r >> 2) + (r & 3);
        bool ok = c <= thr;
        if (PACKED) ok = ok && (c >= lo);
        return ok;
      };
      constexpr bool kMixed = MOD == kModBoth;  // bend needs v as raw left it: the bias comes after
      float add = score.add;
      float rel = (float)(qi - kv0 - 4 * hf), steep = -__builtin_fabsf(score.slope2);
      if constexpr (MOD != kModNone) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[kb][r] = score.raw(sacc[kb][r]);
        if constexpr (MOD == kModSlope) {
          const int side = side_of(kv0);
          score.template slant<kRamp>(sacc[0], 0, side, rel);
          score.template slant<kRamp>(sacc[1], 1, side, rel);
          add = score.slant_add(side, rel, top);
        }
        // Of a tile on one side of the queries all distances are one way from top: -slope2 (|d| - top) is -|slope2 (rel -+ top
        // - c)|. A tile of both sides has only distances below 100, and takes top as a term of its own.
        if constexpr (kMixed) {
          const int side = side_of(kv0);
          if (side == 0) {
            add = __builtin_fmaf(score.slope2, top, add);
            steep = -score.slope2;
          }
          rel -= (float)side * top;
        }
        add -= l2q;
      }
      if (need_mask) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[kb][r] = visible(kb, r) ? sacc[kb][r] : Score<MOD>::template hidden<true>();
      }
      bf16x8 pf[4];
      // dS = P (dP - D) (1 - tanh^2), P = exp2(scale log2(e) S - L log2(e)).
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float y = MOD == kModNone ? __builtin_fmaf(sacc[kb][r], scale_log2, -l2q) : __builtin_fmaf(sacc[kb][r], score.mul, add);
          if constexpr (kMixed)
            y = __builtin_fmaf(steep, __builtin_fabsf(rel - (float)(32 * kb + 8 * (r >> 2) + (r & 3))), y);
          // (P <= 1, see the dK/dV pass; a clamp costs nothing, and the NaN that it drops is in D)
          const float p = SCORED && !CAP ? __builtin_amdgcn_fmed3f(fast_exp2(y), 0.f, 1.f) : fast_exp2(y);
          const float ds = p * (pacc[kb][r] - dq_row);
          pf[2 * kb + (r >> 3)][r & 7] = (__bf16)(CAP ? ds * Score<MOD>::bend(sacc[kb][r]) : ds);
        }
      // dQ^T += K^T dS^T: contraction over the 64 keys in 16-key slabs.
      // The K^T fragments are read only now (the score registers are free after dS): slab by
      // slab, each slab's products issued as soon as its reads have returned while the reads of
      // the slab after next are in flight (lgkmcnt counts LDS reads in issue order).
      uint32_t a0[4], a1[4];
      taddr(kt, a0, a1);
      tr_slab<0, kDB, kRowB>(a0, a1, tf);
      tr_slab<1, kDB, kRowB>(a0, a1, tf);
      slab_wait<2 * kDB, kDB>(tf[0]);
#pragma unroll
      for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[0][db], pf[0], acc[db]);
      tr_slab<2, kDB, kRowB>(a0, a1, tf);
      slab_wait<2 * kDB, kDB>(tf[1]);
#pragma unroll
      for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[1][db], pf[1], acc[db]);
      tr_slab<3, kDB, kRowB>(a0, a1, tf);
      slab_wait<2 * kDB, kDB>(tf[2]);
#pragma unroll
      for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[2][db], pf[2], acc[db]);
      slab_wait<0, kDB>(tf[3]);
#pragma unroll
      for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[3][db], pf[3], acc[db]);
    }
    // This wave's copies of tile t+1 landed; after the barrier nobody reads `cur`, which takes t+2.
    vm_wait0();
    lgkm_wait0();
    asm volatile("s_barrier" ::: "memory");
  };
  // Forward tile t from stage cur, the copies of tile t+1 into stage nxt. S^T = K Q^T is formed per
  // 32-key half: chain 0 (keys kv0 .. +31) carries the copies, and half 0's probabilities are formed
  // while chain 1's products run, half 1's while half 0's O^T products run, so the exps sit in MFMA
  // shadows instead of between the two products. Half 0 is formed against the running maximum m
  // before the tile's maximum is known; the one wave-uniform check after chain 1 raises m (and
  // recomputes half 0) in the rare tile whose maximum exceeds m by kRescaleLog2, exactly as the
  // single-pass online softmax would.
  auto fwd_body = [&](int t, const char* cur, char* nxt) __attribute__((always_inline)) {
    const int kv0 = tile_at(t);
    const bool skip = !wave_has || (causal && kv0 > wq_last) || (PACKED && kv0 + kKT - 1 < w_sst_first) ||
                      (SPAN && kv0 >= w_end_last);
    const char* kt = cur;
    const char* vt = cur + kTile;
    int kb_ = kbase, t0_ = tbase0, t1_ = tbase1;
    asm volatile("" : "+v"(kb_), "+v"(t0_), "+v"(t1_));
    const uint32_t vb = lds_addr(vt);
    uint32_t a0[4], a1[4];
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      a0[db] = vb + (uint32_t)(t0_ ^ (db << 6));
      a1[db] = vb + (uint32_t)(t1_ ^ (db << 6));
    }
    f32x16 s0, s1;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s0[r] = kRamp ? ramp[0][r] : 0.f;
      s1[r] = kRamp ? ramp[1][r] : 0.f;
    }
    // Step i of the 2 kDK products: chain i / kDK, k16 step i % kDK; row fragments two steps ahead.
    constexpr int RA = 2;
    bf16x8 rk[RA + 1];
    auto rd = [&](int i) {
      rk[i % (RA + 1)] = as_bf16x8(lds_read16(kt, 32 * (i / kDK) * kRowB + (kb_ ^ ((i % kDK) << 5))));
    };
    rd(0);
    rd(1);
#pragma unroll
    for (int i = 0; i < kDK; ++i) {
      rd(i + RA);
      s0 = mfma32(rk[i % (RA + 1)], qf[i], s0);
      issue_step(t, nxt, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    // Chain 0 runs for every wave, as it carries the copies; the rest only for a wave with keys of
    // this tile to attend to (the others meet them at the barrier either way).
    if (!skip) {
      // Key kv0 + 4 hf + c (c = 32 kb + 8 (r >> 2) + (r & 3)) is visible to this lane's query iff
      // c <= thr (causal and tail bounds) and, packed, c >= lo (at or after the row's segment
      // start). Only tiles that cross the wave's diagonal, the sequence end or (packed) a segment
      // start are masked (scores of hidden keys set to -inf, so their probabilities are 0); the
      // test is per wave, a scalar branch before each half's softmax.
      const bool need_mask = (causal && kv0 + kKT - 1 > qw0) || (kv0 + kKT > S) || (PACKED && kv0 < w_sst_last) ||
                             (SPAN && kv0 + kKT > w_end_first);
      const int thr = qvalid ? ((SPAN ? my_end - 1 : causal && qi < S - 1 ? qi : S - 1) - kv0 - 4 * hf) : -1;
      const int lo = my_sst - kv0 - 4 * hf;
      {
        auto mask = [&](f32x16& sc, int kb) {
          if (need_mask) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int c = 32 * kb + 8 * (r >> 2) + (r & 3);
              bool ok = c <= thr;
              if (PACKED) ok = ok && (c >= lo);
              sc[r] = ok ? sc[r] : kNegInf;
            }
          }
        };
        // Probability r of half kb against the row bias nb into pf[2 kb + r / 8]; returns it.
        bf16x8 pf[4];
        const int side = (MOD & kModSlope) ? side_of(kv0) : 0;
        const float rel = (float)(qi - kv0 - 4 * hf);
        const float add = (MOD & kModSlope) ? score.slant_add(side, rel, top) : score.add;
        auto form = [&](f32x16& sc, int kb) {  // raw products into v (Score)
          if constexpr (MOD != kModNone) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = score.raw(sc[r]);
            if constexpr (MOD & kModSlope) score.template slant<kRamp>(sc, kb, side, rel);
          }
        };
        auto bias = [&]() { return MOD == kModNone ? ((m == kNegInf) ? 0.f : -m) : FIXED ? add : ((m == kNegInf) ? 0.f : -m) + add; };
        auto prob = [&](const f32x16& sc, int kb, int r, float nb) {
          const float p = fast_exp2(__builtin_fmaf(sc[r], MOD == kModNone ? scale_log2 : score.mul, nb));
          pf[2 * kb + (r >> 3)][r & 7] = (__bf16)p;
          return p;
        };
        // m = -inf only while every key seen by this row is masked; then p = exp2(-inf) = 0.
        float nb = bias();
        form(s0, 0);
        mask(s0, 0);
        // Chain 1, each product followed by an even share of half 0's 16 probabilities (written in
        // this order: the scheduler does not move them across the wave exchange below).
        float l0 = 0.f;
#pragma unroll
        for (int i = kDK; i < 2 * kDK; ++i) {
          if (i + RA < 2 * kDK) rd(i + RA);
          s1 = mfma32(rk[i % (RA + 1)], qf[i - kDK], s1);
#pragma unroll
          for (int r = 16 * (i - kDK) / kDK; r < 16 * (i - kDK + 1) / kDK; ++r) l0 += prob(s0, 0, r, nb);
        }
        // Half 0's speculative values are needed here, not only past the branches below (the mask
        // of half 1, the rescale that may replace them): otherwise the compiler sinks them out of
        // chain 1's shadows.
        asm volatile("" ::"v"(l0), "v"(pf[0]), "v"(pf[1]));
        // Transposed fragments of V (the O^T products' operand) for half 0, after chain 1's row
        // fragments; half 1's go out once these have returned.
        bf16x8 tf[4][4];
        tr_slab<0, kDB, kRowB>(a0, a1, tf);
        tr_slab<1, kDB, kRowB>(a0, a1, tf);
        form(s1, 1);
        mask(s1, 1);
        if constexpr (!FIXED) {
          float mx = kNegInf;
#pragma unroll
          for (int r = 0; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s0[r]), fmaxf(s1[r], fmaxf(s0[r + 1], s1[r + 1])));
          const float mt = MOD == kModNone ? max_xhalf(mx) * scale_log2  // scale_log2 > 0: the max of the scaled scores
                                           : max_xhalf(__builtin_fmaf(mx, score.mul, add));  // add differs by lane half
          // A row raises m only when the tile maximum exceeds it by more than kRescaleLog2: its O and
          // l are then rescaled together and half 0 recomputed; otherwise probabilities up to
          // 2^kRescaleLog2 accumulate against the old m. O / l and L = m + log2(l) are the same
          // either way. The branch is taken by the whole wave when any row needs it (most tiles
          // skip it), but each row decides for itself and the others keep their values bitwise (alpha
          // 1, half 0 recomputed identically): a row's arithmetic depends only on its own scores, so
          // rows of other packed segments sharing the wave come out bitwise the same whatever this
          // row's keys hold.
          const bool up = mt > m + kRescaleLog2;  // false while mt = -inf (all keys hidden)
          if (__builtin_amdgcn_ballot_w64(up) != 0) {
            const float alpha = up ? fast_exp2(m - mt) : 1.f;  // m = -inf: alpha = 0 (O, l are 0)
            m = up ? mt : m;
            l *= alpha;
            lr *= alpha;
#pragma unroll
            for (int db = 0; db < kDB; ++db)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
            nb = bias();
            l0 = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) l0 += prob(s0, 0, r, nb);
          }
        }
        l += l0;
        if constexpr (SCORED) {
          add_rounded(pf[0]);
          add_rounded(pf[1]);
        }
        // O^T += V^T P^T: half 0's two 16-key slabs, each product followed by an even share of half
        // 1's probabilities, then half 1's slabs.
        slab_wait<0, kDB>(tf[0]);
        slab_wait<0, kDB>(tf[1]);
        tr_slab<2, kDB, kRowB>(a0, a1, tf);
        tr_slab<3, kDB, kRowB>(a0, a1, tf);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int db = 0; db < kDB; ++db) {
            acc[db] = mfma32(tf[ks][db], pf[ks], acc[db]);
            const int u = kDB * ks + db;
#pragma unroll
            for (int r = 8 * u / kDB; r < 8 * (u + 1) / kDB; ++r) l += prob(s1, 1, r, nb);
          }
        slab_wait<0, kDB>(tf[2]);
        slab_wait<0, kDB>(tf[3]);
#pragma unroll
        for (int ks = 2; ks < 4; ++ks)
#pragma unroll
          for (int db = 0; db < kDB; ++db) acc[db] = mfma32(tf[ks][db], pf[ks], acc[db]);
        if constexpr (SCORED) {
          add_rounded(pf[2]);
          add_rounded(pf[3]);
        }
      }
    }
    // This wave's copies of tile t+1 landed; after the barrier nobody reads `cur`, which takes t+2.
    vm_wait0();
    lgkm_wait0();
    asm volatile("s_barrier" ::: "memory");
  };
  for (int t = 0; t < ntiles; t += 2) {
    if constexpr (DQ) {
      body(t, lds0, lds1);
      if (t + 1 < ntiles) body(t + 1, lds1, lds0);
    } else {
      fwd_body(t, lds0, lds1);
      if (t + 1 < ntiles) fwd_body(t + 1, lds1, lds0);
    }
  }

  float mul = (DQ && CAP) ? -4.f * scale : scale, lt = 0.f;  // (Score::bend)
  if constexpr (SPLIT) {
    const long rows = (long)B * Hq * S;
    if constexpr (!DQ) {
      lt = l + __shfl_xor(l, 32, 64);
      const float ltr = lr + __shfl_xor(lr, 32, 64);
      if (qvalid && hf == 0)
        *reinterpret_cast<f32x4*>(part + ns * rows * DH + 4 * (split * rows + qrow + qi)) = f32x4{m, lt, ltr, 0.f};
      mul = 1.f;
    }
    if (qvalid) {
      float* ph = part + (split * rows + qrow + qi) * DH;
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
          *reinterpret_cast<f32x4*>(ph + 32 * db + 8 * rq + 4 * hf) =
              f32x4{acc[db][4 * rq] * mul, acc[db][4 * rq + 1] * mul, acc[db][4 * rq + 2] * mul, acc[db][4 * rq + 3] * mul};
    }
    // The padding behind a program's end reads as a write of v0, which the listing check of stores whose data the next
    // instructions write would hold against a last store of v0.
    asm volatile("s_nop 0");
    return;
  }
  if constexpr (!DQ) {
    lt = l + __shfl_xor(l, 32, 64);
    const float by = SCORED ? lr + __shfl_xor(lr, 32, 64) : lt;
    mul = (by > 0.f) ? 1.f / by : 0.f;
  }
  if constexpr (!DQ) {
    // A query that sees nothing: L = +inf, so that the backward's probabilities exp(S - L) are 0.
    if (qvalid && hf == 0) lse_out[qrow + qi] = (SPAN && !(lt > 0.f)) ? -kNegInf : (m + fast_log2(lt)) * kLn2;
  }
  auto quad = [&](int db, int rq) __attribute__((always_inline)) {  // dims 32 db + 8 rq + 4 hf .. + 3
    return u32x2{pack_bf16x2(acc[db][4 * rq] * mul, acc[db][4 * rq + 1] * mul),
                 pack_bf16x2(acc[db][4 * rq + 2] * mul, acc[db][4 * rq + 3] * mul)};
  };
  if constexpr (SCORED && !DQ) {
    if (o_low != nullptr && wave_has) {
      // As O's below, through this wave's quarter of stage 1, rows of DH bytes 16 apart.
      char* ob = lds1 + w * (32 * (DH + 16));
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const u32x2 x = quad(db, rq);
          uint32_t bytes = 0;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t top = (u & 1) ? x[u >> 1] & 0xffff0000u : x[u >> 1] << 16;
            bytes |= below_bf16(acc[db][4 * rq + u] * mul, top) << (8 * u);
          }
          *reinterpret_cast<uint32_t*>(ob + col * (DH + 16) + 32 * db + 8 * rq + 4 * hf) = bytes;
        }
      int8_t* lh = o_low + (qrow + qw0) * DH;
#pragma unroll
      for (int p = 0; p < DH / 32; ++p) {
        const int id = lane + 64 * p, row = id / (DH / 16), c = id % (DH / 16);
        const u32x4 x = *reinterpret_cast<const u32x4*>(ob + row * (DH + 16) + 16 * c);
        if (qw0 + row < S) *reinterpret_cast<u32x4*>(lh + row * DH + 16 * c) = x;
      }
    }
  }
  if constexpr (DH == 96) {
    // Rows of 192 bytes, a line and a half: through LDS measured the same (88.8 and 89.0 us at
    // 2 x 16/4 x 2050, not causal).
    if (!qvalid) return;
    bf16_t* oh = out + (qrow + qi) * DH;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) *reinterpret_cast<u32x2*>(oh + 32 * db + 8 * rq + 4 * hf) = quad(db, rq);
  } else {
    if (!wave_has) return;
    // The wave's 32 rows through its quarter of stage 0 (nobody reads or copies into it past the last
    // barrier), so that a store writes whole rows: 16-byte chunk c of row r at slot c ^ r (head_dim 64:
    // c ^ r / 2) of its 256 (128) bytes. 8 bytes per lane from the accumulator layout wrote a line in 16
    // pieces, which counts where walks are short: packed S = 16384 (~12 key tiles a walk) forward 261 -> 252
    // us and backward 806 -> 792, 4 x 16/4 x 1000 x 128 causal 29.3 -> 27.2 and 100.2 -> 97.8, S = 8192
    // causal 497 -> 492 and 1617 -> 1614.
    char* ob = lds0 + w * (32 * kRowB);
    auto slot = [&](int row, int c) { return row * kRowB + ((c ^ (DH == 64 ? (row >> 1) & 7 : row & 15)) << 4); };
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq)
        *reinterpret_cast<u32x2*>(ob + slot(col, 4 * db + rq) + 8 * hf) = quad(db, rq);
    bf16_t* oh = out + (qrow + qw0) * DH;
#pragma unroll
    for (int p = 0; p < DH / 16; ++p) {
      const int id = lane + 64 * p, row = id / (DH / 8), c = id % (DH / 8);
      const u32x4 x = *reinterpret_cast<const u32x4*>(ob + slot(row, c));
      if (qw0 + row < S) *reinterpret_cast<u32x4*>(oh + row * DH + 8 * c) = x;
    }
  }
}

}  // namespace mtp

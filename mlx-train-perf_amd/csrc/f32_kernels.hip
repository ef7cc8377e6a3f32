// fp32 inputs: the fused linear cross-entropy and flash attention for fp32 hidden states / q, k, v
// (the reference kernels take fp32 as well as bf16: core/loss.py:24, attention/api.py:41-43).
//
// Arithmetic is fp32 end to end: fp32 MFMA products (exact fp32 multiplies, fp32 accumulation;
// v_mfma_f32_32x32x2_f32 in the LCE, v_mfma_f32_16x16x4_f32 in attention), fp32 softmax statistics,
// fp32 outputs and gradients. The algorithms are those of
// the bf16 kernels (lce_kernels.hip, attn_kernels.hip) and of the reference's oracles:
//   LCE forward: per token lse = logsumexp_v(h . w_v) (online over vocab tiles, vocab splits merged
//     by the finalize), tgt = h . w_y, nll = lse - tgt (core/naive.py:9-14, core/chunked.py:35-49);
//   LCE backward: g = (exp(z - lse) - onehot) * ct in fp32 per vocab chunk, dH = g . W_chunk,
//     dW = g^T . H (core/chunked.py:52-90);
//   attention: O = softmax(scale Q K^T + mask) V, L = row logsumexp; backward D = rowsum(dO O),
//     dS = P (dP - D), dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO summed over each kv head's
//     query-head group (attention/reference.py:37-116, attention/api.py:126-194).
//
// MFMA 32x32x2 f32 lane layout (wave64): lane l supplies A[i = l % 32][k = l / 32] and
// B[k = l / 32][j = l % 32]; its 16 results are C[i = 8 (r / 4) + 4 (l / 32) + r % 4][j = l % 32]. Which k a
// lane half contracts at which step is each core's choice (both operands make the same), so that a lane
// reads consecutive k of its row: the register-staged core k = 8 h + s of 16, the copied one
// 8 c + 4 h + s of 32. The 16x16x4 layout stands at the attention kernels.
#include "attn32_core.hpp"
#include "score_gather.hpp"

namespace mtp {
namespace f32k {

__device__ __forceinline__ f32x16 mfma2(float a, float b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void zero(f32x16& a) {
#pragma unroll
  for (int r = 0; r < 16; ++r) a[r] = 0.f;
}
// Key (or query) index, within a 32-block, of accumulator register r of lane half h.
__device__ __forceinline__ int rrow(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// ------------------------------------------------------------------------------------------
// GEMM core: C[128][128] (+)= A[128][K] . B[128][K]^T over K in 16-deep LDS stages, 4 waves of
// 64 x 64 (wave w: A rows 64 (w & 1), B rows 64 (w >> 1)). Operand tiles are staged through
// registers into LDS in one of two layouts:
//   row: [128 rows][16 k] with a 20-float pitch (16-byte fragment reads of 16 lanes hit distinct
//        banks);
//   col: [16 k][128 rows] with a 132-float pitch (the two lane halves read disjoint banks).
// Sources: `RowSrc` (row-major [rows][ld], k along a row), `ColSrc` (k-major [k][ld], rows along a
// k row), and the 4-bit affine head in either role (`Q4RowSrc`, `Q4ColSrc`: w = s * q + b in fp32,
// 8 nibbles per u32, low first, scale and bias per 64 along the hidden dim). Out-of-range elements
// read as zero.
// ------------------------------------------------------------------------------------------
constexpr int kT = 128, kBK = 16, kRowPitch = 20, kColPitch = 132;
constexpr int kTileFloats = 2560;  // >= 128 * 20 and 16 * 132

struct RowSrc {
  static constexpr bool kCol = false;
  const float* p;
  long ld;
  int rows, K;
  bool vec;
  __device__ __forceinline__ float at(int r, int k) const { return (r < rows && k < K) ? p[(long)r * ld + k] : 0.f; }
  __device__ __forceinline__ f32x4 quad(int r, int k) const {
    if (vec && r < rows && k + 3 < K) return *reinterpret_cast<const f32x4*>(p + (long)r * ld + k);
    return f32x4{at(r, k), at(r, k + 1), at(r, k + 2), at(r, k + 3)};
  }
};
struct ColSrc {
  static constexpr bool kCol = true;
  const float* p;  // [k][ld], element (k, r)
  long ld;
  int rows, K;
  bool vec;
  __device__ __forceinline__ float at(int k, int r) const { return (r < rows && k < K) ? p[(long)k * ld + r] : 0.f; }
  __device__ __forceinline__ f32x4 quad(int k, int r) const {
    if (vec && k < K && r + 3 < rows) return *reinterpret_cast<const f32x4*>(p + (long)k * ld + r);
    return f32x4{at(k, r), at(k, r + 1), at(k, r + 2), at(k, r + 3)};
  }
};
// 4-bit head rows v (tile rows) along the hidden dim d (k): W[v][d].
struct Q4Geom {
  const uint32_t* wq;
  const float* sc;
  const float* bi;
  int D;
  __device__ __forceinline__ float w(long v, int d) const {
    const uint32_t word = wq[v * (D >> 3) + (d >> 3)];
    const long g = v * (D >> 6) + (d >> 6);
    return __builtin_fmaf(sc[g], (float)((word >> (4 * (d & 7))) & 0xFu), bi[g]);
  }
};
struct Q4RowSrc {
  static constexpr bool kCol = false;
  Q4Geom q;
  long v0;
  int rows, K;
  __device__ __forceinline__ f32x4 quad(int r, int k) const {
    f32x4 x;
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = (r < rows && k + u < K) ? q.w(v0 + r, k + u) : 0.f;
    return x;
  }
};
// The 4-bit head as the k-major operand: element (k = vocab row, r = hidden index).
struct Q4ColSrc {
  static constexpr bool kCol = true;
  Q4Geom q;
  long v0;
  int rows, K;  // rows: hidden dims from the tile start, K: vocab rows
  int d0;
  __device__ __forceinline__ f32x4 quad(int k, int r) const {
    f32x4 x;
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = (k < K && r + u < rows) ? q.w(v0 + k, d0 + r + u) : 0.f;
    return x;
  }
};

// One operand's share of a stage: thread t fetches quads idx = t + 256 p (p = 0, 1) of the 512.
template <class Src>
__device__ __forceinline__ void fetch(const Src& s, int k0, f32x4 (&x)[2]) {
  const int t = threadIdx.x;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int idx = t + 256 * p;
    if constexpr (Src::kCol) x[p] = s.quad(k0 + (idx >> 5), 4 * (idx & 31));
    else x[p] = s.quad(idx >> 2, k0 + 4 * (idx & 3));
  }
}
template <bool COL>
__device__ __forceinline__ void put(const f32x4 (&x)[2], float* lds) {
  const int t = threadIdx.x;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int idx = t + 256 * p;
    const int off = COL ? (idx >> 5) * kColPitch + 4 * (idx & 31) : (idx >> 2) * kRowPitch + 4 * (idx & 3);
    *reinterpret_cast<f32x4*>(lds + off) = x[p];
  }
}
// Fragments of the wave's two 32-row blocks for the 8 steps of a stage: v[b][s].
template <bool COL>
__device__ __forceinline__ void frags(const float* lds, int r0, float (&v)[2][8]) {
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    if constexpr (COL) {
#pragma unroll
      for (int s = 0; s < 8; ++s) v[b][s] = lds[(8 * h + s) * kColPitch + r0 + 32 * b + i];
    } else {
      const float* row = lds + (r0 + 32 * b + i) * kRowPitch + 8 * h;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(row);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(row + 4);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        v[b][s] = lo[s];
        v[b][4 + s] = hi[s];
      }
    }
  }
}

// acc[bi][bj] = C[64 (w & 1) + 32 bi + ..][64 (w >> 1) + 32 bj + ..]. `lds` holds 4 tiles:
// [stage][A, B].
template <class SA, class SB>
__device__ __forceinline__ void gemm128(const SA& sa, const SB& sb, int K, float* lds, f32x16 (&acc)[2][2]) {
  const int w = threadIdx.x >> 6;
  const int ra = 64 * (w & 1), rb = 64 * (w >> 1);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) zero(acc[i][j]);
  const int nk = (K + kBK - 1) / kBK;
  f32x4 xa[2], xb[2];
  fetch(sa, 0, xa);
  fetch(sb, 0, xb);
  put<SA::kCol>(xa, lds);
  put<SB::kCol>(xb, lds + kTileFloats);
  __syncthreads();
  for (int kt = 0; kt < nk; ++kt) {
    float* cur = lds + (kt & 1) * 2 * kTileFloats;
    float* nxt = lds + ((kt + 1) & 1) * 2 * kTileFloats;
    if (kt + 1 < nk) {
      fetch(sa, (kt + 1) * kBK, xa);
      fetch(sb, (kt + 1) * kBK, xb);
    }
    float fa[2][8], fb[2][8];
    frags<SA::kCol>(cur, ra, fa);
    frags<SB::kCol>(cur + kTileFloats, rb, fb);
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma2(fa[i][s], fb[j][s], acc[i][j]);
    if (kt + 1 < nk) {
      put<SA::kCol>(xa, nxt);
      put<SB::kCol>(xb, nxt + kTileFloats);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------
// The same product on copied tiles (dense operands whose rows are multiples of 16 bytes): 32-deep stages of
// 16 KiB per operand, copied global -> LDS one stage ahead, one barrier per stage; two workgroups per CU.
// The matrix pipe bounds it (4096 MFMA cycles per wave and stage against 32 KiB copied and 16 KiB
// read); the register-staged core above stalls on its loads and LDS writes. N = 1024, D = 512, V = 32000, the
// kernels' times in one trace: forward 363 -> 305 us, gradient tiles 391 -> 343, dH 367 -> 302; the whole
// step 1043 -> 827 us (122 of the 153 TFLOP/s a library fp32 matrix product reaches). Two 256-register
// waves per SIMD: left to a budget of 512 the compiler moved the accumulators between VGPRs and AGPRs
// in every stage.
//   RowOp: k along a row: [128 rows][32 k], chunk c (4 k) of row r at slot c ^ swz32(r); a lane reads chunk
//          2 c + h of its row for the 4 steps of c.
//   ColOp: k-major: [32 k][128 columns]; a lane reads columns 2 i and 2 i + 1 of the k rows of its half, so
//          block b of a wave holds the columns 2 i + b.
// Lane half h contracts k = 8 c + 4 h + s at step s of c, in both. Rows, k and columns past the end read
// as zeros or (columns of a k-major operand) as neighbours whose results are not stored.
// ------------------------------------------------------------------------------------------
constexpr int kDK = 32, kOpB = 16384;
__device__ __forceinline__ int swz32(int r) { return (r ^ ((r >> 3) & 3)) & 7; }
__device__ __forceinline__ int range31(long bytes) { return bytes <= 0 ? 0 : bytes > 0x7fffffffL ? 0x7fffffff : (int)bytes; }

struct RowOp {
  const float* p;  // tile row 0, k = 0
  long ld;
  int rows, K;     // rows from the tile start, contraction length
  uint32_t voff;   // this lane's offset in its wave's copy 0; copy m lies 32 m rows on
  int ck;          // first k of the lane's chunk
  __device__ __forceinline__ RowOp(const float* p_, long ld_, int rows_, int K_) : p(p_), ld(ld_), rows(rows_ < kT ? rows_ : kT), K(K_) {
    const int lane = threadIdx.x & 63, row = 8 * (threadIdx.x >> 6) + (lane >> 3);
    ck = 4 * ((lane & 7) ^ swz32(row));
    voff = 4u * (uint32_t)(row * (int)ld + ck);
  }
  static __device__ __forceinline__ int pos(int b, int i) { return 32 * b + i; }
  __device__ __forceinline__ void copy(int kt, char* dst) const {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), left = K - kt * kDK;
    // (a gradient tile's row may end inside a chunk: its zeros up to the chunk's end are read too)
    const int bytes = left > 0 ? range31(4 * ((rows - 1) * ld + ((left + 3) & ~3))) : 0;
    const uint32_t v = ck < left ? voff : 0x60000000u;  // past the end of its row: nothing
#pragma unroll
    for (int m = 0; m < 4; ++m) lds_copy16(p + kt * kDK, bytes, dst + 1024 * (4 * m + w), v + 128u * m * (uint32_t)ld);
  }
  __device__ __forceinline__ void frags(const char* st, int first, int c, float (&v)[2][4]) const {
    const int i = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1, row = first + i;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(st + row * 128 + (((h ^ swz32(row)) << 4) ^ (c << 5)) + 4096 * b);
#pragma unroll
      for (int s = 0; s < 4; ++s) v[b][s] = x[s];
    }
  }
};
struct ColOp {
  const float* p;  // k = 0, tile column 0
  long ld;
  int cols, K;     // columns from the tile start to the end of the row, contraction length
  uint32_t voff;   // this lane's offset in its wave's copy 0; copy m lies 8 m k rows on
  __device__ __forceinline__ ColOp(const float* p_, long ld_, int cols_, int K_) : p(p_), ld(ld_), cols(cols_), K(K_) {
    const int lane = threadIdx.x & 63;
    voff = 4u * (uint32_t)((2 * (threadIdx.x >> 6) + (lane >> 5)) * (int)ld + 4 * (lane & 31));
  }
  static __device__ __forceinline__ int pos(int b, int i) { return 2 * i + b; }
  __device__ __forceinline__ void copy(int kt, char* dst) const {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), left = K - kt * kDK;
    const int bytes = left > 0 ? range31(4 * ((left - 1) * ld + cols)) : 0;
#pragma unroll
    for (int m = 0; m < 4; ++m) lds_copy16(p + kt * kDK * ld, bytes, dst + 1024 * (4 * m + w), voff + 32u * m * (uint32_t)ld);
  }
  __device__ __forceinline__ void frags(const char* st, int first, int c, float (&v)[2][4]) const {
    const int i = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const f32x2 x = *reinterpret_cast<const f32x2*>(st + (8 * c + 4 * h + s) * 512 + 4 * (first + 2 * i));
      v[0][s] = x[0];
      v[1][s] = x[1];
    }
  }
};
// acc[bi][bj] = C[64 (w & 1) + OA::pos(bi, ..)][64 (w >> 1) + OB::pos(bj, ..)]; s0 and s1 hold A, then B.
template <class OA, class OB>
__device__ __forceinline__ void gemm128_copied(const OA& oa, const OB& ob, int K, char* s0, char* s1, f32x16 (&acc)[2][2]) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ra = 64 * (w & 1), rb = 64 * (w >> 1);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) zero(acc[i][j]);
  const int nk = (K + kDK - 1) / kDK;
  auto stage = [&](int kt, const char* cur, char* nxt) __attribute__((always_inline)) {
    oa.copy(kt + 1, nxt);  // past the end: nothing read, zeros into a stage nobody reads
    ob.copy(kt + 1, nxt + kOpB);
    float fa[2][2][4], fb[2][2][4];  // one chunk pair ahead
    oa.frags(cur, ra, 0, fa[0]);
    ob.frags(cur + kOpB, rb, 0, fb[0]);
    // Keeps the copies up here (the scheduler sank the last one to its wait) and each chunk pair's
    // reads ahead of the products they run under.
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c < 3) {
        oa.frags(cur, ra, c + 1, fa[(c + 1) & 1]);
        ob.frags(cur + kOpB, rb, c + 1, fb[(c + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = mfma2(fa[c & 1][i][s], fb[c & 1][j][s], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    copies_landed();
  };
  oa.copy(0, s0);
  ob.copy(0, s0 + kOpB);
  copies_landed();
  for (int kt = 0; kt < nk; kt += 2) {
    stage(kt, s0, s1);
    if (kt + 1 < nk) stage(kt + 1, s1, s0);
  }
}

__device__ __forceinline__ bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
// Head kinds of the kernels below: dense (any hidden dim), 4-bit, dense on the copied-tile core.
constexpr int kDense = 0, kQ4 = 1, kCopied = 2;
template <int KIND>
constexpr int kStage0 = KIND == kCopied ? 2 * kOpB : 4 * kTileFloats * 4;
template <int KIND>
constexpr int kStage1 = KIND == kCopied ? 2 * kOpB : 16;

// ------------------------------------------------------------------------------------------
// LCE forward: workgroup (128-token tile, vocab split) walks the split's 128-column vocab tiles;
// C[v][t] = W_v . H_t, so each lane owns token columns and keeps an online (max, sum of exp2) per
// token, merged with lane ^ 32 and the other vocab-half wave at the end into part_m/part_s
// [split][N] (log2 domain), which the finalize merges. STAT as in lce_fwd_kernel (lce_kernels.hip).
// ------------------------------------------------------------------------------------------
template <int KIND, int STAT = 0>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void lce32_fwd_kernel(const float* __restrict__ H, const float* __restrict__ W,
                                                        const uint32_t* __restrict__ Wq, const float* __restrict__ Sc,
                                                        const float* __restrict__ Bi, int N, int D, int V, int nsplit,
                                                        float* __restrict__ part_m, float* __restrict__ part_s, float scale2,
                                                        float* __restrict__ part_u, float* __restrict__ gmax, int ldg,
                                                        float* __restrict__ Z, long ldz, ScoreList list) {
  const float c2 = STAT ? scale2 : kLog2e;
  __shared__ float gx[(STAT & kStatGroups) ? kT : 1];
  __shared__ __attribute__((aligned(1024))) char s0[kStage0<KIND>];
  __shared__ __attribute__((aligned(1024))) char s1[kStage1<KIND>];
  float* lds = reinterpret_cast<float*>(s0);
  const int t0 = blockIdx.x * kT, split = blockIdx.y;
  const int vtiles = (V + kT - 1) / kT;
  const int per = (vtiles + nsplit - 1) / nsplit;
  const int vt0 = split * per, vt1 = (vt0 + per < vtiles) ? vt0 + per : vtiles;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wa = w & 1, wb = w >> 1, h = lane >> 5;
  RowSrc hb{H + (long)t0 * D, D, N - t0, D, aligned16(H) && D % 4 == 0};
  float m[2] = {kNegInf, kNegInf}, s[2] = {0.f, 0.f}, u[2] = {0.f, 0.f};
  std::conditional_t<(STAT & kStatEntropy) != 0, TargetCursor<2>, ListCursor<2>> cursor;
  const int tokens[2] = {t0 + 64 * wb + (lane & 31), t0 + 64 * wb + 32 + (lane & 31)};
  if constexpr (STAT & kStatList) cursor.start(list, tokens, N, vt0 * kT);
  for (int vt = vt0; vt < vt1; ++vt) {
    const int v0 = vt * kT;
    f32x16 acc[2][2];
    if constexpr (KIND == kCopied) {
      gemm128_copied(RowOp(W + (long)v0 * D, D, V - v0, D), RowOp(H + (long)t0 * D, D, N - t0, D), D, s0, s1, acc);
    } else if constexpr (KIND == kQ4) {
      Q4RowSrc wa_{Q4Geom{Wq, Sc, Bi, D}, v0, V - v0, D};
      gemm128(wa_, hb, D, lds, acc);
    } else {
      RowSrc wa_{W + (long)v0 * D, D, V - v0, D, aligned16(W) && D % 4 == 0};
      gemm128(wa_, hb, D, lds, acc);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (v0 + 64 * wa + 32 * i + rrow(r, h) >= V) acc[i][j][r] = kNegInf;
      if constexpr (STAT & kStatKeep) {
        const int t = t0 + 64 * wb + 32 * j + (lane & 31);
        if (t < N) {
          float* row = Z + t * ldz + v0 + 64 * wa + 4 * h;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<f32x4*>(row + 32 * i + 8 * q) =
                  f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
      }
    }
    if constexpr (STAT & kStatList) cursor.template take<kT>(list, tokens, acc, v0, 64 * wa, h);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mz = kNegInf;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) mz = fmaxf(mz, acc[i][j][r]);
      if constexpr (STAT & kStatGroups) {  // the tile's maximum of each token: of both halves of both waves
        const float both = fmaxf(mz, __shfl_xor(mz, 32, 64));
        const int tl = 64 * wb + 32 * j + (lane & 31);
        if (wa == 1 && h == 0) gx[tl] = both;
        __syncthreads();
        if (wa == 0 && h == 0 && t0 + tl < N) gmax[(long)(t0 + tl) * ldg + vt] = fmaxf(both, gx[tl]);
      }
      const float mn = fmaxf(m[j], mz * c2);
      const float base = (mn == kNegInf) ? 0.f : mn;
      float sum = 0.f, sumu = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = __builtin_fmaf(acc[i][j][r], c2, -base);
          const float e = fast_exp2(x);
          sum += e;
          if constexpr (STAT & kStatEntropy) sumu = __builtin_fmaf(e, finite_exponent(x), sumu);
        }
      const float f = fast_exp2(m[j] - base);
      if constexpr (STAT & kStatEntropy) u[j] = __builtin_fmaf(s[j], m[j] == kNegInf ? 0.f : m[j] - base, u[j]) * f + sumu;
      s[j] = s[j] * f + sum;
      m[j] = mn;
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float mo = __shfl_xor(m[j], 32, 64), so = __shfl_xor(s[j], 32, 64);
    if constexpr (STAT & kStatEntropy) lse2_merge(m[j], s[j], u[j], mo, so, __shfl_xor(u[j], 32, 64));
    else lse2_merge(m[j], s[j], mo, so);
  }
  __syncthreads();
  float* xm = lds;
  float* xs = lds + 128;
  float* xu = lds + 256;
  if (wa == 1 && h == 0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      xm[64 * wb + 32 * j + (lane & 31)] = m[j];
      xs[64 * wb + 32 * j + (lane & 31)] = s[j];
      if constexpr (STAT & kStatEntropy) xu[64 * wb + 32 * j + (lane & 31)] = u[j];
    }
  }
  __syncthreads();
  if (wa == 0 && h == 0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int tl = 64 * wb + 32 * j + (lane & 31);
      if constexpr (STAT & kStatEntropy) lse2_merge(m[j], s[j], u[j], xm[tl], xs[tl], xu[tl]);
      else lse2_merge(m[j], s[j], xm[tl], xs[tl]);
      if (t0 + tl < N) {
        part_m[(long)split * N + t0 + tl] = m[j];
        part_s[(long)split * N + t0 + tl] = s[j];
        if constexpr (STAT & kStatEntropy) part_u[(long)split * N + t0 + tl] = u[j];
      }
    }
  }
}

// H_t . W_y as an fp32 dot product over the wave (every lane returns the total).
template <int Q4>
__device__ __forceinline__ float row_dot32(const float* __restrict__ h, const float* __restrict__ W,
                                           const uint32_t* __restrict__ Wq, const float* __restrict__ Sc,
                                           const float* __restrict__ Bi, long long y, int D, int lane) {
  float dot = 0.f;
  if constexpr (Q4) {
    const Q4Geom q{Wq, Sc, Bi, D};
    for (int d = lane; d < D; d += 64) dot = __builtin_fmaf(h[d], q.w(y, d), dot);
  } else {
    const float* wr = W + (long)y * D;
    for (int d = lane; d < D; d += 64) dot = __builtin_fmaf(h[d], wr[d], dot);
  }
  return wave_sum(dot);
}

// Per token (one wave each): merge the splits into lse, tgt = H_t . W_y as an fp32 dot product,
// ignore_index rows nll = 0 and tgt = 0, out-of-range targets tgt = 0 (nll = lse).
template <int Q4>
__global__ __launch_bounds__(256) void lce32_finalize_kernel(const float* __restrict__ H, const float* __restrict__ W,
                                                             const uint32_t* __restrict__ Wq, const float* __restrict__ Sc,
                                                             const float* __restrict__ Bi, const int64_t* __restrict__ targets,
                                                             int N, int D, int V, int nsplit, const float* __restrict__ part_m,
                                                             const float* __restrict__ part_s, long long ignore_index,
                                                             float* __restrict__ nll, float* __restrict__ lse,
                                                             float* __restrict__ tgt) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= N) return;
  float mm = kNegInf, ss = 0.f;
  for (int sp = lane; sp < nsplit; sp += 64) lse2_merge(mm, ss, part_m[(long)sp * N + t], part_s[(long)sp * N + t]);
  const float gm = wave_max(mm);
  const float base = (gm == kNegInf) ? 0.f : gm;
  const float gs = wave_sum(ss * fast_exp2(mm - base));
  const float l = (base + fast_log2(gs)) * kLn2;
  const long long y = targets[t];
  const bool ignored = y == ignore_index;
  const bool inrange = y >= 0 && y < (long long)V;
  float dot = 0.f;
  if (!ignored && inrange) dot = row_dot32<Q4>(H + (long)t * D, W, Wq, Sc, Bi, y, D, lane);
  if (lane == 0) {
    lse[t] = l;
    tgt[t] = (ignored || !inrange) ? 0.f : dot;
    nll[t] = ignored ? 0.f : l - ((!inrange) ? 0.f : dot);
  }
}

// Gradient tile of the backward: C[t][v] = H_t . W_v for rows [row0, row0 + nrows) and the chunk's
// columns [c0, c0 + ncols); G[t][v - c0] = (exp(C - lse_t) - [v == y_t]) * coef_t in fp32, coef_t =
// d_nll[t] (0 for ignored rows), 0 past the vocab end (up to a multiple of 4 columns, which the dH
// product reads). AFFINE as in lce_bwd_g_persist_kernel (lce_kernels.hip).
template <int KIND, int AFFINE = 0>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void lce32_bwd_g_kernel(const float* __restrict__ H, const float* __restrict__ W,
                                                          const uint32_t* __restrict__ Wq, const float* __restrict__ Sc,
                                                          const float* __restrict__ Bi, const int64_t* __restrict__ targets,
                                                          const float* __restrict__ lse, const float* __restrict__ dnll,
                                                          int D, int V, long long ignore_index, int row0, int nrows,
                                                          int c0, int ncols, float* __restrict__ G, long ldg,
                                                          AffineRows rows) {
  __shared__ __attribute__((aligned(1024))) char s0[kStage0<KIND>];
  __shared__ __attribute__((aligned(1024))) char s1[kStage1<KIND>];
  float* lds = reinterpret_cast<float*>(s0);
  const int tt = blockIdx.x * kT, vv = blockIdx.y * kT;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wa = w & 1, wb = w >> 1, h = lane >> 5;
  RowSrc hs{H + (long)(row0 + tt) * D, D, nrows - tt, D, aligned16(H) && D % 4 == 0};
  const int v0 = c0 + vv;
  // Per row: coefficient, log2-domain lse and the target's column in the chunk (-1: none), fetched ahead
  // of the product (it has barriers between these writes and the reads below).
  __shared__ float rcoef[kT], rl2[kT];
  __shared__ int ry[kT];  // AFFINE: the bits of beta
  if (AFFINE && threadIdx.x < kT) {
    const int t = row0 + tt + threadIdx.x;
    const bool ok = tt + (int)threadIdx.x < nrows;
    rcoef[threadIdx.x] = ok ? rows.alpha[t] : 0.f;
    rl2[threadIdx.x] = ok ? lse[t] * kLog2e : 0.f;
    ry[threadIdx.x] = __builtin_bit_cast(int, ok && rows.beta ? rows.beta[t] : 0.f);
  } else if (threadIdx.x < kT) {
    const int t = row0 + tt + threadIdx.x;
    const bool ok = tt + (int)threadIdx.x < nrows;
    const long long y = ok ? targets[t] : -1;
    rcoef[threadIdx.x] = ok && y != ignore_index ? dnll[t] : 0.f;
    rl2[threadIdx.x] = ok ? lse[t] * kLog2e : 0.f;
    ry[threadIdx.x] = y >= c0 && y - c0 < ncols ? (int)(y - c0) : -1;
  }
  f32x16 acc[2][2];
  if constexpr (KIND == kCopied) {
    gemm128_copied(RowOp(H + (long)(row0 + tt) * D, D, nrows - tt, D), RowOp(W + (long)v0 * D, D, V - v0, D), D, s0, s1, acc);
  } else if constexpr (KIND == kQ4) {
    Q4RowSrc ws{Q4Geom{Wq, Sc, Bi, D}, v0, V - v0, D};
    gemm128(hs, ws, D, lds, acc);
  } else {
    RowSrc ws{W + (long)v0 * D, D, V - v0, D, aligned16(W) && D % 4 == 0};
    gemm128(hs, ws, D, lds, acc);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int rl = 64 * wa + 32 * i + rrow(r, h), tl = tt + rl;
      if (tl >= nrows) continue;
      const float coef = rcoef[rl], l2 = rl2[rl];
      const int y = ry[rl];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int vl = vv + 64 * wb + 32 * j + (lane & 31);
        if (vl >= ((ncols + 3) & ~3)) continue;
        float g = 0.f;
        if constexpr (AFFINE) {
          const float slope = __builtin_bit_cast(float, y);
          const float p = fast_exp2(__builtin_fmaf(acc[i][j][r], rows.scale2, -l2));
          if (c0 + vl < V && (coef != 0.f || slope != 0.f)) g = p * __builtin_fmaf(slope, finite_exponent(acc[i][j][r]), coef);
        } else if (c0 + vl < V) {
          const float p = fast_exp2(__builtin_fmaf(acc[i][j][r], kLog2e, -l2));
          g = (p - (vl == y ? 1.f : 0.f)) * coef;
        }
        G[(long)tl * ldg + vl] = g;
      }
    }
}

// A row's listed columns of an affine gradient (column < 0: none), one wave per row.
__global__ __launch_bounds__(256) void lce32_bwd_g_columns_kernel(const int* __restrict__ columns,
                                                                  const float* __restrict__ value, int k, int nrows, int c0,
                                                                  int ncols, float* __restrict__ G, long ldg) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= nrows) return;
  for (int i = threadIdx.x & 63; i < k; i += 64) {
    const int y = columns[(long)t * k + i];
    if (y >= c0 && y - c0 < ncols) G[(long)t * ldg + (y - c0)] = value[(long)t * k + i];
  }
}

// The rows of a gather's entries as an operand: past the last entry zeros. Offsets from H in 32 bits: a pass has at most
// kScoreRows tokens, of fewer than 2^15 dims on the copied core.
struct GatherSrc {
  static constexpr bool kCol = false;
  const float* p;
  const int2* entries;
  int D, count, K;
  bool vec;
  __device__ __forceinline__ float at(const float* row, int k) const { return k < K ? row[k] : 0.f; }
  __device__ __forceinline__ f32x4 quad(int r, int k) const {
    if (r >= count) return f32x4{0.f, 0.f, 0.f, 0.f};
    const float* row = p + (long)entries[r].x * D;
    if (vec && k + 3 < K) return *reinterpret_cast<const f32x4*>(row + k);
    return f32x4{at(row, k), at(row, k + 1), at(row, k + 2), at(row, k + 3)};
  }
};
struct GatherOp : RowOp {
  uint32_t off[4];
  __device__ __forceinline__ GatherOp(const float* p_, const int2* entries, int count, int D) : RowOp(p_, D, kT, D) {
    const int first = 8 * (threadIdx.x >> 6) + ((threadIdx.x & 63) >> 3);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int r = first + 32 * m;
      off[m] = r < count ? 4u * ((uint32_t)entries[r].x * (uint32_t)D + (uint32_t)ck) : 0x80000000u;  // out of any range
    }
  }
  __device__ __forceinline__ void copy(int kt, char* dst) const {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), left = K - kt * kDK;
    const bool in = ck < left;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      lds_copy16(p + kt * kDK, left > 0 ? 0x7fffffff : 0, dst + 1024 * (4 * m + w), in ? off[m] : 0x80000000u);
  }
};

// The logits of a gather's entries (GatherPlan): C[v][entry] = W_v . H_token of one group and up to 128 entries.
template <int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void lce32_gather_kernel(const float* __restrict__ H, const float* __restrict__ W, const uint32_t* __restrict__ Wq,
                         const float* __restrict__ Sc, const float* __restrict__ Bi, int D, int V, GatherPlan plan) {
  static_assert(kT == kGroup, "a tile is a group");
  __shared__ __attribute__((aligned(1024))) char s0[kStage0<KIND>];
  __shared__ __attribute__((aligned(1024))) char s1[kStage1<KIND>];
  const GatherTile tile = plan.tiles[blockIdx.x];
  if (tile.count == 0) return;
  const int2* entries = plan.entries + tile.first;
  const int v0 = tile.group * kGroup;
  f32x16 acc[2][2];
  if constexpr (KIND == kCopied) {
    gemm128_copied(RowOp(W + (long)v0 * D, D, V - v0, D), GatherOp(H, entries, tile.count, D), D, s0, s1, acc);
  } else {
    GatherSrc hs{H, entries, D, tile.count, D, aligned16(H) && D % 4 == 0};
    float* lds = reinterpret_cast<float*>(s0);
    if constexpr (KIND == kQ4) {
      Q4RowSrc ws{Q4Geom{Wq, Sc, Bi, D}, v0, V - v0, D};
      gemm128(ws, hs, D, lds, acc);
    } else {
      RowSrc ws{W + (long)v0 * D, D, V - v0, D, aligned16(W) && D % 4 == 0};
      gemm128(ws, hs, D, lds, acc);
    }
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  store_gathered<2, 2>(acc, plan, entries, tile.count, V - v0, 64 * (w & 1), 64 * (w >> 1), lane);
}

// Stores (ACC: adds) a product's tile to C[M][N]: blockIdx.x: 128 rows, blockIdx.y: 128 columns. PA, PB: the
// operands' order of rows within a wave's 64 (the register-staged sources have RowOp's).
template <bool ACC, class PA = RowOp, class PB = RowOp>
__device__ __forceinline__ void store_tile(const f32x16 (&acc)[2][2], int M, int N, float* __restrict__ C, long ldc) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wa = w & 1, wb = w >> 1, h = lane >> 5;
  const int m0 = blockIdx.x * kT, n0 = blockIdx.y * kT;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = m0 + 64 * wa + PA::pos(i, rrow(r, h));
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + 64 * wb + PB::pos(j, lane & 31);
        if (n >= N) continue;
        float* c = C + (long)m * ldc + n;
        *c = ACC ? *c + acc[i][j][r] : acc[i][j][r];
      }
    }
}

// dH[t][d] (+)= sum_v G[t][v] W[v][d] over one chunk: A = G rows, B = the chunk's W rows read k-major.
// dH for one vocab chunk, its contraction (the chunk's columns) split into parts of `per` columns
// (blockIdx.z = part; one part: per >= kcols) so that a small output grid still fills the GPU. With
// one part the tile goes to dH (written by the first chunk, accumulated by the others); with several,
// each part's tile goes to its own fp32 slice part_out[z] and lce32_dh_reduce_kernel sums them in
// part order.
template <int KIND, bool ACC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void lce32_dh_kernel(const float* __restrict__ G, long ldg, const float* __restrict__ W,
                                                       const uint32_t* __restrict__ Wq, const float* __restrict__ Sc,
                                                       const float* __restrict__ Bi, int D, int c0, int kcols, int per,
                                                       int nrows, float* __restrict__ dH) {
  __shared__ __attribute__((aligned(1024))) char s0[kStage0<KIND>];
  __shared__ __attribute__((aligned(1024))) char s1[kStage1<KIND>];
  float* lds = reinterpret_cast<float*>(s0);
  const int m0 = blockIdx.x * kT, n0 = blockIdx.y * kT;
  const int k0 = blockIdx.z * per;
  const int kn = (kcols - k0 < per) ? kcols - k0 : per;
  float* out = dH + (long)blockIdx.z * nrows * D;
  f32x16 acc[2][2];
  if constexpr (KIND == kCopied) {
    gemm128_copied(RowOp(G + (long)m0 * ldg + k0, ldg, nrows - m0, kn), ColOp(W + (long)(c0 + k0) * D + n0, D, D - n0, kn),
                   kn, s0, s1, acc);
    store_tile<ACC, RowOp, ColOp>(acc, nrows, D, out, D);
  } else {
    RowSrc ga{G + (long)m0 * ldg + k0, ldg, nrows - m0, kn, ldg % 4 == 0};
    if constexpr (KIND == kQ4) {
      Q4ColSrc wb{Q4Geom{Wq, Sc, Bi, D}, (long)c0 + k0, D - n0, kn, n0};
      gemm128(ga, wb, kn, lds, acc);
    } else {
      ColSrc wb{W + (long)(c0 + k0) * D + n0, D, D - n0, kn, aligned16(W) && D % 4 == 0};
      gemm128(ga, wb, kn, lds, acc);
    }
    store_tile<ACC>(acc, nrows, D, out, D);
  }
}

// dH (+)= sum over p of parts[p], in part order (deterministic), over the n x d elements.
template <bool ACC>
__global__ __launch_bounds__(256) void lce32_dh_reduce_kernel(const float* __restrict__ parts, int nparts, long count,
                                                              float* __restrict__ dH) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  float x = ACC ? dH[i] : 0.f;
  for (int p = 0; p < nparts; ++p) x += parts[(long)p * count + i];
  dH[i] = x;
}

// dW[v][d] = sum_t G[t][v] H[t][d] for one chunk's vocab rows (all tokens): A = G read k-major
// (k = t), B = H read k-major.
template <int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void lce32_dw_kernel(const float* __restrict__ G, long ldg, const float* __restrict__ H,
                                                       int N, int D, int vrows, float* __restrict__ dW) {
  __shared__ __attribute__((aligned(1024))) char s0[kStage0<KIND>];
  __shared__ __attribute__((aligned(1024))) char s1[kStage1<KIND>];
  const int m0 = blockIdx.x * kT, n0 = blockIdx.y * kT;
  f32x16 acc[2][2];
  if constexpr (KIND == kCopied) {
    gemm128_copied(ColOp(G + m0, ldg, (int)ldg - m0, N), ColOp(H + n0, D, D - n0, N), N, s0, s1, acc);
    store_tile<false, ColOp, ColOp>(acc, vrows, D, dW, D);
  } else {
    ColSrc ga{G + m0, ldg, vrows - m0, N, ldg % 4 == 0};
    ColSrc hb{H + n0, D, D - n0, N, aligned16(H) && D % 4 == 0};
    gemm128(ga, hb, N, reinterpret_cast<float*>(s0), acc);
    store_tile<false>(acc, vrows, D, dW, D);
  }
}

// dK (blockIdx.y 0) or dV (1) = the sum of the nsplit partials in split order. plane: floats, a multiple of 4.
__global__ __launch_bounds__(256) void attn32_dkv_reduce_kernel(const float* __restrict__ part, int nsplit, long plane,
                                                                float* __restrict__ dk, float* __restrict__ dv) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= plane) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int sp = 0; sp < nsplit; ++sp) x += *reinterpret_cast<const f32x4*>(part + (2L * sp + blockIdx.y) * plane + e);
  *reinterpret_cast<f32x4*>((blockIdx.y ? dv : dk) + e) = x;
}

}  // namespace f32k

// ------------------------------------------------------------------------------------------
// Launchers
// ------------------------------------------------------------------------------------------
using namespace f32k;

// Vocab splits of the fp32 forward: about two workgroups per CU.
int lce32_fwd_nsplit(long N, long V) {
  const long rt = (N + kT - 1) / kT, vt = (V + kT - 1) / kT;
  long ns = (2L * kNumCU + rt - 1) / rt;
  if (ns > vt) ns = vt;
  if (ns > 1024) ns = 1024;
  return ns < 1 ? 1 : (int)ns;
}

// The copied-tile core takes dense operands whose rows start at multiples of 16 bytes (the entry points
// check the bases) and whose 128-row tiles stay below the 31-bit offsets of a copy.
static bool copied_tiles(long d, long ld) { return d % 4 == 0 && ld % 4 == 0 && d < (1L << 21) && ld < (1L << 21); }

template <int STAT>
static hipError_t lce32_fwd_tiles(const LceHead32& h, const float* H, int N, int D, int V, const ScoreStats& x, hipStream_t st) {
  const int ns = lce32_fwd_nsplit(N, V);
  auto kernel = h.q4 ? lce32_fwd_kernel<kQ4, STAT> : copied_tiles(D, D) ? lce32_fwd_kernel<kCopied, STAT> : lce32_fwd_kernel<kDense, STAT>;
  hipLaunchKernelGGL(kernel, dim3((N + kT - 1) / kT, ns), dim3(256), 0, st, H, h.w, h.wq, h.sc, h.bi, N, D, V, ns, x.m, x.s,
                     x.scale2, x.u, x.gmax, x.ldg, x.z, x.ldz, x.list);
  return hipGetLastError();
}

hipError_t launch_lce32_stats(const LceHead32& h, const float* H, int N, int D, int V, const ScoreStats& x, hipStream_t st) {
  constexpr int kEntropy = kStatScaled | kStatEntropy, kGroups = kEntropy | kStatGroups;
  if (x.z && x.gmax) return lce32_fwd_tiles<kGroups | kStatKeep>(h, H, N, D, V, x, st);
  if (x.z && x.list.column) return lce32_fwd_tiles<kStatScaled | kStatList | kStatKeep>(h, H, N, D, V, x, st);
  if (x.z) return lce32_fwd_tiles<kEntropy | kStatKeep>(h, H, N, D, V, x, st);
  if (x.gmax && x.list.column) return lce32_fwd_tiles<kGroups | kStatList>(h, H, N, D, V, x, st);
  if (x.gmax) return lce32_fwd_tiles<kGroups>(h, H, N, D, V, x, st);
  if (x.u && x.list.column) return lce32_fwd_tiles<kEntropy | kStatList>(h, H, N, D, V, x, st);
  if (x.u) return lce32_fwd_tiles<kEntropy>(h, H, N, D, V, x, st);
  return lce32_fwd_tiles<kStatScaled | kStatList>(h, H, N, D, V, x, st);
}

hipError_t launch_lce32_gather(const LceHead32& h, const float* H, int D, int V, const GatherPlan& p, hipStream_t st) {
  // The product's core is the forward's, so that a logit is the same number in both.
  auto kernel = h.q4 ? lce32_gather_kernel<kQ4> : copied_tiles(D, D) && D < (1 << 15) ? lce32_gather_kernel<kCopied> : lce32_gather_kernel<kDense>;
  hipLaunchKernelGGL(kernel, dim3(p.max_tiles), dim3(256), 0, st, H, h.w, h.wq, h.sc, h.bi, D, V, p);
  return hipGetLastError();
}

hipError_t launch_lce32_fwd(const LceHead32& h, const float* H, const int64_t* targets, int N, int D, int V,
                            long long ignore_index, float* nll, float* lse, float* tgt, float* ws, hipStream_t st) {
  const int ns = lce32_fwd_nsplit(N, V);
  float* pm = ws;
  float* ps = ws + (long)ns * N;
  ScoreStats stats{};
  stats.m = pm;
  stats.s = ps;
  hipError_t e = lce32_fwd_tiles<0>(h, H, N, D, V, stats, st);
  if (e != hipSuccess) return e;
  const dim3 block(256);
  dim3 fgrid((N + 3) / 4);
  if (h.q4) hipLaunchKernelGGL(lce32_finalize_kernel<1>, fgrid, block, 0, st, H, h.w, h.wq, h.sc, h.bi, targets, N, D, V, ns, pm, ps, ignore_index, nll, lse, tgt);
  else hipLaunchKernelGGL(lce32_finalize_kernel<0>, fgrid, block, 0, st, H, h.w, h.wq, h.sc, h.bi, targets, N, D, V, ns, pm, ps, ignore_index, nll, lse, tgt);
  return hipGetLastError();
}

// Contraction parts of the fp32 dH product of a chunk of kcols columns: about two workgroups per
// CU over the ceil(N/128) x ceil(D/128) output tiles, each part at least 512 columns (32 stages of the
// register-staged core, 16 of the copied one) and a multiple of 16 (the copied core reads zeros past a
// part's end); at most 32. *per receives the columns per part.
int lce32_dh_parts(long N, long D, long kcols, int* per) {
  const long tiles = ((N + kT - 1) / kT) * ((D + kT - 1) / kT);
  long np = (2L * kNumCU + tiles - 1) / tiles;
  if (np > kcols / 512) np = kcols / 512;
  if (np > 32) np = 32;
  if (np < 1) np = 1;
  long pc = (kcols + np - 1) / np;
  pc = (pc + kBK - 1) / kBK * kBK;
  np = (kcols + pc - 1) / pc;
  if (per) *per = (int)(np == 1 ? kcols : pc);
  return (int)np;
}

hipError_t launch_lce32_bwd(const LceHead32& h, const float* H, const int64_t* targets, const float* lse,
                            const float* dnll, int N, int D, int V, long long ignore_index, int chunk, float* dH,
                            float* dW, float* Gbuf, hipStream_t st, const AffineGrad* affine) {
  const long ldg = (long)chunk + 4;
  const bool copied = copied_tiles(D, ldg);
  dim3 block(256);
  for (int c0 = 0; c0 < V; c0 += chunk) {
    const int kc = (V - c0 < chunk) ? V - c0 : chunk;
    dim3 ggrid((N + kT - 1) / kT, (kc + kT - 1) / kT);
    auto gradient = affine ? (h.q4 ? lce32_bwd_g_kernel<kQ4, 1> : copied ? lce32_bwd_g_kernel<kCopied, 1> : lce32_bwd_g_kernel<kDense, 1>)
                           : (h.q4 ? lce32_bwd_g_kernel<kQ4> : copied ? lce32_bwd_g_kernel<kCopied> : lce32_bwd_g_kernel<kDense>);
    if (affine && affine->z) {
      const hipError_t ke = launch_affine_tiles(*affine, lse, N, c0, c0 + kc, (kc + 3) & ~3, ldg, Gbuf, st);
      if (ke != hipSuccess) return ke;
    } else {
      hipLaunchKernelGGL(gradient, ggrid, block, 0, st, H, h.w, h.wq, h.sc, h.bi, targets, lse, dnll, D, V, ignore_index, 0, N,
                         c0, kc, Gbuf, ldg, affine ? affine->rows : AffineRows{});
    }
    if (affine)
      hipLaunchKernelGGL(lce32_bwd_g_columns_kernel, dim3((N + 3) / 4), block, 0, st, affine->columns, affine->value, affine->k,
                         N, c0, kc, Gbuf, ldg);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const bool acc = c0 > 0;
    int per = kc;
    const int np = lce32_dh_parts(N, D, kc, &per);
    dim3 hgrid((N + kT - 1) / kT, (D + kT - 1) / kT, np);
    if (np == 1) {
      if (h.q4) {
        if (acc) hipLaunchKernelGGL((lce32_dh_kernel<kQ4, true>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, dH);
        else hipLaunchKernelGGL((lce32_dh_kernel<kQ4, false>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, dH);
      } else if (copied) {
        if (acc) hipLaunchKernelGGL((lce32_dh_kernel<kCopied, true>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, dH);
        else hipLaunchKernelGGL((lce32_dh_kernel<kCopied, false>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, dH);
      } else {
        if (acc) hipLaunchKernelGGL((lce32_dh_kernel<kDense, true>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, dH);
        else hipLaunchKernelGGL((lce32_dh_kernel<kDense, false>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, dH);
      }
    } else {
      float* parts = Gbuf + (long)N * ldg;   // after the gradient tile: [np][N][D]
      if (h.q4) hipLaunchKernelGGL((lce32_dh_kernel<kQ4, false>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, parts);
      else if (copied) hipLaunchKernelGGL((lce32_dh_kernel<kCopied, false>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, parts);
      else hipLaunchKernelGGL((lce32_dh_kernel<kDense, false>), hgrid, block, 0, st, Gbuf, ldg, h.w, h.wq, h.sc, h.bi, D, c0, kc, per, N, parts);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
      const long count = (long)N * D;
      dim3 rgrid((unsigned)((count + 255) / 256));
      if (acc) hipLaunchKernelGGL(lce32_dh_reduce_kernel<true>, rgrid, block, 0, st, parts, np, count, dH);
      else hipLaunchKernelGGL(lce32_dh_reduce_kernel<false>, rgrid, block, 0, st, parts, np, count, dH);
    }
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (dW) {
      dim3 wgrid((kc + kT - 1) / kT, (D + kT - 1) / kT);
      const float* rows = affine ? static_cast<const float*>(affine->clean) : H;
      if (copied) hipLaunchKernelGGL(lce32_dw_kernel<kCopied>, wgrid, block, 0, st, Gbuf, ldg, rows, N, D, kc, dW + (long)c0 * D);
      else hipLaunchKernelGGL(lce32_dw_kernel<kDense>, wgrid, block, 0, st, Gbuf, ldg, rows, N, D, kc, dW + (long)c0 * D);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

// Splits of each pair of key blocks in the fp32 dK/dV pass. One 8-wave workgroup per CU: the count that
// takes the fewest rounds x items (an item, 32 queries of one head against a pair: about 7 us) plus
// the partials' write and read (28 MB in the time of an item).
int attn32_dkv_splits(int b, int hq, int hkv, int s, int dh) {
  if (b < 1 || hkv < 1 || s < 1 || hq % hkv) return 1;
  const long pairs = ((s + 63) / 64 + 1) / 2, wgs = pairs * b * hkv, items = (long)(hq / hkv) * ((s + kPos - 1) / kPos);
  const long plane = (long)b * hkv * s * dh * 4;
  auto cost = [&](long ns) { return (wgs * ns + kNumCU - 1) / kNumCU * ((items + ns - 1) / ns) * 28000000L + (ns > 1 ? 4 * ns * plane : 0); };
  int best = 1;
  for (int ns = 2; ns <= 16 && ns <= items; ++ns)
    if (cost(ns) < cost(best)) best = ns;
  return best;
}
// D, then, from the next 256-byte boundary, the partials of a split dK/dV pass.
size_t attn32_bwd_workspace(int b, int hq, int hkv, int s, int dh, int ns) {
  return (size_t)b * hq * s * sizeof(float) + (ns > 1 ? 256 + (size_t)ns * 2 * b * hkv * s * dh * sizeof(float) : 0);
}

namespace {
template <int DH>
hipError_t fwd32_dh(const AttnShape& sh, const float* q, const float* k, const float* v, const int32_t* sst, float* o,
                    float* lse, hipStream_t st) {
  const dim3 grid = grid32_q(sh), block(512);
  if (sst) hipLaunchKernelGGL((attn32_q_kernel<DH, kMaskPacked, false>), grid, block, 0, st, q, k, v, nullptr, nullptr, nullptr, nullptr, sst, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, nullptr, 0.f, nullptr, 1, nullptr);
  else hipLaunchKernelGGL((attn32_q_kernel<DH, kMaskPlain, false>), grid, block, 0, st, q, k, v, nullptr, nullptr, nullptr, nullptr, sst, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, nullptr, 0.f, nullptr, 1, nullptr);
  return hipGetLastError();
}
template <int DH>
hipError_t bwd32_dh(const AttnShape& sh, const float* q, const float* k, const float* v, const float* o,
                    const float* lse, const float* d_o, const int32_t* sst, float* dq, float* dk, float* dv,
                    float* dvec, int ns, hipStream_t st) {
  const dim3 qgrid = grid32_q(sh), block(512);
  if (sst) hipLaunchKernelGGL((attn32_q_kernel<DH, kMaskPacked, true>), qgrid, block, 0, st, q, k, v, d_o, o, lse, dvec, sst, dq, nullptr, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, nullptr, 0.f, nullptr, 1, nullptr);
  else hipLaunchKernelGGL((attn32_q_kernel<DH, kMaskPlain, true>), qgrid, block, 0, st, q, k, v, d_o, o, lse, dvec, sst, dq, nullptr, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, nullptr, 0.f, nullptr, 1, nullptr);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  float* part = reinterpret_cast<float*>(((uintptr_t)(dvec + (size_t)sh.b * sh.hq * sh.s) + 255) / 256 * 256);
  const dim3 kgrid(((sh.s + 63) / 64 + 1) / 2 * sh.b * sh.hkv * ns);
  if (sst) hipLaunchKernelGGL((attn32_dkv_kernel<DH, kMaskPacked>), kgrid, block, 0, st, q, k, v, d_o, lse, dvec, sst, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, ns, part, nullptr, 0.f, nullptr);
  else hipLaunchKernelGGL((attn32_dkv_kernel<DH, kMaskPlain>), kgrid, block, 0, st, q, k, v, d_o, lse, dvec, sst, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, ns, part, nullptr, 0.f, nullptr);
  e = hipGetLastError();
  if (e != hipSuccess || ns == 1) return e;
  return launch_attn32_dkv_reduce(part, ns, (long)sh.b * sh.hkv * sh.s * DH, dk, dv, st);
}
}  // namespace

hipError_t launch_attn32_dkv_reduce(const float* part, int ns, long plane, float* dk, float* dv, hipStream_t st) {
  hipLaunchKernelGGL(attn32_dkv_reduce_kernel, dim3((unsigned)((plane / 4 + 255) / 256), 2), dim3(256), 0, st, part, ns, plane, dk, dv);
  return hipGetLastError();
}

hipError_t launch_attn32_fwd(const AttnShape& sh, const float* q, const float* k, const float* v,
                             const int32_t* seg_start, float* o, float* lse, hipStream_t st) {
  switch (sh.dh) {
    case 64: return fwd32_dh<64>(sh, q, k, v, seg_start, o, lse, st);
    case 96: return fwd32_dh<96>(sh, q, k, v, seg_start, o, lse, st);
    case 128: return fwd32_dh<128>(sh, q, k, v, seg_start, o, lse, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_attn32_bwd(const AttnShape& sh, const float* q, const float* k, const float* v, const float* o,
                             const float* lse, const float* d_o, const int32_t* seg_start, float* dq, float* dk,
                             float* dv, float* dvec, int nsplit, hipStream_t st) {
  switch (sh.dh) {
    case 64: return bwd32_dh<64>(sh, q, k, v, o, lse, d_o, seg_start, dq, dk, dv, dvec, nsplit, st);
    case 96: return bwd32_dh<96>(sh, q, k, v, o, lse, d_o, seg_start, dq, dk, dv, dvec, nsplit, st);
    case 128: return bwd32_dh<128>(sh, q, k, v, o, lse, d_o, seg_start, dq, dk, dv, dvec, nsplit, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mtp

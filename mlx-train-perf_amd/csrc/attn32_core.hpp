// The fp32 attention kernels, instantiated by f32_kernels.hip (plain and packed) and attn32_scored.hip (spans, capped
// scores and a bias by distance), and the LDS copies that the fp32 products share with them.
#pragma once
#include "mtp_common.hpp"
#include "mtp_launch.hpp"

namespace mtp {
namespace f32k {

// The waves' copies have landed and their LDS reads are done, for the whole workgroup.
__device__ __forceinline__ void copies_landed() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}
// One global -> LDS copy of a wave: 16 (4) bytes per lane from src + voff (lanes past `bytes` get zeros)
// to dst + 16 lane (4 lane), dst wave-uniform.
__device__ __forceinline__ void lds_copy16(const float* src, int bytes, char* dst, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), (short)0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0, 0);
}
__device__ __forceinline__ void lds_copy4(const float* src, int bytes, char* dst, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), (short)0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 4, voff, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------
// Attention on v_mfma_f32_16x16x4_f32 (lane l: col = l % 16, g = l / 16; it supplies A[col][g] and
// B[g][col] and holds C[4 g + r][col], r < 4). A wave owns 16 positions of one head as the MFMA columns
// (queries: forward and dQ; keys: dK/dV) and keeps their rows and gradients in registers; the 8 waves
// of a workgroup share 32-position tiles of the other side, copied global -> LDS one tile ahead.
//
// The matrix pipe bounds it: a 16x16x4 product takes 32 cycles of its SIMD, so a forward tile is 4096
// MFMA cycles per wave against 32 KiB of LDS reads and ~100 VALU instructions. 32-position waves on
// tiles staged through registers between two barriers left most of it idle: at S = 2048 (16/4 heads,
// head_dim 128, causal) one wave per SIMD waited at the barriers, and the 64 key blocks of dK/dV, of very
// unequal work, were all that 256 CUs had. Hence 16-position waves, which need half the registers, and
// a workgroup of two half-workgroups of 4 waves on two position blocks: under the causal mask the
// mirrored pair (block p and block n - 1 - p), whose work adds up to the same for every pair, with one
// wave of each on every SIMD; otherwise two adjacent blocks, which read the same tiles.
// Measured there: forward 456 -> 177 us, dQ 570 -> 242, dK/dV 2537 -> 322 (4 splits and their sum), 97-109
// TFLOP/s; at S = 8192, 32/8 heads 4.08, 6.19 and 8.13 ms, 133-135 of the 153 TFLOP/s a library fp32
// matrix product reaches.
//
// Row reads (products over head_dim): lane (col, g) reads 16-byte chunks of row col, chunk order
// row_chunk(c, g) -- the contraction may visit head_dim in any order as long as both operands do.
// Column reads (products over the tile's positions): lane (col, g) reads chunk 16 b + col of row
// 4 g + s, one read for four products, whose output rows are head_dims 64 b + 4 i + j (product j, row
// i). Chunk k of row r sits at slot k ^ (r % 16): the 16 lanes of a g, and the lanes 0-7 / 32-39 of a
// read, fall on distinct banks in both.
//
// Masks: key j visible to query i iff j < S, (causal) j <= i, (packed) seg_start[i] <= j; in the
// packed layout (contiguous, ascending, gapless segments) that is "same segment and j <= i". Spans: iff
// start[i] <= j < end[i], neither of which decreases along a row; a query that sees nothing has O = 0 and L = +inf.
// Scores (MOD): cap tanh(x / cap) - slope |i - j| of a scaled product x, tanh by tanhf (an ulp or two: the exponent
// form of the bf16 kernels loses 2^-22 of the cap, more than fp32 results should).
// ------------------------------------------------------------------------------------------
constexpr int kPos = 32;  // positions per LDS tile

__device__ __forceinline__ f32x4 mfma4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <int DH>
struct ALay {
  static constexpr int kRowB = DH == 64 ? 256 : 512;  // 96: chunks 24-31 of a row stay empty (zeros)
  static constexpr int kTile = kPos * kRowB;
  static constexpr int kSlots = kRowB / 16;           // lanes per row of a 1 KiB copy
  static constexpr int kM = kTile / 8192;             // copies per wave and tile
  static constexpr int kC = DH / 16;                  // chunks per lane and row
  static constexpr int kB = DH / 16;                  // 16-row accumulator blocks over head_dim
};

// The per-lane constants of a wave.
template <int DH>
struct ALane {
  using L = ALay<DH>;
  int col, g;
  int rb, rt;            // row-read byte offsets: chunks 0-15 (rb) and, head_dim 96, 16-23 (rt), row `col`
  int cb, ct;            // column-read byte offsets of row 4 g at s = 0
  uint32_t src[L::kM];   // global byte offsets of this lane's copies, from the tile's first row
  __device__ __forceinline__ void init() {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    col = lane & 15;
    g = lane >> 4;
    rb = col * L::kRowB + (((8 * (g >> 1) + (g & 1)) ^ col) << 4);
    rt = col * L::kRowB + (((4 * (g >> 1) + (g & 1)) ^ col) << 4) + 256;
    cb = 4 * g * L::kRowB + ((col ^ (4 * g)) << 4);
    ct = 4 * g * L::kRowB + (((col >> 1) ^ (4 * g)) << 4) + 8 * (col & 1) + 256;
#pragma unroll
    for (int m = 0; m < L::kM; ++m) {
      const int row = (64 / L::kSlots) * (w + 8 * m) + lane / L::kSlots;
      const int c = (lane % L::kSlots) ^ (row & 15);
      src[m] = 16 * c < 4 * DH ? (uint32_t)(row * 4 * DH + 16 * c) : 0x7ffffff0u;  // past the range: zeros
    }
  }
  // Byte offset within a global row of the lane's chunk c.
  __device__ __forceinline__ int row_chunk(int c) const {
    if (DH == 96 && c >= 4) return 16 * (16 + 4 * (g >> 1) + 2 * (c - 4) + (g & 1));
    return 16 * (16 * (c >> 2) + 8 * (g >> 1) + 2 * (c & 3) + (g & 1));
  }
  // Chunk c of tile row 16 half + col.
  __device__ __forceinline__ f32x4 row(const char* tile, int half, int c) const {
    const int off = (DH == 96 && c >= 4) ? (rt ^ ((c - 4) << 5)) : (rb ^ ((c & 3) << 5)) + ((c >> 2) << 8);
    return *reinterpret_cast<const f32x4*>(tile + off + 16 * half * L::kRowB);
  }
  // Four head_dims 64 b + 4 col + j (j < 4) of tile row 16 half + 4 g + s.
  __device__ __forceinline__ f32x4 cols(const char* tile, int half, int s, int b) const {
    return *reinterpret_cast<const f32x4*>(tile + (cb ^ (s << 4)) + (16 * half + s) * L::kRowB + (b << 8));
  }
  // head_dim 96: the last 32, 64 + 2 col + j (j < 2).
  __device__ __forceinline__ f32x2 cols_tail(const char* tile, int half, int s) const {
    return *reinterpret_cast<const f32x2*>(tile + (ct ^ (s << 4)) + (16 * half + s) * L::kRowB);
  }
  // This wave's copies of the 32 rows from position p0 of a [S][DH] matrix (rows past S as zeros;
  // nothing read, zeros written, when not live).
  __device__ __forceinline__ void copy(const float* m, int p0, int S, char* tile, bool live) const {
    const int rows = S - p0 < kPos ? S - p0 : kPos;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < L::kM; ++i)
      lds_copy16(m + (live ? (long)p0 * DH : 0), live ? rows * 4 * DH : 0, tile + 1024 * (w + 8 * i), src[i]);
  }
  // The lane's chunks of a global row as the B operand of the head_dim products.
  __device__ __forceinline__ void load_row(const float* row, bool valid, f32x4 (&x)[L::kC]) const {
#pragma unroll
    for (int c = 0; c < L::kC; ++c) {
      x[c] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (valid) x[c] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(row) + row_chunk(c));
    }
  }
  // acc[half] = tile rows . x (head_dim contraction), the two 16-row chains interleaved.
  __device__ __forceinline__ void dot_rows(const char* tile, const f32x4 (&x)[L::kC], f32x4 (&acc)[2]) const {
    acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < L::kC; ++c) {
      const f32x4 a = row(tile, 0, c), b = row(tile, 1, c);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        acc[0] = mfma4(a[s], x[c][s], acc[0]);
        acc[1] = mfma4(b[s], x[c][s], acc[1]);
      }
    }
  }
  // out += tile^T . p over the tile's 32 rows, p[half][r] the weight of row 16 half + 4 g + r.
  __device__ __forceinline__ void dot_cols(const char* tile, const f32x4 (&p)[2], f32x4 (&out)[L::kB]) const {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int b = 0; b < DH / 64; ++b) {
          const f32x4 a = cols(tile, half, s, b);
#pragma unroll
          for (int j = 0; j < 4; ++j) out[4 * b + j] = mfma4(a[j], p[half][s], out[4 * b + j]);
        }
        if constexpr (DH == 96) {
          const f32x2 a = cols_tail(tile, half, s);
          out[4] = mfma4(a[0], p[half][s], out[4]);
          out[5] = mfma4(a[1], p[half][s], out[5]);
        }
      }
  }
  // Writes acc (head_dim x this lane's position) * mul to the position's global row.
  __device__ __forceinline__ void store_row(float* row, const f32x4 (&acc)[L::kB], float mul) const {
#pragma unroll
    for (int b = 0; b < DH / 64; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(row + 64 * b + 16 * g + 4 * r) =
            f32x4{acc[4 * b][r] * mul, acc[4 * b + 1][r] * mul, acc[4 * b + 2][r] * mul, acc[4 * b + 3][r] * mul};
    if constexpr (DH == 96) {
#pragma unroll
      for (int r = 0; r < 4; r += 2)
        *reinterpret_cast<f32x4*>(row + 64 + 8 * g + 2 * r) =
            f32x4{acc[4][r] * mul, acc[5][r] * mul, acc[4][r + 1] * mul, acc[5][r + 1] * mul};
    }
  }
};
// Scores in the log2 domain: raw(s) is tanh(x / cap) with a cap, else scale2 s; of(v, d, top) the score at distance |d|, its
// bias counted from the highest of the row, that of the key at distance top (top_distance, as in the bf16 kernels).
template <int MOD>
struct Score32 {
  static constexpr bool kCap = MOD & kModCap;
  float scale2, in, cap2, slope2;
  __device__ __forceinline__ float raw(float s) const { return kCap ? tanhf(s * in) : s * scale2; }
  __device__ __forceinline__ float of(float v, float d, float top) const {
    const float y = kCap ? v * cap2 : v;
    return (MOD & kModSlope) ? __builtin_fmaf(-slope2, __builtin_fabsf(d) - top, y) : y;
  }
};
template <int MOD>
__device__ __forceinline__ Score32<MOD> make_score32(float scale, float cap) {
  return Score32<MOD>{scale * kLog2e, (MOD & kModCap) ? scale / cap : 0.f, cap * kLog2e, 0.f};
}
// 2^y of a probability formed again from L: at most 1, where the rounding of y, a difference of two numbers of the scores'
// size, may be far above 0 for scores past 2^29. NaN stays.
__device__ __forceinline__ float prob32(float y) { return fast_exp2(__builtin_elementwise_minimum(y, 0.f)); }
// Sum and maximum over the four lanes (g = 0..3) of a column.
__device__ __forceinline__ float col_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ float col_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
// The two position blocks of pair p out of n: mirrored (the causal mask: equal work per pair) or
// adjacent. The second may be n (none).
__host__ __device__ __forceinline__ void pair_blocks(int p, int n, bool mirror, int& a, int& b) {
  a = mirror ? p : 2 * p;
  b = mirror ? n - 1 - p : 2 * p + 1;
  if (b <= a) b = n;
}
__host__ __device__ __forceinline__ int q_heads32(int G) { return G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1; }

inline dim3 grid32_q(const AttnShape& sh) {
  const int hpw = q_heads32(sh.hq / sh.hkv), R = 16 * (4 / hpw);
  return dim3(((sh.s + R - 1) / R + 1) / 2 * sh.b * (sh.hq / hpw));
}

// Forward (DQ = false) and dQ (DQ = true). A half-workgroup holds q_heads32(G) heads of one GQA group x
// 16 (4 / heads) queries: every K/V tile feeds all of them.
template <int DH, int MASK, bool DQ, int MOD = kModNone>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(DQ ? 2 : 4)))
void attn32_q_kernel(const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v,
                     const float* __restrict__ d_o, const float* __restrict__ o_in, const float* __restrict__ lse_in,
                     float* __restrict__ dvec, const int32_t* __restrict__ seg_start, float* __restrict__ out,
                     float* __restrict__ lse_out, int B, int Hq, int Hkv, int S, float scale, int causal,
                     const int32_t* __restrict__ span_end, float cap, const float* __restrict__ slopes, int nsplit,
                     float* __restrict__ part) {
  // seg_start: the first key that each query sees (packed: its segment's start; span: its span's).
  // Scored calls of few workgroups are split (q_splits, attn32_scored.hip): workgroup `split` of a pair of blocks takes every
  // nsplit-th key tile from tile `split` on, and writes its dQ, or its unnormalized O, maximum and sum, to
  // part[split] ([b][hq][s][dh], the forward's maxima and sums [split][b][hq][s][2] behind all of them).
  constexpr bool PACKED = MASK != kMaskPlain, SPAN = MASK == kMaskSpan, CAP = MOD & kModCap;
  constexpr bool SPLIT = SPAN || MOD != kModNone;
  using L = ALay<DH>;
  __shared__ __attribute__((aligned(1024))) char lds0[2 * L::kTile];  // K, V
  __shared__ __attribute__((aligned(1024))) char lds1[2 * L::kTile];
  const int G = Hq / Hkv, hpw = q_heads32(G), R = 16 * (4 / hpw);
  const int nqb = (S + R - 1) / R, hgb = Hq / hpw, nhg = B * hgb;
  const int ns = SPLIT ? nsplit : 1, split = SPLIT ? blockIdx.x % ns : 0;
  const unsigned wg = SPLIT ? blockIdx.x / ns : blockIdx.x;
  const int hg = wg % nhg, b = hg / hgb, h0 = (hg % hgb) * hpw, kvh = h0 / G;
  int pa, pb;
  pair_blocks((int)(wg / nhg), nqb, causal && !PACKED, pa, pb);
  ALane<DH> ln;
  ln.init();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), u = w & 3;
  const int blk = w < 4 ? pa : pb;
  const int head = h0 + u % hpw, qw0 = blk * R + 16 * (u / hpw), qi = qw0 + ln.col;
  const bool wave_has = blk < nqb && qw0 < S, qvalid = wave_has && qi < S;
  const int wq_last = qw0 + 15 < S ? qw0 + 15 : S - 1;
  const long qrow = (long)(b * Hq + head) * S;
  const float* kh = k + (long)(b * Hkv + kvh) * S * DH;
  const float* vh = v + (long)(b * Hkv + kvh) * S * DH;
  const int32_t* sst = PACKED ? seg_start + (long)b * S : nullptr;
  const float scale_log2 = scale * kLog2e;
  const int32_t* snd = SPAN ? span_end + (long)b * S : nullptr;
  auto in_row = [&](int x) { return x < 0 ? 0 : x < S ? x : S; };  // spans, in range whatever they hold
  Score32<MOD> score = make_score32<MOD>(scale, cap);
  if ((MOD & kModSlope) && slopes) score.slope2 = slopes[head] * kLog2e;

  f32x4 qx[L::kC], dx[DQ ? L::kC : 1];
  ln.load_row(q + (qrow + qi) * DH, qvalid, qx);
  float l2q = 0.f, dq_row = 0.f;
  if constexpr (DQ) {
    ln.load_row(d_o + (qrow + qi) * DH, qvalid, dx);
    f32x4 ox[L::kC];
    ln.load_row(o_in + (qrow + qi) * DH, qvalid, ox);
    float dp = 0.f;
#pragma unroll
    for (int c = 0; c < L::kC; ++c)
#pragma unroll
      for (int s = 0; s < 4; ++s) dp = __builtin_fmaf(dx[c][s], ox[c][s], dp);
    dq_row = col_sum(dp);
    if (qvalid && ln.g == 0 && split == 0) dvec[qrow + qi] = dq_row;
    l2q = qvalid ? lse_in[qrow + qi] * kLog2e : 0.f;
  }
  // Keys of the workgroup: those of its last block (the latest queries) and, packed, from its first
  // block's first segment on (adjacent blocks: one contiguous range).
  const int last = pb < nqb ? pb : pa;
  const int kv_end = SPAN ? in_row(snd[((last + 1) * R < S ? (last + 1) * R : S) - 1])
                          : (causal && (last + 1) * R < S) ? (last + 1) * R : S;
  const int kv_begin = SPAN ? (in_row(sst[pa * R]) / kPos) * kPos : PACKED ? (sst[pa * R] / kPos) * kPos : 0;
  const int ntiles = (SPAN && kv_end <= kv_begin) ? 0 : (kv_end - kv_begin + kPos - 1) / kPos;
  // Span: the end of this lane's, and the smallest and largest of the wave's (its first and last query's).
  const int my_end = (SPAN && qvalid) ? in_row(snd[qi]) : 0;
  const int w_end_first = (SPAN && wave_has) ? in_row(__builtin_amdgcn_readfirstlane(snd[qw0])) : 0;
  const int w_end_last = (SPAN && wave_has) ? in_row(__builtin_amdgcn_readfirstlane(snd[wq_last])) : 0;
  const int my_sst = (PACKED && qvalid) ? sst[qi] : 0;
  const int w_sst_first = (PACKED && wave_has) ? __builtin_amdgcn_readfirstlane(sst[qw0]) : 0;
  const int w_sst_last = (PACKED && wave_has) ? __builtin_amdgcn_readfirstlane(sst[wq_last]) : 0;

  float m = kNegInf, l = 0.f;
  f32x4 acc[L::kB];
#pragma unroll
  for (int i = 0; i < L::kB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  ln.copy(kh, kv_begin + split * kPos, S, lds0, ntiles > split);  // no tile (a segment start past the queries): nothing read
  ln.copy(vh, kv_begin + split * kPos, S, lds0 + L::kTile, ntiles > split);
  copies_landed();
  // The row loads are complete here: tell the compiler, which would wait for them (and for the copies
  // in flight) at their first use.
#pragma unroll
  for (int c = 0; c < L::kC; ++c) {
    asm volatile("" : "+v"(qx[c]));
    if constexpr (DQ) asm volatile("" : "+v"(dx[c]));
  }

  auto body = [&](int t, const char* cur, char* nxt) __attribute__((always_inline)) {
    const int kv0 = kv_begin + t * kPos;
    ln.copy(kh, kv0 + ns * kPos, S, nxt, t + ns < ntiles);
    ln.copy(vh, kv0 + ns * kPos, S, nxt + L::kTile, t + ns < ntiles);
    if (wave_has && !(causal && kv0 > wq_last) && !(PACKED && kv0 + kPos - 1 < w_sst_first) && !(SPAN && kv0 >= w_end_last)) {
      f32x4 sc[2];
      ln.dot_rows(cur, qx, sc);  // S^T = K Q^T
      // Only tiles across the wave's diagonal, the sequence end or a segment start hold hidden pairs.
      const bool need_mask = (causal && kv0 + kPos - 1 > qw0) || kv0 + kPos > S || (PACKED && kv0 < w_sst_last) ||
                             (SPAN && kv0 + kPos > w_end_first);
      const int hi = (SPAN ? my_end - 1 : causal ? (qi < S - 1 ? qi : S - 1) : S - 1) - kv0 - 4 * ln.g;
      const int lo = my_sst - kv0 - 4 * ln.g;
      float rel = 0.f, top = 0.f;
      if constexpr (MOD & kModSlope) {
        int lane = threadIdx.x;
        asm volatile("" : "+v"(lane));  // formed in each tile: the registers are full
        const int i = qw0 + (lane & 15);
        rel = (float)(i - kv0 - 4 * ((lane >> 4) & 3));
        top = top_distance(score.slope2, i, SPAN ? in_row(my_sst) : 0, SPAN ? my_end : causal ? i + 1 : S);
      }
      auto visible = [&](int half, int r) { return 16 * half + r <= hi && (!PACKED || 16 * half + r >= lo); };
      if constexpr (DQ) {
        f32x4 dp[2];
        ln.dot_rows(cur + L::kTile, dx, dp);  // dP^T = V dO^T
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (MOD == kModNone) {
              const float y = __builtin_fmaf(sc[half][r], scale_log2, -l2q);
              sc[half][r] = SPAN ? prob32(y) : fast_exp2(y);
            } else {
              const float v = score.raw(sc[half][r]);
              sc[half][r] = prob32(score.of(v, rel - (float)(16 * half + r), top) - l2q);
              if constexpr (CAP) {  // P (1 - tanh^2): dP, D and the mask come after
                sc[half][r] *= 1.f - v * v;
              }
            }
          }
        if (need_mask) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[half][r] = visible(half, r) ? sc[half][r] : 0.f;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[half][r] *= dp[half][r] - dq_row;
        ln.dot_cols(cur, sc, acc);  // dQ^T += K^T dS^T
      } else {
        float mx = kNegInf;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (MOD == kModNone) sc[half][r] *= scale_log2;
            else sc[half][r] = score.of(score.raw(sc[half][r]), rel - (float)(16 * half + r), top);
          }
        if (need_mask) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[half][r] = visible(half, r) ? sc[half][r] : kNegInf;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fmaxf(sc[0][r], sc[1][r]));
        const float mn = fmaxf(m, col_max(mx));
        const float base = (mn == kNegInf) ? 0.f : mn;
        // O and l are rescaled when some query's maximum rose; alpha is 1 for the others.
        if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
          const float alpha = fast_exp2(m - base);  // m = -inf: 0 (O and l are 0)
          l *= alpha;
#pragma unroll
          for (int i = 0; i < L::kB; ++i) acc[i] *= alpha;
          m = mn;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sc[half][r] = fast_exp2(sc[half][r] - base);
            l += sc[half][r];
          }
        ln.dot_cols(cur + L::kTile, sc, acc);  // O^T += V^T P^T
      }
    }
    copies_landed();
  };
  for (int t = split; t < ntiles; t += 2 * ns) {
    body(t, lds0, lds1);
    if (t + ns < ntiles) body(t + ns, lds1, lds0);
  }
  const long rows = (long)B * Hq * S;
  if constexpr (DQ) {
    if (SPLIT && ns > 1) out = part + split * rows * DH;
    if (qvalid) ln.store_row(out + (qrow + qi) * DH, acc, scale);
  } else {
    const float lt = col_sum(l);
    if (!qvalid) return;
    if (SPLIT && ns > 1) {
      if (ln.g == 0) *reinterpret_cast<f32x2*>(part + ns * rows * DH + 2 * (split * rows + qrow + qi)) = f32x2{m, lt};
      ln.store_row(part + (split * rows + qrow + qi) * DH, acc, 1.f);
      asm volatile("s_nop 0");  // (below)
      return;
    }
    // A query that sees nothing: +inf with spans, so that the backward's exp(S - L) is 0.
    if (ln.g == 0) lse_out[qrow + qi] = (lt > 0.f) ? (m + fast_log2(lt)) * kLn2 : SPAN ? -kNegInf : kNegInf;
    ln.store_row(out + (qrow + qi) * DH, acc, lt > 0.f ? 1.f / lt : 0.f);
  }
  // The padding behind a program's end reads as a write of v0, which the listing check of stores whose data the next
  // instructions write would hold against a last store of v0.
  if constexpr (SPLIT) asm volatile("s_nop 0");
}

// dK, dV: a half-workgroup holds a block of 64 keys of one kv head, each wave 16 of them with their K
// and V rows; items (query head h of the group, 32-query tile t) visit the queries that see the pair of
// blocks. They are dealt to nsplit workgroups, item (h, t) to (h + t) % nsplit (attn32_dkv_splits), so
// that a key's partial sums do not depend on the block it is paired with (one packed segment gives the
// causal result bit for bit); with several, each writes an fp32 partial
// part[split][dK | dV][b][kv head][key][d], which attn32_dkv_reduce_kernel sums in split order.
template <int DH, int MASK, int MOD = kModNone>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void attn32_dkv_kernel(const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v,
                       const float* __restrict__ d_o, const float* __restrict__ lse, const float* __restrict__ dvec,
                       const int32_t* __restrict__ seg_start, float* __restrict__ dk, float* __restrict__ dv, int B,
                       int Hq, int Hkv, int S, float scale, int causal, int nsplit, float* __restrict__ part,
                       const int32_t* __restrict__ span_end, float cap, const float* __restrict__ slopes) {
  constexpr bool PACKED = MASK != kMaskPlain, SPAN = MASK == kMaskSpan, CAP = MOD & kModCap;
  using L = ALay<DH>;
  __shared__ __attribute__((aligned(1024))) char lds0[2 * L::kTile + 512];  // Q, dO, L (32 of 64), D (32 of 64)
  __shared__ __attribute__((aligned(1024))) char lds1[2 * L::kTile + 512];
  const int G = Hq / Hkv, nkb = (S + 63) / 64, nbh = B * Hkv;
  const int split = blockIdx.x % nsplit, bh = (blockIdx.x / nsplit) % nbh, b = bh / Hkv, kvh = bh % Hkv;
  int ba, bb;
  pair_blocks((int)(blockIdx.x / nsplit / nbh), nkb, causal && !PACKED, ba, bb);
  ALane<DH> ln;
  ln.init();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blk = w < 4 ? ba : bb, kw0 = blk * 64 + 16 * (w & 3), kj = kw0 + ln.col;
  const bool wave_has = blk < nkb && kw0 < S, kvalid = wave_has && kj < S;
  const long krow = (long)bh * S;
  const float scale_log2 = scale * kLog2e;
  const int32_t* sst = PACKED ? seg_start + (long)b * S : nullptr;
  const int32_t* send = SPAN ? span_end + (long)b * S : nullptr;
  auto in_row = [&](int x) { return x < 0 ? 0 : x < S ? x : S; };

  f32x4 kx[L::kC], vx[L::kC];
  ln.load_row(k + (krow + kj) * DH, kvalid, kx);
  ln.load_row(v + (krow + kj) * DH, kvalid, vx);
  // Query tiles [t0, t1) see the workgroup's keys; queries my_beg <= q < my_lim see key kj (packed: those of its
  // segment; spans: as start and end do not decrease, those from the first whose span ends past kj to the first
  // whose span starts past it), and the wave's keys none before w_beg or from w_end on.
  Score32<MOD> score = make_score32<MOD>(scale, cap);
  int t0 = causal ? ba * (64 / kPos) : 0;
  int t1 = (S + kPos - 1) / kPos, my_lim = S, w_lim = S, w_end = S;
  int my_beg = 0, w_beg = 0, w_beg_last = 0;
  auto first_over = [&](const int32_t* a, int lo, int x) {  // the first position from lo on with a[i] > x
    int hi = S;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a[mid] > x) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };
  if (SPAN) {
    t0 = __builtin_amdgcn_readfirstlane(first_over(send, 0, ba * 64)) / kPos;
    if (wave_has) {
      my_beg = kvalid ? first_over(send, 0, kj) : S;
      w_beg = __builtin_amdgcn_readfirstlane(my_beg);
      w_beg_last = __builtin_amdgcn_readfirstlane(first_over(send, 0, kw0 + 15 < S ? kw0 + 15 : S - 1));
    }
  }
  if (PACKED) {
    auto above = [&](int x) { return first_over(sst, SPAN ? 0 : x, x); };  // packed: the end of position x's segment
    const int last = bb < nkb ? bb : ba, wl = kw0 + 15 < S ? kw0 + 15 : S - 1;
    t1 = (__builtin_amdgcn_readfirstlane(above(last * 64 + 63 < S ? last * 64 + 63 : S - 1)) + kPos - 1) / kPos;
    if (kvalid) my_lim = above(kj);
    w_lim = __builtin_amdgcn_readfirstlane(my_lim);  // the first key's: the smallest
    if (wave_has) w_end = __builtin_amdgcn_readfirstlane(above(wl));
  }
  struct Item {
    int h, t;
  };
  auto settle = [&](Item x) __attribute__((always_inline)) {  // the first item of this split from x on (h = G: none)
    while (x.h < G && x.t >= t1) {
      ++x.h;
      int r = (split - x.h - t0) % nsplit;
      if (r < 0) r += nsplit;
      x.t = t0 + r;
    }
    return x;
  };

  f32x4 dka[L::kB], dva[L::kB];
#pragma unroll
  for (int i = 0; i < L::kB; ++i) dka[i] = dva[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Copies of an item into a stage: Q and dO rows, L and D (waves 0 and 1, 32 floats each).
  auto copy = [&](Item x, char* st) __attribute__((always_inline)) {
    const bool live = x.h < G;
    const int q0 = x.t * kPos;
    const long qrow = (long)(b * Hq + kvh * G + (live ? x.h : 0)) * S;
    ln.copy(q + qrow * DH, q0, S, st, live);
    ln.copy(d_o + qrow * DH, q0, S, st + L::kTile, live);
    if (w < 2) {
      const int rows = S - q0 < kPos ? S - q0 : kPos;
      lds_copy4((w ? dvec : lse) + qrow + (live ? q0 : 0), live ? rows * 4 : 0, st + 2 * L::kTile + 256 * w,
                  4u * (threadIdx.x & 63));
    }
  };
  auto body = [&](Item x, Item next, const char* cur, char* nxt) __attribute__((always_inline)) {
    copy(next, nxt);
    const int q0 = x.t * kPos;
    if (wave_has && !(causal && q0 + kPos - 1 < kw0) && !(PACKED && q0 >= w_end) && !(SPAN && q0 + kPos - 1 < w_beg)) {
      if ((MOD & kModSlope) && slopes) score.slope2 = slopes[kvh * G + x.h] * kLog2e;
      // The tops of the tile's queries: each formed in a lane, ahead of the products. Without spans 0 for slopes from 0 on.
      f32x4 top[2] = {};
      if constexpr (MOD & kModSlope)
        if (SPAN || score.slope2 < 0.f) {
          const int qi = q0 + (int)(threadIdx.x & 31), at = qi < S ? qi : S - 1;
          const float mine = top_distance(score.slope2, qi, SPAN ? in_row(sst[at]) : 0, SPAN ? in_row(send[at]) : causal ? qi + 1 : S);
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int r = 0; r < 4; ++r) top[half][r] = __shfl(mine, 16 * half + 4 * ln.g + r, 64);
        }
      f32x4 p[2], ds[2];
      ln.dot_rows(cur, kx, p);              // S = Q K^T (queries x this lane's key)
      ln.dot_rows(cur + L::kTile, vx, ds);  // dP = dO V^T
      const float* sl = reinterpret_cast<const float*>(cur + 2 * L::kTile);
      const bool need_mask = (causal && q0 < kw0 + 15) || q0 + kPos > S || (PACKED && q0 + kPos > w_lim) || (SPAN && q0 < w_beg_last);
      const int lo = SPAN ? my_beg - q0 - 4 * ln.g : causal ? kj - q0 - 4 * ln.g : -kPos, hi = my_lim - q0 - 4 * ln.g;
      const float rel = (float)(kj - q0 - 4 * ln.g);
      f32x4 bend[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(sl + 16 * half + 4 * ln.g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (MOD == kModNone) {
            const float y = __builtin_fmaf(p[half][r], scale_log2, -l4[r] * kLog2e);
            p[half][r] = SPAN ? prob32(y) : fast_exp2(y);
          } else {
            const float v = score.raw(p[half][r]);
            if constexpr (CAP) bend[half][r] = 1.f - v * v;
            p[half][r] = prob32(score.of(v, rel - (float)(16 * half + r), top[half][r]) - l4[r] * kLog2e);
          }
        }
      }
      if (need_mask) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool ok = 16 * half + r >= lo && 16 * half + r < hi;
            p[half][r] = ok ? p[half][r] : 0.f;
            if constexpr (CAP) bend[half][r] = ok ? bend[half][r] : 0.f;  // a hidden score may be NaN
          }
      }
      ln.dot_cols(cur + L::kTile, p, dva);  // dV^T += dO^T P
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(sl + 64 + 16 * half + 4 * ln.g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ds[half][r] = p[half][r] * (ds[half][r] - d4[r]);
          if constexpr (CAP) ds[half][r] *= bend[half][r];
        }
      }
      ln.dot_cols(cur, ds, dka);  // dK^T += Q^T dS
    }
    copies_landed();
  };
  Item x = settle(Item{-1, t1});
  if (x.h < G) {
    copy(x, lds0);
    copies_landed();
#pragma unroll
    for (int c = 0; c < L::kC; ++c) asm volatile("" : "+v"(kx[c]), "+v"(vx[c]));
    while (true) {
      const Item y = settle(Item{x.h, x.t + nsplit});
      body(x, y, lds0, lds1);
      if (y.h >= G) break;
      x = settle(Item{y.h, y.t + nsplit});
      body(y, x, lds1, lds0);
      if (x.h >= G) break;
    }
  }
  if (!kvalid) return;
  const long plane = (long)nbh * S * DH;
  if (nsplit > 1) {
    dk = part + 2L * split * plane;
    dv = dk + plane;
  }
  ln.store_row(dk + (krow + kj) * DH, dka, scale);
  ln.store_row(dv + (krow + kj) * DH, dva, 1.f);
}

}  // namespace f32k
}  // namespace mtp

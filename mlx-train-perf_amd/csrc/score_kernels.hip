// Token scoring and distillation over a language-model head (gfx950): what a forward keeps of the logits z = H W^T beside or
// in the place of a target's loss. With x = z / temperature, lse = log sum_v e^x_v and p = e^(x - lse):
//
//   scoring (logprobs): log p_y, the entropy lse - sum p x, the `top` largest logits of a token and their log p;
//   distillation: the divergence of a teacher's list of outcomes (t_k, and the rest as one outcome) from p.
//
// The product is the loss's (lce_fwd_kernel, lce32_fwd_kernel): it leaves a maximum and sums per vocab split and, for the
// alternatives, the maximum of every group of kGroup consecutive logits. The `top` largest logits of a row lie in the
// groups with the `top` largest maxima (a logit outside them has `top` at least as large ahead of it; equal maxima go to the
// lower group, so equal logits to the lower index). So: choose those groups, form their logits again (a product over
// the tokens that want each group: top kGroup / V of the first one, 0.7% for 8 of 151936, in its k order and to its bits),
// choose among them. The logits of a teacher's list, sorted first, the product's tiles put away as they pass (ListCursor) and
// leave out of their sums, so that what a list leaves of 1 is a sum of its own. As a difference of 1 and the list's own
// probabilities it was off by their last digits: 5% of 1.5e-5 at logits of 44.
//
// Up to kFewTokens tokens (kFewTokens32) the logits themselves are kept in the workspace (lce_few_kernel), which leaves two launches;
// where there are not many of them (keep_logits), the product's tiles keep them too.
#include <math.h>

#include <type_traits>

#include "score_gather.hpp"

namespace mtp {
namespace {

// ------------------------------------------------------------------------------------------
// Choice of the K largest keys.
// ------------------------------------------------------------------------------------------
constexpr int kPick = 256;  // threads

// fp32 as an unsigned number of the same order; -0 as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

constexpr int kRanked = 512;  // keys that are ordered by counting
struct PickScratch {
  int4 count[2][kPick / 64];
  int sum[kPick / 64], listed;
  uint32_t least, top[kPick];
  uint64_t list[kRanked];  // keys and their positions, as one number that falls in the order of choice
  int rank[kRanked];
};
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int at) { return (uint64_t)key << 32 | (uint32_t)~at; }
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ int entry_at(uint64_t e) { return (int)~(uint32_t)e; }

// Sum over the threads before this one.
__device__ __forceinline__ int block_before(int mine, PickScratch& s) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int run = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(run, o, 64);
    if (lane >= o) run += up;
  }
  __syncthreads();
  if (lane == 63) s.sum[w] = run;
  __syncthreads();
  int before = run - mine;
  for (int i = 0; i < w; ++i) before += s.sum[i];
  return before;
}

// The K-th largest of M >= K keys, key i at thread i % kPick, register i / kPick (0 past the end: below every number's). Found two
// bits a step, three counts over the keys, so the time does not depend on their order. `above`: how many are larger.
template <int R>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[R], int K, int& above, PickScratch& s) {
  uint32_t least = 0;
  above = 0;
  for (int b = 30; b >= 0; b -= 2) {
    int n1 = 0, n2 = 0, n3 = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      n1 += __popcll(__ballot(key[r] >= (least | 1u << b)));
      n2 += __popcll(__ballot(key[r] >= (least | 2u << b)));
      n3 += __popcll(__ballot(key[r] >= (least | 3u << b)));
    }
    const int w = threadIdx.x >> 6, step = (b >> 1) & 1;
    if ((threadIdx.x & 63) == 0) s.count[step][w] = int4{n1, n2, n3, 0};
    __syncthreads();
    n1 = n2 = n3 = 0;
#pragma unroll
    for (int i = 0; i < kPick / 64; ++i) {
      n1 += s.count[step][i].x;
      n2 += s.count[step][i].y;
      n3 += s.count[step][i].z;
    }
    if (n3 >= K) {
      least |= 3u << b;
    } else if (n2 >= K) {
      least |= 2u << b;
      above = n3;
    } else if (n1 >= K) {
      least |= 1u << b;
      above = n2;
    } else {
      above = n1;
    }
  }
  return least;
}

// The K largest of M >= K keys in LDS, their positions ascending: put(place, position). Equal keys go to the lower position. Ends with
// a barrier. R: at least M / kPick. Returns the K-th largest.
template <int R, class PUT>
__device__ __forceinline__ uint32_t pick_largest(const uint32_t* key, int M, int K, const PUT& put, PickScratch& s) {
  const int tid = threadIdx.x;
  uint32_t mine_keys[R];
#pragma unroll
  for (int r = 0; r < R; ++r) mine_keys[r] = r * kPick + tid < M ? key[r * kPick + tid] : 0u;
  int above;
  const uint32_t least = kth_largest<R>(mine_keys, K, above, s);
  const int equal = K - above;  // how many of the keys that equal the K-th are taken
  const int per = (M + kPick - 1) / kPick, lo = tid * per < M ? tid * per : M, hi = lo + per < M ? lo + per : M;
  int mine = 0;
  for (int i = lo; i < hi; ++i) mine += key[i] == least;
  int seen = block_before(mine, s);
  int taken = 0, rank = seen;
  for (int i = lo; i < hi; ++i) {
    if (key[i] > least) ++taken;
    else if (key[i] == least) taken += rank++ < equal;
  }
  int to = block_before(taken, s);
  for (int i = lo; i < hi; ++i)
    if (key[i] > least || (key[i] == least && seen++ < equal)) put(to++, i);
  __syncthreads();
  return least;
}

// The positions of the keys that are at least `least` to s.list, in no order; how many of them (beyond kRanked: not all listed).
__device__ __forceinline__ int list_from(const uint32_t* key, int M, uint32_t least, PickScratch& s) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  for (int base = 0; base < M; base += kPick) {
    const int i = base + threadIdx.x;
    const bool in = i < M && key[i] >= least;
    const uint64_t who = __ballot(in);
    int first = 0;
    if (lane == 0 && who) first = atomicAdd(&s.listed, __popcll(who));
    first = __builtin_amdgcn_readfirstlane(first) + __popcll(who & ((1ull << lane) - 1));
    if (in && first < kRanked) s.list[first] = entry_of(key[i], i);
  }
  __syncthreads();
  return s.listed;
}
// How many of the n listed come before `mine`.
__device__ __forceinline__ int rank_of(uint64_t mine, int n, const PickScratch& s) {
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) rank += s.list[j] > mine;
  return rank;
}

// pick_largest for keys that mostly differ. The K-th largest of the 256 threads' own maxima is at most the K-th largest key, and
// mostly few more than K keys reach it (every wave finds it by itself, from four of them a lane: no barriers); those are put in
// order by counting. 1187 keys, 8 of them: 8192 rows 95 us with 16 counts over all keys, then 61, and 51 with
// a key and its position as one number to compare.
template <int R>
__device__ __forceinline__ uint32_t pick_few(const uint32_t* key, int M, int K, int* at, PickScratch& s) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t mine = 0;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (r * kPick + tid < M) mine = key[r * kPick + tid] > mine ? key[r * kPick + tid] : mine;
  s.top[tid] = mine;
  __syncthreads();
  uint32_t v[kPick / 64], least = 0;
#pragma unroll
  for (int i = 0; i < kPick / 64; ++i) v[i] = s.top[lane + 64 * i];
  for (int b = 31; b >= 0; --b) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPick / 64; ++i) n += __popcll(__ballot(v[i] >= (least | 1u << b)));
    if (n >= K) least |= 1u << b;
  }
  const int n = list_from(key, M, least, s);
  if (n > kRanked) return pick_largest<R>(key, M, K, [&](int place, int i) { at[place] = i; }, s);
  for (int i = tid; i < n; i += kPick) s.rank[i] = rank_of(s.list[i], n, s);
  __syncthreads();
  for (int i = tid; i < n; i += kPick) {
    if (s.rank[i] >= K) continue;
    const int p = entry_at(s.list[i]);
    if (s.rank[i] == K - 1) s.least = entry_key(s.list[i]);
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) place += s.rank[j] < K && entry_at(s.list[j]) < p;
    at[place] = p;
  }
  __syncthreads();
  return s.least;
}

// ------------------------------------------------------------------------------------------
// Few tokens: the logits [N][ldz] in fp32, and per group of kGroup of them their maximum and, relative to
// it, the two sums. The head is read once and bounds it; a workgroup takes one group: 4 waves of 32 vocab rows, the rows'
// fragments straight from memory to registers, each loaded for the next slab as soon as its product has gone out (a whole slab in
// flight a wave, 8 KiB of a dense head, 4 of a 4-bit one), the tokens' slab (NB blocks of 32) through LDS, one barrier a
// slab. The registers and, up to 16 tokens, the LDS leave room for 5 workgroups a CU: all 1187 groups of 151936 run at once
// (16 tokens over a 4-bit head, 4 workgroups and 5: 157 and 130 us). 4096 x 151936: a dense head's 1.24 GB in 242 us (5.1 TB/s, as
// a library product of one row), a 4-bit head's 0.35 GB in 108, where the vector units are busy for some 60.
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes > 0x7fffffffL ? 0x7fffffff : (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(const __amdgpu_buffer_rsrc_t r, uint32_t voff, int soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}
// LDS written before is seen behind it by the workgroup; loads into registers stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// T: the hidden states' type, and a dense head's and the scales' too (fp32: v_mfma_f32_32x32x2_f32, a lane's 4 values a step
// of 8 k). ROWS: of the tokens' slab (16: the products' upper 16 columns repeat the lower).
template <class T, int Q4, int NB, int ROWS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NB == 1 ? 5 : NB == 2 ? 4 : 2)))
void lce_few_kernel(const T* __restrict__ H, const T* __restrict__ W, const uint32_t* __restrict__ Wq, const T* __restrict__ Sc,
                    const T* __restrict__ Bi, int N, int D, int V, float c2, int ldz, float* __restrict__ Z,
                    float* __restrict__ gmax, float* __restrict__ gs, float* __restrict__ gu) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int kSlab = F32 ? 64 : Q4 ? 256 : 128;               // k
  constexpr int kRow = kSlab * (int)sizeof(T), kBytes = ROWS * kRow;  // a token's, and all of them: tiles of 128 bytes a row
  constexpr int kParts = kBytes / 4096, kChunks = kRow / 16;     // 16-byte chunks: a thread's, and a row's
  constexpr int kWords = Q4 ? kSlab / 16 : 0;                    // a lane's packed words
  constexpr int kLoads = Q4 ? kWords / 4 : kChunks / 2;          // a lane's 16-byte loads of the head
  constexpr int kFrags = Q4 ? kWords : kLoads;                   // products' operands (8 values of a row's k: bf16, or 2 x 4)
  // bf16 4-bit: scales and biases of four slabs, [128 rows][16 groups] each, through LDS: a row's line of them holds 64 groups,
  // and loaded for one slab at a time it did not last in L1 (16 x 4096 x 151936: 138 us against 104).
  constexpr bool kStage = Q4 && !F32;
  constexpr int kScales = kStage ? 2 * 128 * 32 : 0;
  __shared__ __attribute__((aligned(16))) char lds[2 * kBytes + kScales];
  float(*xm)[ROWS] = reinterpret_cast<float(*)[ROWS]>(lds);  // after the product: 4 waves' statistics
  float(*xs)[ROWS] = xm + 4;
  float(*xu)[ROWS] = xm + 8;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, half = lane >> 5, col = lane & 31;
  const int v0 = blockIdx.x * kGroup;
  const int vr = 32 * w + col < V - v0 ? 32 * w + col : V - 1 - v0;  // rows past the end: their logits are replaced
  const int slabs = (D + kSlab - 1) / kSlab;

  // Operand j of a slab is the 16-byte chunk `2 j + half` of a dense row's; of packed words, word kFrags half + j, so that a
  // lane's words lie together. Past the end of a row a load takes the next row's values (past the head zeros),
  // which in_row makes zeros, as the tokens' are (a 4-bit head's scales are): theirs may be infinite.
  u32x4 wa[kLoads];
  const long left = V - v0;
  const __amdgpu_buffer_rsrc_t rw = Q4 ? rows_rsrc(Wq + (long)v0 * (D >> 3), left * (D >> 1))
                                       : rows_rsrc(W + (long)v0 * D, left * D * (long)sizeof(T));
  uint32_t wo = Q4 ? (uint32_t)vr * (uint32_t)(D >> 1) + half * (kSlab / 4) : (uint32_t)vr * (uint32_t)D * (uint32_t)sizeof(T) + 16 * half;
  // Scales and biases of the lane's groups of a slab: two in a word (bf16), or one.
  uint32_t sc = 0, bi = 0;
  u32x4 stage[2];
  auto load_stage = [&](int slab) {  // thread: 8 groups of row tid / 2
    const int row = tid >> 1, g0 = 4 * slab + 8 * (tid & 1), groups = D >> 6;
    const long at = (long)(v0 + row < V ? v0 + row : V - 1) * groups + g0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const bf16_t* p = reinterpret_cast<const bf16_t*>(x ? Bi : Sc) + at;
      stage[x] = zero4();
      if (groups % 8 == 0) {
        if (g0 < groups) stage[x] = *reinterpret_cast<const u32x4*>(p);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (g0 + i < groups) stage[x][i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
      }
    }
  };
  auto put_stage = [&] {
#pragma unroll
    for (int x = 0; x < 2; ++x) lds_write16(lds + 2 * kBytes + 4096 * x, 16 * tid, stage[x]);
  };
  const __amdgpu_buffer_rsrc_t rs = rows_rsrc(Q4 ? Sc + (long)v0 * (D >> 6) : W, Q4 ? left * (D >> 6) * 4 : 0);
  const __amdgpu_buffer_rsrc_t rb = rows_rsrc(Q4 ? Bi + (long)v0 * (D >> 6) : W, Q4 ? left * (D >> 6) * 4 : 0);
  uint32_t so = (uint32_t)vr * (uint32_t)(D >> 6) * 4;
  // The loads' offsets are in the vector operand, which the range is checked for.
  auto load_head = [&](int i) { wa[i] = load16(rw, wo + (Q4 ? 16 : 32) * i, 0); };
  auto next_head = [&] { wo += Q4 ? kSlab / 2 : kRow; };
  auto load_scales = [&] {  // fp32
    sc = __builtin_amdgcn_raw_buffer_load_b32(rs, so, 0, 0);
    bi = __builtin_amdgcn_raw_buffer_load_b32(rb, so, 0, 0);
    so += 4;
  };
  u32x4 ha[kParts];
  auto load_tokens = [&](int slab) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const int id = tid + 256 * p, row = id / kChunks, k = slab * kSlab + (16 / (int)sizeof(T)) * (id % kChunks);
      ha[p] = row < N && k < D ? *reinterpret_cast<const u32x4*>(H + (long)row * D + k) : zero4();
    }
  };
  auto put_tokens = [&](char* dst) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const int id = tid + 256 * p, row = id / kChunks, c = id % kChunks;
      lds_write16(dst + (c >> 3) * (ROWS * 128), lds_off(row, c & 7), ha[p]);
    }
  };
  auto token = [&](const char* cur, int c, int b) {
    return lds_read16(cur + (c >> 3) * (ROWS * 128), lds_off(ROWS == 16 ? col & 15 : 32 * b + col, c & 7));
  };

  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.f;
  auto product4 = [&](const f32x4& a, const u32x4& t, int b) {
    const f32x4 y = __builtin_bit_cast(f32x4, t);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], y[e], acc[b], 0, 0, 0);
  };
  load_tokens(0);
  if constexpr (kStage) load_stage(0);
  else if constexpr (Q4) load_scales();
#pragma unroll
  for (int i = 0; i < kLoads; ++i) load_head(i);
  next_head();
  put_tokens(lds);
  if constexpr (kStage) put_stage();
  lds_barrier();
  int row_left = D * (int)sizeof(T) - 16 * half;  // bytes
  auto in_row = [&](int j) { return 32 * j < row_left ? wa[j] : zero4(); };
  for (int s = 0; s < slabs; ++s, row_left -= kRow) {
    const char* cur = lds + (s & 1) * kBytes;
    load_tokens(s + 1);  // (past the end: zeros)
    if constexpr (kStage) {
      const char* p = lds + 2 * kBytes + 32 * (32 * w + col) + 8 * (s & 3) + 4 * half;
      sc = *reinterpret_cast<const uint32_t*>(p);
      bi = *reinterpret_cast<const uint32_t*>(p + 4096);
      if ((s & 3) == 3) load_stage(s + 1);  // (past the end: zeros)
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < kFrags; ++j) {
      if constexpr (F32 && Q4) {
        const uint32_t q = wa[j >> 2][j & 3];
        const float sf = __uint_as_float(sc), bf = __uint_as_float(bi);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4 a;
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = __builtin_fmaf(sf, (float)((q >> (16 * h + 4 * e)) & 15u), bf);
#pragma unroll
          for (int b = 0; b < NB; ++b) product4(a, token(cur, 8 * half + 2 * j + h, b), b);
        }
      } else if constexpr (F32) {
        const f32x4 a = __builtin_bit_cast(f32x4, in_row(j));
#pragma unroll
        for (int b = 0; b < NB; ++b) product4(a, token(cur, 2 * j + half, b), b);
      } else {
        bf16x8 a;
        if constexpr (Q4) a = as_bf16x8(dequant8(wa[j >> 2][j & 3], j < 8 ? bf16lo(sc) : bf16hi(sc), j < 8 ? bf16lo(bi) : bf16hi(bi)));
        else a = as_bf16x8(in_row(j));
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = mfma32(a, as_bf16x8(token(cur, Q4 ? kFrags * half + j : 2 * j + half, b)), acc[b]);
      }
      if constexpr (Q4) {
        if (F32 && j == kFrags - 1) load_scales();
        if (j % 4 == 3) {
          load_head(j >> 2);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        load_head(j);
        if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
    next_head();
    put_tokens(lds + ((s + 1) & 1) * kBytes);
    lds_barrier();
    if constexpr (kStage) {
      if ((s & 3) == 3) {  // every wave has read its last of the four
        put_stage();
        lds_barrier();
      }
    }
  }

  // acc[b][r]: vocab row 32 w + 8 (r / 4) + 4 half + r % 4 of the group, token 32 b + col.
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int t = 32 * b + col;
    float top = kNegInf;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int row = 32 * w + 8 * q + 4 * half;
      f32x4 z;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        z[u] = v0 + row + u < V ? acc[b][4 * q + u] : kNegInf;
        top = fmaxf(top, z[u]);
      }
      if (t < N && t < ROWS) *reinterpret_cast<f32x4*>(Z + (long)t * ldz + v0 + row) = z;
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == kNegInf ? 0.f : top * c2;
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (v0 + 32 * w + 8 * (r >> 2) + 4 * half + (r & 3) < V) {
        const float x = __builtin_fmaf(acc[b][r], c2, -base), e = fast_exp2(x);
        s += e;
        u = __builtin_fmaf(e, finite_exponent(x), u);
      }
    s += __shfl_xor(s, 32, 64);
    u += __shfl_xor(u, 32, 64);
    if (half == 0 && t < ROWS) {
      xm[w][t] = top;
      xs[w][t] = s;
      xu[w][t] = u;
    }
  }
  __syncthreads();
  for (int t = tid; t < N; t += 256) {
    float top = kNegInf;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, xm[i][t]);
    float m = kNegInf, s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) lse2_merge(m, s, u, xm[i][t] == kNegInf ? kNegInf : xm[i][t] * c2, xs[i][t], xu[i][t]);
    const long o = (long)t * gridDim.x + blockIdx.x;
    gmax[o] = top;
    gs[o] = s;
    gu[o] = u;
  }
}

// ------------------------------------------------------------------------------------------
// The logits of a gather (GatherPlan): C[v][entry] = W_v . H_token, 128 x 128 a workgroup (4 waves of 64 x 64), 64-deep stages
// through registers, a stage ahead. Bound by what it fetches again: the head once (nearly every group is wanted by some token) and
// the hidden rows for every entry (2 D bytes each). 8 of 8192 x 4096 x 151936: 343 us, 250 of them the head's bytes.
// ------------------------------------------------------------------------------------------
template <int Q4>
__global__ __launch_bounds__(256) void lce_gather_kernel(const bf16_t* __restrict__ H, const bf16_t* __restrict__ W,
                                                         const uint32_t* __restrict__ Wq, const bf16_t* __restrict__ Sc,
                                                         const bf16_t* __restrict__ Bi, int D, int V, GatherPlan plan) {
  __shared__ __attribute__((aligned(16))) char lds[2][2][16384];
  const GatherTile tile = plan.tiles[blockIdx.x];
  if (tile.count == 0) return;
  const int2* entries = plan.entries + tile.first;
  const int v0 = tile.group * kGroup;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, half = lane >> 5, col = lane & 31;
  const int wa = w & 1, wb = w >> 1, c = tid & 7;
  const int nk = (D + 63) / 64;

  // Thread: 16-byte chunk c of rows tid / 8 + 32 p of both operands.
  long hrow[4];
  int vrow[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int r = (tid >> 3) + 32 * p;
    hrow[p] = r < tile.count ? (long)entries[r].x * D : -1;
    vrow[p] = v0 + r < V ? v0 + r : V - 1;  // rows past the end: their logits are replaced
  }
  u32x4 a[4], b[4];
  auto load = [&](int kt) {
    const int k = 64 * kt + 8 * c;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      b[p] = hrow[p] >= 0 && k < D ? *reinterpret_cast<const u32x4*>(H + hrow[p] + k) : zero4();
      if constexpr (Q4) {
        const long g = (long)vrow[p] * (D >> 6) + kt;
        a[p] = dequant8(Wq[(long)vrow[p] * (D >> 3) + (k >> 3)], bf16_to_f32(Sc[g]), bf16_to_f32(Bi[g]));
      } else {
        a[p] = k < D ? *reinterpret_cast<const u32x4*>(W + (long)vrow[p] * D + k) : zero4();
      }
    }
  };
  auto put = [&](int s) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int r = (tid >> 3) + 32 * p;
      lds_write16(lds[s][0], lds_off(r, c), a[p]);
      lds_write16(lds[s][1], lds_off(r, c), b[p]);
    }
  };
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  load(0);
  put(0);
  __syncthreads();
  for (int kt = 0; kt < nk; ++kt) {
    const int cur = kt & 1;
    if (kt + 1 < nk) load(kt + 1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      bf16x8 x[2], y[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = as_bf16x8(lds_read16(lds[cur][0], lds_off(64 * wa + 32 * i + col, 2 * ks + half)));
#pragma unroll
      for (int j = 0; j < 2; ++j) y[j] = as_bf16x8(lds_read16(lds[cur][1], lds_off(64 * wb + 32 * j + col, 2 * ks + half)));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma32(x[i], y[j], acc[i][j]);
    }
    if (kt + 1 < nk) put(cur ^ 1);
    __syncthreads();
  }
  store_gathered<2, 2>(acc, plan, entries, tile.count, V - v0, 64 * wa, 64 * wb, lane);
}

// ------------------------------------------------------------------------------------------
// Plan of a gather: entries counted by group, dealt into runs of one group each, the runs cut into tiles. The order of a group's
// entries is that of the atomics and decides nothing: each is a column of its own.
// ------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void zero_counts_kernel(int* __restrict__ counts, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) counts[i] = 0;
}

// counts -> the first entry of each group (in its place), and the tiles.
__global__ __launch_bounds__(1024) void gather_tiles_kernel(int* __restrict__ counts, int groups, GatherTile* __restrict__ tiles,
                                                            int max_tiles) {
  __shared__ int sum_e[16], sum_t[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int per = (groups + 1023) / 1024, lo = tid * per, hi = lo + per < groups ? lo + per : groups;
  int e = 0, t = 0;
  for (int g = lo; g < hi; ++g) {
    e += counts[g];
    t += (counts[g] + kGroup - 1) / kGroup;
  }
  int re = e, rt = t;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int ue = __shfl_up(re, o, 64), ut = __shfl_up(rt, o, 64);
    if (lane >= o) {
      re += ue;
      rt += ut;
    }
  }
  if (lane == 63) {
    sum_e[w] = re;
    sum_t[w] = rt;
  }
  __syncthreads();
  int first = re - e, tile = rt - t, all = 0;
  for (int i = 0; i < 16; ++i) {
    if (i < w) {
      first += sum_e[i];
      tile += sum_t[i];
    }
    all += sum_t[i];
  }
  for (int g = lo; g < hi; ++g) {
    const int n = counts[g];
    counts[g] = first;
    for (int k = 0; k < n; k += kGroup) tiles[tile++] = GatherTile{g, first + k, n - k < kGroup ? n - k : kGroup, 0};
    first += n;
  }
  for (int i = all + tid; i < max_tiles; i += 1024) tiles[i] = GatherTile{0, 0, 0, 0};
}

// groups [N][k] (a row's are its chosen ones; < 0: none) to entries that keep whole groups.
__global__ __launch_bounds__(256) void gather_groups_kernel(const int* __restrict__ groups, long n, int k,
                                                            int* __restrict__ cursor, int2* __restrict__ entries) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n || groups[i] < 0) return;
  entries[atomicAdd(&cursor[groups[i]], 1)] = int2{(int)(i / k), (int)i};
}

__device__ __forceinline__ bool listed(long long id, float lp, const uint8_t* mask, long row, long V) {
  return id >= 0 && id < V && lp != kNegInf && (!mask || mask[row]);
}

constexpr int kPerLane = kScoreTop / 64;

// The column of slot lane + 64 i of row t's list, -1 where the slot is empty: not a token, nothing of the teacher's, or a column
// that an earlier slot has.
__device__ __forceinline__ void load_list(const int64_t* ids, const float* teacher, const uint8_t* mask, long t, long V, int k, int lane,
                                          int (&id)[kPerLane]) {
  bool on[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int s = lane + 64 * i;
    const long long y = s < k ? ids[t * k + s] : -1;
    on[i] = listed(y, s < k ? teacher[t * k + s] : 0.f, mask, t, V);
    id[i] = on[i] ? (int)y : -1;
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    for (int j = 0; j < 64 && 64 * i + j < k; ++j) {
      const int other = __builtin_amdgcn_readlane(id[i], j);
#pragma unroll
      for (int o = 0; o < kPerLane; ++o)
        if (64 * i + j < lane + 64 * o && other >= 0 && other == id[o]) on[o] = false;
    }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    if (!on[i]) id[i] = -1;
}
// A teacher's lists [N][k], one wave a row: its outcomes' columns, ascending and each once (kNoColumn past them), and the slot of
// each. A place is the number of (column, slot) before one's own.
__global__ __launch_bounds__(256) void sort_lists_kernel(const int64_t* __restrict__ ids, const float* __restrict__ teacher,
                                                         const uint8_t* __restrict__ mask, long n, long V, int k,
                                                         int* __restrict__ column, int* __restrict__ slot) {
  const int lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= n) return;
  int id[kPerLane];
  load_list(ids, teacher, mask, t, V, k, lane, id);
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int s = lane + 64 * i;
    const int key = id[i] < 0 ? kNoColumn : id[i];
    int place = 0;
#pragma unroll
    for (int o = 0; o < kPerLane; ++o)
      for (int j = 0; j < 64 && 64 * o + j < k; ++j) {
        const int other = __builtin_amdgcn_readlane(id[o], j);
        const int their = other < 0 ? kNoColumn : other;
        place += their < key || (their == key && 64 * o + j < s);
      }
    if (s < k) {
      column[t * k + place] = key;
      slot[t * k + place] = s;
    }
  }
}

// A target as its row's list of one.
__global__ __launch_bounds__(256) void target_columns_kernel(const int64_t* __restrict__ targets, long long ignore_index, long n, long V,
                                                             int* __restrict__ column) {
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= n) return;
  const long long y = targets[t];
  column[t] = y != ignore_index && y >= 0 && y < V ? (int)y : kNoColumn;
}

// ------------------------------------------------------------------------------------------
// Scoring, per token: the statistics of its row, the target's log probability, the groups to look into (and, where the logits
// were kept, the alternatives themselves). One workgroup a token: bound by the chain of loads, barriers and counts where there are few tokens (12 us
// for 16 x 151936, 15 for 20 alternatives of one), by its vector instructions where there are many (8192: 50).
// ------------------------------------------------------------------------------------------
// Partials of one row: value i at base[i * stride]. m: of x in the log2 domain, or (few tokens) of z, times c2.
struct RowParts {
  const float *m, *s, *u;
  int count;
  long stride, row;  // floats between partials, and between rows
  float m_scale;
};

// put(i, load(i)) for i < n, one i a thread and step, the loads of B steps in flight at once.
template <int B, class LOAD, class PUT>
__device__ __forceinline__ void each(int n, const LOAD& load, const PUT& put) {
  for (int base = threadIdx.x; base < n; base += B * kPick) {
    decltype(load(0)) x[B];
#pragma unroll
    for (int b = 0; b < B; ++b) x[b] = load(base + b * kPick < n ? base + b * kPick : n - 1);
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (base + b * kPick < n) put(base + b * kPick, x[b]);
  }
}

// (m, s, u) of a row, in every thread of the workgroup.
__device__ __forceinline__ void merge_row(const RowParts& p, long t, float& m, float& s, float& u, float (&x)[3][kPick / 64]) {
  m = kNegInf;
  s = u = 0.f;
  const float *pm = p.m + t * p.row, *ps = p.s + t * p.row, *pu = p.u + t * p.row;
  struct Part { float m, s, u; };
  each<5>(p.count, [&](int i) { return Part{pm[i * p.stride], ps[i * p.stride], pu[i * p.stride]}; },
          [&](int, const Part& x) { lse2_merge(m, s, u, x.m == kNegInf ? kNegInf : x.m * p.m_scale, x.s, x.u); });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float mo = __shfl_xor(m, o, 64), so = __shfl_xor(s, o, 64), uo = __shfl_xor(u, o, 64);
    lse2_merge(m, s, u, mo, so, uo);
  }
  if ((threadIdx.x & 63) == 0) {
    x[0][threadIdx.x >> 6] = m;
    x[1][threadIdx.x >> 6] = s;
    x[2][threadIdx.x >> 6] = u;
  }
  __syncthreads();
  m = x[0][0];
  s = x[1][0];
  u = x[2][0];
#pragma unroll
  for (int i = 1; i < kPick / 64; ++i) lse2_merge(m, s, u, x[0][i], x[1][i], x[2][i]);
}

// The log probability of a logit z by norm = (m, log2 s) of its row: relative to the row's largest logit, so that it is right to the
// digits of what it leaves of 0. As z / temperature - lse it had the last digits of a logit: 2e-6 at 32, 1 - p of 8.5e-5 off by 3%.
__device__ __forceinline__ float log_p(float z, float c2, float2 norm) { return (__builtin_fmaf(z, c2, -norm.x) - norm.y) * kLn2; }

// The K largest of a row's candidate logits, ngroups kGroup of them in LDS as keys, in order, with their log probabilities.
// The groups ascend, so positions ascend with the index. `least`: the K-th largest of the groups' maxima (0 with fewer than K
// groups), below which nothing is chosen: mostly a few more than K are left, and each one's place is its count of those before
// it. A target among them takes its log probability from here.
template <int MC>
__device__ __forceinline__ void write_top(const uint32_t* key, const int* group, int ngroups, int K, uint32_t least, int V,
                                          float c2, float2 norm, long t, long long target, const LogprobsOut& out, PickScratch& s) {
  const int M = ngroups * kGroup;
  int n = list_from(key, M, least, s);
  if (n > kRanked || n < K) {  // many equal ones; or logits that are no numbers
    pick_largest<MC / kPick>(key, M, K, [&](int place, int i) { s.list[place] = entry_of(key[i], i); }, s);
    n = K;
  }
  for (int i = threadIdx.x; i < n; i += kPick) {
    const int rank = rank_of(s.list[i], n, s);
    if (rank >= K) continue;
    const int p = entry_at(s.list[i]), id = group[p / kGroup] * kGroup + p % kGroup;
    const float lp = log_p(key_value(entry_key(s.list[i])), c2, norm);
    out.top_ids[t * K + rank] = id < V ? id : -1;
    out.top_logprobs[t * K + rank] = lp;
    if (id == target) out.tgt[t] = out.logprobs[t] = lp;
  }
}

constexpr int kMaxGroups = (int)(kScoreVocab / kGroup);

// KEPT: the logits Z [N][ldz] of few tokens. MG, MC: room for a row's groups and candidates (0: none).
template <bool KEPT, int MG, int MC>
__global__ __launch_bounds__(kPick) void score_rows_kernel(RowParts parts, const float* __restrict__ gmax, int ngroups, int ldg,
                                                           const float* __restrict__ Z, long ldz,
                                                           const int64_t* __restrict__ targets, long long ignore_index, int V,
                                                           float c2, int K, int take, LogprobsOut out,
                                                           int* __restrict__ groups, int* __restrict__ counts,
                                                           uint32_t* __restrict__ floors, float2* __restrict__ norms) {
  __shared__ float x[3][kPick / 64];
  __shared__ float2 norm;
  __shared__ PickScratch scratch;
  __shared__ uint32_t key[MG > MC ? MG : MC > 0 ? MC : 1];
  __shared__ int group[kScoreTop];
  const long t = blockIdx.x;
  const int tid = threadIdx.x;
  const long long y = targets ? targets[t] : 0;
  const bool dead = targets && y == ignore_index;
  if (dead) {
    for (int i = tid; i < K; i += kPick) {
      out.top_ids[t * K + i] = -1;
      out.top_logprobs[t * K + i] = kNegInf;
      if (!KEPT && i < take) groups[t * take + i] = -1;
    }
    if (tid == 0) {
      out.entropy[t] = out.lse[t] = 0.f;
      if (targets) out.logprobs[t] = out.tgt[t] = 0.f;
    }
    return;
  }
  float m, s, u;
  merge_row(parts, t, m, s, u, x);
  const bool in = y >= 0 && y < V;
  if (tid == 0) {
    norm = float2{m, fast_log2(s)};
    const float lse = (m + norm.y) * kLn2;
    out.lse[t] = lse;
    out.entropy[t] = (norm.y - u / s) * kLn2;
    if (targets) out.tgt[t] = out.logprobs[t] = in ? log_p(KEPT ? Z[t * ldz + y] : out.tgt[t], c2, norm) : -lse;
  }
  if constexpr (MG > 0) {
    each<5>(ngroups, [&](int i) { return gmax[t * ldg + i]; }, [&](int i, float x) { key[i] = order_key(x); });
    __syncthreads();
    uint32_t least = pick_few<MG / kPick>(key, ngroups, take, group, scratch);
    if (take < K) least = 0;
    if constexpr (KEPT) {
      each<5>(take * kGroup, [&](int i) { return Z[t * ldz + (long)group[i / kGroup] * kGroup + i % kGroup]; },
              [&](int i, float x) { key[i] = group[i / kGroup] * kGroup + i % kGroup < V ? order_key(x) : 0u; });
      __syncthreads();
      write_top<MC>(key, group, take, K, least, V, c2, norm, t, targets ? y : -1, out, scratch);
    } else if (tid < take) {
      groups[t * take + tid] = group[tid];
      atomicAdd(&counts[group[tid]], 1);
      if (tid == 0) {
        floors[t] = least;
        norms[t] = norm;
      }
    }
  }
}

// After the gather: the alternatives from the chosen groups' logits [N][take][kGroup].
template <int MC>
__global__ __launch_bounds__(kPick) void score_top_kernel(const float* __restrict__ rows, const int* __restrict__ groups,
                                                          const uint32_t* __restrict__ floors, const float2* __restrict__ norms,
                                                          const int64_t* __restrict__ targets, int V, float c2, int K, int take,
                                                          LogprobsOut out) {
  __shared__ PickScratch scratch;
  __shared__ uint32_t key[MC];
  __shared__ int group[kScoreTop];
  const long t = blockIdx.x;
  const int tid = threadIdx.x;
  if (groups[t * take] < 0) return;  // an ignored token
  for (int i = tid; i < take; i += kPick) group[i] = groups[t * take + i];
  each<4>(take * kGroup, [&](int i) { return rows[t * take * kGroup + i]; }, [&](int i, float x) { key[i] = order_key(x); });
  __syncthreads();
  write_top<MC>(key, group, take, K, floors[t], V, c2, norms[t], t, targets ? targets[t] : -1, out, scratch);
}

// ------------------------------------------------------------------------------------------
// Distillation, one wave a token, its list as it came (FEW: few tokens, with their logits Z and every group's maximum and sum)
// or sorted, with the logits picks and the partials of all others. With q_k = p at the list's ids, R the others' sum of p, t_k
// and T = 1 - sum t the teacher's, and f = dL/dq but for a constant (f_R for the rest),
//   forward  sum t log(t / q) + T log(T / R):        f = -t / q,              f_R = -T / R
//   reverse  sum q log(q / t) + R log(R / T):        f = log(q / t),          f_R = log(R / T)
//   jsd      b KL(t | m) + (1 - b) KL(q | m), m = b t + (1 - b) q:  f = (1 - b) log(q / m), f_R = (1 - b) log(R / m_R)
// the gradient by a logit is p (f_R - F) off the list and q (f - F) on it, F = sum q f + R f_R. R and T (but in F) are at least
// kTailFloor. From the partials on in 64 bits: T is a difference, and the products above are what take the time
// (8192 lists of 64: 16 us, their sorting 35, the products 21.6 ms).
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ double log_add(double a, double b) {
  const double hi = fmax(a, b);
  return hi + log1p(exp(fmin(a, b) - hi));
}

constexpr float kLeast = 1.17549435e-38f;

// Few tokens: (base, the sum of 2^(z c2 - base)) over the columns that the wave's list `id` leaves. Groups without a listed
// column give their sums; the others are summed again without it, two columns a lane, eight groups' loads in flight.
struct OffList {
  float base;
  double sum;
};
struct GroupScratch {
  uint32_t listed[kScoreVocab / kGroup / 32];  // bit g: group g has a listed column
  uint32_t columns[kScoreTop][kGroup / 32];    // the listed columns of a group, at the slot of its first one
  int group[kScoreTop], slot[kScoreTop];       // the groups that have some, and that slot
};
__device__ __forceinline__ OffList few_off_list(const RowParts& p, long t, const float* __restrict__ z, const int (&id)[kPerLane], int k,
                                                int lane, GroupScratch& x) {
  static_assert(kGroup == 128, "two columns a lane");
  for (int i = lane; i < (p.count + 31) / 32; i += 64) x.listed[i] = 0u;
  for (int i = lane; i < kScoreTop * (kGroup / 32); i += 64) x.columns[i / (kGroup / 32)][i % (kGroup / 32)] = 0u;
  int first[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) first[i] = -1;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    for (int j = 0; j < 64 && 64 * i + j < k; ++j) {
      const int other = __builtin_amdgcn_readlane(id[i], j);
#pragma unroll
      for (int o = 0; o < kPerLane; ++o)
        if (first[o] < 0 && other >= 0 && id[o] >= 0 && other / kGroup == id[o] / kGroup) first[o] = 64 * i + j;
    }
  __threadfence_block();  // (the wave's own LDS)
  int groups = 0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int g = id[i] / kGroup, c = id[i] % kGroup;
    if (id[i] >= 0) {
      atomicOr(&x.listed[g >> 5], 1u << (g & 31));
      atomicOr(&x.columns[first[i]][c >> 5], 1u << (c & 31));
    }
    const uint64_t firsts = __ballot(first[i] == lane + 64 * i);
    if (first[i] == lane + 64 * i) {
      const int at = groups + __popcll(firsts & ((1ull << lane) - 1));
      x.group[at] = g;
      x.slot[at] = first[i];
    }
    groups += __popcll(firsts);
  }
  __threadfence_block();
  float top = kNegInf, m = kNegInf, s = 0.f;
  for (int i = lane; i < p.count; i += 64) {
    const float mi = p.m[t * p.row + i * p.stride];
    top = fmaxf(top, mi);
    if (!(x.listed[i >> 5] >> (i & 31) & 1)) lse2_merge(m, s, mi == kNegInf ? kNegInf : mi * p.m_scale, p.s[t * p.row + i * p.stride]);
  }
  top = wave_max(top) * p.m_scale;
  const float base = top == kNegInf ? 0.f : top;
  double sum = (double)s * (double)fast_exp2(m - base);
  constexpr int kFlight = 8;
  for (int b = 0; b < groups; b += kFlight) {
    f32x2 v[kFlight];
#pragma unroll
    for (int e = 0; e < kFlight; ++e)
      v[e] = *reinterpret_cast<const f32x2*>(z + (long)x.group[b + e < groups ? b + e : b] * kGroup + 2 * lane);
#pragma unroll
    for (int e = 0; e < kFlight; ++e) {
      if (b + e >= groups) continue;
      const uint32_t listed = x.columns[x.slot[b + e]][lane >> 4] >> (2 * lane & 31);
#pragma unroll
      for (int c = 0; c < 2; ++c) sum += listed >> c & 1 ? 0.0 : (double)fast_exp2(__builtin_fmaf(v[e][c], p.m_scale, -base));
    }
  }
  return {base, wave_sum64(sum)};
}

template <int KIND, bool FEW>
__global__ __launch_bounds__(256) void distill_rows_kernel(RowParts parts, const int* __restrict__ sorted,
                                                           const int* __restrict__ slot, const float* __restrict__ picks,
                                                           const float* __restrict__ Z, long ldz,
                                                           const int64_t* __restrict__ ids, const float* __restrict__ teacher,
                                                           const uint8_t* __restrict__ mask, long n, long V, float c2, double inv_t,
                                                           int k, int renormalize, double beta, float* __restrict__ row_loss,
                                                           int* __restrict__ row_counts, float* __restrict__ lse_out,
                                                           float* __restrict__ rest_out, float* __restrict__ coef,
                                                           int* __restrict__ columns) {
  __shared__ GroupScratch scratch[FEW ? 4 : 1];
  const int lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= n) return;
  // Which slots hold an outcome: a column of its own that the teacher gives something to.
  int id[kPerLane];
  if constexpr (FEW) {
    load_list(ids, teacher, mask, t, V, k, lane, id);
  } else {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int y = lane + 64 * i < k ? sorted[t * k + lane + 64 * i] : kNoColumn;
      id[i] = y == kNoColumn ? -1 : y;
    }
  }
  float lp[kPerLane];
  bool on[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const long o = t * k + lane + 64 * i;
    on[i] = id[i] >= 0;
    lp[i] = on[i] ? teacher[FEW ? o : t * k + slot[o]] : 0.f;
  }
  bool some = false;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) some |= __any(on[i]);
  if (!some) {
    for (int s = lane; s < k; s += 64) {
      coef[t * k + s] = 0.f;
      columns[t * k + s] = -1;
    }
    if (lane == 0) {
      row_loss[t] = lse_out[t] = rest_out[t] = 0.f;
      row_counts[t] = 0;
    }
    return;
  }
  OffList off;
  if constexpr (FEW) {
    off = few_off_list(parts, t, Z + t * ldz, id, k, lane, scratch[threadIdx.x >> 6]);
  } else {
    float m = kNegInf, s = 0.f;
    for (int i = lane; i < parts.count; i += 64)
      lse2_merge(m, s, parts.m[t * parts.row + i * parts.stride], parts.s[t * parts.row + i * parts.stride]);
    off.base = wave_max(m);
    off.sum = wave_sum64((double)s * (double)fast_exp2(off.base == kNegInf ? m : m - off.base));  // (-inf: all is listed)
  }

  // x = z c2 is exact in 64 bits, and the partials' are of the same c2.
  double x[kPerLane], lq[kPerLane], lt[kPerLane], q[kPerLane], p[kPerLane], top = -HUGE_VAL, total = 0.0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    float z = 0.f;
    if (on[i]) z = FEW ? Z[t * ldz + id[i]] : picks[t * k + lane + 64 * i];
    x[i] = (double)z * (double)c2;
    if (on[i]) top = fmax(top, x[i]);
    lt[i] = (double)lp[i];
  }
  top = fmax(wave_max64(top), (double)off.base);
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    q[i] = on[i] ? exp2(x[i] - top) : 0.0;
    total += q[i];
  }
  const double rest = off.sum * exp2((double)off.base - top);
  total = wave_sum64(total) + rest;
  const double lse2 = top + log2(total), left = rest / total;
  constexpr double kLog2 = 0.6931471805599453;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    lq[i] = on[i] ? (x[i] - lse2) * kLog2 : 0.0;
    q[i] /= total;
  }
  if (renormalize) {
    double hi = -HUGE_VAL, sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      lt[i] *= inv_t;
      if (on[i]) hi = fmax(hi, lt[i]);
    }
    hi = wave_max64(hi);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (on[i]) sum += exp(lt[i] - hi);
    hi += log(wave_sum64(sum));
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) lt[i] -= hi;
  }
  double st = 0.0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    p[i] = on[i] ? exp(lt[i]) : 0.0;
    st += p[i];
  }
  const double rq = fmax(left, kTailFloor), rt = renormalize ? 0.0 : fmax(1.0 - wave_sum64(st), kTailFloor);
  double loss = 0.0, qf[kPerLane], sqf = 0.0, frest;
  if constexpr (KIND == kDistillForward) {
    frest = -rt / rq;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      if (on[i]) loss += p[i] * (lt[i] - lq[i]);
      qf[i] = -p[i];
      sqf += qf[i];
    }
    loss = wave_sum64(loss) + (rt > 0.0 ? rt * log(rt / rq) : 0.0);
  } else if constexpr (KIND == kDistillReverse) {
    frest = log(rq / rt);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      qf[i] = on[i] && q[i] != 0.0 ? q[i] * (lq[i] - lt[i]) : 0.0;
      sqf += qf[i];
    }
    loss = wave_sum64(sqf) + rq * frest;
  } else {
    const double a = log(beta), b = log1p(-beta), rm = beta * rt + (1.0 - beta) * rq;
    frest = (1.0 - beta) * log(rq / rm);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      qf[i] = 0.0;
      if (on[i]) {
        const double lm = log_add(a + lt[i], b + lq[i]);
        if (q[i] != 0.0) qf[i] = (1.0 - beta) * q[i] * (lq[i] - lm);
        loss += beta * p[i] * (lt[i] - lm);
      }
      sqf += qf[i];
    }
    loss = wave_sum64(loss + sqf) + rq * frest + (rt > 0.0 ? beta * rt * log(rt / rm) : 0.0);
  }
  const double mean = wave_sum64(sqf) + left * frest;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int slot = lane + 64 * i;
    if (slot < k) {
      coef[t * k + slot] = on[i] ? (float)((qf[i] - q[i] * mean) * inv_t) : 0.f;
      columns[t * k + slot] = on[i] ? id[i] : -1;
    }
  }
  if (lane == 0) {
    row_loss[t] = (float)loss;
    row_counts[t] = 1;
    lse_out[t] = (float)(lse2 * kLog2);
    const float factor = (float)((frest - mean) * inv_t);
    rest_out[t] = factor == 0.f ? kLeast : factor;  // 0 is a row that gets no gradient
  }
}

// The rows' losses as one number, summed in 64 bits in a fixed order, and what a row's gradient is multiplied with. One
// workgroup.
__global__ __launch_bounds__(1024) void distill_reduce_kernel(const float* __restrict__ row_loss,
                                                              const int* __restrict__ row_counts, long n, int mean,
                                                              float* __restrict__ loss, float* __restrict__ scale) {
  __shared__ double sums[16];
  __shared__ long counts[16];
  double s = 0.0;
  long c = 0;
  for (long i = threadIdx.x; i < n; i += 1024) {
    s += (double)row_loss[i];
    c += row_counts[i];
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    c += __shfl_xor(c, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = s;
    counts[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) {
      s += sums[w];
      c += counts[w];
    }
    const double by = mean ? 1.0 / (double)(c > 1 ? c : 1) : 1.0;
    *loss = (float)(s * by);
    *scale = (float)by;
  }
}

// ------------------------------------------------------------------------------------------
// Factors of the backward's gradient tiles (AffineGrad).
// ------------------------------------------------------------------------------------------
// Scoring: dL/dz = (a [v = y] - p (a + b (log p + entropy))) / temperature, a and b the two gradients.
__global__ __launch_bounds__(256) void logprobs_coef_kernel(const float* __restrict__ d_logprobs,
                                                            const float* __restrict__ d_entropy,
                                                            const int64_t* __restrict__ targets, long long ignore_index,
                                                            const float* __restrict__ lse, const float* __restrict__ entropy,
                                                            const float* __restrict__ tgt, long n, long V, float inv_t,
                                                            float* __restrict__ alpha, float* __restrict__ beta,
                                                            int* __restrict__ columns, float* __restrict__ value) {
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= n) return;
  const long long y = targets ? targets[t] : -1;
  const bool dead = targets && y == ignore_index, in = !dead && targets && y >= 0 && y < V;
  const float a = !dead && d_logprobs ? d_logprobs[t] : 0.f, b = !dead && d_entropy ? d_entropy[t] : 0.f;
  const float up = lse[t] - entropy[t], l = in ? finite_exponent(tgt[t]) : 0.f;
  alpha[t] = (b * up - a) * inv_t;
  beta[t] = -b * inv_t * inv_t;
  columns[t] = in ? (int)y : -1;
  value[t] = in ? (-a * expm1f(l) - b * expf(l) * (l + entropy[t])) * inv_t : 0.f;
}

__global__ __launch_bounds__(256) void distill_coef_kernel(const float* __restrict__ d_loss, int per_row,
                                                           const float* __restrict__ scale, const float* __restrict__ rest,
                                                           const float* __restrict__ coef, long n, int k,
                                                           float* __restrict__ alpha, float* __restrict__ value) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * k) return;
  const long t = i / k;
  const float ct = per_row ? d_loss[t] : d_loss[0] * *scale;
  const float c = coef[i];
  value[i] = c == 0.f ? 0.f : c * ct;
  if (i == t * k) {
    const float a = rest[t] == 0.f ? 0.f : rest[t] * ct;
    alpha[t] = a == 0.f && rest[t] != 0.f && ct != 0.f ? kLeast : a;
  }
}

// G = p (alpha + beta z) from kept logits, a row a blockIdx.y, 16 bytes a thread; bound by reading z and writing G (AffineGrad's
// listed columns follow). rest: what rounding leaves (AffineGrad's halves), or null. 1023 x 32000, bf16: 36 us, and with it the step of a
// 4-bit head at 2048 dims 488 -> 407.
template <class G>
__global__ __launch_bounds__(256) void affine_tiles_kernel(const float* __restrict__ Z, long ldz, const float* __restrict__ lse,
                                                           AffineRows rows, int v_begin, int vlim, int cols, long ldg,
                                                           G* __restrict__ out, G* __restrict__ rest) {
  constexpr int kEach = 16 / (int)sizeof(G);
  const long t = blockIdx.y;
  const int c = (blockIdx.x * 256 + threadIdx.x) * kEach, v = v_begin + c;
  if (c >= cols) return;
  const float alpha = rows.alpha[t], beta = rows.beta ? rows.beta[t] : 0.f, l2 = lse[t] * kLog2e;
  const bool live = alpha != 0.f || beta != 0.f;
  float g[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    const f32x4 z = live && v + i < vlim ? *reinterpret_cast<const f32x4*>(Z + t * ldz + v + i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      g[i + u] = live && v + i + u < vlim ? fast_exp2(__builtin_fmaf(z[u], rows.scale2, -l2)) * __builtin_fmaf(beta, finite_exponent(z[u]), alpha) : 0.f;
  }
  if constexpr (sizeof(G) == 2) {
    *reinterpret_cast<u32x4*>(out + t * ldg + c) =
        u32x4{pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]), pack_bf16x2(g[6], g[7])};
    if (!rest) return;
#pragma unroll
    for (int i = 0; i < kEach; ++i) g[i] = bf16_rest(g[i]);
    *reinterpret_cast<u32x4*>(rest + t * ldg + c) =
        u32x4{pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]), pack_bf16x2(g[6], g[7])};
  } else {
    *reinterpret_cast<f32x4*>(out + t * ldg + c) = f32x4{g[0], g[1], g[2], g[3]};
  }
}

// A row whose factors are both 0 gets no gradient and may hold anything, NaN too: in dW = G^T H its zeros would meet that.
__global__ __launch_bounds__(256) void clean_rows_kernel(const uint32_t* __restrict__ h, const float* __restrict__ alpha,
                                                         const float* __restrict__ beta, long row_words, int copies,
                                                         uint32_t* __restrict__ out) {
  const long t = blockIdx.x, all = gridDim.x * row_words;
  const bool live = alpha[t] != 0.f || (beta && beta[t] != 0.f);
  for (long i = threadIdx.x; i < row_words; i += 256) {
    const uint32_t x = live ? h[t * row_words + i] : 0u;
    for (int c = 0; c < copies; ++c) out[c * all + t * row_words + i] = x;
  }
}

__global__ __launch_bounds__(256) void join_halves_kernel(const float* __restrict__ halves, long count, bf16_t* __restrict__ dH) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < count) dH[i] = __builtin_bit_cast(bf16_t, (__bf16)(halves[i] + halves[count + i]));
}

// ------------------------------------------------------------------------------------------
// Host side.
// ------------------------------------------------------------------------------------------
long ceil_div(long a, long b) { return (a + b - 1) / b; }
int groups_of(long v) { return (int)ceil_div(v, kGroup); }

// Room in a workspace, in order; every part starts at a 256-byte boundary.
struct Carver {
  char* base;
  size_t used = 0;
  template <class T>
  T* take(long count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += ((size_t)count * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

struct Scratch {
  bool few, kept;  // kept: the logits are, by the few tokens' kernel or the tiles'
  int groups, ldg, take, max_tiles;  // ldg: floats between the rows of gmax
  long rows, ldz, stage_rows;
  float *m, *s, *u, *gmax, *z, *gs, *gu, *cand, *picks, *row_loss;
  int *chosen, *counts, *column, *slot, *row_counts;
  uint32_t* floors;
  float2* norms;
  int2* entries;
  GatherTile* tiles;
  bf16_t* stage;
  float* stage32;
};

// Whether a forward with alternatives writes its logits rather than forming some again: 4 bytes a logit, against the head read
// once more and five small launches. N x D x V, alternatives; formed again / kept: 333 x 2048 x 32003, 8: 120 / 84 us; 440 x 4096 x
// 151936, 8: 834 / 617; 2000 x 2048 x 32003, 8: 296 / 292; 8000 x 256 x 8000, 8: 341 / 173; 1000 x 512 x 50000, 8: 110 / 116.
bool keep_logits(const ScoreShape& sh) { return 4 * sh.n * sh.v <= kKeptBytes; }
// Tokens of one pass that does: a row is a whole number of groups, which a small vocabulary is far from.
long kept_rows(long n, long ldz) {
  const long most = kKeptBytes / (4 * ldz);
  return n <= most ? n : most < 256 ? most : most / 256 * 256;
}

// k_list: length of a teacher's list (0: scoring, with `top` alternatives).
// logits: the caller's, which keeps them (or, for its size alone, any address).
Scratch carve(const ScoreShape& sh, int f32, int q4, int top, int k_list, float* logits, void* ws, size_t* bytes) {
  Scratch x{};
  Carver c{static_cast<char*>(ws)};
  x.few = f32 ? sh.n <= kFewTokens32 && sh.d % 4 == 0 && sh.d < kScoreDims : sh.n <= kFewTokens;
  x.groups = groups_of(sh.v);
  x.ldg = x.few ? x.groups : (x.groups + 1) / 2 * 2;  // a tile of 256 logits writes both its groups, the last one too
  x.take = top < x.groups ? top : x.groups;
  x.ldz = (long)x.groups * kGroup;
  x.kept = x.few || logits || (top && keep_logits(sh));
  x.rows = x.few || logits ? sh.n : x.kept ? kept_rows(sh.n, x.ldz) : sh.n < kScoreRows ? sh.n : kScoreRows;
  if (x.few) {
    x.z = logits ? logits : c.take<float>(x.rows * x.ldz);
    x.gmax = c.take<float>(x.rows * x.groups);
    x.gs = c.take<float>(x.rows * x.groups);
    x.gu = c.take<float>(x.rows * x.groups);
  } else {
    // (the last block of rows may split the vocabulary into more)
    const long last = sh.n - (sh.n - 1) / x.rows * x.rows;
    auto splits = [&](long n) { return (long)(f32 ? lce32_fwd_nsplit(n, sh.v) : lce_fwd_nsplit(n, sh.v)); };
    const long parts = splits(x.rows) * x.rows > splits(last) * last ? splits(x.rows) * x.rows : splits(last) * last;
    x.m = c.take<float>(parts);
    x.s = c.take<float>(parts);
    if (!k_list) x.u = c.take<float>(parts);
    if (top) {
      x.gmax = c.take<float>(x.rows * x.ldg);
    }
    if (x.kept) x.z = logits ? logits : c.take<float>(x.rows * x.ldz);
    const long entries = x.kept ? 0 : x.rows * x.take;
    if (entries) {
      x.chosen = c.take<int>(entries);
      x.floors = c.take<uint32_t>(x.rows);
      x.norms = c.take<float2>(x.rows);
      x.cand = c.take<float>(entries * kGroup);
      x.counts = c.take<int>(x.groups);
      x.entries = c.take<int2>(entries);
      x.max_tiles = (int)(x.groups + entries / kGroup);  // each group's last tile may be part of one
      if (x.max_tiles > entries) x.max_tiles = (int)entries;
      x.tiles = c.take<GatherTile>(x.max_tiles);
    }
    if (!k_list && !x.kept) x.column = c.take<int>(x.rows);  // the targets'
    if (k_list) {
      x.column = c.take<int>(x.rows * k_list);
      x.slot = c.take<int>(x.rows * k_list);
      x.picks = c.take<float>(x.rows * k_list);
    }
    if (q4 && sh.stage) {
      x.stage_rows = sh.v;
      if (f32) x.stage32 = c.take<float>(sh.v * sh.d);
      else x.stage = c.take<bf16_t>(sh.v * sh.d);
    }
  }
  if (k_list) {
    x.row_loss = c.take<float>(sh.n);
    x.row_counts = c.take<int>(sh.n);
  }
  *bytes = c.used;
  return x;
}

#define MTP_LAUNCHED()                        \
  do {                                        \
    const hipError_t e = hipGetLastError();   \
    if (e != hipSuccess) return e;            \
  } while (0)

template <class T>
hipError_t run_few(const T* H, int q4, const T* w, const uint32_t* wq, const T* sc, const T* bi, const ScoreShape& sh, const Scratch& x,
                   float c2, hipStream_t st) {
  auto run = [&](auto nb, auto rows) {
    constexpr int NB = decltype(nb)::value, ROWS = decltype(rows)::value;
    auto kernel = q4 ? lce_few_kernel<T, 1, NB, ROWS> : lce_few_kernel<T, 0, NB, ROWS>;
    hipLaunchKernelGGL(kernel, dim3(x.groups), dim3(256), 0, st, H, w, wq, sc, bi, (int)sh.n, (int)sh.d, (int)sh.v, c2, (int)x.ldz,
                       x.z, x.gmax, x.gs, x.gu);
    return hipGetLastError();
  };
  if (sh.n <= 16) return run(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  if (sh.n <= 32) return run(std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
  if (sizeof(T) == 4 || sh.n <= 64) return run(std::integral_constant<int, 2>{}, std::integral_constant<int, 64>{});
  return run(std::integral_constant<int, sizeof(T) == 4 ? 2 : 4>{}, std::integral_constant<int, sizeof(T) == 4 ? 64 : 128>{});
}
hipError_t few_logits(const ScoreHead& h, const ScoreShape& sh, const Scratch& x, float c2, hipStream_t st) {
  if (h.f32) return run_few(static_cast<const float*>(h.hidden), h.h32.q4, h.h32.w, h.h32.wq, h.h32.sc, h.h32.bi, sh, x, c2, st);
  return run_few(static_cast<const bf16_t*>(h.hidden), h.h.q4, h.h.w, h.h.wq, h.h.sc, h.h.bi, sh, x, c2, st);
}

// A 4-bit head's rows in fp32 (its group size divides the words of a thread's row).
__global__ __launch_bounds__(256) void dequant32_kernel(const uint32_t* __restrict__ Wq, const float* __restrict__ Sc,
                                                        const float* __restrict__ Bi, long words, float* __restrict__ out) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= words) return;
  const uint32_t q = Wq[i];
  const float s = Sc[i >> 3], b = Bi[i >> 3];
  f32x4 x[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = __builtin_fmaf(s, (float)((q >> (4 * e)) & 15u), b);
  reinterpret_cast<f32x4*>(out)[2 * i] = x[0];
  reinterpret_cast<f32x4*>(out)[2 * i + 1] = x[1];
}

// The head that the product takes: an fp32 4-bit one with a stage is dequantized into it first.
hipError_t staged_head(ScoreHead& h, const ScoreShape& sh, const Scratch& x, hipStream_t st) {
  if (x.stage32 == nullptr) return hipSuccess;
  const hipError_t e = launch_dequant32(h.h32, sh.v, sh.d, x.stage32, st);
  h.h32 = LceHead32{0, x.stage32, nullptr, nullptr, nullptr};
  return e;
}

RowParts row_parts(const Scratch& x, const ScoreHead& h, long n, long v, float c2) {
  if (x.few) return RowParts{x.gmax, x.gs, x.gu, x.groups, 1, x.groups, c2};
  const int ns = h.f32 ? lce32_fwd_nsplit(n, v) : lce_fwd_nsplit(n, v);
  return RowParts{x.m, x.s, x.u ? x.u : x.s, ns, n, 1, 1.f};
}

// The product over rows [r0, r0 + n) with its statistics; k columns a row to picks.
hipError_t tile_stats(const ScoreHead& h, const ScoreShape& sh, const Scratch& x, long r0, long n, float c2, int k, float* picks,
                      hipStream_t st) {
  const ScoreStats stats{c2, x.m, x.s, x.u, x.gmax, x.ldg, x.kept ? x.z : nullptr, x.ldz, ScoreList{k ? x.column : nullptr, picks, k}};
  if (h.f32)
    return launch_lce32_stats(h.h32, static_cast<const float*>(h.hidden) + r0 * sh.d, (int)n, (int)sh.d, (int)sh.v, stats, st);
  return launch_lce_stats(h.h, static_cast<const bf16_t*>(h.hidden) + r0 * sh.d, (int)n, (int)sh.d, (int)sh.v, stats, x.stage,
                          x.stage_rows, st);
}

hipError_t gather(const ScoreHead& h, const ScoreShape& sh, const Scratch& x, long r0, hipStream_t st) {
  const GatherPlan plan{x.entries, x.tiles, x.max_tiles, x.cand};
  if (h.f32) return launch_lce32_gather(h.h32, static_cast<const float*>(h.hidden) + r0 * sh.d, (int)sh.d, (int)sh.v, plan, st);
  return launch_lce_gather(h.h, static_cast<const bf16_t*>(h.hidden) + r0 * sh.d, (int)sh.d, (int)sh.v, plan, st);
}

}  // namespace

hipError_t launch_lce_gather(const LceHead& h, const bf16_t* H, int D, int V, const GatherPlan& p, hipStream_t st) {
  hipLaunchKernelGGL(h.q4 ? lce_gather_kernel<1> : lce_gather_kernel<0>, dim3(p.max_tiles), dim3(256), 0, st, H, h.w, h.wq, h.sc,
                     h.bi, D, V, p);
  return hipGetLastError();
}

// Any address of a caller's logits: whether there are some is all that the sizes depend on.
float* some_logits(int keep) { return keep ? reinterpret_cast<float*>(16) : nullptr; }
size_t logprobs_fwd_workspace(const ScoreShape& sh, int f32, int q4, int top, int keep) {
  size_t bytes;
  carve(sh, f32, q4, top, 0, some_logits(keep), nullptr, &bytes);
  return bytes;
}

hipError_t launch_dequant32(const LceHead32& h, long V, long D, float* out, hipStream_t st) {
  const long words = V * D / 8;
  hipLaunchKernelGGL(dequant32_kernel, dim3((unsigned)ceil_div(words, 256)), dim3(256), 0, st, h.wq, h.sc, h.bi, words, out);
  return hipGetLastError();
}

hipError_t launch_logprobs_fwd(const ScoreHead& head, const ScoreShape& sh, const int64_t* targets, long long ignore_index,
                               int top, const LogprobsOut& o, void* ws, hipStream_t st) {
  size_t bytes;
  ScoreHead h = head;
  const Scratch x = carve(sh, h.f32, h.f32 ? h.h32.q4 : h.h.q4, top, 0, o.logits, ws, &bytes);
  const float c2 = sh.c2;
  const int V = (int)sh.v;
  const hipError_t staged = staged_head(h, sh, x, st);
  if (staged != hipSuccess) return staged;
  for (long r0 = 0; r0 < sh.n; r0 += x.rows) {  // (few tokens, or a caller's logits: one pass)
    const long n = sh.n - r0 < x.rows ? sh.n - r0 : x.rows;
    const LogprobsOut out{o.logprobs ? o.logprobs + r0 : nullptr, o.entropy + r0, top ? o.top_logprobs + r0 * top : nullptr,
                          top ? o.top_ids + r0 * top : nullptr, o.lse + r0, o.tgt ? o.tgt + r0 : nullptr};
    const int64_t* y = targets ? targets + r0 : nullptr;
    if (x.kept) {
      const hipError_t e = x.few ? few_logits(h, sh, x, c2, st) : tile_stats(h, sh, x, r0, n, c2, 0, nullptr, st);
      if (e != hipSuccess) return e;
      auto kernel = !top ? score_rows_kernel<true, 0, 0>
                    : x.take <= 16 && x.groups <= 2048 ? score_rows_kernel<true, 2048, 2048>
                    : x.take <= 64 && x.groups <= 2048 ? score_rows_kernel<true, 2048, 64 * kGroup>
                                                       : score_rows_kernel<true, kMaxGroups, kScoreTop * kGroup>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(kPick), 0, st, row_parts(x, h, n, sh.v, c2), x.gmax, x.groups, x.ldg, x.z,
                         x.ldz, y, ignore_index, V, c2, top, x.take, out, nullptr, nullptr, nullptr, nullptr);
      MTP_LAUNCHED();
      continue;
    }
    hipError_t e;
    if (y) {
      hipLaunchKernelGGL(target_columns_kernel, dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, st, y, ignore_index, n, sh.v, x.column);
      MTP_LAUNCHED();
    }
    e = tile_stats(h, sh, x, r0, n, c2, y ? 1 : 0, out.tgt, st);
    if (e != hipSuccess) return e;
    if (top) {
      hipLaunchKernelGGL(zero_counts_kernel, dim3((unsigned)ceil_div(x.groups, 256)), dim3(256), 0, st, x.counts, x.groups);
      MTP_LAUNCHED();
    }
    auto rows = !top ? score_rows_kernel<false, 0, 0>
                     : x.groups <= 2048 ? score_rows_kernel<false, 2048, 0> : score_rows_kernel<false, kMaxGroups, 0>;
    hipLaunchKernelGGL(rows, dim3((unsigned)n), dim3(kPick), 0, st, row_parts(x, h, n, sh.v, c2), x.gmax, x.groups, x.ldg, nullptr, 0L, y,
                       ignore_index, V, c2, top, x.take, out, x.chosen, x.counts, x.floors, x.norms);
    MTP_LAUNCHED();
    if (!top) continue;
    hipLaunchKernelGGL(gather_tiles_kernel, dim3(1), dim3(1024), 0, st, x.counts, x.groups, x.tiles, x.max_tiles);
    MTP_LAUNCHED();
    hipLaunchKernelGGL(gather_groups_kernel, dim3((unsigned)ceil_div(n * x.take, 256)), dim3(256), 0, st, x.chosen, n * x.take,
                       x.take, x.counts, x.entries);
    MTP_LAUNCHED();
    e = gather(h, sh, x, r0, st);
    if (e != hipSuccess) return e;
    auto best = x.take <= 16 ? score_top_kernel<16 * kGroup> : x.take <= 64 ? score_top_kernel<64 * kGroup> : score_top_kernel<kScoreTop * kGroup>;
    hipLaunchKernelGGL(best, dim3((unsigned)n), dim3(kPick), 0, st, x.cand, x.chosen, x.floors, x.norms, y, V, c2, top, x.take, out);
    MTP_LAUNCHED();
  }
  return hipSuccess;
}

size_t distill_fwd_workspace(const ScoreShape& sh, int f32, int q4, int k, int keep) {
  size_t bytes;
  carve(sh, f32, q4, 0, k, some_logits(keep), nullptr, &bytes);
  return bytes;
}

hipError_t launch_distill_fwd(const ScoreHead& head, const ScoreShape& sh, const int64_t* ids, const float* teacher,
                              const uint8_t* mask, const DistillLoss& p, const DistillOut& o, void* ws, hipStream_t st) {
  size_t bytes;
  ScoreHead h = head;
  const Scratch x = carve(sh, h.f32, h.f32 ? h.h32.q4 : h.h.q4, 0, p.k, o.logits, ws, &bytes);
  const float c2 = sh.c2;
  const hipError_t staged = staged_head(h, sh, x, st);
  if (staged != hipSuccess) return staged;
  float* row_loss = p.reduction == kReduceNone ? o.loss : x.row_loss;
  auto rows = [&](auto few) {
    constexpr bool FEW = decltype(few)::value;
    return p.kind == kDistillForward ? distill_rows_kernel<kDistillForward, FEW>
           : p.kind == kDistillReverse ? distill_rows_kernel<kDistillReverse, FEW> : distill_rows_kernel<kDistillJsd, FEW>;
  };
  auto kernel = x.few ? rows(std::true_type{}) : rows(std::false_type{});
  for (long r0 = 0; r0 < sh.n; r0 += x.rows) {  // (kept: one pass)
    const long n = sh.n - r0 < x.rows ? sh.n - r0 : x.rows;
    const int64_t* id = ids + r0 * p.k;
    const float* lp = teacher + r0 * p.k;
    const uint8_t* see = mask ? mask + r0 : nullptr;
    if (!x.few) {
      hipLaunchKernelGGL(sort_lists_kernel, dim3((unsigned)ceil_div(n, 4)), dim3(256), 0, st, id, lp, see, n, sh.v, p.k, x.column,
                         x.slot);
      MTP_LAUNCHED();
    }
    const hipError_t e = x.few ? few_logits(h, sh, x, c2, st) : tile_stats(h, sh, x, r0, n, c2, p.k, x.picks, st);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(n, 4)), dim3(256), 0, st, row_parts(x, h, n, sh.v, c2), x.column,
                       x.slot, x.picks, x.z, x.ldz, id, lp, see, n, sh.v, c2, p.inv_t, p.k, p.renormalize, p.beta, row_loss + r0,
                       x.row_counts + r0, o.lse + r0, o.rest + r0, o.coef + r0 * p.k, o.columns + r0 * p.k);
    MTP_LAUNCHED();
  }
  if (p.reduction == kReduceNone) return hipSuccess;
  hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), dim3(1024), 0, st, row_loss, x.row_counts, sh.n, p.reduction == kReduceMean,
                     o.loss, o.scale);
  return hipGetLastError();
}

hipError_t launch_logprobs_coef(const float* d_logprobs, const float* d_entropy, const int64_t* targets, long long ignore_index,
                                const float* lse, const float* entropy, const float* tgt, long n, long v, float inv_t,
                                float* alpha, float* beta, int* columns, float* value, hipStream_t st) {
  hipLaunchKernelGGL(logprobs_coef_kernel, dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, st, d_logprobs, d_entropy, targets,
                     ignore_index, lse, entropy, tgt, n, v, inv_t, alpha, beta, columns, value);
  return hipGetLastError();
}

template <class G>
hipError_t affine_tiles(const AffineGrad& a, const float* lse, long n, int v_begin, int vlim, int cols, long ldg, G* g, hipStream_t st) {
  const int each = 16 / (int)sizeof(G);
  for (long r0 = 0; r0 < n; r0 += 32768) {  // blockIdx.y
    const long rows = n - r0 < 32768 ? n - r0 : 32768;
    AffineRows r = a.rows;
    r.alpha += r0;
    if (r.beta) r.beta += r0;
    hipLaunchKernelGGL(affine_tiles_kernel<G>, dim3((unsigned)ceil_div(cols, 256 * each), (unsigned)rows), dim3(256), 0, st, a.z + r0 * a.ldz,
                       a.ldz, lse + r0, r, v_begin, vlim, cols, ldg, g + r0 * ldg, a.halves ? g + (n + r0) * ldg : nullptr);
    MTP_LAUNCHED();
  }
  return hipSuccess;
}
hipError_t launch_affine_tiles(const AffineGrad& a, const float* lse, long n, int v_begin, int vlim, int cols, long ldg, bf16_t* g,
                               hipStream_t st) {
  return affine_tiles(a, lse, n, v_begin, vlim, cols, ldg, g, st);
}
hipError_t launch_affine_tiles(const AffineGrad& a, const float* lse, long n, int v_begin, int vlim, int cols, long ldg, float* g,
                               hipStream_t st) {
  return affine_tiles(a, lse, n, v_begin, vlim, cols, ldg, g, st);
}

hipError_t launch_distill_coef(const float* d_loss, int per_row, const float* scale, const float* rest, const float* coef, long n,
                               int k, float* alpha, float* value, hipStream_t st) {
  hipLaunchKernelGGL(distill_coef_kernel, dim3((unsigned)ceil_div(n * k, 256)), dim3(256), 0, st, d_loss, per_row, scale, rest,
                     coef, n, k, alpha, value);
  return hipGetLastError();
}

hipError_t launch_join_halves(const float* halves, long count, bf16_t* dH, hipStream_t st) {
  hipLaunchKernelGGL(join_halves_kernel, dim3((unsigned)ceil_div(count, 256)), dim3(256), 0, st, halves, count, dH);
  return hipGetLastError();
}

hipError_t launch_clean_rows(const void* hidden, const float* alpha, const float* beta, long n, long row_bytes, int copies, void* out,
                             hipStream_t st) {
  hipLaunchKernelGGL(clean_rows_kernel, dim3((unsigned)n), dim3(256), 0, st, static_cast<const uint32_t*>(hidden), alpha, beta,
                     row_bytes / 4, copies, static_cast<uint32_t*>(out));
  return hipGetLastError();
}

}  // namespace mtp

// Attention with capped scores, a bias by distance and key spans: the plan of a call, and the work orders and key
// ranges that a span backward needs. The kernels are attn_core.hpp's.
#include "attn_scored.hpp"

namespace mtp {

// Workgroup 0 orders the B npb query blocks of the dQ pass (P queries each), workgroup 1 the B nkb 128-key blocks of
// the dK/dV pass, most tiles first; the others fill, for each key, the queries [col_begin, col_end) that see it. Costs are
// looked up twice by the sort, so the first kSchedCosts are kept: 7.3 us at 8192 positions (12.9 with the two searches one
// after the other and the costs searched twice), 5.0 for 4 x 509.
constexpr int kSchedCosts = 4096;
__global__ __launch_bounds__(1024) void attn_span_sched_kernel(const int32_t* __restrict__ start, const int32_t* __restrict__ end,
                                                              int B, int S, int P, int32_t* __restrict__ q_order,
                                                              int32_t* __restrict__ kv_order, int32_t* __restrict__ col_begin,
                                                              int32_t* __restrict__ col_end) {
  if (blockIdx.x >= 2) {
    const long i = (long)(blockIdx.x - 2) * 1024 + threadIdx.x;
    if (i < (long)B * S) {
      const int b = (int)(i / S), pos = (int)(i % S);
      int qb, qe;
      queries_of(start + (long)b * S, end + (long)b * S, S, pos, pos, qb, qe);
      col_begin[i] = qb;
      col_end[i] = qe;
    }
    return;
  }
  __shared__ int kept[kSchedCosts];
  const bool kv = blockIdx.x == 1;
  const int nblk = kv ? (S + 127) / 128 : (S + P - 1) / P, n = B * nblk;
  const int shift = sched_shift(S);
  auto tiles = [&](int from, int to) { return to > from ? (to - from / kKT * kKT + kKT - 1) / kKT : 0; };
  auto in_row = [&](int x) { return x < 0 ? 0 : x < S ? x : S; };
  auto cost = [&](int i) {
    const int b = i / nblk, blk = i % nblk;
    const int32_t *sst = start + (long)b * S, *snd = end + (long)b * S;
    if (kv) {
      const int k0 = blk * 128, klast = (k0 + 127 < S) ? k0 + 127 : S - 1;
      int qb, qe;
      queries_of(sst, snd, S, k0, klast, qb, qe);
      return tiles(qb, qe) >> shift;
    }
    const int q0 = blk * P, q1 = (q0 + P < S) ? q0 + P : S;
    return tiles(in_row(sst[q0]), in_row(snd[q1 - 1])) >> shift;
  };
  for (int i = threadIdx.x; i < n && i < kSchedCosts; i += 1024) kept[i] = cost(i);
  __syncthreads();
  sched_sort(n, [&](int i) { return i < kSchedCosts ? kept[i] : cost(i); }, kv ? kv_order : q_order);
}

namespace {
size_t round256(size_t x) { return (x + 255) / 256 * 256; }
// Heads of a forward or dQ workgroup's group, and its query positions.
int wg_heads(int hq, int hkv) {
  const int G = hq / hkv;
  return (G % 4 == 0) ? 4 : ((G % 2 == 0) ? 2 : 1);
}
int wg_rows(int hq, int hkv) { return 32 * (4 / wg_heads(hq, hkv)); }
int q_grid(const AttnShape& sh) {
  const int P = wg_rows(sh.hq, sh.hkv);
  return (sh.s + P - 1) / P * sh.b * (sh.hq / wg_heads(sh.hq, sh.hkv));
}
// Splits of the dK/dV pass: as many as the plain kernels' table has (for spans, whose layout is on the device, the causal
// mask's), but a split of a key block has at least 2 of its (head, query tile) items where all workgroups run at once, and
// 16 where they take turns: below that its start and the sum of the parts outweigh the shorter walk. A whole step, split
// 8, 4, 2 and 1 times: 4 x 16/4 x 509 x 128 89, 79, 90 and 113 us (4 taken); 2 x 8/8 x 700 x 64 71, 60, 59 and 60 (2);
// 2 x 8/2 x 300 x 128 59, 62, 70 and 86 (8); 1 x 16/8 x 4000 x 128 400 split twice, 472 not at all (2).
int scored_nsplit(int b, int hq, int hkv, int s, int dh, int causal) {
  int ns = attn_dkv_nsplit(b, hq, hkv, s, dh, causal);
  const long wgs = (long)(s + 127) / 128 * b * hkv, items = (long)hq / hkv * ((s + 63) / 64);
  while (ns > 1 && items < ns * (wgs * ns <= kNumCU + kNumCU / 4 ? 2 : 16)) ns /= 2;
  return ns;
}
// Splits of the forward and dQ passes over the keys (1: none): as many as give every CU a workgroup with four tiles of the
// longest walk, or both its places one with eight (spans, whose walks are mostly shorter: sixteen). GPU time of a step,
// unsplit, for one workgroup a CU and for two: 1 x 2/1 x 2932 x 128 211, 106 and 106 us; 1 x 4/1 x 4000 x 64 226, 159 and
// 132; 4 x 16/8 x 509 x 64 (256 workgroups) 61, 61 and 72; windows of 500 in 2 x 4/4 x 4000 x 64 83, 83 and 93, prefixes 197,
// 197 and 163.
int q_splits(int b, int hq, int hkv, int s, bool span) {
  const AttnShape sh{b, hq, hkv, s, 0, 0.f, 0};
  const int wgs = q_grid(sh), tiles = (s + kKT - 1) / kKT;
  auto least = [](int x, int y) { return x < y ? x : y; };
  const int one = least(kNumCU / wgs, tiles / 4), two = least(2 * kNumCU / wgs, tiles / (span ? 16 : 8));
  const int ns = one > two ? one : two;
  return ns < 1 ? 1 : ns > 8 ? 8 : ns;
}
size_t fwd_part_bytes(int b, int hq, int s, int dh, int ns) { return ns > 1 ? (size_t)ns * b * hq * s * (dh + 4) * 4 : 0; }

// O, its bits below bf16 and L from the parts of a split forward: with M the largest maximum,
// O = sum 2^(m - M) O_part / sum 2^(m - M) lr_part. Eight values of a row a thread.
__global__ __launch_bounds__(256) void attn_join_kernel(const float* __restrict__ part, int ns, long rows, int dh, int span,
                                                        bf16_t* __restrict__ o, int8_t* __restrict__ o_low,
                                                        float* __restrict__ lse) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 8, row = e / dh;
  if (row >= rows) return;
  const f32x4* ml = reinterpret_cast<const f32x4*>(part + ns * rows * dh);
  float top = kNegInf, l = 0.f, lr = 0.f;
  for (int sp = 0; sp < ns; ++sp) top = fmaxf(top, ml[sp * rows + row][0]);
  const float base = top == kNegInf ? 0.f : top;
  f32x4 x[2] = {};
  for (int sp = 0; sp < ns; ++sp) {
    const f32x4 v = ml[sp * rows + row];
    const float w = fast_exp2(v[0] - base);  // a part without keys: 2^-inf
    l += w * v[1];
    lr += w * v[2];
    const f32x4* p = reinterpret_cast<const f32x4*>(part + sp * rows * dh + e);
    x[0] += w * p[0];
    x[1] += w * p[1];
  }
  const float mul = lr > 0.f ? 1.f / lr : 0.f;
  u32x4 hi;
  uint32_t low[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = x[j >> 1][2 * (j & 1)] * mul, c = x[j >> 1][2 * (j & 1) + 1] * mul;
    hi[j] = pack_bf16x2(a, c);
    low[j >> 1] |= (below_bf16(a, hi[j] << 16) | below_bf16(c, hi[j] & 0xffff0000u) << 8) << (16 * (j & 1));
  }
  *reinterpret_cast<u32x4*>(o + e) = hi;
  if (o_low) *reinterpret_cast<u32x2*>(o_low + e) = u32x2{low[0], low[1]};
  if (e % dh == 0) lse[row] = l > 0.f ? (top + fast_log2(l)) * kLn2 : span ? -kNegInf : kNegInf;
}
// dQ = the sum of the parts of a split pass, in order.
__global__ __launch_bounds__(256) void attn_dq_sum_kernel(const float* __restrict__ part, int ns, long plane, bf16_t* __restrict__ dq) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= plane) return;
  f32x4 x[2] = {};
  for (int sp = 0; sp < ns; ++sp) {
    const f32x4* p = reinterpret_cast<const f32x4*>(part + sp * plane + e);
    x[0] += p[0];
    x[1] += p[1];
  }
  *reinterpret_cast<u32x4*>(dq + e) = u32x4{pack_bf16x2(x[0][0], x[0][1]), pack_bf16x2(x[0][2], x[0][3]),
                                            pack_bf16x2(x[1][0], x[1][1]), pack_bf16x2(x[1][2], x[1][3])};
}
dim3 eights_grid(long values) { return dim3((unsigned)((values / 8 + 255) / 256)); }

// Whether the workgroups of a span backward's passes take turns, so that their order counts.
bool ordered(int b, int hq, int hkv, int s, int dh) {
  const AttnShape sh{b, hq, hkv, s, dh, 0.f, 0};
  return q_grid(sh) > 2 * kNumCU || (long)(s + 127) / 128 * b * hkv * scored_nsplit(b, hq, hkv, s, dh, 1) > kNumCU;
}
struct Carver {
  char* base;  // null: sizes alone
  size_t at = 0;
  template <class T>
  void take(T*& p, size_t n) {
    p = reinterpret_cast<T*>(base + at);
    at += round256(n * sizeof(T));
  }
};
// What spans add to a backward: its work orders and the queries that see each key.
void carve_plan(Carver& c, int b, int hq, int hkv, int s, ScoredWorkspace* ws) {
  const int P = wg_rows(hq, hkv);
  c.take(ws->q_order, (size_t)b * ((s + P - 1) / P));
  c.take(ws->kv_order, (size_t)b * ((s + 127) / 128));
  c.take(ws->col_begin, (size_t)b * s);
  c.take(ws->col_end, (size_t)b * s);
}
// The parts of a workspace from `base`, with room for the larger split of the two masks; returns the bytes.
size_t carve(int b, int hq, int hkv, int s, int dh, char* base, ScoredWorkspace* ws) {
  const int ns1 = scored_nsplit(b, hq, hkv, s, dh, 1), ns0 = scored_nsplit(b, hq, hkv, s, dh, 0);
  const int ns = ns1 > ns0 ? ns1 : ns0;
  Carver c{base};
  c.take(ws->dvec, (size_t)3 * b * hq * s);
  const int nq = q_splits(b, hq, hkv, s, false);  // (spans: no more)
  const size_t kv_part = ns > 1 ? (size_t)ns * 2 * b * hkv * s * dh : 0, q_part = nq > 1 ? (size_t)nq * b * hq * s * dh : 0;
  c.take(ws->part, kv_part > q_part ? kv_part : q_part);
  carve_plan(c, b, hq, hkv, s, ws);
  return c.at;
}
hipError_t launch_sched(const AttnShape& sh, const AttnScore& sc, const ScoredWorkspace& ws, hipStream_t st) {
  const unsigned fill = (unsigned)(((long)sh.b * sh.s + 1023) / 1024);
  hipLaunchKernelGGL(attn_span_sched_kernel, dim3(2 + fill), dim3(1024), 0, st, sc.start, sc.end, sh.b, sh.s,
                     wg_rows(sh.hq, sh.hkv), ws.q_order, ws.kv_order, ws.col_begin, ws.col_end);
  return hipGetLastError();
}
}  // namespace

size_t attn_scored_bwd_workspace(int b, int hq, int hkv, int s, int dh) {
  ScoredWorkspace ws;
  return carve(b, hq, hkv, s, dh, nullptr, &ws);
}

size_t attn_scored_fwd_workspace(int b, int hq, int hkv, int s, int dh) {
  return fwd_part_bytes(b, hq, s, dh, q_splits(b, hq, hkv, s, false));
}
hipError_t launch_attn_dq_sum(const float* part, int ns, long plane, bf16_t* dq, hipStream_t st) {
  hipLaunchKernelGGL(attn_dq_sum_kernel, eights_grid(plane), dim3(256), 0, st, part, ns, plane, dq);
  return hipGetLastError();
}

size_t attn_scored_plan(int b, int hq, int hkv, int s, int dh) {
  if (!ordered(b, hq, hkv, s, dh)) return 0;
  ScoredWorkspace ws;
  Carver c{nullptr};
  carve_plan(c, b, hq, hkv, s, &ws);
  return c.at;
}

hipError_t launch_attn_scored_fwd(const AttnShape& sh, const AttnScore& sc, const bf16_t* q, const bf16_t* k,
                                  const bf16_t* v, bf16_t* o, int8_t* o_low, int32_t* plan, float* lse,
                                  void* workspace, size_t bytes, hipStream_t st) {
  // The forward of a training step makes the backward's plan, and goes by its order of query blocks too (documents of 64
  // to 2048 in 8192 positions, 16/4 heads, head_dim 128: 62 against 76 us).
  const int32_t* order = nullptr;
  if (plan && sc.start && ordered(sh.b, sh.hq, sh.hkv, sh.s, sh.dh)) {
    ScoredWorkspace ws;
    Carver c{reinterpret_cast<char*>(plan)};
    carve_plan(c, sh.b, sh.hq, sh.hkv, sh.s, &ws);
    const hipError_t e = launch_sched(sh, sc, ws, st);
    if (e != hipSuccess) return e;
    order = ws.q_order;
  }
  int ns = q_splits(sh.b, sh.hq, sh.hkv, sh.s, sc.start != nullptr);
  if (!workspace || bytes < fwd_part_bytes(sh.b, sh.hq, sh.s, sh.dh, ns)) ns = 1;
  float* part = static_cast<float*>(workspace);
  hipError_t e = hipErrorInvalidValue;
  switch (sh.dh) {
    case 64: e = scored_fwd<64>(sh, sc, q, k, v, o, o_low, order, lse, q_grid(sh), ns, part, st); break;
    case 96: e = scored_fwd<96>(sh, sc, q, k, v, o, o_low, order, lse, q_grid(sh), ns, part, st); break;
    case 128: e = scored_fwd<128>(sh, sc, q, k, v, o, o_low, order, lse, q_grid(sh), ns, part, st); break;
    default: break;
  }
  if (e != hipSuccess || ns == 1) return e;
  const long rows = (long)sh.b * sh.hq * sh.s;
  hipLaunchKernelGGL(attn_join_kernel, eights_grid(rows * sh.dh), dim3(256), 0, st, part, ns, rows, sh.dh, sc.start != nullptr,
                     o, o_low, lse);
  return hipGetLastError();
}

hipError_t launch_attn_scored_bwd(const AttnShape& sh, const AttnScore& sc, const bf16_t* q, const bf16_t* k,
                                  const bf16_t* v, const bf16_t* o, const int8_t* o_low, const int32_t* plan,
                                  const float* lse, const bf16_t* d_o, bf16_t* dq, bf16_t* dk, bf16_t* dv, void* workspace,
                                  hipStream_t st) {
  ScoredWorkspace ws;
  carve(sh.b, sh.hq, sh.hkv, sh.s, sh.dh, static_cast<char*>(workspace), &ws);
  ws.nsplit = scored_nsplit(sh.b, sh.hq, sh.hkv, sh.s, sh.dh, sc.start ? 1 : sh.causal);
  ws.nq = q_splits(sh.b, sh.hq, sh.hkv, sh.s, sc.start != nullptr);
  hipError_t e = hipSuccess;
  // Where all workgroups of both passes run at once their order is of no account, and the dQ pass fills the key ranges
  // that the dK/dV pass reads: a launch less (a step of 4 x 16/8 x 509 x 64: 63.2 against
  // 67.5 us of GPU time, 1 x 8/8 x 100 x 128 37.0 against 41.2).
  if (sc.start && !ordered(sh.b, sh.hq, sh.hkv, sh.s, sh.dh)) {
    ws.q_order = ws.kv_order = nullptr;
  } else if (sc.start && plan) {
    Carver c{reinterpret_cast<char*>(const_cast<int32_t*>(plan))};
    carve_plan(c, sh.b, sh.hq, sh.hkv, sh.s, &ws);
  } else if (sc.start) {
    e = launch_sched(sh, sc, ws, st);
    if (e != hipSuccess) return e;
  }
  switch (sh.dh) {
    case 64: e = scored_bwd<64>(sh, sc, ws, q, k, v, o, o_low, lse, d_o, dq, dk, dv, q_grid(sh), st); break;
    case 96: e = scored_bwd<96>(sh, sc, ws, q, k, v, o, o_low, lse, d_o, dq, dk, dv, q_grid(sh), st); break;
    case 128: e = scored_bwd<128>(sh, sc, ws, q, k, v, o, o_low, lse, d_o, dq, dk, dv, q_grid(sh), st); break;
    default: return hipErrorInvalidValue;
  }
  if (e != hipSuccess || ws.nsplit == 1) return e;
  return launch_attn_dkv_reduce(ws.part, ws.nsplit, (long)sh.b * sh.hkv * sh.s * sh.dh, dk, dv, st);
}

}  // namespace mtp

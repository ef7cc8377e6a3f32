// Plain and packed attention: launchers over the kernels of attn_core.hpp, the packed backward's work orders, and
// the sum of split dK/dV passes.
#include "attn_core.hpp"

namespace mtp {

// dK, dV = the sum of the nsplit fp32 partials of the split dK/dV kernel, rounded to bf16 once. Each
// thread sums 8 consecutive elements of one plane (blockIdx.y: 0 dK, 1 dV) over the splits in split
// order, so the result does not depend on scheduling. plane (B Hkv S DH) is a multiple of 8.
__global__ __launch_bounds__(256) void attn_dkv_reduce_kernel(const float* __restrict__ part, int nsplit, long plane,
                                                              bf16_t* __restrict__ dk, bf16_t* __restrict__ dv) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  const int which = blockIdx.y;
  if (e >= plane) return;
  float acc[8] = {};
  for (int sp = 0; sp < nsplit; ++sp) {
    const float* src = part + (2L * sp + which) * plane + e;
    const f32x4 a = *reinterpret_cast<const f32x4*>(src);
    const f32x4 b = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      acc[u] += a[u];
      acc[4 + u] += b[u];
    }
  }
  bf16_t* dst = (which ? dv : dk) + e;
  *reinterpret_cast<u32x4*>(dst) = u32x4{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]),
                                          pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7])};
}

// ------------------------------------------------------------------------------------------
// Launchers
// ------------------------------------------------------------------------------------------
// Work items of the dK/dV kernels (every head_dim): one per (query head of the group, 64-query tile)
// seen by a 128-key block. Under the causal mask key block kb sees the tiles from 128 kb on, so
// block 0 holds the most; without it every block holds ceil(S / 64). The kernel runs one 8-wave
// workgroup per CU. When the heaviest block holds more than ~1.15x a CU's share of all items, or
// there are fewer blocks than CUs, the CUs given light blocks idle while the heaviest runs: the
// block's items are then split over nsplit workgroups (1, 2, 4 or 8: the smallest that brings the
// heaviest workgroup under the share), whose fp32 partials attn_dkv_reduce_kernel sums. At B = 1,
// Hkv = 8 causal this gives 8 splits at S <= 1024, 4 at 2048, 2 at 4096 and 1 from 8192 on.
// Longest-first work orders of a packed backward, one workgroup per order. Workgroup 0 orders the
// B npb query blocks of the dQ pass (P queries each), workgroup 1 the B nkb 128-key blocks of the
// dK/dV pass, by the tile counts their kernels' loops run (from seg_start, exactly as the kernels
// bound them); order[r] is the item of rank r, most tiles first. A counting sort over kSchedBuckets
// buckets of cost >> shift; items of one bucket land in any order, which changes only the schedule:
// every item writes its own outputs.
// Workgroups 2 and up fill seg_end[b][i], the first position after i's segment (the first j > i with
// seg_start[j] > i, S if none), which the dK/dV pass reads instead of searching seg_start per key.
__global__ __launch_bounds__(1024) void attn_sched_kernel(const int32_t* __restrict__ seg_start, int B, int S, int P,
                                                         int32_t* __restrict__ q_order, int32_t* __restrict__ kv_order,
                                                         int32_t* __restrict__ seg_end) {
  if (blockIdx.x >= 2) {
    const long i = (long)(blockIdx.x - 2) * 1024 + threadIdx.x;
    if (i < (long)B * S) {
      const int b = (int)(i / S), pos = (int)(i % S);
      seg_end[i] = first_above(seg_start + (long)b * S, pos, S, pos);
    }
    return;
  }
  const bool kv = blockIdx.x == 1;
  const int nblk = kv ? (S + 127) / 128 : (S + P - 1) / P;
  const int n = B * nblk;
  int32_t* order = kv ? kv_order : q_order;
  const int shift = sched_shift(S);
  auto cost = [&](int i) {
    const int b = i / nblk, blk = i % nblk;
    const int32_t* sst = seg_start + (long)b * S;
    int c;
    if (kv) {
      const int k0 = blk * 128;
      const int klast = (k0 + 127 < S) ? k0 + 127 : S - 1;
      const int q_end = first_above(sst, 0, S, klast);
      const int q_begin = (k0 / kKT) * kKT;
      c = q_end > q_begin ? (q_end - q_begin + kKT - 1) / kKT : 0;
    } else {
      const int q0 = blk * P;
      const int q1 = (q0 + P < S) ? q0 + P : S;
      const int kv0 = (sst[q0] / kKT) * kKT;
      c = (q1 - kv0 + kKT - 1) / kKT;
    }
    return c >> shift;
  };
  sched_sort(n, cost, order);
}

int attn_dkv_nsplit(int b, int hq, int hkv, int s, int dh, int causal) {
  if (b < 1 || hkv < 1 || s < 1 || hq % hkv) return 1;
  const long G = hq / hkv;
  const long nkb = (s + 127) / 128;
  const long heaviest = G * ((s + 63) / 64);
  long total = 0;
  for (long kb = 0; kb < nkb; ++kb) total += G * (causal ? (s - 128 * kb + 63) / 64 : (s + 63) / 64);
  total *= (long)b * hkv;
  for (int ns = 1; ns < 8; ns *= 2)
    if (heaviest * kNumCU * 100 <= 115L * total * ns) return ns;
  return 8;
}

size_t attn_dvec_bytes(int b, int hq, int s) {
  // D (fp32 per query row), rounded up to 256 B so the partials that follow it stay aligned.
  return ((size_t)b * hq * s * sizeof(float) + 255) / 256 * 256;
}

namespace {
size_t round256(size_t x) { return (x + 255) / 256 * 256; }
int fwd_rows(int hq, int hkv) {  // query positions per forward / dQ workgroup
  const int G = hq / hkv;
  return 32 * (4 / ((G % 4 == 0) ? 4 : ((G % 2 == 0) ? 2 : 1)));
}
// Byte offset of the packed work orders: after D and the fp32 dK/dV partials of the larger split.
size_t attn_order_offset(int b, int hq, int hkv, int s, int dh) {
  const int ns1 = attn_dkv_nsplit(b, hq, hkv, s, dh, 1), ns0 = attn_dkv_nsplit(b, hq, hkv, s, dh, 0);
  const int ns = ns1 > ns0 ? ns1 : ns0;
  return attn_dvec_bytes(b, hq, s) + (ns > 1 ? (size_t)ns * 2 * (size_t)b * hkv * s * dh * sizeof(float) : 0);
}
}  // namespace

size_t attn_bwd_workspace(int b, int hq, int hkv, int s, int dh) {
  // D, the fp32 dK/dV partials when either mode splits (the larger split), the two work orders
  // of a packed backward (int32 per dQ query block and per dK/dV key block) and its segment ends
  // (int32 per position).
  const int P = fwd_rows(hq, hkv);
  return attn_order_offset(b, hq, hkv, s, dh) + round256((size_t)b * ((s + P - 1) / P) * 4) +
         round256((size_t)b * ((s + 127) / 128) * 4) + round256((size_t)b * s * 4);
}

namespace {
int fwd_grid(const AttnShape& sh) {
  const int G = sh.hq / sh.hkv;
  const int hpw = (G % 4 == 0) ? 4 : ((G % 2 == 0) ? 2 : 1);
  const int P = 32 * (4 / hpw);
  return ((sh.s + P - 1) / P) * sh.b * (sh.hq / hpw);
}

template <int DH>
hipError_t fwd_dh(const AttnShape& sh, const bf16_t* q, const bf16_t* k, const bf16_t* v, const int32_t* sid,
                  const int32_t* sst, bf16_t* o, float* lse, hipStream_t st) {
  const float sl2 = sh.scale * kLog2e;
  dim3 grid(fwd_grid(sh)), block(256);
  if (sid) hipLaunchKernelGGL((attn_kv_kernel<DH, kMaskPacked, false>), grid, block, 0, st, q, k, v, nullptr, nullptr, nullptr, nullptr, nullptr, sst, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sl2, sh.scale, sh.causal, nullptr, 0.f, nullptr, nullptr, nullptr, nullptr, 1, nullptr);
  else hipLaunchKernelGGL((attn_kv_kernel<DH, kMaskPlain, false>), grid, block, 0, st, q, k, v, nullptr, nullptr, nullptr, nullptr, nullptr, sst, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sl2, sh.scale, sh.causal, nullptr, 0.f, nullptr, nullptr, nullptr, nullptr, 1, nullptr);
  return hipGetLastError();
}

template <int DH>
hipError_t bwd_dh(const AttnShape& sh, const bf16_t* q, const bf16_t* k, const bf16_t* v, const bf16_t* o,
                  const float* lse, const bf16_t* d_o, const int32_t* sid, const int32_t* sst, bf16_t* dq,
                  bf16_t* dk, bf16_t* dv, float* dvec, hipStream_t st) {
  dim3 block(256);
  hipError_t e = hipSuccess;
  // Workspace: D (formed by the dQ pass for the dK/dV pass), the split dK/dV partials, and the
  // packed work orders.
  const float sl2 = sh.scale * kLog2e;
  char* ws = reinterpret_cast<char*>(dvec);
  int32_t* q_order = nullptr;
  int32_t* kv_order = nullptr;
  int32_t* seg_end = nullptr;
  if (sid) {
    const int P = fwd_rows(sh.hq, sh.hkv);
    q_order = reinterpret_cast<int32_t*>(ws + attn_order_offset(sh.b, sh.hq, sh.hkv, sh.s, DH));
    kv_order = q_order + round256((size_t)sh.b * ((sh.s + P - 1) / P) * 4) / 4;
    seg_end = kv_order + round256((size_t)sh.b * ((sh.s + 127) / 128) * 4) / 4;
    const unsigned nse = (unsigned)(((long)sh.b * sh.s + 1023) / 1024);
    hipLaunchKernelGGL(attn_sched_kernel, dim3(2 + nse), dim3(1024), 0, st, sst, sh.b, sh.s, P, q_order, kv_order,
                       seg_end);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  dim3 qgrid(fwd_grid(sh));
  if (sid) hipLaunchKernelGGL((attn_kv_kernel<DH, kMaskPacked, true>), qgrid, block, 0, st, q, k, v, d_o, o, lse, dvec, nullptr, sst, dq, nullptr, sh.b, sh.hq, sh.hkv, sh.s, sl2, sh.scale, sh.causal, q_order, 0.f, nullptr, nullptr, nullptr, nullptr, 1, nullptr);
  else hipLaunchKernelGGL((attn_kv_kernel<DH, kMaskPlain, true>), qgrid, block, 0, st, q, k, v, d_o, o, lse, dvec, nullptr, sst, dq, nullptr, sh.b, sh.hq, sh.hkv, sh.s, sl2, sh.scale, sh.causal, nullptr, 0.f, nullptr, nullptr, nullptr, nullptr, 1, nullptr);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  // Split key blocks write fp32 partials after the D vector in the workspace; the reduce sums them.
  const int ns = attn_dkv_nsplit(sh.b, sh.hq, sh.hkv, sh.s, DH, sh.causal);
  float* part = reinterpret_cast<float*>(ws + attn_dvec_bytes(sh.b, sh.hq, sh.s));
  dim3 sgrid(((sh.s + 127) / 128) * sh.b * sh.hkv * ns);
  if (sid) hipLaunchKernelGGL((attn_bwd_dkv_ab_kernel<DH, kMaskPacked>), sgrid, dim3(512), 0, st, q, k, v, d_o, lse, dvec, seg_end, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sl2, sh.scale, sh.causal, ns, part, kv_order, nullptr, 0.f, nullptr);
  else hipLaunchKernelGGL((attn_bwd_dkv_ab_kernel<DH, kMaskPlain>), sgrid, dim3(512), 0, st, q, k, v, d_o, lse, dvec, sst, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sl2, sh.scale, sh.causal, ns, part, nullptr, nullptr, 0.f, nullptr);
  e = hipGetLastError();
  if (e != hipSuccess || ns == 1) return e;
  const long plane = (long)sh.b * sh.hkv * sh.s * DH;
  dim3 rgrid((unsigned)((plane / 8 + 255) / 256), 2);
  hipLaunchKernelGGL(attn_dkv_reduce_kernel, rgrid, dim3(256), 0, st, part, ns, plane, dk, dv);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_attn_dkv_reduce(const float* part, int ns, long plane, bf16_t* dk, bf16_t* dv, hipStream_t st) {
  hipLaunchKernelGGL(attn_dkv_reduce_kernel, dim3((unsigned)((plane / 8 + 255) / 256), 2), dim3(256), 0, st, part, ns, plane, dk, dv);
  return hipGetLastError();
}

hipError_t launch_attn_fwd(const AttnShape& sh, const bf16_t* q, const bf16_t* k, const bf16_t* v,
                           const int32_t* seg_id, const int32_t* seg_start, bf16_t* o, float* lse,
                           hipStream_t stream) {
  switch (sh.dh) {
    case 64: return fwd_dh<64>(sh, q, k, v, seg_id, seg_start, o, lse, stream);
    case 96: return fwd_dh<96>(sh, q, k, v, seg_id, seg_start, o, lse, stream);
    case 128: return fwd_dh<128>(sh, q, k, v, seg_id, seg_start, o, lse, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_attn_bwd(const AttnShape& sh, const bf16_t* q, const bf16_t* k, const bf16_t* v,
                           const bf16_t* o, const float* lse, const bf16_t* d_o, const int32_t* seg_id,
                           const int32_t* seg_start, bf16_t* dq, bf16_t* dk, bf16_t* dv, float* dvec,
                           hipStream_t stream) {
  switch (sh.dh) {
    case 64: return bwd_dh<64>(sh, q, k, v, o, lse, d_o, seg_id, seg_start, dq, dk, dv, dvec, stream);
    case 96: return bwd_dh<96>(sh, q, k, v, o, lse, d_o, seg_id, seg_start, dq, dk, dv, dvec, stream);
    case 128: return bwd_dh<128>(sh, q, k, v, o, lse, d_o, seg_id, seg_start, dq, dk, dv, dvec, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mtp

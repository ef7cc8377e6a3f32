// fp32 attention with capped scores, a bias by distance and key spans: launches over the kernels of attn32_core.hpp.
#include <type_traits>

#include "attn32_core.hpp"

namespace mtp {
using namespace f32k;

namespace {
// f(MASK, MOD) of the call, as integral constants. A cap without slopes runs the form with both, slopes null.
template <class F>
hipError_t with_form(const AttnScore& sc, F&& f) {
  using std::integral_constant;
  auto mod = [&](auto mask) {
    if (sc.cap > 0.f) return f(mask, integral_constant<int, kModBoth>{});
    if (sc.slopes) return f(mask, integral_constant<int, kModSlope>{});
    if constexpr (decltype(mask)::value == kMaskSpan) return f(mask, integral_constant<int, kModNone>{});
    return hipErrorInvalidValue;
  };
  if (sc.start) return mod(integral_constant<int, kMaskSpan>{});
  return mod(integral_constant<int, kMaskPlain>{});
}

// The 256 bytes that a part of a workspace is padded to.
size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// Splits of the forward and dQ passes (1: none): as many as bring the workgroups of their pairs of query blocks to one a
// CU, each with four key tiles of the longest walk at least (8/2 heads x 1000 x 128, cap and slopes, 4 splits: forward
// 34 + 5 us with the join against 94, dQ 47 + 5 against 128; with 256 workgroups or more one pass leaves no CU idle).
int q_splits(int b, int hq, int hkv, int s) {
  const AttnShape sh{b, hq, hkv, s, 0, 0.f, 0};
  const int wgs = (int)grid32_q(sh).x, tiles = (s + kPos - 1) / kPos;
  int ns = kNumCU / wgs;
  if (ns > tiles / 4) ns = tiles / 4;
  return ns < 1 ? 1 : ns > 8 ? 8 : ns;
}

// O and L from the parts of a split forward: with M the largest maximum, O = sum 2^(m - M) O_part / sum 2^(m - M) l_part.
// Four values of a row a thread.
__global__ __launch_bounds__(256) void attn32_join_kernel(const float* __restrict__ part, int ns, long rows, int dh, int span,
                                                          float* __restrict__ o, float* __restrict__ lse) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 4, row = e / dh;
  if (row >= rows) return;
  const f32x2* ml = reinterpret_cast<const f32x2*>(part + ns * rows * dh);
  float top = kNegInf, l = 0.f;
  for (int sp = 0; sp < ns; ++sp) top = fmaxf(top, ml[sp * rows + row][0]);
  const float base = top == kNegInf ? 0.f : top;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int sp = 0; sp < ns; ++sp) {
    const f32x2 v = ml[sp * rows + row];
    const float w = fast_exp2(v[0] - base);  // a part without keys: 2^-inf
    l += w * v[1];
    x += w * *reinterpret_cast<const f32x4*>(part + sp * rows * dh + e);
  }
  *reinterpret_cast<f32x4*>(o + e) = x * (l > 0.f ? 1.f / l : 0.f);
  if (e % dh == 0) lse[row] = l > 0.f ? (top + fast_log2(l)) * kLn2 : span ? -kNegInf : kNegInf;
}
// dQ = the sum of the parts of a split pass, in order.
__global__ __launch_bounds__(256) void attn32_dq_sum_kernel(const float* __restrict__ part, int ns, long plane, float* __restrict__ dq) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= plane) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int sp = 0; sp < ns; ++sp) x += *reinterpret_cast<const f32x4*>(part + sp * plane + e);
  *reinterpret_cast<f32x4*>(dq + e) = x;
}

dim3 split_grid(const AttnShape& sh, int ns) { return dim3(grid32_q(sh).x * ns); }
dim3 quads_grid(long floats) { return dim3((unsigned)((floats / 4 + 255) / 256)); }

template <int DH>
hipError_t fwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k, const float* v, float* o,
               float* lse, float* part, int ns, hipStream_t st) {
  const hipError_t e = with_form(sc, [&](auto mask, auto mod) {
    hipLaunchKernelGGL((attn32_q_kernel<DH, decltype(mask)::value, false, decltype(mod)::value>), split_grid(sh, ns), dim3(512), 0,
                       st, q, k, v, nullptr, nullptr, nullptr, nullptr, sc.start, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sh.scale,
                       sh.causal, sc.end, sc.cap, sc.slopes, ns, part);
    return hipGetLastError();
  });
  if (e != hipSuccess || ns == 1) return e;
  const long rows = (long)sh.b * sh.hq * sh.s;
  hipLaunchKernelGGL(attn32_join_kernel, quads_grid(rows * DH), dim3(256), 0, st, part, ns, rows, DH, sc.start != nullptr, o, lse);
  return hipGetLastError();
}

template <int DH>
hipError_t bwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k, const float* v, const float* o,
               const float* lse, const float* d_o, float* dq, float* dk, float* dv, float* dvec, float* part, int nq, int ns,
               hipStream_t st) {
  hipError_t e = with_form(sc, [&](auto mask, auto mod) {
    constexpr int MASK = decltype(mask)::value, MOD = decltype(mod)::value;
    hipLaunchKernelGGL((attn32_q_kernel<DH, MASK, true, MOD>), split_grid(sh, nq), dim3(512), 0, st, q, k, v, d_o, o, lse, dvec,
                       sc.start, dq, nullptr, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, sc.end, sc.cap, sc.slopes, nq, part);
    hipError_t e1 = hipGetLastError();
    if (e1 == hipSuccess && nq > 1) {
      const long plane = (long)sh.b * sh.hq * sh.s * DH;
      hipLaunchKernelGGL(attn32_dq_sum_kernel, quads_grid(plane), dim3(256), 0, st, part, nq, plane, dq);
      e1 = hipGetLastError();
    }
    if (e1 != hipSuccess) return e1;
    // (the parts of dQ are read: those of dK and dV take their place)
    hipLaunchKernelGGL((attn32_dkv_kernel<DH, MASK, MOD>), dim3(((sh.s + 63) / 64 + 1) / 2 * sh.b * sh.hkv * ns), dim3(512), 0,
                       st, q, k, v, d_o, lse, dvec, sc.start, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, ns, part,
                       sc.end, sc.cap, sc.slopes);
    return hipGetLastError();
  });
  if (e != hipSuccess || ns == 1) return e;
  return launch_attn32_dkv_reduce(part, ns, (long)sh.b * sh.hkv * sh.s * DH, dk, dv, st);
}

size_t fwd_part_bytes(int b, int hq, int s, int dh, int ns) { return ns > 1 ? (size_t)ns * b * hq * s * (dh + 2) * 4 : 0; }
size_t dvec_bytes(int b, int hq, int s) { return round256((size_t)b * hq * s * 4); }
size_t dq_part_bytes(int b, int hq, int s, int dh, int nq) { return nq > 1 ? (size_t)nq * b * hq * s * dh * 4 : 0; }
size_t dkv_part_bytes(int b, int hkv, int s, int dh, int ns) { return ns > 1 ? (size_t)ns * 2 * b * hkv * s * dh * 4 : 0; }
}  // namespace

size_t attn32_scored_fwd_workspace(int b, int hq, int hkv, int s, int dh) {
  return fwd_part_bytes(b, hq, s, dh, q_splits(b, hq, hkv, s));
}
size_t attn32_scored_bwd_workspace(int b, int hq, int hkv, int s, int dh) {
  const size_t x = dq_part_bytes(b, hq, s, dh, q_splits(b, hq, hkv, s)), y = dkv_part_bytes(b, hkv, s, dh, attn32_dkv_splits(b, hq, hkv, s, dh));
  return dvec_bytes(b, hq, s) + (x > y ? x : y);
}

hipError_t launch_attn32_scored_fwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k,
                                    const float* v, float* o, float* lse, void* workspace, size_t bytes, hipStream_t st) {
  int ns = q_splits(sh.b, sh.hq, sh.hkv, sh.s);
  if (!workspace || bytes < fwd_part_bytes(sh.b, sh.hq, sh.s, sh.dh, ns)) ns = 1;
  float* part = static_cast<float*>(workspace);
  switch (sh.dh) {
    case 64: return fwd<64>(sh, sc, q, k, v, o, lse, part, ns, st);
    case 96: return fwd<96>(sh, sc, q, k, v, o, lse, part, ns, st);
    case 128: return fwd<128>(sh, sc, q, k, v, o, lse, part, ns, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_attn32_scored_bwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k,
                                    const float* v, const float* o, const float* lse, const float* d_o, float* dq,
                                    float* dk, float* dv, void* workspace, size_t bytes, hipStream_t st) {
  float* dvec = static_cast<float*>(workspace);
  const size_t at = dvec_bytes(sh.b, sh.hq, sh.s), room = bytes > at ? bytes - at : 0;
  float* part = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
  int nq = q_splits(sh.b, sh.hq, sh.hkv, sh.s), ns = attn32_dkv_splits(sh.b, sh.hq, sh.hkv, sh.s, sh.dh);
  if (room < dq_part_bytes(sh.b, sh.hq, sh.s, sh.dh, nq)) nq = 1;
  if (room < dkv_part_bytes(sh.b, sh.hkv, sh.s, sh.dh, ns)) ns = 1;
  switch (sh.dh) {
    case 64: return bwd<64>(sh, sc, q, k, v, o, lse, d_o, dq, dk, dv, dvec, part, nq, ns, st);
    case 96: return bwd<96>(sh, sc, q, k, v, o, lse, d_o, dq, dk, dv, dvec, part, nq, ns, st);
    case 128: return bwd<128>(sh, sc, q, k, v, o, lse, d_o, dq, dk, dv, dvec, part, nq, ns, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mtp

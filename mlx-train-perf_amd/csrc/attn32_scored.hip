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

template <int DH>
hipError_t fwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k, const float* v, float* o,
               float* lse, hipStream_t st) {
  return with_form(sc, [&](auto mask, auto mod) {
    hipLaunchKernelGGL((attn32_q_kernel<DH, decltype(mask)::value, false, decltype(mod)::value>), grid32_q(sh), dim3(512), 0, st,
                       q, k, v, nullptr, nullptr, nullptr, nullptr, sc.start, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sh.scale,
                       sh.causal, sc.end, sc.cap, sc.slopes);
    return hipGetLastError();
  });
}

template <int DH>
hipError_t bwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k, const float* v, const float* o,
               const float* lse, const float* d_o, float* dq, float* dk, float* dv, float* dvec, int ns, hipStream_t st) {
  float* part = reinterpret_cast<float*>(((uintptr_t)(dvec + (size_t)sh.b * sh.hq * sh.s) + 255) / 256 * 256);
  const hipError_t e = with_form(sc, [&](auto mask, auto mod) {
    constexpr int MASK = decltype(mask)::value, MOD = decltype(mod)::value;
    hipLaunchKernelGGL((attn32_q_kernel<DH, MASK, true, MOD>), grid32_q(sh), dim3(512), 0, st, q, k, v, d_o, o, lse, dvec,
                       sc.start, dq, nullptr, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, sc.end, sc.cap, sc.slopes);
    const hipError_t e1 = hipGetLastError();
    if (e1 != hipSuccess) return e1;
    hipLaunchKernelGGL((attn32_dkv_kernel<DH, MASK, MOD>), dim3(((sh.s + 63) / 64 + 1) / 2 * sh.b * sh.hkv * ns), dim3(512), 0,
                       st, q, k, v, d_o, lse, dvec, sc.start, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sh.scale, sh.causal, ns, part,
                       sc.end, sc.cap, sc.slopes);
    return hipGetLastError();
  });
  if (e != hipSuccess || ns == 1) return e;
  return launch_attn32_dkv_reduce(part, ns, (long)sh.b * sh.hkv * sh.s * DH, dk, dv, st);
}
}  // namespace

hipError_t launch_attn32_scored_fwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k,
                                    const float* v, float* o, float* lse, hipStream_t st) {
  switch (sh.dh) {
    case 64: return fwd<64>(sh, sc, q, k, v, o, lse, st);
    case 96: return fwd<96>(sh, sc, q, k, v, o, lse, st);
    case 128: return fwd<128>(sh, sc, q, k, v, o, lse, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_attn32_scored_bwd(const AttnShape& sh, const AttnScore& sc, const float* q, const float* k,
                                    const float* v, const float* o, const float* lse, const float* d_o, float* dq,
                                    float* dk, float* dv, float* dvec, int nsplit, hipStream_t st) {
  switch (sh.dh) {
    case 64: return bwd<64>(sh, sc, q, k, v, o, lse, d_o, dq, dk, dv, dvec, nsplit, st);
    case 96: return bwd<96>(sh, sc, q, k, v, o, lse, d_o, dq, dk, dv, dvec, nsplit, st);
    case 128: return bwd<128>(sh, sc, q, k, v, o, lse, d_o, dq, dk, dv, dvec, nsplit, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mtp

// Attention with capped scores, a bias by distance and key spans: the launches of one head_dim over the
// kernels of attn_core.hpp, instantiated by attn_scored_<head_dim>.hip and called from attn_scored.hip.
#pragma once
#include "attn_core.hpp"

namespace mtp {

// A backward call's workspace, in order: D, but for slopes alone the logarithms in the P waves' form, with slopes and a cap
// or spans the tops of the rows' biases (Score), the fp32 parts of a split dQ, then dK/dV pass, and for spans the two work orders (null: none) and
// the queries [col_begin, col_end) that see each key.
struct ScoredWorkspace {
  float* dvec;
  float* part;
  int32_t *q_order, *kv_order, *col_begin, *col_end;
  int nsplit, nq;  // of the dK/dV pass, of the dQ pass
};
hipError_t launch_attn_dq_sum(const float* part, int ns, long plane, bf16_t* dq, hipStream_t st);

template <int DH>
hipError_t scored_fwd(const AttnShape& sh, const AttnScore& sc, const bf16_t* q, const bf16_t* k, const bf16_t* v,
                      bf16_t* o, int8_t* o_low, const int32_t* order, float* lse, int grid, int nsplit, float* part,
                      hipStream_t st);
template <int DH>
hipError_t scored_bwd(const AttnShape& sh, const AttnScore& sc, const ScoredWorkspace& ws, const bf16_t* q,
                      const bf16_t* k, const bf16_t* v, const bf16_t* o, const int8_t* o_low, const float* lse,
                      const bf16_t* d_o, bf16_t* dq, bf16_t* dk, bf16_t* dv, int grid, hipStream_t st);

// The forward under a cap of at most 80 ln 2 runs against a fixed maximum (attn_kv_kernel).
constexpr float kFixedCap = 55.4f;
// f(std::integral_constant<int, MOD>) for the call's score form.
template <class F>
hipError_t with_mod(const AttnScore& sc, F&& f) {
  if (sc.cap > 0.f) {
    if (sc.slopes) return f(std::integral_constant<int, kModBoth>{});
    return f(std::integral_constant<int, kModCap>{});
  }
  if (sc.slopes) return f(std::integral_constant<int, kModSlope>{});
  return f(std::integral_constant<int, kModNone>{});
}

#ifdef MTP_SCORED_DH
template <>
hipError_t scored_fwd<MTP_SCORED_DH>(const AttnShape& sh, const AttnScore& sc, const bf16_t* q, const bf16_t* k,
                                     const bf16_t* v, bf16_t* o, int8_t* o_low, const int32_t* order,
                                     float* lse, int grid, int nsplit, float* part, hipStream_t st) {
  constexpr int DH = MTP_SCORED_DH;
  return with_mod(sc, [&](auto m) {
    constexpr int MOD = decltype(m)::value;
    auto launch = [&](auto whole, auto split) {
      hipLaunchKernelGGL(nsplit > 1 ? split : whole, dim3(grid * nsplit), dim3(256), 0, st, q, k, v, nullptr, nullptr, nullptr, nullptr, sc.end,
                         sc.start, o, lse, sh.b, sh.hq, sh.hkv, sh.s, sh.scale * kLog2e, sh.scale, sh.causal, order,
                         sc.cap, sc.slopes, o_low, nullptr, nullptr, nsplit, part);
      return hipGetLastError();
    };
    // A cap above kFixedCap runs as a cap with slopes of none.
    constexpr int RUN = MOD == kModCap ? kModBoth : MOD;
    const bool fixed = sc.cap <= kFixedCap;
    if (sc.start) {
      if constexpr (MOD == kModCap)
        if (fixed) return launch(attn_kv_kernel<DH, kMaskSpan, false, MOD, true>, attn_kv_kernel<DH, kMaskSpan, false, MOD, true, true>);
      return launch(attn_kv_kernel<DH, kMaskSpan, false, RUN>, attn_kv_kernel<DH, kMaskSpan, false, RUN, false, true>);
    }
    if constexpr (MOD & kModCap)
      if (fixed) return launch(attn_kv_kernel<DH, kMaskPlain, false, MOD, true>, attn_kv_kernel<DH, kMaskPlain, false, MOD, true, true>);
    if constexpr (MOD != kModNone) return launch(attn_kv_kernel<DH, kMaskPlain, false, RUN>, attn_kv_kernel<DH, kMaskPlain, false, RUN, false, true>);
    return hipErrorInvalidValue;
  });
}

template <>
hipError_t scored_bwd<MTP_SCORED_DH>(const AttnShape& sh, const AttnScore& sc, const ScoredWorkspace& ws,
                                     const bf16_t* q, const bf16_t* k, const bf16_t* v, const bf16_t* o,
                                     const int8_t* o_low, const float* lse, const bf16_t* d_o, bf16_t* dq, bf16_t* dk, bf16_t* dv, int grid,
                                     hipStream_t st) {
  constexpr int DH = MTP_SCORED_DH;
  return with_mod(sc, [&](auto m) {
    constexpr int MOD = decltype(m)::value;
    auto launch = [&](auto whole, auto split, auto dkv_kernel) {
      hipLaunchKernelGGL(ws.nq > 1 ? split : whole, dim3(grid * ws.nq), dim3(256), 0, st, q, k, v, d_o, o, lse, ws.dvec, sc.end, sc.start, dq,
                         nullptr, sh.b, sh.hq, sh.hkv, sh.s, sh.scale * kLog2e, sh.scale, sh.causal, ws.q_order, sc.cap,
                         sc.slopes, const_cast<int8_t*>(o_low), ws.q_order ? nullptr : ws.col_begin,
                         ws.q_order ? nullptr : ws.col_end, ws.nq, ws.part);
      hipError_t e = hipGetLastError();
      if (e == hipSuccess && ws.nq > 1) e = launch_attn_dq_sum(ws.part, ws.nq, (long)sh.b * sh.hq * sh.s * sh.dh, dq, st);
      if (e != hipSuccess) return e;
      // (the parts of dQ are read: those of dK and dV take their place)
      hipLaunchKernelGGL(dkv_kernel, dim3((sh.s + 127) / 128 * sh.b * sh.hkv * ws.nsplit), dim3(512), 0, st, q, k, v, d_o,
                         MOD == kModSlope ? lse : ws.dvec + (long)sh.b * sh.hq * sh.s, ws.dvec, ws.col_end, dk, dv, sh.b, sh.hq, sh.hkv, sh.s, sh.scale * kLog2e, sh.scale,
                         sh.causal, ws.nsplit, ws.part, ws.kv_order, ws.col_begin, sc.cap, sc.slopes);
      return hipGetLastError();
    };
    if (sc.start) return launch(attn_kv_kernel<DH, kMaskSpan, true, MOD>, attn_kv_kernel<DH, kMaskSpan, true, MOD, false, true>,
                    attn_bwd_dkv_ab_kernel<DH, kMaskSpan, MOD>);
    if constexpr (MOD != kModNone)
      return launch(attn_kv_kernel<DH, kMaskPlain, true, MOD>, attn_kv_kernel<DH, kMaskPlain, true, MOD, false, true>,
                    attn_bwd_dkv_ab_kernel<DH, kMaskPlain, MOD>);
    return hipErrorInvalidValue;
  });
}
#endif

}  // namespace mtp

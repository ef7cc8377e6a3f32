// The end of a gather's tile (GatherPlan, mtp_launch.hpp), whichever core made it.
#pragma once
#include "mtp_common.hpp"
#include "mtp_launch.hpp"

namespace mtp {

// A wave's logits acc[i][j], rows v = row0 + 32 i + (register's row) of the group, columns entries col0 + 32 j + lane % 32: to
// rows[code] (16 bytes a lane; rows past the vocabulary as -inf), or for a single logit the register that holds it.
template <int NI, int NJ>
__device__ __forceinline__ void store_gathered(const f32x16 (&acc)[NI][NJ], const GatherPlan& plan, const int2* entries,
                                               int count, int vleft, int row0, int col0, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = col0 + 32 * j + (lane & 31);
    const int code = e < count ? entries[e].y : 0;
    if (e >= count) continue;
    if (code >= 0) {
      float* dst = plan.rows + (long)code * kGroup;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int v = row0 + 32 * i + 8 * q + 4 * h;
          f32x4 x;
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = v + u < vleft ? acc[i][j][4 * q + u] : kNegInf;
          *reinterpret_cast<f32x4*>(dst + v) = x;
        }
    } else {
      const int want = (-1 - code) % kGroup - row0;
      float x = 0.f;
      bool here = false;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (want == 32 * i + 8 * (r >> 2) + 4 * h + (r & 3)) {
            x = acc[i][j][r];
            here = true;
          }
      if (here) plan.picks[(-1 - code) / kGroup] = x;
    }
  }
}

}  // namespace mtp

// The end of a gather's tile (GatherPlan, mtp_launch.hpp), whichever core made it.
#pragma once
#include "mtp_common.hpp"
#include "mtp_launch.hpp"

namespace mtp {

// A wave's logits acc[i][j], rows v = row0 + 32 i + (register's row) of the group, columns entries col0 + 32 j + lane % 32: 16
// bytes a lane; rows past the vocabulary as -inf.
template <int NI, int NJ>
__device__ __forceinline__ void store_gathered(const f32x16 (&acc)[NI][NJ], const GatherPlan& plan, const int2* entries,
                                               int count, int vleft, int row0, int col0, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = col0 + 32 * j + (lane & 31);
    if (e >= count) continue;
    float* dst = plan.rows + (long)entries[e].y * kGroup;
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
  }
}

// ------------------------------------------------------------------------------------------
// A forward's listed logits (ScoreList). Each lane follows its token columns' lists up the vocabulary: `next` is the first
// listed column that no tile has passed, `at` its place. A tile's lanes hold the logits of column li = 32 i + 8 (r / 4) + 4 half
// + r % 4 of their wave's part of it, so a listed one is in one lane and one of 16 NI registers: a tree of selects by the bits
// of li finds it (16 NI of them) and a store puts it away. A teacher's list then leaves the tile (its registers become -inf), so
// that the statistics are those of what no list has: what a list leaves of 1 is a sum of its own and no difference.
// Most tiles have none of a wave's tokens' columns, and the rest few.
// ------------------------------------------------------------------------------------------
// acc[BITS' registers from `first`], the one whose index has the bits of li: register bits 0, 1 are bits 0, 1 of li, the ones
// above are its bits 3 and on.
template <int BITS, int NI, int NJ>
__device__ __forceinline__ float select_logit(const f32x16 (&acc)[NI][NJ], int j, int li, int first) {
  if constexpr (BITS == 0) {
    return acc[first >> 4][j][first & 15];
  } else {
    const float lo = select_logit<BITS - 1>(acc, j, li, first), hi = select_logit<BITS - 1>(acc, j, li, first + (1 << (BITS - 1)));
    const int bit = BITS - 1 < 2 ? BITS - 1 : BITS;
    return (li >> bit) & 1 ? hi : lo;
  }
}

template <int NJ>
struct ListCursor {
  int next[NJ], at[NJ];
  // The first listed columns of the tokens t[j] (valid: below N) from v0 on.
  __device__ __forceinline__ void start(const ScoreList& l, const int (&t)[NJ], int N, int v0) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      next[j] = kNoColumn;
      at[j] = 0;
      if (t[j] >= N) continue;
      const int* row = l.column + (long)t[j] * l.k;
      int lo = 0, hi = l.k;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (row[mid] < v0) lo = mid + 1;
        else hi = mid;
      }
      at[j] = lo;
      if (lo < l.k) next[j] = row[lo];
    }
  }
  // The tile [v0, v0 + SIZE): the wave holds its rows [part, part + 32 NI).
  template <int SIZE, int NI>
  __device__ __forceinline__ void take(const ScoreList& l, const int (&t)[NJ], f32x16 (&acc)[NI][NJ], int v0, int part, int half) {
    constexpr int kBits = NI == 4 ? 6 : 5, kWords = NI / 2;
    static_assert(NI == 4 || NI == 2, "16 NI registers");
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      uint32_t taken[kWords] = {};  // registers, as bits
      while (__any(next[j] < v0 + SIZE)) {
        if (next[j] < v0 + SIZE) {
          const int li = next[j] - v0 - part;
          const float z = select_logit<kBits>(acc, j, li, 0);
          if (li >= 0 && li < 32 * NI && ((li >> 2) & 1) == half) {
            l.z[(long)t[j] * l.k + at[j]] = z;
            const int r = (li & 3) | (li >> 3) << 2;
#pragma unroll
            for (int w = 0; w < kWords; ++w) taken[w] |= (r >> 5) == w ? 1u << (r & 31) : 0u;
          }
          ++at[j];
          next[j] = at[j] < l.k ? l.column[(long)t[j] * l.k + at[j]] : kNoColumn;
        }
      }
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        if (__any(taken[w]))
#pragma unroll
          for (int r = 0; r < 32; ++r)
            if (taken[w] >> r & 1) acc[2 * w + (r >> 4)][j][r & 15] = kNegInf;
    }
  }
};

// The same for lists of one, targets, which stay in the statistics: nothing to follow.
template <int NJ>
struct TargetCursor {
  int column[NJ];
  __device__ __forceinline__ void start(const ScoreList& l, const int (&t)[NJ], int N, int) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) column[j] = t[j] < N ? l.column[t[j]] : kNoColumn;
  }
  template <int SIZE, int NI>
  __device__ __forceinline__ void take(const ScoreList& l, const int (&t)[NJ], const f32x16 (&acc)[NI][NJ], int v0, int part, int half) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int li = column[j] - v0 - part;
      const bool here = li >= 0 && li < 32 * NI && ((li >> 2) & 1) == half;
      if (__any(here)) {
        const float z = select_logit<NI == 4 ? 6 : 5>(acc, j, li, 0);
        if (here) l.z[t[j]] = z;
      }
    }
  }
};

}  // namespace mtp

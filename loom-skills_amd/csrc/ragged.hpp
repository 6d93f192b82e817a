// Rows sorted by expert with ragged segments: expert e owns rows offsets[e] .. offsets[e + 1] - 1. The offsets live on the
// device, so every workgroup finds its own segment (one 64-bit ballot or one prefix sum over the experts); values outside
// [0, rows] are clamped and a segment that ends before it starts is empty, so that nothing out of range is touched whatever
// the offsets hold.
#pragma once
#include "common.hpp"

namespace qmm {

constexpr int kMaxRaggedE = 1024;

__device__ __forceinline__ int clamp_row(int v, int rows) { return min(max(v, 0), rows); }

// The nth (from 0) expert that has rows, and its segment [lo, hi); false past the last one. Wave-uniform.
__device__ __forceinline__ bool nth_segment(const int32_t *offsets, int E, int rows, int nth, int &e, int &lo, int &hi) {
  const int lane = threadIdx.x & 63;
  for (int c = 0; c < E; c += 64) {
    const int i = min(c + lane, E - 1);
    const int a = clamp_row(offsets[i], rows), b = clamp_row(offsets[i + 1], rows);
    const bool some = c + lane < E && b > a;
    const unsigned long long mask = __ballot(some);
    const int n = __popcll(mask);
    if (nth < n) {
      const int rank = __popcll(mask & ((1ull << lane) - 1));
      const int l = __ffsll((long long)__ballot(some && rank == nth)) - 1;
      e = __builtin_amdgcn_readfirstlane(c + l);
      lo = __builtin_amdgcn_readlane(a, l);
      hi = __builtin_amdgcn_readlane(b, l);
      return true;
    }
    nth -= n;
  }
  return false;
}

// Row tiles of BM rows, the experts' one after the other: their number, and how many come before the lane's experts (lane l
// owns experts per l .. per l + per - 1).
struct TileScan {
  int total, before, per;
};
template <int BM>
__device__ __forceinline__ TileScan scan_tiles(const int32_t *offsets, int E, int rows) {
  const int lane = threadIdx.x & 63;
  TileScan s;
  s.per = (E + 63) >> 6;
  int own = 0;
  for (int j = 0; j < s.per; ++j) {
    const int i = s.per * lane + j, at = min(i, E - 1);
    const int a = clamp_row(offsets[at], rows), b = clamp_row(offsets[at + 1], rows);
    own += i < E ? (max(b - a, 0) + BM - 1) / BM : 0;
  }
  int sum = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(sum, d, 64);
    sum += lane >= d ? v : 0;
  }
  s.total = __builtin_amdgcn_readlane(sum, 63);
  s.before = sum - own;
  return s;
}
// Expert and segment of row tile t < s.total, and the expert's first tile. Wave-uniform.
template <int BM>
__device__ __forceinline__ void find_tile(const int32_t *offsets, int E, int rows, const TileScan &s, int t, int &e, int &lo,
                                          int &hi, int &first) {
  const int l = __popcll(__ballot(s.before <= t)) - 1;   // before does not fall along the lanes: the last lane at or below t
  first = __builtin_amdgcn_readlane(s.before, l);
  for (e = min(s.per * l, E - 1);; ++e) {
    lo = clamp_row(__builtin_amdgcn_readfirstlane(offsets[e]), rows);
    hi = clamp_row(__builtin_amdgcn_readfirstlane(offsets[e + 1]), rows);
    const int n = (max(hi - lo, 0) + BM - 1) / BM;
    if (t < first + n || e + 1 >= E) return;
    first += n;
  }
}

}  // namespace qmm

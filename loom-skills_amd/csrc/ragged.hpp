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

// Rows of no expert set to zero (QMM_ZERO_REST): workgroup `part` of `parts` that have no other work, beside those that write the
// experts' rows. Offsets that never fall leave the rows before the first segment and behind the last, two runs of bytes; others are
// looked at a row and wave at a time. y: of 2- or 4-byte values at a multiple of their size.
__device__ __forceinline__ void zero_run(u8 *p, int64_t bytes, int thread, int threads) {
  typedef __attribute__((ext_vector_type(4))) u32 u32x4;
  const u32x4 zero = {0, 0, 0, 0};
  const int64_t units = bytes >> 4;
  for (int64_t i = thread; i < units; i += threads) __builtin_memcpy(p + 16 * i, &zero, 16);
  const int left = (int)(bytes & 15) >> 1;   // a last unit by halves
  if (thread < left) {
    const u16 z = 0;
    __builtin_memcpy(p + 16 * units + 2 * thread, &z, 2);
  }
}
__device__ __forceinline__ void zero_rest(const int32_t *offsets, int E, int rows, u8 *y, int64_t row_bytes, int part, int parts) {
  const int lane = threadIdx.x & 63;
  bool falls = false;
  for (int c = 0; c < E; c += 64) {
    const int i = min(c + lane, E - 1);
    falls |= clamp_row(offsets[i + 1], rows) < clamp_row(offsets[i], rows);
  }
  if (!__ballot(falls)) {
    const int first = clamp_row(offsets[0], rows), end = clamp_row(offsets[E], rows);
    const int thread = part * (int)blockDim.x + (int)threadIdx.x, threads = parts * (int)blockDim.x;
    zero_run(y, first * row_bytes, thread, threads);
    zero_run(y + end * row_bytes, (rows - end) * row_bytes, thread, threads);
    return;
  }
  const int waves = (int)blockDim.x >> 6;
  for (int row = part * waves + ((int)threadIdx.x >> 6); row < rows; row += parts * waves) {
    bool in = false;
    for (int c = 0; c < E; c += 64) {
      const int i = min(c + lane, E - 1);
      in |= clamp_row(offsets[i], rows) <= row && row < clamp_row(offsets[i + 1], rows);
    }
    if (!__ballot(in)) zero_run(y + row * row_bytes, row_bytes, lane, 64);
  }
}
// Whether an output's type asks for it, which it does not say any more then.
inline bool zero_rest_asked(int &dtype) {
  const bool asked = dtype >= 0 && (dtype & QMM_ZERO_REST);
  if (asked) dtype &= ~QMM_ZERO_REST;
  return asked;
}
// workgroups for it: they look at the offsets only where every row is an expert's
inline int rest_blocks(int64_t rows, int64_t row_bytes) {
  const int64_t n = rows * row_bytes >> 18;   // 256 KB each, one an XCD at least
  return n < 8 ? 8 : n > 64 ? 64 : (int)n & ~7;
}

}  // namespace qmm

// Products of few rows, y = x W^T, where W is streamed once: 4-bit weights with group scales (w4) or 16-bit weights, dense or
// by expert over ragged segments of rows.
//
//   w4      y[t, r] = sum_g s[r, g] (sum_{c in g} x[t, c] q[r, c] - z[r, g] sum_{c in g} x[t, c])
//   16-bit  y[t, r] = sum_c x[t, c] W[r, c]
//
// v_mfma_f32_16x16x32 with 16 weight rows as B and 16 tokens as A: lane (c, h) = (lane % 16, lane / 16) holds values 8 h .. + 7
// of a 32-value step of weight row c and of token c, and register i of the sums is token 4 h + i, row c, so that a row's scale
// is one register. w4 codes 0 .. 15 are exact in bf16, a bf16 row is its own operand and an f32 value the sum of three bf16
// values (its leading 8 bits, the next 8, the rest: three MFMAs), so every product is exact and every sum f32; the groups' sums
// of x come from an MFMA with ones. Codes and ones enter w4's products times 2^-12 and the scale times 2^12, both exact: the sums of 128
// values times 15 are below 2^11 times the largest of them, so that they stay finite wherever x is; what is lost is below 2^-137 s a
// value (the sums' subnormals).
//
// Memory bounds a row or two (12288 x 4096 7.6 us for 26.8 MB, 3.5 TB/s), the f32 rows' split and the fragments' reads more rows (16 f32
// rows 17 us, 63 44 us): eight waves share a row block along K because a wave's chain of loads is what a small call waits for.
#pragma once
#include <algorithm>
#include <type_traits>

#include "ragged.hpp"

namespace qmm {
namespace few {

typedef __attribute__((ext_vector_type(4))) u32 u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

constexpr int kWaves = 8;
enum Weight { kW4 = 0, kWBF16 = 1, kWF16 = 2 };

struct Args {
  const int32_t *offsets;   // NULL: one segment of all rows
  int E, rows, n, k;
  const u8 *x, *w;
  int64_t w_expert;         // bytes of one expert's matrix
  const u32 *ws;            // w4: (f16 scale, f16 1024 + zero) words [n / 16][groups][16]
  int groups, gshift;       // group of 32-value step i: min(i >> gshift, groups - 1)
  void *y;
  int y_bytes;              // 4: f32; 2: bf16 (w4) or the weights' type
  int parts = 1;            // of K, blocks of the grid's x one after the other; more than one: f32 sums [parts][rows][n] into part
  float *part = nullptr;
  int rest = 0;             // rows of no expert are set to zero, by one more layer of the grid's y
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, u32 bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)bytes, 0x00020000);
}
constexpr u32 kPast = 0x80000000u;   // an offset past every resource: the load gives zeros
__device__ __forceinline__ u32x4 ld(__amdgpu_buffer_rsrc_t r, u32 off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

template <int W>
__device__ __forceinline__ f32x4 mfma(u32x4 x, u32x4 w, f32x4 c) {
  if constexpr (W == kWF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
}
constexpr float kSumScale = 0x1p-12f;   // of w4's codes and ones in bf16
// four codes in the low nibbles of four bytes as two bf16 pairs, times kSumScale: 0000qqqq read as OCP E4M3 is q 2^-9 exactly
__device__ __forceinline__ u32x4 codes(u32 w) {
  const u32 lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
  return u32x4{__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f * kSumScale, false)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f * kSumScale, true)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f * kSumScale, false)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f * kSumScale, true))};
}
// eight f32 values as three exact bf16 parts each
struct Parts {
  u32x4 p[3];
};
__device__ __forceinline__ Parts split(u32x4 a, u32x4 b) {
  Parts o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 u0 = i < 2 ? a[2 * i] : b[2 * i - 4], u1 = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
    const float r0 = u32_as_f32(u0) - u32_as_f32(u0 & 0xFFFF0000u), r1 = u32_as_f32(u1) - u32_as_f32(u1 & 0xFFFF0000u);
    const u32 m0 = f32_as_u32(r0), m1 = f32_as_u32(r1);
    const float l0 = r0 - u32_as_f32(m0 & 0xFFFF0000u), l1 = r1 - u32_as_f32(m1 & 0xFFFF0000u);
    o.p[0][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    o.p[1][i] = __builtin_amdgcn_perm(m1, m0, 0x07060302u);
    o.p[2][i] = __builtin_amdgcn_perm(f32_as_u32(l1), f32_as_u32(l0), 0x07060302u);
  }
  return o;
}

// W: the weights; F32: rows x are f32 (w4 only), else 16-bit; GS: 32-value steps a scale covers within a 128-value tile; TT:
// tiles of 16 tokens at a time; KS: waves that share 16-row blocks of W, each with every KS-th 128-value tile; RB: blocks of a wave
// (a workgroup has 8 RB / KS); TL: rows of x a wave keeps in LDS. Grid: (row blocks of each part of K, experts with rows, layers that
// share a segment's chunks of tokens: all chunks of a dense call; by expert as many as leave few workgroups without one, for a router that
// sends most rows to one expert).
//
// x: up to TL rows are brought into the wave's own LDS, a batch of U tiles at a time and 8 values a lane (f32 rows split into
// their parts there, once instead of once a lane), rows of U x 16 chunks, chunk i of row t at i ^ t; a fragment read past the last
// row reads that one again, its outputs are not stored. With one row a load then brings 1 KB where the fragments' own loads would
// use four lanes. More rows are read as fragments from memory.
template <int W, bool F32, int GS, int TT, int KS, int TL, int RB>
__global__ __launch_bounds__(64 * kWaves, TT > 1 || RB > 2 ? 2 : F32 || RB > 1 || TL > 2 || (TL > 1 && W == kW4) ? 4 : 6) void few_rows_kernel(Args a) {
  constexpr int kParts = F32 ? 3 : 1, kLoads = F32 ? 2 : 1, kES = F32 ? 4 : 2;
  constexpr int U = W == kW4 && !F32 && RB < 4 ? 4 : 2;   // tiles of a wave whose weights are in flight
  constexpr int kBlocks = kWaves / KS * RB;   // of a workgroup
  static_assert(TL == 0 || (TT == 1 && TL <= 16), "staged rows are one tile of tokens");
  __shared__ __align__(16) float red[kWaves][RB * TT][64][4];
  __shared__ __align__(16) u8 xs[TL > 0 ? kWaves : 1][TL > 0 ? kParts : 1][TL > 0 ? TL : 1][U * 256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, h = lane >> 4, part = wave % KS;
  const int KT = (a.k + 127) >> 7, nb = (a.n + 15) >> 4;
  const int groups = (nb + kBlocks - 1) / kBlocks, piece = (int)blockIdx.x / groups, rb0 = ((int)blockIdx.x - piece * groups) * kBlocks;
  const int T0 = (int)((int64_t)KT * piece / a.parts), T1 = (int)((int64_t)KT * (piece + 1) / a.parts);   // this piece's tiles
  int e = 0, lo = 0, hi = a.rows;
  if (a.rest && blockIdx.y == gridDim.y - 1) {
    zero_rest(a.offsets, a.E, a.rows, static_cast<u8 *>(a.y), (int64_t)a.n * a.y_bytes, (int)(blockIdx.z * gridDim.x + blockIdx.x),
              (int)(gridDim.x * gridDim.z));
    return;
  }
  if (a.offsets && !nth_segment(a.offsets, a.E, a.rows, blockIdx.y, e, lo, hi)) return;
  const u8 *w[RB];
  const u32 *ws[RB];
  __amdgpu_buffer_rsrc_t wr[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int rb = min(rb0 + wave / KS * RB + r, nb - 1);   // blocks past the last: that one again, not stored
    const u8 *we = a.w + (int64_t)e * a.w_expert;
    if constexpr (W == kW4) {
      w[r] = we + (int64_t)rb * KT * 1024;
      ws[r] = a.ws + ((int64_t)e * nb + rb) * a.groups * 16 + c;
    } else {
      wr[r] = rsrc(we + (int64_t)rb * 32 * a.k, (u32)(min(16, a.n - 16 * rb) * a.k * 2));
    }
  }
  constexpr u32 one = __builtin_bit_cast(u32, kSumScale) >> 16 | (__builtin_bit_cast(u32, kSumScale) & 0xFFFF0000u);   // in bf16, twice
  const u32x4 ones = {one, one, one, one};

  struct Batch {
    u32x4 q[RB][U][W == kW4 ? 1 : 4];
    u32 sc[RB][U][4 / GS];
    u32x4 x[TL > 0 ? TL * U / 4 + (TL * U % 4 != 0) : 1][kLoads];   // 8 values a lane
  };
  constexpr int kX = TL * U * 16;   // chunks of 8 values of a batch's staged rows

  constexpr int kRows = TL > 0 ? TL : 16 * TT;   // at a time
  for (int t0 = lo + (int)blockIdx.z * kRows; t0 < hi; t0 += (int)gridDim.z * kRows) {
    const int rows = min(kRows, hi - t0);
    const __amdgpu_buffer_rsrc_t xr = rsrc(a.x + (int64_t)t0 * a.k * kES, (u32)rows * (u32)a.k * kES);
    f32x4 acc[RB][TT];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};

    constexpr bool kLds = TL > 0;
    {
      // batch at tb: tiles tb, tb + KS, ... (past the last: that one again, not used)
      auto load = [&](int tb, Batch &b) __attribute__((always_inline)) {
        if constexpr (kLds) {
#pragma unroll
          for (int i = 0; 64 * i < kX; ++i) {
            const int at = 64 * i + lane, t = at / (U * 16), u = at / 16 % U, k = 128 * (tb + KS * u) + 8 * (at & 15);
            const u32 off = k < a.k && t < TL ? ((u32)t * (u32)a.k + (u32)k) * kES : kPast;
#pragma unroll
            for (int p = 0; p < kLoads; ++p) b.x[i][p] = ld(xr, off + 16 * p);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = min(tb + KS * u, T1 - 1);
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            if constexpr (W == kW4) {
              b.q[r][u][0] = *reinterpret_cast<const u32x4 *>(w[r] + (int64_t)t * 1024 + 16 * lane);
#pragma unroll
              for (int g = 0; g < 4 / GS; ++g) b.sc[r][u][g] = ws[r][min((4 * t + GS * g) >> a.gshift, a.groups - 1) * 16];
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int kk = 128 * t + 32 * j + 8 * h;
                b.q[r][u][j] = ld(wr[r], kk < a.k ? (u32)(c * a.k + kk) * 2u : kPast);
              }
            }
          }
        }
      };
      auto use = [&](int tb, const Batch &b) __attribute__((always_inline)) {
        if constexpr (kLds) {
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int i = 0; 64 * i < kX; ++i) {
            const int at = 64 * i + lane, t = at / (U * 16), ch = (at % (U * 16)) ^ t;
            if (kX % 64 == 0 || t < TL) {
              if constexpr (F32) {
                const Parts v = split(b.x[i][0], b.x[i][kLoads - 1]);
#pragma unroll
                for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(&xs[wave][p][t][16 * ch]) = v.p[p];
              } else {
                *reinterpret_cast<u32x4 *>(&xs[wave][0][t][16 * ch]) = b.x[i][0];
              }
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = tb + KS * u;
          if (t >= T1) break;
          u32x4 xv[TT][4][kLds ? 1 : kLoads];
          if constexpr (!kLds) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int p = 0; p < kLoads; ++p) {
                  const int kk = 128 * t + 32 * j + 8 * h;
                  xv[tt][j][p] = ld(xr, kk < a.k ? ((u32)(16 * tt + c) * (u32)a.k + (u32)kk) * kES + 16 * p : kPast);
                }
          }
#pragma unroll
          for (int g = 0; g < 4 / GS; ++g) {
            f32x4 dot[RB][TT], sum[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
              sum[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int r = 0; r < RB; ++r) dot[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int jj = 0; jj < GS; ++jj) {
              const int j = GS * g + jj;
              u32x4 wf[RB];
#pragma unroll
              for (int r = 0; r < RB; ++r) {
                if constexpr (W == kW4) wf[r] = codes(b.q[r][u][0][j]);
                else wf[r] = b.q[r][u][j];
              }
#pragma unroll
              for (int tt = 0; tt < TT; ++tt) {
                Parts xp;
                if constexpr (kLds) {
                  const int row = min(c, rows - 1), ch = (16 * u + 4 * j + h) ^ row;
#pragma unroll
                  for (int p = 0; p < kParts; ++p) xp.p[p] = *reinterpret_cast<const u32x4 *>(&xs[wave][p][row][16 * ch]);
                } else if constexpr (F32) {
                  xp = split(xv[tt][j][0], xv[tt][j][kLds ? 0 : kLoads - 1]);
                } else {
                  xp.p[0] = xv[tt][j][0];
                }
#pragma unroll
                for (int p = kParts - 1; p >= 0; --p) {
                  if constexpr (W == kW4) {
#pragma unroll
                    for (int r = 0; r < RB; ++r) dot[r][tt] = mfma<W>(xp.p[p], wf[r], dot[r][tt]);
                    sum[tt] = mfma<W>(xp.p[p], ones, sum[tt]);
                  } else {
#pragma unroll
                    for (int r = 0; r < RB; ++r) acc[r][tt] = mfma<W>(xp.p[p], wf[r], acc[r][tt]);
                  }
                }
              }
            }
            if constexpr (W == kW4) {
#pragma unroll
              for (int r = 0; r < RB; ++r) {
                const float s = f16_to_f32(b.sc[r][u][g]) * (1.f / kSumScale), z = (float)(b.sc[r][u][g] >> 16 & 15u);
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    acc[r][tt][i] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[tt][i], dot[r][tt][i]), acc[r][tt][i]);
              }
            }
          }
        }
      };
      Batch b;
      for (int tb = T0 + part; tb < T1; tb += KS * U) {
        load(tb, b);
        use(tb, b);
      }
    }

    auto store = [&](int token, int row, float v) __attribute__((always_inline)) {   // token of the chunk
      if (token < rows && row < a.n) {
        const int64_t at = (int64_t)(t0 + token) * a.n + row;
        if (a.parts > 1) a.part[(int64_t)piece * a.rows * a.n + at] = v;
        else if (a.y_bytes == 4) static_cast<float *>(a.y)[at] = v;
        else if constexpr (W == kWF16) static_cast<_Float16 *>(a.y)[at] = (_Float16)v;
        else static_cast<__bf16 *>(a.y)[at] = (__bf16)v;
      }
    };
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) *reinterpret_cast<f32x4 *>(red[wave][r * TT + tt][lane]) = acc[r][tt];
    __syncthreads();
    // output (block v / (256 TT), token, row v % 16): the block's waves' sums in order
    for (int v = tid; v < 256 * TT * kBlocks; v += 64 * kWaves) {
      const int b = v / (256 * TT), token = (v >> 4) % (16 * TT), r = v & 15, l = ((token & 15) >> 2) * 16 + r;
      if (token >= rows) continue;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) s += red[b / RB * KS + i][b % RB * TT + (token >> 4)][l][token & 3];
      store(token, 16 * (rb0 + b) + r, s);
    }
    __syncthreads();
  }
}

// All extents are checked by the callers.
template <int W, bool F32, int GS, int TT, int KS, int TL, int RB = 1>
int launch(const Args &a, int slots, hipStream_t s) {
  constexpr int kRows = TL > 0 ? TL : 16 * TT;
  const int per = 16 * kWaves / KS * RB, blocks = (a.n + per - 1) / per;
  const int most = (a.rows + kRows - 1) / kRows;   // chunks of a segment that holds all rows
  const int chunks = a.offsets ? max(1, min(most / 4, 2048 / (blocks * slots))) : min(most, 65535);
  few_rows_kernel<W, F32, GS, TT, KS, TL, RB><<<dim3((unsigned)(blocks * a.parts), slots + (a.rest ? 1 : 0), (unsigned)chunks), dim3(64 * kWaves), 0, s>>>(a);
  return launch_status();
}
// us in a graph on inputs out of cache. x in LDS (TL) against fragments from memory: one dense row, w4 12288 x 4096 7.6 against 9.7,
// 4096 x 12288 8.6 and 12.7, f32 4096 x 4096 6.0 and 8.2; two or four dense rows no difference. By expert with a row each: 16-bit 8
// rows 1536 x 2048 11.9 and 13.8, but 32 rows of 32 experts 2880 x 2880 56 and 40 (experts hit more often are walked two rows at a
// time). w4 with two waves a row block where the blocks fill the chip: 104 rows of 128 experts 1536 x 2048 28 against 47 with
// eight, 30 without LDS; f32 rows with four, two blocks each, 38 against 47.
//
// Row blocks of a wave (RB) share its reads of x, their split into bf16 parts and the groups' sums, which is most of the work from
// f32 rows or five bf16 rows on: as many as leave each CU a workgroup, one, two and three at 12288 x 4096: 8 rows bf16 12.1, 11.2,
// 10.1, f32 26.8, 18.5, 16.4; 63 rows bf16 47.6, 39.2, 23.2, f32 89, 71, 44 (four: 45, and 82 against 50 in groups of 64, spilling);
// at 6144 x 4096 16 rows 10.6, 8.0, 8.5, at 4096 x 4096 6.7, 7.9; 2 rows bf16 9.8, 10.1, 10.0; 300 rows of 128 experts 1536 x 2048
// bf16 49, 44, 39, f32 109, 74, 60. 16-bit weights (no sums, no split): 64 rows of 32 experts 2880 x 2880 79 and 86.
template <int W, bool F32, int GS, int RB>
int launch_rb(const Args &a, int avg, int slots, hipStream_t s) {
  if (avg <= 16) return launch<W, F32, GS, 1, 8, 0, RB>(a, slots, s);
  return avg <= 32 ? launch<W, F32, GS, 2, 8, 0, RB>(a, slots, s) : launch<W, F32, GS, 4, 8, 0, RB>(a, slots, s);
}
template <int W, bool F32, int GS>
int launch_tt(const Args &a, hipStream_t s) {
  const int slots = a.offsets ? min(a.E, a.rows) : 1;
  const int avg = (a.rows + slots - 1) / slots;   // tokens at a time: as many as a segment may hold
  const int64_t blocks = (int64_t)((a.n + 15) / 16) * slots;
  if (a.rows == 1) return launch<W, F32, GS, 1, 8, 1>(a, slots, s);
  if constexpr (W != kW4) {
    if (avg == 1 && a.rows <= 8) return launch<W, F32, GS, 1, 8, 2>(a, slots, s);
  } else {
    if (avg == 1 && blocks >= 2048) {
      if constexpr (F32) return launch<W, F32, GS, 1, 4, 4, 2>(a, slots, s);
      else return launch<W, F32, GS, 1, 2, 4>(a, slots, s);
    }
    if (F32 || a.offsets || avg >= 5) {
      if (blocks > 512) return launch_rb<W, F32, GS, 3>(a, avg, slots, s);
      if (blocks > 256) return launch_rb<W, F32, GS, 2>(a, avg, slots, s);
    }
  }
  return launch_rb<W, F32, GS, 1>(a, avg, slots, s);
}

// In how many parts K is taken, where the row blocks leave most CUs without work and a wave's chain of tiles is long (by us a tile as
// measured at K = 4096). us without and with: 31 f32 rows 150 x 12128 43 and 11, 63 f32 rows 1024 x 8192 58 and 21, 2048 x 4096 32 and
// 21, 5 f32 rows 512 x 12288 15.6 and 8.2, 32 bf16 rows 512 x 12288 24 and 10; the host takes 4 more a call.
inline int parts_of(int64_t rows, int64_t n, int64_t k, int E, bool f32) {
  const int64_t slots = std::min<int64_t>(E, rows), avg = (rows + slots - 1) / slots, blocks = (n + 15) / 16 * slots;
  if (avg <= 1 || avg > 64) return 1;
  const float tiles = (float)k / (128.f * kWaves), us = tiles * (f32 ? 2.4f : 1.1f) * (avg <= 16 ? 1.f : avg <= 32 ? 1.7f : 3.3f);
  int p = 1;
  while (p < 16 && blocks * 2 * p <= 256 && tiles >= 2.f * p && us / p > 10.f) p *= 2;
  return p;
}

}  // namespace few
}  // namespace qmm

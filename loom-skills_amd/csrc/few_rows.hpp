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
// of x come from an MFMA with ones.
#pragma once
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
// four codes in the low nibbles of four bytes as two bf16 pairs: 0000qqqq read as OCP E4M3 is q 2^-9 exactly
__device__ __forceinline__ u32x4 codes(u32 w) {
  const u32 lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
  return u32x4{__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true))};
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
// tiles of 16 tokens at a time. Grid: (16-row blocks of W, experts with rows, token chunks of a dense call).
template <int W, bool F32, int GS, int TT>
__global__ __launch_bounds__(64 * kWaves) void few_rows_kernel(Args a) {
  constexpr int kParts = F32 ? 3 : 1, kLoads = F32 ? 2 : 1, kES = F32 ? 4 : 2;
  constexpr int U = W == kW4 ? 4 : 2;   // tiles of a wave whose weights are in flight
  __shared__ __align__(16) float red[kWaves][TT][64][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, h = lane >> 4, rb = blockIdx.x;
  int e = 0, lo = 0, hi = a.rows;
  if (a.offsets && !nth_segment(a.offsets, a.E, a.rows, blockIdx.y, e, lo, hi)) return;
  const int KT = (a.k + 127) >> 7, nb = (a.n + 15) >> 4;
  const u8 *w = a.w + (int64_t)e * a.w_expert;
  const u32 *ws = nullptr;
  __amdgpu_buffer_rsrc_t wr;
  if constexpr (W == kW4) {
    w += (int64_t)rb * KT * 1024;
    ws = a.ws + ((int64_t)e * nb + rb) * a.groups * 16 + c;
  } else {
    wr = rsrc(w + (int64_t)rb * 32 * a.k, (u32)(min(16, a.n - 16 * rb) * a.k * 2));
  }
  const u32 one = W == kWF16 ? 0x3C003C00u : 0x3F803F80u;
  const u32x4 ones = {one, one, one, one};

  for (int t0 = lo + (int)blockIdx.z * 16 * TT; t0 < hi; t0 += (int)gridDim.z * 16 * TT) {
    const __amdgpu_buffer_rsrc_t xr = rsrc(a.x + (int64_t)t0 * a.k * kES, (u32)min(16 * TT, hi - t0) * (u32)a.k * kES);
    f32x4 acc[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int tb = wave; tb < KT; tb += kWaves * U) {
      u32x4 q[U][W == kW4 ? 1 : 4];
      u32 sc[U][4 / GS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = min(tb + kWaves * u, KT - 1);
        if constexpr (W == kW4) {
          q[u][0] = *reinterpret_cast<const u32x4 *>(w + (int64_t)t * 1024 + 16 * lane);
#pragma unroll
          for (int g = 0; g < 4 / GS; ++g) sc[u][g] = ws[min((4 * t + GS * g) >> a.gshift, a.groups - 1) * 16];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int kk = 128 * t + 32 * j + 8 * h;
            q[u][j] = ld(wr, kk < a.k ? (u32)(c * a.k + kk) * 2u : kPast);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = tb + kWaves * u;
        if (t >= KT) break;
        u32x4 xv[TT][4][kLoads];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int p = 0; p < kLoads; ++p) {
              const int kk = 128 * t + 32 * j + 8 * h;
              xv[tt][j][p] = ld(xr, kk < a.k ? ((u32)(16 * tt + c) * (u32)a.k + (u32)kk) * kES + 16 * p : kPast);
            }
#pragma unroll
        for (int g = 0; g < 4 / GS; ++g) {
          f32x4 dot[TT], sum[TT];
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) dot[tt] = sum[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int jj = 0; jj < GS; ++jj) {
            const int j = GS * g + jj;
            u32x4 wf;
            if constexpr (W == kW4) wf = codes(q[u][0][j]);
            else wf = q[u][j];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
              Parts xp;
              if constexpr (F32) xp = split(xv[tt][j][0], xv[tt][j][kLoads - 1]);
              else xp.p[0] = xv[tt][j][0];
#pragma unroll
              for (int p = kParts - 1; p >= 0; --p) {
                if constexpr (W == kW4) {
                  dot[tt] = mfma<W>(xp.p[p], wf, dot[tt]);
                  sum[tt] = mfma<W>(xp.p[p], ones, sum[tt]);
                } else {
                  acc[tt] = mfma<W>(xp.p[p], wf, acc[tt]);
                }
              }
            }
          }
          if constexpr (W == kW4) {
            const float s = f16_to_f32(sc[u][g]), z = (float)(sc[u][g] >> 16 & 15u);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[tt][i] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[tt][i], dot[tt][i]), acc[tt][i]);
          }
        }
      }
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) *reinterpret_cast<f32x4 *>(red[wave][tt][lane]) = acc[tt];
    __syncthreads();
    for (int v = tid; v < 256 * TT; v += 64 * kWaves) {   // output (token v / 16, row v % 16), the waves' sums in order
      const int token = v >> 4, r = v & 15, l = ((token & 15) >> 2) * 16 + r;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) s += red[i][token >> 4][l][token & 3];
      if (t0 + token < hi && 16 * rb + r < a.n) {
        const int64_t at = (int64_t)(t0 + token) * a.n + 16 * rb + r;
        if (a.y_bytes == 4) static_cast<float *>(a.y)[at] = s;
        else if constexpr (W == kWF16) static_cast<_Float16 *>(a.y)[at] = (_Float16)s;
        else static_cast<__bf16 *>(a.y)[at] = (__bf16)s;
      }
    }
    __syncthreads();
  }
}

// Rows behind the last segment are not written. All extents are checked by the callers.
template <int W, bool F32, int GS>
int launch_tt(const Args &a, hipStream_t s) {
  const int slots = a.offsets ? min(a.E, a.rows) : 1;
  const int avg = a.offsets ? (a.rows + a.E - 1) / a.E : a.rows;   // tokens at a time: as many as a segment may hold
  const dim3 blk(64 * kWaves);
  const unsigned nb = (unsigned)((a.n + 15) / 16);
  auto chunks = [&](int tt) { return a.offsets ? 1u : (unsigned)min((a.rows + 16 * tt - 1) / (16 * tt), 65535); };
  if (avg <= 16) few_rows_kernel<W, F32, GS, 1><<<dim3(nb, slots, chunks(1)), blk, 0, s>>>(a);
  else if (avg <= 32) few_rows_kernel<W, F32, GS, 2><<<dim3(nb, slots, chunks(2)), blk, 0, s>>>(a);
  else few_rows_kernel<W, F32, GS, 4><<<dim3(nb, slots, chunks(4)), blk, 0, s>>>(a);
  return launch_status();
}

}  // namespace few
}  // namespace qmm

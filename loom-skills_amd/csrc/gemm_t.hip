// The transposed product of GGUF-block weights, Y = X W: the gradient of a projection y = x W^T with respect to x, where W
// stays quantized and frozen.
//
//   qmm_gemm_t        Y[t, c] = inv[t] (sum_f X16[t, 0, f] W[f, c] + sum_f X16[t, 1, f] W2[f, c]),  c < k, f < n
//   qmm_grad_operand  X16 and inv from gradient rows: the row-scaled f16 form of qmm_row_scale_f16 over all parts of a row,
//                     each part's n values padded with zeros to a multiple of 64
//
// W [n, k] holds its values along c, the output's columns, so the sum runs down the matrix's rows. W is dequantized to f16
// with the forward GEMM's roundings (deq_f16.hpp), so the gradient is that of the product that the forward GEMM computes;
// fp32 accumulation.
//
// Design (v_mfma_f32_32x32x16_f16, eight waves a workgroup, one workgroup a CU). A workgroup owns BM rows x 256 columns, one
// super-block column of W, and walks down the rows f 64 at a time. The MFMA wants 8 consecutive f of one column in a lane,
// the blocks hold consecutive columns of one f, so the weights are transposed on their way into LDS: a thread takes one code
// dword of four rows f .. f + 3 (32 neighbouring lanes a row's 128 code bytes), interleaves the rows' bytes with v_perm, so
// that the two f16 halves of every packed instruction are two rows f of one column with the two rows' scales, and stores
// four f16 (f .. f + 3 of a column) at a time. Each weight is dequantized once per workgroup.
//   - LDS rows are 64 f = 128 bytes, one a column (weights) or an output row (activations); chunk i of 16 bytes lies at
//     i ^ swizzle(c), so that the 16 columns or rows that a fragment read covers at a time (256 bytes, all 64 banks), and the
//     8 columns, 4 apart, that a weight store covers, lie in different banks. Both are double-buffered: one barrier a step.
//   - X16 goes straight into LDS (buffer_load ... lds) a step ahead; code dwords and block headers are loaded two and three
//     steps ahead into registers.
//   - Between a step's MFMAs the wave brings in the next step's weights.
//   - Scales: 64 rows x 8 sub-blocks are one (f16(d sc), f16(-dmin m)) pair a thread, decoded one step ahead into an LDS table
//     [sub-block][f], from which a thread reads its four rows' scales as 8 bytes.
// Few output tiles are split along f over the grid's y: each part writes its f32 sums to the workspace and a second launch
// adds the parts in order. 2048 rows, two Q4_K matrices of 12288 x 4096: 386 us, 1.07 PFLOP/s, the matrix pipe 0.57 busy at
// the clock the power limit leaves it (an f16 library product of the shape 304 to 497 us by its orientation).
#include "act_quant.hpp"
#include "gemm_tile_kernel.hpp"

using namespace qmm;

namespace {

enum { kQ4K = tile::kQ4K, kQ4KT = tile::kQ4KT, kQ6K = tile::kQ6K, kQ40 = tile::kQ40 };
typedef __attribute__((ext_vector_type(4))) u32 u32x4;
typedef __attribute__((ext_vector_type(2))) u32 u32x2;

constexpr int kBN = 256, kBF = 64, kThreads = 512;
constexpr int kBBytes = kBN * kBF * 2, kRun = 72, kTable = 16 * kRun * 2;   // LDS bytes of a step's weights and
                                                                             // scale table (runs of 64 f16, 16 bytes apart)
constexpr int kGroupM = 8;

// The 16-byte chunk of an LDS row of 128 bytes is moved by this much: bits 1-3 of the column (bit 0 picks the row's half of
// the banks) for the reads, bits 4 and 5 for the stores, whose columns differ in bits 2-4 (Q4_0: 2, 3 and 5).
__device__ __forceinline__ int swizzle(int c) { return ((c >> 1) & 7) ^ ((c >> 4) & 1) ^ ((c >> 5) & 1); }

struct GArgs {
  int T, K, n, n64;
  const _Float16 *x16;         // [T, parts, n64]
  const float *scales;         // [T, 2]
  const u8 *w, *w2;
  void *y;
  int y_bf16;
  float *part;                 // splits > 1: [splits, T, K]
  int tiles_m, tiles_n, splits;
};

// a thread's raw words of a step: a code dword of four rows (Q6_K: the low and the high bits), and the header of the one row
// whose scales it decodes
template <int WF>
struct Raw {
  u32 q[4], qh[WF == kQ6K ? 4 : 1];
};
template <int WF>
struct Head {
  uint4 v;
};

template <int WF, int BM>
__global__ __launch_bounds__(kThreads, 2) void gemm_t_kernel(GArgs a) {
  constexpr int NI = BM / 64, kABytes = BM * 128;
  extern __shared__ __align__(1024) u8 smem[];   // weights [2], activations [2], scale tables [2]
  u8 *const bs = smem, *const as = smem + 2 * kBBytes, *const ts = as + 2 * kABytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 31, h = lane >> 5;

  // XCD-aware order: workgroup b runs on XCD b % 8, which gets a contiguous range of tiles in groups of kGroupM row tiles,
  // rows fastest: the tiles of an XCD at a time share weight columns and activation rows in its L2
  const int per = (int)(gridDim.x / 8);
  const int t = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if (t >= a.tiles_m * a.tiles_n) return;
  const int g = t / (kGroupM * a.tiles_n), gm = min(kGroupM, a.tiles_m - g * kGroupM), gt = t - g * kGroupM * a.tiles_n;
  const int m0 = (g * kGroupM + gt % gm) * BM, cb = gt / gm;

  const int per_matrix = a.n64 / kBF, steps = a.w2 ? 2 * per_matrix : per_matrix;
  const int s0 = (int)((int64_t)blockIdx.y * steps / a.splits), s1 = (int)((int64_t)(blockIdx.y + 1) * steps / a.splits);
  const int R = steps * kBF;   // values of an activation row

  // ---- activations, straight into LDS: load i of a wave is rows 8 (8 i + wave) .. + 7, lane l's 16 bytes chunk
  // (l % 8) ^ swizzle(row) of row l / 8
  constexpr int ND = BM / 64;
  const uint64_t xa = (uint64_t)a.x16;
  const u32x4 xrs = {(u32)xa, (u32)(xa >> 32) & 0xFFFFu, (u32)((int64_t)a.T * R * 2), 0x00020000u};
  u32 aoff[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int r = 8 * (8 * i + wave) + (lane >> 3), row = m0 + r;
    aoff[i] = row < a.T ? (u32)row * (u32)R * 2u + (u32)(((lane & 7) ^ swizzle(r)) * 16) : 0x80000000u;   // rows past T: zeros
  }
  const u32 lds0 = (u32)(uintptr_t)(__attribute__((address_space(3))) u8 *)as;
  auto load_x = [&](int buf, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
      tile::lds_load16(xrs, aoff[i], (u32)(s * 128), __builtin_amdgcn_readfirstlane(lds0 + (u32)(buf * kABytes + (8 * i + wave) * 1024)));
  };

  // vmcnt(0), as the builtin: the compiler, which does not count the loads into LDS, then knows that its own have landed too
  auto wait_loads = []() __attribute__((always_inline)) { __builtin_amdgcn_s_waitcnt(0x0F70); };

  // ---- weights: rows 4 fq .. + 3 of a step, code dword dw of the super-block (Q4_0: of its eight blocks)
  const int64_t RB = tile::row_bytes_of(WF, a.K);
  const int fq = 2 * wave + h, dw = lc;
  auto matrix = [&](int s) { return s >= per_matrix ? a.w2 : a.w; };
  auto first_row = [&](int s) { return (s >= per_matrix ? s - per_matrix : s) * kBF; };
  // address of byte `at` of super-block cb of row f (tiled: `at` in the tiled unit, for row 0 of 16)
  auto row_at = [&](const u8 *m, int f) {
    f = min(f, a.n - 1);   // rows past n (multiplied by zero activations and zero scales) read the last one
    if constexpr (WF == kQ4KT) return m + (int64_t)(f >> 4) * 16 * RB + (int64_t)(cb >> 1) * 4608;
    else return m + (int64_t)f * RB + (int64_t)cb * (WF == kQ6K ? 210 : 144);
  };
  auto load_codes = [&](int s, Raw<WF> &r) __attribute__((always_inline)) {
    const u8 *m = matrix(s);
    const int f0 = first_row(s) + 4 * fq;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u8 *b = row_at(m, f0 + i);
      if constexpr (WF == kQ4K) {
        r.q[i] = *reinterpret_cast<const u32 *>(b + 16 + 4 * dw);
      } else if constexpr (WF == kQ4KT) {   // code bytes 16 pc .. of the super-block, pc = 4 h' + q, in plane q
        const int pc = dw >> 2, rr = min(f0 + i, a.n - 1) & 15;
        r.q[i] = *reinterpret_cast<const u32 *>(b + 512 + 1024 * (pc & 3) + 16 * (4 * rr + 2 * (cb & 1) + (pc >> 2)) + 4 * (dw & 3));
      } else if constexpr (WF == kQ6K) {    // ql byte 4 dw of half dw / 16, and the qh byte of the same values
        r.q[i] = ld4u(b + 4 * dw);
        r.qh[i] = ld4u(b + 128 + 32 * (dw >> 4) + 4 * (dw & 7));
      } else {
        r.q[i] = ld4u(b + 18 * (dw >> 2) + 2 + 4 * (dw & 3));
      }
    }
  };
  // the header words of row tid / 8 of a step, for sub-block tid % 8
  auto load_head = [&](int s, Head<WF> &hd) __attribute__((always_inline)) {
    const int f = first_row(s) + (tid >> 3), g8 = tid & 7;
    const u8 *b = row_at(matrix(s), f);
    if constexpr (WF == kQ4K) hd.v = ld16(b);
    else if constexpr (WF == kQ4KT) hd.v = ld16(b + 32 * (min(f, a.n - 1) & 15) + 16 * (cb & 1));
    else if constexpr (WF == kQ6K)
      hd.v = make_uint4(*reinterpret_cast<const u16 *>(b + 192 + 2 * g8), *reinterpret_cast<const u16 *>(b + 208), 0u, 0u);
    else hd.v = make_uint4(*reinterpret_cast<const u16 *>(b + 18 * g8), 0u, 0u, 0u);
  };
  // the scale table of a step, f16: Q4_K [2 (d sc, -dmin m)][8 sub-blocks][64 f], Q6_K [16 runs][64 f], Q4_0 [8 blocks][64 f]
  auto decode = [&](int buf, int s, const Head<WF> &hd) __attribute__((always_inline)) {
    _Float16 *tb = reinterpret_cast<_Float16 *>(ts + buf * kTable);
    const int fr = tid >> 3, g8 = tid & 7;
    const bool live = first_row(s) + fr < a.n;
    if constexpr (WF == kQ4K || WF == kQ4KT) {
      u32 sc, mn;
      q4k_scale_min(hd.v.y, hd.v.z, hd.v.w, g8, sc, mn);
      const float d = f16_to_f32(hd.v.x) * (float)sc, m = -(f16_to_f32(hd.v.x >> 16) * (float)mn);
      tb[g8 * kRun + fr] = (_Float16)(live ? d : 0.f);
      tb[(8 + g8) * kRun + fr] = (_Float16)(live ? m : 0.f);
    } else if constexpr (WF == kQ6K) {
      const float d = f16_to_f32(hd.v.y);
      const float a0 = d * (float)(signed char)(hd.v.x & 0xFFu), a1 = d * (float)(signed char)(hd.v.x >> 8);
      tb[(2 * g8) * kRun + fr] = (_Float16)(live ? a0 : 0.f);
      tb[(2 * g8 + 1) * kRun + fr] = (_Float16)(live ? a1 : 0.f);
    } else {
      const u16 d = live ? (u16)hd.v.x : (u16)0;
      tb[g8 * kRun + fr] = __builtin_bit_cast(_Float16, d);
    }
  };
  // columns (in the tile) of the four low-nibble values of the thread's dword; the high nibbles lie kHigh further
  constexpr int kHigh = WF == kQ6K ? 64 : WF == kQ40 ? 16 : 32;
  const int col0 = WF == kQ6K ? 128 * (dw >> 4) + 4 * (dw & 15) : WF == kQ40 ? 32 * (dw >> 2) + 4 * (dw & 3) : 64 * (dw >> 3) + 4 * (dw & 7);
  auto dequant = [&](int buf, const Raw<WF> &r, int s) __attribute__((always_inline)) {   // s: nibble
    const _Float16 *tb = reinterpret_cast<const _Float16 *>(ts + buf * kTable);
    u8 *out = bs + buf * kBBytes;
    const int c0 = col0 + kHigh * s;
    const int run = WF == kQ6K ? c0 >> 4 : c0 >> 5;   // the values' scale
    const u32x2 sc = *reinterpret_cast<const u32x2 *>(tb + run * kRun + 4 * fq);
    u32x2 mn = {0u, 0u};
    if constexpr (WF == kQ4K || WF == kQ4KT) mn = *reinterpret_cast<const u32x2 *>(tb + (8 + run) * kRun + 4 * fq);
    u32 nb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      nb[i] = (s ? r.q[i] >> 4 : r.q[i]) & 0x0F0F0F0Fu;
      if constexpr (WF == kQ6K) {   // group 2 s + (dw / 8) % 2 of the half: bits 2 group of the qh byte
        const int gb = 4 * s + 2 * ((dw >> 3) & 1);
        nb[i] |= ((r.qh[i] >> gb) & 0x03030303u) << 4;
      }
    }
    u32 o[4][2];   // [column][pair of rows]
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const u32 lo = __builtin_amdgcn_perm(nb[2 * p + 1], nb[2 * p], 0x05010400u);   // columns 0, 1: (row 2p, row 2p + 1)
      const u32 hi = __builtin_amdgcn_perm(nb[2 * p + 1], nb[2 * p], 0x07030602u);   // columns 2, 3
      const h2 ds = as_h2(sc[p]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32 b = c < 2 ? lo : hi;
        if constexpr (WF == kQ4K || WF == kQ4KT) {
          const h2 q = c & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 512.0f, true)
                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 512.0f, false);
          o[c][p] = as_u32(__builtin_elementwise_fma(q, ds, as_h2(mn[p])));
        } else {   // (1024 + code) - (1024 + 32 or 8) exactly, then one rounding multiply
          const h2 q = as_h2(__builtin_amdgcn_perm(0x64646464u, b, c & 1 ? 0x04030402u : 0x04010400u));
          o[c][p] = as_u32((q + as_h2(WF == kQ6K ? 0xE420E420u : 0xE408E408u)) * ds);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int cc = c0 + c;
      *reinterpret_cast<u32x2 *>(out + cc * 128 + (((fq >> 1) ^ swizzle(cc)) * 16) + 8 * (fq & 1)) = u32x2{o[c][0], o[c][1]};
    }
  };

  f32x16 acc[NI][2];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  // the wave's BM / 2 rows x 64 columns
  const int wm = wave >> 2, wn = wave & 3;
  // A step's products from buffer buf; part(kk) is work for the vector pipe and LDS beside the MFMAs of K16 step kk, which read
  // their fragments a K16 step ahead.
  auto multiply = [&](int buf, auto part) __attribute__((always_inline)) {
    const u8 *ab = as + buf * kABytes + (wm * (BM / 2) + lc) * 128, *bb = bs + buf * kBBytes + (64 * wn + lc) * 128;
    const int sw = swizzle(lc);   // 32 more rows or columns flip its bit 0
    f16x8 af[2][NI], bf[2][2];
    auto read = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) bf[kk & 1][j] = *reinterpret_cast<const f16x8 *>(bb + j * 4096 + (((2 * kk + h) ^ sw ^ j) * 16));
#pragma unroll
      for (int i = 0; i < NI; ++i)
        af[kk & 1][i] = *reinterpret_cast<const f16x8 *>(ab + i * 4096 + (((2 * kk + h) ^ sw ^ ((wm * NI + i) & 1)) * 16));
    };
    read(0);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk < 3) read(kk + 1);
      part(kk);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[kk & 1][i], bf[kk & 1][j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // ---- step s multiplies buffer s % 2 while step s + 1 is brought into the other one, with the scale table that step s - 1
  // has decoded; slot s % 2 of the registers holds the codes of step s (headers: of step s + 1). A step's loads, the codes of
  // step s + 2, the headers of s + 3 and the activations of s + 1, are issued at its start and awaited at its end. Loads past
  // the last step repeat it.
  auto clamp = [&](int s) { return min(s, s1 - 1); };
  Raw<WF> raw[2];
  Head<WF> head[2];
  load_head(s0, head[1]);
  load_codes(s0, raw[0]);
  load_head(clamp(s0 + 1), head[0]);
  load_codes(clamp(s0 + 1), raw[1]);
  load_x(0, s0);
  decode(0, s0, head[1]);
  load_head(clamp(s0 + 2), head[1]);
  __syncthreads();
  dequant(0, raw[0], 0);
  dequant(0, raw[0], 1);
  decode(1, clamp(s0 + 1), head[0]);
  wait_loads();
  __syncthreads();
  auto step = [&](auto parity, int s) __attribute__((always_inline)) {
    constexpr int cur = decltype(parity)::value, nx = cur ^ 1;
    load_codes(clamp(s + 2), raw[cur]);
    load_head(clamp(s + 3), head[cur]);
    load_x(nx, clamp(s + 1));
    multiply(cur, [&](int kk) __attribute__((always_inline)) {
      if (kk == 0) decode(cur, clamp(s + 2), head[nx]);
      else if (kk < 3) dequant(nx, raw[nx], kk - 1);
    });
    wait_loads();
    __syncthreads();
  };
  int s = s0;
  for (; s + 1 < s1; s += 2) {
    step(std::integral_constant<int, 0>{}, s);
    step(std::integral_constant<int, 1>{}, s + 1);
  }
  if (s < s1) multiply(0, [](int) {});   // the last of an odd count

  // ---- accumulator register r of a block is row 8 (r / 4) + 4 h + r % 4, column lc
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = m0 + wm * (BM / 2) + 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
      if (row >= a.T) continue;
      const float inv = a.splits > 1 ? 1.f : a.scales[2 * row + 1];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int64_t o = (int64_t)row * a.K + cb * kBN + 64 * wn + 32 * j + lc;
        if (a.splits > 1) a.part[(int64_t)blockIdx.y * a.T * a.K + o] = acc[i][j][r];
        else store_val(a.y, a.y_bf16, o, acc[i][j][r] * inv);
      }
    }
}

// the parts' sums in order, times the row's inverse scale; four values a thread (K % 256 == 0)
__global__ __launch_bounds__(256) void gemm_t_join_kernel(int64_t quads, int K, int splits, const float *__restrict__ part,
                                                          const float *__restrict__ scales, void *__restrict__ y, int y_bf16) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  f32x4 s = reinterpret_cast<const f32x4 *>(part)[i];
  for (int z = 1; z < splits; ++z) s += reinterpret_cast<const f32x4 *>(part)[(int64_t)z * quads + i];
  const float inv = scales[2 * (4 * i / K) + 1];
#pragma unroll
  for (int q = 0; q < 4; ++q) store_val(y, y_bf16, 4 * i + q, s[q] * inv);
}

// 2^-e brings the largest magnitude m into [2^13, 2^14), up to the largest floats' 2^127 (e = 114): gradients are small, so e may
// be negative (the forward operand's is not); a row of zeros or subnormals, or with infinities, takes e = 0 (NaN values are passed over and stay NaN)
__device__ __forceinline__ int grad_exponent(float m) {
  const int biased = (int)((f32_as_u32(m) >> 23) & 255u);
  return biased == 0 || biased == 255 ? 0 : max(biased - 140, -126);
}
__device__ __forceinline__ float pow2(int e) { return u32_as_f32((u32)(127 + e) << 23); }
// the row's maximum over a workgroup of NT threads
template <int NT>
__device__ __forceinline__ float block_max(float m) {
  __shared__ float part[NT / 64];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = part[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, part[i]);
  return m;
}

// A row's parts x n values into the f16 operand, a workgroup a row. n % 8 == 0, 16-byte aligned rows of at most 8 NT J values:
// the row is read once, into registers.
template <int NT, int J>
__global__ __launch_bounds__(NT) void grad_operand_kernel(int64_t rows, int parts, int n, int n64, const void *__restrict__ x, int bf,
                                                          _Float16 *__restrict__ x16, float *__restrict__ scales) {
  const int64_t row = item_index();
  if (row >= rows) return;
  const int chunks = parts * (n / 8), padded = parts * (n64 / 8);
  float v[J][8], m = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) load8_act(x, bf, 8 * (row * chunks + min((int)threadIdx.x + NT * j, chunks - 1)), v[j]);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[j][i]));   // past the row its last chunk again
  const int e = grad_exponent(block_max<NT>(m));
  const float sc = pow2(-e);
  if (threadIdx.x == 0) *reinterpret_cast<float2 *>(scales + 2 * row) = make_float2(sc, pow2(e));
  f16x8 *const out = reinterpret_cast<f16x8 *>(x16) + row * padded;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (int)threadIdx.x + NT * j, p = c >= n / 8 ? 1 : 0;   // two parts at most
    f16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (_Float16)(v[j][i] * sc);
    if (c < chunks) out[c + p * ((n64 - n) / 8)] = o;
  }
  const int pad = (n64 - n) / 8;   // fewer than 8 chunks a part
  if ((int)threadIdx.x < parts * pad) {
    const int p = (int)threadIdx.x / pad;
    out[p * (n64 / 8) + n / 8 + (int)threadIdx.x % pad] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}
// any n and alignment: the row is read twice, the second time from L2 (2048 rows of 2 x 12288 bf16: 77 us, 33 above)
__global__ __launch_bounds__(256) void grad_operand_any_kernel(int64_t rows, int parts, int n, int n64, const void *__restrict__ x, int bf,
                                                               _Float16 *__restrict__ x16, float *__restrict__ scales) {
  const int64_t row = item_index(), in0 = row * parts * n, out0 = row * parts * n64;
  if (row >= rows) return;
  const int total = parts * n;
  float m = 0.f;
  for (int c = threadIdx.x; c < total; c += 256) m = fmaxf(m, fabsf(load_val(x, bf, in0 + c)));
  const int e = grad_exponent(block_max<256>(m));
  const float sc = pow2(-e);
  if (threadIdx.x == 0) {
    scales[2 * row] = sc;
    scales[2 * row + 1] = pow2(e);
  }
  for (int p = 0; p < parts; ++p)
    for (int c = threadIdx.x; c < n64; c += 256)
      x16[out0 + (int64_t)p * n64 + c] = c < n ? (_Float16)(load_val(x, bf, in0 + (int64_t)p * n + c) * sc) : (_Float16)0.f;
}

int64_t n64_of(int64_t n) { return (n + kBF - 1) / kBF * kBF; }
// The rows of a tile and the parts along f: the least time, where every CU walks its share of (tile, part) pairs. Measured with
// a full chip (Q4_K, K = 4096, two matrices of 12288 rows): a step of 64 rows of W takes a tile of 64 output rows 0.84 us, 128
// 1.25, 256 1.92; the parts' sums cost their f32 traffic and a launch. 2048 rows: 386 us in two parts of 256-row tiles, 461 on
// 128-row tiles, 645 on 64; 100 rows: 47 in 16 parts of 128-row tiles, 59 in eight of 64-row tiles, 406 in one part; 4096
// rows 738 / 914 / 1290. A matrix of 768 rows, K = 2048: 14.0 us at 100 rows on 64-row tiles, 16.4 on 128.
struct Plan { int bm, splits; };
Plan plan_of(int64_t rows, int64_t k, int64_t n, bool two) {
  const int64_t steps = n64_of(n) / kBF * (two ? 2 : 1);
  Plan best{0, 1};
  double least = 0;
  for (int bm : {64, 128, 256}) {
    const double step = bm == 64 ? 0.84 : bm == 128 ? 1.25 : 1.92;
    const int64_t tiles = (rows + bm - 1) / bm * (k / kBN);
    for (int64_t s = 1; s <= 32 && s <= (steps + 3) / 4; ++s) {
      const double t = (double)((tiles * s + 255) / 256) * (double)((steps + s - 1) / s) * step + (s > 1 ? 3 + 2e-6 * (double)(s * rows * k) : 0);
      if (!best.bm || t < least) { best = Plan{bm, (int)s}; least = t; }
    }
  }
  return best;
}

template <int WF, int BM>
int launch(const GArgs &a, hipStream_t s) {
  constexpr int kLds = 2 * (kBBytes + BM * 128 + kTable);
  static std::atomic<unsigned> raised{0};
  const void *fn = reinterpret_cast<const void *>(&gemm_t_kernel<WF, BM>);
  if (int st = raise_dyn_lds(fn, kLds, raised)) return st;
  const int tiles = a.tiles_m * a.tiles_n;
  gemm_t_kernel<WF, BM><<<dim3((unsigned)(8 * ((tiles + 7) / 8)), (unsigned)a.splits), kThreads, kLds, s>>>(a);
  if (int st = launch_status()) return st;
  if (a.splits > 1) {
    const int64_t quads = (int64_t)a.T * a.K / 4;
    gemm_t_join_kernel<<<(unsigned)((quads + 255) / 256), 256, 0, s>>>(quads, a.K, a.splits, a.part, a.scales, a.y, a.y_bf16);
    return launch_status();
  }
  return QMM_OK;
}

template <int WF>
int dispatch(int bm, const GArgs &a, hipStream_t s) {
  if (bm == 64) return launch<WF, 64>(a, s);
  return bm == 128 ? launch<WF, 128>(a, s) : launch<WF, 256>(a, s);
}

int check_shape(int fmt, int64_t rows, int64_t k, int64_t n, bool two) {
  if (fmt != QMM_Q4_K && fmt != QMM_Q4_KT && fmt != QMM_Q6_K && fmt != QMM_Q4_0) return QMM_ERR_FORMAT;
  if (rows <= 0 || k <= 0 || n <= 0 || rows > (1 << 24) || k > (1 << 20) || n > (1 << 24) || k % 256) return QMM_ERR_SHAPE;
  if (fmt == QMM_Q4_KT && (n % 16 || k % 512)) return QMM_ERR_SHAPE;   // whole 16-row blocks of whole 512-value units
  if (rows * n64_of(n) * (two ? 2 : 1) * 2 >= (1ll << 31)) return QMM_ERR_SHAPE;   // activations: 32-bit buffer offsets
  return QMM_OK;
}

}  // namespace

extern "C" int qmm_grad_operand(int64_t rows, int parts, int64_t n, const void *x, int x_dtype, void *x16, float *scales,
                                qmm_stream_t stream) {
  if (!x || !x16 || !scales) return QMM_ERR_NULL;
  if (x_dtype != QMM_F32 && x_dtype != QMM_BF16) return QMM_ERR_DTYPE;
  if (parts != 1 && parts != 2) return QMM_ERR_RANGE;
  if (rows <= 0 || n <= 0 || rows > (1 << 24) || n > (1 << 24)) return QMM_ERR_SHAPE;
  if (!aligned(x, x_dtype == QMM_BF16 ? 2 : 4) || !aligned(x16, 16) || !aligned(scales, 4)) return QMM_ERR_ALIGN;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t chunks = parts * (n / 8);
  auto go = [&](auto *kernel, int threads) {
    kernel<<<item_grid(rows), threads, 0, s>>>(rows, parts, (int)n, (int)n64_of(n), x, x_dtype == QMM_BF16,
                                               static_cast<_Float16 *>(x16), scales);
    return launch_status();
  };
  if (n % 8 || !aligned(x, 16) || !aligned(scales, 8) || chunks > 8192) return go(grad_operand_any_kernel, 256);
  if (chunks <= 256) return go(grad_operand_kernel<256, 1>, 256);
  if (chunks <= 1024) return go(grad_operand_kernel<512, 2>, 512);
  if (chunks <= 2048) return go(grad_operand_kernel<1024, 2>, 1024);
  if (chunks <= 4096) return go(grad_operand_kernel<1024, 4>, 1024);
  return go(grad_operand_kernel<1024, 8>, 1024);
}

extern "C" int64_t qmm_gemm_t_workspace_size(int fmt, int64_t rows, int64_t k, int64_t n, int two) {
  if (check_shape(fmt, rows, k, n, two != 0) != QMM_OK) return -1;
  const int s = plan_of(rows, k, n, two != 0).splits;
  return s > 1 ? s * rows * k * 4 : 0;
}

extern "C" int qmm_gemm_t(int fmt, int64_t rows, int64_t k, int64_t n, const void *x, const float *scales, const void *w,
                          const void *w2, void *y, int y_dtype, void *workspace, int64_t workspace_bytes,
                          qmm_stream_t stream) {
  if (int st = check_shape(fmt, rows, k, n, w2 != nullptr)) return st;
  if (!x || !scales || !w || !y) return QMM_ERR_NULL;
  if (y_dtype != QMM_F32 && y_dtype != QMM_BF16) return QMM_ERR_DTYPE;
  const size_t wal = fmt == QMM_Q4_K || fmt == QMM_Q4_KT ? 16 : fmt == QMM_Q6_K ? 4 : 2;
  if (!aligned(x, 16) || !aligned(scales, 4) || !aligned(w, wal) || !aligned(w2, wal) || !aligned(y, y_dtype == QMM_BF16 ? 2 : 4))
    return QMM_ERR_ALIGN;
  GArgs a{};
  const Plan plan = plan_of(rows, k, n, w2 != nullptr);
  const int bm = plan.bm;
  a.splits = plan.splits;
  if (a.splits > 1) {
    if (!workspace || workspace_bytes < a.splits * rows * k * 4) return QMM_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return QMM_ERR_ALIGN;
  }
  a.T = (int)rows; a.K = (int)k; a.n = (int)n; a.n64 = (int)n64_of(n);
  a.x16 = static_cast<const _Float16 *>(x); a.scales = scales;
  a.w = static_cast<const u8 *>(w); a.w2 = static_cast<const u8 *>(w2);
  a.y = y; a.y_bf16 = y_dtype == QMM_BF16; a.part = static_cast<float *>(workspace);
  a.tiles_m = (int)((rows + bm - 1) / bm); a.tiles_n = (int)(k / kBN);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (fmt) {
    case QMM_Q6_K: return dispatch<kQ6K>(bm, a, s);
    case QMM_Q4_0: return dispatch<kQ40>(bm, a, s);
    case QMM_Q4_KT: return dispatch<kQ4KT>(bm, a, s);
    default: return dispatch<kQ4K>(bm, a, s);
  }
}

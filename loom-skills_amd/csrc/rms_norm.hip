// Root-mean-square norm with the residual's addition, written as the operand of the product that follows:
//
//   h = x + residual;   y[c] = (h[c] r) weight[c],   r = 1 / sqrt(sum h^2 / k + eps)
//
//   out QMM_F32 / QMM_BF16   y
//   out QMM_F16              the row-scaled f16 operand of qmm_row_scale_f16(y), scales (2^-e, 2^e)
//   out QMM_Q8               planar Q8_1 of qmm_quant_q8(y)
//   out QMM_MXFP8            E4M3 codes and E8M0 scales of qmm_quant_mxfp8(y)
//
// h is f32 (the norm does not see the rounding of a bf16 h), its squares are summed in f32 in a fixed tree, and y is rounded
// once, by the output form; the operand forms have the bits of the quantizer applied to the f32 y.
//
// k % 8 == 0 and rows on 16 bytes: one pass over memory, a row lives in registers (8 J values a lane, L lanes a row) between
// the sum of its squares and its output, so x and residual are read once and h and y written once, which is what bounds it.
// Rows of up to 512 values take 16, 32 or 64 lanes of a wave (up to 16 rows a workgroup, no barrier), longer ones a workgroup.
// Four neighbouring lanes hold a 32-value group, so an 8-bit scale is two lane exchanges. 4096 x 4096 bf16 with a residual into
// f16: 29.6 us for 134 MB, 4.5 TB/s (25.7 where part of the inputs is in the last-level cache); 65536 x 128 bf16 9.0 us, 3.7 TB/s.
//
// Other k and addresses (f32, bf16 and f16 outputs): a workgroup of 256 threads a row, a value a load, x and residual read twice
// (into f16 three times) from memory and then L2. Its instructions bound it (vector pipes 0.90 busy at 65536 x 100), with most
// lanes idle in short rows: 65536 x 100 bf16 57 us (65536 x 104: 9.0), 4096 x 4095 with a residual 77, into f16 107, 333 x 2881
// 15 (333 x 2880: 5.0).
//
// The backward pass, with hn = h r the normed row and g = weight dy:
//
//   dx = dh + r (g - hn mean_c(g hn));   dweight[c] = sum_rows dy hn
//
// the same layout: sum h^2 and sum g h are one exchange, h, dy and dh are read once and dx written once. For dweight a
// workgroup walks its rows with the column's sum in registers and writes one partial row; a second launch adds the partial
// rows in a fixed order. Memory bounds it (inputs out of cache): 4096 x 4096 bf16 rows with dh 31 us for dx (134 MB, 4.3 TB/s), 48
// with dweight (512 workgroups, a row's loads awaited before the next row's); 65536 x 128 15 and 20. Rows of more than 8192
// values are read twice, with dweight three times: 1024 x 12288 29 and 53. Other k and addresses take that kernel a value a load,
// 512 threads a row, and a column a thread for dweight: 65536 x 100 169 and 526, 4096 x 4095 97 and 125, 333 x 2881 12 and 20.
#include "act_quant.hpp"
#include "bfly.hpp"
#include "epilogue.hpp"

using namespace qmm;

namespace {

constexpr int kMaxK = 32768;   // 1024 lanes of 32 values

struct NArgs {
  int64_t rows, k;
  const void *x, *res, *weight;
  void *h, *out, *scales;
  float eps;
  int x_bf16, res_bf16, w_bf16;
};

__device__ __forceinline__ float norm_rate(float sum, int64_t k, float eps) { return 1.0f / sqrtf(sum / (float)k + eps); }

// the f16 operand's exponent of a row whose largest magnitude is m (qmm_row_scale_f16)
__device__ __forceinline__ int f16_exponent(float m) { return min(max((int)((f32_as_u32(m) >> 23) & 255u) - 140, 0), 100); }
__device__ __forceinline__ float pow2(int e) { return u32_as_f32((u32)(127 + e) << 23); }

__device__ __forceinline__ u32 bf16_pair(float a, float b) {
  return (u32)__builtin_bit_cast(u16, (__bf16)a) | ((u32)__builtin_bit_cast(u16, (__bf16)b) << 16);
}
// 8 values to element offset e of a bf16 or f32 array
__device__ __forceinline__ void store8(void *p, int bf, int64_t e, const float (&v)[8]) {
  if (bf) {
    *reinterpret_cast<v4u *>(static_cast<u16 *>(p) + e) =
        v4u{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
  } else {
    float *f = static_cast<float *>(p) + e;
    *reinterpret_cast<v4u *>(f) = v4u{f32_as_u32(v[0]), f32_as_u32(v[1]), f32_as_u32(v[2]), f32_as_u32(v[3])};
    *reinterpret_cast<v4u *>(f + 4) = v4u{f32_as_u32(v[4]), f32_as_u32(v[5]), f32_as_u32(v[6]), f32_as_u32(v[7])};
  }
}

// v over the row's L lanes (a power of two): a butterfly in the wave, then the waves in order through LDS
template <int L, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *part) {
  constexpr int W = L < 64 ? L : 64;
#pragma unroll
  for (int off = W / 2; off >= 1; off >>= 1) {
    const float o = __shfl_xor(v, off, kWave);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  if constexpr (L > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < L / 64; ++i) v = MAX ? fmaxf(v, part[i]) : v + part[i];
  }
  return v;
}

// L lanes a row, chunk l + L j of 8 values in lane l: k % 8 == 0 (k % 32 for the 8-bit outputs), 16-byte aligned rows
template <int OUT, int L, int J>
__global__ __launch_bounds__(L < 256 ? 256 : L) void rms_norm_kernel(NArgs a) {
  constexpr int kRows = L < 256 ? 256 / L : 1;
  __shared__ float part[2][L > 64 ? L / 64 : 1];
  const int l = threadIdx.x % L;
  const int64_t first = item_index() * kRows, row_ = first + threadIdx.x / L;
  if (first >= a.rows) return;
  const bool alive = row_ < a.rows;
  const int64_t row = alive ? row_ : a.rows - 1;   // lanes of rows past the last stay for the exchanges and store nothing
  const int chunks = (int)(a.k / 8);
  const int64_t r0 = row * a.k;
  float v[J][8];
#pragma unroll
  for (int j = 0; j < J; ++j) load8_act(a.x, a.x_bf16, r0 + 8 * min(l + L * j, chunks - 1), v[j]);
  if (a.res) {
    float t[J][8];
#pragma unroll
    for (int j = 0; j < J; ++j) load8_act(a.res, a.res_bf16, r0 + 8 * min(l + L * j, chunks - 1), t[j]);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] += t[j][i];
  }
  float w[J][8];
#pragma unroll
  for (int j = 0; j < J; ++j) load8_act(a.weight, a.w_bf16, 8 * min(l + L * j, chunks - 1), w[j]);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(v[j][i], v[j][i], s);
    sum += l + L * j < chunks ? s : 0.f;
  }
  if (a.h) {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (alive && l + L * j < chunks) store8(a.h, a.res_bf16, r0 + 8 * (l + L * j), v[j]);
  }
  const float rate = norm_rate(row_reduce<L, false>(sum, part[0]), a.k, a.eps);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rate * w[j][i];

  if constexpr (OUT == QMM_F16) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = l + L * j < chunks ? fmaxf(m, fabsf(v[j][i])) : m;
    const int e = f16_exponent(row_reduce<L, true>(m, part[1]));
    const float sc = pow2(-e);
    if (alive && l == 0) *reinterpret_cast<float2 *>(static_cast<float *>(a.scales) + 2 * row) = make_float2(sc, pow2(e));
#pragma unroll
    for (int j = 0; j < J; ++j) {
      f16x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (_Float16)(v[j][i] * sc);
      if (alive && l + L * j < chunks) *reinterpret_cast<f16x8 *>(static_cast<_Float16 *>(a.out) + r0 + 8 * (l + L * j)) = o;
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = l + L * j;
      const bool in = alive && c < chunks;
      const int64_t e = r0 + 8 * c;
      if constexpr (OUT == QMM_Q8) {
        u32 c0, c1;
        float d16, s;
        q8_group4(v[j], c0, c1, d16, s);
        if (in) {
          *reinterpret_cast<v2u *>(static_cast<u8 *>(a.out) + e) = v2u{c0, c1};
          if ((l & 3) == 0)
            reinterpret_cast<float2 *>(static_cast<u8 *>(a.out) + a.rows * a.k)[e / 32] = make_float2(d16, s);
        }
      } else if constexpr (OUT == QMM_MXFP8) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[j][i]));
        m = fmaxf(m, xshfl<1>(m));
        m = fmaxf(m, xshfl<2>(m));
        const int sx = mxfp8_exponent(m);
        u32 o[2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
          o[q] = (u32)e4m3_pack2<true>(v[j][4 * q + 2], v[j][4 * q + 3], sx, e4m3_pack2<false>(v[j][4 * q], v[j][4 * q + 1], sx, 0));
        if (in) {
          *reinterpret_cast<v2u *>(static_cast<u8 *>(a.out) + e) = v2u{o[0], o[1]};
          if ((l & 3) == 0) static_cast<u8 *>(a.scales)[e / 32] = (u8)(sx + 127);
        }
      } else if (in) {
        store8(a.out, OUT == QMM_BF16, e, v[j]);
      }
    }
  }
}

// Any k and alignment (f32, bf16 and f16 outputs): a workgroup a row, thread t the values t, t + 256, ... . x and residual
// are read again for the output (they come from L2); every value is read before the thread that owns it overwrites it, so
// h and out may be x or residual here too.
template <int OUT>
__global__ __launch_bounds__(256) void rms_norm_any_kernel(NArgs a) {
  __shared__ float part[2][4];
  const int64_t row = item_index(), r0 = row * a.k;
  if (row >= a.rows) return;
  auto at = [](const void *p, int bf, int64_t i) {
    return bf ? bf16_to_f32(static_cast<const u16 *>(p)[i]) : static_cast<const float *>(p)[i];
  };
  auto put = [](void *p, int bf, int64_t i, float v) {
    if (bf) static_cast<u16 *>(p)[i] = __builtin_bit_cast(u16, (__bf16)v);
    else static_cast<float *>(p)[i] = v;
  };
  auto sum_at = [&](int64_t c) { return at(a.x, a.x_bf16, r0 + c) + (a.res ? at(a.res, a.res_bf16, r0 + c) : 0.f); };
  float sum = 0.f;
  for (int64_t c = threadIdx.x; c < a.k; c += 256) {
    const float h = sum_at(c);
    sum = __builtin_fmaf(h, h, sum);
  }
  const float rate = norm_rate(row_reduce<256, false>(sum, part[0]), a.k, a.eps);
  auto value = [&](int64_t c, float h) { return h * rate * at(a.weight, a.w_bf16, c); };
  int e = 0;
  if constexpr (OUT == QMM_F16) {
    float m = 0.f;
    for (int64_t c = threadIdx.x; c < a.k; c += 256) m = fmaxf(m, fabsf(value(c, sum_at(c))));
    e = f16_exponent(row_reduce<256, true>(m, part[1]));
    if (threadIdx.x == 0) {
      static_cast<float *>(a.scales)[2 * row] = pow2(-e);
      static_cast<float *>(a.scales)[2 * row + 1] = pow2(e);
    }
  }
  for (int64_t c = threadIdx.x; c < a.k; c += 256) {
    const float h = sum_at(c), y = value(c, h);
    if (a.h) put(a.h, a.res_bf16, r0 + c, h);
    if constexpr (OUT == QMM_F16) static_cast<_Float16 *>(a.out)[r0 + c] = (_Float16)(y * pow2(-e));
    else put(a.out, OUT == QMM_BF16, r0 + c, y);
  }
}

template <int OUT, int L, int J>
int launch(const NArgs &a, hipStream_t s) {
  constexpr int kRows = L < 256 ? 256 / L : 1;
  rms_norm_kernel<OUT, L, J><<<item_grid((a.rows + kRows - 1) / kRows), L < 256 ? 256 : L, 0, s>>>(a);
  return launch_status();
}

template <int OUT>
int dispatch(const NArgs &a, bool vec, hipStream_t s) {
  if (!vec) {
    if constexpr (OUT == QMM_F32 || OUT == QMM_BF16 || OUT == QMM_F16) {
      rms_norm_any_kernel<OUT><<<item_grid(a.rows), 256, 0, s>>>(a);
      return launch_status();
    } else {
      return QMM_ERR_ALIGN;
    }
  }
  const int64_t chunks = a.k / 8;
  if (chunks <= 16) return launch<OUT, 16, 1>(a, s);
  if (chunks <= 32) return launch<OUT, 32, 1>(a, s);
  if (chunks <= 64) return launch<OUT, 64, 1>(a, s);
  if (chunks <= 256) return launch<OUT, 256, 1>(a, s);
  if (chunks <= 512) return launch<OUT, 256, 2>(a, s);
  if (chunks <= 1024) return launch<OUT, 512, 2>(a, s);
  if (chunks <= 2048) return launch<OUT, 1024, 2>(a, s);
  return launch<OUT, 1024, 4>(a, s);
}

// ---- backward
struct BArgs {
  int64_t rows, k;
  const void *h, *weight, *dy, *dh;
  void *dx;
  float *part;                 // [workgroups, k] partial dweight rows, or NULL
  float *rate;                 // rms_norm_grad_long_kernel with part: [rows]
  float eps;
  int h_bf16, w_bf16, dy_bf16, dh_bf16, dx_bf16;
};

// two sums over the row's L lanes
template <int L>
__device__ __forceinline__ void row_reduce2(float &u, float &v, float2 *part) {
  constexpr int W = L < 64 ? L : 64;
#pragma unroll
  for (int off = W / 2; off >= 1; off >>= 1) {
    u += __shfl_xor(u, off, kWave);
    v += __shfl_xor(v, off, kWave);
  }
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_float2(u, v);
    __syncthreads();
    u = part[0].x;
    v = part[0].y;
#pragma unroll
    for (int i = 1; i < L / 64; ++i) {
      u += part[i].x;
      v += part[i].y;
    }
  }
}

// lanes and chunks as rms_norm_kernel; row group g = blockIdx.x, + gridDim.x, ... (without DW one group a workgroup, up to
// the most workgroups of a grid)
template <int L, int J, bool DW>
__global__ __launch_bounds__(L < 256 ? 256 : L) void rms_norm_grad_kernel(BArgs a) {
  constexpr int kRows = L < 256 ? 256 / L : 1;
  __shared__ float2 part[2][L > 64 ? L / 64 : 1];   // in turn: a wave may still read the last row's
  const int l = threadIdx.x % L, chunks = (int)(a.k / 8);
  float w[J][8], acc[DW ? J : 1][8];
#pragma unroll
  for (int j = 0; j < J; ++j) load8_act(a.weight, a.w_bf16, 8 * min(l + L * j, chunks - 1), w[j]);
  if constexpr (DW) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[j][i] = 0.f;
  }
  const int64_t groups = (a.rows + kRows - 1) / kRows;
  int turn = 0;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x, turn ^= 1) {
    const int64_t row_ = g * kRows + threadIdx.x / L;
    const bool alive = row_ < a.rows;
    const int64_t r0 = (alive ? row_ : a.rows - 1) * a.k;
    float h[J][8], d[J][8], e[J][8];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t at = r0 + 8 * min(l + L * j, chunks - 1);
      load8_act(a.h, a.h_bf16, at, h[j]);
      load8_act(a.dy, a.dy_bf16, at, d[j]);
      if (a.dh) load8_act(a.dh, a.dh_bf16, at, e[j]);
    }
    float hh = 0.f, gh = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float u = 0.f, v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        u = __builtin_fmaf(h[j][i], h[j][i], u);
        v = __builtin_fmaf(d[j][i] * w[j][i], h[j][i], v);
      }
      hh += l + L * j < chunks ? u : 0.f;
      gh += l + L * j < chunks ? v : 0.f;
    }
    row_reduce2<L>(hh, gh, part[turn]);
    const float rate = norm_rate(hh, a.k, a.eps), mean = rate * (gh / (float)a.k);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hn = h[j][i] * rate;
        o[i] = rate * __builtin_fmaf(-hn, mean, d[j][i] * w[j][i]);
        if (a.dh) o[i] += e[j][i];
        if constexpr (DW) acc[j][i] = alive ? __builtin_fmaf(d[j][i], hn, acc[j][i]) : acc[j][i];
      }
      if (alive && l + L * j < chunks) store8(a.dx, a.dx_bf16, r0 + 8 * (l + L * j), o);
    }
  }
  if constexpr (DW) {
    if constexpr (kRows == 1) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (l + L * j < chunks) store8(a.part, 0, (int64_t)blockIdx.x * a.k + 8 * (l + L * j), acc[j]);
    } else {   // the workgroup's rows side by side, added in order
      static_assert(J == 1, "short rows are one chunk a lane");
      __shared__ float sums[kRows][8 * L];
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[threadIdx.x / L][8 * l + i] = acc[0][i];
      __syncthreads();
      for (int c = threadIdx.x; c < a.k; c += 256) {
        float v = sums[0][c];
#pragma unroll
        for (int q = 1; q < kRows; ++q) v += sums[q][c];
        a.part[(int64_t)blockIdx.x * a.k + c] = v;
      }
    }
  }
}

// Rows of more than 8192 values (V = 8; in registers they spill), any k and alignment (V = 1): a workgroup a row, which is read
// twice, the second time from L2
template <int V>
__global__ __launch_bounds__(512) void rms_norm_grad_long_kernel(BArgs a) {
  __shared__ float2 part[8];
  const int64_t row = item_index(), r0 = row * a.k;
  if (row >= a.rows) return;
  auto load = [](const void *p, int bf, int64_t at, float (&v)[V]) __attribute__((always_inline)) {
    if constexpr (V == 8) load8_act(p, bf, at, v);
    else v[0] = load_val(p, bf, at);
  };
  float hh = 0.f, gh = 0.f;
  for (int64_t c = V * threadIdx.x; c < a.k; c += V * 512) {
    float h[V], d[V], w[V];
    load(a.h, a.h_bf16, r0 + c, h);
    load(a.dy, a.dy_bf16, r0 + c, d);
    load(a.weight, a.w_bf16, c, w);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      hh = __builtin_fmaf(h[i], h[i], hh);
      gh = __builtin_fmaf(d[i] * w[i], h[i], gh);
    }
  }
  row_reduce2<512>(hh, gh, part);
  const float rate = norm_rate(hh, a.k, a.eps), mean = rate * (gh / (float)a.k);
  if (a.part && threadIdx.x == 0) a.rate[row] = rate;
  for (int64_t c = V * threadIdx.x; c < a.k; c += V * 512) {
    float h[V], d[V], w[V], e[V];
    load(a.h, a.h_bf16, r0 + c, h);
    load(a.dy, a.dy_bf16, r0 + c, d);
    load(a.weight, a.w_bf16, c, w);
    if (a.dh) load(a.dh, a.dh_bf16, r0 + c, e);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      d[i] = rate * __builtin_fmaf(-(h[i] * rate), mean, d[i] * w[i]);
      if (a.dh) d[i] += e[i];
    }
    if constexpr (V == 8) store8(a.dx, a.dx_bf16, r0 + c, d);
    else store_val(a.dx, a.dx_bf16, r0 + c, d[0]);
  }
}
// and its partial dweight rows: 256 columns a workgroup, rows blockIdx.y, + gridDim.y, ...
__global__ __launch_bounds__(256) void rms_norm_dweight_part_kernel(BArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.k) return;
  float v = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
    v = __builtin_fmaf(load_val(a.dy, a.dy_bf16, row * a.k + c), load_val(a.h, a.h_bf16, row * a.k + c) * a.rate[row], v);
  a.part[(int64_t)blockIdx.y * a.k + c] = v;
}

// dweight from n partial rows: 32 columns a workgroup, thread row q adds rows q, q + 32, ...; the 32 sums in order
__global__ __launch_bounds__(1024) void rms_norm_dweight_kernel(const float *__restrict__ part, int n, int64_t k, float *__restrict__ dw) {
  __shared__ float sums[32][33];
  const int x = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + x;
  float v = 0.f;
  if (c < k)
#pragma unroll 8
    for (int i = q; i < n; i += 32) v += part[(int64_t)i * k + c];
  sums[q][x] = v;
  __syncthreads();
  if (q == 0 && c < k) {
#pragma unroll
    for (int i = 1; i < 32; ++i) v += sums[i][x];
    dw[c] = v;
  }
}

// Partial rows of dweight: enough workgroups to keep their loads in flight, few enough that the partial rows are a small part
// of the traffic (1024 / 512, us in a graph on one set of inputs: 16384 x 2048 bf16 55 / 71, 65536 x 128 17 / 19; two chunks a
// lane 4096 x 4096 36 / 35, 2048 x 8192 44 / 38; long rows 1024 x 12288 64 / 55, 47 with 128)
constexpr int64_t kParts = 1024, kParts2 = 512, kPartsLong = 128;

template <int L, int J>
int launch_grad(const BArgs &a, float *dw, hipStream_t s) {
  constexpr int kRows = L < 256 ? 256 / L : 1, kThreads = L < 256 ? 256 : L;
  const int64_t groups = (a.rows + kRows - 1) / kRows;
  if (!dw) {
    rms_norm_grad_kernel<L, J, false><<<item_grid(groups).x, kThreads, 0, s>>>(a);
    return launch_status();
  }
  constexpr int64_t kMost = J == 1 ? kParts : kParts2;
  const unsigned n = (unsigned)(groups < kMost ? groups : kMost);
  rms_norm_grad_kernel<L, J, true><<<n, kThreads, 0, s>>>(a);
  if (int st = launch_status()) return st;
  rms_norm_dweight_kernel<<<(unsigned)((a.k + 31) / 32), 1024, 0, s>>>(a.part, (int)n, a.k, dw);
  return launch_status();
}

}  // namespace

extern "C" int qmm_rms_norm(int64_t rows, int64_t k, const void *x, int x_dtype, const void *residual, int res_dtype,
                            const void *weight, int w_dtype, float eps, void *h, int out_dtype, void *out,
                            void *out_scales, qmm_stream_t stream) {
  if (!x || !weight || !out || (h && !residual)) return QMM_ERR_NULL;
  const bool q8 = out_dtype == QMM_Q8, mx = out_dtype == QMM_MXFP8, f16 = out_dtype == QMM_F16;
  if ((mx || f16) && !out_scales) return QMM_ERR_NULL;
  auto val = [](int d) { return d == QMM_F32 || d == QMM_BF16; };
  if (!val(x_dtype) || !val(w_dtype) || (residual && !val(res_dtype))) return QMM_ERR_DTYPE;
  if (!q8 && !mx && !f16 && !val(out_dtype)) return QMM_ERR_DTYPE;
  if (!(eps >= 0.f)) return QMM_ERR_RANGE;
  if (rows <= 0 || rows > (1ll << 24) || k <= 0 || k > kMaxK || ((q8 || mx) && k % 32)) return QMM_ERR_SHAPE;
  auto size = [](int d) { return d == QMM_F32 ? (size_t)4 : (size_t)2; };
  if (!aligned(x, size(x_dtype)) || !aligned(weight, size(w_dtype)) || (residual && !aligned(residual, size(res_dtype))) ||
      (h && !aligned(h, size(res_dtype))) || (q8 || mx ? !aligned(out, 16) : !aligned(out, size(out_dtype))) ||
      (f16 && !aligned(out_scales, 8)))
    return QMM_ERR_ALIGN;
  const bool vec = k % 8 == 0 && aligned(x, 16) && aligned(weight, 16) && aligned(residual, 16) && aligned(h, 16) && aligned(out, 16);
  const NArgs a{rows, k, x, residual, weight, h, out, out_scales, eps, x_dtype == QMM_BF16, res_dtype == QMM_BF16, w_dtype == QMM_BF16};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (out_dtype) {
    case QMM_F32: return dispatch<QMM_F32>(a, vec, s);
    case QMM_BF16: return dispatch<QMM_BF16>(a, vec, s);
    case QMM_F16: return dispatch<QMM_F16>(a, vec, s);
    case QMM_Q8: return dispatch<QMM_Q8>(a, vec, s);
    default: return dispatch<QMM_MXFP8>(a, vec, s);
  }
}

extern "C" int64_t qmm_rms_norm_grad_workspace_size(int64_t rows, int64_t k) {
  if (rows <= 0 || rows > (1ll << 24) || k <= 0 || k > kMaxK) return -1;
  return 4 * ((rows < kParts ? rows : kParts) * k + rows);
}

extern "C" int qmm_rms_norm_grad(int64_t rows, int64_t k, const void *h, int h_dtype, const void *weight, int w_dtype,
                                 float eps, const void *dy, int dy_dtype, const void *dh, int dh_dtype, void *dx,
                                 int dx_dtype, float *dweight, void *workspace, int64_t workspace_bytes,
                                 qmm_stream_t stream) {
  if (!h || !weight || !dy || !dx) return QMM_ERR_NULL;
  auto val = [](int d) { return d == QMM_F32 || d == QMM_BF16; };
  if (!val(h_dtype) || !val(w_dtype) || !val(dy_dtype) || !val(dx_dtype) || (dh && !val(dh_dtype))) return QMM_ERR_DTYPE;
  if (!(eps >= 0.f)) return QMM_ERR_RANGE;
  const int64_t need = qmm_rms_norm_grad_workspace_size(rows, k);
  if (need < 0) return QMM_ERR_SHAPE;
  auto size = [](int d) { return d == QMM_F32 ? (size_t)4 : (size_t)2; };
  if (!aligned(h, size(h_dtype)) || !aligned(weight, size(w_dtype)) || !aligned(dy, size(dy_dtype)) ||
      !aligned(dx, size(dx_dtype)) || (dh && !aligned(dh, size(dh_dtype))) || !aligned(dweight, 4))
    return QMM_ERR_ALIGN;
  if (dweight) {
    if (!workspace || workspace_bytes < need) return QMM_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return QMM_ERR_ALIGN;
  }
  BArgs a{rows, k, h, weight, dy, dh, dx, dweight ? static_cast<float *>(workspace) : nullptr, nullptr, eps,
          h_dtype == QMM_BF16, w_dtype == QMM_BF16, dy_dtype == QMM_BF16, dh_dtype == QMM_BF16, dx_dtype == QMM_BF16};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t chunks = k / 8;
  const bool vec = k % 8 == 0 && aligned(h, 16) && aligned(weight, 16) && aligned(dy, 16) && aligned(dh, 16) && aligned(dx, 16);
  if (vec && chunks <= 16) return launch_grad<16, 1>(a, dweight, s);
  if (vec && chunks <= 32) return launch_grad<32, 1>(a, dweight, s);
  if (vec && chunks <= 64) return launch_grad<64, 1>(a, dweight, s);
  if (vec && chunks <= 256) return launch_grad<256, 1>(a, dweight, s);
  if (vec && chunks <= 512) return launch_grad<256, 2>(a, dweight, s);
  if (vec && chunks <= 1024) return launch_grad<512, 2>(a, dweight, s);
  const unsigned n = (unsigned)(rows < kPartsLong ? rows : kPartsLong);
  if (dweight) a.rate = a.part + (int64_t)n * k;
  if (vec) rms_norm_grad_long_kernel<8><<<item_grid(rows), 512, 0, s>>>(a);
  else rms_norm_grad_long_kernel<1><<<item_grid(rows), 512, 0, s>>>(a);
  if (int st = launch_status()) return st;
  if (!dweight) return QMM_OK;
  rms_norm_dweight_part_kernel<<<dim3((unsigned)((k + 255) / 256), n), 256, 0, s>>>(a);
  if (int st = launch_status()) return st;
  rms_norm_dweight_kernel<<<(unsigned)((k + 31) / 32), 1024, 0, s>>>(a.part, (int)n, k, dweight);
  return launch_status();
}

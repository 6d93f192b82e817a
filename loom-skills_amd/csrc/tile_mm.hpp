// C = A B over 16-bit operands on v_mfma_f32_32x32x16, one matrix or one an expert over ragged segments of rows:
//
//   forward          Y[t, r]   = sum_c X[t, c] W_e[r, c]        t in expert e's segment
//   input gradient   dX[t, c]  = sum_r dY[t, r] W_e[r, c]
//   weight gradient  dW_e[r,c] = sum_t dY[t, r] X[t, c]         t over expert e's segment
//
// with W_e as 16-bit rows or as 4-bit codes with group scales, dequantized to f16 on their way into LDS: f16(s (q - z)), the
// one rounding (q - z is exact).
//
// A workgroup owns BM x BN outputs, WM x WN waves of (BM / WM) x (BN / WN), and walks the sum 64 values at a time through ST
// LDS buffers. An operand whose memory rows run along the sum (kRow) keeps them: LDS rows of 64 values, 16-byte chunk i at
// i ^ (row / 2 % 8), so that the 16 rows a fragment read covers at a time lie in all banks. One whose memory rows run along the
// outputs (kCol) keeps those too, 64 LDS rows of BM or BN values, and is transposed by ds_read_b64_tr_b16 (16 lanes read a
// 4 x 16 block and get its columns): chunk i of LDS row k at i ^ (4 (k % 4)) ^ (k / 4 % 4), for the reads (four rows x 64 bytes at
// a time) and the stores of dequantized weights (16 rows of one chunk). 16-bit operands go straight into LDS
// (buffer_load ... lds), rows past a segment's end and values past a row's end as zeros. The fragments of the next 16 values
// are read while the MFMAs of these run, and the barrier of a step stands before its last 16 values' MFMAs, so that the next
// step's first reads run under them.
//
// The MFMAs bound a full round of 256 x 256 tiles (a step of 64 values 1.56 us on every CU, by 4096 x 4096 outputs of 4096 and 8192
// values: 1.38 PFLOP/s, at the clock the power limit holds; a library product of 8192^3 reaches 1.55), a launch the rounds it takes and
// each tile's start and end (the operands' first loads, 128 KB of outputs; 8 us a further round of 4096 x 4096 outputs). Kernels alone,
// least and mean of 21 calls: 16384 rows of 32 experts 2880 x 2880 forward 315 and 340 us, 0.86 PFLOP/s, in four rounds, the last a
// little over half full; their weights' gradient 378 and 397 with eight steps a tile. Many experts of few rows are bound by memory: 8000
// rows of 128 experts 768 x 2048, dW writes 0.8 GB in 144 us (164 and 175 among calls of dx, which it evicts from the last-level cache).
#pragma once
#include <algorithm>
#include <type_traits>

#include "ragged.hpp"

namespace qmm {
namespace tmm {

typedef __attribute__((ext_vector_type(4))) u32 u32x4;
typedef __attribute__((ext_vector_type(2))) u32 u32x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(2))) _Float16 h2;

enum Src { kRow = 0, kCol = 1, kW4Col = 2 };
enum Sum { kSumFixed = 0, kSumRagged = 1 };   // what the segments cut: A's rows (kSumFixed) or the sum (the weight gradient)
constexpr u32 kPast = 0x80000000u;            // an offset past every resource: the load gives zeros
constexpr int kGroupM = 8;

struct Args {
  const int32_t *offsets;      // NULL: one segment of all rows
  int E, rows;
  int M, N, K;                 // outputs M x N (kSumFixed: M unused), sum of K values (kSumRagged: K unused)
  const u8 *a, *b;
  int64_t a_row, b_row;        // bytes from one memory row to the next (w4: unused)
  int64_t b_expert;            // bytes from one expert's matrix to the next
  const u32 *ws;               // w4: (f16 scale, f16 1024 + zero) words [E][ceil(rows of W / 16)][groups][16]
  int w_blocks, w_tiles;       // w4: 16-row blocks and 128-value tiles of an expert's matrix
  int groups, gshift;          // w4: group of 32-value step i: min(i >> gshift, groups - 1)
  const float *scales;         // [rows, 2] or NULL: output row t times scales[t, 1]
  void *y;
  int y_type;                  // QMM_F32, QMM_BF16 or QMM_F16
  int stream;                  // weight gradient: whole 128-byte lines a row, past what the caches hold
  int tiles_n;
  int splits;                  // parts of the sum, one a layer of the grid (y); more than one: f32 sums [splits][outputs] into part
  float *part;
  int rest;                    // kSumFixed: the layer's first workgroups, a multiple of eight, which set the rows of no expert to zero (ragged.hpp); 0: none
};

template <int DT>
__device__ __forceinline__ f32x16 mfma(u32x4 x, u32x4 w, f32x16 c) {
  if constexpr (DT == QMM_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
}

// 16 bytes a lane from a buffer resource into LDS at lds + 16 lane (wave-uniform lds); lanes past the resource's end write
// zeros. Written out so that the compiler's wait counting stays with the register loads; the caller waits before the barrier.
__device__ __forceinline__ void lds_load16(u32x4 rsrc, u32 voff, u32 lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(rsrc), "s"(lds)
               : "m0", "memory");
}
// every load has landed, every LDS access of this wave is done, and the same holds for the workgroup's other waves
__device__ __forceinline__ void wait_all_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// the same but for the wave's last N loads
template <int N>
__device__ __forceinline__ void wait_but_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// bytes past 0 (every extent here is below 2^31: at most 256 rows of 2^21 bytes)
__device__ __forceinline__ u32x4 resource(const u8 *p, int bytes) {
  const uint64_t at = (uint64_t)p;
  return u32x4{(u32)__builtin_amdgcn_readfirstlane((int)(u32)at), (u32)__builtin_amdgcn_readfirstlane((int)((u32)(at >> 32) & 0xFFFFu)),
               (u32)__builtin_amdgcn_readfirstlane(max(bytes, 0)), 0x00020000u};
}

__device__ __forceinline__ h2 as_h2(u32 v) { return __builtin_bit_cast(h2, v); }
// eight weights f16(s (q - z)) from a code word (low nibbles values 0 .. 3, high nibbles 4 .. 7) and a scale word
__device__ __forceinline__ u32x4 dequant(u32 q, u32 sc) {
  const u32 lo = q & 0x0F0F0F0Fu, hi = (q >> 4) & 0x0F0F0F0Fu;
  const h2 v = as_h2(sc), s = {v.x, v.x}, z = {v.y, v.y};
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // 0x6400 | q is 1024 + q; the difference is exact
    const h2 c = as_h2(__builtin_amdgcn_perm(0x64646464u, i < 2 ? lo : hi, i & 1 ? 0x04030402u : 0x04010400u));
    o[i] = __builtin_bit_cast(u32, (c - z) * s);
  }
  return o;
}

// 32 output rows mb .. of a wave (those below m_end), columns nb .. nb + 32 NJ - 1 (those below N), through its own LDS: the sums
// of a lane are one column of 16 rows, a store covers neighbouring columns. scales: of the segment's rows, or NULL.
template <int NJ>
constexpr int stage_pitch() { return NJ * 32 + 8; }   // floats; 4 rows apart is 32 banks apart
template <int NJ, bool STREAM = false>
__device__ __forceinline__ void store_rows(const Args &a, float *stage, const f32x16 (&acc)[NJ], int64_t out0, int mb, int m_end, int nb,
                                           const float *scales, int lane) {
  constexpr int kPitch = stage_pitch<NJ>();
  const int c = lane & 31, h = lane >> 5;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) stage[((r & 3) + 8 * (r >> 2) + 4 * h) * kPitch + 32 * j + c] = acc[j][r];
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  auto store = [&](auto *y) __attribute__((always_inline)) {
    using T = std::remove_reference_t<decltype(*y)>;
    constexpr int V = 16 / sizeof(T), L = 32 * NJ / V;   // values a lane, lanes a row: a store covers neighbouring lines
    typedef __attribute__((ext_vector_type(V))) T TV;
    const int col = (lane % L) * V, n = nb + col;
    auto pass = [&](int r0, auto whole) __attribute__((always_inline)) {
      const int r = r0 + lane / L, m = mb + r;
      if (m < m_end && n < a.N) {
        const float *const from = stage + r * kPitch + col;
        const float sc = scales ? scales[2 * (int64_t)m + 1] : 1.f;
        T *const to = y + out0 + (int64_t)m * a.N + n;
        if (decltype(whole)::value || n + V <= a.N) {
          TV o;
#pragma unroll
          for (int x = 0; x < V; ++x) o[x] = (T)(from[x] * sc);
          if constexpr (STREAM) __builtin_nontemporal_store(o, reinterpret_cast<TV *>(to));
          else __builtin_memcpy(to, &o, 16);   // at any address: the GPU's memory takes them
        } else {
#pragma unroll 1
          for (int x = 0; n + x < a.N; ++x) to[x] = (T)(from[x] * sc);
        }
      }
    };
    if (nb + 32 * NJ <= a.N) {
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 64 / L) pass(r0, std::true_type{});
    } else {
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += 64 / L) pass(r0, std::false_type{});
    }
  };
  if (a.y_type == QMM_F32) store(static_cast<float *>(a.y));
  else if (a.y_type == QMM_BF16) store(static_cast<__bf16 *>(a.y));
  else store(static_cast<_Float16 *>(a.y));
}

template <int SRC>
__device__ __forceinline__ int chunk_swizzle(int row) {
  if constexpr (SRC == kRow) return (row >> 1) & 7;
  else return ((row & 3) << 2) ^ ((row >> 2) & 3);
}

// The workgroup among those of a layer of the sum (the grid's y). HIP refuses 2^32 threads along a grid's dimension: what passes 2^21
// workgroups lies along z.
constexpr int kGridX = 1 << 21;
__device__ __forceinline__ int workgroup() { return (int)(blockIdx.z * kGridX + blockIdx.x); }
inline dim3 tile_grid(int64_t tiles, int rest, int layers) {
  const int64_t n = (tiles + 7) / 8 * 8 + rest, x = std::min<int64_t>(n, kGridX);
  return dim3((unsigned)x, (unsigned)layers, (unsigned)((n + x - 1) / x));
}
constexpr int64_t kMaxTiles = 1 << 30;   // more have outputs that no card holds

// The workgroup's output tile where the segments cut A's rows: expert, segment, first row in it, column tile; false for a workgroup
// too many. Workgroup i runs on XCD i % 8, which takes a contiguous range of tiles: an expert's in groups of kGroupM row tiles,
// rows fastest, so that the tiles that an XCD works on at a time share operands in its L2.
template <int BM>
__device__ __forceinline__ bool row_tile(const Args &a, int &e, int &lo, int &hi, int &m0, int &nt) {
  TileScan sc{(a.rows + BM - 1) / BM, 0, 1};
  if (a.offsets) sc = scan_tiles<BM>(a.offsets, a.E, a.rows);
  const int total = sc.total * a.tiles_n, per = (total + 7) >> 3;
  const int wg = workgroup() - a.rest, i = wg >> 3;
  int t = (wg & 7) * per + i, first = 0;
  if (i >= per || t >= total) return false;
  if (a.offsets) find_tile<BM>(a.offsets, a.E, a.rows, sc, t / a.tiles_n, e, lo, hi, first);
  t -= first * a.tiles_n;
  const int own = a.offsets ? (max(hi - lo, 1) + BM - 1) / BM : sc.total;   // the expert's row tiles
  const int g = t / (kGroupM * a.tiles_n), gm = max(1, min(kGroupM, own - g * kGroupM)), gt = t - g * kGroupM * a.tiles_n;
  m0 = (g * kGroupM + gt % gm) * BM;
  nt = gt / gm;
  return true;
}
// whether the workgroup is one of those for the rows of no expert, which are done then
__device__ __forceinline__ bool rest_done(const Args &a) {
  const int part = workgroup();
  if (part >= a.rest) return false;
  if (blockIdx.y == 0)
    zero_rest(a.offsets, a.E, a.rows, static_cast<u8 *>(a.y), (int64_t)a.N * (a.y_type == QMM_F32 ? 4 : 2), part, a.rest);
  return true;
}
// first step of part i of n
__device__ __forceinline__ int part_of(int steps, int n, int i) { return (int)((int64_t)steps * i / n); }
// the outputs of a sum in parts: the layer's f32 sums
__device__ __forceinline__ void to_part(Args &a, int64_t outputs) {
  if (a.splits == 1) return;
  a.y = a.part + blockIdx.y * outputs;
  a.y_type = QMM_F32;
  a.scales = nullptr;
}

// The P parts added in order, the rows scaled and rounded: a workgroup a tile of 16 rows x 64 columns (by the segments, so that rows
// of no expert stay as they are) or, without offsets, of all rows; a thread four columns of a row, its loads all in
// flight.
constexpr int kJoinRows = 16, kJoinCols = 64;
template <int P>
static __global__ __launch_bounds__(256) void join_kernel(Args a, int64_t outputs) {
  int e = 0, lo = 0, hi = a.rows, m0, nt;
  if (!row_tile<kJoinRows>(a, e, lo, hi, m0, nt)) return;
  const int m = m0 + (int)(threadIdx.x >> 4), n = nt * kJoinCols + 4 * (int)(threadIdx.x & 15);
  const int own = min(4, a.N - n);   // columns of the thread
  if (m >= hi - lo || own <= 0) return;
  const int64_t at = (int64_t)(lo + m) * a.N + n;
  f32x4 part[P], v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const float *src = a.part + p * outputs + at;
    if (own == 4) {
      __builtin_memcpy(&part[p], src, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[p][i] = src[min(i, own - 1)];
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) v += part[p];
  v *= a.scales ? a.scales[2 * (int64_t)(lo + m) + 1] : 1.f;
  auto store = [&](auto *y) __attribute__((always_inline)) {
    using T = std::remove_reference_t<decltype(*y)>;
    const T o[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    if (own == 4) {
      __builtin_memcpy(y + at, o, sizeof(o));
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < own) y[at + i] = o[i];
    }
  };
  if (a.y_type == QMM_F32) store(static_cast<float *>(a.y));
  else if (a.y_type == QMM_BF16) store(static_cast<__bf16 *>(a.y));
  else store(static_cast<_Float16 *>(a.y));
}
// row tiles that offsets may give at most
inline int64_t most_row_tiles(const Args &a, int bm) {
  return a.offsets ? std::min<int64_t>((int64_t)a.rows / bm + a.E, a.rows) : (a.rows + bm - 1) / bm;
}

// DT: QMM_BF16 or QMM_F16; SA, SB: the operands' sources; GS: 32-value steps a w4 scale covers (1, 2; 4: more); ST: steps in LDS,
// whose loads go out ST - 1 steps ahead
template <int DT, int SA, int SB, int SUM, int BM, int BN, int WM, int WN, int GS, int ST>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_mm_kernel(Args a) {
  constexpr int NW = WM * WN, NT = 64 * NW, NI = BM / WM / 32, NJ = BN / WN / 32;
  constexpr int kA = BM * 128, kB = BN * 128;             // LDS bytes of a step's operands
  constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;       // 1 KB loads a wave and step
  constexpr bool kW4 = SB == kW4Col;
  static_assert(SA == kRow || BM >= 128, "a transposed operand is at least 128 wide");
  static_assert(SB == kRow || BN >= 128, "a transposed operand is at least 128 wide");
  static_assert(ST == 2 || (ST == 4 && !kW4), "a power of two; the wait's count is of direct loads alone");
  extern __shared__ __align__(1024) u8 smem[];            // A [ST], B [ST]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  int e = 0, lo = 0, hi = a.rows, m0, nt;
  if constexpr (SUM == kSumFixed) {
    if (rest_done(a)) return;
    if (!row_tile<BM>(a, e, lo, hi, m0, nt)) return;
  } else {
    // every XCD takes an eighth of every expert's tiles, one expert after the other: experts differ in their rows
    const int tiles_m = (a.M + BM - 1) / BM, per_e = tiles_m * a.tiles_n, per = (per_e + 7) >> 3;
    const int i = workgroup() >> 3;
    e = i / per;
    const int r = (workgroup() & 7) * per + i - e * per;
    if (e >= a.E || r >= per_e) return;
    m0 = (r % tiles_m) * BM;
    nt = r / tiles_m;
    lo = clamp_row(__builtin_amdgcn_readfirstlane(a.offsets[e]), a.rows);
    hi = clamp_row(__builtin_amdgcn_readfirstlane(a.offsets[e + 1]), a.rows);
  }
  const int n0 = nt * BN;
  // the wave's blocks of 32 rows rb0 .. rb0 + rows_of - 1 and columns cb0 .. cb0 + NJ - 1. Where a tile has outputs in half or a
  // quarter of its columns only, twice or four times as many waves share those, with fewer rows each.
  const int fold = NI >= 4 && WN >= 4 && n0 + BN / 4 >= a.N ? 4 : NI >= 2 && WN >= 2 && n0 + BN / 2 >= a.N ? 2 : 1;
  const int across = WN / fold, rows_of = NI / fold;
  const int rb0 = wave / across * rows_of, cb0 = wave % across * NJ;
  const int seg = max(hi - lo, 0);                        // the segment's rows
  const int m_end = SUM == kSumFixed ? seg : a.M;         // outputs m0 .. min(m0 + BM, m_end) - 1
  const int K = SUM == kSumFixed ? a.K : seg, S = (K + 63) >> 6;
  const int S0 = part_of(S, a.splits, blockIdx.y), S1 = part_of(S, a.splits, blockIdx.y + 1);   // this layer's steps

  // ---- straight into LDS: load i of a wave is 1 KB of the step, lane l's 16 bytes a chunk of row (i NW + wave) ROWS + l / CH
  u32 aoff[LA], boff[LB];
  int acol[SA == kRow ? LA : 1], bcol[SB == kRow ? LB : 1];   // kRow: first value of the lane's chunk
  auto place = [&](auto src, int R, int first, int end, int64_t stride, int i, u32 &off, int &col) __attribute__((always_inline)) {
    constexpr int SRC = decltype(src)::value;
    const int CH = SRC == kRow ? 8 : R / 8;
    const int row = (i * NW + wave) * (64 / CH) + lane / CH, ch = (lane & (CH - 1)) ^ chunk_swizzle<SRC>(row);
    if constexpr (SRC == kRow) {
      off = (u32)((int64_t)row * stride + 16 * ch);
      col = 8 * ch;
    } else {
      off = first + 8 * ch < end ? (u32)((int64_t)row * stride + 16 * ch) : kPast;
      col = 0;
    }
  };
#pragma unroll
  for (int i = 0; i < LA; ++i)
    place(std::integral_constant<int, SA>{}, BM, m0, a.M, a.a_row, i, aoff[i], acol[SA == kRow ? i : 0]);
  if constexpr (!kW4) {
#pragma unroll
    for (int i = 0; i < LB; ++i)
      place(std::integral_constant<int, SB>{}, BN, n0, a.N, a.b_row, i, boff[i], bcol[SB == kRow ? i : 0]);
  }
  // where the tile's operands start, and the bytes from there to the end of what it may read
  const u8 *ap, *bp = a.b;
  if constexpr (SUM == kSumFixed) {
    ap = a.a + (int64_t)(lo + m0) * a.a_row;
    if constexpr (!kW4) bp += (int64_t)e * a.b_expert + (SB == kRow ? (int64_t)n0 * a.b_row : (int64_t)n0 * 2);
    else bp += (int64_t)e * a.b_expert;
  } else {
    ap = a.a + (int64_t)lo * a.a_row + (int64_t)m0 * 2;
    bp += (int64_t)lo * a.b_row + (int64_t)n0 * 2;
  }
  const u32 lds0 = (u32)(uintptr_t)(__attribute__((address_space(3))) u8 *)smem;
  const int a_row = (int)a.a_row, b_row = (int)a.b_row;
  const int a_bytes = SA == kRow ? min(BM, m_end - m0) * a_row : 0, b_bytes = SB == kRow ? min(BN, a.N - n0) * b_row : 0;
  // past the last step (s >= S) the loads give zeros: kRow by the values' check, kCol by the rows left
  auto load_a = [&](int s, int i) __attribute__((always_inline)) {
    const u32 dst = __builtin_amdgcn_readfirstlane(lds0 + (u32)((s & (ST - 1)) * kA + (i * NW + wave) * 1024));
    if constexpr (SA == kRow)
      lds_load16(resource(ap + (int64_t)s * 128, a_bytes - s * 128), 64 * s + acol[i] < K ? aoff[i] : kPast, dst);
    else
      lds_load16(resource(ap + (int64_t)s * 64 * a_row, min(64, K - 64 * s) * a_row - m0 * 2), aoff[i], dst);
  };
  auto load_b = [&](int s, int i) __attribute__((always_inline)) {
    const u32 dst = __builtin_amdgcn_readfirstlane(lds0 + (u32)(ST * kA + (s & (ST - 1)) * kB + (i * NW + wave) * 1024));
    if constexpr (SB == kRow)
      lds_load16(resource(bp + (int64_t)s * 128, b_bytes - s * 128), 64 * s + bcol[i] < K ? boff[i] : kPast, dst);
    else if constexpr (SB == kCol)
      lds_load16(resource(bp + (int64_t)s * 64 * b_row, min(64, K - 64 * s) * b_row - n0 * 2), boff[i], dst);
  };

  // ---- w4: unit tid of a step's 2 BN is a lane's 16 bytes of a 16-row x 128-value tile. Rows and tiles past the end read the last
  // ones: their outputs are not stored, and in the sum A is zero there.
  static_assert(!kW4 || 2 * BN <= NT, "a unit a thread");
  constexpr int kScales = 4 / GS;
  u32 cw[4], cs[kScales];
  auto load_w4 = [&](int s) __attribute__((always_inline)) {
    const int l = tid & 63, b = tid >> 6;
    const int rb = min(4 * s + (b & 3), a.w_blocks - 1), t = min((n0 >> 7) + (b >> 2), a.w_tiles - 1);
    const u32x4 v = *reinterpret_cast<const u32x4 *>(bp + ((int64_t)rb * a.w_tiles + t) * 1024 + 16 * l);
#pragma unroll
    for (int j = 0; j < 4; ++j) cw[j] = v[j];
    const u32 *sp = a.ws + ((int64_t)e * a.w_blocks + rb) * a.groups * 16 + (l & 15);
#pragma unroll
    for (int g = 0; g < kScales; ++g) cs[g] = sp[min((4 * t + GS * g) >> a.gshift, a.groups - 1) * 16];
  };
  auto store_w4 = [&](int s) __attribute__((always_inline)) {
    const int l = tid & 63, b = tid >> 6;
    if (2 * BN < NT && tid >= 2 * BN) return;
    u8 *out = smem + 2 * kA + (s & 1) * kB;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 16 * (b & 3) + (l & 15), ch = 16 * (b >> 2) + 4 * j + (l >> 4);
      *reinterpret_cast<u32x4 *>(out + row * (BN * 2) + ((ch ^ chunk_swizzle<SB>(row)) * 16)) = dequant(cw[j], cs[j / GS]);
    }
  };

  // ---- fragments: lane (c, h) = (l % 32, l / 32) holds values 8 h .. + 7 of the 16 of row or column c
  const int c = lane & 31, h = lane >> 5, p = lane & 15, q = (lane >> 4) & 1;
  const u32 row_base = (u32)(c * 128 + ((h ^ ((c >> 1) & 7)) * 16));
  auto read_row = [&](u32 at, int blk, int kk) __attribute__((always_inline)) {   // rows 32 blk .. of the operand at `at`
    return *reinterpret_cast<const u32x4 *>(smem + ((at + row_base) ^ (u32)(kk * 32)) + blk * 4096);
  };
  auto read_col = [&](u32 at, int RS, int blk, int kk) __attribute__((always_inline)) {   // columns 32 blk ..
    u32x4 v;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int kr = p >> 2, k = 8 * h + 4 * t + kr;
      const int ch = ((4 * blk) ^ (kr << 2)) + ((2 * q + ((p & 3) >> 1)) ^ (2 * h + t));
      const u8 *src = smem + at + (16 * kk) * RS + k * RS + ch * 16 + (p & 1) * 8;
      const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(src));
      const u32x2 d = __builtin_bit_cast(u32x2, r);
      v[2 * t] = d.x;
      v[2 * t + 1] = d.y;
    }
    return v;
  };
  auto read_a = [&](int s, int i, int kk) __attribute__((always_inline)) {
    const u32 at = (u32)((s & (ST - 1)) * kA);
    if constexpr (SA == kRow) return read_row(at, rb0 + i, kk);
    else return read_col(at, BM * 2, rb0 + i, kk);
  };
  auto read_b = [&](int s, int j, int kk) __attribute__((always_inline)) {
    const u32 at = (u32)(ST * kA + (s & (ST - 1)) * kB);
    if constexpr (SB == kRow) return read_row(at, cb0 + j, kk);
    else return read_col(at, BN * 2, cb0 + j, kk);
  };

  f32x16 acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  constexpr int kGap = 128 / (NI * NJ) + 1;   // w4: vector instructions between two MFMAs
  constexpr int kLoads = LA + (kW4 ? 0 : LB);
  // of a step's loads, those that go out past the barrier; the rest follow a phase later (w4: none, that phase has the weights)
  constexpr int kFirst = kW4 ? kLoads : (kLoads + 1) / 2;
  auto load_one = [&](int s, int l) __attribute__((always_inline)) {
    if (l < LA) load_a(s, l);
    else if constexpr (!kW4) load_b(s, l - LA);
  };
  u32x4 fa[2][NI], fb[2][NJ];
  // the walk along the sum with the wave's first NA 32-row blocks; every wave meets every barrier
  auto walk = [&](auto blocks) __attribute__((always_inline)) {
    constexpr int NA = decltype(blocks)::value;
    auto read = [&](int set, int s, int kk) __attribute__((always_inline)) {
      if constexpr (NA > 0) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[set][j] = read_b(s, j, kk);
#pragma unroll
        for (int i = 0; i < NA; ++i) fa[set][i] = read_a(s, i, kk);
      }
    };
    auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mfma<DT>(fa[set][i], fb[set][j], acc[i][j]);
    };
    auto multiply_loading = [&](int set, int s, int first, int end) __attribute__((always_inline)) {   // loads of step s between
#pragma unroll
      for (int m = 0; m < (NA * NJ > end - first ? NA * NJ : end - first); ++m) {
        if (m < end - first) load_one(s, first + m);
        if (m < NA * NJ) acc[m / NJ][m % NJ] = mfma<DT>(fa[set][m / NJ], fb[set][m % NJ], acc[m / NJ][m % NJ]);
        if (m < end - first) __builtin_amdgcn_sched_barrier(0);
      }
    };
    read(0, S0, 0);
    for (int s = S0; s < S1; ++s) {
#pragma unroll
      for (int kk = 0; kk < 3; ++kk) {
        read((kk + 1) & 1, s, kk + 1);
        __builtin_amdgcn_sched_barrier(0);
        // the next step's weights, whose buffer the last barrier has freed: late in the step, their loads are one step old then
        if constexpr (kW4) {
          if (kk == 2) store_w4(s + 1);
        }
        if (kk == 0) multiply_loading(0, s + ST - 1, kFirst, kLoads);
        else multiply(kk & 1);
        if constexpr (kW4) {
          if (kk > 0) {
#pragma unroll
            for (int m = 0; m < NA * NJ; ++m) {   // an MFMA, then vector instructions of the weights
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x002, kGap, 0);
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (ST == 2) wait_all_barrier();
      else wait_but_barrier<(ST - 2) * kLoads>();   // the next step's loads have landed
      read(0, s + 1, 0);   // past the last step: what the buffer holds, not used
      if constexpr (kW4) load_w4(s + 2);
      __builtin_amdgcn_sched_barrier(0);
      multiply_loading(1, s + ST, 0, kFirst);   // past the last step: zeros
    }
    wait_all_barrier();   // the buffers are the outputs' staging areas next
  };

  // blocks of 32 rows of the wave that hold outputs at all (the last tile of a segment is often nearly empty)
  const int live = n0 + cb0 * 32 < a.N ? min(max((m_end - m0 - rb0 * 32 + 31) >> 5, 0), rows_of) : 0;
  if (S1 > S0) {
#pragma unroll
    for (int t = 0; t < ST - 1; ++t)
#pragma unroll
      for (int l = 0; l < kLoads; ++l) load_one(S0 + t, l);
    if constexpr (kW4) {
      load_w4(S0);
      store_w4(S0);
      load_w4(S0 + 1);
    }
    if constexpr (ST == 2) wait_all_barrier();
    else wait_but_barrier<(ST - 2) * kLoads>();
#pragma unroll
    for (int l = 0; l < kFirst; ++l) load_one(S0 + ST - 1, l);
    if (live == NI) walk(std::integral_constant<int, NI>{});
    else if (live == 0) walk(std::integral_constant<int, 0>{});
    else if (NI > 1 && live == 1) walk(std::integral_constant<int, 1>{});
    else if (NI > 2 && live == 2) walk(std::integral_constant<int, NI < 2 ? NI : 2>{});
    else if (NI > 3) walk(std::integral_constant<int, NI < 3 ? NI : 3>{});
  }

  // ---- outputs (every wave is past its last read of the operands)
  constexpr int kStage = 32 * stage_pitch<NJ>();
  static_assert(kStage * 4 * NW <= ST * (kA + kB), "the staging areas fit the operands' buffers");
  const int64_t out0 = SUM == kSumFixed ? (int64_t)lo * a.N : (int64_t)e * a.M * a.N;
  to_part(a, SUM == kSumFixed ? (int64_t)a.rows * a.N : (int64_t)a.E * a.M * a.N);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if (i >= live) break;
    float *const stage = reinterpret_cast<float *>(smem) + wave * kStage;
    const int mb = m0 + (rb0 + i) * 32, nb = n0 + cb0 * 32;
    if constexpr (SUM == kSumRagged) {
      if (a.stream) store_rows<NJ, true>(a, stage, acc[i], out0, mb, m_end, nb, nullptr, lane);
      else store_rows<NJ>(a, stage, acc[i], out0, mb, m_end, nb, nullptr, lane);
    } else {
      store_rows<NJ>(a, stage, acc[i], out0, mb, m_end, nb, a.scales ? a.scales + 2 * (int64_t)lo : nullptr, lane);
    }
  }
}

// ------------------------------------------------------------------------------------------------------ host
// A tile shape and in how many parts the sum is taken (more where few tiles would walk a long sum): the least estimated time, that
// is the workgroups that a CU gets times (turns along the sum times a turn's time + a start and end), or what one workgroup alone
// takes if that is more, and the parts' way through memory. A shape's figures (us a turn over the workgroups that share a CU on
// launches that fill the chip, their start and end, a turn of one workgroup on a CU) are no measurements of their own: they are those with which the choice comes closest
// to the fastest of all shapes and parts, measured on 800 calls of 1e8 to 2e11 operations: 2 to 3.5 % slower than it on average.
struct Shape {
  int bm, bn;
  float turn, ends, alone;
  int depth = 2;   // steps in LDS
};
struct Plan {
  int shape, splits;
};
// what qmm_tile_plan says of it
inline int64_t plan_word(const Shape &t, const Plan &p) {
  return (int64_t)p.splits << 40 | (int64_t)t.depth << 32 | (int64_t)t.bm << 16 | t.bn;
}
// turns: of a workgroup (the longest); mean: of them all, for what a CU's workgroups take together; tiles_of(shape): workgroups without
// a split; outputs: of the whole call
template <int COUNT, class T>
Plan least_time(const Shape (&shapes)[COUNT], int64_t turns, float mean, int64_t outputs, T tiles_of) {
  Plan best{0, 1};
  float least = 0.f;
  for (int i = 0; i < COUNT; ++i) {
    const int64_t tiles = std::max<int64_t>(tiles_of(shapes[i]), 1);
    for (int p = 1; p <= 16; p *= 2) {
      if (p > 1 && (turns < 4 * p || tiles * p > 1024 || outputs * p > (16 << 20))) break;
      const float t = (float)((turns + p - 1) / p), each = mean < (float)turns ? mean / p : t;
      const float busy = (float)((tiles * p + 255) / 256) * (each * shapes[i].turn + shapes[i].ends), one = t * shapes[i].alone + 5.5f;
      const float us = std::max(busy, one) + (p > 1 ? 4.5f + (float)(outputs * (2 * p + 1)) * 0.8e-6f : 0.f);
      if ((i == 0 && p == 1) || us < least) best = {i, p}, least = us;
    }
  }
  return best;
}
// row tiles to expect: a segment's last tile is half empty on average and segments differ, hardly an expert is without rows
inline int64_t expected_row_tiles(int64_t rows, int E, int bm) {
  if (E == 1) return (rows + bm - 1) / bm;
  const int64_t hit = std::min<int64_t>(E, rows);
  return std::max<int64_t>(rows / bm + hit * 3 / 5, hit);
}
// 16-bit weights: the last two have four steps in LDS instead of two, one workgroup a CU, for launches that leave CUs without a
// second one to hide a step's loads behind (us, 512 rows of 4 experts 2880 x 2880 32 -> 20, 2000 rows 2048 x 2048 30 -> 24; 8000 rows of
// 128 experts 768 x 2048 95 either way, dx 105 -> 122); 16384 rows of 32 experts 2880 x 2880 320, 363, 447 with the first three.
// 4-bit ones: gradients of 2048 x 4096 x 12288 301, 247, 315, 227.
constexpr Shape kTiles[] = {{256, 256, 1.4f, 7.f, 1.4f}, {128, 128, 0.47f, 3.2f, 0.9f}, {64, 128, 0.4f, 1.f, 0.7f},
                            {64, 128, 0.38f, 4.4f, 0.36f, 4}, {128, 128, 0.55f, 5.3f, 0.5f, 4}};
constexpr Shape kTilesW4[] = {{256, 256, 1.93f, 8.3f, 1.5f}, {128, 128, 0.54f, 3.4f, 0.8f}, {64, 128, 0.36f, 1.2f, 0.5f},
                              {256, 128, 1.03f, 5.f, 1.f}};
template <int COUNT>
Plan plan_rows(const Shape (&shapes)[COUNT], int64_t rows, int E, int64_t N, int64_t K) {   // the segments cut A's rows
  return least_time(shapes, (K + 63) / 64, (float)((K + 63) / 64), rows * N,
                    [&](const Shape &t) { return expected_row_tiles(rows, E, t.bm) * ((N + t.bn - 1) / t.bn); });
}
// The segments cut the sum: E M N outputs, however few rows there are; the longest segment is taken as 1.4 times the average. us with
// the shapes in turn: 16384 rows of 32 experts 2880 x 2880 380 and 462, 8000 of 128 768 x 2048 into bf16 145, 159, 222, 15314 of 16 1216 x 264
// 85, 60, 48, 2000 of two 2048 x 1024 44, 28, 21, 500 of four 1024 x 1024 12, 7, 7, 15313 of three 248 x 824 in four parts 44, 31, 26.
constexpr Shape kTilesSum[] = {{256, 256, 1.35f, 6.8f, 1.35f}, {128, 128, 0.46f, 2.2f, 1.1f}, {128, 128, 0.52f, 5.3f, 0.57f, 4}};
inline Plan plan_sum(int64_t rows, int E, int64_t M, int64_t N) {
  const float mean = E == 1 ? (float)(rows / 64 + 1) : (float)rows / (64.f * (float)E) + 1.f;
  return least_time(kTilesSum, (E == 1 ? rows : rows * 7 / (5 * E)) / 64 + 1, mean, E * M * N,
                    [&](const Shape &t) { return (int64_t)E * ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn); });
}
inline int64_t part_bytes(const Plan &p, int64_t outputs) { return p.splits > 1 ? p.splits * outputs * 4 : 0; }

// the plan's parts in the caller's workspace
inline int in_parts(Args &a, const Plan &p, int64_t outputs, void *workspace, int64_t bytes) {
  a.splits = p.splits;
  a.part = static_cast<float *>(workspace);
  if (p.splits == 1) return QMM_OK;
  if (!workspace || bytes < part_bytes(p, outputs)) return QMM_ERR_WORKSPACE;
  return aligned(workspace, 16) ? QMM_OK : QMM_ERR_ALIGN;
}
inline int launch_join(const Args &in, int64_t rows, int64_t outputs, hipStream_t s) {
  Args a = in;
  a.tiles_n = (a.N + kJoinCols - 1) / kJoinCols;
  a.rows = (int)rows;
  a.rest = 0;
  const int64_t tiles = most_row_tiles(a, kJoinRows) * a.tiles_n;
  if (tiles > kMaxTiles) return QMM_ERR_SHAPE;
  const dim3 grid = tile_grid(tiles, 0, 1);
  switch (a.splits) {
    case 2: join_kernel<2><<<grid, dim3(256), 0, s>>>(a, outputs); break;
    case 4: join_kernel<4><<<grid, dim3(256), 0, s>>>(a, outputs); break;
    case 8: join_kernel<8><<<grid, dim3(256), 0, s>>>(a, outputs); break;
    default: join_kernel<16><<<grid, dim3(256), 0, s>>>(a, outputs); break;
  }
  return launch_status();
}

template <int DT, int SA, int SB, int SUM, int BM, int BN, int WM, int WN, int GS, int ST = 2>
int launch(const Args &in, hipStream_t s) {
  Args a = in;
  a.tiles_n = (a.N + BN - 1) / BN;
  const int64_t tiles = SUM == kSumRagged ? ((int64_t)((a.M + BM - 1) / BM) * a.tiles_n + 7) / 8 * 8 * a.E : most_row_tiles(a, BM) * a.tiles_n;
  if (tiles > kMaxTiles) return QMM_ERR_SHAPE;
  constexpr int lds = ST * (BM + BN) * 128;
  auto *fn = tile_mm_kernel<DT, SA, SB, SUM, BM, BN, WM, WN, GS, ST>;
  static std::atomic<unsigned> raised{0};
  if (int st = raise_dyn_lds(reinterpret_cast<const void *>(fn), lds, raised)) return st;
  fn<<<tile_grid(tiles, a.rest, a.splits), dim3(64 * WM * WN), lds, s>>>(a);
  if (int st = launch_status()) return st;
  if (a.splits == 1) return QMM_OK;
  if (SUM == kSumFixed) return launch_join(a, a.rows, (int64_t)a.rows * a.N, s);
  a.offsets = nullptr;   // every matrix is written
  a.scales = nullptr;
  return launch_join(a, (int64_t)a.E * a.M, (int64_t)a.E * a.M * a.N, s);
}
template <int DT, int SA, int SB, int GS>
int launch_shape(const Args &a, int shape, hipStream_t s) {
  if constexpr (SB == kW4Col) {
    if (shape == 3) return launch<DT, SA, SB, kSumFixed, 256, 128, 4, 2, GS>(a, s);
  } else {
    if (shape == 3) return launch<DT, SA, SB, kSumFixed, 64, 128, 1, 4, GS, 4>(a, s);
    if (shape == 4) return launch<DT, SA, SB, kSumFixed, 128, 128, 2, 4, GS, 4>(a, s);
  }
  switch (shape) {
    case 0: return launch<DT, SA, SB, kSumFixed, 256, 256, 2, 4, GS>(a, s);
    case 1: return launch<DT, SA, SB, kSumFixed, 128, 128, 2, 2, GS>(a, s);
    default: return launch<DT, SA, SB, kSumFixed, 64, 128, 1, 4, GS>(a, s);
  }
}

}  // namespace tmm
}  // namespace qmm

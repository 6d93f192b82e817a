// Many rows times 4-bit weights with group scales: the f16 operand's product, the weights taken from global memory straight into
// registers.
//
//   y[t, r] = scales[t] sum_c x16[t, c] f16(s[r, g] (q[r, c] - z[r, g]))
//
// What stands beside the MFMAs is the dequantization, 15 instructions a lane and 8 values against NI MFMAs of 32 x 32 x 16. A lane
// of the MFMA's B operand holds 8 values of a row, which is one word of a packed tile (16 rows x 128 values): its two 16-byte
// pieces of a tile are its operands of eight MFMA steps, and no other wave of the workgroup repeats them: four waves share 32 NI
// rows and own 32 NJ columns each. x goes straight into LDS 128 values at a time (rows of 256 bytes, chunk i at i ^ row % 16, for
// conflict-free fragment reads), double buffered; codes, scales and x of the next 128 values are loaded before this one's MFMAs,
// and one barrier ends the turn. Weights dequantized into LDS and read as fragments from there: 496 us at 8192 x 8192 x 4096
// against 469 here, 131 against 99 at 8000 rows of 128 experts 1536 x 2048.
#include "w4_mm.hpp"

namespace qmm {
using namespace tmm;

namespace {

// NI: blocks of 32 rows a workgroup; NJ: blocks of 32 columns a wave. Four waves a SIMD of the smallest tile (8000 rows of 128 experts
// 1536 x 2048 96 us, three 98).
template <int NI, int NJ, int GS>
__global__ __launch_bounds__(256, NI * NJ == 2 ? 4 : 2) void w4_gemm_kernel(Args a) {
  constexpr int kRows = 32 * NI, kTurn = kRows * 256, LX = 2 * NI;   // LDS bytes of 128 values of x, and a wave's loads of them
  constexpr int G = 4 / GS, kStage = 32 * stage_pitch<NJ>();
  extern __shared__ __align__(1024) u8 smem[];   // x [2]; then the staging areas
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  int e = 0, lo = 0, hi = a.rows, m0, nt;
  if (rest_done(a)) return;
  if (!row_tile<kRows>(a, e, lo, hi, m0, nt)) return;
  const int n0 = nt * 128 * NJ + wave * 32 * NJ, rows = min(kRows, max(hi - lo, 0) - m0), T = (a.K + 127) >> 7;
  const int T0 = part_of(T, a.splits, blockIdx.y), T1 = part_of(T, a.splits, blockIdx.y + 1);   // this layer's turns

  // x: load i of a wave is rows 4 (4 i + wave) .. + 3
  const u8 *xp = a.a + (int64_t)(lo + m0) * a.a_row;
  const int a_row = (int)a.a_row, x_bytes = rows * a_row;
  const u32 lds0 = (u32)(uintptr_t)(__attribute__((address_space(3))) u8 *)smem;
  u32 off[LX];
  int col[LX];
#pragma unroll
  for (int i = 0; i < LX; ++i) {
    const int row = 4 * (4 * i + wave) + (lane >> 4), ch = (lane & 15) ^ (row & 15);
    off[i] = (u32)(row * a_row + 16 * ch);
    col[i] = 8 * ch;
  }
  auto load_x = [&](int t, int buf) __attribute__((always_inline)) {   // past K: zeros
#pragma unroll
    for (int i = 0; i < LX; ++i)
      lds_load16(resource(xp + (int64_t)t * 256, x_bytes - t * 256), 128 * t + col[i] < a.K ? off[i] : kPast,
                 __builtin_amdgcn_readfirstlane(lds0 + (u32)(buf * kTurn + (4 * i + wave) * 1024)));
  };

  // the lane's columns' codes and scales; columns past the last read its row block's neighbours and are not stored
  const u8 *wp[NJ];
  const u32 *sp[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int64_t rb = (int64_t)e * a.w_blocks + min((n0 >> 4) + 2 * j + (c >> 4), a.w_blocks - 1);
    wp[j] = a.b + rb * a.w_tiles * 1024 + (16 * h + (c & 15)) * 16;
    sp[j] = a.ws + rb * a.groups * 16 + (c & 15);
  }
  struct Turn {
    u32x4 q[NJ][2];   // words i: values 32 i + 8 h .. and 32 i + 16 + 8 h ..
    u32 s[NJ][G];
  };
  auto load_w = [&](int t, Turn &w) __attribute__((always_inline)) {
    t = min(t, T - 1);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int p = 0; p < 2; ++p) w.q[j][p] = *reinterpret_cast<const u32x4 *>(wp[j] + (int64_t)t * 1024 + 512 * p);
#pragma unroll
      for (int g = 0; g < G; ++g) w.s[j][g] = sp[j][min((4 * t + GS * g) >> a.gshift, a.groups - 1) * 16];
    }
  };

  f32x16 acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  auto walk = [&](auto blocks) __attribute__((always_inline)) {
    constexpr int NA = decltype(blocks)::value;
    auto turn = [&](int t, int buf, const Turn &w, Turn &next) __attribute__((always_inline)) {
      load_x(t + 1, buf ^ 1);
      load_w(t + 1, next);
      __builtin_amdgcn_sched_barrier(0);
      const u8 *x = smem + buf * kTurn;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        u32x4 fa[NA > 0 ? NA : 1], fb[NJ];
#pragma unroll
        for (int i = 0; i < NA; ++i)
          fa[i] = *reinterpret_cast<const u32x4 *>(x + (32 * i + c) * 256 + (((2 * kk + h) ^ (c & 15)) * 16));
        if constexpr (NA > 0) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) fb[j] = dequant(w.q[j][kk & 1][kk >> 1], w.s[j][(kk >> 1) / GS]);
        }
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = mfma<QMM_F16>(fa[i], fb[j], acc[i][j]);
      }
      wait_all_barrier();
    };
    Turn w0, w1;
    load_x(T0, 0);
    load_w(T0, w0);
    wait_all_barrier();
    int t = T0;
    for (; t + 1 < T1; t += 2) {
      turn(t, 0, w0, w1);
      turn(t + 1, 1, w1, w0);
    }
    if (t < T1) turn(t, 0, w0, w1);
  };
  const int live = n0 < a.N ? (rows + 31) >> 5 : 0;
  if (live == NI) walk(std::integral_constant<int, NI>{});
  else if (live == 0) walk(std::integral_constant<int, 0>{});
  else if (live == 1) walk(std::integral_constant<int, 1>{});
  else if (NI > 2 && live == 2) walk(std::integral_constant<int, NI < 2 ? NI : 2>{});
  else if (NI > 2) walk(std::integral_constant<int, NI < 3 ? NI : 3>{});

  to_part(a, (int64_t)a.rows * a.N);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if (i >= live) break;
    store_rows<NJ>(a, reinterpret_cast<float *>(smem) + wave * kStage, acc[i], (int64_t)lo * a.N, m0 + 32 * i, hi - lo, n0,
                   a.scales ? a.scales + 2 * (int64_t)lo : nullptr, lane);
  }
}

template <int NI, int NJ, int GS>
int launch_one(const Args &in, hipStream_t s) {
  Args a = in;
  a.tiles_n = (a.N + 128 * NJ - 1) / (128 * NJ);
  const int64_t tiles = most_row_tiles(a, 32 * NI) * a.tiles_n;
  if (tiles > kMaxTiles) return QMM_ERR_SHAPE;
  constexpr int stage = 4 * 32 * stage_pitch<NJ>() * 4, x = 2 * 32 * NI * 256, lds = stage > x ? stage : x;
  auto *fn = w4_gemm_kernel<NI, NJ, GS>;
  static std::atomic<unsigned> raised{0};
  if (int st = raise_dyn_lds(reinterpret_cast<const void *>(fn), lds, raised)) return st;
  fn<<<tile_grid(tiles, a.rest, a.splits), dim3(256), lds, s>>>(a);
  if (int st = launch_status()) return st;
  return a.splits == 1 ? QMM_OK : launch_join(a, a.rows, (int64_t)a.rows * a.N, s);
}
template <int NI, int NJ>
int launch_gs(const Args &a, int gs, hipStream_t s) {
  return gs == 1 ? launch_one<NI, NJ, 1>(a, s) : gs == 2 ? launch_one<NI, NJ, 2>(a, s) : launch_one<NI, NJ, 4>(a, s);
}

}  // namespace

// Figures as those of tile_mm.hpp's shapes, for turns of 128 values: 2 % from the fastest choice on average. us at 8192 x 8192 x 4096 64
// x 128 559, 64 x 256 525, 128 x 128 525, 128 x 256 469, at 333 x 12288 x 4096 52, 65, 58, 65, at 2048 x 4096 x 12288 223, 218, 203, 199, at
// 8000 rows of 128 experts 1536 x 2048 96, 100, 118, 110.
static constexpr Shape shapes[] = {{64, 128, 0.5f, 1.f, 0.55f}, {64, 256, 1.06f, 1.5f, 1.05f}, {128, 128, 1.06f, 1.5f, 1.05f},
                                   {128, 256, 1.83f, 2.5f, 1.9f}};
const Shape &w4_gemm_shape(int shape) { return shapes[shape]; }
Plan w4_gemm_plan(int64_t rows, int E, int64_t N, int64_t K) {
  return least_time(shapes, (K + 127) / 128, (float)((K + 127) / 128), rows * N,
                    [&](const Shape &t) { return expected_row_tiles(rows, E, t.bm) * ((N + t.bn - 1) / t.bn); });
}
int w4_gemm(const Args &a, int shape, int gs, hipStream_t s) {
  switch (shape) {
    case 0: return launch_gs<2, 1>(a, gs, s);
    case 1: return launch_gs<2, 2>(a, gs, s);
    case 2: return launch_gs<4, 1>(a, gs, s);
    default: return launch_gs<4, 2>(a, gs, s);
  }
}

}  // namespace qmm

// 4-bit weights with group scales and zero points, W[r, c] = s[r, c / group] (q[r, c] - z[r, c / group]): argument checks, the
// layout's one-time preparation and the choice of the kernel by the operand's type.
//
//   qmm_w4_pack   codes, scales, zero points -> tiles and scale words
//   qmm_w4_mm     y = x W^T: f32 / bf16 rows on few_rows.hpp (exact products), the row-scaled f16 operand on tile_mm.hpp
//   qmm_w4_mm_t   dx = dy W on tile_mm.hpp
//
// Tiles of 16 rows x 128 values, 1 KB each, so that every load is a contiguous run of a wave: lane 16 h + r holds values
// 32 j + 8 h .. + 7 of row r in its word j (0 .. 3), the eight values of one lane of a 32-value MFMA step; values 0 - 3 of the
// eight are the low nibbles of the word's bytes and 4 - 7 the high ones, so that one mask gives four neighbouring values.
#include "w4_mm.hpp"

using namespace qmm;

namespace {

constexpr int64_t kMaxSide = 1 << 20, kMaxRows = 1 << 24;

int64_t blocks(int64_t n) { return (n + 15) / 16; }
int64_t tiles(int64_t k) { return (k + 127) / 128; }
int64_t groups_of(int64_t k, int64_t group) { return (k + group - 1) / group; }
// a group is 32 2^i values, or whole rows
bool shape_ok(int64_t n, int64_t k, int64_t group) {
  if (n <= 0 || n > kMaxSide || k <= 0 || k > kMaxSide || k % 32) return false;
  return group >= k || (group >= 32 && (group & (group - 1)) == 0);
}
// 32-value step i lies in group i >> shift
int group_shift(int64_t k, int64_t group) {
  if (group >= k) return 31;
  int s = 0;
  while ((32ll << s) < group) ++s;
  return s;
}
// 32-value steps of a 128-value tile that share a scale
int group_steps(int64_t k, int64_t group) { return group >= k || group >= 128 ? 4 : (int)(group / 32); }

// thread: a lane's 16 bytes of a tile, [experts][n / 16][k / 128][64]
__global__ void w4_pack_kernel(const u8 *codes, u32 *w, int n, int k, int64_t items) {
  const int64_t at = item_index() * 256 + threadIdx.x;
  if (at >= items) return;
  const int nb = (n + 15) >> 4, nt = (k + 127) >> 7, l = (int)(at & 63);
  const int64_t tile = at >> 6, block = tile / nt, e = block / nb;
  const int r = (int)(block - e * nb) * 16 + (l & 15), c0 = (int)(tile - block * nt) * 128 + 8 * (l >> 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    u32 v = 0;
    const int c = c0 + 32 * j;
    if (r < n && c < k) {
      const u8 *q = codes + (e * n + r) * (int64_t)k + c;
#pragma unroll
      for (int b = 0; b < 4; ++b) v |= (u32)((q[b] & 15) | (q[4 + b] & 15) << 4) << (8 * b);
    }
    w[4 * at + j] = v;
  }
}
// thread: a scale word, [experts][n / 16][groups][16]
__global__ void w4_scales_kernel(const u16 *scales, const u8 *zeros, u32 *ws, int n, int groups, int64_t items) {
  const int64_t at = item_index() * 256 + threadIdx.x;
  if (at >= items) return;
  const int nb = (n + 15) >> 4;
  const int64_t i = at >> 4, block = i / groups, e = block / nb;
  const int r = (int)(block - e * nb) * 16 + (int)(at & 15), g = (int)(i - block * groups);
  u32 v = 0x64000000u;
  if (r < n) {
    const int64_t src = (e * n + r) * (int64_t)groups + g;
    v |= scales[src] | (zeros ? (u32)(zeros[src] & 15) : 8u) << 16;
  }
  ws[at] = v;
}

int check(int64_t rows, int64_t k, int64_t n, int64_t group, int E, const int32_t *offsets, const void *x, const void *w,
          const void *ws, const void *y, int &y_dtype, int &rest) {
  rest = zero_rest_asked(y_dtype) && offsets;
  if (!shape_ok(n, k, group) || rows < 0 || rows > kMaxRows) return QMM_ERR_SHAPE;
  if (E < 1 || E > kMaxRaggedE || (!offsets && E != 1)) return QMM_ERR_RANGE;
  if (y_dtype != QMM_F32 && y_dtype != QMM_BF16) return QMM_ERR_DTYPE;
  if (rows && (!x || !w || !ws || !y)) return QMM_ERR_NULL;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(ws, 16) || !aligned(offsets, 4) || !aligned(y, y_dtype == QMM_F32 ? 4 : 2))
    return QMM_ERR_ALIGN;
  return QMM_OK;
}

tmm::Args tile_args(int64_t rows, int64_t k, int64_t n, int64_t group, int E, const int32_t *offsets, const void *x,
                    const float *scales, const void *w, const void *ws, void *y, int y_dtype, int64_t N, int rest) {
  tmm::Args a{};
  a.offsets = offsets;
  a.E = E;
  a.rows = (int)rows;
  a.a = static_cast<const u8 *>(x);
  a.b = static_cast<const u8 *>(w);
  a.b_expert = blocks(n) * tiles(k) * 1024;
  a.ws = static_cast<const u32 *>(ws);
  a.w_blocks = (int)blocks(n);
  a.w_tiles = (int)tiles(k);
  a.groups = (int)groups_of(k, group);
  a.gshift = group_shift(k, group);
  a.scales = scales;
  a.y = y;
  a.y_type = y_dtype;
  a.N = (int)N;
  a.splits = 1;
  a.rest = rest ? rest_blocks(rows, N * (y_dtype == QMM_F32 ? 4 : 2)) : 0;
  return a;
}

bool sizes_ok(int64_t rows, int64_t k, int64_t n, int E) {
  return shape_ok(n, k, k) && rows >= 0 && rows <= kMaxRows && E >= 1 && E <= kMaxRaggedE;
}

}  // namespace

extern "C" int64_t qmm_w4_bytes(int64_t n, int64_t k) {
  return shape_ok(n, k, k) ? blocks(n) * tiles(k) * 1024 : -1;
}
extern "C" int64_t qmm_w4_scale_bytes(int64_t n, int64_t k, int64_t group) {
  return shape_ok(n, k, group) ? blocks(n) * groups_of(k, group) * 64 : -1;
}

extern "C" int qmm_w4_pack(int E, int64_t n, int64_t k, int64_t group, const uint8_t *codes, const void *scales,
                           const uint8_t *zeros, void *w, void *ws, qmm_stream_t stream) {
  if (!shape_ok(n, k, group)) return QMM_ERR_SHAPE;
  if (E < 1 || E > kMaxRaggedE) return QMM_ERR_RANGE;
  if (!codes || !scales || !w || !ws) return QMM_ERR_NULL;
  if (!aligned(w, 16) || !aligned(ws, 16) || !aligned(scales, 2)) return QMM_ERR_ALIGN;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t g = groups_of(k, group), units = E * blocks(n) * tiles(k) * 64, words = E * blocks(n) * g * 16;
  w4_pack_kernel<<<item_grid((units + 255) / 256), 256, 0, s>>>(codes, static_cast<u32 *>(w), (int)n, (int)k, units);
  w4_scales_kernel<<<item_grid((words + 255) / 256), 256, 0, s>>>(static_cast<const u16 *>(scales), zeros,
                                                                  static_cast<u32 *>(ws), (int)n, (int)g, words);
  return launch_status();
}

extern "C" int64_t qmm_w4_mm_workspace_size(int64_t rows, int64_t k, int64_t n, int E, int x_dtype) {
  if (!sizes_ok(rows, k, n, E)) return -1;
  if (!rows) return 0;
  if (x_dtype == QMM_F16) return tmm::part_bytes(w4_gemm_plan(rows, E, n, k), rows * n);
  return tmm::part_bytes({0, few::parts_of(rows, n, k, E, x_dtype == QMM_F32)}, rows * n);
}
extern "C" int64_t qmm_w4_mm_t_workspace_size(int64_t rows, int64_t k, int64_t n, int E) {
  if (!sizes_ok(rows, k, n, E)) return -1;
  return rows ? tmm::part_bytes(tmm::plan_rows(tmm::kTilesW4, rows, E, k, n), rows * k) : 0;
}

extern "C" int qmm_w4_mm(int64_t rows, int64_t k, int64_t n, int64_t group, int E, const int32_t *offsets, const void *x,
                         int x_dtype, const float *x_scales, const void *w, const void *ws, void *y, int y_dtype,
                         void *workspace, int64_t workspace_bytes, qmm_stream_t stream) {
  if (x_dtype != QMM_F32 && x_dtype != QMM_BF16 && x_dtype != QMM_F16) return QMM_ERR_DTYPE;
  int rest;
  if (int st = check(rows, k, n, group, E, offsets, x, w, ws, y, y_dtype, rest)) return st;
  if (!aligned(x_scales, 4)) return QMM_ERR_ALIGN;
  if (rows == 0) return QMM_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (x_dtype == QMM_F16) {
    tmm::Args a = tile_args(rows, k, n, group, E, offsets, x, x_scales, w, ws, y, y_dtype, n, rest);
    a.a_row = 2 * k;
    a.K = (int)k;
    const tmm::Plan p = w4_gemm_plan(rows, E, n, k);
    if (int st = in_parts(a, p, rows * n, workspace, workspace_bytes)) return st;
    return w4_gemm(a, p.shape, group_steps(k, group), s);
  }
  few::Args a{offsets, E, (int)rows, (int)n, (int)k, static_cast<const u8 *>(x), static_cast<const u8 *>(w),
              blocks(n) * tiles(k) * 1024, static_cast<const u32 *>(ws), (int)groups_of(k, group),
              group_shift(k, group), y, y_dtype == QMM_F32 ? 4 : 2};
  tmm::Args join = tile_args(rows, k, n, group, E, offsets, x, nullptr, w, ws, y, y_dtype, n, 0);
  const tmm::Plan p = {0, few::parts_of(rows, n, k, E, x_dtype == QMM_F32)};
  if (int st = in_parts(join, p, rows * n, workspace, workspace_bytes)) return st;
  a.parts = p.splits;
  a.part = join.part;
  a.rest = rest;
  if (int st = w4_few(a, x_dtype == QMM_F32, group_steps(k, group), s)) return st;
  return p.splits > 1 ? tmm::launch_join(join, rows, rows * n, s) : QMM_OK;
}

extern "C" int qmm_w4_mm_t(int64_t rows, int64_t k, int64_t n, int64_t group, int E, const int32_t *offsets, const void *x,
                           const float *scales, const void *w, const void *ws, void *y, int y_dtype, void *workspace,
                           int64_t workspace_bytes, qmm_stream_t stream) {
  int rest;
  if (int st = check(rows, k, n, group, E, offsets, x, w, ws, y, y_dtype, rest)) return st;
  if (rows && !scales) return QMM_ERR_NULL;
  if (!aligned(scales, 4)) return QMM_ERR_ALIGN;
  if (rows == 0) return QMM_OK;
  tmm::Args a = tile_args(rows, k, n, group, E, offsets, x, scales, w, ws, y, y_dtype, k, rest);
  a.K = (int)((n + 63) / 64 * 64);
  a.a_row = 2 * (int64_t)a.K;
  const tmm::Plan p = tmm::plan_rows(tmm::kTilesW4, rows, E, k, n);
  if (int st = in_parts(a, p, rows * k, workspace, workspace_bytes)) return st;
  return w4_gemm_t(a, p.shape, group_steps(k, group), reinterpret_cast<hipStream_t>(stream));
}

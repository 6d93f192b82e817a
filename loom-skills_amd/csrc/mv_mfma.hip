// Products of a few rows (a batch of decoding sequences, drafted tokens) with the epilogue of qmm_linear / qmm_ffn_gate_up, on
// the bf16 MFMA with exact operands:
//
//   v[t, r] = sum_k x[t, k] W[r, k],   W in Q4_0 / Q4_K / Q6_K / MXFP4 blocks or MXFP4 split planes,
//   x bf16 rows, f32 rows, or planar Q8_1
//
// The matvec kernels read and unpack every weight once per two or four tokens and take an fma per product: their time grows
// with the tokens (4096 x 4096 f32 rows, Q6_K: 16 us at two tokens, 482 at 63). Here a weight is unpacked once per 16 tokens,
// into its integer code (at most 6 bits, exact in bf16) or its E2M1 value, and 16 x 16 x 32 products take one
// v_mfma_f32_16x16x32_bf16. The activations are exact too: a bf16 row is its own operand, a Q8_1 code is an integer below 128,
// and an f32 value is the sum of three bf16 values (its leading 8 bits, the next 8, the rest: three MFMAs). So every product is
// exact and every sum f32, as in the matvec kernels; the block scales join after the MFMA, in f32:
//
//   Q4_0    d (dot - 8 S)          Q4_K  (d sc) dot - (dmin m) S        S the block's sum of x (an MFMA with ones, or Q8_1's)
//   Q6_K    (d sc) dot a 16-value run (a second MFMA with the other run's lanes zero); codes as 16 (h - 2) + l from the two
//           parts that are stored, each exact
//   MXFP4   2^e dot                Q8_1: times the group's da
//
// What bounds it: the vector instructions that unpack weights and split activations (30 - 90 a group of 16 rows x 32 values) in
// large calls (Q6_K 12288 x 4096 at 63 rows: vector pipes 0.67 busy on f32 rows, 0.65 on Q8_1, MFMA 0.32 and 0.19, waves waiting
// 0.33 and 0.40 of their time); in small ones those and the wait for loads alike (Q4_0 6144 x 2048, five f32 rows: 0.50, waiting
// 0.42). Gate and up at once: Q4_0 2 x 6144 x 2048 13.4 us at five f32 rows, 18.5 at 33 bf16 rows; Q6_K 2 x 4096 x 4096 21.0 at 17
// Q8_1 rows. Loads are coalesced (neighbouring lanes on neighbouring bytes, through the wave's own LDS): with every lane reading
// its own row the address unit took 64 cycles a load and was the bound (12288 x 4096 Q4_0, bf16 rows, two tokens: 32 us).
//
// A workgroup: RT tiles of 16 weight rows (of each of NM matrices) x TT tiles of 16 tokens, eight waves. A wave takes whole
// chunks of 256 values of all its rows (chunk v, v + 8, ...): it brings the rows' bytes into its own LDS, then the tokens' values
// 64 at a time, the next chunk's and the next 64 values' loads in flight. Its sums stay in registers (four a pair of tiles: lane
// (c, q) = (lane % 16, lane / 16), register i is token 4 q + i, row c, so a row's scale is one register) and the waves' meet in
// LDS at the end, in order. A token's result does not depend on the tokens beside it.
// MFMA operands: lane (c, q) holds 8 K values of token c / weight row c, K positions F::kpos(q) .. + 7 of a 32-value group.
#include <type_traits>

#include "epilogue.hpp"
#include "rowdot.hpp"

using namespace qmm;

namespace {

typedef __attribute__((ext_vector_type(4))) u32 u32x4;
typedef __attribute__((ext_vector_type(2))) u32 u32x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

constexpr int kWaves = 8;
enum XType { kXF32 = 0, kXBF16 = 1, kXQ8 = 2 };

__device__ __forceinline__ bf16x8 as_frag(u32 a, u32 b, u32 c, u32 d) { return __builtin_bit_cast(bf16x8, u32x4{a, b, c, d}); }
__device__ __forceinline__ f32x4 mfma(bf16x8 x, bf16x8 w, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w, c, 0, 0, 0); }
// the codes in the low nibbles of four bytes as bf16 pairs: 0000qqqq read as OCP E4M3 is q 2^-9 exactly
__device__ __forceinline__ bf16x8 code_frag(u32 n0, u32 n1) {
  return as_frag(__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(n0, 512.f, false)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(n0, 512.f, true)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(n1, 512.f, false)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(n1, 512.f, true)));
}
__device__ __forceinline__ u32 ld2any(const u8 *p) {
  typedef u16 u16_a1 __attribute__((aligned(1)));
  return *reinterpret_cast<const u16_a1 *>(p);
}
__device__ __forceinline__ u32 lds4(const u8 *p) { return *reinterpret_cast<const u32 *>(p); }

// A format's chunk of 256 values of 16 rows. kPiece bytes a lane and load, kPieces pieces a row, kLoads loads; a row's chunk is
// kChunk bytes in memory (kGroup a 32-value group) and lies kStride apart in LDS (gcd with the 64 banks' 256 bytes at most 16:
// a read of one place in 16 rows meets 16 banks). Side: what a lane keeps of row c in registers. unpack: group g of row c;
// apply: its terms joined into y.
struct FQ40 {   // 18-byte blocks: d, 16 bytes (low nibbles values 0..15)
  static constexpr int kPiece = 4, kPieces = 36, kChunk = 144, kGroup = 18, kStride = 144;
  static constexpr bool kSum = true;
  struct Side {};
  struct U { bf16x8 w; float d; };
  static __device__ __forceinline__ int kpos(int q) { return 8 * q; }
  static __device__ __forceinline__ void side(Side &, const u8 *, const u8 *, int) {}
  static __device__ __forceinline__ void unpack(U &u, const u8 *l, const Side &, int g, int q) {
    // the codes start at 18 g + 2: two bytes into a dword for even g
    const u8 *p = l + 18 * g + 8 * (q & 1) + (g & 1 ? 2 : 0);
    u32 a = lds4(p), b = lds4(p + 4);
    u.d = f16_to_f32(*reinterpret_cast<const u16 *>(l + 18 * g));
    if (!(g & 1)) {
      const u32 c = lds4(p + 8);
      a = __builtin_amdgcn_alignbit(b, a, 16);
      b = __builtin_amdgcn_alignbit(c, b, 16);
    }
    const int sh = 4 * (q >> 1);
    u.w = code_frag((a >> sh) & 0x0F0F0F0Fu, (b >> sh) & 0x0F0F0F0Fu);
  }
  template <class D, class J>
  static __device__ __forceinline__ void apply(const U &u, D dot, const f32x4 &S, J join) {
    const f32x4 v = dot(u.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) join(u.d, __builtin_fmaf(-8.f, S[i], v[i]), i);
  }
};

struct FQ4K {   // header, then pages of 32 bytes (low nibbles one group, high nibbles the next)
  static constexpr int kPiece = 16, kPieces = 9, kChunk = 144, kGroup = 18, kStride = 144;
  static constexpr bool kSum = true;
  struct Side {};
  struct U { bf16x8 w; float ds, dm; };
  static __device__ __forceinline__ int kpos(int q) { return 8 * q; }
  static __device__ __forceinline__ void side(Side &, const u8 *, const u8 *, int) {}
  static __device__ __forceinline__ void unpack(U &u, const u8 *l, const Side &, int g, int q) {
    const u32x2 n = *reinterpret_cast<const u32x2 *>(l + 16 + 32 * (g >> 1) + 8 * q);
    const u32x4 h = *reinterpret_cast<const u32x4 *>(l);
    const int sh = 4 * (g & 1);
    u.w = code_frag((n.x >> sh) & 0x0F0F0F0Fu, (n.y >> sh) & 0x0F0F0F0Fu);
    u32 sc, mn;
    q4k_scale_min(h.y, h.z, h.w, g, sc, mn);
    u.ds = f16_to_f32(h.x) * (float)sc;
    u.dm = f16_to_f32(h.x >> 16) * (float)mn;
  }
  template <class D, class J>
  static __device__ __forceinline__ void apply(const U &u, D dot, const f32x4 &S, J join) {
    const f32x4 v = dot(u.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) join(1.f, __builtin_fmaf(u.ds, v[i], -(u.dm * S[i])), i);
  }
};

struct FQ6K {   // 208 bytes in LDS (ql, qh, 16 scales), d in a register; 16-value runs have their own scale
  static constexpr int kPiece = 4, kPieces = 52, kChunk = 210, kGroup = 26, kStride = 208;
  static constexpr bool kSum = false;
  struct Side { u32 d; };
  struct U { bf16x8 lo[2], hi[2]; float s[2]; };
  static __device__ __forceinline__ int kpos(int q) { return 8 * q; }
  static __device__ __forceinline__ void side(Side &s, const u8 *row, const u8 *, int chunk) {
    s.d = *reinterpret_cast<const u16 *>(row + 210 * (int64_t)chunk + 208);
  }
  // 16 (h - 2) of the two-bit parts h of four bytes, as bf16 pairs: -32, -16, 0, 16 by table
  static __device__ __forceinline__ void high(u32 s, u32 &a, u32 &b) {
    const u32 hi = __builtin_amdgcn_perm(0u, 0x4100C1C2u, s), lo = __builtin_amdgcn_perm(0u, 0x80008000u, s);
    a = __builtin_amdgcn_perm(hi, lo, 0x05010400u);
    b = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
  }
  static __device__ __forceinline__ void unpack(U &u, const u8 *l, const Side &sd, int g, int q) {
    const int hb = g >> 2, j = g & 3;   // group j of half hb: ql bytes 32 (j % 2) .., nibble j / 2; qh bits 2 j
    const u32x2 ql = *reinterpret_cast<const u32x2 *>(l + 64 * hb + 32 * (j & 1) + 8 * q);
    const u32x2 qh = *reinterpret_cast<const u32x2 *>(l + 128 + 32 * hb + 8 * q);
    const u32 sc = *reinterpret_cast<const u16 *>(l + 192 + 2 * g);
    const int sh = 4 * (j >> 1);
    const u32x4 lo = __builtin_bit_cast(u32x4, code_frag((ql.x >> sh) & 0x0F0F0F0Fu, (ql.y >> sh) & 0x0F0F0F0Fu));
    u32x4 hi;
    u32 a, b;
    high((qh.x >> (2 * j)) & 0x03030303u, a, b);
    hi.x = a; hi.y = b;
    high((qh.y >> (2 * j)) & 0x03030303u, a, b);
    hi.z = a; hi.w = b;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    const float d = f16_to_f32(sd.d);
#pragma unroll
    for (int run = 0; run < 2; ++run) {   // the run's 16 values are those of lanes q / 2 = run
      const bool mine = (q >> 1) == run;
      u.lo[run] = __builtin_bit_cast(bf16x8, mine ? lo : zero);
      u.hi[run] = __builtin_bit_cast(bf16x8, mine ? hi : zero);
      u.s[run] = d * (float)(signed char)((sc >> (8 * run)) & 0xFFu);
    }
  }
  template <class D, class J>
  static __device__ __forceinline__ void apply(const U &u, D dot, const f32x4 &, J join) {
#pragma unroll
    for (int run = 0; run < 2; ++run) {
      const f32x4 v = dot(u.lo[run], u.hi[run]);
#pragma unroll
      for (int i = 0; i < 4; ++i) join(u.s[run], v[i], i);
    }
  }
};

// E2M1 pairs of a byte, low nibble first
template <int B>
__device__ __forceinline__ u32 fp4_pair(u32 w) { return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, B)); }

struct FMX {   // 17-byte blocks: E8M0, 16 bytes (low nibbles values 0..15)
  static constexpr int kPiece = 4, kPieces = 34, kChunk = 136, kGroup = 17, kStride = 136;
  static constexpr bool kSum = false;
  struct Side {};
  struct U { bf16x8 w; float s; };
  static __device__ __forceinline__ int kpos(int q) { return 8 * q; }
  static __device__ __forceinline__ void side(Side &, const u8 *, const u8 *, int) {}
  static __device__ __forceinline__ void unpack(U &u, const u8 *l, const Side &, int g, int q) {
    const int at = 17 * g + 1, sh8 = 8 * (at & 3);
    const u8 *p = l + (at & ~3) + 8 * (q & 1);
    u32 n[2] = {lds4(p), lds4(p + 4)};
    if (sh8) {
      const u32 c = lds4(p + 8);
      n[0] = __builtin_amdgcn_alignbit(n[1], n[0], sh8);
      n[1] = __builtin_amdgcn_alignbit(c, n[1], sh8);
    }
    u32 w[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // four nibbles of four bytes, as two pairs in bytes 0 and 2
      const u32 v = (n[i] >> (4 * (q >> 1))) & 0x0F0F0F0Fu, b = v | (v >> 4);
      w[2 * i] = fp4_pair<0>(b);
      w[2 * i + 1] = fp4_pair<2>(b);
    }
    u.w = as_frag(w[0], w[1], w[2], w[3]);
    u.s = e8m0_scale(l[17 * g]);
  }
  template <class D, class J>
  static __device__ __forceinline__ void apply(const U &u, D dot, const f32x4 &, J join) {
    const f32x4 v = dot(u.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) join(u.s, v[i], i);
  }
};

struct FMXS {   // split planes: 16 nibble bytes a block in pairs order, the E8M0 bytes in a plane of their own
  static constexpr int kPiece = 16, kPieces = 8, kChunk = 128, kGroup = 16, kStride = 144;
  static constexpr bool kSum = false;
  struct Side { u32x2 e; };
  struct U { bf16x8 w; float s; };
  static __device__ __forceinline__ int kpos(int q) { return 8 * q; }
  static __device__ __forceinline__ void side(Side &, const u8 *, const u8 *, int) {}
  static __device__ __forceinline__ void unpack(U &u, const u8 *l, const Side &sd, int g, int q) {
    const u32 w = lds4(l + 16 * g + 4 * q);
    u.w = as_frag(fp4_pair<0>(w), fp4_pair<1>(w), fp4_pair<2>(w), fp4_pair<3>(w));
    u.s = e8m0_scale((sd.e[g >> 2] >> (8 * (g & 3))) & 0xFFu);
  }
  template <class D, class J>
  static __device__ __forceinline__ void apply(const U &u, D dot, const f32x4 &, J join) {
    const f32x4 v = dot(u.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) join(u.s, v[i], i);
  }
};

struct MArgs {
  int n, tokens, chunks, groups;   // rows of a matrix, tokens, chunks and 32-value groups of a row (even)
  int64_t k, rb, sb;               // values, bytes and scale bytes of a row
  const void *x;                   // rows, or the planar Q8_1 codes
  const float *meta;               // Q8_1: (d, code sum) [tokens][k / 32]
  const u8 *w, *ws, *w2, *ws2;
};

template <int XT>
constexpr int x_size() { return XT == kXF32 ? 4 : XT == kXBF16 ? 2 : 1; }
// LDS bytes of 16 tokens' 64 values: a token's bytes and 16 more (Q8_1: then its two groups' pairs)
template <int XT>
constexpr int x_stride() { return 64 * x_size<XT>() + (XT == kXQ8 ? 32 : 16); }
template <class F, int XT, int RT, int NM, int TT>
constexpr int own_bytes() { return RT * NM * 16 * F::kStride + TT * 16 * x_stride<XT>(); }

template <class F, int XT, int RT, int NM, int TT>
__global__ __launch_bounds__(64 * kWaves) void mv_mfma_kernel(MArgs a, Epi ep) {
  constexpr int NX = XT == kXF32 ? 3 : 1, NL = (16 * F::kPieces + 63) / 64, MR = NM * RT;
  constexpr int kOwn = own_bytes<F, XT, RT, NM, TT>();
  extern __shared__ __align__(16) u8 smem[];   // [wave][kOwn]; at the end the waves' sums [wave][MR][TT][256]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q = lane >> 4;
  // workgroup b runs on XCD b % 8 = blockIdx.x % 8: the token tiles of a row block follow each other there and share its
  // weights in L2
  const int row0 = ((int)blockIdx.y * 8 + (int)(blockIdx.x & 7)) * (16 * RT), t0 = (int)(blockIdx.x >> 3) * (16 * TT);
  if (row0 >= a.n) return;
  u8 *const own = smem + wave * kOwn, *const xl = own + MR * 16 * F::kStride;

  // ---- weights: load i of a tile is pieces 64 i + lane of its 16 rows' chunks in order (rows past n: row n - 1); byte offsets
  // fit 32 bits (qmm_mv_mfma_fits)
  u32 woff[RT][NL];
  int wpiece[NL];   // the piece's first byte in its row's chunk, past the chunk for lanes without one
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int idx = 64 * i + lane, r = idx / F::kPieces, p = idx % F::kPieces;
    wpiece[i] = r < 16 ? p * F::kPiece : 1 << 20;
#pragma unroll
    for (int k = 0; k < RT; ++k) woff[k][i] = (u32)min(row0 + 16 * k + min(r, 15), a.n - 1) * (u32)a.rb + (u32)(p * F::kPiece);
  }
  typedef typename std::conditional<F::kPiece == 16, u32x4, u32>::type Piece;
  typedef Piece __attribute__((aligned(F::kPiece == 16 ? 16 : 1))) PieceU;
  Piece wv[MR][NL];
  typename F::Side side[MR];
  auto load_w = [&](int ch) __attribute__((always_inline)) {
    const int valid = min(8, a.groups - 8 * ch) * F::kGroup;   // bytes of the chunk that lie in the row
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const u8 *base = (m ? a.w2 : a.w) + (int64_t)ch * F::kChunk;
#pragma unroll
      for (int k = 0; k < RT; ++k) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          if (wpiece[i] + F::kPiece <= valid) wv[m * RT + k][i] = *reinterpret_cast<const PieceU *>(base + woff[k][i]);
          if constexpr (F::kGroup % 4 == 1) {   // 17-byte blocks: the last chunk can end inside a dword, perhaps the tensor too
            if (wpiece[i] + 2 == valid) wv[m * RT + k][i] = ld2any(base + woff[k][i]);
          }
        }
        const int64_t row = min(row0 + 16 * k + c, a.n - 1);
        if constexpr (std::is_same_v<F, FMXS>) {   // the row's eight E8M0 bytes (fewer in the last chunk: pairs)
          const u8 *s = (m ? a.ws2 : a.ws) + row * a.sb + 8 * ch;
          const int left = min(8, a.groups - 8 * ch);
          u32 e[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) e[h] = *reinterpret_cast<const u16 *>(s + (2 * h < left ? 2 * h : 0));
          side[m * RT + k].e = u32x2{e[0] | (e[1] << 16), e[2] | (e[3] << 16)};
        } else {
          F::side(side[m * RT + k], (m ? a.w2 : a.w) + row * a.rb, nullptr, ch);
        }
      }
    }
  };
  auto store_w = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < MR; ++t)
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int idx = 64 * i + lane;
        const int at = F::kStride == F::kPieces * F::kPiece ? F::kPiece * idx : (idx / F::kPieces) * F::kStride + (idx % F::kPieces) * F::kPiece;
        if (NL * 64 == 16 * F::kPieces || idx < 16 * F::kPieces)
          *reinterpret_cast<Piece *>(own + t * 16 * F::kStride + at) = wv[t][i];
      }
  };

  // ---- activations, 64 values of 16 tokens: 16-byte pieces, LX lanes a token (tokens past the last: the last)
  constexpr int LX = 4 * x_size<XT>(), NLX = LX / 4;   // lanes a token, loads a tile
  // pieces in flight (four are a chunk), in slots of their own; fewer where their registers would cost a workgroup a CU
  // (Q6_K on Q8_1, 12288 x 4096: 20 us with one, 25 with two)
  constexpr int kDeepX = std::is_same_v<F, FQ6K> ? 1 : XT == kXF32 || TT == 2 ? 2 : 4;
  u32x4 xv[kDeepX][TT][NLX], mv[kDeepX][TT];
  const u8 *xp[TT][NLX];
  const u8 *mp[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
#pragma unroll
    for (int i = 0; i < NLX; ++i)
      xp[t][i] = static_cast<const u8 *>(a.x) + (int64_t)min(t0 + 16 * t + (64 * i + lane) / LX, a.tokens - 1) * a.k * x_size<XT>() + 16 * (lane % LX);
    mp[t] = XT == kXQ8 ? reinterpret_cast<const u8 *>(a.meta + (int64_t)min(t0 + 16 * t + c, a.tokens - 1) * a.groups * 2) : nullptr;
  }
  // piece p of the wave's chunk ch, or of the chunk after it (p >= 4); past the row the last piece, which is not used
  auto load_x = [&](int ch, int p) __attribute__((always_inline)) {
    const int slot = p % kDeepX, at = min(4 * (ch + p / 4 * kWaves) + p % 4, a.groups / 2 - 1);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int i = 0; i < NLX; ++i) xv[slot][t][i] = *reinterpret_cast<const u32x4 *>(xp[t][i] + (int64_t)at * 64 * x_size<XT>());
      if constexpr (XT == kXQ8) mv[slot][t] = *reinterpret_cast<const u32x4 *>(mp[t] + (int64_t)at * 16);   // two groups' pairs
    }
  };
  auto store_x = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      u8 *to = xl + t * 16 * x_stride<XT>();
#pragma unroll
      for (int i = 0; i < NLX; ++i)
        *reinterpret_cast<u32x4 *>(to + ((64 * i + lane) / LX) * x_stride<XT>() + 16 * (lane % LX)) = xv[slot][t][i];
      if constexpr (XT == kXQ8) *reinterpret_cast<u32x4 *>(to + c * x_stride<XT>() + 64) = mv[slot][t];   // four lanes the same
    }
  };
  // the operand's bf16 parts: 8 values of token c, group e (0, 1) of the 64
  auto operand = [&](int t, int e, bf16x8 (&x)[NX]) __attribute__((always_inline)) {
    const u8 *p = xl + (16 * t + c) * x_stride<XT>() + (32 * e + F::kpos(q)) * x_size<XT>();
    if constexpr (XT == kXBF16) {
      x[0] = *reinterpret_cast<const bf16x8 *>(p);
    } else if constexpr (XT == kXQ8) {
      const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
      u32 o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32 d = v[i >> 1] >> (16 * (i & 1));
        const float f0 = (float)(signed char)(d & 0xFFu), f1 = (float)(signed char)((d >> 8) & 0xFFu);
        o[i] = __builtin_amdgcn_perm(f32_as_u32(f1), f32_as_u32(f0), 0x07060302u);   // the upper halves: exact
      }
      x[0] = as_frag(o[0], o[1], o[2], o[3]);
    } else {
      const u32x4 v[2] = {*reinterpret_cast<const u32x4 *>(p), *reinterpret_cast<const u32x4 *>(p + 16)};
      u32 o[3][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32 hi[2], mid[2], lo[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const u32 b = v[i >> 1][2 * (i & 1) + s];
          hi[s] = b & 0xFFFF0000u;
          const float r = u32_as_f32(b) - u32_as_f32(hi[s]);   // of an infinity: NaN, as the row's outputs then are
          mid[s] = f32_as_u32(r) & 0xFFFF0000u;
          lo[s] = f32_as_u32(r - u32_as_f32(mid[s]));
        }
        o[0][i] = __builtin_amdgcn_perm(hi[1], hi[0], 0x07060302u);
        o[1][i] = __builtin_amdgcn_perm(mid[1], mid[0], 0x07060302u);
        o[2][i] = __builtin_amdgcn_perm(lo[1], lo[0], 0x07060302u);
      }
#pragma unroll
      for (int s = 0; s < 3; ++s) x[s] = as_frag(o[s][0], o[s][1], o[s][2], o[s][3]);
    }
  };

  f32x4 y[MR][TT];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int t = 0; t < TT; ++t) y[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const u32 one2 = 0x3F803F80u;   // (1, 1)
  const bf16x8 ones = as_frag(one2, one2, one2, one2);

  if (wave < a.chunks) {
    load_w(wave);
#pragma unroll
    for (int p = 0; p < kDeepX; ++p) load_x(wave, p);
  }
  for (int ch = wave; ch < a.chunks; ch += kWaves) {
    store_w();
    typename F::Side now[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) now[m] = side[m];
    if (ch + kWaves < a.chunks) load_w(ch + kWaves);
#pragma unroll
    for (int p = 0; p < 4; ++p) {   // 64 values
      if (8 * ch + 2 * p >= a.groups) break;
      store_x(p % kDeepX);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      load_x(ch, p + kDeepX);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int g = 2 * p + e;
        typename F::U u[MR];
#pragma unroll
        for (int m = 0; m < MR; ++m) F::unpack(u[m], own + m * 16 * F::kStride + c * F::kStride, now[m], g, q);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          bf16x8 x[NX];
          operand(t, e, x);
          f32x4 S = zero, da = zero;
          if constexpr (XT == kXQ8) {
            const u8 *mt = xl + (16 * t + 4 * q) * x_stride<XT>() + 64 + 8 * e;   // tokens 4 q + i
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 v = *reinterpret_cast<const float2 *>(mt + i * x_stride<XT>());
              da[i] = v.x;
              S[i] = v.y;
            }
          } else if constexpr (F::kSum) {   // the smallest parts first
#pragma unroll
            for (int s = NX - 1; s >= 0; --s) S = mfma(x[s], ones, S);
          }
          auto dot = [&](auto... w) __attribute__((always_inline)) {
            f32x4 v = zero;
#pragma unroll
            for (int s = NX - 1; s >= 0; --s) ((v = mfma(x[s], w, v)), ...);
            return v;
          };
#pragma unroll
          for (int m = 0; m < MR; ++m)
            F::apply(u[m], dot, S, [&](float d, float v, int i) __attribute__((always_inline)) {
              y[m][t][i] = __builtin_fmaf(XT == kXQ8 ? d * da[i] : d, v, y[m][t][i]);
            });
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }

  // ---- the waves' sums meet, in place of their own areas
  float *meet = reinterpret_cast<float *>(smem);
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) meet[((wave * MR + m) * TT + t) * 256 + 16 * (4 * q + i) + c] = y[m][t][i];
  __syncthreads();
  for (int o = tid; o < 256 * RT * TT; o += 64 * kWaves) {
    const int t = o / (16 * RT), rr = o % (16 * RT), row = row0 + rr, at = 16 * (t & 15) + (rr & 15);
    if (t0 + t >= a.tokens || row >= a.n) continue;
    float v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      auto sum = [&](int k) { return meet[((k * MR + m * RT + (rr >> 4)) * TT + (t >> 4)) * 256 + at]; };
      v[m] = sum(0);
#pragma unroll
      for (int k = 1; k < kWaves; ++k) v[m] += sum(k);
    }
    const int64_t out = (int64_t)(t0 + t) * a.n + row;
    if constexpr (NM == 2) epi_store2(ep, out, row, v[0], v[NM - 1]);
    else epi_store(ep, out, row, v[0]);
  }
}

template <class F, int XT, int RT, int NM, int TT>
int launch_t(const MArgs &a, const Epi &ep, hipStream_t s) {
  constexpr int kOwn = own_bytes<F, XT, RT, NM, TT>(), kMeet = RT * NM * TT * 1024;
  constexpr int kLds = kWaves * (kOwn > kMeet ? kOwn : kMeet);
  static_assert(kLds <= 160 * 1024, "LDS of a workgroup");
  const void *fn = reinterpret_cast<const void *>(&mv_mfma_kernel<F, XT, RT, NM, TT>);
  static std::atomic<unsigned> raised{0};
  if (int st = raise_dyn_lds(fn, kLds, raised)) return st;
  const dim3 grid((unsigned)(8 * ((a.tokens + 16 * TT - 1) / (16 * TT))), (unsigned)((a.n + 128 * RT - 1) / (128 * RT)));
  mv_mfma_kernel<F, XT, RT, NM, TT><<<grid, 64 * kWaves, kLds, s>>>(a, ep);
  return launch_status();
}
template <class F, int XT, int NM>
int launch(const MArgs &a, const Epi &ep, hipStream_t s) {
  // Two row tiles of one matrix share a wave's activations where that leaves two workgroups a CU, or where an XCD's 32 CUs
  // take them in one round and single tiles in more (f32 and Q8_1 rows, whose operands are made from the loaded values: f32
  // rows, five tokens, Q4_0 6144 x 2048 8.8 -> 7.4 us, 8192 x 8192 24.9 -> 21.0, Q6_K 40.3 -> 32.9; Q8_1 33 tokens Q4_0
  // 2720 x 8192 32.1 -> 21.7; bf16 rows 5.7 and 5.6, 13.1 and 13.5, 20.7 and 22.5). Two token tiles share its unpacked
  // weights past 16 tokens.
  constexpr int kMost = NM == 2 ? 1 : 2, TT = XT == kXF32 ? 1 : 2;
  const bool wide = a.tokens > 16;
  const int tiles = wide ? (a.tokens + 16 * TT - 1) / (16 * TT) : 1;
  auto round = [&](int rows) { return ((a.n + rows - 1) / rows + 7) / 8 * tiles; };   // workgroups of an XCD
  const bool one_round = XT != kXBF16 && round(16) > 32 && round(32) <= 32;
  if (one_round || (int64_t)((a.n + 31) / 32) * tiles >= 512)
    return wide ? launch_t<F, XT, kMost, NM, TT>(a, ep, s) : launch_t<F, XT, kMost, NM, 1>(a, ep, s);
  return wide ? launch_t<F, XT, 1, NM, TT>(a, ep, s) : launch_t<F, XT, 1, NM, 1>(a, ep, s);
}
template <class F, int NM>
int launch_x(int x_dtype, const MArgs &a, const Epi &ep, hipStream_t s) {
  if (x_dtype == QMM_F32) return launch<F, kXF32, NM>(a, ep, s);
  if (x_dtype == QMM_BF16) return launch<F, kXBF16, NM>(a, ep, s);
  if constexpr (std::is_same_v<F, FQ4K> || std::is_same_v<F, FMX>) return QMM_ERR_FORMAT;   // Q8_1: not taken here
  else return launch<F, kXQ8, NM>(a, ep, s);
}
template <int NM>
int launch_f(int fmt, int x_dtype, const MArgs &a, const Epi &ep, hipStream_t s) {
  switch (fmt) {
    case QMM_Q4_0: return launch_x<FQ40, NM>(x_dtype, a, ep, s);
    case QMM_Q4_K: return launch_x<FQ4K, NM>(x_dtype, a, ep, s);
    case QMM_Q6_K: return launch_x<FQ6K, NM>(x_dtype, a, ep, s);
    case QMM_MXFP4: return launch_x<FMX, NM>(x_dtype, a, ep, s);
    default: return launch_x<FMXS, NM>(x_dtype, a, ep, s);
  }
}

}  // namespace

// Whether qmm_mv_mfma takes a call (the matvec kernels take the others). us at 12288 x 4096 and 4096 x 12288, here against the
// matvec kernels: Q6_K bf16 rows 17 and 18 / 25 and 28 at one token; two tokens: Q4_0 f32 25, 27 / 30, 23, bf16 12, 12 / 14, 18,
// Q4_K f32 22, 24 / 29, 23, bf16 (K not the fast kernel's 4096 or 8192) 12 / 17, MXFP4 f32 21, 24 / 21, 23; split planes bf16
// 12, 13 / 10, 11 at two and 12, 13 / 17, 15 at three; Q8_1 rows: Q4_0 15, 15 / 16, 15 at four, Q6_K 21, 23 / 36, 38 at eight
// (20, 23 / 21, 21 at four), split planes 16, 17 / 20, 18 at three. At 63 tokens: Q6_K f32 105 / 1442, bf16 44 / 863, Q8_1
// 56 / 227.
bool qmm_mv_mfma_fits(int fmt, int x_dtype, int64_t k, int64_t n, int64_t tokens) {
  if (fmt != QMM_Q4_0 && fmt != QMM_Q4_K && fmt != QMM_Q6_K && fmt != QMM_MXFP4 && fmt != QMM_MXFP4S) return false;
  if (k % 64 || (x_dtype == QMM_Q8 && (fmt == QMM_Q4_K || fmt == QMM_MXFP4))) return false;
  if (n > (1 << 22) || tokens > (1 << 20) || k > (1 << 20)) return false;   // 32-bit rows, tokens and chunks; the grid
  if (n * row_bytes(fmt, k) >= (1ll << 32)) return false;                      // byte offsets of weight rows
  if (x_dtype == QMM_Q8) return tokens >= (fmt == QMM_MXFP4S ? 3 : fmt == QMM_Q4_0 ? 4 : 5);
  if (fmt == QMM_Q6_K && x_dtype == QMM_BF16) return tokens >= 1;
  if (fmt == QMM_MXFP4S || (fmt == QMM_Q4_K && x_dtype == QMM_BF16 && (k == 4096 || k == 8192))) return tokens >= 3;
  return tokens >= 2;
}

int qmm_mv_mfma(int fmt, int x_dtype, int64_t k, int64_t n, int64_t tokens, const void *x, const void *w, const void *ws,
                const void *w2, const void *ws2, hipStream_t s, const Epi &ep) {
  if (!x || !w || (fmt == QMM_MXFP4S && (!ws || (w2 && !ws2)))) return QMM_ERR_NULL;
  if (n <= 0 || row_bytes(fmt, k) == 0) return QMM_ERR_SHAPE;
  const size_t wal = fmt == QMM_Q4_K || fmt == QMM_MXFP4S ? 16 : fmt == QMM_MXFP4 ? 1 : 4;   // as the matvec kernels take them
  if (!aligned(x, 16) || !aligned(w, wal) || !aligned(w2, wal)) return QMM_ERR_ALIGN;
  if (fmt == QMM_MXFP4S && (!aligned(ws, 2) || !aligned(ws2, 2))) return QMM_ERR_ALIGN;
  MArgs a{};
  a.n = (int)n; a.tokens = (int)tokens; a.k = k;
  a.groups = (int)(k / 32); a.chunks = (a.groups + 7) / 8;
  a.rb = row_bytes(fmt, k); a.sb = fmt == QMM_MXFP4S ? k / 32 : 0;
  a.x = x;
  a.meta = x_dtype == QMM_Q8 ? reinterpret_cast<const float *>(static_cast<const u8 *>(x) + tokens * k) : nullptr;
  a.w = static_cast<const u8 *>(w); a.w2 = static_cast<const u8 *>(w2);
  a.ws = static_cast<const u8 *>(ws ? ws : w); a.ws2 = static_cast<const u8 *>(ws2 ? ws2 : w2);
  return w2 ? launch_f<2>(fmt, x_dtype, a, ep, s) : launch_f<1>(fmt, x_dtype, a, ep, s);
}

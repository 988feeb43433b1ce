// Device pieces shared by the block-scaled fp8 kernels: block amax and
// codes, the tile search over groups, fragments of 128 codes.
#pragma once
#include <type_traits>

#include "smoe_common.hpp"
#include "smoe_fp8_blocks.hpp"

namespace smoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr float kE4m3Max = 448.0f;

// Constant memory that every lane of a wave reads at one address (s_load)
typedef const float __attribute__((address_space(4)))* uniform_f32;
__device__ __forceinline__ uniform_f32 as_uniform(const float* p) {
  return (uniform_f32)(reinterpret_cast<uintptr_t>(p));
}

// amax over |v| as bit patterns: the largest unsigned word is the largest
// magnitude, NaN above infinity above the rest, so a block with a NaN has a NaN
// scale.
__device__ __forceinline__ uint32_t amax_bits(uint32_t m, float v) {
  return max(m, __float_as_uint(v) & 0x7FFFFFFFu);
}
// ... over the 16 lanes of a DPP row
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(dpp_i<kDppXor1>(static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(dpp_i<kDppXor2>(static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(dpp_i<kDppHalfMirror>(static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(dpp_i<kDppMirror>(static_cast<int>(v))));
  return v;
}
// ... over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ uint32_t quarters_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
  return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)));
}

// scale = max(amax / 448, 1e-12), the quotient an IEEE one; a NaN stays
__device__ __forceinline__ float block_scale(uint32_t amax) {
  const float s = __fdiv_rn(__uint_as_float(amax), kE4m3Max);
  return s < 1e-12f ? 1e-12f : s;
}

// Quotients by one divisor, as good as correctly rounded ones: r the correctly
// rounded reciprocal, q0 = x r, e = x - q0 s, q0 + e r (P. Markstein, IBM J.
// Res. Dev. 34, 1990).  His theorem asks for a q0 within a unit, which this one
// exceeds by half a unit at times; but the sum is within 12 * 2^-49 (of x / s
// brought to 1 .. 2) before it is rounded, and the few pairs where that could
// move a quotient over the middle between two codes are tried one by one in
// tests/test_fp8_blocks_quotient.py: the code is always that of the rounded
// x / s.  Below 2^-10, where e could underflow, the code is 0 either way.  4
// operations for an IEEE division's 12.  s = infinity: 0 for finite x, NaN for
// infinite x.
struct Divisor {
  float r, s;
};
__device__ __forceinline__ Divisor divisor(float s) {
  return {__fdiv_rn(1.0f, s), s == INFINITY ? 0.0f : s};
}
__device__ __forceinline__ float quotient(float x, Divisor d) {
  const float q = mul_rn(x, d.r);
  return copysignf(fmaf(fmaf(-q, d.s, x), d.r, q), x);  // x = -0 keeps its sign
}

// Four e4m3 codes of values that a block's scale has brought to +-448 (plus
// half a unit in the last place of the quotient, which rounds to 448): round
// to nearest even, NaN to NaN.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}

// Eight elements from column c of a row that ends at cols, 0 past the end;
// one 16- or 32-byte load where the row's start and c allow it (vec).
template <int XDT>
__device__ __forceinline__ void load_cols8(const void* row, int c, int cols, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    if constexpr (XDT == SMOE_F32) {
      const f32x4* p = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(row) + c);
      const f32x4 a = p[0], b = p[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = a[j];
        v[4 + j] = b[j];
      }
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(row) + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint16_t h = static_cast<uint16_t>(a[j >> 1] >> (16 * (j & 1)));
        v[j] = XDT == SMOE_BF16 ? bf2f(h) : static_cast<float>(__builtin_bit_cast(_Float16, h));
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float x = 0.f;
    if (c + j < cols) {
      if constexpr (XDT == SMOE_F32) x = reinterpret_cast<const float*>(row)[c + j];
      else if constexpr (XDT == SMOE_BF16) x = bf2f(reinterpret_cast<const uint16_t*>(row)[c + j]);
      else x = static_cast<float>(reinterpret_cast<const _Float16*>(row)[c + j]);
    }
    v[j] = x;
  }
}

template <int XDT>
constexpr int elt_bytes() { return XDT == SMOE_F32 ? 4 : 2; }

__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = amax_bits(m, v[j]);
  return m;
}

__device__ __forceinline__ u32x2 codes8(const float (&v)[8], float sc) {
  const Divisor d = divisor(sc);
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = quotient(v[j], d);
  return u32x2{pack_e4m3(q[0], q[1], q[2], q[3]), pack_e4m3(q[4], q[5], q[6], q[7])};
}

// Block b (row b / nblk, column block b % nblk) of 1 x 128 blocks by the
// sixteen lanes of a DPP row, eight elements each.  Every lane of the wave
// calls it (blocks past `total` compute on the last one and store nothing).
template <int XDT>
__device__ __forceinline__ void quant_row_block(const BlockQuant& q, int nblk, int64_t total, int64_t b, int l16) {
  const uint32_t bc = static_cast<uint32_t>(b < total ? b : total - 1);  // total <= 2^28
  const int64_t row = bc / static_cast<uint32_t>(nblk);  // a 64-bit division is longer than the rest
  const int kb = static_cast<int>(bc - static_cast<uint32_t>(row) * nblk);
  const int c = kb * kFp8Block + 8 * l16;
  const char* rp = reinterpret_cast<const char*>(q.x) + row * q.ldx * elt_bytes<XDT>();
  const bool vec = (reinterpret_cast<uintptr_t>(q.x) | static_cast<uintptr_t>(q.ldx * elt_bytes<XDT>())) % 16 == 0;
  float v[8];
  load_cols8<XDT>(rp, c, q.cols, vec, v);
  const float sc = block_scale(row16_max(amax8(v)));
  if (b >= total) return;
  if (l16 == 0) q.scale[row * q.s_row + kb * q.s_col] = sc;
  if (c < q.ld_out) *reinterpret_cast<u32x2*>(q.codes + row * q.ld_out + c) = codes8(v, sc);
}

// Four output channels n .. n + 3 of row r (those below N_out)
template <int ODT, typename P>
__device__ __forceinline__ void store4(const P& p, int64_t r, int n, const float (&o)[4]) {
  const int64_t at = r * p.ldo + n;
  if constexpr (ODT == SMOE_F32) {
    float* po = reinterpret_cast<float*>(p.out) + at;
    if (n + 3 < p.N_out && (reinterpret_cast<uintptr_t>(po) & 15) == 0) {
      *reinterpret_cast<f32x4*>(po) = f32x4{o[0], o[1], o[2], o[3]};
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (n + v < p.N_out) po[v] = o[v];
    }
  } else {
    uint16_t* po = reinterpret_cast<uint16_t*>(p.out) + at;
    if (n + 3 < p.N_out && (reinterpret_cast<uintptr_t>(po) & 7) == 0) {
      *reinterpret_cast<u32x2*>(po) = u32x2{pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3])};
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (n + v < p.N_out) po[v] = f2bf(o[v]);
    }
  }
}

// Rows of the 64 groups from b on: first, end and BM-row tiles of group
// b + lane; off: the G + 1 offsets, in global memory or LDS.
template <typename O>
__device__ __forceinline__ void groups64(O off, int G, int BM, int b, int& lo, int& hi, int& t) {
  const int i = b + static_cast<int>(threadIdx.x & 63);
  const int ic = i < G ? i : G - 1;
  lo = off[ic];
  hi = off[ic + 1];
  t = i < G ? (hi - lo + BM - 1) / BM : 0;
}

// Tiles of BM rows x BN channels in all.  P: BlockGemm or MxGemm.
template <int BM, int BN, typename P, typename O>
__device__ __forceinline__ int count_tiles(const P& p, O off) {
  int tiles = 0;
  if (p.G == 0) {
    tiles = (p.single_rows + BM - 1) / BM;
  } else {
    for (int b = 0; b < p.G; b += 64) {
      int lo, hi, t;
      groups64(off, p.G, BM, b, lo, hi, t);
      tiles += __builtin_amdgcn_readlane(wave_incl_scan(t), 63);
    }
  }
  return tiles * ((p.N_out + BN - 1) / BN);
}

// Tile bid of T, for a workgroup of id bid modulo 8: group by group; within a
// group SUPER row tiles at a time, over them strip by strip with the strip's row
// tiles next to each other, so that the rows in use stay in an L2 while the
// strips' weights pass.  Workgroup ids are dealt to the 8 XCDs round robin and
// each XCD takes one contiguous part of the order.  SUPER: an XCD holds 32 tiles
// of 256 rows (64 of 128) at a time (32768 routed rows, 1024 -> 2816 SwiGLU, 256
// rows a tile: 2 row tiles 250 us, 4 252, 8 260, 16 256; 1024 -> 5632: 119, 117,
// 118, 121).
template <int BM, int BN, typename P, typename O>
__device__ __forceinline__ void tile_at(const P& p, O off, int T, int bid, int& g, int& m0, int& mrows, int& n0) {
  const int strips = (p.N_out + BN - 1) / BN;
  const int x = bid & 7, base = T >> 3, rem = T & 7;
  const int logical = x * base + min(x, rem) + (bid >> 3);
  int lo = 0, hi = p.single_rows, in = logical;
  g = 0;
  if (p.G > 0) {
    int acc = 0;
    for (int b = 0; b < p.G; b += 64) {
      int l, h, t;
      groups64(off, p.G, BM, b, l, h, t);
      const int incl = wave_incl_scan(t) * strips + acc;
      const uint64_t m = __ballot(logical < incl);
      if (m) {
        const int f = __builtin_ctzll(m);
        g = b + f;
        in = logical - __builtin_amdgcn_readlane(incl - t * strips, f);
        lo = __builtin_amdgcn_readlane(l, f);
        hi = __builtin_amdgcn_readlane(h, f);
        break;
      }
      acc = __builtin_amdgcn_readlane(incl, 63);
    }
  }
  const int tm = (hi - lo + BM - 1) / BM;
  constexpr int SUPER = BM == 256 ? 4 : 8;
  const int super = in / (SUPER * strips), rest = in - super * SUPER * strips;
  const int sr = min(SUPER, tm - super * SUPER);  // row tiles of this part
  const int strip = sr == SUPER ? rest / SUPER : rest / sr;  // uniform: a shift but for the last part
  m0 = lo + (super * SUPER + rest - strip * sr) * BM;
  mrows = min(BM, hi - m0);
  n0 = strip * BN;
}

// The tile of workgroup bid, if there is one
template <int BM, int BN, typename P>
__device__ __forceinline__ bool block_tile(const P& p, int bid, int& g, int& m0, int& mrows, int& n0) {
  const int T = count_tiles<BM, BN>(p, p.grp_off);
  if (bid >= T) return false;
  tile_at<BM, BN>(p, p.grp_off, T, bid, g, m0, mrows, n0);
  return true;
}

// keeps the first `left` bytes
__device__ __forceinline__ u32x4 cut16(u32x4 v, int left) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int n = left - 4 * d;
    v[d] &= n >= 4 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
  }
  return v;
}

// The codes past the end of K in a stage of `rows` 128-byte rows (swizzled as
// sw_chunk says), set to code 0: what lies behind a row's end may decode to
// NaN, in either operand.  left: bytes of the stage that belong to K.
__device__ __forceinline__ void cut_stage(uint8_t* stage, int rows, int left, int tid, int threads) {
  const int c0 = left >> 4, per = 8 - c0;  // the first chunk that is not whole
  for (int e = tid; e < rows * per; e += threads) {
    const int r = e / per, c = c0 + e % per;
    u32x4* at = reinterpret_cast<u32x4*>(stage + r * 128 + (sw_chunk<8>(r, c) << 4));
    u32x4 v = c == c0 ? *at : u32x4{0u, 0u, 0u, 0u};
    if (c == c0) v = cut16(v, left & 15);
    *at = v;
  }
}

// 32 codes of a lane as four bf16 MFMA operands (every e4m3 value is a bf16)
__device__ __forceinline__ void widen_frag(i32x8 f, bf16x8 (&o)[4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const u32x2 a = fp8x4_to_bf16x4(static_cast<uint32_t>(f[2 * p]));
    const u32x2 b = fp8x4_to_bf16x4(static_cast<uint32_t>(f[2 * p + 1]));
    o[p] = __builtin_bit_cast(bf16x8, u32x4{a.x, a.y, b.x, b.y});
  }
}

template <typename F>
inline int by_xdt(int dt, F&& f) {
  switch (dt) {
    case SMOE_F32: return f(std::integral_constant<int, SMOE_F32>{});
    case SMOE_BF16: return f(std::integral_constant<int, SMOE_BF16>{});
    case SMOE_F16: return f(std::integral_constant<int, SMOE_F16>{});
    default: return SMOE_EUNSUPPORTED;
  }
}


}  // namespace smoe

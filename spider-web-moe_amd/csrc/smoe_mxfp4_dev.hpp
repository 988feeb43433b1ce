// Device pieces shared by the microscaled 4-bit kernels: a block's power of
// two, codes, fragments of 32 codes.
#pragma once
#include "smoe_fp8_blocks_dev.hpp"
#include "smoe_mxfp4.hpp"

namespace smoe {

// Biased exponent of a block's power of two from its largest magnitude (bit
// pattern): that of the magnitude less 2, the exponent of e2m1's largest values
// (magnitudes of 7 and more units then round to 6), at least 0 (2^-127); 255
// (NaN) for an infinity or a NaN.
__device__ __forceinline__ int mx_scale_byte(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23);
  return e == 255 ? 255 : max(e - 2, 0);
}
// The power of two itself (byte < 255)
__device__ __forceinline__ float mx_scale_value(int byte) {
  return __uint_as_float(byte > 0 ? static_cast<uint32_t>(byte) << 23 : 0x00400000u);
}

// Four codes in 16 bits of values and their block's power of two: to nearest
// even, past 6 to 6 (v_cvt_scalef32_pk_fp4_f32; 2^22 bit patterns, every tie and
// both ends of the exponents compared with the definition).  Blocks without a
// power of two hold code 0.
__device__ __forceinline__ uint32_t mx_codes4(float a, float b, float c, float d, int byte) {
  const float s = mx_scale_value(byte);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c, d, s, 1);
  return byte == 255 ? 0u : w;
}
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], int byte) {
  const float s = mx_scale_value(byte);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  return byte == 255 ? 0u : w;
}

// amax over the four lanes of a quad
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(dpp_i<kDppXor1>(static_cast<int>(v))));
  return max(v, static_cast<uint32_t>(dpp_i<kDppXor2>(static_cast<int>(v))));
}

// 128 columns (four blocks) by the sixteen lanes of a DPP row, eight elements
// each: this lane's codes, and in the row's first lane the four scales.  Every
// lane of the wave calls it.
__device__ __forceinline__ uint32_t mx_quant128(const float (&v)[8], uint32_t& scales) {
  const int byte = mx_scale_byte(quad_max(amax8(v)));
  scales = static_cast<uint32_t>(byte) | static_cast<uint32_t>(dpp_i<0x104>(byte)) << 8 |  // row_shl 4, 8, 12
           static_cast<uint32_t>(dpp_i<0x108>(byte)) << 16 | static_cast<uint32_t>(dpp_i<0x10C>(byte)) << 24;
  return mx_codes8(v, byte);
}

// Piece b (row b / npc, columns 128 (b % npc) ..) of x by the sixteen lanes of
// a DPP row.  Every lane of the wave calls it (pieces past `total` compute on
// the last one and store nothing).
template <int XDT>
__device__ __forceinline__ void mx_quant_piece(const MxQuant& q, int npc, int64_t total, int64_t b, int l16) {
  const uint32_t bc = static_cast<uint32_t>(b < total ? b : total - 1);  // total <= 2^28
  const int64_t row = bc / static_cast<uint32_t>(npc);
  const int kb = static_cast<int>(bc - static_cast<uint32_t>(row) * npc);
  const int c = kb * 128 + 8 * l16;
  const char* rp = reinterpret_cast<const char*>(q.x) + row * q.ldx * elt_bytes<XDT>();
  const bool vec = (reinterpret_cast<uintptr_t>(q.x) | static_cast<uintptr_t>(q.ldx * elt_bytes<XDT>())) % 16 == 0;
  float v[8];
  load_cols8<XDT>(rp, c, q.cols, vec, v);
  uint32_t scales;
  const uint32_t codes = mx_quant128(v, scales);
  if (b >= total) return;
  if (l16 == 0) *reinterpret_cast<uint32_t*>(q.scale + row * q.s_row + kb * q.s_word) = scales;
  if (c / 2 < q.ld_codes) *reinterpret_cast<uint32_t*>(q.codes + row * q.ld_codes + c / 2) = codes;
}

// Word i of the planes, rows fastest
inline __host__ __device__ int64_t mx_plane_words(const MxPlanes& p) {
  return static_cast<int64_t>(p.groups) * p.rows * ((p.blocks + 3) / 4);
}
__device__ __forceinline__ void mx_plane_word(const MxPlanes& p, uint32_t i) {
  const uint32_t rest = i / static_cast<uint32_t>(p.rows), r = i - rest * p.rows, nd = (p.blocks + 3) / 4;
  const uint32_t g = rest / nd, s = rest - g * nd;
  uint32_t w = *reinterpret_cast<const uint32_t*>(p.src + (static_cast<int64_t>(g) * p.rows + r) * p.ld + 4 * s);
  const int left = p.blocks - 4 * static_cast<int>(s);
  if (left < 4) w = (w & ((1u << 8 * left) - 1u)) | (0x7F7F7F7Fu << 8 * left);
  p.dst[static_cast<int64_t>(rest) * (mx_plane_pitch(p.rows) / 4) + r] = w;
}

// The matrix instruction on 128 k: lane l holds 32 codes of row l % 16 of each
// operand and their scale in byte `S` of its scale register.  Products and sums
// are those of the values, rounded as f32 sums are: a block's 32 products, which
// are multiples of a quarter up to 36, add exactly, and an instruction's sum
// with its accumulator was off by at most 3 * 2^-24 of the magnitudes (measured,
// scales of 2^-27 to 2^23 in one sum).  No products are cut, as they are between
// e4m3 operands: one form serves bf16 and f32 outputs.
template <int S>
__device__ __forceinline__ f32x4 mx_mfma(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x4 acc) {
  const i32x8 a = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w), 0, 0, 0, 0};
  const i32x8 b = {static_cast<int>(x.x), static_cast<int>(x.y), static_cast<int>(x.z), static_cast<int>(x.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, S, static_cast<int>(ws), S, static_cast<int>(xs));
}

// erfc(a) = exp(-a^2) t P(t), t = 1 / (1 + 0.3 a), P of degree 8 fitted to
// exp(a^2) erfc(a) / t on 0 <= a <= 13 by reweighted least squares: within 3e-8
// of it, so that in f32 the GELU below is within 4e-6 of its value also where
// that is small (1 + erf loses 2^-25 of one there, and a block of small
// activations is quantized by its own largest).
__device__ __forceinline__ float gelu_tail(float x) {
  const float a = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.0f));
  float y = fmaf(-0.12786658f, t, 0.47773516f);
  y = fmaf(y, t, -0.49654815f);
  y = fmaf(y, t, 0.5302056f);
  y = fmaf(y, t, -0.08285845f);
  y = fmaf(y, t, 0.21002072f);
  y = fmaf(y, t, 0.14956778f);
  y = fmaf(y, t, 0.17054613f);
  y = fmaf(y, t, 0.1691978f);
  const float h = 0.5f * x * (t * y * __builtin_amdgcn_exp2f(x * x * -0.72134752f));  // log2(e) / 2
  return x < 0.f ? h : (x > 13.f ? x : x - h);
}

}  // namespace smoe

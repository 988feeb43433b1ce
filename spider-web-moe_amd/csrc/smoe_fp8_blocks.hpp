// Block-scaled fp8 (e4m3 codes, one f32 scale for each 1 x 128 block of
// activations and each 128 x 128 block of weights): arguments of the
// quantizer and of the products on such operands, shared by their
// translation unit and the C entry points.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smoe.h"

namespace smoe {

constexpr int kFp8Block = 128;
inline int fp8_blocks_of(int n) { return n / kFp8Block + (n % kFp8Block != 0); }  // any n >= 0

// x [groups * rows, cols] (rows ldx elements apart) -> codes (rows ld_out
// bytes apart, code 0 past cols) and the scale of block (row block r of
// group g, column block c) at scale[(g * row_blocks + r) * s_row + c * s_col].
struct BlockQuant {
  const void* x = nullptr;
  int x_dtype = SMOE_BF16;
  int64_t ldx = 0;
  int groups = 1, rows = 0, cols = 0, block_rows = 1;
  uint8_t* codes = nullptr;
  int64_t ld_out = 0;
  float* scale = nullptr;
  int64_t s_row = 0, s_col = 0;
};
int launch_quantize_fp8_blocks(const BlockQuant& q, hipStream_t s);

enum BlockEpi : int {
  BLK_LINEAR = 0,  // out = acc + bias                        (f32 / bf16)
  BLK_GELU = 1,    // out = gelu_erf(acc + bias)              (f32 / bf16)
  BLK_UP_GELU = 2,    // codes and scales of gelu_erf(acc + bias), per row and 128 channels
  BLK_UP_SWIGLU = 3,  // codes and scales of silu(gate) * (up + bias)
  BLK_DOWN = 4,    // out f32 = (acc + bias) * row_scale
};

// C[row, n] = sum over 128-wide blocks b of K of
//   xs[a_row, b] * ws[n / 128, b] * (codes of X[a_row, b] . codes of W_g[n, b])
struct BlockGemm {
  int epi = BLK_LINEAR;
  const uint8_t* X = nullptr;  // codes, rows ldx bytes apart
  int64_t ldx = 0;
  const float* xs = nullptr;   // scale of (row r, block b): xs[r * xs_row + b * xs_col]
  int64_t xs_row = 0, xs_col = 0;
  const int32_t* a_rows = nullptr;  // plan row -> X row; nullptr = identity
  // instead of X / xs (linear_quantizes_inside): x [single_rows, K] itself,
  // rows ld_float elements apart, quantized by the product's workgroups
  const void* x_float = nullptr;
  int x_dtype = SMOE_BF16;
  int64_t ld_float = 0;
  const uint8_t* W = nullptr;  // codes [G, N_out (SwiGLU: gate rows, then up rows), K]
  int64_t w_gstride = 0, ldw = 0;
  const float* ws = nullptr;   // [G, row blocks (SwiGLU: gate's, then up's), blocks of K]
  int64_t ws_gstride = 0;
  int K = 0, N_out = 0;        // N_out: output channels
  const int32_t* grp_off = nullptr;  // [G + 1]; G == 0: one group of single_rows rows
  int G = 0, single_rows = 0;
  int max_rows = 0;            // worst-case total rows (grid sizing)
  const float* bias = nullptr;
  int64_t bias_gstride = 0;
  const float* row_scale = nullptr;  // BLK_DOWN
  void* out = nullptr;
  int out_dtype = SMOE_F32;
  int64_t ldo = 0;             // elements (codes: bytes)
  bool wide = false;           // BLK_UP_*, BLK_DOWN: products summed in f32 (BLK_LINEAR, BLK_GELU: with f32 outputs)
  float* out_scale = nullptr;  // BLK_UP_*: scale of (row, block): out_scale[block * os_col + row]
  int64_t os_col = 0;
};
int launch_gemm_fp8_blocks(const BlockGemm& g, hipStream_t s);
// the dense products of a few rows (smoe_fp8_blocks_few.hip)
bool gemm_blocks_few_fits(const BlockGemm& g);
int launch_gemm_blocks_few(const BlockGemm& g, hipStream_t s);
// whether a linear product of N rows takes x_float
bool linear_quantizes_inside(int N, int K);

// A small step's dispatch plan (smoe_dispatch_plan's: offsets [E + 1], rows,
// row weights, tokrow [N, K]) and the quantized messages in one launch.
struct PrepArgs {
  const int32_t* idx = nullptr;
  const float* w = nullptr;
  int N = 0, K = 0, E = 0;
  int32_t *off = nullptr, *rows = nullptr, *tokrow = nullptr;
  float* roww = nullptr;
};
bool prep_fits(int N, int K, int E);
int launch_prep(const PrepArgs& a, const BlockQuant& q, hipStream_t s);

// The expert step of a few tokens (N * K <= 16) in two launches.
struct TokensArgs {
  const void* msg = nullptr;  // [N, H] f32 / bf16
  int msg_dtype = SMOE_BF16;
  const int32_t* idx = nullptr;
  const float* w = nullptr;
  int N = 0, K = 0, E = 0, H = 0, U = 0;
  int act_fn = SMOE_ACT_GELU;
  const uint8_t *w_up = nullptr, *w_down = nullptr;
  const float *s_up = nullptr, *s_down = nullptr, *b_up = nullptr, *b_down = nullptr;
  float* act = nullptr;  // f32 [N * K, U], 16-byte aligned
  void* out = nullptr;   // [N, H]
  int out_dtype = SMOE_BF16;
};
bool tokens_fit(int N, int K, int H, int U);
int launch_tokens(const TokensArgs& a, hipStream_t s);

}  // namespace smoe

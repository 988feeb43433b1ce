// Microscaled 4-bit floating point: blocks of 32 values along a row as e2m1
// codes and one power of two.  Arguments of the quantizer and of the products
// on such operands, shared by their translation units and the C entry points.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smoe.h"
#include "smoe_fp8_blocks.hpp"

namespace smoe {

constexpr int kMxBlock = 32;
inline int64_t mx_blocks_of(int64_t n) { return n / kMxBlock + (n % kMxBlock != 0); }  // any n >= 0
inline int64_t mx_code_pitch(int64_t n) { return 16 * mx_blocks_of(n); }               // whole blocks
inline int64_t mx_scale_pitch(int64_t n) { return (mx_blocks_of(n) + 3) / 4 * 4; }     // whole words

// x [rows, cols] (rows ldx elements apart) -> codes two a byte, the even column
// in the low half (rows ld_codes bytes apart, code 0 past cols), and the blocks'
// powers of two as biased exponents, word by word (four blocks): word kb of row
// r at scale + r * s_row + kb * s_word.
struct MxQuant {
  const void* x = nullptr;
  int x_dtype = SMOE_BF16;
  int64_t ldx = 0;
  int64_t rows = 0;
  int cols = 0;
  uint8_t* codes = nullptr;
  int64_t ld_codes = 0;
  uint8_t* scale = nullptr;
  int64_t s_row = 0, s_word = 0;
};
// The large products read scales in planes: word s of every row of a group
// side by side (plane pitch: the rows rounded up to 4), so that 16-byte DMAs
// fetch a stage's: 4-byte ones, a word a row, take a cycle a lane.  The weights'
// come in rows: src [groups * rows, ld] -> dst words [groups, mx_scale_pitch / 4,
// pitch], 127 (1) for blocks past the end.
inline __host__ __device__ int64_t mx_plane_pitch(int64_t rows) { return (rows + 3) / 4 * 16; }  // bytes
struct MxPlanes {
  const uint8_t* src = nullptr;
  int64_t ld = 0;
  int groups = 0, rows = 0;  // groups == 0: none
  int blocks = 0;            // of a row
  uint32_t* dst = nullptr;
};
constexpr int64_t kMxPlaneWords = 0xfffffe00ll;  // words that a call lays out in planes at most
int launch_quantize_mxfp4(const MxQuant& q, const MxPlanes (&planes)[2], hipStream_t s);
int launch_dequantize_mxfp4(const uint8_t* codes, int64_t ld_codes, const uint8_t* scale, int64_t ld_scale,
                            int64_t rows, int cols, void* out, int out_dtype, hipStream_t s);

enum MxEpi : int {
  MX_LINEAR = 0,     // out = acc + bias                       (f32 / bf16)
  MX_GELU = 1,       // out = gelu_erf(acc + bias)             (f32 / bf16)
  MX_UP_GELU = 2,    // codes and scales of gelu_erf(acc + bias)
  MX_UP_SWIGLU = 3,  // codes and scales of silu(gate) * (up + bias)
  MX_DOWN = 4,       // out f32 = (acc + bias) * row_scale
};

// C[row, n] = sum over k of the values of X[a_row, k] and W_g[n, k]
struct MxGemm {
  int epi = MX_LINEAR;
  const uint8_t* X = nullptr;  // codes, rows ldx bytes apart (code 0 past K within a block)
  int64_t ldx = 0;
  // scales: in planes (ws_plane > 0: the large products) or in rows ld_.. bytes apart
  const uint8_t* xs = nullptr;
  int64_t xs_plane = 0, ld_xs = 0;
  const int32_t* a_rows = nullptr;  // plan row -> X row (MX_UP_*; the others: identity)
  int64_t x_rows = 0;               // MX_UP_*: rows of X
  // instead of X / xs (mx_linear_quantizes_inside): x [single_rows, K] itself,
  // rows ld_float elements apart, quantized by the product's workgroups
  const void* x_float = nullptr;
  int x_dtype = SMOE_BF16;
  int64_t ld_float = 0;
  const uint8_t* W = nullptr;  // codes [G, N_out (SwiGLU: gate rows, then up rows), ldw]
  int64_t w_gstride = 0, ldw = 0;
  const uint8_t* ws = nullptr;
  int64_t ws_gstride = 0, ws_plane = 0, ld_ws = 0;
  int K = 0, N_out = 0;              // N_out: output channels
  const int32_t* grp_off = nullptr;  // [G + 1]; G == 0: one group of single_rows rows
  int G = 0, single_rows = 0;
  int max_rows = 0;                  // worst-case total rows (grid sizing)
  const float* bias = nullptr;
  int64_t bias_gstride = 0;
  const float* row_scale = nullptr;  // MX_DOWN
  void* out = nullptr;
  int out_dtype = SMOE_F32;
  int64_t ldo = 0;               // elements (codes: bytes)
  uint8_t* out_scale = nullptr;  // MX_UP_*
  int64_t os_plane = 0, ld_os = 0;
  bool dry = false;  // says whether the launch would be refused, and launches nothing
};
int launch_gemm_mxfp4(const MxGemm& g, hipStream_t s);
int launch_gemm_mx_mid(const MxGemm& g, hipStream_t s);  // smoe_mxfp4_mid.hip
// the dense products of a few rows (smoe_mxfp4_few.hip)
bool gemm_mx_few_fits(const MxGemm& g);
int launch_gemm_mx_few(const MxGemm& g, hipStream_t s);
// grouped products of decode steps (smoe_mxfp4_few.hip)
bool gemm_mx_stream_fits(const MxGemm& g);
int launch_gemm_mx_stream(const MxGemm& g, hipStream_t s);
// Dense products of up to this many rows run on gemm_mx_few, whatever N_out is
constexpr int kMxFewRows = 24;
// whether a linear product of N rows takes x_float
bool mx_linear_quantizes_inside(int N, int K);
// whether a product runs on large tiles, with scales in planes (ws_plane > 0; the
// other kernels read rows of scales and refuse planes)
bool mx_large_linear(int N, int N_out);
bool mx_large_experts(int N, int K, int E);

// A small step's dispatch plan (prep_fits) and the quantized messages in one launch
int launch_prep_mx(const PrepArgs& a, const MxQuant& q, hipStream_t s);

// The expert step of a few tokens (N * K <= 16) in two launches.
struct MxTokensArgs {
  const void* msg = nullptr;  // [N, H] f32 / bf16
  int msg_dtype = SMOE_BF16;
  const int32_t* idx = nullptr;
  const float* w = nullptr;
  int N = 0, K = 0, E = 0, H = 0, U = 0;
  int act_fn = SMOE_ACT_GELU;
  const uint8_t *w_up = nullptr, *w_down = nullptr;  // codes, whole rows
  const uint8_t *s_up = nullptr, *s_down = nullptr;  // scales, mx_scale_pitch apart
  const float *b_up = nullptr, *b_down = nullptr;
  float* act = nullptr;  // f32 [N * K, U], 16-byte aligned
  void* out = nullptr;   // [N, H]
  int out_dtype = SMOE_BF16;
};
bool mx_tokens_fit(int N, int K, int H, int U);
int launch_mx_tokens(const MxTokensArgs& a, hipStream_t s);

}  // namespace smoe

// Microscaled 4-bit steps of a few rows: dense products and expert steps whose
// waves load the weights' fragments straight into registers, and the launch
// that makes a small step's plan and quantizes its messages.
#include "smoe_internal.hpp"
#include "smoe_mxfp4_dev.hpp"
#include "smoe_small_plan.hpp"

namespace smoe {

int device_cus();
namespace {

// A lane's part of 256 k of a row: blocks 2 q and 2 q + 1 (q = lane / 16; the
// four lanes of a row cover 128 contiguous bytes), one for each of two matrix
// instructions, and their scales side by side.
struct Piece {
  u32x4 lo, hi;
  uint32_t s;
};
// Piece b of a row of nb blocks; blocks past the end are the row's first one,
// at scale 1 (the other operand's codes are 0 there)
__device__ __forceinline__ Piece load_piece(const uint8_t* codes, const uint8_t* scale, int b, int q, int nb) {
  const int c = 8 * b + 2 * q;
  const bool l = c < nb, h = c + 1 < nb;
  Piece p;
  p.lo = *reinterpret_cast<const u32x4*>(codes + (l ? 16 * c : 0));
  p.hi = *reinterpret_cast<const u32x4*>(codes + (h ? 16 * c + 16 : 0));
  const uint32_t s = *reinterpret_cast<const uint16_t*>(scale + (l ? c : 0));  // rows are whole words
  p.s = (l ? s & 0xFFu : 127u) | (h ? s & 0xFF00u : 127u << 8);
  return p;
}
__device__ __forceinline__ Piece cut_piece(Piece p, int b, int q, int nb) {  // of X: code 0 past the end
  const u32x4 zero = {0u, 0u, 0u, 0u};
  if (8 * b + 2 * q >= nb) p.lo = zero;
  if (8 * b + 2 * q + 1 >= nb) p.hi = zero;
  return p;
}
__device__ __forceinline__ f32x4 product(const Piece& w, const Piece& x, f32x4 acc) {
  acc = mx_mfma<0>(w.lo, w.s, x.lo, x.s, acc);
  return mx_mfma<1>(w.hi, w.s, x.hi, x.s, acc);
}

// Rows quantized into LDS: 256 k of a row as 128 bytes, a row 16 bytes more than
// that (rows a multiple of 256 bytes apart would meet in one bank), then its
// scales, 8 bytes for 256 k.
struct XLds {
  uint8_t* base;
  int ks, pitch, rows;
  __device__ __forceinline__ XLds(uint8_t* b, int ks_, int rows_) : base(b), ks(ks_), pitch(ks_ * 128 + 16), rows(rows_) {}
  __device__ __forceinline__ uint8_t* codes(int r) const { return base + r * pitch; }
  __device__ __forceinline__ uint8_t* scale(int r) const { return base + rows * pitch + r * ks * 8; }
  __device__ __forceinline__ Piece load(int r, int b, int q) const {
    const uint8_t* c = codes(r) + 128 * b + 32 * q;
    return {*reinterpret_cast<const u32x4*>(c), *reinterpret_cast<const u32x4*>(c + 16),
            *reinterpret_cast<const uint16_t*>(scale(r) + 8 * b + 2 * q)};
  }
};
constexpr int xlds_row(int64_t k) { return static_cast<int>((k + 255) / 256) * 136 + 16; }  // bytes a row

// Row r of the `rows` rows, its columns 128 h .., by the sixteen lanes of a DPP
// row: every lane of a wave comes along, `live` or not.
template <int XDT>
__device__ __forceinline__ void quant_to_lds(const XLds& x, const void* row, int r, int h, int cols, bool vec, int l16, bool live) {
  float v[8];
  load_cols8<XDT>(row, 128 * h + 8 * l16, live ? cols : 0, vec, v);
  uint32_t scales;
  const uint32_t codes = mx_quant128(v, scales);
  if (!live) return;
  *reinterpret_cast<uint32_t*>(x.codes(r) + 64 * h + 4 * l16) = codes;
  if (l16 == 0) *reinterpret_cast<uint32_t*>(x.scale(r) + 4 * h) = scales;
}

// Dense products of 16 MT rows: 16 channels a workgroup, four waves taking
// every fourth 256 of K straight into registers, D of them at once; their sums
// are added through LDS in wave order.
//
// XQ: -1 X is codes; else its dtype (x_float), which the workgroup quantizes
// into LDS while its first weights are on their way: one launch for a few tokens.
// Latency bounds it: 1 x 2048 -> 1408 4.4 us, about an empty launch.
template <int EPI, int ODT, int MT, int XQ>
__global__ __launch_bounds__(256, 4) void k_mx_few(const MxGemm p) {
  constexpr int BM = 16 * MT, NW = 4, D = MT == 1 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) float red[NW * MT * 256];
  extern __shared__ __attribute__((aligned(16))) uint8_t xbuf[];  // XQ >= 0
  const int strips = (p.N_out + 15) / 16;
  const int m0 = static_cast<int>(blockIdx.x) / strips * BM, n0 = static_cast<int>(blockIdx.x) % strips * 16;
  const int mrows = min(BM, p.single_rows - m0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int nb = (p.K + kMxBlock - 1) / kMxBlock, KS = (nb + 7) / 8;
  const int64_t wr = min(n0 + l16, p.N_out - 1);
  const uint8_t *wrow = p.W + wr * p.ldw, *wsrow = p.ws + wr * p.ld_ws;
  const uint8_t *xrow[MT], *xsrow[MT];
  const XLds xl(xbuf, KS, mrows);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t r = XQ >= 0 ? 0 : m0 + min(16 * i + l16, mrows - 1);  // rows past the end: a valid one, never stored
    xrow[i] = p.X + r * p.ldx;
    xsrow[i] = p.xs + r * p.ld_xs;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool first = true;
  for (int b0 = wave; b0 < KS || (XQ >= 0 && first); b0 += D * NW) {
    Piece w[D], x[D][MT];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = min(b0 + d * NW, KS - 1);  // past the end: the last one again, not used
      w[d] = load_piece(wrow, wsrow, b, q, nb);
      if constexpr (XQ < 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i) x[d][i] = load_piece(xrow[i], xsrow[i], b, q, nb);
      }
    }
    if constexpr (XQ >= 0) {
      if (first) {
        const bool vec = (reinterpret_cast<uintptr_t>(p.x_float) | static_cast<uintptr_t>(p.ld_float * elt_bytes<XQ>())) % 16 == 0;
        const int total = mrows * 2 * KS;  // pieces of 128 columns
        for (int e0 = wave * 4; e0 < total; e0 += NW * 4) {  // uniform
          const int e = min(e0 + q, total - 1), r = e / (2 * KS);
          quant_to_lds<XQ>(xl, reinterpret_cast<const char*>(p.x_float) + static_cast<int64_t>(m0 + r) * p.ld_float * elt_bytes<XQ>(),
                           r, e - r * 2 * KS, p.K, vec, l16, e0 + q < total);
        }
        __syncthreads();
        first = false;
      }
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < MT; ++i) x[d][i] = xl.load(min(16 * i + l16, mrows - 1), min(b0 + d * NW, KS - 1), q);
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = b0 + d * NW;
      if (b >= KS) break;  // uniform
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (XQ < 0 && 8 * b + 8 > nb) x[d][i] = cut_piece(x[d][i], b, q, nb);
        acc[i] = product(w[d], x[d][i], acc[i]);
      }
    }
  }

  // lane: channels 4 q + v of row l16 of each 16 x 16 tile
#pragma unroll
  for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(red + (wave * MT + i) * 256 + lane * 4) = acc[i];
  __syncthreads();
  const int i = wave;  // a tile a wave
  const int r = 16 * i + l16, n = n0 + 4 * q;
  if (i >= MT || r >= mrows) return;
  f32x4 sum = *reinterpret_cast<const f32x4*>(red + i * 256 + lane * 4);
#pragma unroll
  for (int w = 1; w < NW; ++w) sum += *reinterpret_cast<const f32x4*>(red + (w * MT + i) * 256 + lane * 4);
  float o[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float y = sum[v] + (p.bias && n + v < p.N_out ? p.bias[n + v] : 0.f);
    o[v] = EPI == MX_GELU ? gelu_tail(y) : y;
  }
  store4<ODT>(p, m0 + r, n, o);
}

// -------------------------------------------------- decode-size experts ----
// Grouped products of decode steps, a few rows a group.  The weights' bytes bound
// them, and a workgroup of few rows has too little to do between two barriers of
// a staged pipeline: here a strip of a group's channels (32 for the up products,
// a block of activations; 16 for the down product) is a workgroup, its four waves
// take every fourth 256 of K, and weights and rows go straight into registers,
// D pieces at once, without a barrier; the waves' sums are added through LDS in
// wave order.  16 rows at a time: a group with more reads its strip again, from
// the L2.  32 tokens, 2 of 16 experts of 1024 x 2816 (SwiGLU, 49 MB of weights):
// 14.2 us the up product, 7.5 the down one.  At 64 tokens, whose up product now runs
// on staged tiles (11.2), the two took 14.4 and 7.8 here; with non-temporal weight
// loads 15.2 and 8.8; with blocks q and q + 4 a lane, so that a load covers whole
// 64-byte pieces, 17.2 and 8.2.
template <int EPI>
__global__ __launch_bounds__(256, 4) void k_mx_stream(const MxGemm p) {
  constexpr bool SWIGLU = EPI == MX_UP_SWIGLU, UP = EPI == MX_UP_GELU || SWIGLU;
  constexpr int NT = SWIGLU ? 4 : (UP ? 2 : 1), CH = UP ? 32 : 16, D = SWIGLU ? 1 : (UP ? 2 : 3), NW = 4;
  __shared__ __attribute__((aligned(16))) float red[NW * NT * 256];
  const int strips = p.N_out / CH;  // N_out % 32 == 0
  const int g = static_cast<int>(blockIdx.x) / strips, n0 = (static_cast<int>(blockIdx.x) - g * strips) * CH;
  const int lo = p.grp_off[g], hi = p.grp_off[g + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int nb = (p.K + kMxBlock - 1) / kMxBlock, KS = (nb + 7) / 8;
  const uint8_t *wrow[NT], *wsrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {  // SwiGLU: two tiles of gate rows, two of up rows
    const int64_t r = n0 + 16 * (t & 1) + l16 + (t >= 2 ? p.N_out : 0);
    wrow[t] = p.W + g * p.w_gstride + r * p.ldw;
    wsrow[t] = p.ws + g * p.ws_gstride + r * p.ld_ws;
  }
  for (int m0 = lo; m0 < hi; m0 += 16) {
    const int mrows = min(16, hi - m0);
    const int r = m0 + min(l16, mrows - 1);  // rows past the end: a valid one, never stored
    const int64_t xr = p.a_rows ? p.a_rows[r] : r;
    const uint8_t *xrow = p.X + xr * p.ldx, *xsrow = p.xs + xr * p.ld_xs;
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int b0 = wave; b0 < KS; b0 += D * NW) {
      Piece w[D][NT], x[D];
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int b = b0 + d * NW;
        if (b >= KS) break;  // uniform
#pragma unroll
        for (int t = 0; t < NT; ++t) w[d][t] = load_piece(wrow[t], wsrow[t], b, q, nb);
        x[d] = load_piece(xrow, xsrow, b, q, nb);
      }
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int b = b0 + d * NW;
        if (b >= KS) break;  // uniform
        if (8 * b + 8 > nb) x[d] = cut_piece(x[d], b, q, nb);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = product(w[d][t], x[d], acc[t]);
      }
    }
    if (m0 > lo) __syncthreads();  // the rows before are read
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(red + (wave * NT + t) * 256 + lane * 4) = acc[t];
    __syncthreads();
    if (wave) continue;
    f32x4 sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      sum[t] = *reinterpret_cast<const f32x4*>(red + t * 256 + lane * 4);
#pragma unroll
      for (int u = 1; u < NW; ++u) sum[t] += *reinterpret_cast<const f32x4*>(red + (u * NT + t) * 256 + lane * 4);
    }
    // lane: channels 4 q + v of each tile, of row l16
    const int64_t row = m0 + l16;
    const bool live = l16 < mrows;
    const float* bias = p.bias ? p.bias + g * p.bias_gstride + n0 + 4 * q : nullptr;
    if constexpr (UP) {
      float y[2][4], m = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float b = bias ? bias[16 * h + v] : 0.f;
          if constexpr (SWIGLU) y[h][v] = silu(sum[h][v]) * (sum[NT - 2 + h][v] + b);
          else y[h][v] = gelu_tail(sum[h][v] + b);
          m = __builtin_elementwise_maximum(m, fabsf(y[h][v]));  // a NaN stays
        }
      const int byte = mx_scale_byte(quarters_max(__float_as_uint(m) & 0x7FFFFFFFu));
      if (!live) continue;
      uint8_t* to = static_cast<uint8_t*>(p.out) + row * p.ldo + n0 / 2 + 2 * q;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint16_t*>(to + 8 * h) = static_cast<uint16_t>(mx_codes4(y[h][0], y[h][1], y[h][2], y[h][3], byte));
      if (q == 0) p.out_scale[row * p.ld_os + n0 / 32] = static_cast<uint8_t>(byte);
    } else {
      if (!live) continue;
      const float rs = p.row_scale[row];
      f32x4 o;
#pragma unroll
      for (int v = 0; v < 4; ++v) o[v] = (sum[0][v] + (bias ? bias[v] : 0.f)) * rs;
      *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + row * p.ldo + n0 + 4 * q) = o;
    }
  }
}

// ------------------------------------------------- a few tokens' experts ----
// At most kTokensMax (token, slot) entries: the whole expert step in two launches
// that keep the dispatch plan in registers and quantize their own operands.  Bound
// by the latency of the two: 1 token, 2 of 64 experts of 2048 x 1408 5.7 and 5.9 us
// (weights of 6 MB, 1.3 us of a copy's rate).

// Up product of one expert's rows and 16 channels (SwiGLU: of gate and up):
// four waves take every fourth 256 of K, the rows' messages are quantized into
// LDS under the first weights' loads; activations leave in f32 at their plan
// rows.
template <bool SWIGLU, int XDT>
__global__ __launch_bounds__(256, 4) void k_mx_tokens_up(const MxTokensArgs a) {
  constexpr int NT = SWIGLU ? 2 : 1, D = SWIGLU ? 2 : 4;
  __shared__ __attribute__((aligned(16))) float red[4 * NT * 256];
  __shared__ int s_tok[kTokensMax];
  extern __shared__ __attribute__((aligned(16))) uint8_t xbuf[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int NK = a.N * a.K, strips = (a.U + 15) / 16;
  const int o = blockIdx.x / strips, n0 = (blockIdx.x - o * strips) * 16;
  const Entry en = plan_entries(a.idx, a.w, NK, a.K, a.E);
  const bool mine = en.keep && en.ord == o;
  const uint64_t mask = __ballot(mine);
  if (!mask) return;  // uniform: fewer experts than that have rows
  const int f = __builtin_ctzll(mask);
  const int e = __builtin_amdgcn_readlane(en.e, f), row0 = __builtin_amdgcn_readlane(en.row, f);
  const int rows = __popcll(mask);  // <= N <= kTokensMax
  if (wave == 0 && mine) s_tok[en.row - row0] = lane / a.K;

  const int nb = a.H / kMxBlock, KS = (nb + 7) / 8;
  const int64_t sp = (nb + 3) / 4 * 4;
  const XLds xl(xbuf, KS, rows);
  const uint8_t *wrow[NT], *wsrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t r = static_cast<int64_t>(e) * NT * a.U + j * a.U + n0 + l16;  // U % 32 == 0
    wrow[j] = a.w_up + r * 16 * nb;
    wsrow[j] = a.s_up + r * sp;
  }
  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool first = true;
  for (int b0 = wave; b0 < KS || first; b0 += 4 * D) {
    Piece w[D][NT];
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int j = 0; j < NT; ++j) w[d][j] = load_piece(wrow[j], wsrow[j], min(b0 + 4 * d, KS - 1), q, nb);
    if (first) {
      __syncthreads();  // s_tok
      const bool vec = (reinterpret_cast<uintptr_t>(a.msg) | static_cast<uintptr_t>(a.H) * elt_bytes<XDT>()) % 16 == 0;
      const int total = rows * 2 * KS;
      for (int i0 = wave * 4; i0 < total; i0 += 16) {  // uniform
        const int i = min(i0 + q, total - 1), r = i / (2 * KS);
        quant_to_lds<XDT>(xl, reinterpret_cast<const char*>(a.msg) + static_cast<int64_t>(s_tok[r]) * a.H * elt_bytes<XDT>(), r,
                          i - r * 2 * KS, a.H, vec, l16, i0 + q < total);
      }
      __syncthreads();
      first = false;
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = b0 + 4 * d;
      if (b >= KS) break;  // uniform
      const Piece x = xl.load(min(l16, rows - 1), b, q);
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[j] = product(w[d][j], x, acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) *reinterpret_cast<f32x4*>(red + (wave * NT + j) * 256 + lane * 4) = acc[j];
  __syncthreads();
  if (wave > 0 || l16 >= rows) return;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 1; u < 4; ++u) acc[j] += *reinterpret_cast<const f32x4*>(red + (u * NT + j) * 256 + lane * 4);
  const int c = n0 + 4 * q;
  f32x4 y;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float b = a.b_up ? a.b_up[static_cast<int64_t>(e) * a.U + c + v] : 0.f;
    y[v] = SWIGLU ? silu(acc[0][v]) * (acc[NT - 1][v] + b) : gelu_tail(acc[0][v] + b);
  }
  *reinterpret_cast<f32x4*>(a.act + static_cast<int64_t>(row0 + l16) * a.U + c) = y;
}

// Down products of every expert that has rows, 16 channels a workgroup: a
// tile's 16 columns are the tokens, a token's column holds its row of the expert
// at hand (a token without one leaves its sum as it is).  Eight waves take every
// eighth (expert, 256 of K); an expert's part of a wave's sum is weighted as it
// is added, the waves' sums are added in wave order.
template <int ODT>
__global__ __launch_bounds__(512, 4) void k_mx_tokens_down(const MxTokensArgs a) {
  constexpr int D = 4;
  __shared__ __attribute__((aligned(16))) float red[8 * 256];
  __shared__ int s_row[kTokensMax * kTokensMax], s_exp[kTokensMax];
  __shared__ float s_w[kTokensMax * kTokensMax];
  extern __shared__ __attribute__((aligned(16))) uint8_t xbuf[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int NK = a.N * a.K, n0 = blockIdx.x * 16;
  const Entry en = plan_entries(a.idx, a.w, NK, a.K, a.E);
  const int rows = __popcll(__ballot(en.keep));
  int experts = 0;
  for (int i = 0; i < NK; ++i) {
    const int k = __builtin_amdgcn_readlane(en.keep ? en.ord + 1 : 0, i);
    experts = max(experts, k);
  }
  for (int i = tid; i < kTokensMax * kTokensMax; i += 512) s_row[i] = -1;
  __syncthreads();
  if (wave == 0 && en.keep) {
    const int at = en.ord * kTokensMax + lane / a.K;
    s_row[at] = en.row;
    s_w[at] = en.w;
    s_exp[en.ord] = en.e;  // equal from every entry of the expert
  }
  const int nb = a.U / kMxBlock, KS = (nb + 7) / 8;
  const int64_t sp = (nb + 3) / 4 * 4;
  const XLds xl(xbuf, KS, rows);
  const int total = rows * 2 * KS;
  for (int i0 = wave * 4; i0 < total; i0 += 32) {  // uniform; U % 32 == 0: whole vectors
    const int i = min(i0 + q, total - 1), r = i / (2 * KS);
    quant_to_lds<SMOE_F32>(xl, a.act + static_cast<int64_t>(r) * a.U, r, i - r * 2 * KS, a.U, true, l16, i0 + q < total);
  }
  __syncthreads();
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int items = experts * KS;
  for (int i0 = wave; i0 < items; i0 += 8 * D) {
    Piece w[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = min(i0 + 8 * d, items - 1), o = i / KS;
      const int64_t r = static_cast<int64_t>(s_exp[o]) * a.H + n0 + l16;  // H % 32 == 0
      w[d] = load_piece(a.w_down + r * 16 * nb, a.s_down + r * sp, i - o * KS, q, nb);
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = i0 + 8 * d;
      if (i >= items) break;  // uniform
      const int o = i / KS;
      const int r = s_row[o * kTokensMax + l16], rc = max(r, 0);
      const f32x4 part = product(w[d], xl.load(rc, i - o * KS, q), f32x4{0.f, 0.f, 0.f, 0.f});
      const float sc = s_w[o * kTokensMax + l16];
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[v] = r >= 0 ? fmaf(part[v], sc, acc[v]) : acc[v];
    }
  }
  *reinterpret_cast<f32x4*>(red + wave * 256 + lane * 4) = acc;
  __syncthreads();
  if (wave > 0 || l16 >= a.N) return;
#pragma unroll
  for (int u = 1; u < 8; ++u) acc += *reinterpret_cast<const f32x4*>(red + u * 256 + lane * 4);
  const int n = n0 + 4 * q;
  if (a.b_down)
    for (int o = 0; o < experts; ++o) {
      const int at = o * kTokensMax + l16;
      if (s_row[at] < 0) continue;
#pragma unroll
      for (int v = 0; v < 4; ++v)
        acc[v] = fmaf(a.b_down[static_cast<int64_t>(s_exp[o]) * a.H + n + v], s_w[at], acc[v]);
    }
  const int64_t at = static_cast<int64_t>(l16) * a.H + n;
  if constexpr (ODT == SMOE_F32) {
#pragma unroll
    for (int v = 0; v < 4; ++v) reinterpret_cast<float*>(a.out)[at + v] = acc[v];
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v) reinterpret_cast<uint16_t*>(a.out)[at + v] = f2bf(acc[v]);
  }
}

// A small step's plan and its quantized messages in one launch: workgroup 0
// makes the plan, the others quantize 64 pieces each.  The plan bounds it: 64
// tokens, 2 of 16 experts 3.0 us, 777 tokens, 4 of 32 experts 5.7 us.
template <int KB, int T>
__global__ __launch_bounds__(1024) void k_prep_mx(const PrepArgs a, const MxQuant mq, int npc, int64_t total) {
  if (blockIdx.x > 0) {
    const int64_t b = (static_cast<int64_t>(blockIdx.x - 1) * 1024 + threadIdx.x) >> 4;
    if (mq.x_dtype == SMOE_F32) mx_quant_piece<SMOE_F32>(mq, npc, total, b, threadIdx.x & 15);
    else mx_quant_piece<SMOE_BF16>(mq, npc, total, b, threadIdx.x & 15);
    return;
  }
  prep_plan<KB, T>(a);
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

template <int EPI, int ODT, int MT, int XQ>
int go_few(const MxGemm& a, hipStream_t s) {
  const int64_t grid = (static_cast<int64_t>(a.single_rows) + 16 * MT - 1) / (16 * MT) * ((static_cast<int64_t>(a.N_out) + 15) / 16);
  if (grid * 256 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  if (a.dry) return SMOE_OK;
  const size_t lds = XQ >= 0 ? static_cast<size_t>(std::min(16 * MT, a.single_rows)) * xlds_row(a.K) : 0;
  SMOE_LAUNCH((k_mx_few<EPI, ODT, MT, XQ>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, s, a);
  return rc();
}

template <int EPI, int ODT>
int go_rows(const MxGemm& a, hipStream_t s) {
  if (a.x_float) return by_xdt(a.x_dtype, [&](auto xd) { return go_few<EPI, ODT, 1, decltype(xd)::value>(a, s); });
  return a.single_rows <= 16 ? go_few<EPI, ODT, 1, -1>(a, s) : go_few<EPI, ODT, 2, -1>(a, s);
}

// LDS for quantized rows beside a kernel's own
constexpr int64_t kXLds = 49152;

}  // namespace

// Whole calls in a graph, us, this kernel and tiles: 17 x 2048 -> 1408 5.9 and 6.9,
// 24 rows 6.4 and 7.0, 48 rows 6.6 and 7.2; 24 x 1000 -> 2800 6.3 and 6.2, 40 rows
// 7.7 and 6.3.  With many channels it reads every row once for 16 of them, and tiles
// would be ahead: 24 x 1024 -> 5632 8.0 and 6.1, 17 x 4096 -> 40000 34.7 and 19.8.
bool gemm_mx_few_fits(const MxGemm& a) { return a.G == 0 && a.ws_plane == 0 && a.single_rows <= kMxFewRows; }

// Up to one row tile, and while each workgroup's own quantizing costs about what a
// launch does.  Inside and by a launch of its own, us in a graph (from the host a
// launch is 4 more): into 1408 channels 1 x 4096 4.3 and 5.7, 4 x 1024 4.3 and 5.9,
// 16 x 1024 6.6 and 6.8, 4 x 4096 6.7 and 6.2, 8 x 2048 6.7 and 6.3, 2 x 8192 8.1 and
// 7.9; past it 16 x 1536 8.0 and 6.5, 8 x 4096 10.0 and 6.5; into 50257 channels 4 x
// 1024 21.0 and 28.0, 8 x 2048 32.4 and 33.1, past it 8 x 4096 47.9 and 33.9.
bool mx_linear_quantizes_inside(int N, int K) {
  return N <= 16 && static_cast<int64_t>(N) * K <= 16384 && static_cast<int64_t>(N) * xlds_row(K) <= kXLds;
}

int launch_gemm_mx_few(const MxGemm& a, hipStream_t s) {
  if (a.ws_plane) return SMOE_EINVAL;  // the kernel reads rows of scales
  const bool f32 = a.out_dtype == SMOE_F32;
  if (a.epi == MX_LINEAR) return f32 ? go_rows<MX_LINEAR, SMOE_F32>(a, s) : go_rows<MX_LINEAR, SMOE_BF16>(a, s);
  if (a.epi == MX_GELU) return f32 ? go_rows<MX_GELU, SMOE_F32>(a, s) : go_rows<MX_GELU, SMOE_BF16>(a, s);
  return SMOE_EINVAL;
}

// Up to 4 rows a group on average, and up to 8 where the staged kernel's tiles (32
// rows, 64 channels of SwiGLU or 128) do not give every CU one.  Both products and
// the plan, us, streamed and staged: 64 experts of 2048 x 1408, 64 tokens (2 rows)
// 40.1 and 41.5, 128 tokens (4 rows) 45.5 and 46.8; 32 experts of 1024 x 1408, 32
// tokens (4 rows) 23.7 and 25.2; 16 experts of 1024 x 2816, SwiGLU, 32 tokens (4
// rows) 26.3 and 26.5, 64 tokens (8 rows) 30.8 and 27.0, but only the down product,
// of 128 tiles, streamed 26.6; 12 experts of 544 x 1184, 32 tokens (8 rows) 15.4
// and 18.5; 8 experts of 256 x 512, 32 tokens (8 rows) 11.8 and 15.3, 64 tokens (16
// rows) 16.2 and 15.2.
bool gemm_mx_stream_fits(const MxGemm& a) {
  if (a.G < 1 || a.ws_plane != 0) return false;
  const int ch = a.epi == MX_UP_SWIGLU ? 64 : 128;
  const int64_t tiles = static_cast<int64_t>(std::min(a.G, a.max_rows)) * ((a.N_out - 1) / ch + 1);
  return a.max_rows <= (tiles <= device_cus() ? 8ll : 4ll) * a.G;
}

int launch_gemm_mx_stream(const MxGemm& a, hipStream_t s) {
  const bool up = a.epi == MX_UP_GELU || a.epi == MX_UP_SWIGLU;
  const int64_t grid = static_cast<int64_t>(a.G) * (a.N_out / (up ? 32 : 16));
  if (a.ws_plane || a.N_out % 32 || (!up && a.epi != MX_DOWN) || grid * 256 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  if (a.dry) return SMOE_OK;
  const dim3 g(static_cast<unsigned>(grid)), b(256);
  if (a.epi == MX_UP_GELU) SMOE_LAUNCH((k_mx_stream<MX_UP_GELU>), g, b, 0, s, a);
  else if (a.epi == MX_UP_SWIGLU) SMOE_LAUNCH((k_mx_stream<MX_UP_SWIGLU>), g, b, 0, s, a);
  else SMOE_LAUNCH((k_mx_stream<MX_DOWN>), g, b, 0, s, a);
  return rc();
}

int launch_prep_mx(const PrepArgs& a, const MxQuant& q, hipStream_t s) {
  const int npc = (q.cols - 1) / 128 + 1;
  const int64_t total = q.rows * npc, wgs = (total + 63) / 64 + 1;
  if (!prep_fits(a.N, a.K, a.E) || wgs * 1024 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  return by_prep(a.N, a.K, [&](auto kb, auto t) {
    SMOE_LAUNCH((k_prep_mx<decltype(kb)::value, decltype(t)::value>), dim3(static_cast<unsigned>(wgs)), dim3(1024),
                prep_lds(a), s, a, q, npc, total);
    return rc();
  });
}

bool mx_tokens_fit(int N, int K, int H, int U) {
  return N * static_cast<int64_t>(K) <= kTokensMax && static_cast<int64_t>(N) * xlds_row(H) <= kXLds &&
         static_cast<int64_t>(N) * K * xlds_row(U) <= kXLds;
}

int launch_mx_tokens(const MxTokensArgs& a, hipStream_t s) {
  const dim3 up(static_cast<unsigned>(std::min(a.E, a.N * a.K) * ((a.U + 15) / 16)));
  const size_t lds_up = static_cast<size_t>(a.N) * xlds_row(a.H);
  const size_t lds_down = static_cast<size_t>(a.N) * a.K * xlds_row(a.U);
  const bool f32 = a.msg_dtype == SMOE_F32;
  if (a.act_fn == SMOE_ACT_SWIGLU) {
    if (f32) hipLaunchKernelGGL((k_mx_tokens_up<true, SMOE_F32>), up, dim3(256), lds_up, s, a);
    else hipLaunchKernelGGL((k_mx_tokens_up<true, SMOE_BF16>), up, dim3(256), lds_up, s, a);
  } else {
    if (f32) hipLaunchKernelGGL((k_mx_tokens_up<false, SMOE_F32>), up, dim3(256), lds_up, s, a);
    else hipLaunchKernelGGL((k_mx_tokens_up<false, SMOE_BF16>), up, dim3(256), lds_up, s, a);
  }
  const dim3 down(static_cast<unsigned>((a.H + 15) / 16));
  if (a.out_dtype == SMOE_F32) hipLaunchKernelGGL((k_mx_tokens_down<SMOE_F32>), down, dim3(512), lds_down, s, a);
  else hipLaunchKernelGGL((k_mx_tokens_down<SMOE_BF16>), down, dim3(512), lds_down, s, a);
  return rc();
}

}  // namespace smoe

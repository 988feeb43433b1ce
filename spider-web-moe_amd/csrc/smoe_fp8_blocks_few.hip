// Block-scaled fp8 steps of a few rows: dense products and expert steps whose
// waves load the weights' fragments straight into registers, and the launch
// that makes a decode step's plan and quantizes its messages.
#include "smoe_fp8_blocks_dev.hpp"
#include "smoe_internal.hpp"
#include "smoe_routing.hpp"

namespace smoe {
namespace {

// A lane's 32 codes of a 128-wide block: bytes 16 q .. + 15 of both halves
// (q = lane / 16), so that one load instruction covers whole 64-byte pieces
// of 16 rows.  Both operands pair the same k, in whatever order.
struct Piece {
  u32x4 lo, hi;
};
__device__ __forceinline__ Piece load_piece(const uint8_t* row, int k0, int q, int K) {
  const int a = k0 + 16 * q, b = a + 64;  // chunks past K: the row's first one, cut before use
  return {*reinterpret_cast<const u32x4*>(row + (a < K ? a : 0)),
          *reinterpret_cast<const u32x4*>(row + (b < K ? b : 0))};
}
__device__ __forceinline__ Piece cut_piece(Piece p, int q, int left) {
  return {cut16(p.lo, left - 16 * q), cut16(p.hi, left - 64 - 16 * q)};
}
__device__ __forceinline__ i32x8 frag_of(const Piece& p) {
  return __builtin_bit_cast(i32x8, (uint32_t __attribute__((ext_vector_type(8)))){
                                       p.lo.x, p.lo.y, p.lo.z, p.lo.w, p.hi.x, p.hi.y, p.hi.z, p.hi.w});
}

template <bool WIDE>
__device__ __forceinline__ f32x4 block_product(const Piece& w, const Piece& x) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if constexpr (WIDE) {
    bf16x8 a[4], b[4];
    widen_frag(frag_of(w), a);
    widen_frag(frag_of(x), b);
    f32x4 part = zero;
#pragma unroll
    for (int u = 0; u < 4; ++u) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[u], b[u], part, 0, 0, 0);
    return part;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(frag_of(w), frag_of(x), zero, 0, 0, 0, 0, 0, 0);
  }
}

// Dense products of 16 MT rows: 16 channels a workgroup, four waves taking
// every fourth block of K straight into registers, D blocks at once; their sums
// are added through LDS in wave order.
//
// XQ: -1 X is codes; else its dtype (x_float), which the workgroup quantizes
// into LDS while its first weights are on their way: one launch for a few
// tokens (1 x 2048 -> 1408: 4.8 us; quantizer and product 3 + 4.2).
template <int EPI, int ODT, bool WIDE, int MT, int XQ>
__global__ __launch_bounds__(256, 4) void k_blocks_few(const BlockGemm p) {
  constexpr int BM = 16 * MT, NW = 4, D = MT == 1 ? 4 : (WIDE ? 2 : 3);
  __shared__ __attribute__((aligned(16))) float red[NW * MT * 256];
  extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];  // XQ >= 0
  const int strips = (p.N_out + 15) / 16;
  const int m0 = static_cast<int>(blockIdx.x) / strips * BM, n0 = static_cast<int>(blockIdx.x) % strips * 16;
  const int mrows = min(BM, p.single_rows - m0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int KB = (p.K + 127) / 128;

  const uint8_t* wrow = p.W + static_cast<int64_t>(min(n0 + l16, p.N_out - 1)) * p.ldw;
  const uint8_t* xrow[MT];
  const float* srow[MT];
  const int ldl = KB * 128;  // XQ: row pitch in LDS
  float* const xsl = reinterpret_cast<float*>(xlds + BM * ldl);  // [KB][BM]
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t r = XQ >= 0 ? 0 : m0 + min(16 * i + l16, mrows - 1);  // rows past the end: a valid one, never stored
    xrow[i] = p.X + r * p.ldx;
    srow[i] = p.xs + r * p.xs_row;
  }
  const float* wsp = p.ws + static_cast<int64_t>(n0 / 128) * KB;

  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  bool first = true;
  for (int b0 = wave; b0 < KB || (XQ >= 0 && first); b0 += D * NW) {
    Piece w[D], x[D][MT];
    float xsv[D][MT], ws[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = min(b0 + d * NW, KB - 1);  // past the end: the last block again, not used
      w[d] = load_piece(wrow, 128 * b, q, p.K);
      if constexpr (XQ < 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          x[d][i] = load_piece(xrow[i], 128 * b, q, p.K);
          xsv[d][i] = srow[i][b * p.xs_col];
        }
      }
      ws[d] = wsp[b];
    }
    if constexpr (XQ >= 0) {
      if (first) {  // sixteen lanes quantize a block
        constexpr int XD = XQ;
        const bool vec = (reinterpret_cast<uintptr_t>(p.x_float) | static_cast<uintptr_t>(p.ld_float * elt_bytes<XD>())) % 16 == 0;
        for (int e = tid >> 4; e < mrows * KB; e += NW * 4) {
          const int r = e / KB, b = e - r * KB;
          const char* rp = reinterpret_cast<const char*>(p.x_float) + static_cast<int64_t>(m0 + r) * p.ld_float * elt_bytes<XD>();
          float v[8];
          load_cols8<XD>(rp, 128 * b + 8 * l16, p.K, vec, v);
          const float sc = block_scale(row16_max(amax8(v)));
          if (l16 == 0) xsl[b * BM + r] = sc;
          *reinterpret_cast<u32x2*>(xlds + r * ldl + 128 * b + 8 * l16) = codes8(v, sc);
        }
        __syncthreads();
        first = false;
      }
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int b = min(b0 + d * NW, KB - 1);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int r = min(16 * i + l16, mrows - 1);
          x[d][i] = load_piece(xlds + r * ldl, 128 * b, q, ldl);
          xsv[d][i] = xsl[b * BM + r];
        }
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = b0 + d * NW;
      if (b >= KB) break;  // uniform
      const int left = p.K - 128 * b;
      if (left < 128) {  // uniform: the last block of a ragged K
        w[d] = cut_piece(w[d], q, left);
        if constexpr (XQ < 0)
#pragma unroll
          for (int i = 0; i < MT; ++i) x[d][i] = cut_piece(x[d][i], q, left);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f32x4 part = block_product<WIDE>(w[d], x[d][i]);
        const float sc = xsv[d][i] * ws[d];
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[i][v] = fmaf(part[v], sc, acc[i][v]);
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
    o[v] = EPI == BLK_GELU ? gelu_erf(y) : y;
  }
  store4<ODT>(p, m0 + r, n, o);
}

// ------------------------------------------------- a few tokens' experts ----
// At most 16 (token, slot) entries: the whole expert step in two launches that
// keep the dispatch plan in registers and quantize their own operands.
//
// The plan, by one wave, lane j = entry j (token j / K): an id's slots of one
// token merged into the first (weights added in slot order from 0, as
// smoe_dispatch_plan adds them), ids outside [0, E) and sums that are not > 0
// left out.  row: the entry's place among the kept ones by (expert, token);
// ord: how many smaller experts have rows.
struct Entry {
  int e, row, ord;
  float w;
  bool keep;
};
__device__ __forceinline__ Entry plan_entries(const int32_t* __restrict__ idx, const float* __restrict__ w, int NK,
                                              int K, int E) {
  const int j = threadIdx.x & 63;
  const int jc = min(j, NK - 1), t = jc / K;
  const int e = idx[jc];
  const float wj = w[jc];
  Entry r{e, 0, 0, 0.f, j < NK && e >= 0 && e < E};
  for (int i = 0; i < NK; ++i) {
    const int ei = __builtin_amdgcn_readlane(e, i);
    const float wi = lane_f(wj, i);
    const bool same = ei == e && i / K == t;
    r.keep = r.keep && !(same && i < j);
    r.w = same ? r.w + wi : r.w;
  }
  r.keep = r.keep && r.w > 0.f;
  const uint64_t kept = __ballot(r.keep);
  bool lead = r.keep;  // the expert's first kept entry
  for (int i = 0; i < NK; ++i) {
    const int ei = __builtin_amdgcn_readlane(e, i);
    const bool k = kept >> i & 1;
    lead = lead && !(k && ei == e && i < j);
    r.row += k && (ei < e || (ei == e && i < j)) ? 1 : 0;
  }
  const uint64_t leads = __ballot(lead);
  for (int i = 0; i < NK; ++i)
    r.ord += (leads >> i & 1) && __builtin_amdgcn_readlane(e, i) < e ? 1 : 0;
  return r;
}

constexpr int kTokensMax = 16;  // entries (and so tokens, experts and rows)

// Up product of one expert's rows and 16 channels (SwiGLU: of gate and up):
// four waves take every fourth block of K, the rows' messages are quantized
// into LDS under the first weights' loads; activations leave in f32 at their
// plan rows.  Bound by the latency of its loads: 2 of 64 experts, 2048 -> 1408,
// 5.8 MB in 6 us.
template <bool SWIGLU, int XDT, bool WIDE>
__global__ __launch_bounds__(256, 4) void k_tokens_up(const TokensArgs a) {
  constexpr int NT = SWIGLU ? 2 : 1, D = SWIGLU ? 3 : 4;
  __shared__ __attribute__((aligned(16))) float red[4 * NT * 256];
  __shared__ int s_tok[kTokensMax];
  extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
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

  const int KB = (a.H + 127) / 128, ldl = KB * 128;
  float* const xsl = reinterpret_cast<float*>(xlds + a.N * ldl);  // [KB][N]
  const uint8_t* wrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
    wrow[j] = a.w_up + (static_cast<int64_t>(e) * NT * a.U + j * a.U + n0 + l16) * a.H;  // U % 16 == 0
  const int ub = (a.U + 127) / 128;
  const float* wsp = a.s_up + (static_cast<int64_t>(e) * NT * ub + n0 / 128) * KB;
  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool first = true;
  for (int b0 = wave; b0 < KB || first; b0 += 4 * D) {
    Piece w[D][NT];
    float ws[D][NT];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = min(b0 + 4 * d, KB - 1);  // past the end: the last block again, not used
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        w[d][j] = load_piece(wrow[j], 128 * b, q, a.H);
        ws[d][j] = wsp[j * ub * KB + b];
      }
    }
    if (first) {
      __syncthreads();  // s_tok
      const bool vec = (reinterpret_cast<uintptr_t>(a.msg) | static_cast<uintptr_t>(a.H) * elt_bytes<XDT>()) % 16 == 0;
      for (int i = tid >> 4; i < rows * KB; i += 16) {
        const int r = i / KB, b = i - r * KB;
        const char* rp = reinterpret_cast<const char*>(a.msg) + static_cast<int64_t>(s_tok[r]) * a.H * elt_bytes<XDT>();
        float v[8];
        load_cols8<XDT>(rp, 128 * b + 8 * l16, a.H, vec, v);
        const float sc = block_scale(row16_max(amax8(v)));
        if (l16 == 0) xsl[b * a.N + r] = sc;
        *reinterpret_cast<u32x2*>(xlds + r * ldl + 128 * b + 8 * l16) = codes8(v, sc);
      }
      __syncthreads();
      first = false;
    }
    const int r = min(l16, rows - 1);
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = b0 + 4 * d;
      if (b >= KB) break;  // uniform
      const Piece x = load_piece(xlds + r * ldl, 128 * b, q, ldl);
      const float xs = xsl[b * a.N + r];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (a.H - 128 * b < 128) w[d][j] = cut_piece(w[d][j], q, a.H - 128 * b);
        const f32x4 part = block_product<WIDE>(w[d][j], x);
        const float sc = xs * ws[d][j];
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[j][v] = fmaf(part[v], sc, acc[j][v]);
      }
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
    y[v] = SWIGLU ? silu(acc[0][v]) * (acc[NT - 1][v] + b) : gelu_erf(acc[0][v] + b);
  }
  *reinterpret_cast<f32x4*>(a.act + static_cast<int64_t>(row0 + l16) * a.U + c) = y;
}

// Down products of every expert that has rows, 16 channels a workgroup, added
// over the experts as they are multiplied: a tile's 16 columns are the tokens,
// a token's column holds its row of the expert at hand (a token without one
// leaves its sum as it is) and its weight goes into the scale.  Eight waves
// take every eighth (expert, block of K), their sums added in wave order.
// 2 experts, 1408 -> 2048: 7 us, the quantizing of 1408 activations before the
// first product among them (in the up product's epilogue it would need all of a
// block's workgroups).
template <int ODT>
__global__ __launch_bounds__(512, 4) void k_tokens_down(const TokensArgs a) {
  constexpr int D = 4;
  constexpr bool WIDE = ODT == SMOE_F32;
  __shared__ __attribute__((aligned(16))) float red[8 * 256];
  __shared__ int s_row[kTokensMax * kTokensMax], s_exp[kTokensMax];
  __shared__ float s_w[kTokensMax * kTokensMax];
  extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
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
  const int KB = (a.U + 127) / 128, ldl = KB * 128, hb = (a.H + 127) / 128;
  float* const xsl = reinterpret_cast<float*>(xlds + rows * ldl);  // [KB][rows]
  const bool vec = reinterpret_cast<uintptr_t>(a.act) % 16 == 0;  // U % 16 == 0
  for (int i = tid >> 4; i < rows * KB; i += 32) {
    const int r = i / KB, b = i - r * KB;
    float v[8];
    load_cols8<SMOE_F32>(a.act + static_cast<int64_t>(r) * a.U, 128 * b + 8 * l16, a.U, vec, v);
    const float sc = block_scale(row16_max(amax8(v)));
    if (l16 == 0) xsl[b * rows + r] = sc;
    *reinterpret_cast<u32x2*>(xlds + r * ldl + 128 * b + 8 * l16) = codes8(v, sc);
  }
  __syncthreads();
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int items = experts * KB;
  for (int i0 = wave; i0 < items; i0 += 8 * D) {
    Piece w[D];
    float ws[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = min(i0 + 8 * d, items - 1), o = i / KB, b = i - o * KB;
      const int64_t e = s_exp[o];
      w[d] = load_piece(a.w_down + (e * a.H + n0 + l16) * a.U, 128 * b, q, a.U);  // H % 16 == 0
      ws[d] = a.s_down[(e * hb + n0 / 128) * KB + b];
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = i0 + 8 * d;
      if (i >= items) break;  // uniform
      const int o = i / KB, b = i - o * KB;
      const int r = s_row[o * kTokensMax + l16], rc = max(r, 0);
      if (a.U - 128 * b < 128) w[d] = cut_piece(w[d], q, a.U - 128 * b);
      const f32x4 part = block_product<WIDE>(w[d], load_piece(xlds + rc * ldl, 128 * b, q, ldl));
      const float sc = xsl[b * rows + rc] * ws[d] * s_w[o * kTokensMax + l16];
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

// words of 64 tokens an expert takes: an odd number
__host__ __device__ inline int prep_pitch(int N) { return ((N + 63) / 64) | 1; }

// The plan of a decode step or a short prompt (K <= KB, N <= 1024 T) and its
// quantized messages in one launch: workgroup 0 makes the plan (the one
// smoe_dispatch_plan makes), the others quantize 64 blocks each.
//
// T tokens per thread, their slots in registers: ids that occur twice are
// merged into their first slot (weights added in slot order from 0), ids
// outside [0, E) and sums that are not > 0 left out.  Every kept (token,
// expert) sets the token's bit in the expert's masks, one word for 64 tokens,
// by an LDS atomic OR (its result does not depend on the order); a row is then
// the expert's offset, its counts in the words before and the bits below.
// LDS: E * P masks, then as many counts; an odd pitch P, without which the
// experts' words of 64 tokens meet in one bank; after them the plan's rows.
// 777 tokens of 1024 channels, top-4 of 32: 15.6 -> 5.9 us against ranking by
// ballots through memory; what is left is the plan's one workgroup.
template <int KB, int T>
__global__ __launch_bounds__(1024) void k_prep(const PrepArgs a, const BlockQuant bq, int nblk, int64_t total) {
  extern __shared__ unsigned long long mask[];
  __shared__ int tot[kPlanMaxG], goff[kPlanMaxG + 1], wsum[4];
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    auto run = [&](auto xd) {
      quant_row_block<decltype(xd)::value>(bq, nblk, total,
                                           (static_cast<int64_t>(blockIdx.x - 1) * 1024 + tid) >> 4, tid & 15);
    };
    if (bq.x_dtype == SMOE_F32) run(std::integral_constant<int, SMOE_F32>{});
    else run(std::integral_constant<int, SMOE_BF16>{});
    return;
  }
  const int N = a.N, K = a.K, E = a.E, C = (N + 63) / 64, P = prep_pitch(N);
  uint16_t* before = reinterpret_cast<uint16_t*>(mask + E * P);
  int id[T][KB];
  float w[T][KB], sum[T][KB];
  bool use[T][KB];
#pragma unroll
  for (int u = 0; u < T; ++u)
#pragma unroll
    for (int j = 0; j < KB; ++j) {  // unconditional loads at clamped indices
      const int at = min(u * 1024 + tid, N - 1) * K + min(j, K - 1);
      id[u][j] = a.idx[at];
      w[u][j] = a.w[at];
    }
  for (int i = tid; i < E * P; i += 1024) mask[i] = 0ull;
#pragma unroll
  for (int u = 0; u < T; ++u)
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      use[u][j] = u * 1024 + tid < N && j < K && id[u][j] >= 0 && id[u][j] < E;
      sum[u][j] = 0.f;
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        if (i < j) use[u][j] = use[u][j] && id[u][i] != id[u][j];  // its first slot speaks for an id
        sum[u][j] = i < K && id[u][i] == id[u][j] ? sum[u][j] + w[u][i] : sum[u][j];
      }
      use[u][j] = use[u][j] && sum[u][j] > 0.f;
    }
  __syncthreads();
  const int c = tid >> 6, lane = tid & 63;
  const unsigned long long bit = 1ull << lane;
#pragma unroll
  for (int u = 0; u < T; ++u)
#pragma unroll
    for (int j = 0; j < KB; ++j)
      if (use[u][j]) atomicOr(&mask[id[u][j] * P + 16 * u + c], bit);
  __syncthreads();
  if constexpr (T == 1) {  // a thread an expert
    if (tid < E) {
      int n = 0;
      for (int i = 0; i < C; ++i) {
        before[tid * P + i] = static_cast<uint16_t>(n);
        n += __popcll(mask[tid * P + i]);
      }
      tot[tid] = n;
    }
  } else {
    for (int e = c; e < E; e += 16) {  // a wave an expert, a lane a word: C <= 64
      const int n = lane < C ? __popcll(mask[e * P + lane]) : 0;
      const int upto = wave_incl_scan(n);
      if (lane < C) before[e * P + lane] = static_cast<uint16_t>(upto - n);
      if (lane == 63) tot[e] = upto;
    }
  }
  __syncthreads();
  block_group_offsets(tot, E, goff, wsum);
  for (int g = tid; g <= E; g += 1024) a.off[g] = goff[g];
  int row[T][KB];
#pragma unroll
  for (int u = 0; u < T; ++u) {
    const int t = u * 1024 + tid;
    int n = 0;
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      int rank = 0;  // among the token's experts, ascending
#pragma unroll
      for (int i = 0; i < KB; ++i) rank += use[u][i] && id[u][i] < id[u][j] ? 1 : 0;
      if (!use[u][j]) continue;
      const int at = id[u][j] * P + 16 * u + c;
      row[u][j] = goff[id[u][j]] + before[at] + __popcll(mask[at] & (bit - 1ull));
      a.tokrow[t * K + rank] = row[u][j];
      ++n;
    }
    for (int j = n; j < K && t < N; ++j) a.tokrow[t * K + j] = -1;
  }
  __syncthreads();  // the masks are read
  // rows and their weights leave in order: scattered from here, each store of a
  // wave took a cycle per lane
  float* const lw = reinterpret_cast<float*>(mask);
  uint16_t* const lt = reinterpret_cast<uint16_t*>(lw + N * K);
#pragma unroll
  for (int u = 0; u < T; ++u)
#pragma unroll
    for (int j = 0; j < KB; ++j)
      if (use[u][j]) {
        lw[row[u][j]] = sum[u][j];
        lt[row[u][j]] = static_cast<uint16_t>(u * 1024 + tid);
      }
  __syncthreads();
  for (int r = tid; r < goff[E]; r += 1024) {
    a.rows[r] = lt[r];
    a.roww[r] = lw[r];
  }
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

template <int EPI, int ODT, bool WIDE, int MT, int XQ>
int go_few(const BlockGemm& a, hipStream_t s) {
  const int64_t grid = (static_cast<int64_t>(a.single_rows) + 16 * MT - 1) / (16 * MT) * ((static_cast<int64_t>(a.N_out) + 15) / 16);
  if (grid * 256 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  const size_t lds = XQ >= 0 ? static_cast<size_t>(16 * MT) * fp8_blocks_of(a.K) * 132 : 0;
  SMOE_LAUNCH((k_blocks_few<EPI, ODT, WIDE, MT, XQ>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, s, a);
  return rc();
}

template <int EPI, int ODT, bool WIDE>
int go_rows(const BlockGemm& a, hipStream_t s) {
  if (a.x_float) return by_xdt(a.x_dtype, [&](auto xd) { return go_few<EPI, ODT, WIDE, 1, decltype(xd)::value>(a, s); });
  return a.single_rows <= 16 ? go_few<EPI, ODT, WIDE, 1, -1>(a, s) : go_few<EPI, ODT, WIDE, 2, -1>(a, s);
}

}  // namespace

// Up to 24 rows (24 x 2816 -> 1024: 6.5 us, tiles through LDS 7.9; 32 x 2048 ->
// 1408: 7.9 and 6.6).
bool gemm_blocks_few_fits(const BlockGemm& a) { return a.G == 0 && a.single_rows <= 24; }

bool linear_quantizes_inside(int N, int K) {
  return N <= 16 && static_cast<int64_t>(N) * K <= 16384 && 16 * static_cast<int64_t>(fp8_blocks_of(K)) * 132 <= 49152;
}

int launch_gemm_blocks_few(const BlockGemm& a, hipStream_t s) {
  const bool f32 = a.out_dtype == SMOE_F32;
  if (a.epi == BLK_LINEAR) return f32 ? go_rows<BLK_LINEAR, SMOE_F32, true>(a, s) : go_rows<BLK_LINEAR, SMOE_BF16, false>(a, s);
  if (a.epi == BLK_GELU) return f32 ? go_rows<BLK_GELU, SMOE_F32, true>(a, s) : go_rows<BLK_GELU, SMOE_BF16, false>(a, s);
  return SMOE_EINVAL;
}

// Up to 8192 choices, which the plan's one workgroup holds in registers and LDS,
// against three launches and the quantizer's.  Whole steps of 1500 tokens: top-4
// of 32 69 -> 65 us, top-2 of 96 44 -> 34; 4096 tokens, top-2 of 64: 181 -> 175.
bool prep_fits(int N, int K, int E) {
  return K <= 16 && N <= 4096 && N * K <= 8192 && E <= kPlanMaxG &&
         E * prep_pitch(N) <= 6300;  // 62 KB of LDS
}

int launch_prep(const PrepArgs& a, const BlockQuant& q, hipStream_t s) {
  const int nblk = fp8_blocks_of(q.cols);
  const int64_t total = static_cast<int64_t>(q.rows) * nblk, wgs = (total + 63) / 64 + 1;
  if (!prep_fits(a.N, a.K, a.E) || wgs * 1024 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  const size_t lds = std::max(static_cast<size_t>(a.E) * prep_pitch(a.N) * 10, static_cast<size_t>(a.N) * a.K * 6);
  auto go = [&](auto kb, auto t) {
    SMOE_LAUNCH((k_prep<decltype(kb)::value, decltype(t)::value>), dim3(static_cast<unsigned>(wgs)), dim3(1024), lds, s,
                a, q, nblk, total);
    return rc();
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  using I8 = std::integral_constant<int, 8>;
  using I16 = std::integral_constant<int, 16>;
  if (a.N <= 1024) return a.K <= 2 ? go(I2{}, I1{}) : a.K <= 4 ? go(I4{}, I1{}) : a.K <= 8 ? go(I8{}, I1{}) : go(I16{}, I1{});
  if (a.N <= 2048) return a.K <= 2 ? go(I2{}, I2{}) : a.K <= 4 ? go(I4{}, I2{}) : go(I8{}, I2{});
  return a.K <= 2 ? go(I2{}, I4{}) : go(I4{}, I4{});
}

// LDS of the two launches: quantized rows of up to N messages or N * K
// activations, and their scales
constexpr int64_t kTokensLds = 49152;

bool tokens_fit(int N, int K, int H, int U) {
  return N * static_cast<int64_t>(K) <= kTokensMax && static_cast<int64_t>(N) * fp8_blocks_of(H) * 132 <= kTokensLds &&
         static_cast<int64_t>(N) * K * fp8_blocks_of(U) * 132 <= kTokensLds;
}

int launch_tokens(const TokensArgs& a, hipStream_t s) {
  const dim3 up(static_cast<unsigned>(std::min(a.E, a.N * a.K) * ((a.U + 15) / 16)));
  const size_t lds_up = static_cast<size_t>(a.N) * fp8_blocks_of(a.H) * 132;
  const size_t lds_down = static_cast<size_t>(a.N) * a.K * fp8_blocks_of(a.U) * 132;
  const bool f32 = a.msg_dtype == SMOE_F32, wide = a.out_dtype == SMOE_F32;
  auto go_up = [&](auto sw, auto w) {
    constexpr bool SW = decltype(sw)::value, WD = decltype(w)::value;
    if (f32) hipLaunchKernelGGL((k_tokens_up<SW, SMOE_F32, WD>), up, dim3(256), lds_up, s, a);
    else hipLaunchKernelGGL((k_tokens_up<SW, SMOE_BF16, WD>), up, dim3(256), lds_up, s, a);
  };
  using Y = std::true_type;
  using N = std::false_type;
  if (a.act_fn == SMOE_ACT_SWIGLU) wide ? go_up(Y{}, Y{}) : go_up(Y{}, N{});
  else wide ? go_up(N{}, Y{}) : go_up(N{}, N{});
  const dim3 down(static_cast<unsigned>((a.H + 15) / 16));
  if (a.out_dtype == SMOE_F32) hipLaunchKernelGGL((k_tokens_down<SMOE_F32>), down, dim3(512), lds_down, s, a);
  else hipLaunchKernelGGL((k_tokens_down<SMOE_BF16>), down, dim3(512), lds_down, s, a);
  return rc();
}

}  // namespace smoe

// Microscaled 4-bit products of decode steps, short prompts and middle sizes:
// operands, scales among them, as the user's tensors hold them, through LDS.
#include "smoe_common.hpp"
#include "smoe_internal.hpp"
#include "smoe_mxfp4_dev.hpp"

namespace smoe {

int device_cus();

namespace {

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

// BM rows x BN weight rows a workgroup (SwiGLU: BN / 2 gate channels and the
// up channels of the same outputs), 256 k (128 bytes of codes and 8 of scales a
// row) a stage through an LDS ring of NS stages filled by DMA.  WM x WN waves,
// wave tile BM / WM rows x BN / WN weight rows (SwiGLU: half gate, half up).
// The matrix instruction takes the scales beside the codes, so a stage is 2
// instructions for each 16 x 16 tile straight into the f32 accumulators.
//
// A lane's 32 codes and their scale: the instruction wants lane q = l / 16 to
// hold one block of each row; with blocks 2 q and 2 q + 1 of a stage in its two
// steps the two scales are neighbours, one 16-bit LDS read whose bytes the two
// instructions name.  The DMA puts block 2 q at chunk q and 2 q + 1 at q + 4, so
// that the fragment reads keep the conflict-free pattern of 128-byte rows.
//
// The weights' bytes and the stages' latency bound it: 777 tokens, 4 of 32 experts of
// 1024 x 1408 (GELU) 14.4 us the up product and 11-14 the down one, 23 MB of weights
// each; 200 x 1000 -> 2800 5.9 us.
template <int EPI, int ODT, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_gemm_mx_mid(const MxGemm p) {
  constexpr bool SWIGLU = EPI == MX_UP_SWIGLU, UP = EPI == MX_UP_GELU || SWIGLU;
  constexpr int NW = WM * WN, CH = SWIGLU ? BN / 2 : BN, CHW = CH / WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static_assert(TM % 16 == 0 && TN % (SWIGLU ? 64 : 32) == 0, "whole blocks of 32 channels a wave");
  constexpr int XB = BM * 128, WB = BN * 128, SB = (BM + BN) * 8, STAGE = XB + WB + SB;
  constexpr int XI = BM / 8, WI = BN / 8, SI = SB / 256;  // DMA instructions of a stage (fewer than waves: some load the same)
  constexpr int X_LD = (XI + NW - 1) / NW, W_LD = (WI + NW - 1) / NW, S_LD = (SI + NW - 1) / NW, LD = X_LD + W_LD + S_LD;
  static_assert((XI % NW == 0 || NW % XI == 0) && (WI % NW == 0 || NW % WI == 0) && SB % 256 == 0, "whole DMA instructions");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * STAGE];
  int g, m0, mrows, n0;
  if (!block_tile<BM, CH>(p, blockIdx.x, g, m0, mrows, n0)) return;  // uniform
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int nb = (p.K + kMxBlock - 1) / kMxBlock, KS = (nb + 7) / 8, nd = (nb + 3) / 4;

  // the weight row of row r of the tile
  auto wrow = [&](int r) {
    const int w = r / TN, t = r % TN;
    const int ch = SWIGLU ? n0 + CHW * w + t % CHW : n0 + r;
    return static_cast<int64_t>(min(ch, p.N_out - 1)) + (SWIGLU && t >= CHW ? p.N_out : 0);
  };
  auto xrow = [&](int r) {  // rows past the end: a valid one, never stored
    const int pr = m0 + min(r, mrows - 1);
    return static_cast<int64_t>(p.a_rows ? p.a_rows[pr] : pr);
  };
  // DMA sources: lane i of instruction j loads 16 bytes of row 8 j + i / 8, the
  // block that belongs at the chunk the swizzle puts at i % 8 (the same one for
  // every instruction of a wave: their rows are a multiple of 16 apart, or it
  // has one)
  static_assert(8 * NW % 16 == 0, "one chunk per lane");
  const int cl = sw_chunk<8>(8 * wave + (lane >> 3), lane & 7);
  const int blk = 2 * (cl & 3) + (cl >> 2);
  const uint8_t* xsrc[X_LD];
  const uint8_t* wsrc[W_LD];
  const uint8_t* ssrc[S_LD];
#pragma unroll
  for (int j = 0; j < X_LD; ++j) xsrc[j] = p.X + xrow(8 * ((NW * j + wave) % XI) + (lane >> 3)) * p.ldx;
#pragma unroll
  for (int j = 0; j < W_LD; ++j) wsrc[j] = p.W + g * p.w_gstride + wrow(8 * ((NW * j + wave) % WI) + (lane >> 3)) * p.ldw;
#pragma unroll
  for (int j = 0; j < S_LD; ++j) {  // 32 rows' two words of scales an instruction, X's rows before W's
    const int r = 32 * ((NW * j + wave) % SI) + (lane >> 1);
    ssrc[j] = r < BM ? p.xs + xrow(r) * p.ld_xs : p.ws + g * p.ws_gstride + wrow(r - BM) * p.ld_ws;
  }
  // DMA d of stage s; what lies past K is the row's first chunk or word instead, cut before use
  auto issue = [&](int s) {
    uint8_t* base = ring + (s % NS) * STAGE;
    const int at = 8 * s + blk < nb ? (8 * s + blk) * 16 : 0;
    const int sat = 2 * s + (lane & 1) < nd ? (2 * s + (lane & 1)) * 4 : 0;
#pragma unroll
    for (int d = 0; d < X_LD; ++d)
      __builtin_amdgcn_global_load_lds((gbl_vptr)(xsrc[d] + at), (lds_vptr)(base + (NW * d + wave) % XI * 1024), 16, 0, 0);
#pragma unroll
    for (int d = 0; d < W_LD; ++d)
      __builtin_amdgcn_global_load_lds((gbl_vptr)(wsrc[d] + at), (lds_vptr)(base + XB + (NW * d + wave) % WI * 1024), 16, 0, 0);
#pragma unroll
    for (int d = 0; d < S_LD; ++d)
      __builtin_amdgcn_global_load_lds((gbl_vptr)(ssrc[d] + sat), (lds_vptr)(base + XB + WB + (NW * d + wave) % SI * 256), 4, 0, 0);
  };
  const int fr = lane & 15, q = lane >> 4;
  const int flo = fr * 128 + (sw_chunk<8>(fr, q) << 4);  // step h: flo ^ 64 h

  f32x4 acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (s < KS) issue(s);

  auto stage = [&](int s) {
    const uint8_t* sx = ring + (s % NS) * STAGE;
    const uint8_t* ss = sx + XB + WB + 2 * q;
    uint32_t xsc[FM], wsc[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) wsc[j] = *reinterpret_cast<const uint16_t*>(ss + (BM + wn * TN + j * 16 + fr) * 8);
#pragma unroll
    for (int i = 0; i < FM; ++i) xsc[i] = *reinterpret_cast<const uint16_t*>(ss + (wm * TM + i * 16 + fr) * 8);
    auto step = [&](auto h) {
      constexpr int H = decltype(h)::value;
      u32x4 w[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) w[j] = *reinterpret_cast<const u32x4*>(sx + XB + (wn * TN + j * 16) * 128 + (flo ^ (64 * H)));
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(sx + (wm * TM + i * 16) * 128 + (flo ^ (64 * H)));
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[j][i] = mx_mfma<H>(w[j], wsc[j], x, xsc[i], acc[j][i]);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
  };
  // The last stage of a K that ends inside it: code 0 for what lies past K in
  // the rows, and scale 1 in both operands (a byte of another row may be NaN).
  // The weights' codes there may be anything: none of them is NaN.
  auto cut = [&](int s) {
    const int left = nb - 8 * s;
    if (left >= 8) return;  // uniform
    uint8_t* base = ring + (s % NS) * STAGE;
    const int per = 8 - left;
    for (int e = tid; e < BM * per; e += NW * 64) {
      const int r = e / per, b = left + e % per;
      *reinterpret_cast<u32x4*>(base + r * 128 + (sw_chunk<8>(r, (b >> 1) | (b & 1) << 2) << 4)) = u32x4{0u, 0u, 0u, 0u};
    }
    for (int e = tid; e < (BM + BN) * per; e += NW * 64) base[XB + WB + e / per * 8 + left + e % per] = 127;
    lds_barrier();
  };
  // own part of a stage landed (the later ones may be on their way); after the
  // barrier everybody's, and nobody reads the stage before any more
  if (KS >= NS) wait_vmcnt<(NS - 1) * LD>();
  else wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  cut(0);
  stage(0);
  int s = 1;
  for (; s - 1 + NS < KS; ++s) {
    wait_vmcnt<(NS - 2) * LD>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    issue(s - 1 + NS);
    stage(s);
  }
  for (; s < KS; ++s) {
    wait_vmcnt<0>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    cut(s);
    stage(s);
  }

  // epilogue: lane holds channels 4 q + v of row fr of each 16 x 16 tile
  const float* bias = p.bias ? p.bias + g * p.bias_gstride : nullptr;
  if constexpr (UP) {
    // a block of 32 channels is two tiles of one wave: its amax by the four
    // lanes of a row; codes and scales leave through the ring in whole rows
    constexpr int JN = SWIGLU ? FN / 2 : FN, CPR = CH / 32;  // 16-byte chunks (blocks) a row
    static_assert(BM * CH / 2 + BM * CPR <= NS * STAGE, "staging in the ring");
    uint8_t* stg = ring;
    uint8_t* sst = ring + BM * (CH / 2);
    __syncthreads();  // every wave is done with the ring
#pragma unroll
    for (int b = 0; b < JN / 2; ++b) {
      const int c = n0 + CHW * wn + 32 * b;
      float bb[2][4] = {};
      if (bias && c < p.N_out) {  // uniform: N_out % 32 == 0
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) bb[j][v] = bias[c + 16 * j + 4 * q + v];
      }
      const int cb = wn * (CHW / 32) + b;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        float y[2][4];
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if constexpr (SWIGLU) y[j][v] = silu(acc[2 * b + j][i][v]) * (acc[JN + 2 * b + j][i][v] + bb[j][v]);
            else y[j][v] = gelu_tail(acc[2 * b + j][i][v] + bb[j][v]);
            m = __builtin_elementwise_maximum(m, fabsf(y[j][v]));  // a NaN stays
          }
        const int byte = mx_scale_byte(quarters_max(__float_as_uint(m) & 0x7FFFFFFFu));
        const int r = wm * TM + i * 16 + fr;
        uint8_t* to = stg + r * (CH / 2) + (sw_chunk<CPR>(r, cb) << 4) + 2 * q;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<uint16_t*>(to + 8 * j) = static_cast<uint16_t>(mx_codes4(y[j][0], y[j][1], y[j][2], y[j][3], byte));
        if (q == 0) sst[r * CPR + cb] = static_cast<uint8_t>(byte);
      }
    }
    __syncthreads();
    uint8_t* out = static_cast<uint8_t*>(p.out);
    for (int e = tid; e < BM * CPR; e += NW * 64) {
      const int r = e / CPR, c = e % CPR;
      if (r < mrows && n0 + 32 * c < p.N_out) {
        *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(m0 + r) * p.ldo + n0 / 2 + 16 * c) =
            *reinterpret_cast<const u32x4*>(stg + r * (CH / 2) + (sw_chunk<CPR>(r, c) << 4));
        p.out_scale[static_cast<int64_t>(m0 + r) * p.ld_os + n0 / 32 + c] = sst[r * CPR + c];
      }
    }
  } else {
    float b4[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int n = n0 + wn * TN + j * 16 + 4 * q + v;
        b4[j][v] = (bias && n < p.N_out) ? bias[n] : 0.f;
      }
    auto value = [&](int j, int i, float rs, float (&o)[4]) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float y = acc[j][i][v] + b4[j][v];
        o[v] = EPI == MX_GELU ? gelu_tail(y) : (EPI == MX_DOWN ? y * rs : y);
      }
    };
    // whole 16-byte chunks: the tile is staged in the ring (chunk c of row r at
    // c ^ (r & 7)) and leaves in whole rows
    constexpr int EB = ODT == SMOE_F32 ? 4 : 2, CPR = BN * EB / 16;
    constexpr int PASS = BM * BN * EB <= NS * STAGE ? 1 : 2, FP = FM / PASS, TP = TM / PASS;
    static_assert(BM / PASS * BN * EB <= NS * STAGE && FM % PASS == 0, "staging in the ring");
    const bool whole = (static_cast<int64_t>(p.N_out) * EB) % 16 == 0 && (p.ldo * EB) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    if (whole) {
#pragma unroll
      for (int h = 0; h < PASS; ++h) {
        __syncthreads();  // every wave is done with the ring (or the pass before)
#pragma unroll
        for (int i = h * FP; i < (h + 1) * FP; ++i) {
          const int r = wm * TM + i * 16 + fr, lr = wm * TP + (i - h * FP) * 16 + fr;
          const float rs = EPI == MX_DOWN ? p.row_scale[m0 + min(r, mrows - 1)] : 1.f;
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            float o[4];
            value(j, i, rs, o);
            const int c4 = wn * (TN / 4) + j * 4 + q;  // group of four channels
            if constexpr (ODT == SMOE_F32)
              *reinterpret_cast<f32x4*>(ring + (lr * CPR + (c4 ^ (lr & 7))) * 16) = f32x4{o[0], o[1], o[2], o[3]};
            else
              *reinterpret_cast<u32x2*>(ring + (lr * CPR + ((c4 >> 1) ^ (lr & 7))) * 16 + (c4 & 1) * 8) =
                  u32x2{pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3])};
          }
        }
        __syncthreads();
        for (int e = tid; e < BM / PASS * CPR; e += NW * 64) {
          const int lr = e / CPR, c = e % CPR;
          const int r = lr / TP * TM + h * FP * 16 + lr % TP;
          if (r < mrows && n0 + c * (16 / EB) < p.N_out) {
            u32x4* to = reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p.out) + ((m0 + static_cast<int64_t>(r)) * p.ldo + n0) * EB + c * 16);
            const u32x4 o = *reinterpret_cast<const u32x4*>(ring + (lr * CPR + (c ^ (lr & 7))) * 16);
            if constexpr (EPI == MX_DOWN) __builtin_nontemporal_store(o, to);
            else *to = o;
          }
        }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = wm * TM + i * 16 + fr;
        if (r >= mrows) continue;
        float o[4];
        value(j, i, EPI == MX_DOWN ? p.row_scale[m0 + r] : 1.f, o);
        store4<ODT>(p, m0 + r, n0 + wn * TN + j * 16 + 4 * q, o);
      }
  }
}

template <int EPI, int ODT, int BM, int BN, int WM, int WN, int NS>
int go_tile(const MxGemm& a, hipStream_t s) {
  constexpr int CH = EPI == MX_UP_SWIGLU ? BN / 2 : BN;
  const int rows = a.G > 0 ? a.max_rows : a.single_rows;
  // at most one partly filled row tile for every group with rows
  const int64_t tiles = (static_cast<int64_t>(rows) + BM - 1) / BM + (a.G > 0 ? std::min(a.G, rows) : 0);
  const int64_t grid = tiles * ((static_cast<int64_t>(a.N_out) + CH - 1) / CH);
  if (grid * 64 * WM * WN > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  if (a.dry) return SMOE_OK;
  SMOE_LAUNCH((k_gemm_mx_mid<EPI, ODT, BM, BN, WM, WN, NS>), dim3(static_cast<unsigned>(grid)),
              dim3(64 * WM * WN), 0, s, a);
  return rc();
}

// Tiles of BM rows and CH channels: over groups, as if the rows were spread
// evenly (the host does not know the counts).
int64_t tiles_of(const MxGemm& a, int BM, int CH) {
  const int64_t strips = (static_cast<int64_t>(a.N_out) + CH - 1) / CH;
  if (a.G == 0) return (static_cast<int64_t>(a.single_rows) + BM - 1) / BM * strips;
  const int64_t per = (static_cast<int64_t>(a.max_rows) + a.G - 1) / a.G;
  return std::min(a.G, a.max_rows) * ((per + BM - 1) / BM) * strips;
}

// 32 x 64 tiles where they leave no CU a second one, 64 x 64 up to four for a CU.
// Whole products with the activations' quantizer, us, in a graph: 100 x 1000 ->
// 2800 6.7 (two waves a tile 7.1; three stages 6.9), 30 x 2048 -> 1408 7.4 (8.1);
// 200 x 1000 -> 2800 7.4 on 64 x 64 and 8.4 on 64 x 128, 777 x 2816 -> 1024 10.8
// and 13.0, 1500 x 1024 -> 1408 10.1 and 10.7 on 128 x 128.
template <int EPI, int ODT>
int go_dense(const MxGemm& a, hipStream_t s) {
  const int64_t cus = device_cus();
  if (tiles_of(a, 32, 64) <= cus) return go_tile<EPI, ODT, 32, 64, 2, 2, 4>(a, s);
  if (tiles_of(a, 64, 64) <= 4 * cus) return go_tile<EPI, ODT, 64, 64, 2, 2, 3>(a, s);
  return go_tile<EPI, ODT, 128, 128, 2, 2, 2>(a, s);
}

// 128 weight rows a tile (SwiGLU: 64 channels; 256 rows on eight waves left fewer
// workgroups: 800 tokens over 16 experts of 1024 x 2816 37 us for both products and
// the plan, 41.4 before), two stages (the third takes LDS from a workgroup beside:
// 1024 tokens over 64 experts of 2048 x 1408 59.6 and 64.6), and rows by the groups'
// average: 32 up to 56 (400 tokens over 32 experts of 1024 x 1408, 50 rows, 29.6;
// on 64 rows 32.1), 64 up to 112 (777 tokens, 97 rows, 36.6; on 128 rows 42.3, on
// 32 rows 48.0), 128 (1500 tokens over 16 SwiGLU experts, 188 rows, 50.6; on 64
// rows 58.8), fewer where those tiles do not give every CU one.
template <int EPI>
int go_grouped(const MxGemm& a, hipStream_t s) {
  constexpr int O = SMOE_F32, CH = EPI == MX_UP_SWIGLU ? 64 : 128;
  const int64_t cus = device_cus(), per = (static_cast<int64_t>(a.max_rows) + a.G - 1) / a.G;
  int BM = per <= 56 ? 32 : (per <= 112 ? 64 : 128);
  while (BM > 32 && tiles_of(a, BM, CH) < cus) BM /= 2;
  if (BM == 32) return go_tile<EPI, O, 32, 128, 2, 2, 2>(a, s);
  if (BM == 64) return go_tile<EPI, O, 64, 128, 2, 2, 2>(a, s);
  return go_tile<EPI, O, 128, 128, 2, 2, 2>(a, s);
}

}  // namespace

int launch_gemm_mx_mid(const MxGemm& a, hipStream_t s) {
  if (a.ws_plane || a.ld_ws % 4 || a.ld_xs % 4) return SMOE_EINVAL;
  const bool f32 = a.out_dtype == SMOE_F32;
  switch (a.epi) {
    case MX_LINEAR: return f32 ? go_dense<MX_LINEAR, SMOE_F32>(a, s) : go_dense<MX_LINEAR, SMOE_BF16>(a, s);
    case MX_GELU: return f32 ? go_dense<MX_GELU, SMOE_F32>(a, s) : go_dense<MX_GELU, SMOE_BF16>(a, s);
    case MX_UP_GELU: return go_grouped<MX_UP_GELU>(a, s);
    case MX_UP_SWIGLU: return go_grouped<MX_UP_SWIGLU>(a, s);
    case MX_DOWN: return go_grouped<MX_DOWN>(a, s);
    default: return SMOE_EINVAL;
  }
}

}  // namespace smoe

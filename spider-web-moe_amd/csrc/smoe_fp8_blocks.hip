// Block-scaled fp8: the quantizer (e4m3 codes with one f32 scale per 1 x 128
// or 128 x 128 block) and the products on such operands, dense and grouped by
// expert.
#include "smoe_common.hpp"
#include "smoe_fp8_blocks_dev.hpp"
#include "smoe_internal.hpp"

namespace smoe {
namespace {

// 1 x 128 blocks (quant_row_block), sixteen a workgroup.
template <int XDT>
__global__ __launch_bounds__(256) void k_quant_row_blocks(const BlockQuant q, int nblk, int64_t total) {
  quant_row_block<XDT>(q, nblk, total, (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4,
                       threadIdx.x & 15);
}

// 128 x 128 blocks: a workgroup holds a block, thread t the columns
// 8 (t % 16) .. + 7 of rows t / 16, t / 16 + 16, ..
template <int XDT>
__global__ __launch_bounds__(256) void k_quant_square_blocks(const BlockQuant q, int rblk, int nblk) {
  __shared__ float red[4];
  const int kb = blockIdx.x % nblk;
  const int64_t grb = blockIdx.x / nblk;  // group * row blocks + row block
  const int64_t g = grb / rblk;
  const int r0 = static_cast<int>(grb - g * rblk) * kFp8Block;
  const int c = kb * kFp8Block + 8 * (threadIdx.x & 15);
  const bool vec = (reinterpret_cast<uintptr_t>(q.x) | static_cast<uintptr_t>(q.ldx * elt_bytes<XDT>())) % 16 == 0;
  float v[8][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + (threadIdx.x >> 4) + 16 * i;
    const char* rp = reinterpret_cast<const char*>(q.x) + (g * q.rows + min(r, q.rows - 1)) * q.ldx * elt_bytes<XDT>();
    load_cols8<XDT>(rp, c, r < q.rows ? q.cols : 0, vec, v[i]);
    m = nan_max(m, amax8(v[i]));
  }
  m = row16_nan_max(m);
  m = nan_max(m, __shfl_xor(m, 16));
  m = nan_max(m, __shfl_xor(m, 32));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const float sc = block_scale(nan_max(nan_max(red[0], red[1]), nan_max(red[2], red[3])));
  if (threadIdx.x == 0) q.scale[grb * q.s_row + kb * q.s_col] = sc;
  if (c >= q.ld_out) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + (threadIdx.x >> 4) + 16 * i;
    if (r < q.rows)
      *reinterpret_cast<u32x2*>(q.codes + (g * q.rows + r) * q.ld_out + c) = codes8(v[i], sc);
  }
}

// ------------------------------------------------------------------ GEMM ----
// 128 rows x 128 output channels a workgroup (SwiGLU: 128 gate and the 128
// up channels of the same outputs), K one block of 128 a stage through a
// two-stage LDS ring filled by DMA; wave tile 64 x 64 channels (SwiGLU 32
// gate + 32 up).  A block's products are summed by the matrix instruction
// from zero and enter the f32 accumulators times the block's two scales.
//
// The f8f6f4 instruction sums a block below f32 precision (measured on normal
// codes: 1.5e-5 of the sum, 1 / 100 of a bf16 rounding), which suits outputs
// of 8 to 16 bits.  WIDE (f32 outputs): the codes are widened to bf16, exactly,
// and multiplied at a quarter of the rate with f32 sums.
template <int EPI, int ODT, bool WIDE>
__global__ __launch_bounds__(EPI == BLK_UP_SWIGLU ? 512 : 256, 2) void k_gemm_blocks(const BlockGemm p) {
  constexpr bool SWIGLU = EPI == BLK_UP_SWIGLU, UP = EPI == BLK_UP_GELU || SWIGLU;
  constexpr int BM = 128, BN = 128, WN = SWIGLU ? 4 : 2, NW = 2 * WN, WROWS = 64 * WN;
  constexpr int NS = 2, XB = BM * 128, WB = WROWS * 128, SCB = BM * 4, STAGE = XB + WB + SCB;
  constexpr int X_LD = BM / 8 / NW, W_LD = WROWS / 8 / NW;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * STAGE];
  int g, m0, mrows, n0;
  if (!block_tile<BM, BN>(p, blockIdx.x, g, m0, mrows, n0)) return;  // uniform
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int KB = (p.K + 127) / 128;

  // DMA sources: lane i of instruction j loads 16 bytes of row
  // 8 (NW j + wave) + i / 8, the chunk that the swizzle puts at i % 8
  const uint8_t* xsrc[X_LD];
  const uint8_t* wsrc[W_LD];
  int xc[X_LD], wc[W_LD];
#pragma unroll
  for (int j = 0; j < X_LD; ++j) {
    const int r = 8 * (NW * j + wave) + (lane >> 3);
    const int pr = m0 + min(r, mrows - 1);  // rows past the tile's end: a valid row, never stored
    xc[j] = 16 * sw_chunk<8>(r, lane & 7);
    xsrc[j] = p.X + static_cast<int64_t>(p.a_rows ? p.a_rows[pr] : pr) * p.ldx;
  }
#pragma unroll
  for (int j = 0; j < W_LD; ++j) {
    const int r = 8 * (NW * j + wave) + (lane >> 3);
    const int ch = SWIGLU ? n0 + 32 * (r >> 6) + (r & 31) : n0 + r;
    const int64_t row = min(ch, p.N_out - 1) + (SWIGLU && (r & 32) ? p.N_out : 0);
    wc[j] = 16 * sw_chunk<8>(r, lane & 7);
    wsrc[j] = p.W + g * p.w_gstride + row * p.ldw;
  }
  // the rows' scales: waves of even number load rows 0-63, of odd number 64-127
  const int sr = 64 * (wave & 1) + lane;
  const int spr = m0 + min(sr, mrows - 1);
  const float* ssrc = p.xs + static_cast<int64_t>(p.a_rows ? p.a_rows[spr] : spr) * p.xs_row;
  auto issue = [&](int s) {
    uint8_t* base = ring + (s % NS) * STAGE;
    const int k0 = s * 128;
#pragma unroll
    for (int j = 0; j < X_LD; ++j)  // chunks past K: the row's first one, cut before use
      __builtin_amdgcn_global_load_lds((gbl_vptr)(xsrc[j] + (k0 + xc[j] < p.K ? k0 + xc[j] : 0)),
                                       (lds_vptr)(base + (NW * j + wave) * 1024), 16, 0, 0);
#pragma unroll
    for (int j = 0; j < W_LD; ++j)
      __builtin_amdgcn_global_load_lds((gbl_vptr)(wsrc[j] + (k0 + wc[j] < p.K ? k0 + wc[j] : 0)),
                                       (lds_vptr)(base + XB + (NW * j + wave) * 1024), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((gbl_vptr)(ssrc + s * p.xs_col),
                                     (lds_vptr)(base + XB + WB + 256 * (wave & 1)), 4, 0, 0);
  };
  const int fr = lane & 15, q = lane >> 4;
  auto frag = [&](const uint8_t* op, int r) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(op + r * 128 + (sw_chunk<8>(r, 2 * q) << 4));
    const u32x4 hi = *reinterpret_cast<const u32x4*>(op + r * 128 + (sw_chunk<8>(r, 2 * q + 1) << 4));
    return __builtin_bit_cast(i32x8, (uint32_t __attribute__((ext_vector_type(8)))){
                                         lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
  };

  f32x4 acc[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* wsp = p.ws + g * p.ws_gstride + static_cast<int64_t>(n0 / 128) * KB;
  const float* wsp_up = wsp + static_cast<int64_t>((p.N_out + 127) / 128) * KB;  // SwiGLU

  issue(0);
  for (int s = 0; s < KB; ++s) {
    // own part of stage s landed; after the barrier everybody's, and nobody
    // reads stage s - 1 any more
    wait_vmcnt<0>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    if (s + 1 < KB) issue(s + 1);  // into the slot of stage s - 1
    const uint8_t* sx = ring + (s % NS) * STAGE;
    const float* sc = reinterpret_cast<const float*>(sx + XB + WB) + wm * 64;
    i32x8 xf[4], wf[4];
    float xsv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xf[i] = frag(sx, wm * 64 + i * 16 + fr);
      xsv[i] = sc[i * 16 + fr];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) wf[j] = frag(sx + XB, wn * 64 + j * 16 + fr);
    const int left = p.K - s * 128;
    if (left < 128) {  // uniform: the last stage of a ragged K
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xf[i] = cut_frag(xf[i], left - 32 * q);
        wf[i] = cut_frag(wf[i], left - 32 * q);
      }
    }
    const float w0 = wsp[s], w1 = SWIGLU ? wsp_up[s] : 0.f;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if constexpr (WIDE) {
      bf16x8 xw[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) widen_frag(xf[i], xw[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 ww[4];
        widen_frag(wf[j], ww);
        const float wsc = SWIGLU && j >= 2 ? w1 : w0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 part = zero;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[u], xw[i][u], part, 0, 0, 0);
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[j][i][v] = fmaf(part[v], xsv[i] * wsc, acc[j][i][v]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float wsc = SWIGLU && j >= 2 ? w1 : w0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf[i], zero, 0, 0, 0,
                                                                              0, 0, 0);
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[j][i][v] = fmaf(part[v], xsv[i] * wsc, acc[j][i][v]);
        }
      }
    }
  }

  // epilogue: lane holds channels 4 q + v of row fr of each 16 x 16 tile
  const float* bias = p.bias ? p.bias + g * p.bias_gstride : nullptr;
  if constexpr (UP) {
    // activations of 128 channels: amax per row over the wave's channels, then
    // over the waves of the row through LDS; codes staged in the ring
    constexpr int JN = SWIGLU ? 2 : 4;
    const int cw = SWIGLU ? 32 * wn : 64 * wn;  // the wave's first channel of the 128
    float* red = reinterpret_cast<float*>(ring);  // [WN][BM]
    uint8_t* stg = ring + WN * BM * 4;            // [BM][128], 16-byte chunks swizzled by row
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = 0.f;
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int c = cw + j * 16 + 4 * q;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const bool in = n0 + c + v < p.N_out;
        const float b = bias && in ? bias[n0 + c + v] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y;
          if constexpr (SWIGLU) y = silu(acc[j][i][v]) * (acc[j + 2][i][v] + b);
          else y = gelu_erf(acc[j][i][v] + b);
          y = in ? y : 0.f;
          acc[j][i][v] = y;
          m[i] = nan_max(m[i], fabsf(y));
        }
      }
    }
    __syncthreads();  // every wave is done with the ring
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = nan_max(m[i], __shfl_xor(m[i], 16));
      m[i] = nan_max(m[i], __shfl_xor(m[i], 32));
      if (q == 0) red[wn * BM + wm * 64 + i * 16 + fr] = m[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = wm * 64 + i * 16 + fr;
      float a = red[r];
#pragma unroll
      for (int w = 1; w < WN; ++w) a = nan_max(a, red[w * BM + r]);
      const float sc = block_scale(a);
      if (wn == 0 && q == 0 && r < mrows) p.out_scale[(n0 / 128) * p.os_col + m0 + r] = sc;
#pragma unroll
      for (int j = 0; j < JN; ++j) {
        const int c = cw + j * 16 + 4 * q;
        *reinterpret_cast<uint32_t*>(stg + r * 128 + (((c >> 4) ^ (r & 7)) << 4) + (c & 15)) =
            pack_e4m3(__fdiv_rn(acc[j][i][0], sc), __fdiv_rn(acc[j][i][1], sc),
                      __fdiv_rn(acc[j][i][2], sc), __fdiv_rn(acc[j][i][3], sc));
      }
    }
    __syncthreads();
    uint8_t* out = reinterpret_cast<uint8_t*>(p.out);
    for (int e = tid; e < BM * 8; e += NW * 64) {
      const int r = e >> 3, c = e & 7;
      if (r < mrows && n0 + 16 * c < p.N_out)  // N_out % 16 == 0: whole chunks
        *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(m0 + r) * p.ldo + n0 + 16 * c) =
            *reinterpret_cast<const u32x4*>(stg + r * 128 + ((c ^ (r & 7)) << 4));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + wn * 64 + j * 16 + 4 * q;
      float b4[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) b4[v] = (bias && n + v < p.N_out) ? bias[n + v] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = wm * 64 + i * 16 + fr;
        if (r >= mrows) continue;
        float o[4];
        const float rs = EPI == BLK_DOWN ? p.row_scale[m0 + r] : 1.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float y = acc[j][i][v] + b4[v];
          o[v] = EPI == BLK_GELU ? gelu_erf(y) : (EPI == BLK_DOWN ? y * rs : y);
        }
        store4<ODT>(p, m0 + r, n, o);
      }
    }
  }
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

}  // namespace

int launch_quantize_fp8_blocks(const BlockQuant& q, hipStream_t s) {
  if (q.groups < 0 || q.rows < 0 || q.cols < 1 || q.ldx < q.cols || q.ld_out < q.cols || q.ld_out % 16 ||
      reinterpret_cast<uintptr_t>(q.codes) % 16 || (q.block_rows != 1 && q.block_rows != kFp8Block))
    return SMOE_EINVAL;
  if (q.groups == 0 || q.rows == 0) return SMOE_OK;
  const int nblk = fp8_blocks_of(q.cols), rblk = fp8_blocks_of(q.rows);
  if (q.ld_out > static_cast<int64_t>(nblk) * kFp8Block) return SMOE_EINVAL;
  const bool square = q.block_rows != 1;
  const int64_t total = square ? static_cast<int64_t>(q.groups) * rblk * nblk
                               : static_cast<int64_t>(q.groups) * q.rows * nblk;
  const int64_t wgs = square ? total : (total + 15) / 16;
  if (wgs > 0x7fffffff) return SMOE_EINVAL;
  return by_xdt(q.x_dtype, [&](auto xd) {
    constexpr int XD = decltype(xd)::value;
    if (square)
      hipLaunchKernelGGL((k_quant_square_blocks<XD>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, s, q, rblk, nblk);
    else
      hipLaunchKernelGGL((k_quant_row_blocks<XD>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, s, q, nblk, total);
    return rc();
  });
}

int launch_gemm_fp8_blocks(const BlockGemm& a, hipStream_t s) {
  const int rows = a.G > 0 ? a.max_rows : a.single_rows;
  if (rows <= 0) return SMOE_OK;
  if (a.K < 1 || a.N_out < 1 || a.ldx < a.K || a.ldw < a.K || a.ldx % 16 || a.ldw % 16 || a.w_gstride % 16)
    return SMOE_EINVAL;
  if (gemm_blocks_few_fits(a)) return launch_gemm_blocks_few(a, s);
  if (a.x_float) return SMOE_EINVAL;
  // at most one partly filled row tile for every group with rows
  const int64_t tiles = (rows + 127) / 128 + (a.G > 0 ? std::min(a.G, rows) : 0);
  const int64_t grid = tiles * ((a.N_out + 127) / 128);
  if (grid > 0x7fffffff) return SMOE_EINVAL;
  auto go = [&](auto epi, auto odt, auto wide) {
    constexpr int EPI = decltype(epi)::value;
    SMOE_LAUNCH((k_gemm_blocks<EPI, decltype(odt)::value, decltype(wide)::value>),
                dim3(static_cast<unsigned>(grid)), dim3(EPI == BLK_UP_SWIGLU ? 512 : 256), 0, s, a);
    return rc();
  };
  using F = std::integral_constant<int, SMOE_F32>;
  using B = std::integral_constant<int, SMOE_BF16>;
  using T = std::true_type;
  using N = std::false_type;
  const bool f32 = a.out_dtype == SMOE_F32;
  switch (a.epi) {
    case BLK_LINEAR: {
      using E = std::integral_constant<int, BLK_LINEAR>;
      return f32 ? go(E{}, F{}, T{}) : go(E{}, B{}, N{});
    }
    case BLK_GELU: {
      using E = std::integral_constant<int, BLK_GELU>;
      return f32 ? go(E{}, F{}, T{}) : go(E{}, B{}, N{});
    }
    case BLK_UP_GELU: return go(std::integral_constant<int, BLK_UP_GELU>{}, F{}, N{});
    case BLK_UP_SWIGLU: return go(std::integral_constant<int, BLK_UP_SWIGLU>{}, F{}, N{});
    case BLK_DOWN: return go(std::integral_constant<int, BLK_DOWN>{}, F{}, N{});
    default: return SMOE_EINVAL;
  }
}

}  // namespace smoe

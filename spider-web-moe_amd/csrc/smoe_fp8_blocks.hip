// Block-scaled fp8: the quantizer (e4m3 codes with one f32 scale per 1 x 128
// or 128 x 128 block) and the products on such operands, dense and grouped by
// expert.
#include "smoe_common.hpp"
#include "smoe_fp8_blocks_dev.hpp"
#include "smoe_internal.hpp"

namespace smoe {

int device_cus();

namespace {

// 1 x 128 blocks (quant_row_block), sixteen a workgroup, a block's 128 columns
// by 16 lanes in one load each.  Bound by the bytes: bf16 16384 x 1024 in 12.8
// us, 51 MB at 4.0 TB/s.
template <int XDT>
__global__ __launch_bounds__(256) void k_quant_row_blocks(const BlockQuant q, int nblk, int64_t total) {
  quant_row_block<XDT>(q, nblk, total, (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4,
                       threadIdx.x & 15);
}

// 128 x 128 blocks: a workgroup holds a block in registers (one read, one
// write), thread t the columns 8 (t % 16) .. + 7 of rows t / 16, t / 16 + 16, ..
// Bound by the bytes: bf16 16384 x 2816, 138 MB, one call after another 26.8 us
// at 5.2 TB/s (30.8 with plain stores).
template <int XDT>
__global__ __launch_bounds__(256) void k_quant_square_blocks(const BlockQuant q, int rblk, int nblk) {
  __shared__ uint32_t red[4];
  const int kb = blockIdx.x % nblk;
  const uint32_t grb = blockIdx.x / nblk;  // group * row blocks + row block
  const int64_t g = grb / static_cast<uint32_t>(rblk);
  const int r0 = static_cast<int>(grb - g * rblk) * kFp8Block;
  const int c = kb * kFp8Block + 8 * (threadIdx.x & 15);
  const bool vec = (reinterpret_cast<uintptr_t>(q.x) | static_cast<uintptr_t>(q.ldx * elt_bytes<XDT>())) % 16 == 0;
  float v[8][8];
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + (threadIdx.x >> 4) + 16 * i;
    const char* rp = reinterpret_cast<const char*>(q.x) + (g * q.rows + min(r, q.rows - 1)) * q.ldx * elt_bytes<XDT>();
    load_cols8<XDT>(rp, c, r < q.rows ? q.cols : 0, vec, v[i]);
    m = max(m, amax8(v[i]));
  }
  m = quarters_max(row16_max(m));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const float sc = block_scale(max(max(red[0], red[1]), max(red[2], red[3])));
  if (threadIdx.x == 0) q.scale[grb * q.s_row + kb * q.s_col] = sc;
  if (c >= q.ld_out) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + (threadIdx.x >> 4) + 16 * i;
    if (r < q.rows)  // past the L2s, which would write them back at the kernel's end
      __builtin_nontemporal_store(codes8(v[i], sc), reinterpret_cast<u32x2*>(q.codes + (g * q.rows + r) * q.ld_out + c));
  }
}

// ------------------------------------------------------------------ GEMM ----
// BM rows x BN weight rows a workgroup (SwiGLU: BN / 2 gate channels and the
// up channels of the same outputs), K one block of 128 a stage through an LDS
// ring of NS stages filled by DMA.  WM x WN waves, wave tile BM / WM rows x 64
// weight rows (SwiGLU 32 gate + 32 up).  A block's products are summed by the
// matrix instruction from zero and enter the f32 accumulators times the
// block's two scales.
//
// The f8f6f4 instruction cuts products: of eight neighbouring k each one
// toward zero to a multiple of 2^(e - 13), e the largest sum of two operands'
// exponents among them, so by less than 2^-13 of the eight's largest product;
// the eights are added in f32 (measured with single products beside a large
// one, at every place).  On normal codes that is 1.5e-5 of the sum, 1 / 100 of a
// bf16 rounding; where large products cancel it can be all of it.  It suits
// outputs of 8 to 16 bits, whose operands were themselves rounded by up to 2^-4.
// WIDE (f32 outputs): the codes are widened to bf16, exactly, and multiplied at
// half the rate with f32 sums (16384 x 1024 -> 5632: 265 to 288 us).
//
// 16384 x 1024 -> 5632 in bf16: 118 to 124 us, 1.5 to 1.6 PFLOP/s.  Stages alone
// 86 (a stage of 256 x 256 tiles: 2048 cycles of products beside 1536 of LDS
// reads for its fragments), the output's way through the LDS 15, its stores 20.
template <int EPI, int ODT, bool WIDE, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_gemm_blocks(const BlockGemm p) {
  constexpr bool SWIGLU = EPI == BLK_UP_SWIGLU, UP = EPI == BLK_UP_GELU || SWIGLU;
  constexpr int NW = WM * WN, CH = SWIGLU ? BN / 2 : BN, CHW = CH / WN, TM = BM / WM, FM = TM / 16;
  static_assert(BN == 64 * WN && TM % 16 == 0 && (BM == 32 || BM == 64 || BM == 128 || BM == 256), "wave tile: 64 weight rows");
  static_assert(!UP || CH % 128 == 0, "activations are quantized in blocks of 128 channels");
  constexpr int XB = BM * 128, WB = BN * 128, SR = BM < 64 ? 64 : BM, STAGE = XB + WB + SR * 4;
  constexpr int XI = BM / 8;  // DMA instructions of a stage's rows (fewer than waves: some load the same)
  constexpr int X_LD = (XI + NW - 1) / NW, W_LD = BN / 8 / NW, LD = X_LD + W_LD + 1;
  static_assert((XI % NW == 0 || NW % XI == 0) && W_LD * NW * 8 == BN && NW % (SR / 64) == 0, "whole DMA instructions");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * STAGE];
  int g, m0, mrows, n0;
  if (!block_tile<BM, CH>(p, blockIdx.x, g, m0, mrows, n0)) return;  // uniform
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int KB = (p.K + 127) / 128;

  // DMA sources: lane i of instruction j loads 16 bytes of row
  // 8 (NW j + wave) + i / 8, the chunk cl that the swizzle puts at i % 8 (the
  // same one for every j: 4 NW j is a multiple of 8)
  static_assert(4 * NW % 8 == 0, "one chunk per lane");
  const int cl = 16 * sw_chunk<8>(8 * wave + (lane >> 3), lane & 7);
  const uint8_t* xsrc[X_LD];
  const uint8_t* wsrc[W_LD];
#pragma unroll
  for (int j = 0; j < X_LD; ++j) {
    const int pr = m0 + min(8 * ((NW * j + wave) % XI) + (lane >> 3), mrows - 1);  // rows past the end: a valid one, never stored
    xsrc[j] = p.X + static_cast<int64_t>(p.a_rows ? p.a_rows[pr] : pr) * p.ldx;
  }
#pragma unroll
  for (int j = 0; j < W_LD; ++j) {
    const int r = 8 * (NW * j + wave) + (lane >> 3);
    const int ch = SWIGLU ? n0 + 32 * (r >> 6) + (r & 31) : n0 + r;
    const int64_t row = min(ch, p.N_out - 1) + (SWIGLU && (r & 32) ? p.N_out : 0);
    wsrc[j] = p.W + g * p.w_gstride + row * p.ldw;
  }
  // the rows' scales: wave w loads rows 64 (w % (SR / 64)) .. + 63
  const int sw = wave % (SR / 64);
  const int spr = m0 + min(64 * sw + lane, mrows - 1);
  const float* ssrc = p.xs + static_cast<int64_t>(p.a_rows ? p.a_rows[spr] : spr) * p.xs_row;
  // DMA d of stage s: X_LD of rows, W_LD of weights, one of the rows' scales
  auto issue_one = [&](int s, int d) {
    uint8_t* base = ring + (s % NS) * STAGE;
    const int at = s * 128 + cl < p.K ? s * 128 + cl : 0;  // chunks past K: the row's first one, cut before use
    if (d < X_LD)
      __builtin_amdgcn_global_load_lds((gbl_vptr)(xsrc[d < X_LD ? d : 0] + at), (lds_vptr)(base + (NW * d + wave) % XI * 1024), 16, 0, 0);
    else if (d < X_LD + W_LD)
      __builtin_amdgcn_global_load_lds((gbl_vptr)(wsrc[d >= X_LD && d < X_LD + W_LD ? d - X_LD : 0] + at),
                                       (lds_vptr)(base + XB + (NW * (d - X_LD) + wave) * 1024), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds((gbl_vptr)(ssrc + s * p.xs_col), (lds_vptr)(base + XB + WB + 256 * sw), 4, 0, 0);
  };
  const int fr = lane & 15, q = lane >> 4;
  // fragment of 16 rows from tile row 16 t on: row fr, chunks q and q + 4 (both
  // operands pair the same k, in whatever order); the swizzle is the same for
  // every t.  Chunks 2 q and 2 q + 1 meet in the same banks: a ds_read_b128
  // serves lanes 0-3, 12-15, 20-23, 24-27 together (half the LDS cycles were
  // conflicts).
  const int flo = fr * 128 + (sw_chunk<8>(fr, q) << 4), fhi = flo ^ 64;
  auto frag = [&](const uint8_t* op) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(op + flo);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(op + fhi);
    return __builtin_bit_cast(i32x8, (uint32_t __attribute__((ext_vector_type(8)))){
                                         lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
  };

  f32x4 acc[4][FM];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int nblk = (p.N_out + 127) / 128;
  const int cblk = min((n0 + CHW * wn) / 128, nblk - 1);  // the wave's channels' block of weight scales
  const float* wsp = p.ws + g * p.ws_gstride + static_cast<int64_t>(cblk) * KB;
  const float* wsp_up = wsp + static_cast<int64_t>(nblk) * KB;  // SwiGLU

  // The weight scales of a stage are uniform: scalar loads, a stage ahead.  As
  // vector loads each made the wave wait for every DMA issued before it.
  const uniform_f32 wsc = as_uniform(wsp), wsc_up = as_uniform(wsp_up);
  float nw0 = wsc[0], nw1 = SWIGLU ? wsc_up[0] : 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (s < KB) {
#pragma unroll
      for (int d = 0; d < LD; ++d) issue_one(s, d);
    }
  // A stage's last ROT rows of fragments are multiplied after the barrier that
  // opens the next stage, each weight fragment replaced by the next stage's
  // after its last use: otherwise the matrix unit waits there for the LDS
  // (80 KB at 128 bytes a cycle with 256 x 256 tiles).
  // Step t: TA steps of those rows, weights outside, then the rows before them.
  // Under the product of a step the four multiply-adds that bring the step LAG
  // before into the accumulators and, in the stage's first half, the DMAs of a
  // later one.  (16384 x 1024 -> 5632: DMAs over the
  // whole stage 139, over its first half 132.)
  constexpr int ROT = FM >= 4 ? 2 : 1, TA = 4 * ROT, STEPS = 4 * FM, LAG = 2;
  constexpr bool CARRY = FM > ROT;  // the last steps' multiply-adds go under the next stage's first ones
  i32x8 wf[4], xa[ROT];
  float za0[ROT], za1[ROT], zb0[2], zb1[2];  // the scales of the last ROT rows, of row i before them: [i % 2]
  f32x4 part[4];
  auto product = [&](const i32x8& w, const i32x8& x) {
    f32x4 now = {0.f, 0.f, 0.f, 0.f};
    if constexpr (WIDE) {
      bf16x8 ww[4], xw[4];
      widen_frag(w, ww);
      widen_frag(x, xw);
#pragma unroll
      for (int u = 0; u < 4; ++u) now = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[u], xw[u], now, 0, 0, 0);
    } else {
      now = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, now, 0, 0, 0, 0, 0, 0);
    }
    return now;
  };
  auto add = [&](int t) {
    const int j = t < TA ? t / ROT : t % 4, i = t < TA ? FM - ROT + t % ROT : (t - TA) / 4;
    const float z0 = t < TA ? za0[t % ROT] : zb0[i % 2], z1 = t < TA ? za1[t % ROT] : zb1[i % 2];
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[j][i][v] = fmaf(part[t % 4][v], SWIGLU && j >= 2 ? z1 : z0, acc[j][i][v]);
  };
  // the last ROT rows of the stage before; `fill(j)`: the weights' fragment j is free
  auto last_rows = [&](auto fill, auto dma) {
#pragma unroll
    for (int t = 0; t < TA; ++t) {
      part[t % 4] = product(wf[t / ROT], xa[t % ROT]);
      __builtin_amdgcn_sched_barrier(0);
      if (t % ROT == ROT - 1) fill(t / ROT);
      if (t >= LAG) add(t - LAG);
      else if (CARRY) add(STEPS + t - LAG);
      dma(t);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!CARRY) {
#pragma unroll
      for (int t = TA - LAG; t < TA; ++t) add(t);
    }
  };
  // stage s, whose part of the ring holds for every wave when it is called;
  // `more`: stage s - 1 + NS is requested meanwhile, into the slot of stage s - 1
  auto stage = [&](int s, auto first, auto more) {
    const uint8_t* sx = ring + (s % NS) * STAGE;
    const float* sc = reinterpret_cast<const float*>(sx + XB + WB) + wm * TM + fr;
    const float w0 = nw0, w1 = nw1;
    const int ns = min(s + 1, KB - 1);
    nw0 = wsc[ns];
    if (SWIGLU) nw1 = wsc_up[ns];
    auto xfrag = [&](int i) { return frag(sx + (wm * TM + i * 16) * 128); };
    auto fill = [&](int j) { wf[j] = frag(sx + XB + (wn * 64 + j * 16) * 128); };
    auto dma = [&](int t) {
      if constexpr (decltype(more)::value) {
#pragma unroll
        for (int d = 0; d < LD; ++d)
          if (d * STEPS / (2 * LD) == t) issue_one(s - 1 + NS, d);
      }
    };
    i32x8 xf = xfrag(0);
    float xsv = sc[0];
    if constexpr (decltype(first)::value) {
#pragma unroll
      for (int j = 0; j < 4; ++j) fill(j);
    } else {
      last_rows(fill, dma);
    }
#pragma unroll
    for (int i = 0; i < FM - ROT; ++i) {
      i32x8 nx = xf;
      float nv[ROT];
      if (i + 1 < FM - ROT) {
        nx = xfrag(i + 1);
        nv[0] = sc[(i + 1) * 16];
      } else {
#pragma unroll
        for (int u = 0; u < ROT; ++u) {
          xa[u] = xfrag(FM - ROT + u);
          nv[u] = sc[(FM - ROT + u) * 16];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = TA + 4 * i + j;
        part[t % 4] = product(wf[j], xf);
        __builtin_amdgcn_sched_barrier(0);
        if (t - LAG >= (decltype(first)::value ? TA : 0)) add(t - LAG);
        if (j == LAG - 1) {
          zb0[i % 2] = xsv * w0;
          zb1[i % 2] = xsv * w1;
        }
        dma(t);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i + 1 < FM - ROT) {
        xf = nx;
        xsv = nv[0];
      } else {
#pragma unroll
        for (int u = 0; u < ROT; ++u) {
          za0[u] = nv[u] * w0;
          za1[u] = nv[u] * w1;
        }
      }
    }
    if constexpr (FM == ROT) {
      xa[0] = xf;
      za0[0] = xsv * w0;
      za1[0] = xsv * w1;
    }
  };
  auto cut = [&](int s) {
    if (s == KB - 1 && p.K - s * 128 < 128) {  // uniform: the last stage of a ragged K
      cut_stage(ring + (s % NS) * STAGE, BM + BN, p.K - s * 128, tid, NW * 64);
      lds_barrier();
    }
  };
  // own part of a stage landed (the later ones may be on their way); after the
  // barrier everybody's, and nobody reads the stage before any more.  Two
  // loops: a branch around each DMA made the compiler move the multiply-adds
  // away from the products they should hide under.
  if (KB >= NS) wait_vmcnt<(NS - 1) * LD>();
  else wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  cut(0);
  stage(0, std::true_type{}, std::false_type{});
  int s = 1;
  for (; s - 1 + NS < KB; ++s) {
    wait_vmcnt<(NS - 2) * LD>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    stage(s, std::false_type{}, std::true_type{});
  }
  for (; s < KB; ++s) {
    wait_vmcnt<0>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    cut(s);
    stage(s, std::false_type{}, std::false_type{});
  }
  last_rows([](int) {}, [](int) {});
  if constexpr (CARRY) {
#pragma unroll
    for (int t = TA - LAG; t < TA; ++t) add(t);
  }

  // epilogue: lane holds channels 4 q + v of row fr of each 16 x 16 tile
  const float* bias = p.bias ? p.bias + g * p.bias_gstride : nullptr;
  if constexpr (UP) {
    // amax per row over the wave's channels, then over the waves of a block
    // of 128 channels through LDS; codes staged in the ring
    constexpr int JN = SWIGLU ? 2 : 4, BW = 128 / CHW;  // BW waves share a block
    uint32_t* red = reinterpret_cast<uint32_t*>(ring);     // [WN][BM]
    Divisor* div = reinterpret_cast<Divisor*>(red + WN * BM);  // [CH / 128][BM]
    uint8_t* stg = ring + (WN + 2 * (CH / 128)) * BM * 4;      // [BM][CH], 16-byte chunks swizzled by row
    static_assert((WN + 2 * (CH / 128)) * BM * 4 + BM * CH <= NS * STAGE, "staging in the ring");
    uint32_t m[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) m[i] = 0u;
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int c = n0 + CHW * wn + j * 16;
      if (c < p.N_out) {  // uniform: N_out % 16 == 0
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (bias) {
#pragma unroll
          for (int v = 0; v < 4; ++v) b[v] = bias[c + 4 * q + v];
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float y;
            if constexpr (SWIGLU) y = silu(acc[j][i][v]) * (acc[j + 2][i][v] + b[v]);
            else y = gelu_erf(acc[j][i][v] + b[v]);
            acc[j][i][v] = y;
            m[i] = amax_bits(m[i], y);
          }
      } else {
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    __syncthreads();  // every wave is done with the ring
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      m[i] = quarters_max(m[i]);
      if (q == 0) red[wn * BM + wm * TM + i * 16 + fr] = m[i];
    }
    __syncthreads();
    for (int e = tid; e < CH / 128 * BM; e += NW * 64) {
      const int blk = e / BM, r = e % BM;
      uint32_t a = red[blk * BW * BM + r];
#pragma unroll
      for (int w = 1; w < BW; ++w) a = max(a, red[(blk * BW + w) * BM + r]);
      const float sc = block_scale(a);
      div[e] = divisor(sc);
      if (r < mrows && n0 + 128 * blk < p.N_out) p.out_scale[(n0 / 128 + blk) * p.os_col + m0 + r] = sc;
    }
    __syncthreads();
    // the quantizer's own quotients (with the reciprocal alone 1 of 15 ties went
    // to the other code), one division for a row's block
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r = wm * TM + i * 16 + fr;
      const Divisor d = div[wn / BW * BM + r];
#pragma unroll
      for (int j = 0; j < JN; ++j) {
        const int c = CHW * wn + j * 16 + 4 * q;
        *reinterpret_cast<uint32_t*>(stg + r * CH + (((c >> 4) ^ (r & 7)) << 4) + (c & 15)) =
            pack_e4m3(quotient(acc[j][i][0], d), quotient(acc[j][i][1], d), quotient(acc[j][i][2], d),
                      quotient(acc[j][i][3], d));
      }
    }
    __syncthreads();
    uint8_t* out = reinterpret_cast<uint8_t*>(p.out);
    for (int e = tid; e < BM * (CH / 16); e += NW * 64) {
      const int r = e / (CH / 16), c = e % (CH / 16);
      if (r < mrows && n0 + 16 * c < p.N_out)  // N_out % 16 == 0: whole chunks
        *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(m0 + r) * p.ldo + n0 + 16 * c) =
            *reinterpret_cast<const u32x4*>(stg + r * CH + ((c ^ (r & 7)) << 4));
    }
  } else {
    float b4[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int n = n0 + wn * 64 + j * 16 + 4 * q + v;
        b4[j][v] = (bias && n < p.N_out) ? bias[n] : 0.f;
      }
    auto value = [&](int j, int i, float rs, float (&o)[4]) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float y = acc[j][i][v] + b4[j][v];
        o[v] = EPI == BLK_GELU ? gelu_erf(y) : (EPI == BLK_DOWN ? y * rs : y);
      }
    };
    // whole 16-byte chunks: the tile is staged in the ring (chunk c of row r at
    // c ^ (r & 7)) and leaves in whole rows.  Straight from the registers a row
    // is written in 32- or 64-byte pieces, which reach memory as twice the
    // write requests.
    constexpr int EB = ODT == SMOE_F32 ? 4 : 2, CPR = BN * EB / 16;
    constexpr int PASS = BM * BN * EB <= NS * STAGE ? 1 : 2, FP = FM / PASS, TP = TM / PASS;
    static_assert(BM / PASS * BN * EB <= NS * STAGE, "staging in the ring");
    const bool whole = (static_cast<int64_t>(p.N_out) * EB) % 16 == 0 && (p.ldo * EB) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    if (whole) {
#pragma unroll
      for (int h = 0; h < PASS; ++h) {
        __syncthreads();  // every wave is done with the ring (or the pass before)
#pragma unroll
        for (int i = h * FP; i < (h + 1) * FP; ++i) {
          const int r = wm * TM + i * 16 + fr, lr = wm * TP + (i - h * FP) * 16 + fr;
          const float rs = EPI == BLK_DOWN ? p.row_scale[m0 + min(r, mrows - 1)] : 1.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float o[4];
            value(j, i, rs, o);
            const int c4 = wn * 16 + j * 4 + q;  // group of four channels
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
            // past the L2s, where they would push the operands out (256 x 256
            // tiles, 16384 x 1024 -> 5632: 124 -> 118 us) or be written back at the
            // kernel's end (f32 rows, 777 tokens, top-4, 1408 -> 1024: 15.6 -> 14.6)
            if constexpr (BM == 256 || EPI == BLK_DOWN) __builtin_nontemporal_store(o, to);
            else *to = o;
          }
        }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = wm * TM + i * 16 + fr;
        if (r >= mrows) continue;
        float o[4];
        value(j, i, EPI == BLK_DOWN ? p.row_scale[m0 + r] : 1.f, o);
        store4<ODT>(p, m0 + r, n0 + wn * 64 + j * 16 + 4 * q, o);
      }
  }
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

template <int EPI, int ODT, bool WIDE, int BM, int BN, int WM, int WN, int NS>
int go_tile(const BlockGemm& a, hipStream_t s) {
  constexpr int CH = EPI == BLK_UP_SWIGLU ? BN / 2 : BN;
  const int rows = a.G > 0 ? a.max_rows : a.single_rows;
  // at most one partly filled row tile for every group with rows
  const int64_t tiles = (static_cast<int64_t>(rows) + BM - 1) / BM + (a.G > 0 ? std::min(a.G, rows) : 0);
  const int64_t grid = tiles * ((static_cast<int64_t>(a.N_out) + CH - 1) / CH);
  if (grid * 64 * WM * WN > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  SMOE_LAUNCH((k_gemm_blocks<EPI, ODT, WIDE, BM, BN, WM, WN, NS>), dim3(static_cast<unsigned>(grid)),
              dim3(64 * WM * WN), 0, s, a);
  return rc();
}

// Tiles of BM rows and CH channels: over groups, as if the rows were spread
// evenly (the host does not know the counts).
int64_t tiles_of(const BlockGemm& a, int BM, int CH) {
  const int64_t strips = (static_cast<int64_t>(a.N_out) + CH - 1) / CH;
  if (a.G == 0) return (static_cast<int64_t>(a.single_rows) + BM - 1) / BM * strips;
  const int64_t per = (static_cast<int64_t>(a.max_rows) + a.G - 1) / a.G;
  return std::min(a.G, a.max_rows) * ((per + BM - 1) / BM) * strips;
}

// Dense products: the smallest tile that one round of the CUs covers, since a
// tile alone on its CU takes about as long as its stages' bytes (200 x 1000 ->
// 2800: 128 x 128 tiles 10.0 us, 32 x 64 6.6, 64 x 64 6.3); past one round 64 x
// 128 and 128 x 128 (2048 rows: 17.0 and 15.4), whose workgroups share a CU, and
// 256 x 256, which reads the operands least often, once it fills about two
// thirds of the CUs (8192 x 1024 -> 5632: 72 -> 64 us; 2048 x 1000 -> 2800, 88 such
// tiles: 15.4 -> 20.5).
template <int EPI, int ODT, bool WIDE>
int go_dense(const BlockGemm& a, hipStream_t s) {
  const int64_t cus = device_cus();
  if (tiles_of(a, 32, 64) <= cus) return go_tile<EPI, ODT, WIDE, 32, 64, 2, 1, 4>(a, s);
  if (tiles_of(a, 64, 64) <= cus) return go_tile<EPI, ODT, WIDE, 64, 64, 4, 1, 4>(a, s);
  if (tiles_of(a, 64, 128) <= cus) return go_tile<EPI, ODT, WIDE, 64, 128, 2, 2, 3>(a, s);
  if constexpr (!WIDE) {
    if (tiles_of(a, 256, 256) * 8 >= cus * 5) return go_tile<EPI, ODT, WIDE, 256, 256, 2, 4, 2>(a, s);
  }
  if (tiles_of(a, 128, 128) <= cus) return go_tile<EPI, ODT, WIDE, 64, 128, 2, 2, 2>(a, s);
  return go_tile<EPI, ODT, WIDE, 128, 128, 2, 2, 2>(a, s);
}

// Grouped products: the row tile by the rows a group has on average, smaller
// where that leaves CUs without a tile; a third stage where a tile has its CU
// for itself.  Whole expert steps: 32 rows up to 40 a group (64 tokens, top-2 of
// 64: 77 us with 64-row tiles, 72 with 32, 59 with the third stage), 64 up to
// 112 (777 tokens, top-4 of 32: 49 us with 128-row tiles, 45 with 64, 52 with
// 32), 128 above (1500 tokens, top-2 of 16 SwiGLU: 81, 84, 114), 256 from 512 on
// (6000 tokens: 208 -> 181 us; 2500: 102 -> 119).  GELU's up product keeps 128
// rows, whose two workgroups a CU hide one's epilogue under the other's products
// (6000 tokens, top-4 of 32: 183 us with 256, 172).  WIDE has no registers for
// 256 rows and keeps 128 (16384 tokens, top-2 of 16 SwiGLU: up 581 us, down 252;
// 254 and 129 without).
template <int EPI, bool WIDE>
int go_grouped(const BlockGemm& a, hipStream_t s) {
  constexpr int O = SMOE_F32;
  constexpr bool SW = EPI == BLK_UP_SWIGLU;
  const int64_t cus = device_cus(), per = (static_cast<int64_t>(a.max_rows) + a.G - 1) / a.G;
  if constexpr (EPI != BLK_UP_GELU && !WIDE) {
    if (per >= 512 && tiles_of(a, 256, SW ? 128 : 256) * 8 >= cus * 5) return go_tile<EPI, O, WIDE, 256, 256, 2, 4, 2>(a, s);
  }
  int BM = per <= (SW ? 28 : 40) ? 32 : (per <= 112 ? 64 : 128);
  while (BM > 32 && tiles_of(a, BM, 128) < cus) BM /= 2;
  if constexpr (SW) {  // 256 weight rows a stage: one workgroup a CU with two stages already
    if (BM == 32) return go_tile<EPI, O, WIDE, 32, 256, 2, 4, 3>(a, s);
    if (BM == 64) return go_tile<EPI, O, WIDE, 64, 256, 2, 4, 3>(a, s);
    return go_tile<EPI, O, WIDE, 128, 256, 2, 4, 2>(a, s);
  } else {
    if constexpr (EPI == BLK_DOWN) {  // its channels need not come in blocks of 128
      if (tiles_of(a, 32, 128) * 8 <= cus * 5) return go_tile<EPI, O, WIDE, 32, 64, 2, 1, 4>(a, s);
    }
    const bool deep = tiles_of(a, BM, 128) <= 2 * cus;
    if (BM == 32 && deep) return go_tile<EPI, O, WIDE, 32, 128, 2, 2, 3>(a, s);
    if (BM == 32) return go_tile<EPI, O, WIDE, 32, 128, 2, 2, 2>(a, s);
    if (BM == 64 && deep) return go_tile<EPI, O, WIDE, 64, 128, 2, 2, 3>(a, s);
    if (BM == 64) return go_tile<EPI, O, WIDE, 64, 128, 2, 2, 2>(a, s);
    return go_tile<EPI, O, WIDE, 128, 128, 2, 2, 2>(a, s);
  }
}

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
  if (wgs * 256 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
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
  const bool f32 = a.out_dtype == SMOE_F32;
  switch (a.epi) {
    case BLK_LINEAR: return f32 ? go_dense<BLK_LINEAR, SMOE_F32, true>(a, s) : go_dense<BLK_LINEAR, SMOE_BF16, false>(a, s);
    case BLK_GELU: return f32 ? go_dense<BLK_GELU, SMOE_F32, true>(a, s) : go_dense<BLK_GELU, SMOE_BF16, false>(a, s);
    case BLK_UP_GELU: return a.wide ? go_grouped<BLK_UP_GELU, true>(a, s) : go_grouped<BLK_UP_GELU, false>(a, s);
    case BLK_UP_SWIGLU: return a.wide ? go_grouped<BLK_UP_SWIGLU, true>(a, s) : go_grouped<BLK_UP_SWIGLU, false>(a, s);
    case BLK_DOWN: return a.wide ? go_grouped<BLK_DOWN, true>(a, s) : go_grouped<BLK_DOWN, false>(a, s);
    default: return SMOE_EINVAL;
  }
}

}  // namespace smoe

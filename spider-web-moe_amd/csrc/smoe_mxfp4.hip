// Microscaled 4-bit floating point: the quantizer and its inverse, and the
// products on such operands, dense and grouped by expert.
#include "smoe_common.hpp"
#include "smoe_internal.hpp"
#include "smoe_mxfp4_dev.hpp"

namespace smoe {

int device_cus();

namespace {

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

// 128 columns of a row by 16 lanes (mx_quant_piece), sixteen pieces a workgroup;
// behind them workgroups for the planes, 256 words each.  Bytes bound it: a piece
// is read once, its amax goes over quads of lanes, the conversion instruction
// rounds.  16384 x 1024 bf16 and the planes of 5632 weight rows 10.0 us, 16384 x
// 2816 23.8 us (4.9 TB/s).
template <int XDT>
__global__ __launch_bounds__(256) void k_quant_mx(const MxQuant q, int npc, int64_t total, uint32_t quant_wgs,
                                                  const MxPlanes p0, const MxPlanes p1) {
  if (blockIdx.x < quant_wgs) {
    mx_quant_piece<XDT>(q, npc, total, (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4, threadIdx.x & 15);
    return;
  }
  const uint32_t i = (blockIdx.x - quant_wgs) * 256 + threadIdx.x, n0 = static_cast<uint32_t>(mx_plane_words(p0));
  if (i < n0) mx_plane_word(p0, i);
  else if (i - n0 < static_cast<uint32_t>(mx_plane_words(p1))) mx_plane_word(p1, i - n0);
}

// The values of codes: eight columns a thread.  Exact but for f16, whose range
// is smaller.  Bound by the bytes written: 16384 x 2816 to bf16 27.8 us, 4.2 TB/s.
template <int ODT>
__global__ __launch_bounds__(256) void k_dequant_mx(const uint8_t* __restrict__ codes, int64_t ld_codes,
                                                    const uint8_t* __restrict__ scale, int64_t ld_scale,
                                                    int cols, int npt, int64_t total, void* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const uint32_t iu = static_cast<uint32_t>(i);  // total < 2^32
  const int64_t row = iu / static_cast<uint32_t>(npt);
  const int c = static_cast<int>(iu - static_cast<uint32_t>(row) * npt) * 8;
  const uint8_t* cp = codes + row * ld_codes + c / 2;
  const int n = min(8, cols - c);
  uint32_t w = 0u;
  if (n == 8 && reinterpret_cast<uintptr_t>(cp) % 4 == 0) {
    w = *reinterpret_cast<const uint32_t*>(cp);
  } else {
    for (int j = 0; j < (n + 1) / 2; ++j) w |= static_cast<uint32_t>(cp[j]) << (8 * j);
  }
  const int byte = scale[row * ld_scale + c / kMxBlock];
  const float s = byte == 255 ? __uint_as_float(0x7FC00000u) : mx_scale_value(byte);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int m = (w >> (4 * j)) & 7;
    // 0, 0.5, then 1.m at exponents 0 .. 2
    const float a = m < 2 ? 0.5f * m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
    v[j] = ((w >> (4 * j)) & 8 ? -a : a) * s;
  }
  const int64_t at = row * cols + c;
  if constexpr (ODT == SMOE_F32) {
    float* o = static_cast<float*>(out) + at;
    if (n == 8 && reinterpret_cast<uintptr_t>(o) % 16 == 0) {
      *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      for (int j = 0; j < n; ++j) o[j] = v[j];
    }
  } else {
    uint16_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      h[j] = ODT == SMOE_BF16 ? f2bf(v[j]) : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[j]));
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    if (n == 8 && reinterpret_cast<uintptr_t>(o) % 16 == 0) {
      u32x4 p;
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = h[2 * j] | static_cast<uint32_t>(h[2 * j + 1]) << 16;
      *reinterpret_cast<u32x4*>(o) = p;
    } else {
      for (int j = 0; j < n; ++j) o[j] = h[j];
    }
  }
}

// ------------------------------------------------------------------ GEMM ----
// Where chunk c of row r of a stage lies (an involution).  Rows are 64 bytes;
// the four groups of lanes that a ds_read_b128 serves together (0-3, 12-15,
// 20-23, 24-27: rows 4 R .. of R = 0 and 3 at one chunk, 1 and 2 at its
// neighbour) meet in four different quarters of the banks.
__device__ __forceinline__ int mx_chunk(int r, int c) {
  const int R = (r >> 2) & 3;
  return c ^ ((R & 1) << 1 ^ (R >> 1) * 3);
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int kNowhere = static_cast<int>(0x80000000u);  // an offset that a buffer store drops

// BM rows x BN weight rows a tile (SwiGLU: BN / 2 gate channels and the up
// channels of the same outputs), 128 k (64 bytes of codes and 4 of scales a row)
// a stage through an LDS ring of NS stages filled by DMA.  WM x WN waves, wave
// tile BM / WM rows x BN / WN weight rows (SwiGLU: half gate, half up).  The
// matrix instruction takes the scales beside the codes, so a stage is one
// instruction for each 16 x 16 tile straight into the f32 accumulators.
//
// A workgroup walks over the tiles bid, bid + grid, ..: the next tile's first
// stages are requested before the last products and the epilogue, which uses no
// LDS.  For that a lane holds four rows of one channel of each 16 x 16 tile, and
// channels are dealt to the tiles so that the lane's are neighbours: a row leaves
// in 256-byte pieces of 16 lanes, and a block of 32 activations is quantized by a
// quad of lanes.
//
// The last two of a stage's FN steps come after the barrier that opens the next
// stage, over the latency of that stage's first fragments.
//
// The matrix instructions bound it, with their operands from LDS close behind.
// 128 x 256 tiles and two workgroups a CU, one's epilogue under the other's
// products: 16384 x 1024 -> 5632 bf16 70 us (2.7 PFLOP/s; 86 in one tile a
// workgroup, 55 of them the loop without DMA and epilogue), 32768 rows of 16
// experts of 1024 x 2816 135 us the up product (SwiGLU, 2.8 PFLOP/s) and 85 the
// down one (2.2: some 264 row tiles x 4 are two rounds of the 512 workgroups and a
// few tiles of a third; evenly loaded, 256 x 4, it takes 75); in the first calls after an idle second 150-167 (178 in
// one tile a workgroup) and 88-99.  Slower: 256 x 256 on four waves (one a SIMD),
// 128 x 128, and eight waves of 64 x 64.
template <int EPI, int ODT, int BM, int BN, int WM, int WN, int NS, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_gemm_mx(const MxGemm p) {
  constexpr bool SWIGLU = EPI == MX_UP_SWIGLU, UP = EPI == MX_UP_GELU || SWIGLU, GATHER = UP;
  constexpr int NW = WM * WN, CH = SWIGLU ? BN / 2 : BN, CHW = CH / WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int JC = SWIGLU ? FN / 2 : FN;  // channels of a lane
  static_assert(TM % 16 == 0 && TM <= 64 && FN >= 4 && (JC == 4 || JC == 8 || (!SWIGLU && !UP && JC == 2)), "wave tile");
  constexpr int XI = BM / 16, WI = BN / 16;  // DMA instructions of a stage (fewer than waves: some load the same)
  // scales: BN words of the weights by channel, then the rows', from the one at or
  // before the first whose word is 16-byte aligned; GATHER: the rows' word by word
  constexpr int SLOTS = BN / 4 + (GATHER ? 0 : BM / 4 + 1), SI = (SLOTS + 63) / 64, GI = GATHER ? (BM + 63) / 64 : 0;
  constexpr int XB = XI * 1024, WB = WI * 1024, XS = SI * 1024 - (GATHER ? 0 : (64 * SI - BN / 4) * 16), STAGE = XB + WB + SI * 1024 + GI * 256;
  constexpr int X_LD = (XI + NW - 1) / NW, W_LD = (WI + NW - 1) / NW, S_LD = (SI + NW - 1) / NW, G_LD = (GI + NW - 1) / NW, LD = X_LD + W_LD + S_LD + G_LD;
  static_assert((XI % NW == 0 || NW % XI == 0) && (WI % NW == 0 || NW % WI == 0), "whole DMA instructions");
  constexpr int EB = UP ? 0 : (ODT == SMOE_F32 ? 4 : 2);
  constexpr int STORES = UP ? FM * 8 : FM * 4 * (JC * EB / 16 > 0 ? JC * EB / 16 : 1);  // of a wave and tile
  static_assert((NS - 1) * LD < 64, "counted by vmcnt");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * STAGE];
  __shared__ int s_off[257];
  __shared__ __attribute__((aligned(16))) i32x4 s_tile[NW][8];  // a wave's: tiles requested, not yet finished
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, q = lane >> 4;
  const int nb = (p.K + kMxBlock - 1) / kMxBlock, KS = (nb + 3) / 4;
  for (int i = tid; i <= p.G && p.G > 0; i += NW * 64) s_off[i] = p.grp_off[i];
  __syncthreads();
  const int T = count_tiles<BM, CH>(p, s_off);
  if (static_cast<int>(blockIdx.x) >= T) return;  // uniform

  // a lane's number anew: what is computed from it stays where it is used (kept
  // over the products it would take their registers)
  auto anew = [](int v) {
    asm volatile("" : "+v"(v));
    return v;
  };
  // The channel of weight row r, from the tile's first (SwiGLU: of its half):
  // tile j = t / 16 of its wave, place c = t % 16; lane c's channels of a wave are
  // JC c + j, in f32 4 c + j % 4 of every 64
  auto channel = [](int r) {
    const int w = r / TN, t = r % TN, j = (t >> 4) % JC, c = t & 15;
    return CHW * w + (EB == 4 ? 64 * (j >> 2) + 4 * c + (j & 3) : JC * c + j);
  };
  // DMA sources of the tile that is requested: lane i of instruction j loads 16
  // bytes of row 16 j + i / 4, the block whose chunk lies at i % 4 (the same one
  // for every j), or slot 64 j + i of the scales
  // (an address is a base of the tile's and 32 bits of a lane's: launch_gemm_mxfp4
  // checks that they suffice)
  const int blk = mx_chunk(lane >> 2, lane & 3);
  const uint8_t *xbase = nullptr, *wbase = nullptr;
  uint32_t xoff[X_LD], woff[W_LD];
  const uint8_t* ssrc[S_LD];
  int64_t splane[S_LD];
  uint32_t goff[G_LD > 0 ? G_LD : 1];
  int pbid = blockIdx.x, ps = 0;  // tile and stage to request next
  int asked = 0;                  // tiles
  auto sources = [&] {
    int g, m0, mrows, n0;
    tile_at<BM, CH>(p, s_off, T, pbid, g, m0, mrows, n0);
    const int ln = anew(lane);
    s_tile[wave][asked++ & 7] = i32x4{g, m0, mrows, n0};  // every lane the same
    // rows past the end: a valid one, never stored
    auto xrow = [&](int r) {
      const int pr = min(r, mrows - 1);
      return static_cast<uint32_t>(GATHER ? p.a_rows[m0 + pr] : pr);
    };
    xbase = p.X + (GATHER ? 0 : m0 * p.ldx);
    wbase = p.W + g * p.w_gstride + n0 * p.ldw;
#pragma unroll
    for (int j = 0; j < X_LD; ++j)
      xoff[j] = xrow(16 * ((NW * j + wave) % XI) + (ln >> 2)) * static_cast<uint32_t>(p.ldx) + blk * 16;
#pragma unroll
    for (int j = 0; j < W_LD; ++j) {  // SwiGLU: gate rows, then up
      const int r = 16 * ((NW * j + wave) % WI) + (ln >> 2);
      woff[j] = static_cast<uint32_t>(min(channel(r), p.N_out - 1 - n0) + (SWIGLU && r % TN >= TN / 2 ? p.N_out : 0)) *
                    static_cast<uint32_t>(p.ldw) + blk * 16;
    }
#pragma unroll
    for (int j = 0; j < S_LD; ++j) {
      const int t = min(64 * ((NW * j + wave) % SI) + ln, SLOTS - 1);
      const bool up = SWIGLU && t >= BN / 8, wt = t < BN / 4;
      const int64_t at = wt ? min(n0 + 4 * (up ? t - BN / 8 : t), p.N_out - 1) + (up ? p.N_out : 0)
                            : min((m0 & ~3) + 4 * (t - BN / 4), m0 + mrows - 1);
      ssrc[j] = (wt ? p.ws + g * p.ws_gstride : p.xs) + (at & ~3ll) * 4;  // whole slots: planes are
      splane[j] = wt ? p.ws_plane : p.xs_plane;
    }
#pragma unroll
    for (int j = 0; j < G_LD; ++j) goff[j] = xrow(min(64 * ((NW * j + wave) % (GI > 0 ? GI : 1)) + ln, BM - 1)) * 4;
  };
  // The next stage of the sequence (behind the last one that one again, never
  // read): its tile's sources, then DMA d of it into slot `base`.  Blocks past K
  // are the row's first one instead, cut before use.
  uint32_t fwd = 0;  // bytes from the block of stage 0 to this stage's (an offset holds 16 blk, which may go again)
  auto next_stage = [&] {
    if (ps == KS && pbid + static_cast<int>(gridDim.x) < T) {  // uniform
      pbid += gridDim.x;
      ps = 0;
      sources();
    }
    ps = min(ps, KS - 1) + 1;
    fwd = 4 * (ps - 1) + blk < nb ? 64u * (ps - 1) : -16u * blk;
  };
  auto dma = [&](uint8_t* base, int d) {
    if (d < X_LD) {
      __builtin_amdgcn_global_load_lds((gbl_vptr)(xbase + (xoff[d < X_LD ? d : 0] + fwd)), (lds_vptr)(base + (NW * d + wave) % XI * 1024), 16, 0, 0);
    } else if (d < X_LD + W_LD) {
      const int e = d - X_LD;
      __builtin_amdgcn_global_load_lds((gbl_vptr)(wbase + (woff[e >= 0 && e < W_LD ? e : 0] + fwd)), (lds_vptr)(base + XB + (NW * e + wave) % WI * 1024), 16, 0, 0);
    } else if (d < X_LD + W_LD + S_LD) {
      const int e = d - X_LD - W_LD, i = e >= 0 && e < S_LD ? e : 0;
      __builtin_amdgcn_global_load_lds((gbl_vptr)(ssrc[i] + (ps - 1) * splane[i]), (lds_vptr)(base + XB + WB + (NW * e + wave) % SI * 1024), 16, 0, 0);
    } else {
      const int e = d - X_LD - W_LD - S_LD, i = e >= 0 && e < G_LD ? e : 0;
      __builtin_amdgcn_global_load_lds((gbl_vptr)(p.xs + (ps - 1) * p.xs_plane + goff[i]), (lds_vptr)(base + XB + WB + XS + (NW * e + wave) % (GI > 0 ? GI : 1) * 256), 4, 0, 0);
    }
  };
  // The last stage of a K that ends inside it: code 0 for what lies past K in
  // the rows.  The weights' codes there may be anything: none of them is NaN, nor
  // is a scale there.
  auto cut = [&](int s, uint8_t* base) {
    const int left = nb - 4 * s;
    if (left >= 4) return;  // uniform
    const int per = 4 - left;
    for (int e = anew(tid); e < BM * per; e += NW * 64) {
      const int r = e / per, b = left + e % per;
      *reinterpret_cast<u32x4*>(base + r * 64 + (mx_chunk(r, b) << 4)) = u32x4{0u, 0u, 0u, 0u};
    }
    lds_barrier();
  };

  const int flo = fr * 64 + (mx_chunk(fr, q) << 4);
  u32x4 x[FM], w[FN];
  uint32_t xsc[FM], wsc[FN];
  f32x4 acc[FN][FM];
  const int wch = (CHW * wn + (EB == 4 ? 4 : JC) * fr) * 4;  // the lane's first channel's word
  int shift = 0;  // rows before the tile's first in the first slot
  uint8_t *cur = ring, *prev = ring + (NS - 1) * STAGE;  // slots of this stage and of the one before
  bool stored = false;                                   // a tile's stores lie behind
  // Stage s of a tile: its DMAs landed (own ones by the count, in which the
  // stages requested since, and the stores of the tile before if they are newer,
  // may be under way; everybody's behind the barrier, after which nobody reads
  // the slot before any more), and that slot filled again.
  auto open = [&](int s) {
    constexpr int C = (NS - 2) * LD;
    wait_lgkm0();
    if (stored && s < NS - 1) wait_vmcnt<(C + STORES < 63 ? C + STORES : 63)>();
    else wait_vmcnt<C>();
    __builtin_amdgcn_s_barrier();
    if (s == KS - 1) cut(s, cur);
    next_stage();
  };
  auto read_w = [&](int j) { w[j] = *reinterpret_cast<const u32x4*>(cur + XB + (wn * TN + j * 16) * 64 + flo); };
  auto products = [&](int j) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = mx_mfma<0>(x[i], xsc[i], w[j], wsc[j], acc[j][i]);
    __builtin_amdgcn_sched_barrier(0);
  };
  // The products of an open stage but for the last two steps', which run
  // (`before`: those of the stage before) over the latency of its first reads
  auto stage = [&](auto before) {
    const uint8_t* sc = cur + XB + WB + q;
    const uint8_t* sx = sc + XS + (wm * TM + fr + shift) * 4;
    u32x4 nx[FM];
    uint32_t nxs[FM];
    u32x4 nwv[FN / 4];
    read_w(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      nx[i] = *reinterpret_cast<const u32x4*>(cur + (wm * TM + i * 16) * 64 + flo);
      nxs[i] = sx[i * 64];
    }
    // the lane's channels' words, four at a time: byte q of each
#pragma unroll
    for (int h = 0; h < FN / 4; ++h)
      nwv[h] = *reinterpret_cast<const u32x4*>(cur + XB + WB + wch + (4 * h >= JC ? CH * 4 : 0) + 4 * h % JC * (EB == 4 ? 64 : 4));
    read_w(1);
    if constexpr (FN > 4) read_w(2);  // w[2], w[3] of four still hold the stage before
    // the DMAs go under the products, evenly: all at once they hold up every wave
    // of the workgroup (16384 x 1024 -> 5632: 75 us)
    constexpr int FIRST = decltype(before)::value ? 0 : 2;
    auto dmas = [&](int step) {
#pragma unroll
      for (int d = 0; d < LD; ++d)
        if (max(d * FN / LD, FIRST) == step) dma(prev, d);
    };
    if constexpr (decltype(before)::value) {
      products(FN - 2);
      dmas(0);
      products(FN - 1);
      dmas(1);
    }
    if constexpr (FN == 4) read_w(2);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      x[i] = nx[i];
      xsc[i] = nxs[i];
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) wsc[j] = nwv[j / 4][j % 4] >> (8 * q);
#pragma unroll
    for (int j = 0; j < FN - 2; ++j) {
      if (j + 3 < FN) read_w(j + 3);
      products(j);
      dmas(j + 2);
    }
    prev = cur;
    cur = cur + STAGE == ring + NS * STAGE ? ring : cur + STAGE;
  };
  static_assert(FN >= 4, "steps of a stage");

  sources();
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    next_stage();
#pragma unroll
    for (int d = 0; d < LD; ++d) dma(ring + i * STAGE, d);
  }
  static_assert(NS <= 8, "s_tile: at most NS - 1 tiles ahead");
  for (int bid = blockIdx.x, turn = 0; bid < T; bid += gridDim.x, ++turn) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    open(0);
    float rows_w[(TM + 63) / 64];  // MX_DOWN: the weights of the wave's rows lane, lane + 64
    const i32x4 tile = s_tile[wave][turn & 7];
    const int cg = __builtin_amdgcn_readfirstlane(tile.x), cm0 = __builtin_amdgcn_readfirstlane(tile.y),
              cmrows = __builtin_amdgcn_readfirstlane(tile.z), cn0 = __builtin_amdgcn_readfirstlane(tile.w);
    if constexpr (!GATHER) shift = cm0 & 3;
    if constexpr (EPI == MX_DOWN) {
#pragma unroll
      for (int h = 0; h < (TM + 63) / 64; ++h) rows_w[h] = p.row_scale[cm0 + min(wm * TM + 64 * h + lane, cmrows - 1)];
    }
    stage(std::false_type{});
    if constexpr (EPI == MX_DOWN) {
#pragma unroll
      for (int h = 0; h < (TM + 63) / 64; ++h) rows_w[h] = __int_as_float(anew(__float_as_int(rows_w[h])));  // here, not behind the last DMAs
    }
#pragma unroll 1
    for (int s = 1; s < KS; ++s) {
      open(s);
      stage(std::true_type{});
    }
    products(FN - 2);
    products(FN - 1);

    // epilogue: lane (q, fr) holds channels ch0 .. of rows 4 q + v of each 16
    const int row0 = wm * TM, eq = anew(q), ef = anew(fr);
    const int ch0 = cn0 + CHW * wn + (EB == 4 ? 4 : JC) * ef;  // the lane's first channel
    float bias[JC];
#pragma unroll
    for (int j = 0; j < JC; ++j) bias[j] = 0.f;
    if (p.bias) {  // uniform; such loads wait for every DMA under way
#pragma unroll
      for (int j = 0; j < JC; ++j) {
        const int ch = ch0 + (EB == 4 ? 64 * (j >> 2) + (j & 3) : j);
        bias[j] = p.bias[cg * p.bias_gstride + min(ch, p.N_out - 1)];
      }
    }
    // A buffer ends behind the tile's last row: what a lane holds past it is not
    // stored (the range check counts the scalar offset of a row too)
    const int rows_left = max(cmrows - row0, 0);
    if constexpr (UP) {
      const int64_t rb = static_cast<int64_t>(cm0) + row0;
      const int ldo = static_cast<int>(p.ldo);
      const rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(static_cast<uint8_t*>(p.out) + rb * p.ldo, 0, rows_left * ldo, 0x00027000);
      // the scales of the wave's channels: four blocks a plane, TM rows of it
      const int64_t plane0 = (cn0 + CHW * wn) / 128;
      const rsrc_t osc = __builtin_amdgcn_make_buffer_rsrc(p.out_scale + plane0 * p.os_plane + rb * 4, 0, rows_left * 4, 0x00027000);
      const bool in = ch0 < p.N_out;                // N_out % 32 == 0: whole blocks
      const bool word = ch0 / 128 * 128 < p.N_out;  // blocks behind the last one of its word get scale 1
      const int to = in ? eq * 4 * ldo + ch0 / 2 : kNowhere;
      const int sto = word && ef % (32 / JC) == 0 ? eq * 16 + ch0 / 32 - static_cast<int>(plane0) * 4 : kNowhere;
      if (p.bias) {  // uniform
#pragma unroll
        for (int j = 0; j < JC; ++j)
#pragma unroll
          for (int i = 0; i < FM; ++i) acc[FN - JC + j][i] += bias[j];
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float y[JC], m = 0.f;
#pragma unroll
          for (int j = 0; j < JC; ++j) {
            if constexpr (SWIGLU) y[j] = silu(acc[j][i][v]) * acc[JC + j][i][v];
            else y[j] = gelu_tail(acc[j][i][v]);
            m = __builtin_elementwise_maximum(m, fabsf(y[j]));  // a NaN stays
          }
          uint32_t mb = quad_max(__float_as_uint(m) & 0x7FFFFFFFu);
          if constexpr (JC == 4) mb = max(mb, static_cast<uint32_t>(dpp_i<kDppHalfMirror>(static_cast<int>(mb))));
          // mx_scale_byte and mx_scale_value at once; the codes of a block whose
          // scale is NaN do not matter
          const int two = max(static_cast<int>(mb & 0x7F800000u) - 0x01000000, 0x00400000);
          const float sv = __int_as_float(two);
          uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], sv, 0);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], sv, 1);
          if constexpr (JC == 8) {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[JC - 4], y[JC - 3], sv, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[JC - 2], y[JC - 1], sv, 3);
          }
          const int byte = mb >= 0x7F800000u ? 255 : two >> 23;
          const int rr = i * 16 + v;
          if constexpr (JC == 4) __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(c), out, to, rr * ldo, 0);
          else __builtin_amdgcn_raw_buffer_store_b32(c, out, to, rr * ldo, 0);
          __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(in ? byte : 127), osc, sto, rr * 4, 0);
        }
    } else {
      // whole vectors of a row, or its elements one by one (then the stores are
      // not counted: waited for)
      const bool whole = (static_cast<int64_t>(p.N_out) * EB) % 16 == 0 && (p.ldo * EB) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
      auto value = [&](int j, int i, int v, float rs) {
        const float y = acc[j][i][v] + bias[j];
        return EPI == MX_GELU ? gelu_tail(y) : (EPI == MX_DOWN ? y * rs : y);
      };
      const int ldb = static_cast<int>(p.ldo) * EB;
      const rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(static_cast<uint8_t*>(p.out) + (static_cast<int64_t>(cm0) + row0) * ldb, 0,
                                                           rows_left * ldb, 0x00027000);
      if (whole) {
        // a row's offset in the lanes' registers, not in the scalar one, with which
        // 16-byte stores gave wrong values here where the next vector operation
        // wrote their data's registers (two of 16 columns, GELU)
        constexpr int HS = EB == 4 ? JC / 4 : 1;
        int to[HS];
#pragma unroll
        for (int h = 0; h < HS; ++h) to[h] = ch0 + 64 * h < p.N_out ? eq * 4 * ldb + (ch0 + 64 * h) * EB : kNowhere;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int rr = i * 16 + v, at = rr * ldb;
            const float rs = EPI == MX_DOWN ? __shfl(rows_w[i / 4], (rr + 4 * eq) & 63) : 1.f;
            if constexpr (EB == 4) {
#pragma unroll
              for (int h = 0; h < HS; ++h) {
                const f32x4 o = {value(4 * h, i, v, rs), value(4 * h + 1, i, v, rs), value(4 * h + 2, i, v, rs), value(4 * h + 3, i, v, rs)};
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), out, to[h] + at, 0, 2);
              }
            } else {
              const u32x2 a = {pack_bf2(value(0, i, v, rs), value(1, i, v, rs)), pack_bf2(value(2, i, v, rs), value(3, i, v, rs))};
              if constexpr (JC == 4) {
                __builtin_amdgcn_raw_buffer_store_b64(a, out, to[0] + at, 0, 2);
              } else {
                const u32x4 o = {a.x, a.y, pack_bf2(value(JC - 4, i, v, rs), value(JC - 3, i, v, rs)),
                                 pack_bf2(value(JC - 2, i, v, rs), value(JC - 1, i, v, rs))};
                __builtin_amdgcn_raw_buffer_store_b128(o, out, to[0] + at, 0, 2);
              }
            }
          }
      } else {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int r = row0 + i * 16 + 4 * eq + v;
            const float rs = EPI == MX_DOWN ? __shfl(rows_w[i / 4], (r - row0) & 63) : 1.f;
#pragma unroll
            for (int j = 0; j < JC; ++j) {
              const int ch = ch0 + (EB == 4 ? 64 * (j >> 2) + (j & 3) : j);
              if (r < cmrows && ch < p.N_out) {
                const int64_t at = (static_cast<int64_t>(cm0) + r) * p.ldo + ch;
                if constexpr (EB == 4) static_cast<float*>(p.out)[at] = value(j, i, v, rs);
                else static_cast<uint16_t*>(p.out)[at] = f2bf(value(j, i, v, rs));
              }
            }
          }
        wait_vmcnt<0>();
      }
    }
    stored = true;
  }
  wait_vmcnt<0>();  // nothing may land in the LDS of the workgroup that comes next
}

// Tiles of 128 x 256, two workgroups a CU
template <int EPI, int ODT>
int go(const MxGemm& a, hipStream_t s) {
  constexpr int BM = 128, CH = EPI == MX_UP_SWIGLU ? 128 : 256;
  const int rows = a.G > 0 ? a.max_rows : a.single_rows;
  // at most one partly filled row tile for every group with rows
  const int64_t tiles = (static_cast<int64_t>(rows) + BM - 1) / BM + (a.G > 0 ? std::min(a.G, rows) : 0);
  const int64_t all = tiles * ((static_cast<int64_t>(a.N_out) + CH - 1) / CH);
  if (all > 0x7fff0000ll) return SMOE_EINVAL;  // tiles are counted in 32 bits
  if (a.dry) return SMOE_OK;
  const int64_t grid = std::min<int64_t>(all, std::max<int64_t>(device_cus() * 2 / 8 * 8, 8));
  SMOE_LAUNCH((k_gemm_mx<EPI, ODT, BM, 256, 2, 2, 3, 2>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
  return rc();
}

}  // namespace

int launch_quantize_mxfp4(const MxQuant& q, const MxPlanes (&planes)[2], hipStream_t s) {
  if (q.rows < 0 || q.cols < 1 || q.ldx < q.cols || q.ld_codes < mx_code_pitch(q.cols) || q.ld_codes % 16 ||
      q.s_row % 4 || q.s_word % 4 || reinterpret_cast<uintptr_t>(q.codes) % 16 || reinterpret_cast<uintptr_t>(q.scale) % 4)
    return SMOE_EINVAL;
  if (q.rows == 0) return SMOE_OK;
  const int npc = (q.cols - 1) / 128 + 1;
  if (q.ld_codes > 64 * static_cast<int64_t>(npc) || q.rows > ((1 << 28) - 16) / npc) return SMOE_EINVAL;
  const int64_t total = q.rows * npc, wgs = (total + 15) / 16;
  const int64_t words = mx_plane_words(planes[0]) + mx_plane_words(planes[1]), all = wgs + (words + 255) / 256;
  if (words > kMxPlaneWords) return SMOE_EINVAL;
  return by_xdt(q.x_dtype, [&](auto xd) {
    auto go = [&](int64_t grid, int64_t quant_wgs) {
      hipLaunchKernelGGL((k_quant_mx<decltype(xd)::value>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, q, npc,
                         total, static_cast<uint32_t>(quant_wgs), planes[0], planes[1]);
      return rc();
    };
    if (all * 256 <= 0xffffffffll) return go(all, wgs);  // threads of a launch
    const int r = go(wgs, wgs);
    return r != SMOE_OK ? r : go(all - wgs, 0);
  });
}

int launch_dequantize_mxfp4(const uint8_t* codes, int64_t ld_codes, const uint8_t* scale, int64_t ld_scale, int64_t rows,
                            int cols, void* out, int out_dtype, hipStream_t s) {
  if (rows < 0 || cols < 1 || ld_codes < (cols + 1ll) / 2 || ld_scale < mx_blocks_of(cols)) return SMOE_EINVAL;
  if (rows == 0) return SMOE_OK;
  const int npt = (cols - 1) / 8 + 1;
  if (rows > 0xfffffe00ll / npt) return SMOE_EINVAL;  // threads of a launch
  const int64_t total = rows * npt;
  return by_xdt(out_dtype, [&](auto od) {
    hipLaunchKernelGGL((k_dequant_mx<decltype(od)::value>), dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0,
                       s, codes, ld_codes, scale, ld_scale, cols, npt, total, out);
    return rc();
  });
}

int launch_gemm_mxfp4(const MxGemm& a, hipStream_t s) {
  const int rows = a.G > 0 ? a.max_rows : a.single_rows;
  if (rows <= 0) return SMOE_OK;
  const int64_t pitch = mx_code_pitch(a.K);
  if (a.K < 1 || a.N_out < 1 || a.ldw < pitch || a.ldw % 16 || a.w_gstride % 16 || a.ws_gstride % 4) return SMOE_EINVAL;
  if (!a.x_float && (a.ldx < pitch || a.ldx % 16 || a.xs_plane % 4)) return SMOE_EINVAL;
  if (gemm_mx_few_fits(a)) return launch_gemm_mx_few(a, s);
  if (a.x_float) return SMOE_EINVAL;
  if (gemm_mx_stream_fits(a)) return launch_gemm_mx_stream(a, s);
  if (a.ws_plane == 0) return launch_gemm_mx_mid(a, s);
  if (a.ws_plane % 16 || a.xs_plane % 16) return SMOE_EINVAL;
  // 32-bit offsets: weight rows of a tile (SwiGLU: and those of the up half), rows
  // of X of a tile (gathered: all), a wave's rows of the output
  const bool up = a.epi == MX_UP_GELU || a.epi == MX_UP_SWIGLU;
  const int64_t lim = (1ll << 32) - (1 << 20);
  if (a.ldw > lim / 512 || a.ldx > lim / 512 || a.N_out > (1 << 22) ||
      (a.epi == MX_UP_SWIGLU && (a.N_out + 256ll) * a.ldw > lim) || (up && a.x_rows > lim / a.ldx))
    return SMOE_EINVAL;
  const bool f32 = a.out_dtype == SMOE_F32;
  switch (a.epi) {
    case MX_LINEAR: return f32 ? go<MX_LINEAR, SMOE_F32>(a, s) : go<MX_LINEAR, SMOE_BF16>(a, s);
    case MX_GELU: return f32 ? go<MX_GELU, SMOE_F32>(a, s) : go<MX_GELU, SMOE_BF16>(a, s);
    case MX_UP_GELU: return go<MX_UP_GELU, SMOE_F32>(a, s);
    case MX_UP_SWIGLU: return go<MX_UP_SWIGLU, SMOE_F32>(a, s);
    case MX_DOWN: return go<MX_DOWN, SMOE_F32>(a, s);
    default: return SMOE_EINVAL;
  }
}

// From 160 pieces of 256 x 256 outputs on (tiles of 128 x 256 for more than 320 of
// the 512 workgroups), and 512 rows a group; a workspace's size goes by it, so it is
// the same on every device.  Whole calls in a graph, us, middle and large kernel:
// 1024 x 1024 -> 5632 (88 pieces) 14.8 and 15.1, 1792 (154) 20.5 and 18.5, 2048
// (176) 20.4 and 18.4, 4096 (352) 30.2 and 28.4; 2048 x 2816 -> 4096 (128) 27.0 and
// 32.5, -> 5120 (160) 33.6 and 33.1; 10240 x 2816 -> 1024 (160) 41.8 and 42.6, 16384
// (256) 56.3 and 54.8; 512 x 1024 -> 20480 (160) 18.9 and 17.0.  Where one or two
// row tiles meet a vocabulary the middle one would be ahead: 40 x 1024 -> 50257 13.7
// and 28.7, 128 rows 21.3 and 35.2, 256 rows 35.6 and 39.3.
// Expert steps at 384, 512, 640 and 768 rows a group: 16 experts of 1024 x 2816
// (SwiGLU) 74.1, 96.1, 115.2, 128.6 and 80.8, 96.1, 107.1, 117.1; 32 of 1024 x 1408
// 89.4, 110.4, 123.2, 139.6 and 87.8, 114.4, 124.9, 134.4; 64 of 2048 x 1408 281.6,
// 356.1, 424.9, 495.2 and 271.5, 332.4, 398.1, 467.8 (from 192 on, 171.2 and 166.6);
// 8 of 256 x 512 stay behind (1024 rows 34.2 and 39.7).
bool mx_large_linear(int N, int N_out) {
  return N > kMxFewRows && (static_cast<int64_t>(N) + 255) / 256 * ((static_cast<int64_t>(N_out) + 255) / 256) >= 160;
}
bool mx_large_experts(int N, int K, int E) { return static_cast<int64_t>(N) * K >= 512ll * E; }

}  // namespace smoe

// Block-scaled fp8 products of a few rows per group (decode steps): the
// weights are streamed once, each wave loading the fragments it multiplies
// straight into registers, and what a step needs besides (dispatch plan,
// quantized messages) comes from one launch.
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

// 16 MT rows of one group.  UP: 128 channels a workgroup, 8 waves of 16
// channels (SwiGLU: 16 gate and 16 up), each over the whole of K, whose
// activations are quantized where they are.  Else: 16 NT channels, 4 waves
// taking every fourth block of K, their sums added through LDS in wave order.
//
// XQ: -1 X is codes; else its dtype, dense rows (a.x_float, a.ld_float), which
// the workgroup quantizes into LDS while its first weights are on their way.
//
// A wave loads D blocks' fragments at once and then multiplies them; what
// hides the latency is the number of waves (UP 2, else 4 or more on a SIMD).
template <int EPI, int ODT, bool WIDE, int MT, int NT, int XQ>
__global__ __launch_bounds__((EPI == BLK_UP_GELU || EPI == BLK_UP_SWIGLU) ? 512 : 256, 4)
void k_blocks_few(const BlockGemm p) {
  constexpr bool SWIGLU = EPI == BLK_UP_SWIGLU, UP = EPI == BLK_UP_GELU || SWIGLU;
  constexpr int BM = 16 * MT, BN = UP ? 128 : 16 * NT, NW = UP ? 8 : 4, STEP = UP ? 1 : 4;
  constexpr int D = MT == 1 ? (SWIGLU ? 3 : 4) : (WIDE || SWIGLU ? 2 : 3);
  static_assert(!UP || NT == (SWIGLU ? 2 : 1), "one or two weight tiles a wave");
  __shared__ __attribute__((aligned(16))) float red[UP ? 8 * BM : NW * MT * NT * 64 * 4];
  uint32_t* const redm = reinterpret_cast<uint32_t*>(red);  // UP: amax bits [8][BM]
  extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];  // XQ >= 0
  int g, m0, mrows, n0;
  if (!block_tile<BM, BN>(p, blockIdx.x, g, m0, mrows, n0)) return;  // uniform
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int q = lane >> 4, l16 = lane & 15;
  const int KB = (p.K + 127) / 128;

  const uint8_t* wrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int ch = UP ? n0 + 16 * wave + l16 : n0 + 16 * j + l16;
    const int64_t row = min(ch, p.N_out - 1) + (SWIGLU && j ? p.N_out : 0);
    wrow[j] = p.W + g * p.w_gstride + row * p.ldw;
  }
  const uint8_t* xrow[MT];
  const float* srow[MT];
  const int ldl = KB * 128;  // XQ: row pitch in LDS
  float* const xsl = reinterpret_cast<float*>(xlds + BM * ldl);  // [KB][BM]
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int pr = m0 + min(16 * i + l16, mrows - 1);  // rows past the end: a valid one, never stored
    const int64_t r = XQ >= 0 ? 0 : (p.a_rows ? p.a_rows[pr] : pr);
    xrow[i] = p.X + r * p.ldx;
    srow[i] = p.xs + r * p.xs_row;
  }
  const float* wsp = p.ws + g * p.ws_gstride + static_cast<int64_t>(n0 / 128) * KB;
  const float* wsp_up = wsp + static_cast<int64_t>((p.N_out + 127) / 128) * KB;  // SwiGLU

  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  bool first = true;
  for (int b0 = UP ? 0 : wave; b0 < KB || (XQ >= 0 && first); b0 += D * STEP) {
    Piece w[D][NT], x[D][MT];
    float xsv[D][MT], ws0[D], ws1[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int b = min(b0 + d * STEP, KB - 1);  // past the end: the last block again, not used
#pragma unroll
      for (int j = 0; j < NT; ++j) w[d][j] = load_piece(wrow[j], 128 * b, q, p.K);
      if constexpr (XQ < 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          x[d][i] = load_piece(xrow[i], 128 * b, q, p.K);
          xsv[d][i] = srow[i][b * p.xs_col];
        }
      }
      ws0[d] = wsp[b];
      ws1[d] = SWIGLU ? wsp_up[b] : 0.f;
    }
    if constexpr (XQ >= 0) {
      if (first) {  // sixteen lanes quantize a block
        constexpr int XD = XQ;
        for (int e = tid >> 4; e < mrows * KB; e += NW * 4) {
          const int r = e / KB, b = e - r * KB;
          const char* rp = reinterpret_cast<const char*>(p.x_float) + static_cast<int64_t>(m0 + r) * p.ld_float * elt_bytes<XD>();
          const bool vec = (reinterpret_cast<uintptr_t>(p.x_float) | static_cast<uintptr_t>(p.ld_float * elt_bytes<XD>())) % 16 == 0;
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
        const int b = min(b0 + d * STEP, KB - 1);
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
      const int b = b0 + d * STEP;
      if (b >= KB) break;  // uniform
      const int left = p.K - 128 * b;
      if (left < 128) {  // uniform: the last block of a ragged K
#pragma unroll
        for (int j = 0; j < NT; ++j) w[d][j] = cut_piece(w[d][j], q, left);
        if constexpr (XQ < 0)
#pragma unroll
          for (int i = 0; i < MT; ++i) x[d][i] = cut_piece(x[d][i], q, left);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const f32x4 part = block_product<WIDE>(w[d][j], x[d][i]);
          const float sc = xsv[d][i] * (SWIGLU && j ? ws1[d] : ws0[d]);
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[j][i][v] = fmaf(part[v], sc, acc[j][i][v]);
        }
    }
  }

  // lane: channels 4 q + v of row l16 of each 16 x 16 tile
  const float* bias = p.bias ? p.bias + g * p.bias_gstride : nullptr;
  if constexpr (UP) {
    const int c = n0 + 16 * wave + 4 * q;
    float y[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      uint32_t m = 0u;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const bool in = c + v < p.N_out;
        const float b = bias && in ? bias[c + v] : 0.f;
        float t;
        if constexpr (SWIGLU) t = silu(acc[0][i][v]) * (acc[NT - 1][i][v] + b);
        else t = gelu_erf(acc[0][i][v] + b);
        y[i][v] = in ? t : 0.f;
        m = amax_bits(m, y[i][v]);
      }
      m = quarters_max(m);
      if (q == 0) redm[wave * BM + 16 * i + l16] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = 16 * i + l16;
      uint32_t a = redm[r];
#pragma unroll
      for (int w = 1; w < 8; ++w) a = max(a, redm[w * BM + r]);
      const float sc = block_scale(a);
      const Divisor dv = divisor(sc);
      if (r >= mrows) continue;
      if (wave == 0 && q == 0) p.out_scale[(n0 / 128) * p.os_col + m0 + r] = sc;
      if (c < p.N_out)  // N_out % 16 == 0: four channels of one side
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + static_cast<int64_t>(m0 + r) * p.ldo + c) =
            pack_e4m3(quotient(y[i][0], dv), quotient(y[i][1], dv), quotient(y[i][2], dv), quotient(y[i][3], dv));
    }
  } else {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        *reinterpret_cast<f32x4*>(red + ((wave * NT + j) * MT + i) * 256 + lane * 4) = acc[j][i];
    __syncthreads();
    for (int t = wave; t < NT * MT; t += NW) {  // a tile a wave
      const int j = t / MT, i = t % MT;
      f32x4 s = *reinterpret_cast<const f32x4*>(red + t * 256 + lane * 4);
#pragma unroll
      for (int w = 1; w < NW; ++w) s += *reinterpret_cast<const f32x4*>(red + (w * NT * MT + t) * 256 + lane * 4);
      const int r = 16 * i + l16, n = n0 + 16 * j + 4 * q;
      if (r >= mrows) continue;
      const float rs = EPI == BLK_DOWN ? p.row_scale[m0 + r] : 1.f;
      float o[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float y = s[v] + (bias && n + v < p.N_out ? bias[n + v] : 0.f);
        o[v] = EPI == BLK_GELU ? gelu_erf(y) : (EPI == BLK_DOWN ? y * rs : y);
      }
      store4<ODT>(p, m0 + r, n, o);
    }
  }
}

// The merged slots of one token (merge_token's result) from registers: the
// ids that occur, ascending, each with its slots' weights added in slot order
// from 0; ids outside [0, E) and sums that are not > 0 left out, -1 padded.
template <int KB>
__device__ __forceinline__ void merge_slots(const int32_t* ti, const float* tw, int K, int E, int32_t* og, float* ow) {
  int id[KB];
  float w[KB], sum[KB];
  bool use[KB];
#pragma unroll
  for (int j = 0; j < KB; ++j) {  // unconditional loads at clamped indices
    id[j] = ti[min(j, K - 1)];
    w[j] = tw[min(j, K - 1)];
  }
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    use[j] = j < K && id[j] >= 0 && id[j] < E;
    sum[j] = 0.f;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      if (i < j) use[j] = use[j] && id[i] != id[j];  // its first slot speaks for an id
      sum[j] = i < K && id[i] == id[j] ? sum[j] + w[i] : sum[j];
    }
    use[j] = use[j] && sum[j] > 0.f;
  }
  int n = 0;
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    int rank = 0;
#pragma unroll
    for (int i = 0; i < KB; ++i) rank += use[i] && id[i] < id[j] ? 1 : 0;
    if (use[j]) {
      og[rank] = id[j];
      ow[rank] = sum[j];
      ++n;
    }
  }
  for (int j = n; j < K; ++j) {
    og[j] = -1;
    ow[j] = 0.f;
  }
}

// The plan of a decode step or a short prompt and its quantized messages in
// one launch (K <= KB): workgroup 0 merges every token's slots, ranks, scans and
// scatters (smoe_routing.hpp: the same plan as smoe_dispatch_plan), the
// others quantize 64 blocks each.
template <int KB>
__global__ __launch_bounds__(1024) void k_prep(const PrepArgs a, const BlockQuant bq, int nblk, int64_t total) {
  __shared__ int32_t sg[kPrepMaxEntries];
  __shared__ float sw[kPrepMaxEntries];
  __shared__ int cc[kPlanMaxG * (kPrepMaxN / 64)], tot[kPlanMaxG], goff[kPlanMaxG + 1], wsum[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  if (blockIdx.x > 0) {
    auto run = [&](auto xd) {
      quant_row_block<decltype(xd)::value>(bq, nblk, total,
                                           (static_cast<int64_t>(blockIdx.x - 1) * 1024 + tid) >> 4, tid & 15);
    };
    if (bq.x_dtype == SMOE_F32) run(std::integral_constant<int, SMOE_F32>{});
    else run(std::integral_constant<int, SMOE_BF16>{});
    return;
  }
  const int N = a.N, K = a.K, E = a.E, C = (N + 63) / 64;
  if (tid < N) merge_slots<KB>(a.idx + tid * K, a.w + tid * K, K, E, sg + tid * K, sw + tid * K);
  __syncthreads();
  const int win = a.win, W = (E + win - 1) / win;
  for (int item = wave; item < C * W; item += 16) {
    const int c = item / W;
    rank_chunk(sg, sw, N, K, E, 1, c * 64, (item % W) * win, win, cc + c, cc + c, C, a.tokrow);
  }
  __syncthreads();
  for (int g = wave; g < E; g += 16) {
    const int v = lane < C ? cc[g * C + lane] : 0;
    const int incl = wave_incl_scan(v);
    if (lane < C) cc[g * C + lane] = incl - v;
    if (lane == 63) tot[g] = incl;
  }
  __syncthreads();
  block_group_offsets(tot, E, goff, wsum);
  for (int g = tid; g <= E; g += 1024) a.off[g] = goff[g];
  if (tid < N) scatter_token(sg, sw, tid, K, E, cc + (tid >> 6), C, goff, a.rows, a.roww, a.tokrow);
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

template <int EPI, int ODT, bool WIDE, int MT, int NT, int XQ>
int go_few(const BlockGemm& a, hipStream_t s) {
  constexpr bool UP = EPI == BLK_UP_GELU || EPI == BLK_UP_SWIGLU;
  constexpr int BM = 16 * MT, BN = UP ? 128 : 16 * NT;
  const int rows = a.G > 0 ? a.max_rows : a.single_rows;
  const int64_t tiles = (rows + BM - 1) / BM + (a.G > 0 ? std::min(a.G, rows) : 0);
  const int64_t grid = tiles * ((a.N_out + BN - 1) / BN);
  if (grid > 0x7fffffff) return SMOE_EINVAL;
  const int KB = fp8_blocks_of(a.K);
  const size_t lds = XQ >= 0 ? static_cast<size_t>(BM) * KB * 132 : 0;
  SMOE_LAUNCH((k_blocks_few<EPI, ODT, WIDE, MT, NT, XQ>), dim3(static_cast<unsigned>(grid)), dim3(UP ? 512 : 256), lds, s, a);
  return rc();
}

template <int EPI, int ODT, bool WIDE, int NT>
int go_rows(const BlockGemm& a, int mt, hipStream_t s) {
  if constexpr (EPI == BLK_LINEAR || EPI == BLK_GELU) {
    if (a.x_float)
      return by_xdt(a.x_dtype, [&](auto xd) { return go_few<EPI, ODT, WIDE, 1, NT, decltype(xd)::value>(a, s); });
  }
  return mt == 1 ? go_few<EPI, ODT, WIDE, 1, NT, -1>(a, s) : go_few<EPI, ODT, WIDE, 2, NT, -1>(a, s);
}

}  // namespace

bool gemm_blocks_few_fits(const BlockGemm& a) {
  if (a.G == 0) return a.single_rows <= 32;
  return a.max_rows <= 24 * static_cast<int64_t>(a.G);
}

bool linear_quantizes_inside(int N, int K) {
  return N <= 16 && static_cast<int64_t>(N) * K <= 16384 && 16 * static_cast<int64_t>(fp8_blocks_of(K)) * 132 <= 49152;
}

int launch_gemm_blocks_few(const BlockGemm& a, hipStream_t s) {
  const int mt = a.G == 0 ? (a.single_rows <= 16 ? 1 : 2) : (a.max_rows <= 8 * static_cast<int64_t>(a.G) ? 1 : 2);
  const bool f32 = a.out_dtype == SMOE_F32;
  switch (a.epi) {
    case BLK_LINEAR: return f32 ? go_rows<BLK_LINEAR, SMOE_F32, true, 1>(a, mt, s) : go_rows<BLK_LINEAR, SMOE_BF16, false, 1>(a, mt, s);
    case BLK_GELU: return f32 ? go_rows<BLK_GELU, SMOE_F32, true, 1>(a, mt, s) : go_rows<BLK_GELU, SMOE_BF16, false, 1>(a, mt, s);
    case BLK_UP_GELU: return go_rows<BLK_UP_GELU, SMOE_F32, false, 1>(a, mt, s);
    case BLK_UP_SWIGLU: return go_rows<BLK_UP_SWIGLU, SMOE_F32, false, 2>(a, mt, s);
    case BLK_DOWN: return go_rows<BLK_DOWN, SMOE_F32, false, 1>(a, mt, s);
    default: return SMOE_EINVAL;
  }
}

bool prep_fits(int N, int K, int E) {
  return N <= kPrepMaxN && K <= 16 && N * K <= kPrepMaxEntries && E <= kPlanMaxG;
}

int launch_prep(const PrepArgs& args, const BlockQuant& q, hipStream_t s) {
  PrepArgs a = args;
  const int C = (a.N + 63) / 64;
  a.win = 64;  // narrower rank windows until the 16 waves have work
  while (a.win > 8 && C * ((a.E + a.win - 1) / a.win) < 16) a.win >>= 1;
  const int nblk = fp8_blocks_of(q.cols);
  const int64_t total = static_cast<int64_t>(q.rows) * nblk, wgs = (total + 63) / 64 + 1;
  if (wgs > 0x7fffffff) return SMOE_EINVAL;
  const dim3 grid(static_cast<unsigned>(wgs)), block(1024);
  if (a.K <= 2) hipLaunchKernelGGL((k_prep<2>), grid, block, 0, s, a, q, nblk, total);
  else if (a.K <= 4) hipLaunchKernelGGL((k_prep<4>), grid, block, 0, s, a, q, nblk, total);
  else if (a.K <= 8) hipLaunchKernelGGL((k_prep<8>), grid, block, 0, s, a, q, nblk, total);
  else hipLaunchKernelGGL((k_prep<16>), grid, block, 0, s, a, q, nblk, total);
  return rc();
}

}  // namespace smoe

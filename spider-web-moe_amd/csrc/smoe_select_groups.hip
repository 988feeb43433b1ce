// Group-limited expert routing and its gradient (the entry points
// smoe_select_groups / smoe_select_groups_backward).
//
//   s_e = softmax(z)_e or sigmoid(z_e)         scores, 0 where z_e = -inf
//   c_e = s_e + bias_e                         what is compared; -inf where masked
//   a group's value: the sum of its two largest c (of one where it has only one)
//   chosen: the K largest c of the top_groups groups of largest value
//   w_j = scale * s_j / max(sum of the chosen s, 1e-9), or scale * s_j
//
// Ties go to the lower index, NaN compares as +infinity.
#include "smoe_common.hpp"
#include "smoe_internal.hpp"

namespace smoe {
namespace {

template <int DT>
__device__ __forceinline__ float load_logit(const void* z, int64_t i) {
  if constexpr (DT == SMOE_F32) return reinterpret_cast<const float*>(z)[i];
  else if constexpr (DT == SMOE_BF16) return bf2f(reinterpret_cast<const uint16_t*>(z)[i]);
  else return static_cast<float>(reinterpret_cast<const _Float16*>(z)[i]);
}

// A wave's token: lane l holds experts V l .. V l + V - 1, in one load where
// rows keep its alignment (E % V == 0: the base of the array is aligned or the
// caller passes vec = false); -inf past E.
template <int DT, int V>
__device__ __forceinline__ void load_logits(const void* z, int64_t base, int E, bool vec, float (&v)[V]) {
  const int e0 = V * static_cast<int>(threadIdx.x & 63);
  if constexpr (V == 4) {
    if (vec) {  // uniform
      const int64_t at = base + (e0 < E ? e0 : 0);
      if constexpr (DT == SMOE_F32) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(z) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i];
      } else {
        const u32x2 a = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint16_t*>(z) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint16_t h = static_cast<uint16_t>(a[i >> 1] >> (16 * (i & 1)));
          v[i] = DT == SMOE_BF16 ? bf2f(h) : static_cast<float>(__builtin_bit_cast(_Float16, h));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = e0 + i < E ? v[i] : -INFINITY;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float x = load_logit<DT>(z, base + (e0 + i < E ? e0 + i : 0));
    v[i] = e0 + i < E ? x : -INFINITY;
  }
}

// ---- the same arithmetic in f32 and in f64 ----
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float min_of(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double min_of(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float exp_of(float a) { return expf(a); }
__device__ __forceinline__ double exp_of(double a) { return exp(a); }
__device__ __forceinline__ float wave_max_of(float v) { return wave_max(v); }
__device__ __forceinline__ double wave_max_of(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum_of(float v) { return wave_sum(v); }
__device__ __forceinline__ double wave_sum_of(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float lane_of(float v, int l) { return lane_f(v, l); }
__device__ __forceinline__ double lane_of(double v, int l) { return __shfl(v, l); }
// lane ^ (1 << step), or a lane that holds the same after the steps before
template <int STEP>
__device__ __forceinline__ float partner(float v) {
  if constexpr (STEP == 0) return dpp_f<kDppXor1>(v);
  else if constexpr (STEP == 1) return dpp_f<kDppXor2>(v);
  else if constexpr (STEP == 2) return dpp_f<kDppHalfMirror>(v);
  else if constexpr (STEP == 3) return dpp_f<kDppMirror>(v);
  else return __shfl_xor(v, 1 << STEP);
}
template <int STEP>
__device__ __forceinline__ double partner(double v) { return __shfl_xor(v, 1 << STEP); }

// LDS of a wave's own: what any lane wrote before is read by any lane after
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct SelectArgs {
  int E, K, sigmoid, groups, top_groups, renorm;
  const float* bias;
  float scale;
};

// The choice of one token (z: its logits, -inf past E).  Lane j < K returns
// slot j: its expert and score.  Returns whether every comparison that decided
// was by more than `tol` (scaled as below); T = double with tol 0 always is.
//
// Error of c in f32: the score is off by at most 2^-20 of the largest score
// (expf 1 ulp, its argument |z - max| 2^-24 times at most e^-t t < 0.4 of it, a
// sum of 10 levels, a division), the sum by 2^-24 of |c|.  Two compared values
// differ by twice that, two groups' values by four times and a rounding: with
// 2^-18 of the largest score and 2^-21 of the magnitudes that were added as the
// border, order in f32 is order.
template <typename T, int V>
__device__ __forceinline__ bool choose(const float (&z)[V], const SelectArgs& a, T* group_lds, int& slot_e,
                                       T& slot_s) {
  const int lane = threadIdx.x & 63, e0 = V * lane, E = a.E;
  const T ninf = -INFINITY;
  T s[V], c[V];
  T smax = 1;
  if (a.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = z[v] == -INFINITY ? T(0) : T(1) / (T(1) + exp_of(-T(z[v])));
  } else {
    float m = -INFINITY;  // of the numbers: a NaN makes the sum, and so every score, NaN
#pragma unroll
    for (int v = 0; v < V; ++v) m = z[v] > m ? z[v] : m;
    m = wave_max(m);
    T part = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = z[v] == -INFINITY ? T(0) : exp_of(T(z[v]) - T(m));
      part += s[v];
    }
    const T sum = wave_sum_of(part);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = z[v] == -INFINITY ? T(0) : s[v] / sum;
    smax = T(1) / sum;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const T b = a.bias && e0 + v < E ? T(a.bias[e0 + v]) : T(0);
    c[v] = z[v] == -INFINITY ? ninf : min_of(s[v] + b, T(INFINITY));  // NaN -> +infinity
  }
  const T border = smax * T(0x1p-18f);
  bool sure = true;
  bool open[V];
#pragma unroll
  for (int v = 0; v < V; ++v) open[v] = e0 + v < E;
  if (a.groups > 1) {
    const int per = E / a.groups;
    const int lanes = per / V;  // of a group
    T mine[V];                  // the value of each expert's group
    int gid[V];
    if (per % V == 0 && (lanes & (lanes - 1)) == 0) {  // uniform: groups are aligned runs of 2^n lanes
      T x = c[0], y = ninf;                            // the two largest
#pragma unroll
      for (int v = 1; v < V; ++v) {
        y = max_of(y, min_of(x, c[v]));
        x = max_of(x, c[v]);
      }
      auto merge = [&](T px, T py) {
        y = max_of(min_of(x, px), max_of(y, py));
        x = max_of(x, px);
      };
      if (lanes >= 2) merge(partner<0>(x), partner<0>(y));
      if (lanes >= 4) merge(partner<1>(x), partner<1>(y));
      if (lanes >= 8) merge(partner<2>(x), partner<2>(y));
      if (lanes >= 16) merge(partner<3>(x), partner<3>(y));
      if (lanes >= 32) merge(partner<4>(x), partner<4>(y));
      if (lanes >= 64) merge(partner<5>(x), partner<5>(y));
      const T value = y == ninf ? x : min_of(x + y, T(INFINITY));
      const int g = lane / lanes;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        mine[v] = value;
        gid[v] = g;
      }
      int ahead = 0;
      for (int o = 0; o < a.groups; ++o) {
        const T w = lane_of(value, o * lanes);
        ahead += w > value || (w == value && o < g) ? 1 : 0;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) open[v] = open[v] && ahead < a.top_groups;
    } else {
      // any other shape: through LDS, [0, 256) the values of c, then of the groups
      wave_sync();
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (e0 + v < E) group_lds[e0 + v] = c[v];
      wave_sync();
      T gval[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {  // this lane's groups: V lane + v
        T x = ninf, y = ninf;
        if (e0 + v < a.groups)
          for (int i = 0; i < per; ++i) {
            const T w = group_lds[(e0 + v) * per + i];
            y = max_of(y, min_of(x, w));
            x = max_of(x, w);
          }
        gval[v] = y == ninf ? x : min_of(x + y, T(INFINITY));
      }
      wave_sync();  // every value of c is read
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (e0 + v < a.groups) group_lds[e0 + v] = gval[v];
      wave_sync();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (e0 + v >= E) continue;
        gid[v] = (e0 + v) / per;
        mine[v] = group_lds[gid[v]];
        int ahead = 0;
        for (int o = 0; o < a.groups; ++o) {
          const T w = group_lds[o];
          ahead += w > mine[v] || (w == mine[v] && o < gid[v]) ? 1 : 0;
        }
        open[v] = ahead < a.top_groups;
      }
    }
    if constexpr (sizeof(T) == 4) {
      T low = INFINITY, high = ninf, cmag = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (e0 + v >= E) continue;
        if (c[v] != ninf) cmag = max_of(cmag, T(fabsf(c[v])));
        if (open[v]) low = min_of(low, mine[v]);
        else high = max_of(high, mine[v]);
      }
      low = -wave_max_of(-low);
      high = wave_max_of(high);
      cmag = wave_max_of(cmag);
      sure = high == ninf || low - high > border + T(0x1p-21f) * cmag;
    }
  }
  T last = 0;
  slot_e = 0;
  slot_s = 0;
  // one more than K: the first that is left out decides too
  const int rounds = sizeof(T) == 4 ? a.K + 1 : a.K;
#pragma unroll 1
  for (int j = 0; j < rounds; ++j) {
    T best = ninf, bs = 0;
    int bv = -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool take = open[v] && (bv < 0 || c[v] > best);
      best = take ? c[v] : best;
      bs = take ? s[v] : bs;
      bv = take ? v : bv;
    }
    const T top = wave_max_of(best);
    const uint64_t at = __ballot(bv >= 0 && best == top);
    if (!at) break;  // uniform: nothing is left (the round after the last pick)
    const int src = __builtin_ctzll(at);  // the lowest lane: the lowest index
    if constexpr (sizeof(T) == 4)
      if (j > 0 && top != ninf) sure = sure && last - top > border + T(0x1p-21f) * max_of(fabsf(last), fabsf(top));
    last = top;
    const int e = V * src + __builtin_amdgcn_readlane(bv, src);
    const T sc = lane_of(bs, src);
    if (lane == j) {
      slot_e = e;
      slot_s = sc;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) open[v] = open[v] && e0 + v != e;
  }
  return sure;
}

// One wave per token.  The choice is made in f32 and, where two values that
// decide lie nearer than f32 tells apart, once more in f64, so that it is the
// order of the real values.  16384 tokens over 256 experts in 8 groups, top 8 of
// 4 groups: 37 us with normal f32 logits (about 1 token in 100 needs both), 60
// at most, where every token does (uniform, saturated or equal logits).  Bound
// by instructions: about 1200 a token, half of them the K rounds of a maximum
// over the wave; the bytes are 4 us.
template <int DT, int V>
__global__ __launch_bounds__(256) void k_select_groups(const void* __restrict__ logits, int N, bool vec,
                                                       const SelectArgs a, float* __restrict__ top_w,
                                                       int32_t* __restrict__ top_idx) {
  __shared__ double lds[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  if (t >= N) return;  // wave-uniform; no workgroup barrier below
  float z[V];
  load_logits<DT, V>(logits, static_cast<int64_t>(t) * a.E, a.E, vec, z);
  int e;
  float s;
  if (!choose<float, V>(z, a, reinterpret_cast<float*>(lds[wave]), e, s)) {  // uniform
    double d;
    choose<double, V>(z, a, lds[wave], e, d);
    s = static_cast<float>(d);
  }
  const float total = wave_sum(lane < a.K ? s : 0.f);
  if (lane >= a.K) return;
  const float w = a.renorm ? s / (total < 1e-9f ? 1e-9f : total) : s;
  top_w[static_cast<int64_t>(t) * a.K + lane] = w * a.scale;
  top_idx[static_cast<int64_t>(t) * a.K + lane] = e;
}

// d loss / d z_e.  With S = sum of the chosen s and g_j = d loss / d w_j:
//   renorm, S >= 1e-9: ds_j = scale / S * (g_j - g_0 - sum_i (g_i - g_0) s_i / S),
//                      g_0 that of the first slot: 0 where the weights cannot
//                      change the loss (one slot, or equal g), and no worse else
//   renorm, otherwise: ds_j = scale / 1e-9 * g_j       (the clamped sum is a constant)
//   else               ds_j = scale * g_j
//   sigmoid: dz_e = ds_e s_e (1 - s_e);  softmax: dz_e = s_e (ds_e - sum_i s_i ds_i)
// An expert chosen in several slots takes all their gradients; ids outside
// [0, E) none.  One wave per token, lane j < K the slot j as well: 16384 tokens
// over 256 experts in 15.6 us, 34 MB at 2.2 TB/s.
template <int DT, int V>
__global__ __launch_bounds__(256) void k_select_groups_bwd(const void* __restrict__ logits, int N, bool vec,
                                                           const SelectArgs a,
                                                           const int32_t* __restrict__ top_idx,
                                                           const float* __restrict__ d_w,
                                                           void* __restrict__ d_logits) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= N) return;  // wave-uniform
  const int E = a.E, K = a.K, e0 = V * lane;
  const int64_t base = static_cast<int64_t>(t) * E;
  const int64_t slot = static_cast<int64_t>(t) * K + (lane < K ? lane : 0);
  const int id_in = top_idx[slot];
  const float g = d_w[slot];
  float z[V];
  load_logits<DT, V>(logits, base, E, vec, z);
  const bool used = lane < K && id_in >= 0 && id_in < E;
  const int id = used ? id_in : -1;
  const float zs = load_logit<DT>(logits, base + (used ? id : 0));  // the slot's logit
  float m = -INFINITY, sum = 1.f;
  if (!a.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) m = z[v] > m ? z[v] : m;
    m = wave_max(m);
    float part = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) part += z[v] == -INFINITY ? 0.f : expf(z[v] - m);
    sum = wave_sum(part);
  }
  // score and its slope (sigmoid: s (1 - s) without the cancellation)
  auto score = [&](float x, float& slope) {
    if (x == -INFINITY) {
      slope = 0.f;
      return 0.f;
    }
    if (!a.sigmoid) {
      slope = 1.f;
      return expf(x - m) / sum;
    }
    const float u = expf(-fabsf(x)), big = 1.f / (1.f + u), small = u / (1.f + u);
    slope = big * small;
    return x >= 0.f ? big : (x < 0.f ? small : x);
  };
  float unused;
  const float ss = used ? score(zs, unused) : 0.f;
  const float total = wave_sum(ss);
  const bool over = total >= 1e-9f || total != total;
  const float f = a.renorm ? a.scale / (over ? total : 1e-9f) : a.scale;
  const bool centred = a.renorm && over;  // uniform
  const uint64_t slots = __ballot(used);
  const float gc = centred && slots ? g - lane_f(g, __builtin_ctzll(slots)) : g;
  const float dot = wave_sum(used ? gc * ss : 0.f);
  const float ds_slot = used ? f * (gc - (centred ? dot / total : 0.f)) : 0.f;
  const float mean = a.sigmoid ? 0.f : wave_sum(used ? ss * ds_slot : 0.f);
  float d[V];
#pragma unroll
  for (int v = 0; v < V; ++v) d[v] = 0.f;
#pragma unroll 1
  for (int j = 0; j < K; ++j) {
    const int e = __builtin_amdgcn_readlane(id, j);
    const float dj = lane_f(ds_slot, j);
#pragma unroll
    for (int v = 0; v < V; ++v) d[v] += e0 + v == e ? dj : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float slope;
    const float s = score(z[v], slope);
    if (a.sigmoid) d[v] = d[v] == 0.f ? 0.f : d[v] * slope;
    else d[v] = s * (d[v] - mean);
  }
  if constexpr (V == 4) {
    if (vec) {
      if (e0 >= E) return;
      if constexpr (DT == SMOE_F32) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(d_logits) + base + e0) = f32x4{d[0], d[1], d[2], d[3]};
      } else if constexpr (DT == SMOE_BF16) {
        *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(d_logits) + base + e0) =
            u32x2{pack_bf2(d[0], d[1]), pack_bf2(d[2], d[3])};
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) reinterpret_cast<_Float16*>(d_logits)[base + e0 + v] = static_cast<_Float16>(d[v]);
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (e0 + v >= E) continue;
    if constexpr (DT == SMOE_F32) reinterpret_cast<float*>(d_logits)[base + e0 + v] = d[v];
    else if constexpr (DT == SMOE_BF16) reinterpret_cast<uint16_t*>(d_logits)[base + e0 + v] = f2bf(d[v]);
    else reinterpret_cast<_Float16*>(d_logits)[base + e0 + v] = static_cast<_Float16>(d[v]);
  }
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

template <typename F>
int by_zdt(int dt, F&& f) {
  switch (dt) {
    case SMOE_F32: return f(std::integral_constant<int, SMOE_F32>{});
    case SMOE_BF16: return f(std::integral_constant<int, SMOE_BF16>{});
    case SMOE_F16: return f(std::integral_constant<int, SMOE_F16>{});
    default: return SMOE_EUNSUPPORTED;
  }
}

// experts a lane holds: E <= 64, <= 128, <= 256
template <typename F>
int by_lane(int E, F&& f) {
  if (E <= 64) return f(std::integral_constant<int, 1>{});
  if (E <= 128) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}

// whether rows of E logits load (and store) as vectors of four
bool vec4(const void* p, int zdt, int E) {
  return E % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (zdt == SMOE_F32 ? 16 : 8) == 0;
}

}  // namespace

int launch_select_groups(const void* logits, int zdt, int N, int E, int K, int sigmoid, const float* bias,
                         int groups, int top_groups, int renorm, float scale, float* top_w,
                         int32_t* top_idx, hipStream_t s) {
  if (N <= 0) return SMOE_OK;
  const SelectArgs a{E, K, sigmoid, groups, top_groups, renorm, bias, scale};
  return by_zdt(zdt, [&](auto dt) {
    return by_lane(E, [&](auto v) {
      hipLaunchKernelGGL((k_select_groups<decltype(dt)::value, decltype(v)::value>), dim3((N + 3) / 4), dim3(256), 0,
                         s, logits, N, vec4(logits, zdt, E), a, top_w, top_idx);
      return rc();
    });
  });
}

int launch_select_groups_bwd(const void* logits, int zdt, int N, int E, int K, int sigmoid, int renorm,
                             float scale, const int32_t* top_idx, const float* d_w, void* d_logits,
                             hipStream_t s) {
  if (N <= 0) return SMOE_OK;
  const SelectArgs a{E, K, sigmoid, 1, 1, renorm, nullptr, scale};
  return by_zdt(zdt, [&](auto dt) {
    return by_lane(E, [&](auto v) {
      hipLaunchKernelGGL((k_select_groups_bwd<decltype(dt)::value, decltype(v)::value>), dim3((N + 3) / 4), dim3(256),
                         0, s, logits, N, vec4(logits, zdt, E) && vec4(d_logits, zdt, E), a, top_idx, d_w, d_logits);
      return rc();
    });
  });
}

}  // namespace smoe

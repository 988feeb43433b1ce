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

constexpr int kSgMaxE = 256;

template <int DT>
__device__ __forceinline__ float load_logit(const void* z, int64_t i) {
  if constexpr (DT == SMOE_F32) return reinterpret_cast<const float*>(z)[i];
  else if constexpr (DT == SMOE_BF16) return bf2f(reinterpret_cast<const uint16_t*>(z)[i]);
  else return static_cast<float>(reinterpret_cast<const _Float16*>(z)[i]);
}

__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ double key64(double v) { return fmin(v, static_cast<double>(INFINITY)); }

// One wave per token, lane l holding experts l, l + 64, ..; all in 64 bits, so
// that which of two near scores is the larger does not depend on how an exp
// rounds.
template <int DT>
__global__ __launch_bounds__(256) void k_select_groups(const void* __restrict__ logits, int N, int E,
                                                       int K, int sigmoid, const float* __restrict__ bias,
                                                       int groups, int top_groups, int renorm, float scale,
                                                       float* __restrict__ top_w,
                                                       int32_t* __restrict__ top_idx) {
  constexpr int V = kSgMaxE / 64;
  __shared__ double cs[4][kSgMaxE], gv[4][kSgMaxE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  const bool live = t < N;
  const int64_t base = static_cast<int64_t>(live ? t : N - 1) * E;
  double s[V], key[V];
  bool cand[V];
  double mx = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 64 * v;
    s[v] = e < E ? load_logit<DT>(logits, base + e) : -INFINITY;
    cand[v] = e < E;
    mx = (s[v] > mx || s[v] != s[v]) ? s[v] : mx;
  }
  double sum = 0.0;
  if (!sigmoid) {
    mx = wave_max64(mx);
#pragma unroll
    for (int v = 0; v < V; ++v) sum += s[v] == -INFINITY ? 0.0 : exp(s[v] - mx);
    sum = wave_sum64(sum);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 64 * v;
    const bool masked = s[v] == -INFINITY;
    s[v] = masked ? 0.0 : (sigmoid ? 1.0 / (1.0 + exp(-s[v])) : exp(s[v] - mx) / sum);
    key[v] = masked ? -INFINITY : key64(s[v] + (bias && e < E ? static_cast<double>(bias[e]) : 0.0));
    if (e < E) cs[wave][e] = key[v];
  }
  __syncthreads();
  if (groups > 1) {
    const int per = E / groups;
    for (int g = lane; g < groups; g += 64) {
      double a = -INFINITY, b = -INFINITY;
      for (int i = 0; i < per; ++i) {
        const double x = cs[wave][g * per + i];
        b = fmax(b, fmin(a, x));
        a = fmax(a, x);
      }
      gv[wave][g] = b == -INFINITY ? a : key64(a + b);
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane + 64 * v;
      if (e >= E) continue;
      const int g = e / per;
      int before = 0;
      for (int o = 0; o < groups; ++o)
        before += gv[wave][o] > gv[wave][g] || (gv[wave][o] == gv[wave][g] && o < g);
      cand[v] = before < top_groups;
    }
  }
  double slot = 0.0, total = 0.0;
  int slot_i = 0;
  for (int j = 0; j < K; ++j) {
    double bv = -INFINITY, bs = 0.0;
    int bi = 1 << 20;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane + 64 * v;
      if (cand[v] && (key[v] > bv || (key[v] == bv && e < bi))) {
        bv = key[v];
        bi = e;
        bs = s[v];
      }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const double ov = __shfl_xor(bv, o), os = __shfl_xor(bs, o);
      const int oi = __shfl_xor(bi, o);
      if (ov > bv || (ov == bv && oi < bi)) {
        bv = ov;
        bi = oi;
        bs = os;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) cand[v] = cand[v] && lane + 64 * v != bi;
    total += bs;
    if (lane == j) {
      slot = bs;
      slot_i = bi;
    }
  }
  if (live && lane < K) {
    const double w = renorm ? slot / (total < 1e-9 ? 1e-9 : total) : slot;
    top_w[static_cast<int64_t>(t) * K + lane] = static_cast<float>(w * scale);
    top_idx[static_cast<int64_t>(t) * K + lane] = slot_i;
  }
}

// d loss / d z_e.  With S = sum of the chosen s and g_j = d loss / d w_j:
//   renorm, S > 1e-9:  ds_j = scale / S * (g_j - sum_i g_i s_i / S)
//   renorm, otherwise: ds_j = scale / 1e-9 * g_j       (the clamped sum is a constant)
//   else               ds_j = scale * g_j
//   sigmoid: dz_e = ds_e s_e (1 - s_e);  softmax: dz_e = s_e (ds_e - sum_i s_i ds_i)
// An expert chosen in several slots takes all their gradients; ids outside
// [0, E) none.
template <int DT>
__global__ __launch_bounds__(256) void k_select_groups_bwd(const void* __restrict__ logits, int N, int E,
                                                           int K, int sigmoid, int renorm, float scale,
                                                           const int32_t* __restrict__ top_idx,
                                                           const float* __restrict__ d_w,
                                                           void* __restrict__ d_logits) {
  constexpr int V = kSgMaxE / 64;
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= N) return;  // wave-uniform
  const int64_t base = static_cast<int64_t>(t) * E;
  float z[V], s[V], om[V], ds[V];
  float mx = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 64 * v;
    z[v] = e < E ? load_logit<DT>(logits, base + e) : -INFINITY;
    mx = fmaxf(mx, z[v]);
    ds[v] = 0.f;
  }
  float sum = 1.f;
  if (!sigmoid) {
    mx = wave_max(mx);
    float part = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) part += z[v] == -INFINITY ? 0.f : expf(z[v] - mx);
    sum = wave_sum(part);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool masked = z[v] == -INFINITY;
    if (sigmoid) {  // 1 - s without the cancellation
      const float x = expf(-fabsf(z[v]));
      const float big = 1.f / (1.f + x), small = x / (1.f + x);
      s[v] = masked ? 0.f : (z[v] >= 0.f ? big : (z[v] < 0.f ? small : z[v]));
      om[v] = z[v] >= 0.f ? small : (z[v] < 0.f ? big : z[v]);
    } else {
      s[v] = masked ? 0.f : expf(z[v] - mx) / sum;
      om[v] = 1.f;
    }
  }
  const int id = lane < K ? top_idx[static_cast<int64_t>(t) * K + lane] : -1;
  const float g = lane < K ? d_w[static_cast<int64_t>(t) * K + lane] : 0.f;
  float total = 0.f, dot = 0.f;
  for (int j = 0; j < K; ++j) {
    const int e = __shfl(id, j);
    const float gj = __shfl(g, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 64 * v == e) {
        total += s[v];
        dot += gj * s[v];
        ds[v] += gj;
      }
  }
  total = wave_sum(total);
  dot = wave_sum(dot);
  const bool over = total >= 1e-9f || total != total;
  const float f = renorm ? scale / (over ? total : 1e-9f) : scale;
  const float sub = renorm && over ? dot / total : 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float n = 0.f;  // how many slots chose the expert
    for (int j = 0; j < K; ++j) n += lane + 64 * v == __shfl(id, j) ? 1.f : 0.f;
    ds[v] = n > 0.f ? f * (ds[v] - n * sub) : 0.f;
  }
  float mean = 0.f;
  if (!sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) mean += s[v] * ds[v];
    mean = wave_sum(mean);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 64 * v;
    if (e >= E) continue;
    const float d = sigmoid ? (ds[v] == 0.f ? 0.f : ds[v] * s[v] * om[v]) : s[v] * (ds[v] - mean);
    if constexpr (DT == SMOE_F32) reinterpret_cast<float*>(d_logits)[base + e] = d;
    else if constexpr (DT == SMOE_BF16) reinterpret_cast<uint16_t*>(d_logits)[base + e] = f2bf(d);
    else reinterpret_cast<_Float16*>(d_logits)[base + e] = static_cast<_Float16>(d);
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

}  // namespace

int launch_select_groups(const void* logits, int zdt, int N, int E, int K, int sigmoid, const float* bias,
                         int groups, int top_groups, int renorm, float scale, float* top_w,
                         int32_t* top_idx, hipStream_t s) {
  if (N <= 0) return SMOE_OK;
  return by_zdt(zdt, [&](auto dt) {
    hipLaunchKernelGGL((k_select_groups<decltype(dt)::value>), dim3((N + 3) / 4), dim3(256), 0, s, logits,
                       N, E, K, sigmoid, bias, groups, top_groups, renorm, scale, top_w, top_idx);
    return rc();
  });
}

int launch_select_groups_bwd(const void* logits, int zdt, int N, int E, int K, int sigmoid, int renorm,
                             float scale, const int32_t* top_idx, const float* d_w, void* d_logits,
                             hipStream_t s) {
  if (N <= 0) return SMOE_OK;
  return by_zdt(zdt, [&](auto dt) {
    hipLaunchKernelGGL((k_select_groups_bwd<decltype(dt)::value>), dim3((N + 3) / 4), dim3(256), 0, s,
                       logits, N, E, K, sigmoid, renorm, scale, top_idx, d_w, d_logits);
    return rc();
  });
}

}  // namespace smoe

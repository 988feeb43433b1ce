// Balance loss of a router and its gradient (the entry points
// smoe_balance_loss / smoe_balance_loss_backward).
//
// Per sequence of T tokens, of which n are not masked:
//   p_t    = softmax(z_t), or sigmoid(z_t) over its sum       0 where z = -inf
//   c_e    = how many of the tokens' choices are expert e      (ids outside [0, E) none)
//   load_e = c_e / sum of c;  P_e = sum over t of p_te / n
//   loss   = E sum_e load_e P_e
// The counts have no gradient.  With u_e = E load_e - 1 (the p of a token add
// up to 1, so a constant may go: where the load is even u is 0 exactly, and so
// is the gradient)
//   dz_te  = dloss / n * p_te (u_e - sum_i p_ti u_i)           softmax
//            the same times 1 - sigmoid(z_te)                  sigmoid
#include "smoe_common.hpp"
#include "smoe_internal.hpp"

namespace smoe {
namespace {

template <int DT>
__device__ __forceinline__ float logit(const void* z, int64_t i) {
  if constexpr (DT == SMOE_F32) return reinterpret_cast<const float*>(z)[i];
  else if constexpr (DT == SMOE_BF16) return bf2f(reinterpret_cast<const uint16_t*>(z)[i]);
  else return static_cast<float>(reinterpret_cast<const _Float16*>(z)[i]);
}

// Experts e0 .. e0 + V - 1 of a token, -inf past E; one load where the rows'
// alignment allows it (vec)
template <int DT, int V>
__device__ __forceinline__ void load_row(const void* z, int64_t base, int e0, int E, bool vec, float (&v)[V]) {
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
    const float x = logit<DT>(z, base + (e0 + i < E ? e0 + i : 0));
    v[i] = e0 + i < E ? x : -INFINITY;
  }
}

// e^x within (3 + 2.3 |x|) 2^-24 of its value (the product's rounding, the
// constant's, the instruction's), 0 below 2^-126.  With the argument split, so that
// |x| plays no part, 8 sequences of 2048 tokens over 256 experts take 13.4 us
// forward instead of 12.8, 2^20 tokens over 64 experts 198 instead of 188.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// p of a token whose experts lie in SEG lanes, V each, and with sigmoid also
// 1 - sigmoid(z).  t = exp(-|z|) gives both sigmoid(z) and 1 - sigmoid(z): they
// are 1 / (1 + t) and t / (1 + t).  A token whose logits are all below -16 takes
// the largest out first, exp(z - m) / (1 + t): the shares of far negative logits
// are those of their exponentials (above, a t that is 0 has a share below e^-71).
template <int SEG, int V>
__device__ __forceinline__ void shares(const float (&z)[V], bool sigmoid, float (&p)[V], float (&rest)[V]) {
  float m = -INFINITY;  // of the numbers: a NaN makes the sum, and so every share, NaN
#pragma unroll
  for (int v = 0; v < V; ++v) m = fmaxf(m, z[v]);
  m = seg_max<SEG>(m);
  float sum = 0.f;
  if (sigmoid) {  // uniform
    float one[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float t = exp_of(-fabsf(z[v]));
      one[v] = __builtin_amdgcn_rcpf(1.f + t);
      const float far = t * one[v];
      p[v] = z[v] > 0.f ? one[v] : far;
      rest[v] = z[v] > 0.f ? far : one[v];
    }
    if (__builtin_amdgcn_ballot_w64(m < -16.f)) {  // uniform
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float e = z[v] == -INFINITY ? 0.f : exp_of(z[v] - m) * one[v];
        p[v] = m < -16.f ? e : p[v];
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = z[v] == -INFINITY ? 0.f : exp_of(z[v] - m);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sum += p[v];
  sum = seg_sum<SEG>(sum);
  const float r = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] *= r;
}

struct BalanceArgs {
  const void* logits;
  const int32_t* idx;
  const uint8_t* mask;  // or nullptr
  int S, T, E, K;
  bool sigmoid, vec;
  int rows, chunks;     // tokens of a workgroup; workgroups of a sequence
  float* part_p;        // [S * chunks, E] sums of p
  int32_t* part_c;      // [S * chunks, E + 1] counts, then tokens
  float* loss;          // [S]
  int32_t* counts;      // [S, E]
  float* slope;         // [S, E] u / n, or nullptr
};

// A sequence's loss from its chunks' sums by NT threads (chunk i's at
// sum_p + i * E, cnt + i * (E + 1)): sums over the chunks in 64 bits, in a fixed
// order, by NT / P slices of P >= E threads.
template <int NT>
__device__ __forceinline__ void finish(const BalanceArgs& a, int seq, int chunks, const float* sum_p, const int32_t* cnt) {
  __shared__ double s_sum[NT], s_red[NT / 64];
  __shared__ int s_cnt[NT], s_n[NT / 64], s_tot[NT / 64];
  const int tid = threadIdx.x, E = a.E;
  int P = 16;
  while (P < E) P *= 2;  // <= 256 <= NT
  const int e = tid % P, slice = tid / P, slices = NT / P;
  double sum = 0.0;
  int c = 0, n = 0;
  if (e < E) {
#pragma unroll 8
    for (int i = slice; i < chunks; i += slices) {
      sum += static_cast<double>(sum_p[static_cast<int64_t>(i) * E + e]);
      c += cnt[static_cast<int64_t>(i) * (E + 1) + e];
    }
  }
  for (int i = tid; i < chunks; i += NT) n += cnt[static_cast<int64_t>(i) * (E + 1) + E];
  s_sum[tid] = sum;
  s_cnt[tid] = c;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o);
  if ((tid & 63) == 0) s_n[tid >> 6] = n;
  __syncthreads();
  sum = 0.0;
  c = 0;
  if (tid < P)
    for (int i = 0; i < slices; ++i) {
      sum += s_sum[i * P + tid];
      c += s_cnt[i * P + tid];
    }
  n = 0;
  for (int w = 0; w < NT / 64; ++w) n += s_n[w];
  int tot = c;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) tot += __shfl_xor(tot, o);
  if ((tid & 63) == 0) s_tot[tid >> 6] = tot;
  __syncthreads();
  tot = 0;
  for (int w = 0; w < NT / 64; ++w) tot += s_tot[w];
  const double load = tot > 0 ? static_cast<double>(c) / tot : 0.0;
  double term = c > 0 ? load * sum : (sum != sum ? sum : 0.0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) term += __shfl_xor(term, o);
  if ((tid & 63) == 0) s_red[tid >> 6] = term;
  __syncthreads();
  if (tid == 0) {
    double l = 0.0;
    for (int w = 0; w < NT / 64; ++w) l += s_red[w];
    a.loss[seq] = static_cast<float>(n > 0 ? l * E / n : 0.0);
  }
  if (tid < E) {
    a.counts[static_cast<int64_t>(seq) * E + tid] = c;
    if (a.slope) {  // E c and tot are whole numbers: 0 exactly where they are equal (49 * (1 / 49) is not 1)
      const double u = (static_cast<double>(E) * c - tot) / std::max(tot, 1);
      a.slope[static_cast<int64_t>(seq) * E + tid] = tot > 0 && n > 0 ? static_cast<float>(u / n) : 0.f;
    }
  }
}

// `rows` tokens of a sequence a workgroup, kTokens * 64 / SEG a wave at a time
// (their logits are loaded together); the shares' sums stay in registers, the
// counts in LDS.  With one chunk a sequence the workgroup goes on to the loss
// itself.  The logits are read once; latency and the exponentials bound it.  8
// sequences of 2048 tokens over 256 experts, sigmoid: 9.7 us, 1.7 TB/s (a token at
// a time in 128 workgroups 36.6; accurate expf and a second exponential for
// the sigmoid 11.9).
template <int DT, int SEG, int V>
__global__ __launch_bounds__(256) void k_balance_part(const BalanceArgs a) {
  constexpr int PW = 64 / SEG, kTokens = SEG == 16 ? 2 : 4;
  __shared__ float s_p[4 * PW * SEG * V];
  __shared__ int32_t s_c[257];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int seq = blockIdx.x / a.chunks, chunk = blockIdx.x - seq * a.chunks;
  const int E = a.E, e0 = V * (lane % SEG);
  const int t0 = chunk * a.rows, t1 = min(t0 + a.rows, a.T);
  const int64_t first = static_cast<int64_t>(seq) * a.T;
  for (int i = tid; i <= E; i += 256) s_c[i] = 0;
  __syncthreads();
  // counts: ids are few beside the logits
  for (uint32_t i = tid; i < static_cast<uint32_t>(t1 - t0) * a.K; i += 256) {
    const int id = a.idx[(first + t0) * a.K + i];
    const bool on = !a.mask || a.mask[first + t0 + i / static_cast<uint32_t>(a.K)];
    if (on && id >= 0 && id < E) atomicAdd(&s_c[id], 1);
  }
  // f32 sums of at most kRun trips (128 tokens a lane: 2^-17 of the sum), those in
  // 64 bits: a workgroup's tokens grow with the batch
  constexpr int kRun = 128 / kTokens;
  float sum[V];
  double runs[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sum[v] = 0.f;
    runs[v] = 0.0;
  }
  int n = 0, trips = 0;
  for (int t = t0 + wave * PW; t < t1; t += 4 * PW * kTokens) {  // uniform
    float z[kTokens][V];
    bool on[kTokens];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const int mine = t + u * 4 * PW + lane / SEG;
      const int64_t at = first + min(mine, t1 - 1);
      on[u] = mine < t1 && (!a.mask || a.mask[at]);
      load_row<DT, V>(a.logits, at * E, e0, E, a.vec, z[u]);
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      float p[V], rest[V];
      shares<SEG, V>(z[u], a.sigmoid, p, rest);
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] += on[u] ? p[v] : 0.f;  // a masked token's may be NaN
      n += on[u] && lane % SEG == 0 ? 1 : 0;
    }
    if (++trips == kRun) {  // uniform
      trips = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        runs[v] += static_cast<double>(sum[v]);
        sum[v] = 0.f;
      }
    }
  }
  if (n) atomicAdd(&s_c[E], n);
#pragma unroll
  for (int v = 0; v < V; ++v) s_p[(wave * PW + lane / SEG) * SEG * V + e0 + v] = static_cast<float>(runs[v] + static_cast<double>(sum[v]));
  __syncthreads();
  float all = 0.f;
  if (tid < E)
    for (int i = 0; i < 4 * PW; ++i) all += s_p[i * SEG * V + tid];
  if (a.chunks == 1) {
    __syncthreads();
    if (tid < E) s_p[tid] = all;
    __syncthreads();
    finish<256>(a, seq, 1, s_p, s_c);
    return;
  }
  if (tid < E) a.part_p[static_cast<int64_t>(blockIdx.x) * E + tid] = all;
  for (int i = tid; i <= E; i += 256) a.part_c[static_cast<int64_t>(blockIdx.x) * (E + 1) + i] = s_c[i];
}

// One workgroup a sequence; latency bounds it: 8 sequences of 64 chunks of 256
// experts 5.0-5.8 us.
__global__ __launch_bounds__(1024) void k_balance_loss(const BalanceArgs a) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * a.chunks;
  finish<1024>(a, blockIdx.x, a.chunks, a.part_p + at * a.E, a.part_c + at * (a.E + 1));
}

// Logits in, gradients out, 64 / SEG tokens a wave: bound by both.  16384 tokens
// over 256 experts, f32: 10.0 us, 3.4 TB/s (with expf and a division for
// 1 - sigmoid 14.7).
template <int DT, int SEG, int V>
__global__ __launch_bounds__(256) void k_balance_bwd(const BalanceArgs a, const float* __restrict__ d_loss,
                                                     void* __restrict__ d_logits) {
  constexpr int PW = 64 / SEG;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.E, e0 = V * (lane % SEG);
  const int64_t N = static_cast<int64_t>(a.S) * a.T;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * PW;
  if (t0 >= N) return;  // uniform
  const int64_t mine = t0 + lane / SEG, at = mine < N ? mine : N - 1;
  const int64_t seq = at / a.T;
  const bool on = !a.mask || a.mask[at];
  float z[V], p[V], rest[V], u[V];
  load_row<DT, V>(a.logits, at * E, e0, E, a.vec, z);
#pragma unroll
  for (int v = 0; v < V; ++v) u[v] = e0 + v < E ? a.slope[seq * E + e0 + v] : 0.f;
  const float dl = d_loss[seq];
  shares<SEG, V>(z, a.sigmoid, p, rest);
  float dot = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) dot = fmaf(p[v], u[v], dot);
  dot = seg_sum<SEG>(dot);
  float d[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    d[v] = dl * (p[v] * (u[v] - dot));
    if (a.sigmoid) d[v] *= rest[v];
    d[v] = on ? d[v] : 0.f;
  }
  if (mine >= N || e0 >= E) return;
  const int64_t o = mine * E + e0;
  if constexpr (V == 4) {
    if (a.vec) {
      if constexpr (DT == SMOE_F32) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(d_logits) + o) = f32x4{d[0], d[1], d[2], d[3]};
      } else if constexpr (DT == SMOE_BF16) {
        *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(d_logits) + o) =
            u32x2{pack_bf2(d[0], d[1]), pack_bf2(d[2], d[3])};
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) reinterpret_cast<_Float16*>(d_logits)[o + v] = static_cast<_Float16>(d[v]);
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (e0 + v >= E) continue;
    if constexpr (DT == SMOE_F32) reinterpret_cast<float*>(d_logits)[o + v] = d[v];
    else if constexpr (DT == SMOE_BF16) reinterpret_cast<uint16_t*>(d_logits)[o + v] = f2bf(d[v]);
    else reinterpret_cast<_Float16*>(d_logits)[o + v] = static_cast<_Float16>(d[v]);
  }
}

int rc() { return hipGetLastError() == hipSuccess ? SMOE_OK : SMOE_EHIP; }

// f(dtype, lanes of a token, experts of a lane)
template <typename F>
int by_shape(int dt, int E, F&& f) {
  auto lanes = [&](auto d) {
    using I1 = std::integral_constant<int, 1>;
    using I4 = std::integral_constant<int, 4>;
    if (E <= 16) return f(d, std::integral_constant<int, 16>{}, I1{});
    if (E <= 64) return f(d, std::integral_constant<int, 16>{}, I4{});
    if (E <= 128) return f(d, std::integral_constant<int, 32>{}, I4{});
    return f(d, std::integral_constant<int, 64>{}, I4{});
  };
  switch (dt) {
    case SMOE_F32: return lanes(std::integral_constant<int, SMOE_F32>{});
    case SMOE_BF16: return lanes(std::integral_constant<int, SMOE_BF16>{});
    case SMOE_F16: return lanes(std::integral_constant<int, SMOE_F16>{});
    default: return SMOE_EUNSUPPORTED;
  }
}

// whether rows of E logits load (and store) as vectors of four
bool vec4(const void* p, int dt, int E) {
  return E % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (dt == SMOE_F32 ? 16 : 8) == 0;
}

}  // namespace

// Tokens of a workgroup.  A short sequence is one launch, up to two times what a
// workgroup has in flight: 128 tokens of up to 64 experts (one launch 7.2 us, two
// 7.7), 64 of up to 128 (7.0 and 7.5), 32 of up to 256 (7.2 and 7.9; 64 tokens
// 10.9 and 8.0).  Else about 512 workgroups over the batch, and at least 32
// tokens each: 8 sequences of 2048 tokens over 256 experts, both kernels, 13.4 us
// (16 tokens each 14.1, 64 tokens 22.8).  At most 256 chunks a sequence, since one workgroup
// adds them up: 16384 tokens over 256 experts as one sequence 22.1 us (512 chunks
// 23.6, 128 chunks 32.2 before the shares had one exponential).
int balance_rows(int64_t S, int64_t T, int E) {
  const int64_t one = 2048 / (E <= 64 ? 16 : (E <= 128 ? 32 : 64));
  if (T <= one) return static_cast<int>(one);
  return static_cast<int>(std::max({int64_t{32}, (S * T + 511) / 512, (T + 255) / 256}));
}
int balance_chunks(int64_t S, int64_t T, int E) {
  const int64_t r = balance_rows(S, T, E);
  return static_cast<int>(std::max<int64_t>(1, (T + r - 1) / r));
}

int launch_balance_loss(const void* logits, int dt, int S, int T, int E, int K, int sigmoid, const int32_t* idx,
                        const uint8_t* mask, float* loss, int32_t* counts, float* slope, float* part_p,
                        int32_t* part_c, hipStream_t s) {
  const BalanceArgs a{logits, idx, mask, S, T, E, K, sigmoid != 0, vec4(logits, dt, E), balance_rows(S, T, E),
                      balance_chunks(S, T, E), part_p, part_c, loss, counts, slope};
  const int64_t grid = static_cast<int64_t>(S) * a.chunks;
  if (grid * 256 > 0xffffffffll) return SMOE_EINVAL;  // threads of a launch
  const int r = by_shape(dt, E, [&](auto d, auto seg, auto v) {
    hipLaunchKernelGGL((k_balance_part<decltype(d)::value, decltype(seg)::value, decltype(v)::value>),
                       dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
    return rc();
  });
  if (r != SMOE_OK || a.chunks == 1) return r;
  hipLaunchKernelGGL(k_balance_loss, dim3(S), dim3(1024), 0, s, a);
  return rc();
}

int launch_balance_loss_bwd(const void* logits, int dt, int S, int T, int E, int sigmoid, const uint8_t* mask,
                            const float* slope, const float* d_loss, void* d_logits, hipStream_t s) {
  BalanceArgs a{};
  a.logits = logits;
  a.mask = mask;
  a.S = S;
  a.T = T;
  a.E = E;
  a.sigmoid = sigmoid != 0;
  a.vec = vec4(logits, dt, E) && vec4(d_logits, dt, E);
  a.slope = const_cast<float*>(slope);
  return by_shape(dt, E, [&](auto d, auto seg, auto v) {
    constexpr int PW = 4 * (64 / decltype(seg)::value);
    const int64_t grid = (static_cast<int64_t>(S) * T + PW - 1) / PW;
    if (grid * 256 > 0xffffffffll) return static_cast<int>(SMOE_EINVAL);  // threads of a launch
    hipLaunchKernelGGL((k_balance_bwd<decltype(d)::value, decltype(seg)::value, decltype(v)::value>),
                       dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a, d_loss, d_logits);
    return rc();
  });
}

}  // namespace smoe

// Dispatch plans of small steps, made inside the launches of the block-scaled
// fp8 and microscaled 4-bit expert steps: in registers for a few entries, by bit
// masks for a decode step or a short prompt.
#pragma once
#include <algorithm>
#include <type_traits>

#include "smoe_common.hpp"
#include "smoe_fp8_blocks.hpp"
#include "smoe_routing.hpp"

namespace smoe {

constexpr int kTokensMax = 16;  // entries (and so tokens, experts and rows)

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

// words of 64 tokens an expert takes: an odd number
__host__ __device__ inline int prep_pitch(int N) { return ((N + 63) / 64) | 1; }

// The plan of a decode step or a short prompt (K <= KB, N <= 1024 T) by one
// workgroup of 1024 threads: the one smoe_dispatch_plan makes.
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
__device__ __forceinline__ void prep_plan(const PrepArgs& a) {
  extern __shared__ unsigned long long mask[];
  __shared__ int tot[kPlanMaxG], goff[kPlanMaxG + 1], wsum[4];
  const int tid = threadIdx.x;
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

// LDS of prep_plan
inline size_t prep_lds(const PrepArgs& a) {
  return std::max(static_cast<size_t>(a.E) * prep_pitch(a.N) * 10, static_cast<size_t>(a.N) * a.K * 6);
}
// f(KB, T) of the smallest prep_plan that takes N tokens of K slots (prep_fits)
template <typename F>
inline int by_prep(int N, int K, F&& f) {
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  using I8 = std::integral_constant<int, 8>;
  using I16 = std::integral_constant<int, 16>;
  if (N <= 1024) return K <= 2 ? f(I2{}, I1{}) : K <= 4 ? f(I4{}, I1{}) : K <= 8 ? f(I8{}, I1{}) : f(I16{}, I1{});
  if (N <= 2048) return K <= 2 ? f(I2{}, I2{}) : K <= 4 ? f(I4{}, I2{}) : f(I8{}, I2{});
  return K <= 2 ? f(I2{}, I4{}) : f(I4{}, I4{});
}

}  // namespace smoe

// Routing of tokens to experts, forward and backward.
//
//   s = softmax(z) or sigmoid(z) over a token's E experts,  c = s + bias (the bias steers the choice alone)
//   groups of E / G experts: kept are the G' groups with the largest sum of their `best` largest c
//   chosen: the k largest c of the kept groups, in falling order; equal ones by ascending number
//   w = scale s / sum of the chosen s (or scale s)
//   aux = aux_coef E sum_e f_e mean(s_e / sum s) + z_coef mean(logsumexp(z)^2),  f_e = share of all choices that fell on e
//
// LPT lanes share a token, each with VPL experts in registers (groups of four neighbours, so that the lanes' 16-byte
// loads join up). Few lanes per token keep the shuffles of the k arg-max rounds few; the rounds bound the kernel, not
// memory. The order must be that of the exact scores: without a bias it is that of the logits, which are compared as
// they are; with one, or for sums over a group, scores are compared in fp32, and a token where two neighbours of the
// order are nearer than fp32 errors is decided again in 64 bits.
#include "fmb_api.h"
#include "launch.cuh"
#include "rows.cuh"

namespace fmb {

constexpr int ROUTE_THREADS = 128;
constexpr int TAKEN = static_cast<int>(0x80000000);        // below the key of every value

struct RouteParams {
  const void* logits;
  long long ld, tokens;
  const float* bias;               // [E] or null
  float* weights;                  // [tokens, k]
  int* idx;                        // [tokens, k]
  int* counts;                     // [E], added to
  float* partial;                  // [blocks, E + 1]: sums of s / sum s and of lse^2, or null
  int E, k, softmax, groups, gsize, top_groups, best, renorm, vec;
  float scale;
};

// Whole numbers in the order of the values; NaN counts as the largest, -0 as 0.
__device__ __forceinline__ int order_key(float v) {
  v += 0.f;
  if (v != v) return 0x7fffffff;
  const int b = __float_as_int(v);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float order_value(int key) { return __int_as_float(key ^ ((key >> 31) & 0x7fffffff)); }

template <int LPT> __device__ __forceinline__ int expert_of(int i, int lane) { return (i >> 2) * (LPT * 4) + lane * 4 + (i & 3); }

template <typename T, int LPT, int VPL>
__device__ __forceinline__ void load_logits(const T* row, int lane, int E, int vec, float (&z)[VPL]) {
#pragma unroll
  for (int i = 0; i < VPL; i += 4) {
    const int e = expert_of<LPT>(i, lane);
    if (vec) {
      float f[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
      if (e < E) load_f32<T, 4>(row + e, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) z[i + j] = f[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[i + j] = e + j < E ? to_f32(row[e + j]) : -CUDART_INF_F;
    }
  }
}

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }

// A token's choice in 64 bits by its LPT lanes: writes the chosen experts to pick[0, k). Rare: the loops are plain.
template <typename T, int LPT>
__device__ __noinline__ void choose_exactly(const RouteParams& p, const T* row, int lane, double* c, double* g, int* pick) {
  double top = -CUDART_INF, sum = 0.0;
  if (p.softmax) {
    for (int e = lane; e < p.E; e += LPT) top = fmax(top, static_cast<double>(to_f32(row[e])));
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -CUDART_INF) top = 0.0;
    for (int e = lane; e < p.E; e += LPT) sum += exp(static_cast<double>(to_f32(row[e])) - top);
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum == 0.0) sum = 1.0;
  }
  for (int e = lane; e < p.E; e += LPT) {
    const double z = to_f32(row[e]);
    double v = (p.softmax ? exp(z - top) / sum : 1.0 / (1.0 + exp(-z))) + (p.bias != nullptr ? static_cast<double>(p.bias[e]) : 0.0);
    c[e] = v != v ? CUDART_INF : v;
  }
  __syncwarp();
  unsigned kept = 0xffffffffu;
  if (p.groups > 1) {
    for (int n = lane; n < p.groups; n += LPT) {
      double a = -CUDART_INF, b = -CUDART_INF;             // the two largest
      for (int e = n * p.gsize; e < (n + 1) * p.gsize; ++e) {
        if (c[e] > a) { b = a; a = c[e]; } else if (c[e] > b) b = c[e];
      }
      const double v = p.best > 1 && p.gsize > 1 ? a + b : a;
      g[n] = v != v ? CUDART_INF : v;
    }
    __syncwarp();
    kept = 0;
    for (int n = 0; n < p.groups; ++n) {
      int ahead = 0;
      for (int m = 0; m < p.groups; ++m) ahead += g[m] > g[n] || (g[m] == g[n] && m < n);
      if (ahead < p.top_groups) kept |= 1u << n;
    }
  }
  if (p.bias == nullptr)                                   // among the kept ones the order of the logits is the scores'
    for (int e = lane; e < p.E; e += LPT) {
      const double z = to_f32(row[e]);
      c[e] = z != z ? CUDART_INF : z;
    }
  double last = CUDART_INF;
  int last_e = -1;
  for (int j = 0; j < p.k; ++j) {
    double bv = -CUDART_INF;
    int be = 0x7fffffff;
    for (int e = lane; e < p.E; e += LPT) {
      const double v = c[e];
      const bool open = p.groups == 1 || (kept >> (e / p.gsize) & 1);
      const bool after = v < last || (v == last && e > last_e);
      if (open && after && (v > bv || (v == bv && e < be))) { bv = v; be = e; }
    }
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oe = __shfl_xor_sync(0xffffffffu, be, o);
      if (ov > bv || (ov == bv && oe < be)) { bv = ov; be = oe; }
    }
    if (lane == 0) pick[j] = be;
    last = bv;
    last_e = be;
  }
  __syncwarp();
}

template <typename T, int LPT, int VPL, bool AUX>
__global__ void __launch_bounds__(ROUTE_THREADS) route_fwd_kernel(const RouteParams p) {
  constexpr int TPB = ROUTE_THREADS / LPT;                 // tokens that a block has in hand
  constexpr int MOST_K = LPT * VPL < FMB_ROUTE_MAX_K ? LPT * VPL : FMB_ROUTE_MAX_K, PER = (MOST_K + LPT - 1) / LPT;
  extern __shared__ double s_mem[];                        // c in 64 bits [TPB, E] and of groups [TPB, groups], when needed
  __shared__ int s_pick[TPB][MOST_K + 1], s_key[TPB][MOST_K + 1];
  extern __shared__ int s_dyn[];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x % LPT, slot = threadIdx.x / LPT;
  const bool by_logit = p.bias == nullptr, check_order = !by_logit, grouped = p.groups > 1;
  const bool check_groups = grouped && !(by_logit && p.best == 1);
  const bool exact_too = check_order || check_groups;
  // How far a score in fp32 may be from the exact one, as a part of it: expf is within 2 units, the sum 1 + e and the
  // division within half of one each; a softmax divides by a sum of up to 512 terms, 35 roundings deep. Scores are at
  // most 1, so two scores of a group and two of another one are within 4 times that.
  const float off = p.softmax ? 2.6e-6f : 4e-7f;
  double* c64 = s_mem + static_cast<size_t>(slot) * p.E;
  double* g64 = s_mem + static_cast<size_t>(TPB) * p.E + slot * p.groups;
  float* c32 = reinterpret_cast<float*>(c64);              // read for the last time before the first store of 64 bits
  int* s_count = s_dyn + (exact_too || grouped ? 2 * TPB * (p.E + p.groups) : 0);            // [E]
  float* s_acc = reinterpret_cast<float*>(s_count + p.E);                             // [E + 1]
  for (int e = threadIdx.x; e < p.E; e += ROUTE_THREADS) s_count[e] = 0;
  if (AUX)
    for (int e = threadIdx.x; e <= p.E; e += ROUTE_THREADS) s_acc[e] = 0.f;
  __syncthreads();
  float acc[AUX ? VPL : 1], acc_z = 0.f;
#pragma unroll
  for (int i = 0; i < (AUX ? VPL : 1); ++i) acc[i] = 0.f;

  for (long long base = static_cast<long long>(blockIdx.x) * TPB; base < p.tokens; base += static_cast<long long>(gridDim.x) * TPB) {
    const bool live = base + slot < p.tokens;
    const long long token = live ? base + slot : p.tokens - 1;       // lanes without a token go along with the last one
    const T* row = static_cast<const T*>(p.logits) + token * p.ld;
    float z[VPL];
    load_logits<T, LPT, VPL>(row, lane, p.E, p.vec, z);
    float top = 0.f, mass = 1.f;
    if (p.softmax || AUX) {
      top = z[0];
#pragma unroll
      for (int i = 1; i < VPL; ++i) top = fmaxf(top, z[i]);
      top = lanes_max<LPT>(top);
      if (top == -CUDART_INF_F) top = 0.f;                  // a row of nothing but -inf: scores of 0
      mass = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) mass += expert_of<LPT>(i, lane) < p.E ? expf(z[i] - top) : 0.f;
      mass = lanes_sum<LPT>(mass);
      if (mass == 0.f) mass = 1.f;
    }
    if constexpr (AUX) {
      float norm = 1.f;
      if (!p.softmax) {
        norm = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) norm += expert_of<LPT>(i, lane) < p.E ? sigmoid(z[i]) : 0.f;
        norm = lanes_sum<LPT>(norm);
        if (norm == 0.f) norm = 1.f;
      }
      if (live) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (expert_of<LPT>(i, lane) < p.E) acc[i] += p.softmax ? expf(z[i] - top) / mass : sigmoid(z[i]) / norm;
        const float lse = top + logf(mass);
        if (lane == 0) acc_z += lse * lse;
      }
    }
    int key[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = expert_of<LPT>(i, lane);
      float c = z[i];
      if (!by_logit) c = (p.softmax ? expf(c - top) / mass : sigmoid(c)) + (e < p.E ? __ldg(p.bias + e) : 0.f);
      key[i] = e < p.E ? order_key(c) : TAKEN;
    }
    bool doubt = false;
    if (grouped) {
      // scores of the groups: each lane takes some of them from shared memory
      __syncwarp();
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = expert_of<LPT>(i, lane);
        if (e < p.E) {
          float c = order_value(key[i]);
          if (by_logit && p.best > 1) c = p.softmax ? expf(z[i] - top) / mass : sigmoid(z[i]);
          c32[e] = key[i] == 0x7fffffff ? CUDART_INF_F : c;
        }
      }
      __syncwarp();
      float* g32 = reinterpret_cast<float*>(g64);
      for (int n = lane; n < p.groups; n += LPT) {
        float a = -CUDART_INF_F, b = -CUDART_INF_F;
        for (int e = n * p.gsize; e < (n + 1) * p.gsize; ++e) {
          const float v = c32[e];
          b = fmaxf(b, fminf(a, v));
          a = fmaxf(a, v);
        }
        const float v = p.best > 1 && p.gsize > 1 ? a + b : a;
        g32[n] = v != v ? CUDART_INF_F : v;
      }
      __syncwarp();
      unsigned kept = 0;
      for (int n = lane; n < p.groups; n += LPT) {
        const float mine = g32[n];
        int ahead = 0;
        for (int m = 0; m < p.groups; ++m) {
          const float v = g32[m];
          ahead += v > mine || (v == mine && m < n);
          if (check_groups && m != n) doubt |= !(fabsf(v - mine) > 4.f * off + 2.4e-7f * (fabsf(v) + fabsf(mine)));
        }
        if (ahead < p.top_groups) kept |= 1u << n;
      }
#pragma unroll
      for (int o = LPT / 2; o > 0; o >>= 1) kept |= __shfl_xor_sync(0xffffffffu, kept, o);
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = expert_of<LPT>(i, lane);
        if (e < p.E && !(kept >> (e / p.gsize) & 1)) key[i] = TAKEN;
      }
    }
    // k rounds of arg-max, and one more to see how far behind the next one is
    const int rounds = check_order ? p.k + 1 : p.k;
    for (int j = 0; j < rounds; ++j) {
      int bk = TAKEN, be = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (key[i] > bk) { bk = key[i]; be = expert_of<LPT>(i, lane); }
#pragma unroll
      for (int o = LPT / 2; o > 0; o >>= 1) {
        const int ok = __shfl_xor_sync(0xffffffffu, bk, o), oe = __shfl_xor_sync(0xffffffffu, be, o);
        if (ok > bk || (ok == bk && oe < be)) { bk = ok; be = oe; }
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (expert_of<LPT>(i, lane) == be) key[i] = TAKEN;
      if (lane == 0) { s_pick[slot][j] = be; s_key[slot][j] = bk; }
    }
    __syncwarp();
    if (check_order) {
      for (int j = lane; j < p.k; j += LPT) {
        const int ka = s_key[slot][j], kb = s_key[slot][j + 1];
        if (kb == TAKEN) continue;                          // every expert is chosen
        const int ea = s_pick[slot][j], eb = s_pick[slot][j + 1];
        const float a = order_value(ka), b = order_value(kb), ba = p.bias[ea], bb = p.bias[eb];
        const bool near = !(a - b > off * (fabsf(a - ba) + fabsf(b - bb)) + 1.2e-7f * (fabsf(a) + fabsf(b)) + 1e-37f);
        const bool same = j + 1 < p.k && ka == kb && ba == bb && to_f32(row[ea]) == to_f32(row[eb]);    // in any precision
        doubt |= near && !same;
      }
    }
    if (exact_too) {
      unsigned who = __ballot_sync(0xffffffffu, doubt);
      if (who) {                                            // some token of this warp: all its lanes go, the others keep theirs
        const unsigned seg = LPT == 32 ? 0xffffffffu : ((1u << LPT) - 1u) << (threadIdx.x % 32 / LPT * LPT);
        const bool mine = (who & seg) != 0;
        int keep[PER];
#pragma unroll
        for (int n = 0; n < PER; ++n) keep[n] = n * LPT + lane < p.k ? s_pick[slot][n * LPT + lane] : 0;
        __syncwarp();
        choose_exactly<T, LPT>(p, row, lane, c64, g64, s_pick[slot]);
        if (!mine) {
#pragma unroll
          for (int n = 0; n < PER; ++n)
            if (n * LPT + lane < p.k) s_pick[slot][n * LPT + lane] = keep[n];
        }
        __syncwarp();
      }
    }
    // weights of the chosen, each by a lane of its own
    float sum = 0.f, best = -CUDART_INF_F, chosen[PER];
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int j = n * LPT + lane;
      chosen[n] = j < p.k ? to_f32(row[s_pick[slot][j]]) : -CUDART_INF_F;
      best = fmaxf(best, chosen[n]);
    }
    best = lanes_max<LPT>(best);
    // shares of the chosen alone are taken around their own maximum: they may all lie far below the row's
    const float from = !p.renorm ? top : best == -CUDART_INF_F ? 0.f : best;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      if (n * LPT + lane < p.k) {
        chosen[n] = p.softmax ? expf(chosen[n] - from) / (p.renorm ? 1.f : mass) : sigmoid(chosen[n]);
        sum += chosen[n];
      }
    }
    sum = lanes_sum<LPT>(sum);
    if (!p.softmax && p.renorm && __any_sync(0xffffffffu, sum < 1e-30f && best > -CUDART_INF_F)) {
      // sigmoids that vanish in fp32 still have shares: s = e^z there
      float far = 0.f;
#pragma unroll
      for (int n = 0; n < PER; ++n)
        if (n * LPT + lane < p.k) far += expf(to_f32(row[s_pick[slot][n * LPT + lane]]) - from);
      far = lanes_sum<LPT>(far);
      if (sum < 1e-30f && best > -CUDART_INF_F) {
#pragma unroll
        for (int n = 0; n < PER; ++n)
          if (n * LPT + lane < p.k) chosen[n] = expf(to_f32(row[s_pick[slot][n * LPT + lane]]) - from);
        sum = far;
      }
    }
    const float by = !p.renorm ? p.scale : sum == 0.f ? 0.f : p.scale / sum;      // nothing to share out: weights of 0
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int j = n * LPT + lane;
      if (j < p.k && live) {
        const int e = s_pick[slot][j];
        p.weights[token * p.k + j] = chosen[n] * by;
        p.idx[token * p.k + j] = e;
        atomicAdd(&s_count[e], 1);
      }
    }
    __syncwarp();
  }
  if constexpr (AUX) {
    for (int who = 0; who < TPB; ++who) {                   // tokens' sums one slot after another: a fixed order
      __syncthreads();
      if (slot == who) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (expert_of<LPT>(i, lane) < p.E) s_acc[expert_of<LPT>(i, lane)] += acc[i];
        if (lane == 0) s_acc[p.E] += acc_z;
      }
    }
  }
  __syncthreads();
  if (AUX)
    for (int e = threadIdx.x; e <= p.E; e += ROUTE_THREADS) p.partial[static_cast<long long>(blockIdx.x) * (p.E + 1) + e] = s_acc[e];
  for (int e = threadIdx.x; e < p.E; e += ROUTE_THREADS)
    if (s_count[e]) atomicAdd(p.counts + e, s_count[e]);    // whole numbers: the order does not matter
}

// aux from the blocks' sums and the counts: one block, 32 columns x 32 groups of rows at a time.
__global__ void __launch_bounds__(1024)
route_aux_kernel(const float* __restrict__ partial, const int* __restrict__ counts, float* __restrict__ aux, int blocks, int E,
                 long long tokens, int k, float aux_coef, float z_coef) {
  __shared__ float red[32][33];
  __shared__ float s_part[32];
  pdl_wait();
  pdl_launch_dependents();
  float out = 0.f;                                          // of lane 0 of each warp: its columns' terms
  const float inv_n = 1.f / static_cast<float>(tokens);
  for (int c0 = 0; c0 <= E; c0 += 32) {
    const int c = c0 + threadIdx.x;
    float s = 0.f;
    if (c <= E)
      for (int r = threadIdx.y; r < blocks; r += 32) s += partial[static_cast<long long>(r) * (E + 1) + c];
    __syncthreads();
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = lanes_sum<32>(red[threadIdx.x][threadIdx.y]);
    const int mine = c0 + threadIdx.y;
    if (mine < E) {
      const float f = static_cast<float>(counts[mine]) / (static_cast<float>(tokens) * static_cast<float>(k));
      out += aux_coef * static_cast<float>(E) * f * (s * inv_n);
    } else if (mine == E) {
      out += z_coef * (s * inv_n);
    }
  }
  if (threadIdx.x == 0) s_part[threadIdx.y] = out;
  __syncthreads();
  if (threadIdx.y == 0) {
    out = lanes_sum<32>(s_part[threadIdx.x]);
    if (threadIdx.x == 0) *aux = out;
  }
}

struct RouteGrad {
  const void* logits;
  long long ld, tokens;
  const float* weights;            // of the forward pass
  const int* idx;
  const float* dweights;           // [tokens, k] or null
  const float* daux;               // one number or null
  const int* counts;
  void* dlogits;                   // [tokens, E] contiguous
  int E, k, softmax, renorm, vec;
  float scale, aux_coef, z_coef;
};

// Gradient of the logits. Of renormalised softmax weights and of sigmoid scores it is zero but for the chosen experts
// (DENSE false: zeros and k values per token, the logits' rows are not read); otherwise every expert has one.
template <typename T, int LPT, int VPL, bool DENSE>
__global__ void __launch_bounds__(ROUTE_THREADS) route_bwd_kernel(const RouteGrad p) {
  constexpr int TPB = ROUTE_THREADS / LPT;
  constexpr int MOST_K = LPT * VPL < FMB_ROUTE_MAX_K ? LPT * VPL : FMB_ROUTE_MAX_K, PER = (MOST_K + LPT - 1) / LPT;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x % LPT;
  const long long token0 = static_cast<long long>(blockIdx.x) * TPB + threadIdx.x / LPT;
  const bool live = token0 < p.tokens;
  const long long token = live ? token0 : p.tokens - 1;
  const T* row = static_cast<const T*>(p.logits) + token * p.ld;
  T* out = static_cast<T*>(p.dlogits) + token * p.E;
  // the chosen experts' scores and the gradient of the scores
  int e[PER];
  float w[PER], dw[PER], s[PER];
  float dot = 0.f;
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int j = n * LPT + lane;
    e[n] = -1;
    w[n] = dw[n] = s[n] = 0.f;
    if (j < p.k) {
      e[n] = p.idx[token * p.k + j];
      w[n] = p.weights[token * p.k + j];
      dw[n] = p.dweights != nullptr ? p.dweights[token * p.k + j] : 0.f;
      if (!p.softmax) s[n] = sigmoid(to_f32(row[e[n]]));
      dot += w[n] * dw[n];
    }
  }
  dot = lanes_sum<LPT>(dot);
  float dz[PER];                                            // the part of the weights, on the chosen experts
  float flow = 0.f;                                         // not renormalised softmax: sum of w dw, which all experts share
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    // d w_j / d s_i = scale (delta_ij - s_j / S) / S and d s / d z = s (s (1 - s)): both leave a factor w_j
    dz[n] = w[n] * (p.renorm ? (p.scale == 0.f ? 0.f : dw[n] - dot / p.scale) : dw[n]);
    if (!p.softmax) dz[n] *= 1.f - s[n];
  }
  if (p.softmax && !p.renorm) flow = dot;
  if constexpr (!DENSE) {
#pragma unroll
    for (int i = 0; i < VPL; i += 4) {
      const int at = expert_of<LPT>(i, lane);
      if (p.vec) {
        if (live && at < p.E) {
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(out + at) = make_uint4(0, 0, 0, 0);
          else *reinterpret_cast<uint2*>(out + at) = make_uint2(0, 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (live && at + j < p.E) out[at + j] = from_f32<T>(0.f);
      }
    }
    __syncwarp();
#pragma unroll
    for (int n = 0; n < PER; ++n)
      if (live && e[n] >= 0) out[e[n]] = from_f32<T>(dz[n]);
  } else {
    float z[VPL];
    load_logits<T, LPT, VPL>(row, lane, p.E, p.vec, z);
    float top = z[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) top = fmaxf(top, z[i]);
    top = lanes_max<LPT>(top);
    if (top == -CUDART_INF_F) top = 0.f;
    float mass = 0.f, norm = 0.f, pull = 0.f;
    const float up = p.daux != nullptr ? *p.daux : 0.f;
    const float per_f = up * p.aux_coef * static_cast<float>(p.E) / (static_cast<float>(p.tokens) * static_cast<float>(p.tokens) * static_cast<float>(p.k));
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int at = expert_of<LPT>(i, lane);
      if (at < p.E) {
        const float x = expf(z[i] - top);
        mass += x;
        const float share = p.softmax ? x : sigmoid(z[i]);
        norm += share;
        pull += share * static_cast<float>(__ldg(p.counts + at));
      }
    }
    mass = lanes_sum<LPT>(mass);
    norm = lanes_sum<LPT>(norm);
    if (mass == 0.f) mass = 1.f;                            // as in the forward pass: scores of 0
    if (norm == 0.f) norm = 1.f;
    pull = lanes_sum<LPT>(pull) / norm;                     // mean count under the token's shares
    const float zt = up * p.z_coef * 2.f / static_cast<float>(p.tokens) * (top + logf(mass));
    auto whole = [&](float v, int at) {                     // what an expert's logit gets without the chosen one's own part
      const float x = expf(v - top) / mass;
      const float ds = per_f * (static_cast<float>(__ldg(p.counts + at)) - pull);
      if (p.softmax) return x * (ds - flow + zt);
      const float sg = sigmoid(v);
      return ds / norm * sg * (1.f - sg) + x * zt;
    };
#pragma unroll
    for (int i = 0; i < VPL; i += 4) {
      const int at = expert_of<LPT>(i, lane);
      if (live) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = at + j < p.E ? whole(z[i + j], at + j) : 0.f;
        if (p.vec) {
          if (at < p.E) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + at) = make_float4(f[0], f[1], f[2], f[3]);
            else {
              const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
              *reinterpret_cast<uint2*>(out + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at + j < p.E) out[at + j] = from_f32<T>(f[j]);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int n = 0; n < PER; ++n)
      if (live && e[n] >= 0) out[e[n]] = from_f32<T>(whole(to_f32(row[e[n]]), e[n]) + dz[n]);
  }
}

template <typename T, int LPT, int VPL>
int route_fwd_run(const RouteParams& p, int blocks, cudaStream_t stream) {
  constexpr int TPB = ROUTE_THREADS / LPT;
  const bool room = p.bias != nullptr || p.groups > 1;
  const size_t smem = (room ? sizeof(double) * TPB * (p.E + p.groups) : 0) + sizeof(int) * (2 * p.E + 1);
  auto kernel = p.partial != nullptr ? route_fwd_kernel<T, LPT, VPL, true> : route_fwd_kernel<T, LPT, VPL, false>;
  // at most 16 (256 + 32) or 8 (512 + 32) values of 64 bits: with the static arrays below the 48 KB that need no opting in
  return launch_pdl(kernel, dim3(blocks), dim3(ROUTE_THREADS), smem, stream, p) == cudaSuccess ? 0 : -3;
}

template <typename T, int LPT, int VPL> int route_bwd_run(const RouteGrad& p, bool dense, cudaStream_t stream) {
  constexpr int TPB = ROUTE_THREADS / LPT;
  const dim3 grid(static_cast<unsigned>((p.tokens + TPB - 1) / TPB));
  const cudaError_t e = dense ? launch_pdl(route_bwd_kernel<T, LPT, VPL, true>, grid, dim3(ROUTE_THREADS), 0, stream, p)
                              : launch_pdl(route_bwd_kernel<T, LPT, VPL, false>, grid, dim3(ROUTE_THREADS), 0, stream, p);
  return e == cudaSuccess ? 0 : -3;
}

// lanes per token by the number of experts
inline int route_lanes(int E) { return E <= 8 ? 1 : E <= 16 ? 2 : E <= 32 ? 4 : E <= 256 ? 8 : 16; }

}  // namespace fmb

using namespace fmb;

extern "C" int fmb_route_blocks(long long tokens, int E) {
  const int per = ROUTE_THREADS / route_lanes(E);
  const long long need = (tokens + per - 1) / per, most = 4LL * sm_count();
  return static_cast<int>(need < 1 ? 1 : need < most ? need : most);
}

#define FMB_ROUTE(T, RUN, ...)                                       \
  do {                                                               \
    if (E <= 8) return RUN<T, 1, 8>(__VA_ARGS__);                    \
    if (E <= 16) return RUN<T, 2, 8>(__VA_ARGS__);                   \
    if (E <= 32) return RUN<T, 4, 8>(__VA_ARGS__);                   \
    if (E <= 64) return RUN<T, 8, 8>(__VA_ARGS__);                   \
    if (E <= 128) return RUN<T, 8, 16>(__VA_ARGS__);                 \
    if (E <= 256) return RUN<T, 8, 32>(__VA_ARGS__);                 \
    return RUN<T, 16, 32>(__VA_ARGS__);                              \
  } while (0)

extern "C" int fmb_route_fwd(const void* logits, long long ld, int dtype, const float* bias, float* weights, int* idx,
                             int* counts, float* partial, float* aux, long long tokens, int E, int k, int softmax, int groups,
                             int top_groups, int best, int renorm, float scale, float aux_coef, float z_coef, int blocks,
                             cudaStream_t stream) {
  if (E < 1 || E > FMB_ROUTE_MAX_EXPERTS || k < 1 || k > FMB_ROUTE_MAX_K || k > E || groups < 1 || groups > 32 || E % groups ||
      top_groups < 1 || top_groups > groups || k > E / groups * top_groups || best < 1 || best > 2 || blocks < 1)
    return -2;
  if (cudaMemsetAsync(counts, 0, E * sizeof(int), stream) != cudaSuccess) return -3;
  if (tokens <= 0) return 0;
  RouteParams p = {};
  p.logits = logits; p.ld = ld; p.tokens = tokens; p.bias = bias; p.weights = weights; p.idx = idx; p.counts = counts;
  p.partial = partial; p.E = E; p.k = k; p.softmax = softmax; p.groups = groups; p.gsize = E / groups; p.top_groups = top_groups;
  p.best = best; p.renorm = renorm; p.scale = scale;
  p.vec = E % 4 == 0 && ld % 4 == 0 && aligned16(logits);
  int rc = -1;
  if (dtype == FMB_BF16) rc = [&]() -> int { FMB_ROUTE(__nv_bfloat16, route_fwd_run, p, blocks, stream); }();
  else if (dtype == FMB_F32) rc = [&]() -> int { FMB_ROUTE(float, route_fwd_run, p, blocks, stream); }();
  if (rc != 0 || partial == nullptr) return rc;
  return launch_pdl(route_aux_kernel, dim3(1), dim3(32, 32), 0, stream, partial, counts, aux, blocks, E, tokens, k, aux_coef,
                    z_coef) == cudaSuccess ? 0 : -3;
}

extern "C" int fmb_route_bwd(const void* logits, long long ld, int dtype, const float* weights, const int* idx,
                             const float* dweights, const float* daux, const int* counts, void* dlogits, long long tokens, int E,
                             int k, int softmax, int renorm, float scale, float aux_coef, float z_coef, cudaStream_t stream) {
  if (E < 1 || E > FMB_ROUTE_MAX_EXPERTS || k < 1 || k > FMB_ROUTE_MAX_K || k > E) return -2;
  if (tokens <= 0) return 0;
  RouteGrad p = {};
  p.logits = logits; p.ld = ld; p.tokens = tokens; p.weights = weights; p.idx = idx; p.dweights = dweights; p.daux = daux;
  p.counts = counts; p.dlogits = dlogits; p.E = E; p.k = k; p.softmax = softmax; p.renorm = renorm; p.scale = scale;
  p.aux_coef = aux_coef; p.z_coef = z_coef;
  p.vec = E % 4 == 0 && ld % 4 == 0 && aligned16(logits) && aligned16(dlogits);
  const bool dense = daux != nullptr || (softmax && !renorm);
  if (dtype == FMB_BF16) FMB_ROUTE(__nv_bfloat16, route_bwd_run, p, dense, stream);
  if (dtype == FMB_F32) FMB_ROUTE(float, route_bwd_run, p, dense, stream);
  return -1;
}

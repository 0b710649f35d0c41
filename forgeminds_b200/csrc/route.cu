// Routing of tokens to experts, forward and backward.
//
//   s = softmax(z) or sigmoid(z) over a token's E experts,  c = s + bias (the bias steers the choice alone)
//   groups of E / G experts: kept are the G' groups with the largest sum of their `best` largest c
//   chosen: the k largest c of the kept groups, in falling order; equal ones by ascending number
//   w = scale s / sum of the chosen s (or scale s)
//   aux = aux_coef E sum_e f_e mean(s_e / sum s) + z_coef mean(logsumexp(z)^2),  f_e = share of all choices that fell on e
//
// Forward: LPT lanes share a token, each with VPL neighbouring experts. The order must be that of the exact scores. What
// is compared are whole numbers of 32 bits: 23 bits of the score in fixed point, 9 of the expert's number, so that one
// maximum finds value and expert and no two are equal. Each lane lists its four largest by a network once; a round of the
// choice is then a maximum over the lanes' first ones. A token where two neighbours of the order are nearer than the errors
// of score and fixed point, and not equal by their inputs, is decided again, in 64 bits where it must be; so is one with NaN
// or +inf, and one of which a lane has given away its four.
// Bound by these instructions (600 per token of 256 experts in 8 groups and 8 choices), not by memory: 65536 such tokens in
// 58 us at two thirds of the issue slots, 17 us of memory traffic; their backward pass, all zeros but for 8 values, 16 us. With
// the auxiliary losses, whose gradient is dense, 152 and 126 us (two accurate exponentials an expert each).
#include "fmb_api.h"
#include "launch.cuh"
#include "rows.cuh"

namespace fmb {

constexpr int ROUTE_THREADS = 128;
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

// A token's choice in 64 bits by its LPT lanes: writes the chosen experts to pick[0, k). c, g: shared memory for E scores
// and the groups'. Rare, and tens of thousands of cycles long: a pair of neighbours alone is put in order without it.
template <typename T, int LPT, int VPL>
__device__ __forceinline__ void choose_exactly(const RouteParams& p, const T* row, int lane, double* c, double* g, int* pick) {
  const int e0 = lane * VPL;
  double own[VPL];
  double top = -CUDART_INF, sum = 0.0;
  unsigned open = 0;                                       // experts of this lane that can be chosen
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    own[i] = e0 + i < p.E ? static_cast<double>(to_f32(row[e0 + i])) : -CUDART_INF;
    if (e0 + i < p.E) open |= 1u << i;
    top = fmax(top, own[i]);
  }
  if (p.softmax) {
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -CUDART_INF) top = 0.0;
#pragma unroll 1
    for (int e = lane; e < p.E; e += LPT) sum += exp(static_cast<double>(to_f32(row[e])) - top);
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum == 0.0) sum = 1.0;
  }
  auto biased = [&](int e) {                               // NaN is the largest
    const double v = c[e] + (p.bias != nullptr ? static_cast<double>(p.bias[e]) : 0.0);
    return v != v ? CUDART_INF : v;
  };
  if (p.bias != nullptr || p.groups > 1) {
#pragma unroll 1
    for (int e = lane; e < p.E; e += LPT) {
      const double z = to_f32(row[e]);
      c[e] = p.softmax ? exp(z - top) / sum : 1.0 / (1.0 + exp(-z));
    }
    __syncwarp();
  }
  if (p.groups > 1) {
    for (int n = lane; n < p.groups; n += LPT) {
      double a = -CUDART_INF, b = -CUDART_INF;             // the two largest, and where they are
      int at_a = n * p.gsize, at_b = p.gsize > 1 ? at_a + 1 : at_a;
      for (int e = n * p.gsize; e < (n + 1) * p.gsize; ++e) {
        const double v = biased(e);
        if (v > a || e == n * p.gsize) {
          b = a;
          at_b = e == n * p.gsize ? at_b : at_a;
          a = v;
          at_a = e;
        } else if (v > b || e == n * p.gsize + 1) {
          b = v;
          at_b = e;
        }
      }
      // scores and biases are added apart: groups with the same logits and the same biases in another order are equal
      double v = a;
      if (p.best > 1 && p.gsize > 1) {
        v = c[at_a] + c[at_b];
        if (p.bias != nullptr) v += static_cast<double>(p.bias[at_a]) + static_cast<double>(p.bias[at_b]);
      }
      g[n] = v != v ? CUDART_INF : v;
    }
    __syncwarp();
    unsigned kept = 0;
    for (int n = lane; n < p.groups; n += LPT) {
      int ahead = 0;
      for (int m = 0; m < p.groups; ++m) ahead += g[m] > g[n] || (g[m] == g[n] && m < n);
      if (ahead < p.top_groups) kept |= 1u << n;
    }
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) kept |= __shfl_xor_sync(0xffffffffu, kept, o);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (e0 + i < p.E && !(kept >> ((e0 + i) / p.gsize) & 1)) open &= ~(1u << i);
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {                          // without a bias the order of the logits is the scores'
    if (p.bias != nullptr && e0 + i < p.E) own[i] = biased(e0 + i);
    if (own[i] != own[i]) own[i] = CUDART_INF;
  }
  for (int j = 0; j < p.k; ++j) {
    double bv = -CUDART_INF;
    int be = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if ((open >> i & 1) && (own[i] > bv || be == 0x7fffffff)) { bv = own[i]; be = e0 + i; }
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oe = __shfl_xor_sync(0xffffffffu, be, o);
      if (ov > bv || (ov == bv && oe < be)) { bv = ov; be = oe; }
    }
    if (lane == 0) pick[j] = be;
    if (be >= e0 && be < e0 + VPL) open &= ~(1u << (be - e0));
  }
  __syncwarp();
}

// 1 / (1 + e^-z) for comparisons: within 6e-7 (2^x to 2^-22, its argument to a unit, one addition, one reciprocal)
__device__ __forceinline__ float sigmoid_near(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + exp2_unit(z * -1.4426950408889634f)));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr int NUMBER_BITS = 9, FIXED = 1 << 23;            // a key: 23 bits of score, then 511 - expert
constexpr unsigned NUMBER = (1u << NUMBER_BITS) - 1;
// y up to 2^24 - 1, from 2^23 on rounded to a whole number by the addition that brought it there; less (or NaN) counts as 2^23
__device__ __forceinline__ unsigned route_key(float y, int e) {
  return (__float_as_uint(fmaxf(y, 8388608.f)) << NUMBER_BITS) + (NUMBER - e);
}
__device__ __forceinline__ unsigned key_score(unsigned key) { return key >> NUMBER_BITS; }
__device__ __forceinline__ int key_expert(unsigned key) { return NUMBER - (key & NUMBER); }

template <int W> __device__ __forceinline__ unsigned lanes_umax(unsigned v) {
  if constexpr (W == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Falling order of N keys in registers: Batcher's merge exchange, no branches (19 exchanges for 8, 63 for 16).
template <int N> __device__ __forceinline__ void sort_falling(unsigned (&v)[N]) {
  if constexpr (N > 1)
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const unsigned a = v[i + j], b = v[i + j + k];
            v[i + j] = max(a, b);
            v[i + j + k] = min(a, b);
          }
}

// The four largest (or all, of fewer) in falling order: fours sorted, then merged with the best four so far (32 minima and
// maxima for 8, where the whole order takes 38; and the rounds move four registers, not eight).
constexpr int LIST = 4;
template <int N, int L> __device__ __forceinline__ void top_falling(const unsigned (&v)[N], unsigned (&list)[L]) {
  static_assert(L == (N < LIST ? N : LIST) && (N <= LIST || N % LIST == 0), "whole fours");
#pragma unroll
  for (int i = 0; i < L; ++i) list[i] = v[i];
  sort_falling(list);
#pragma unroll
  for (int from = L; from < N; from += L) {
    unsigned more[L];
#pragma unroll
    for (int i = 0; i < L; ++i) more[i] = v[from + i];
    sort_falling(more);
#pragma unroll
    for (int i = 0; i < L; ++i) list[i] = max(list[i], more[L - 1 - i]);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (!(i & o)) {
          const unsigned a = list[i], b = list[i + o];
          list[i] = max(a, b);
          list[i + o] = min(a, b);
        }
  }
}

// VPL neighbouring experts' logits; -inf where there is none
template <typename T, int VPL> __device__ __forceinline__ void load_own(const T* row, int e0, int E, int vec, float (&z)[VPL]) {
  constexpr int BYTES = VPL * sizeof(T);
  if (vec) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) z[i] = -CUDART_INF_F;
    if (e0 < E) {
      if constexpr (BYTES >= 16) load_f32<T, VPL>(row + e0, z);
      else if constexpr (BYTES == 8 && sizeof(T) == 4) {
        const float2 f = __ldg(reinterpret_cast<const float2*>(row + e0));
        z[0] = f.x; z[1] = f.y;
      } else if constexpr (BYTES == 8) load_f32<T, 4>(row + e0, z);
      else if constexpr (BYTES == 4 && sizeof(T) == 2) {
        const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(row + e0));
        z[0] = __uint_as_float(u << 16); z[1] = __uint_as_float(u & 0xffff0000u);
      } else z[0] = to_f32(row[e0]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) z[i] = e0 + i < E ? to_f32(row[e0 + i]) : -CUDART_INF_F;
  }
}

// Keys of a lane's experts by their scores, and by their logits (without a bias the order is the same). bias: in fixed
// point. fp32 logits: 32 units below the largest one in 23 bits.
template <int VPL>
__device__ __forceinline__ void keys_by_score(bool softmax, const float (&z)[VPL], const float (&bias)[VPL], float top, float inv_mass,
                                              float unit, int e0, unsigned (&key)[VPL]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const float c = softmax ? exp2_unit((z[i] - top) * 1.4426950408889634f) * inv_mass : sigmoid_near(z[i]);
    key[i] = route_key(fmaf(c, unit, bias[i]), e0 + i);
  }
}
// bf16: the 16 bits themselves, turned so that their order is the numbers' (and -0 is 0): no two logits share a score.
template <typename T, int VPL>
__device__ __forceinline__ void keys_by_logit(const float (&z)[VPL], float high, int e0, unsigned (&key)[VPL]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if constexpr (sizeof(T) == 2) {
      const unsigned b = __float_as_uint(z[i] + 0.f);
      key[i] = ((b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u)) >> 16 << NUMBER_BITS) + (NUMBER - (e0 + i));
    } else {
      key[i] = route_key(fmaf(z[i] - high, 262144.f, 16777215.f), e0 + i);
    }
  }
}
__device__ __forceinline__ float fixed_bias(float bias, float lo, float unit) { return fmaf(bias - lo, unit, 8388608.f); }

// One round of a choice: the largest first key of LPT lanes, whose lane moves on to its next one.
template <int LPT, int N> __device__ __forceinline__ unsigned take_largest(unsigned (&list)[N]) {
  const unsigned w = lanes_umax<LPT>(list[0]);
  if (list[0] == w) {
#pragma unroll
    for (int i = 0; i + 1 < N; ++i) list[i] = list[i + 1];
    list[N - 1] = 0;
  }
  return w;
}

// Whether expert b comes before expert a by their exact scores (sigmoids with their biases).
__device__ __forceinline__ bool sigmoid_ahead(float za, float zb, float bias_a, float bias_b, bool lower) {
  const double a = 1.0 / (1.0 + exp(-static_cast<double>(za))) + static_cast<double>(bias_a);
  const double b = 1.0 / (1.0 + exp(-static_cast<double>(zb))) + static_cast<double>(bias_b);
  return b > a || (b == a && lower);
}

// The same for softmax scores with their biases, from the row's largest logit and its fp32 sum of exponentials: 1 and 0, or
// -1 where the sum's error (of some 25 roundings, and of the terms' own 2e-7: 2e-6, taken twice) leaves it open.
__device__ __forceinline__ int softmax_ahead(float za, float zb, float bias_a, float bias_b, float top, float mass) {
  const double s = (exp(static_cast<double>(zb) - top) - exp(static_cast<double>(za) - top)) / mass;
  const double ahead = s + (static_cast<double>(bias_b) - static_cast<double>(bias_a));
  return fabs(ahead) > 4e-6 * fabs(s) + 1e-14 ? ahead > 0.0 : -1;
}

// The choice of a warp's tokens where some neighbours j, j + 1 of key[0, k + 2) are closer than `apart`, or a token is in
// doubt already: pairs that stand alone are put in order, other tokens decided again. Writes pick[0, k).
template <typename T, int LPT, int VPL>
__device__ __forceinline__ void settle(const RouteParams& p, const T* row, int lane, unsigned apart, bool doubt, bool flat_bias,
                                       float top, float mass,
                                       const unsigned* key, int* pick, double* c64, double* g64) {
  const bool biased = p.bias != nullptr;
  auto close = [&](int j) { return key[j] != 0 && key[j + 1] != 0 && key_score(key[j]) - key_score(key[j + 1]) < apart; };
  for (int j = lane; j < p.k; j += LPT) pick[j] = min(key_expert(key[j]), p.E - 1);
  __syncwarp();
  for (int j = lane; j < p.k; j += LPT) {
    doubt |= key[j] == 0;                                  // fewer keys than choices
    if (!close(j)) continue;
    const int a = key_expert(key[j]), b = key_expert(key[j + 1]);
    const float za = to_f32(row[a]), zb = to_f32(row[b]);
    if (za == zb && (!biased || p.bias[a] == p.bias[b])) {
      // equal in any precision, and the lower number is first; at the last choice the next one might belong before both
      doubt |= j == p.k - 1 && close(j + 1);
    } else if ((j > 0 && close(j - 1)) || close(j + 1)) {
      doubt = true;
    } else {
      const int ahead = !biased ? zb > za || (zb == za && b < a)
                        : p.softmax ? softmax_ahead(za, zb, p.bias[a], p.bias[b], top, mass)
                                    : sigmoid_ahead(za, zb, p.bias[a], p.bias[b], b < a);
      doubt |= ahead < 0;
      if (ahead > 0) {
        pick[j] = b;
        if (j + 1 < p.k) pick[j + 1] = a;
      }
    }
  }
  __syncwarp();
  unsigned who = __ballot_sync(0xffffffffu, doubt);
  if (who == 0) return;
  // a row of one logit throughout (an untrained router, a padded token) is in order as it is, with equal biases
  bool flat = flat_bias;
  for (int e = lane; e < p.E; e += LPT) flat &= to_f32(row[e]) == to_f32(row[0]);
  who = __ballot_sync(0xffffffffu, !flat);
  const unsigned seg = LPT == 32 ? 0xffffffffu : ((1u << LPT) - 1u) << (threadIdx.x % 32 / LPT * LPT);
  flat = (who & seg) == 0;
  who = __ballot_sync(0xffffffffu, doubt && !flat);
  if (who == 0) return;
  constexpr int MOST_K = LPT * VPL < FMB_ROUTE_MAX_K ? LPT * VPL : FMB_ROUTE_MAX_K, PER = (MOST_K + LPT - 1) / LPT;
  int keep[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) keep[n] = n * LPT + lane < p.k ? pick[n * LPT + lane] : 0;
  __syncwarp();
  choose_exactly<T, LPT, VPL>(p, row, lane, c64, g64, pick);
  if ((who & seg) == 0) {                                  // the other tokens keep theirs
#pragma unroll
    for (int n = 0; n < PER; ++n)
      if (n * LPT + lane < p.k) pick[n * LPT + lane] = keep[n];
  }
  __syncwarp();
}

// What is the same for all tokens of a thread
template <int LPT, int VPL> struct RouteLane {
  int lane, e0;
  bool biased, grouped, by_score;                          // by_score: else the order of the logits is the scores'
  bool whole_lanes, has_group, two_best;                   // whole_lanes: groups are a power of two of whole lanes
  int span;
  unsigned own_group;
  __device__ __forceinline__ explicit RouteLane(const RouteParams& p) {
    lane = threadIdx.x % LPT;
    e0 = lane * VPL;
    biased = p.bias != nullptr;
    grouped = p.groups > 1;
    by_score = biased || (grouped && p.best > 1);
    span = p.gsize / VPL;
    whole_lanes = p.gsize % VPL == 0 && (span & (span - 1)) == 0 && span <= LPT;
    own_group = grouped && whole_lanes ? lane / span : 0;
    has_group = own_group < static_cast<unsigned>(p.groups);
    two_best = p.best > 1 && p.gsize > 1;
  }
};

// Shared memory of a token: for the choice in 64 bits scores [E] and groups' [groups], keys [k + 2] and choices [k]; and
// the block's counts [E]
struct RouteRoom {
  double *c64, *g64;
  unsigned* key;
  int *pick, *count;
};

// The fixed point of biased scores: what 0 is, steps per score, and how near two scores may be without being told apart
struct RouteScale {
  float lo, unit, error;                                   // error: twice that of a score of 1, in steps
  unsigned near;                                           // how near sigmoid scores may be without being told apart
  bool bad_bias, flat_bias;                                // NaN or +inf: every choice is made in 64 bits; one finite bias for all
};

// Chooses for the LPT lanes' token and writes its weights, choice and counts. Not EXACT: returns false, and writes nothing
// for any token of the warp, if one of them is left open by 32 bits or by the lists of its lanes. `loaded` is called once
// the logits are used up. acc, acc_z: sums for the auxiliary loss.
template <typename T, int LPT, int VPL, bool EXACT, bool AUX, typename F>
__device__ __forceinline__ bool decide(const RouteParams& p, const RouteLane<LPT, VPL>& me, const RouteScale& scale, const RouteRoom& room,
                                       int token, bool live, const T* row, const float (&z)[VPL], const float (&bias)[VPL],
                                       float* acc, float& acc_z, F&& loaded) {
  constexpr int MOST_K = LPT * VPL < FMB_ROUTE_MAX_K ? LPT * VPL : FMB_ROUTE_MAX_K, PER = (MOST_K + LPT - 1) / LPT;
  constexpr int L = EXACT || VPL < LIST ? VPL : LIST;
  const int lane = me.lane, e0 = me.e0;
  float top = z[0], mass = 1.f;
#pragma unroll
  for (int i = 1; i < VPL; ++i) top = max_or_nan(top, z[i]);
  bool doubt = scale.bad_bias || !(top < CUDART_INF_F);     // NaN or +inf, or an order that fp32 leaves open
  if (p.softmax || AUX || !me.biased) top = lanes_max<LPT>(top);
  const float high = top;                                   // (of this lane alone where nothing needs the row's)
  if (p.softmax || AUX) {
    if (top == -CUDART_INF_F) top = 0.f;                    // a row of nothing but -inf: scores of 0
    mass = 0.f;
    float share[AUX ? VPL : 1], norm = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float e = e0 + i < p.E ? expf(z[i] - top) : 0.f;
      mass += e;
      if constexpr (AUX) {
        share[i] = p.softmax ? e : e0 + i < p.E ? sigmoid(z[i]) : 0.f;
        norm += share[i];
      }
    }
    mass = lanes_sum<LPT>(mass);
    if (mass == 0.f) mass = 1.f;
    if constexpr (AUX) {
      norm = lanes_sum<LPT>(norm);
      const float by = norm == 0.f ? 1.f : 1.f / norm;
      if (live) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) acc[i] += share[i] * by;
      }
    }
  }
  if constexpr (AUX) {
    if (live) {
      const float lse = top + logf(mass);
      if (lane == 0) acc_z += lse * lse;
    }
  }
  float inv_mass = 1.f;
  unsigned near = scale.near;
  if (p.softmax) {                                          // no score is above the largest one's, 1 / mass, and errors are in proportion
    inv_mass = __fdividef(1.f, mass);
    near = static_cast<unsigned>(fminf(fmaf(scale.error, inv_mass, 4.f), 1e6f));
  }
  // fixed-point scores and keys; first, second: the lane's two largest for its group where the lists do not hold them
  unsigned key[VPL], list[L], first = 0, second = 0;
  const bool lists_serve = me.biased || !me.by_score;
  unsigned* s_n = reinterpret_cast<unsigned*>(room.c64);    // groups that are no whole lanes: the token's fixed-point scores
  auto see = [&](unsigned v, int e) {
    if (e < p.E) {
      if (!lists_serve) {
        second = max(second, min(first, v));
        first = max(first, v);
      }
      if (!me.whole_lanes) s_n[e] = key_score(v);
    }
  };
  if (me.grouped && !me.whole_lanes) __syncwarp();          // the scores of the token before have been read
  if (me.by_score) {
    keys_by_score<VPL>(p.softmax, z, bias, top, inv_mass, scale.unit, e0, key);
    if (me.grouped && !(lists_serve && me.whole_lanes)) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) see(key[i], e0 + i);
    }
  }
  if (!me.biased) {
    keys_by_logit<T, VPL>(z, high, e0, key);
    if (me.grouped && !me.by_score && !me.whole_lanes) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) see(key[i], e0 + i);
    }
  }
  loaded();
  if (e0 + VPL > p.E) {                                     // the last expert's key is above 0: its number is
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (e0 + i >= p.E) key[i] = 0;
  }
  auto make_list = [&]() {
    if constexpr (L == VPL) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) list[i] = key[i];
      sort_falling(list);
    } else {
      top_falling(key, list);
    }
  };
  const unsigned by_logit = sizeof(T) == 2 ? 0u : 4u;       // bf16 logits' keys are exact
  if (me.grouped) {
    unsigned low = 0, out = 0;                              // the lowest group kept and the highest left out
    if (me.whole_lanes) {
      make_list();
      unsigned a = lists_serve ? list[0] : first, b = lists_serve ? (L > 1 ? list[L > 1 ? 1 : 0] : 0u) : second;
      for (int o = 1; o < me.span; o *= 2) {                // the lane's two largest, then the group's
        const unsigned oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
        b = max(max(b, ob), min(a, oa));
        a = max(a, oa);
      }
      // the group's score above 31 - its number, the same in all its lanes
      unsigned mine = me.has_group ? (key_score(a) + (me.two_best ? key_score(b) : 0u)) << 5 | (31 - me.own_group) : 0u;
      const unsigned whole = mine;
#pragma unroll 1
      for (int n = 0; n < p.top_groups; ++n) {
        low = lanes_umax<LPT>(mine);
        mine = mine == low ? 0 : mine;
      }
      out = lanes_umax<LPT>(mine);
      if (whole < low || !me.has_group) {                   // a group that is left out
#pragma unroll
        for (int i = 0; i < L; ++i) list[i] = 0;
      }
    } else {
      __syncwarp();
      unsigned* s_g = reinterpret_cast<unsigned*>(room.g64);
      int per = 1;                                          // lanes for a group
      while (2 * per * p.groups <= LPT) per *= 2;
      for (int n0 = 0; n0 < p.groups; n0 += LPT / per) {
        const int n = n0 + lane / per;
        unsigned a = 0, b = 0;
        if (n < p.groups)
          for (int e = n * p.gsize + lane % per; e < (n + 1) * p.gsize; e += per) {
            const unsigned v = s_n[e];
            b = max(b, min(a, v));
            a = max(a, v);
          }
        for (int o = 1; o < per; o *= 2) {
          const unsigned oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
          b = max(max(b, ob), min(a, oa));
          a = max(a, oa);
        }
        if (n < p.groups && lane % per == 0) s_g[n] = (a + (me.two_best ? b : 0u)) << 5 | (31 - n);
      }
      __syncwarp();
      unsigned kept = 0;
      for (int n = lane; n < p.groups; n += LPT) {
        int ahead = 0;
        for (int m = 0; m < p.groups; ++m) ahead += s_g[m] > s_g[n];
        if (ahead < p.top_groups) kept |= 1u << n;
        if (ahead == p.top_groups - 1) low = s_g[n];
        if (ahead >= p.top_groups) out = max(out, s_g[n]);
      }
#pragma unroll
      for (int o = LPT / 2; o > 0; o >>= 1) kept |= __shfl_xor_sync(0xffffffffu, kept, o);
      low = lanes_umax<LPT>(low);
      out = lanes_umax<LPT>(out);
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (e0 + i < p.E && !(kept >> ((e0 + i) / p.gsize) & 1)) key[i] = 0;
      __syncwarp();
      make_list();
    }
    const unsigned apart = me.by_score ? 2 * near : by_logit;
    doubt |= p.top_groups < p.groups && (low >> 5) - (out >> 5) < apart;
  } else {
    make_list();
  }
  const bool longer = L < VPL && list[L - 1] != 0;          // there may be more behind the list
  // k rounds of the largest first key, each kept by a lane of its own, and one more to see how far behind the next one is
  unsigned mine[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    mine[n] = 0;
#pragma unroll 4
    for (int j = n * LPT; j < (n + 1) * LPT && j < p.k; ++j) {
      const unsigned w = take_largest<LPT>(list);
      if (lane == j - n * LPT) mine[n] = w;
    }
  }
  const unsigned next = take_largest<LPT>(list);
  bool open = longer && list[0] == 0;                       // this lane has given away its whole list
  const unsigned apart = me.biased ? near : by_logit;
  int pick[PER];
  unsigned after[PER];
  bool hit = false;                                         // neighbours of the order that are too near to tell
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int j = n * LPT + lane;
    after[n] = __shfl_down_sync(0xffffffffu, mine[n], 1, LPT);
    if (n + 1 < PER) {
      const unsigned turn = __shfl_sync(0xffffffffu, mine[n + 1 < PER ? n + 1 : n], 0, LPT);
      if (lane == LPT - 1) after[n] = turn;
    }
    if (j == p.k - 1) after[n] = next;
    pick[n] = min(key_expert(mine[n]), p.E - 1);            // (a token in doubt may have fewer keys than choices)
    if (j < p.k) {
      open |= mine[n] == 0;
      hit |= after[n] != 0 && key_score(mine[n]) - key_score(after[n]) < apart;
    }
  }
  open |= doubt;
  if (__any_sync(0xffffffffu, hit || open)) {               // one token of this warp, or more: all its lanes go
    const unsigned then = take_largest<LPT>(list);
    if constexpr (EXACT) {
#pragma unroll
      for (int n = 0; n < PER; ++n)
        if (n * LPT + lane < p.k) room.key[n * LPT + lane] = mine[n];
      if (lane == 0) {
        room.key[p.k] = next;
        room.key[p.k + 1] = then;
      }
      __syncwarp();
      settle<T, LPT, VPL>(p, row, lane, apart, doubt, !me.biased || scale.flat_bias, top, mass, room.key, room.pick, room.c64, room.g64);
#pragma unroll
      for (int n = 0; n < PER; ++n)
        if (n * LPT + lane < p.k) pick[n] = room.pick[n * LPT + lane];
      __syncwarp();
    } else {
      // neighbours that are equal by their inputs are in order; at the last choice the next one might belong before both
      if (hit) {
#pragma unroll
        for (int n = 0; n < PER; ++n) {
          const int j = n * LPT + lane;
          if (j < p.k && after[n] != 0 && key_score(mine[n]) - key_score(after[n]) < apart) {
            const int b = key_expert(after[n]);
            open |= to_f32(row[pick[n]]) != to_f32(row[b]) || (me.biased && p.bias[pick[n]] != p.bias[b]);
            open |= j == p.k - 1 && then != 0 && key_score(next) - key_score(then) < apart;
          }
        }
      }
      if (__any_sync(0xffffffffu, open)) return false;
    }
  }
  // weights of the chosen, each by a lane of its own
  float sum = 0.f, best = -CUDART_INF_F, chosen[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int j = n * LPT + lane;
    chosen[n] = j < p.k ? to_f32(row[pick[n]]) : -CUDART_INF_F;
    best = fmaxf(best, chosen[n]);
  }
  if (p.softmax) best = lanes_max<LPT>(best);
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
  if (!p.softmax && p.renorm && __any_sync(0xffffffffu, sum < 1e-30f)) {
    // sigmoids that vanish in fp32 still have shares: s = e^z there
    const float peak = lanes_max<LPT>(best), around = peak == -CUDART_INF_F ? 0.f : peak;
    float far = 0.f, share[PER];
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      share[n] = n * LPT + lane < p.k ? expf(to_f32(row[pick[n]]) - around) : 0.f;
      far += share[n];
    }
    far = lanes_sum<LPT>(far);
    if (sum < 1e-30f) {
#pragma unroll
      for (int n = 0; n < PER; ++n) chosen[n] = share[n];
      sum = far;
    }
  }
  const float by = !p.renorm ? p.scale : sum == 0.f ? 0.f : p.scale / sum;      // nothing to share out: weights of 0
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int j = n * LPT + lane;
    if (j < p.k && live) {
      const int e = pick[n];
      p.weights[static_cast<long long>(token) * p.k + j] = chosen[n] * by;
      p.idx[static_cast<long long>(token) * p.k + j] = e;
      atomicAdd(room.count + e, 1);
    }
  }
  __syncwarp();
  return true;
}

template <typename T> __device__ __forceinline__ const T* route_row(const RouteParams& p, int token) {
  return static_cast<const T*>(p.logits) + static_cast<long long>(token) * p.ld;
}
template <int VPL>
__device__ __forceinline__ void load_bias(const RouteParams& p, int e0, const RouteScale& scale, float (&bias)[VPL]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) bias[i] = fixed_bias(p.bias != nullptr && e0 + i < p.E ? p.bias[e0 + i] : 0.f, scale.lo, scale.unit);
}

// A warp's tokens once more, with whole lists and what 64 bits take. Everything is loaded here again and the code stands
// inline, in a loop of its own: as a call from the middle of the loop over the tokens it made that loop spill (67 us where
// this takes 58, 65536 tokens of 256 experts).
template <typename T, int LPT, int VPL>
__device__ __forceinline__ void decide_again(const RouteParams& p, RouteScale scale, RouteRoom room, int token, bool live) {
  const RouteLane<LPT, VPL> me(p);
  const T* row = route_row<T>(p, token);
  float z[VPL], bias[VPL], none = 0.f;
  load_own<T, VPL>(row, me.e0, p.E, p.vec, z);
  load_bias<VPL>(p, me.e0, scale, bias);
  decide<T, LPT, VPL, true, false>(p, me, scale, room, token, live, row, z, bias, nullptr, none, [] {});
}

template <typename T, int LPT, int VPL, bool AUX>
__global__ void __launch_bounds__(ROUTE_THREADS, VPL > 8 ? 3 : 6) route_fwd_kernel(const __grid_constant__ RouteParams p) {
  constexpr int TPB = ROUTE_THREADS / LPT;                 // tokens that a block has in hand
  constexpr int MOST_K = LPT * VPL < FMB_ROUTE_MAX_K ? LPT * VPL : FMB_ROUTE_MAX_K;
  extern __shared__ double s_mem[];                        // for the choice in 64 bits: scores [TPB, E], groups [TPB, groups]
  __shared__ unsigned s_key[TPB][MOST_K + 2];
  __shared__ int s_pick[TPB][MOST_K];
  __shared__ float s_range[2][ROUTE_THREADS / 32];
  const int slot = threadIdx.x / LPT;
  int* s_count = reinterpret_cast<int*>(s_mem + static_cast<size_t>(TPB) * (p.E + p.groups));   // [E]
  float* s_acc = reinterpret_cast<float*>(s_count + p.E);                                       // [E + 1]
  const RouteRoom room = {s_mem + static_cast<size_t>(slot) * p.E, s_mem + static_cast<size_t>(TPB) * p.E + slot * p.groups,
                          s_key[slot], s_pick[slot], s_count};
  pdl_wait();
  pdl_launch_dependents();
  const RouteLane<LPT, VPL> me(p);
  const int e0 = me.e0;
  for (int e = threadIdx.x; e < p.E; e += ROUTE_THREADS) s_count[e] = 0;
  if (AUX)
    for (int e = threadIdx.x; e <= p.E; e += ROUTE_THREADS) s_acc[e] = 0.f;
  // the range of scores in fixed point: [0, 1] and what the finite biases add
  RouteScale scale = {0.f, 1.f, 0.f, 0, false, false};
  float range = 1.f, bias[VPL];
  if (me.biased) {
    float a = CUDART_INF_F, b = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      bias[i] = e0 + i < p.E ? p.bias[e0 + i] : 0.f;
      scale.bad_bias |= !(bias[i] < CUDART_INF_F);
      if (e0 + i < p.E && fabsf(bias[i]) < CUDART_INF_F) { a = fminf(a, bias[i]); b = fmaxf(b, bias[i]); }
    }
    a = -lanes_max<32>(-a);
    b = lanes_max<32>(b);
    if (threadIdx.x % 32 == 0) { s_range[0][threadIdx.x / 32] = a; s_range[1][threadIdx.x / 32] = b; }
    __syncthreads();
    for (int w = 0; w < ROUTE_THREADS / 32; ++w) { a = fminf(a, s_range[0][w]); b = fmaxf(b, s_range[1][w]); }
    if (a <= b) { scale.lo = a; range = (b - a) + 1.f; }      // ((1 + b) - a would lose a unit of b's, which may be anything)
    bool same = a == b;
#pragma unroll
    for (int i = 0; i < VPL; ++i) same &= e0 + i >= p.E || bias[i] == a;
    scale.flat_bias = __all_sync(0xffffffffu, same);
  }
  __syncthreads();
  // Steps per score, so few less that no rounding goes past the last one: the range is off by two units of 2^-24 of itself,
  // the quotient and a bias without the lowest by one each (two steps in all), a score may be 2^-21 above 1 (four), and two
  // additions round to a step (one): seven at the most. And what the bias adds to the fixed point.
  scale.unit = static_cast<float>(FIXED - 16) / range;
  load_bias<VPL>(p, e0, scale, bias);
  // How far a score may be from the exact one. Sigmoid: s (1 - s) <= 1/4 of the error of e^-z (2^-22, and its argument's
  // rounding, 3.3e-7 at |z| = 5.5 and less in s beyond), 1.8e-7 from addition and reciprocal: 3.4e-7. Softmax, divided by a
  // sum of up to 512 terms some 30 roundings deep: 3e-6 of the score. Then a step of the fixed point. Two of those, and one
  // more, where a token's scores are taken: closer than that is too near.
  scale.error = (p.softmax ? 6e-6f : 6.8e-7f) * scale.unit;
  scale.near = static_cast<unsigned>(fminf(scale.error + 4.f, 1e6f));
  float acc[AUX ? VPL : 1], acc_z = 0.f;
#pragma unroll
  for (int i = 0; i < (AUX ? VPL : 1); ++i) acc[i] = 0.f;

  const int last = static_cast<int>(p.tokens) - 1;          // (fewer than 2^31 tokens)
  const int stride = gridDim.x * TPB;
  float z[VPL];                                             // lanes without a token go along with the last one
  load_own<T, VPL>(route_row<T>(p, min(static_cast<int>(blockIdx.x) * TPB + slot, last)), e0, p.E, p.vec, z);
  for (int base = blockIdx.x * TPB; base <= last;) {
    // 32 steps, of which those with an undecided token are taken again afterwards
    const int begin = base;
    unsigned again = 0;
    for (unsigned bit = 1; bit != 0 && base <= last; bit <<= 1, base += stride) {
      const int token = min(base + slot, last);
      const bool done = decide<T, LPT, VPL, false, AUX>(p, me, scale, room, token, base + slot <= last, route_row<T>(p, token), z, bias, acc,
                                                        acc_z, [&] {
        if (base + stride <= last) load_own<T, VPL>(route_row<T>(p, min(base + stride + slot, last)), e0, p.E, p.vec, z);
      });
      if (!done) again |= bit;
    }
    if (again != 0) {
      for (; again != 0; again &= again - 1) {
        const int at = begin + (__ffs(again) - 1) * stride + slot;
        decide_again<T, LPT, VPL>(p, scale, room, min(at, last), at <= last);
      }
      if (base <= last) load_own<T, VPL>(route_row<T>(p, min(base + slot, last)), e0, p.E, p.vec, z);
      load_bias<VPL>(p, e0, scale, bias);
    }
  }
  if constexpr (AUX) {
    for (int who = 0; who < TPB; ++who) {                   // tokens' sums one slot after another: a fixed order
      __syncthreads();
      if (slot == who) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (e0 + i < p.E) s_acc[e0 + i] += acc[i];
        if (me.lane == 0) s_acc[p.E] += acc_z;
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
      if (p.renorm) w[n] = p.scale == 0.f ? 0.f : w[n] / p.scale;      // the share: of a single choice exactly 1
      dot += w[n] * dw[n];
    }
  }
  dot = lanes_sum<LPT>(dot);
  float dz[PER];                                            // the part of the weights, on the chosen experts
  float flow = 0.f;                                         // not renormalised softmax: sum of w dw, which all experts share
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    // d w_j / d s_i = scale (delta_ij - s_j / S) / S and d s / d z = s (s (1 - s)): both leave a factor w_j
    dz[n] = p.renorm ? p.scale * w[n] * (dw[n] - dot) : w[n] * dw[n];
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
int route_fwd_run(RouteParams p, int blocks, cudaStream_t stream) {
  constexpr int TPB = ROUTE_THREADS / LPT, BYTES = VPL * sizeof(T) < 16 ? VPL * sizeof(T) : 16;
  // values of 64 bits of the block's 16, 8 or 4 tokens, counts and sums: with the kernel's static arrays (keys and choices of
  // each token, ranges) no opt-in is needed
  constexpr int MOST_E = LPT * VPL, MOST_K = MOST_E < FMB_ROUTE_MAX_K ? MOST_E : FMB_ROUTE_MAX_K;
  static_assert(sizeof(double) * TPB * (MOST_E + FMB_ROUTE_MAX_GROUPS) + sizeof(int) * (2 * MOST_E + 1) +
                sizeof(int) * TPB * (2 * MOST_K + 2) + sizeof(float) * ROUTE_THREADS / 16 <= 48 * 1024, "beyond 48 KB a kernel has to opt in");
  const size_t smem = sizeof(double) * TPB * (p.E + p.groups) + sizeof(int) * (2 * p.E + 1);
  p.vec = p.E % VPL == 0 && p.ld % VPL == 0 && reinterpret_cast<uintptr_t>(p.logits) % BYTES == 0;
  auto kernel = p.partial != nullptr ? route_fwd_kernel<T, LPT, VPL, true> : route_fwd_kernel<T, LPT, VPL, false>;
  return launch_pdl(kernel, dim3(blocks), dim3(ROUTE_THREADS), smem, stream, p) == cudaSuccess ? 0 : -3;
}

template <typename T, int LPT, int VPL> int route_bwd_run(const RouteGrad& p, bool dense, cudaStream_t stream) {
  constexpr int TPB = ROUTE_THREADS / LPT;
  const dim3 grid(static_cast<unsigned>((p.tokens + TPB - 1) / TPB));
  const cudaError_t e = dense ? launch_pdl(route_bwd_kernel<T, LPT, VPL, true>, grid, dim3(ROUTE_THREADS), 0, stream, p)
                              : launch_pdl(route_bwd_kernel<T, LPT, VPL, false>, grid, dim3(ROUTE_THREADS), 0, stream, p);
  return e == cudaSuccess ? 0 : -3;
}

// Lanes per token in the forward pass: 8 where 8 experts for each hold them all (a warp then serves four tokens), up to a
// warp beyond (its maximum over the lanes is one instruction).
inline int route_lanes(int E) { return E <= 64 ? 8 : E <= 128 ? 16 : 32; }

}  // namespace fmb

using namespace fmb;

extern "C" int fmb_route_blocks(long long tokens, int E) {
  const int per = ROUTE_THREADS / route_lanes(E);
  const long long need = (tokens + per - 1) / per, most = (E <= 256 ? 6LL : 3LL) * sm_count();      // as many as are resident
  return static_cast<int>(need < 1 ? 1 : need < most ? need : most);
}

#define FMB_ROUTE_FWD(T, ...)                                        \
  do {                                                               \
    if (E <= 8) return route_fwd_run<T, 8, 1>(__VA_ARGS__);          \
    if (E <= 16) return route_fwd_run<T, 8, 2>(__VA_ARGS__);         \
    if (E <= 32) return route_fwd_run<T, 8, 4>(__VA_ARGS__);         \
    if (E <= 64) return route_fwd_run<T, 8, 8>(__VA_ARGS__);         \
    if (E <= 128) return route_fwd_run<T, 16, 8>(__VA_ARGS__);       \
    if (E <= 256) return route_fwd_run<T, 32, 8>(__VA_ARGS__);       \
    return route_fwd_run<T, 32, 16>(__VA_ARGS__);                    \
  } while (0)
#define FMB_ROUTE_BWD(T, ...)                                        \
  do {                                                               \
    if (E <= 8) return route_bwd_run<T, 1, 8>(__VA_ARGS__);          \
    if (E <= 16) return route_bwd_run<T, 2, 8>(__VA_ARGS__);         \
    if (E <= 32) return route_bwd_run<T, 4, 8>(__VA_ARGS__);         \
    if (E <= 64) return route_bwd_run<T, 8, 8>(__VA_ARGS__);         \
    if (E <= 128) return route_bwd_run<T, 8, 16>(__VA_ARGS__);       \
    if (E <= 256) return route_bwd_run<T, 8, 32>(__VA_ARGS__);       \
    return route_bwd_run<T, 16, 32>(__VA_ARGS__);                    \
  } while (0)

extern "C" int fmb_route_fwd(const void* logits, long long ld, int dtype, const float* bias, float* weights, int* idx,
                             int* counts, float* partial, float* aux, long long tokens, int E, int k, int softmax, int groups,
                             int top_groups, int best, int renorm, float scale, float aux_coef, float z_coef, int blocks,
                             cudaStream_t stream) {
  if (E < 1 || E > FMB_ROUTE_MAX_EXPERTS || k < 1 || k > FMB_ROUTE_MAX_K || k > E || groups < 1 || groups > FMB_ROUTE_MAX_GROUPS || E % groups ||
      top_groups < 1 || top_groups > groups || k > E / groups * top_groups || best < 1 || best > 2 || blocks < 1)
    return -2;
  if (cudaMemsetAsync(counts, 0, E * sizeof(int), stream) != cudaSuccess) return -3;
  if (tokens <= 0) return 0;
  if (tokens > 0x7fff0000LL) return -2;                    // steps over the tokens stay within 31 bits
  RouteParams p = {};
  p.logits = logits; p.ld = ld; p.tokens = tokens; p.bias = bias; p.weights = weights; p.idx = idx; p.counts = counts;
  p.partial = partial; p.E = E; p.k = k; p.softmax = softmax; p.groups = groups; p.gsize = E / groups; p.top_groups = top_groups;
  p.best = best; p.renorm = renorm; p.scale = scale;
  int rc = -1;
  if (dtype == FMB_BF16) rc = [&]() -> int { FMB_ROUTE_FWD(__nv_bfloat16, p, blocks, stream); }();
  else if (dtype == FMB_F32) rc = [&]() -> int { FMB_ROUTE_FWD(float, p, blocks, stream); }();
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
  if (dtype == FMB_BF16) FMB_ROUTE_BWD(__nv_bfloat16, p, dense, stream);
  if (dtype == FMB_F32) FMB_ROUTE_BWD(float, p, dense, stream);
  return -1;
}

// Rotary positions for queries and keys in one launch.
//
//   u = a cos - b sin,  v = a sin + b cos        for each of R/2 pairs (a, b) of a head's first R values,
//   pairs (i, i + R/2), or (2i, 2i + 1) when interleaved; the other D - R values are copied. The backward pass is
//   the same rotation with -sin.
//
// Bound by HBM bandwidth: three operations per value. The angle depends on the token alone, so a thread takes one
// vector of pairs and walks over heads with cos and sin in registers; the tables (fp32) are read once per token.
#include "fmb_api.h"
#include "launch.cuh"
#include "rows.cuh"

namespace fmb {

struct RotaryTensor {
  const void* src;
  void* dst;                       // contiguous [B, T, H, D]
  long long sb, st, sh;            // strides of src in elements; the head dimension is contiguous
  int heads;
};

struct RotaryParams {
  RotaryTensor q, k;
  const float *cos, *sin;          // [table, R / 2], rows `ldt` apart
  const void* positions;           // null: the token's place in its sequence
  long long pos_b;                 // elements between the positions of two sequences (0: shared)
  long long ldt, table;
  unsigned tokens, token0;         // all tokens, and the first one of this launch
  int T, D, R, wide_pos, units, rot_units, groups, per_group;
  float sign;
};

constexpr int BATCH = 4;

// One item: unit `u` of a token (VEC pairs, or two vectors of VEC copied values) in `per_group` heads.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const unsigned per_token = static_cast<unsigned>(p.units) * p.groups;
  const unsigned item = blockIdx.x * 256u + threadIdx.x;             // fewer than 2^31 items per launch
  const unsigned local = item / per_token;
  const unsigned token = p.token0 + local;
  if (token >= p.tokens) return;
  const unsigned rest = item - local * per_token;
  const int group = rest / p.units, unit = rest - group * p.units;
  const int b = token / p.T, t = token - b * p.T;
  const bool turn = unit < p.rot_units;
  float c[VEC], s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) { c[j] = 1.f; s[j] = 0.f; }
  if (turn) {
    long long pos = t;
    if (p.positions != nullptr) {
      const long long at = b * p.pos_b + t;
      pos = p.wide_pos ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
    }
    if (pos >= p.table) {                                            // beyond the table there is no angle: say so loudly
#pragma unroll
      for (int j = 0; j < VEC; ++j) { c[j] = CUDART_NAN_F; s[j] = CUDART_NAN_F; }
    } else if (pos >= 0) {                                           // a negative position marks padding: left unturned
      const float *cr = p.cos + pos * p.ldt + unit * VEC, *sr = p.sin + pos * p.ldt + unit * VEC;
      if constexpr (VEC % 4 == 0) {
        load_f32<float, VEC>(cr, c);
        load_f32<float, VEC>(sr, s);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { c[j] = cr[j]; s[j] = sr[j]; }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] *= p.sign;
    }
  }
  // where the two vectors of pairs, or the two that are copied (the second may not be there), lie in a head
  const int first = turn ? (INTER ? 2 * VEC * unit : VEC * unit) : p.R + 2 * VEC * (unit - p.rot_units);
  const int second = INTER || !turn ? first + VEC : first + p.R / 2;
  const bool two = turn || second < p.D;
  const int h_end = min((group + 1) * p.per_group, p.q.heads + p.k.heads);
  auto place = [&](int h, const T*& src, T*& dst) {
    const bool is_k = h >= p.q.heads;
    const RotaryTensor& x = is_k ? p.k : p.q;
    const int hh = is_k ? h - p.q.heads : h;
    src = static_cast<const T*>(x.src) + b * x.sb + t * x.st + hh * x.sh;
    dst = static_cast<T*>(x.dst) + (static_cast<long long>(token) * x.heads + hh) * p.D;
  };
  if constexpr (VEC == Vec16<T>::N) {
    // BATCH heads are loaded before the first of them is stored: a thread has 128 bytes on their way
    for (int h = group * p.per_group; h < h_end; h += BATCH) {
      uint4 ra[BATCH], rb[BATCH];
      T* dst[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (h + i < h_end) {
          const T* src;
          place(h + i, src, dst[i]);
          ra[i] = *reinterpret_cast<const uint4*>(src + first);
          if (two) rb[i] = *reinterpret_cast<const uint4*>(src + second);
        }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (h + i >= h_end) break;
        if (turn) {
          float x0[VEC], x1[VEC], y0[VEC], y1[VEC];
          Vec16<T>::unpack(ra[i], x0);
          Vec16<T>::unpack(rb[i], x1);
          if constexpr (INTER) {
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              y0[2 * j] = x0[2 * j] * c[j] - x0[2 * j + 1] * s[j];
              y0[2 * j + 1] = x0[2 * j] * s[j] + x0[2 * j + 1] * c[j];
              y1[2 * j] = x1[2 * j] * c[VEC / 2 + j] - x1[2 * j + 1] * s[VEC / 2 + j];
              y1[2 * j + 1] = x1[2 * j] * s[VEC / 2 + j] + x1[2 * j + 1] * c[VEC / 2 + j];
            }
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              y0[j] = x0[j] * c[j] - x1[j] * s[j];
              y1[j] = x0[j] * s[j] + x1[j] * c[j];
            }
          }
          ra[i] = Vec16<T>::pack(y0);
          rb[i] = Vec16<T>::pack(y1);
        }
        *reinterpret_cast<uint4*>(dst[i] + first) = ra[i];
        if (two) *reinterpret_cast<uint4*>(dst[i] + second) = rb[i];
      }
    }
  } else {
    static_assert(VEC == 1, "single values otherwise");
#pragma unroll 2
    for (int h = group * p.per_group; h < h_end; ++h) {
      const T* src;
      T* dst;
      place(h, src, dst);
      const T va = src[first], vb = two ? src[second] : va;
      if (turn) {
        const float a = to_f32(va), e = to_f32(vb);
        dst[first] = from_f32<T>(a * c[0] - e * s[0]);
        dst[second] = from_f32<T>(a * s[0] + e * c[0]);
      } else {
        dst[first] = va;
        if (two) dst[second] = vb;
      }
    }
  }
}

template <typename T, bool INTER>
cudaError_t rotary_launch(RotaryParams p, bool vec, cudaStream_t stream) {
  const int n = vec ? Vec16<T>::N : 1, heads = p.q.heads + p.k.heads;
  p.rot_units = p.R / 2 / n;
  p.units = p.rot_units + ((p.D - p.R) / n + 1) / 2;
  // Few tokens: a thread per head, for latency. Many: up to eight heads per thread, for the tables' sake.
  const long long lanes = static_cast<long long>(p.tokens) * p.units;
  const long long room = static_cast<long long>(sm_count()) * 2048;
  int per = 1;
  while (per < 8 && per < heads && lanes * heads / (2 * per) >= room) per *= 2;
  p.per_group = per;
  p.groups = (heads + per - 1) / per;
  const long long per_token = static_cast<long long>(p.units) * p.groups;
  const long long most = 0x7fffff00LL / per_token;                   // tokens whose items 31 bits can number
  cudaError_t e = most > 0 ? cudaSuccess : cudaErrorInvalidValue;
  for (long long lo = 0; e == cudaSuccess && lo < p.tokens; lo += most) {
    p.token0 = static_cast<unsigned>(lo);
    const long long items = (p.tokens - lo < most ? p.tokens - lo : most) * per_token;
    const unsigned blocks = static_cast<unsigned>((items + 255) / 256);
    e = vec ? launch_pdl(rotary_kernel<T, Vec16<T>::N, INTER>, dim3(blocks), dim3(256), 0, stream, p)
            : launch_pdl(rotary_kernel<T, 1, INTER>, dim3(blocks), dim3(256), 0, stream, p);
  }
  return e;
}

}  // namespace fmb

using namespace fmb;

extern "C" int fmb_rotary(const FmbRotaryTensor* q, const FmbRotaryTensor* k, const float* cos, const float* sin,
                          long long ldt, long long table, const void* positions, int wide_positions, long long pos_b,
                          long long batch, int T, int D, int R, int interleaved, float sign, int dtype, cudaStream_t stream) {
  if (q == nullptr || k == nullptr || D <= 0 || R < 0 || R > D || R % 2 || q->heads < 0 || k->heads < 0) return -2;
  const int heads = q->heads + k->heads;
  const long long tokens = batch * T;
  if (tokens <= 0 || heads == 0) return 0;
  if (tokens > 0x7fffffffLL) return -2;
  RotaryParams p = {};
  p.q = {q->src, q->dst, q->sb, q->st, q->sh, q->heads};
  p.k = {k->src, k->dst, k->sb, k->st, k->sh, k->heads};
  p.cos = cos; p.sin = sin; p.ldt = ldt; p.table = table;
  p.positions = positions; p.wide_pos = wide_positions; p.pos_b = pos_b;
  p.tokens = static_cast<unsigned>(tokens); p.T = T; p.D = D; p.R = R; p.sign = sign;
  const int n = dtype == FMB_BF16 ? 8 : 4;
  auto fits = [&](const FmbRotaryTensor* x) {
    return x->heads == 0 || (aligned16(x->src) && aligned16(x->dst) && x->sb % n == 0 && x->st % n == 0 && x->sh % n == 0);
  };
  const bool vec = D % n == 0 && R % (2 * n) == 0 && fits(q) && fits(k) && aligned16(cos) && aligned16(sin) && ldt % 4 == 0;
  cudaError_t e;
  if (dtype == FMB_BF16)
    e = interleaved ? rotary_launch<__nv_bfloat16, true>(p, vec, stream) : rotary_launch<__nv_bfloat16, false>(p, vec, stream);
  else if (dtype == FMB_F32)
    e = interleaved ? rotary_launch<float, true>(p, vec, stream) : rotary_launch<float, false>(p, vec, stream);
  else
    return -1;
  return e == cudaSuccess ? 0 : -3;
}

// Rotary positions for queries and keys in one launch.
//
//   u = a cos - b sin,  v = a sin + b cos        for each of R/2 pairs (a, b) of a head's first R values,
//   pairs (i, i + R/2), or (2i, 2i + 1) when interleaved; the other D - R values are copied. The backward pass is
//   the same rotation with -sin.
//
// Bound by HBM bandwidth: three operations per value. The angle depends on the token alone, so a thread takes one
// vector of pairs and walks over heads with cos and sin in registers; the tables (fp32) are read once per token.
// 65536 tokens, 32 + 8 heads of 128, half of them turned, bf16: 205 us, 6.6 TB/s.
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

// The token, unit and heads of this thread's item; false where there is none.
struct Item {
  unsigned token;
  int b, t, unit, h, h_end;
};
__device__ __forceinline__ bool item_of(const RotaryParams& p, Item& it) {
  const unsigned per_token = static_cast<unsigned>(p.units) * p.groups;
  const unsigned item = blockIdx.x * 256u + threadIdx.x;             // fewer than 2^31 items per launch
  const unsigned local = item / per_token, rest = item - local * per_token;
  it.token = p.token0 + local;
  const int group = rest / p.units;
  it.unit = rest - group * p.units;
  it.b = it.token / p.T;
  it.t = it.token - it.b * p.T;
  it.h = group * p.per_group;
  it.h_end = min(it.h + p.per_group, p.q.heads + p.k.heads);
  return it.token < p.tokens;
}
__device__ __forceinline__ long long position_of(const RotaryParams& p, const Item& it) {
  if (p.positions == nullptr) return it.t;
  const long long at = it.b * p.pos_b + it.t;
  return p.wide_pos ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
}
template <typename T> __device__ __forceinline__ void head_of(const RotaryParams& p, const Item& it, int h, const T*& src, T*& dst) {
  const bool is_k = h >= p.q.heads;
  const RotaryTensor& x = is_k ? p.k : p.q;
  const int hh = is_k ? h - p.q.heads : h;
  src = static_cast<const T*>(x.src) + it.b * x.sb + it.t * x.st + hh * x.sh;
  dst = static_cast<T*>(x.dst) + (static_cast<long long>(it.token) * x.heads + hh) * p.D;
}

// One item: unit `u` of a token (VEC pairs, or two vectors of VEC copied values) in `per_group` heads.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryParams p) {
  pdl_wait();
  pdl_launch_dependents();
  Item it;
  if (!item_of(p, it)) return;
  const int unit = it.unit;
  bool turn = unit < p.rot_units;
  const int first = turn ? (INTER ? 2 * VEC * unit : VEC * unit) : p.R + 2 * VEC * (unit - p.rot_units);
  // where the two vectors of pairs, or the two that are copied (the second may not be there), lie in a head
  const int second = INTER || !turn ? first + VEC : first + p.R / 2;
  const bool two = turn || second < p.D;
  float c[VEC], s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) { c[j] = 1.f; s[j] = 0.f; }
  if (turn) {
    const long long pos = position_of(p, it);
    if (pos >= p.table) {                                            // beyond the table there is no angle: say so loudly
#pragma unroll
      for (int j = 0; j < VEC; ++j) { c[j] = CUDART_NAN_F; s[j] = CUDART_NAN_F; }
    } else if (pos < 0) {                                            // a negative position marks padding: copied
      turn = false;
    } else {
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
  if constexpr (VEC == Vec16<T>::N) {
    // BATCH heads are loaded before the first of them is stored: a thread has 128 bytes on their way
    for (int h = it.h; h < it.h_end; h += BATCH) {
      uint4 ra[BATCH], rb[BATCH];
      T* dst[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (h + i < it.h_end) {
          const T* src;
          head_of<T>(p, it, h + i, src, dst[i]);
          ra[i] = *reinterpret_cast<const uint4*>(src + first);
          if (two) rb[i] = *reinterpret_cast<const uint4*>(src + second);
        }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (h + i >= it.h_end) break;
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
    for (int h = it.h; h < it.h_end; ++h) {
      const T* src;
      T* dst;
      head_of<T>(p, it, h, src, dst);
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

// Heads of whole vectors of which R values are no whole vectors of pairs. One item: one vector of a head, where a value's
// partner is its neighbour (INTER), or lies R / 2 away and is loaded by itself.
template <typename T, bool INTER>
__global__ void __launch_bounds__(256) rotary_mixed_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int N = Vec16<T>::N;
  pdl_wait();
  pdl_launch_dependents();
  Item it;
  if (!item_of(p, it)) return;
  const int first = it.unit * N, half = p.R / 2;
  float c[N], s[N];
  int away[N];                                                       // of the partner
  unsigned turns = 0;                                                // values that are turned
  const long long pos = first < p.R ? position_of(p, it) : -1;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = first + j;
    const bool upper = INTER ? e % 2 : e >= half;
    away[j] = INTER ? (upper ? -1 : 1) : upper ? -half : half;
    c[j] = 1.f;
    s[j] = 0.f;
    if (e < p.R && pos >= 0) {
      turns |= 1u << j;
      const long long at = pos * p.ldt + (INTER ? e / 2 : upper ? e - half : e);
      c[j] = pos < p.table ? p.cos[at] : CUDART_NAN_F;
      s[j] = pos < p.table ? p.sin[at] * (upper ? p.sign : -p.sign) : CUDART_NAN_F;
    }
  }
  // Heads that are loaded before the first of them is stored (four with single partners cost occupancy). 32768 tokens, 32
  // heads of 128: 50 values turned in halves 145 us (four 163), as neighbours 100 (one at a time 139); their bytes 82.
  constexpr int HEADS = INTER ? BATCH : BATCH / 2;
  for (int h = it.h; h < it.h_end; h += HEADS) {
    uint4 u[HEADS];
    T other[HEADS][INTER ? 1 : N], *dst[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      if (h + i < it.h_end) {
        const T* src;
        head_of<T>(p, it, h + i, src, dst[i]);
        u[i] = *reinterpret_cast<const uint4*>(src + first);
        if constexpr (!INTER) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (turns >> j & 1) other[i][j] = src[first + j + away[j]];
        }
      }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      if (h + i >= it.h_end) break;
      if (turns != 0) {
        float x[N], y[N];
        Vec16<T>::unpack(u[i], x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          y[j] = x[j];
          if (turns >> j & 1) y[j] = x[j] * c[j] + (INTER ? x[j ^ 1] : to_f32(other[i][INTER ? 0 : j])) * s[j];
        }
        u[i] = Vec16<T>::pack(y);
      }
      *reinterpret_cast<uint4*>(dst[i] + first) = u[i];
    }
  }
}

enum class Form { VECTORS, MIXED, SINGLE };

template <typename T, bool INTER>
cudaError_t rotary_launch(RotaryParams p, Form form, cudaStream_t stream) {
  const int n = form == Form::SINGLE ? 1 : Vec16<T>::N, heads = p.q.heads + p.k.heads;
  p.rot_units = p.R / 2 / n;
  p.units = form == Form::MIXED ? p.D / n : p.rot_units + ((p.D - p.R) / n + 1) / 2;
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
    e = form == Form::VECTORS ? launch_pdl(rotary_kernel<T, Vec16<T>::N, INTER>, dim3(blocks), dim3(256), 0, stream, p)
        : form == Form::MIXED ? launch_pdl(rotary_mixed_kernel<T, INTER>, dim3(blocks), dim3(256), 0, stream, p)
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
  const bool whole = D % n == 0 && fits(q) && fits(k);
  const Form form = !whole ? Form::SINGLE : R % (2 * n) == 0 && aligned16(cos) && aligned16(sin) && ldt % 4 == 0 ? Form::VECTORS : Form::MIXED;
  cudaError_t e;
  if (dtype == FMB_BF16)
    e = interleaved ? rotary_launch<__nv_bfloat16, true>(p, form, stream) : rotary_launch<__nv_bfloat16, false>(p, form, stream);
  else if (dtype == FMB_F32)
    e = interleaved ? rotary_launch<float, true>(p, form, stream) : rotary_launch<float, false>(p, form, stream);
  else
    return -1;
  return e == cudaSuccess ? 0 : -3;
}

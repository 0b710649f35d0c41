// Distillation from the K largest logits of a teacher: loss and gradient over rows of student logits.
//
//   p_k = softmax over the row's kept teacher logits / tau   (or exp(t_k / tau - lse) when the teacher's normaliser is known)
//   q   = softmax(student / tau)
//   row = sum_k p_k (log p_k - log q[index_k]),   gradient = (q sum_k p_k - p scattered to index) scale / tau
//
// A slot whose index is outside [0, V), or whose teacher logit is -inf, does not count; a row without slots that
// count has no loss and no gradient. An index that stands twice in a row counts twice.
// Bound by HBM bandwidth: one exponential per student logit and pass. Sums and statistics are fp32; exponentials are
// 2^x of the special function unit (relative error 2^-22) with the argument folded into one multiply-add.
#include "fmb_api.h"
#include "launch.cuh"
#include "rows.cuh"

namespace fmb {

constexpr int KL_THREADS = 512;
constexpr float LOG2E = 1.4426950408889634f;

template <typename TT> __device__ __forceinline__ bool slot_counts(long long at, TT value, int V) {
  return at >= 0 && at < V && !(to_f32(value) == -CUDART_INF_F);
}

// Rows that have a slot that counts. One warp per row.
template <typename TT>
__global__ void __launch_bounds__(256)
kl_topk_count_kernel(const TT* __restrict__ values, const long long* __restrict__ index, int* __restrict__ count,
                     long long rows, int V, int K) {
  __shared__ int s_n;
  if (threadIdx.x == 0) s_n = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (long long row = blockIdx.x * 8LL + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8LL) {
    bool any = false;
    for (int k = lane; k < K; k += 32) any |= slot_counts(index[row * K + k], values[row * K + k], V);
    n += __any_sync(0xffffffffu, any) ? 1 : 0;
  }
  if (lane == 0 && n) atomicAdd(&s_n, n);
  __syncthreads();
  if (threadIdx.x == 0 && s_n) atomicAdd(count, s_n);      // whole numbers: the order does not matter
}

struct KlParams {
  const void* student;
  long long ld;                    // elements between rows
  const void* values;              // [rows, K]
  const long long* index;          // [rows, K]
  const float* lse;                // [rows] or null
  float* row_loss;                 // [rows]
  float2* stats;                   // [rows]: (maximum, sum of exponentials)
  void* grad;                      // [rows, V] contiguous (its pitch is ldg), or null
  long long ldg;
  const int* count;                // rows that count (mean), or null
  int* ticket;                     // 0 before the launch; the block that makes it `blocks` adds the rows' losses
  float* loss;                     // the sum (mean) of row_loss, or null
  const float* upstream;           // backward: gradient of the loss, one number or one per row
  int upstream_rows, skip_one;     // skip_one: the gradient is there already for an upstream of 1
  long long rows;
  int V, K;
  float tau;
};

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = lanes_sum<32>(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < (blockDim.x >> 5) ? scratch[threadIdx.x & 31] : 0.f;
  return lanes_sum<32>(v);
}
__device__ __forceinline__ float block_max(float v, float* scratch) {
  v = lanes_max<32>(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < (blockDim.x >> 5) ? scratch[threadIdx.x & 31] : -CUDART_INF_F;
  return lanes_max<32>(v);
}

// Teacher's side of a row into shared memory: index (-1 where a slot does not count), p and log p. Returns sum p.
template <typename TT>
__device__ __forceinline__ float teacher_row(const KlParams& p, long long row, int* s_at, float* s_p, float* s_logp,
                                             float* scratch) {
  const TT* tv = static_cast<const TT*>(p.values) + row * p.K;
  const long long* ti = p.index + row * p.K;
  const float inv_tau = 1.f / p.tau;
  float top = -CUDART_INF_F;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const long long at = ti[k];
    const bool ok = slot_counts(at, tv[k], p.V);
    const float t = to_f32(tv[k]) * inv_tau;
    s_at[k] = ok ? static_cast<int>(at) : -1;
    s_logp[k] = ok ? t : -CUDART_INF_F;
    if (ok) top = fmaxf(top, t);
  }
  float base;
  if (p.lse != nullptr) {
    base = p.lse[row];
    __syncthreads();
  } else {
    top = block_max(top, scratch);
    if (top == -CUDART_INF_F) top = 0.f;                   // nothing counts (or NaN alone, which the sum carries on)
    float s = 0.f;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) s += expf(s_logp[k] - top);
    base = top + logf(block_sum(s, scratch));
  }
  float mass = 0.f;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const float lp = s_logp[k] - base;
    const float pk = s_at[k] >= 0 ? expf(lp) : 0.f;
    s_logp[k] = lp;
    s_p[k] = pk;
    mass += pk;
  }
  return block_sum(mass, scratch);
}

template <typename T> __device__ __forceinline__ int head_of(const T* p, int V) {
  const int to = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
  return to < V ? to : V;
}

// The gradient of one row, `total` = sum of exponentials around `mc` = maximum * c.
template <typename T>
__device__ __forceinline__ void write_gradient(const KlParams& p, const T* sr, T* gr, const int* s_at, const float* s_p, float c,
                                               float mc, float share, float scale) {
  constexpr int N = Vec16<T>::N;
  const float a = share * scale;
  const int head = head_of(sr, p.V);
  const bool wide = ((reinterpret_cast<uintptr_t>(sr) ^ reinterpret_cast<uintptr_t>(gr)) & 15) == 0;
  const int nv = wide ? (p.V - head) / N : 0, body = wide ? head + nv * N : 0;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    float f[N];
    Vec16<T>::unpack(reinterpret_cast<const uint4*>(sr + head)[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = exp2_unit(fmaf(f[j], c, -mc)) * a;
    reinterpret_cast<uint4*>(gr + head)[i] = Vec16<T>::pack(f);
  }
  if (wide)
    for (int i = threadIdx.x; i < head; i += blockDim.x) gr[i] = from_f32<T>(exp2_unit(fmaf(to_f32(sr[i]), c, -mc)) * a);
  for (int i = body + threadIdx.x; i < p.V; i += blockDim.x) gr[i] = from_f32<T>(exp2_unit(fmaf(to_f32(sr[i]), c, -mc)) * a);
}

template <typename T, typename TT, bool FWD>
__global__ void __launch_bounds__(KL_THREADS) kl_topk_kernel(const KlParams p) {
  constexpr int N = Vec16<T>::N;
  extern __shared__ float s_teacher[];                     // p, log p, index, student logit at index: K each
  __shared__ float scratch[32];
  __shared__ int s_last;
  pdl_wait();
  pdl_launch_dependents();
  float *s_p = s_teacher, *s_logp = s_p + p.K;
  int* s_at = reinterpret_cast<int*>(s_logp + p.K);
  float* s_x = reinterpret_cast<float*>(s_at + p.K);
  const float c = LOG2E / p.tau, inv_tau = 1.f / p.tau;
  const float per_row = p.count != nullptr ? 1.f / static_cast<float>(max(*p.count, 1)) : 1.f;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float up = 1.f;
    if constexpr (!FWD) {
      up = p.upstream[p.upstream_rows ? row : 0];
      if (p.skip_one && up == 1.f) continue;
    }
    __syncthreads();
    const T* sr = static_cast<const T*>(p.student) + row * p.ld;
    T* gr = p.grad != nullptr ? static_cast<T*>(p.grad) + row * p.ldg : nullptr;
    const float mass = teacher_row<TT>(p, row, s_at, s_p, s_logp, scratch);
    bool some = false;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) some |= s_at[k] >= 0;
    if (!__syncthreads_or(some)) {
      if (FWD && threadIdx.x == 0) { p.row_loss[row] = 0.f; p.stats[row] = make_float2(0.f, 1.f); }
      if (gr != nullptr)
        for (int i = threadIdx.x; i < p.V; i += blockDim.x) gr[i] = from_f32<T>(0.f);
      continue;
    }
    float m, total;
    if constexpr (FWD) {
      float tm = -CUDART_INF_F, ts = 0.f;                  // this thread's maximum and sum around it
      const int head = head_of(sr, p.V), nv = (p.V - head) / N;
      auto add = [&](float top, auto&& sum) {
        if (top > tm) {
          ts *= tm == -CUDART_INF_F ? 0.f : exp2_unit((tm - top) * c);
          tm = top;
        }
        ts += sum(tm == -CUDART_INF_F ? 0.f : tm * c);
      };
      for (int i = threadIdx.x; i < nv; i += blockDim.x) {
        float f[N];
        Vec16<T>::unpack(reinterpret_cast<const uint4*>(sr + head)[i], f);
        float top = f[0];
#pragma unroll
        for (int j = 1; j < N; ++j) top = fmaxf(top, f[j]);
        add(top, [&](float mc) {
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < N; ++j) s += exp2_unit(fmaf(f[j], c, -mc));
          return s;
        });
      }
      for (int i = threadIdx.x; i < p.V - nv * N; i += blockDim.x) {
        const float f = to_f32(sr[i < head ? i : i + nv * N]);
        add(f, [&](float mc) { return exp2_unit(fmaf(f, c, -mc)); });
      }
      m = block_max(tm, scratch);
      total = block_sum(tm == -CUDART_INF_F ? ts : ts * exp2_unit((tm - m) * c), scratch);
      if (threadIdx.x == 0) p.stats[row] = make_float2(m, total);
      float part = 0.f;
      const float log_total = logf(total);
      for (int k = threadIdx.x; k < p.K; k += blockDim.x)
        if (s_at[k] >= 0) {
          const float x = to_f32(sr[s_at[k]]);
          s_x[k] = x;
          if (!(s_p[k] == 0.f)) part += s_p[k] * (s_logp[k] - ((x - m) * inv_tau - log_total));
        }
      part = block_sum(part, scratch);
      if (threadIdx.x == 0) p.row_loss[row] = part;
    } else {
      const float2 st = p.stats[row];
      m = st.x;
      total = st.y;
      for (int k = threadIdx.x; k < p.K; k += blockDim.x)
        if (s_at[k] >= 0) s_x[k] = to_f32(sr[s_at[k]]);
    }
    if (gr == nullptr) continue;
    const float mc = m * c, share = mass / total, scale = per_row * up * inv_tau;
    __syncthreads();                                       // all of the teacher's logits are read: gr may be sr itself
    write_gradient<T>(p, sr, gr, s_at, s_p, c, mc, share, scale);
    __syncthreads();
    // an index that stands more than once: each of its slots writes the same sum, taken in slot order
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
      if (s_at[k] < 0) continue;
      float want = 0.f;
      for (int j = 0; j < p.K; ++j) want += s_at[j] == s_at[k] ? s_p[j] : 0.f;
      gr[s_at[k]] = from_f32<T>((exp2_unit(fmaf(s_x[k], c, -mc)) * share - want) * scale);
    }
  }
  if constexpr (FWD) {
    if (p.loss == nullptr) return;
    // the last block to finish adds the rows in a fixed order
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    float v = 0.f;
    for (long long i = threadIdx.x; i < p.rows; i += blockDim.x) v += __ldcg(p.row_loss + i);
    v = block_sum(v, scratch);
    if (threadIdx.x == 0) *p.loss = v * per_row;
  }
}

template <typename T, typename TT>
int kl_run(KlParams p, bool fwd, int* ws, bool mean, const int* count, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(p.K) * 16;
  cudaError_t e = cudaSuccess;
  if (fwd) {
    if (cudaMemsetAsync(ws, 0, 2 * sizeof(int), stream) != cudaSuccess) return -3;
    p.ticket = ws + 1;
  }
  if (mean) {
    if (count == nullptr) {
      count = ws;
      if (fwd) {
        const long long blocks = (p.rows + 7) / 8 < 4LL * sm_count() ? (p.rows + 7) / 8 : 4LL * sm_count();
        e = launch_pdl(kl_topk_count_kernel<TT>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                       static_cast<const TT*>(p.values), p.index, ws, p.rows, p.V, p.K);
        if (e != cudaSuccess) return -3;
      }
    }
    p.count = count;
  }
  const long long blocks = p.rows < 4LL * sm_count() ? p.rows : 4LL * sm_count();
  e = fwd ? launch_pdl(kl_topk_kernel<T, TT, true>, dim3(static_cast<unsigned>(blocks)), dim3(KL_THREADS), smem, stream, p)
          : launch_pdl(kl_topk_kernel<T, TT, false>, dim3(static_cast<unsigned>(blocks)), dim3(KL_THREADS), smem, stream, p);
  return e == cudaSuccess ? 0 : -3;
}

int kl_dispatch(const KlParams& p, int dtype, int t_dtype, bool fwd, int* ws, bool mean, const int* count, cudaStream_t stream) {
  if (dtype == FMB_BF16 && t_dtype == FMB_BF16) return kl_run<__nv_bfloat16, __nv_bfloat16>(p, fwd, ws, mean, count, stream);
  if (dtype == FMB_BF16 && t_dtype == FMB_F32) return kl_run<__nv_bfloat16, float>(p, fwd, ws, mean, count, stream);
  if (dtype == FMB_F32 && t_dtype == FMB_BF16) return kl_run<float, __nv_bfloat16>(p, fwd, ws, mean, count, stream);
  if (dtype == FMB_F32 && t_dtype == FMB_F32) return kl_run<float, float>(p, fwd, ws, mean, count, stream);
  return -1;
}

}  // namespace fmb

using namespace fmb;

extern "C" int fmb_kl_topk_fwd(const void* student, long long ld, const void* values, const long long* index, const float* lse,
                               float* row_loss, float* stats, void* grad, long long ldg, const int* count, int* ws, float* loss,
                               long long rows, int V, int K, float tau, int mean, int dtype, int t_dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || K <= 0 || K > FMB_KL_MAX_KEEP || !(tau > 0.f)) return -2;
  KlParams p = {};
  p.student = student; p.ld = ld; p.values = values; p.index = index; p.lse = lse; p.row_loss = row_loss;
  p.stats = reinterpret_cast<float2*>(stats); p.grad = grad; p.ldg = ldg; p.loss = loss; p.rows = rows; p.V = V; p.K = K;
  p.tau = tau;
  return kl_dispatch(p, dtype, t_dtype, true, ws, mean != 0, count, stream);
}

extern "C" int fmb_kl_topk_bwd(const void* student, long long ld, const void* values, const long long* index, const float* lse,
                               const float* stats, void* grad, long long ldg, const int* count, const float* upstream,
                               int upstream_rows, int skip_one, long long rows, int V, int K, float tau, int dtype, int t_dtype,
                               cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || K <= 0 || K > FMB_KL_MAX_KEEP || !(tau > 0.f) || upstream == nullptr) return -2;
  KlParams p = {};
  p.student = student; p.ld = ld; p.values = values; p.index = index; p.lse = lse;
  p.stats = const_cast<float2*>(reinterpret_cast<const float2*>(stats)); p.grad = grad; p.ldg = ldg; p.upstream = upstream;
  p.upstream_rows = upstream_rows; p.skip_one = skip_one; p.rows = rows; p.V = V; p.K = K; p.tau = tau;
  return kl_dispatch(p, dtype, t_dtype, false, nullptr, count != nullptr, count, stream);
}

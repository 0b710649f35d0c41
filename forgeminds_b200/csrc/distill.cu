// Distillation from the K largest logits of a teacher: loss and gradient over rows of student logits.
//
//   p_k = softmax over the row's kept teacher logits / tau   (or exp(t_k / tau - lse) when the teacher's normaliser is known)
//   q   = softmax(student / tau)
//   row = sum_k p_k (log p_k - log q[index_k]),   gradient = (q sum_k p_k - p scattered to index) scale / tau
//
// A slot whose index is outside [0, V), or whose teacher logit is -inf, does not count; a row without slots that
// count has no loss and no gradient. An index that stands twice in a row counts twice.
// Bound by HBM bandwidth: one exponential per student logit and pass. Sums and statistics are fp32; exponentials are
// 2^x of the special function unit (relative error 2^-22). Their argument is a difference of logits, taken before it is
// scaled: m / tau of a large logit, or of a small tau, is rounded to more than the exponent can bear, and of a mask of the
// type's lowest value it overflows (folded into one multiply-add, x / tau - m / tau, such rows were NaN).
#include "fmb_api.h"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "rows.cuh"

namespace fmb {

constexpr int KL_THREADS = 512;
constexpr int KL_COUNT_BLOCKS = 256, KL_COUNT_ROWS = 4;
constexpr float LOG2E = 1.4426950408889634f;

template <typename TT> __device__ __forceinline__ bool slot_counts(long long at, TT value, int V) {
  return at >= 0 && at < V && !(to_f32(value) == -CUDART_INF_F);
}

// Scratch of a forward pass: rows that count, the ticket, rows given out, then the blocks' parts of the count. Nothing has to
// be cleared before the count kernel, which leaves one part per block and clears the two counters.
constexpr int WS_COUNT = 0, WS_TICKET = 1, WS_TAKEN = 2, WS_PARTS = 4;
static_assert(WS_PARTS + KL_COUNT_BLOCKS == FMB_KL_SCRATCH, "the caller's scratch");

// Rows that have a slot that counts. A warp looks at the first 32 slots of four rows at once, which nearly always settles
// them (8192 rows of 64: 6.9 us with all slots of one row after another, 4.4 with this).
template <typename TT>
__global__ void __launch_bounds__(256)
kl_topk_count_kernel(const TT* __restrict__ values, const long long* __restrict__ index, int* __restrict__ ws,
                     long long rows, int V, int K) {
  __shared__ int s_n;
  if (threadIdx.x == 0) s_n = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (long long row = (blockIdx.x * 8LL + (threadIdx.x >> 5)) * KL_COUNT_ROWS; row < rows; row += gridDim.x * 8LL * KL_COUNT_ROWS) {
    long long at[KL_COUNT_ROWS];
    TT value[KL_COUNT_ROWS];
#pragma unroll
    for (int i = 0; i < KL_COUNT_ROWS; ++i) {
      at[i] = -1;
      value[i] = from_f32<TT>(0.f);
      if (row + i < rows && lane < K) {
        at[i] = index[(row + i) * K + lane];
        value[i] = values[(row + i) * K + lane];
      }
    }
#pragma unroll
    for (int i = 0; i < KL_COUNT_ROWS; ++i) {
      bool any = __any_sync(0xffffffffu, slot_counts(at[i], value[i], V));
      for (int k = 32 + lane; !any && row + i < rows && k - lane < K; k += 32)
        any = __any_sync(0xffffffffu, k < K && slot_counts(index[(row + i) * K + min(k, K - 1)], values[(row + i) * K + min(k, K - 1)], V));
      n += any ? 1 : 0;
    }
  }
  if (lane == 0 && n) atomicAdd(&s_n, n);
  __syncthreads();
  if (threadIdx.x == 0) {
    ws[WS_PARTS + blockIdx.x] = s_n;
    if (blockIdx.x == 0) ws[WS_TICKET] = ws[WS_TAKEN] = 0;
  }
}

struct KlParams {
  const void* student;
  long long ld;                    // elements between rows
  const void* values;              // [rows, K]
  const long long* index;          // [rows, K]
  const float* lse;                // [rows] or null
  float* row_loss;                 // [rows]
  float2* stats;                   // [rows]: (a logit that is the maximum or near it, sum of exponentials around it)
  void* grad;                      // [rows, V] contiguous (its pitch is ldg), or null
  long long ldg;
  const int* count;                // rows that count (mean), or null
  int* parts;                      // scratch whose parts the count is the sum of, and where it is then left; or null
  int n_parts;
  int* ticket;                     // 0 before the launch; the block that makes it `blocks` adds the rows' losses
  int* taken;                      // 0 before the launch: rows that have been given out
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

// What the losses are divided by: 1, the count that is given, or the sum of the parts, which every block takes and leaves
// beside them for the backward pass.
__device__ __forceinline__ float rows_that_count(const KlParams& p, int* scratch) {
  if (p.parts == nullptr) return p.count != nullptr ? static_cast<float>(max(*p.count, 1)) : 1.f;
  int n = 0;
  for (int i = threadIdx.x; i < p.n_parts; i += blockDim.x) n += p.parts[WS_PARTS + i];
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) n += scratch[w];
  if (threadIdx.x == 0) p.parts[WS_COUNT] = n;
  return static_cast<float>(max(n, 1));
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
    const float t = to_f32(tv[k]);
    s_at[k] = ok ? static_cast<int>(at) : -1;
    s_logp[k] = ok ? t : -CUDART_INF_F;
    if (ok) top = fmaxf(top, t);
  }
  float base = 0.f;
  if (p.lse != nullptr) {
    const float lse = p.lse[row];
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) s_logp[k] = fmaf(s_logp[k], inv_tau, -lse);
    __syncthreads();
  } else {
    top = block_max(top, scratch);
    if (top == -CUDART_INF_F) top = 0.f;                   // nothing counts (or NaN alone, which the sum carries on)
    float s = 0.f;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
      s_logp[k] = (s_logp[k] - top) * inv_tau;
      s += expf(s_logp[k]);
    }
    base = logf(block_sum(s, scratch));
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

// The gradient of one row, `share` = sum p / sum of exponentials around `m`.
template <typename T>
__device__ __forceinline__ void write_gradient(const KlParams& p, const T* sr, T* gr, const int* s_at, const float* s_p, float c,
                                               float m, float share, float scale) {
  constexpr int N = Vec16<T>::N;
  const float a = share * scale;
  const int head = head_of(sr, p.V);
  const bool wide = ((reinterpret_cast<uintptr_t>(sr) ^ reinterpret_cast<uintptr_t>(gr)) & 15) == 0;
  const int nv = wide ? (p.V - head) / N : 0, body = wide ? head + nv * N : 0;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    float f[N];
    Vec16<T>::unpack(reinterpret_cast<const uint4*>(sr + head)[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = exp2_unit((f[j] - m) * c) * a;
    reinterpret_cast<uint4*>(gr + head)[i] = Vec16<T>::pack(f);
  }
  if (wide)
    for (int i = threadIdx.x; i < head; i += blockDim.x) gr[i] = from_f32<T>(exp2_unit((to_f32(sr[i]) - m) * c) * a);
  for (int i = body + threadIdx.x; i < p.V; i += blockDim.x) gr[i] = from_f32<T>(exp2_unit((to_f32(sr[i]) - m) * c) * a);
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
  if (!FWD && p.skip_one && !p.upstream_rows && *p.upstream == 1.f) return;
  __shared__ int s_parts[KL_THREADS / 32];
  const float per_row = 1.f / rows_that_count(p, s_parts);
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
        ts += sum(tm == -CUDART_INF_F ? 0.f : tm);
      };
      for (int i = threadIdx.x; i < nv; i += blockDim.x) {
        float f[N];
        Vec16<T>::unpack(reinterpret_cast<const uint4*>(sr + head)[i], f);
        float top = f[0];
#pragma unroll
        for (int j = 1; j < N; ++j) top = fmaxf(top, f[j]);
        add(top, [&](float from) {
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < N; ++j) s += exp2_unit((f[j] - from) * c);
          return s;
        });
      }
      for (int i = threadIdx.x; i < p.V - nv * N; i += blockDim.x) {
        const float f = to_f32(sr[i < head ? i : i + nv * N]);
        add(f, [&](float from) { return exp2_unit((f - from) * c); });
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
    const float share = mass / total, scale = per_row * up * inv_tau;
    __syncthreads();                                       // all of the teacher's logits are read: gr may be sr itself
    write_gradient<T>(p, sr, gr, s_at, s_p, c, m, share, scale);
    __syncthreads();
    // an index that stands more than once: each of its slots writes the same sum, taken in slot order
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
      if (s_at[k] < 0) continue;
      float want = 0.f;
      for (int j = 0; j < p.K; ++j) want += s_at[j] == s_at[k] ? s_p[j] : 0.f;
      gr[s_at[k]] = from_f32<T>((exp2_unit((s_x[k] - m) * c) * share - want) * scale);
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

// ------------------------------------------------------------------ rows that stay in shared memory
// A row is split over the CTAs of a cluster, at most 64 KB for each so that three of them share an SM: the logits are read
// from memory once, and the sum of exponentials and the gradient are taken from there. A thread keeps to its own 16-byte
// vectors, and as soon as the gradient has used one, the same place receives the next row's: loads, exponentials and stores
// of the SM's CTAs overlap. The sum is one pass: exponentials are taken around a logit that is within 2^8 of the largest so
// far, and the threads' sums are brought to the row's largest such logit afterwards (a pass for the maximum before it cost
// 3 % more). Few threads per row (256, or 128), because the reductions and the row's bookkeeping cost each
// warp as much as some fifty vectors do. Kept logit k belongs to thread k, whose maximum and sums join the row's own
// reductions. The CTAs of a row exchange (maximum, sum around it, loss) once. Rows are given out one by one: clusters that
// find no place at first, while an earlier kernel still holds some SMs, would otherwise be a second wave.
// Measured, with gradient and the count of rows, bf16, one call behind another: 8192 x 32000 in 185 us (5.7 TB/s of logits and
// gradient; one block per row that reads it twice took twice as long), 4096 x 128259 over four CTAs in 460 us (4.6 TB/s): there
// a row's CTAs wait for one another for a fifth of the time. Exponents folded into one multiply-add, which is wrong for some
// rows (see the top), took 181 and 440. Both exponentials of a logit together hold the special function unit for 60 % of the
// time, half of the issue slots are used.

// m: a logit near the maximum of the CTA's own; s: sum of exponentials around it; over the kept logits that are held here
// a: sum e (log e - (x - m) / tau), w: sum e, which brings a to the row's m
struct KlPart {
  float m, s, a, w;
};

// A row of V values: `head` of them before the first 16-byte boundary, then nv whole vectors, then the rest. The up to
// 2 N - 2 values outside the vectors are held singly by the first threads of the row's first CTA.
template <typename T> struct KlRow {
  static constexpr int N = Vec16<T>::N;
  const T* at;
  int head, nv;
  __device__ __forceinline__ KlRow(const T* p, int V) : at(p), head(head_of(p, V)) { nv = (V - head) / N; }
  __device__ __forceinline__ const uint4* vectors() const { return reinterpret_cast<const uint4*>(at + head); }
  __device__ __forceinline__ int single(int t) const { return t < head ? t : nv * N + t; }       // of thread t
};

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

constexpr int KL_ROW_THREADS = 256;                        // most of a CTA: the kept logits that it can take
constexpr int KL_MARKS = 1024;                             // words of the marks by which an index that stands twice is found
constexpr int KL_ROW_BYTES = 64 * 1024;                    // most of a row in one CTA, and
constexpr int KL_ROW_MOST = 192 * 1024;                    // where eight CTAs of that do not hold it

template <typename T, typename TT, int THREADS>
__global__ void __launch_bounds__(THREADS, 3 * KL_ROW_THREADS / THREADS)
kl_topk_row_kernel(const __grid_constant__ KlParams p, int split, int per_cta) {
  constexpr int N = Vec16<T>::N, H = N / 2, WARPS = THREADS / 32;
  extern __shared__ uint4 s_row[];                         // [per_cta]: this CTA's part of the row
  __shared__ unsigned s_marks[KL_MARKS];
  __shared__ int s_at[THREADS];
  __shared__ float s_e[THREADS];
  __shared__ KlPart s_part[2][8];
  __shared__ float2 s_max[WARPS];
  __shared__ float4 s_sum[WARPS];
  __shared__ float scratch[32], s_single[2 * N];
  __shared__ int s_last;
  __shared__ int2 s_given[2];                              // rows that this CTA is told
  for (int i = threadIdx.x; i < KL_MARKS; i += THREADS) s_marks[i] = 0;
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  // tells a row (two at the start) to all CTAs of this one's cluster; they see it behind the next barrier
  auto give = [&](int which, int a, int b) {
    for (int i = 0; i < split; ++i) {
      if (split > 1) {
        const uint32_t to = mapa_shared(smem_u32(&s_given[which]), i);
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(to), "r"(a) : "memory");
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(to + 4), "r"(b) : "memory");
      } else {
        s_given[which] = make_int2(a, b);
      }
    }
  };
  const float c = LOG2E / p.tau, inv_tau = 1.f / p.tau;
  const float counted = rows_that_count(p, s_at), scale = inv_tau / counted;
  const int first = rank * per_cta;                        // this CTA's first vector
  const bool slot = threadIdx.x < p.K;
  const F2 c2 = f2(c, c);
  const float slack = 8.f / c;
  float single = -CUDART_INF_F;
  // vectors of this CTA in a row
  auto held = [&](const KlRow<T>& r) { return min(per_cta, r.nv - first); };
  const uint32_t s_mine = smem_u32(s_row);
  auto fetch = [&](const uint4* from, int i) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s_mine + i * 16), "l"(from + i) : "memory");
  };
  auto load_single = [&](const KlRow<T>& r) {
    return rank == 0 && static_cast<int>(threadIdx.x) < p.V - r.nv * N ? to_f32(r.at[r.single(threadIdx.x)]) : -CUDART_INF_F;
  };
  // This thread's kept logit. The loads for the next row are issued a row ahead and looked at when that row begins: a
  // comparison where they are issued would hold the CTA up for their 2800 cycles.
  long long slot_index = -1;
  TT slot_value = from_f32<TT>(0.f);
  float lse = 0.f;
  auto load_slot = [&](long long r) {
    slot_index = -1;
    if (p.lse != nullptr && r < p.rows) lse = p.lse[r];
    if (slot && r < p.rows) {
      slot_index = p.index[r * p.K + threadIdx.x];
      slot_value = static_cast<const TT*>(p.values)[r * p.K + threadIdx.x];
    }
  };
  if (split > 1) cluster_sync_all();                       // every CTA of the row runs before one writes to another
  if (rank == 0 && threadIdx.x == 0) {
    const int first_row = atomicAdd(p.taken, 2);
    give(0, first_row, first_row + 1);
  }
  if (split > 1) cluster_sync_all();
  else __syncthreads();
  long long row = s_given[0].x, next = s_given[0].y;
  if (row < p.rows) {
    const KlRow<T> r(static_cast<const T*>(p.student) + row * p.ld, p.V);
    const int n = held(r);
    for (int i = threadIdx.x; i < n; i += THREADS) fetch(r.vectors() + first, i);
    single = load_single(r);
    load_slot(row);
  }
  int side = 0;
  while (row < p.rows) {
    side ^= 1;
    int after = 0;                                         // the row after the next one
    if (rank == 0 && threadIdx.x == 0 && next < p.rows) after = atomicAdd(p.taken, 1);
    const KlRow<T> r(static_cast<const T*>(p.student) + row * p.ld, p.V);
    const int n = held(r);
    const int at = slot_counts(slot_index, slot_value, p.V) ? static_cast<int>(slot_index) : -1;
    const float t = at >= 0 ? to_f32(slot_value) : -CUDART_INF_F;
    asm volatile("cp.async.wait_all;" ::: "memory");       // its own copies: other threads read them behind a barrier
    // one pass: exponentials of this thread's logits around `around`, which need not be their maximum, only within 2^8 of it
    float around = single;
    F2 sums = f2(single == -CUDART_INF_F ? 0.f : 1.f, 0.f), more = f2(0.f, 0.f);
    {
      float limit = around + slack;
      F2 less = f2(0.f, 0.f);
      auto start = [&](float top) {                        // rare, but for the first vector
        const float k = around == -CUDART_INF_F ? 0.f : exp2_unit((around - top) * c);
        sums = f2_mul(sums, f2(k, k));
        more = f2_mul(more, f2(k, k));
        around = top;
        limit = top + slack;
        less = f2(-top, -top);
      };
      if (around != -CUDART_INF_F) less = f2(-around, -around);
#pragma unroll 2
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint4 x = s_row[i];
        float f[N], top;
        Vec16<T>::unpack(x, f);
        if constexpr (sizeof(T) == 2) {
          const uint32_t u = max_bf16x2(max_bf16x2(x.x, x.y), max_bf16x2(x.z, x.w));
          top = fmaxf(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
        } else {
          top = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
        }
        if (!(top <= limit)) start(top);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const float2 o = f2_mul(f2_add(f2(f[2 * j], f[2 * j + 1]), less), c2);
          if (j % 2) more = f2_add(more, f2(exp2_unit(o.x), exp2_unit(o.y)));
          else sums = f2_add(sums, f2(exp2_unit(o.x), exp2_unit(o.y)));
        }
      }
      sums = f2_add(sums, more);
    }
    float m = lanes_max<32>(around);
    float ref = lanes_max<32>(t);
    if (lane == 0) s_max[warp] = make_float2(m, ref);
    if (threadIdx.x < 2 * N) s_single[threadIdx.x] = single;
    const bool some = __syncthreads_or(at >= 0);
    {
      const float2 o = s_max[lane % WARPS];
      m = lanes_max<WARPS>(o.x);
      ref = lanes_max<WARPS>(o.y);
    }
    if (ref == -CUDART_INF_F) ref = 0.f;                   // nothing counts, or NaN alone
    const float logit = p.lse != nullptr ? fmaf(t, inv_tau, -lse) : (t - ref) * inv_tau;      // log of e below
    const KlRow<T> rn(static_cast<const T*>(p.student) + next * p.ld, p.V);
    const int nn = next < p.rows ? held(rn) : 0;
    float next_single = next < p.rows ? load_single(rn) : -CUDART_INF_F;
    load_slot(next);
    // sums: exponentials of the student, e of the teacher, and KlPart's a and w
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float s = (sums.x + sums.y) * (around == -CUDART_INF_F ? 0.f : exp2_unit((around - m) * c)), e = 0.f, a = 0.f, xk = 0.f;
    bool mine = false, twice = false;                      // whether the student's logit at the index is held here
    int mark = -1;
    if (at >= 0) {
      const int v = at - r.head, own = v - first * N;
      if (v < 0 || v >= r.nv * N) {
        mine = rank == 0;
        xk = s_single[v < 0 ? at : at - r.nv * N];
      } else if (own >= 0 && own < per_cta * N) {
        mine = true;
        xk = to_f32(reinterpret_cast<const T*>(s_row)[own]);
      }
      e = expf(logit);
      if (mine && !(e == 0.f)) a = e * (logit - (xk - base) * inv_tau);
      // a mark that is set already: an index that stands twice, or in a few rows of a hundred two that share a mark
      const unsigned h = static_cast<unsigned>(at) * 2654435761u >> 17;
      mark = h >> 5;
      twice = atomicOr(s_marks + mark, 1u << (h & 31)) >> (h & 31) & 1;
    }
    if (slot) {
      s_at[threadIdx.x] = at;
      s_e[threadIdx.x] = e;
    }
    s = lanes_sum<32>(s);
    float mass = lanes_sum<32>(e);
    a = lanes_sum<32>(a);
    float w = 0.f;
    if (split > 1) w = lanes_sum<32>(mine ? e : 0.f);
    if (lane == 0) s_sum[warp] = make_float4(s, mass, a, w);
    if (rank == 0 && threadIdx.x == 0) give(side, next < p.rows ? after : static_cast<int>(p.rows), 0);
    twice = __syncthreads_or(twice);                       // also: every logit at an index has been taken from the row's copy
    if (mark >= 0) s_marks[mark] = 0;                      // the next row's first mark is behind another barrier
    {
      const float4 o = s_sum[lane % WARPS];
      s = lanes_sum<WARPS>(o.x);
      mass = lanes_sum<WARPS>(o.y);
      a = lanes_sum<WARPS>(o.z);
      if (split > 1) w = lanes_sum<WARPS>(o.w);
    }
    if (split > 1) {
      if (threadIdx.x < split) {                           // a copy of this CTA's part for each of the row's CTAs
        const uint32_t to = mapa_shared(smem_u32(&s_part[side][rank]), threadIdx.x);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(a) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 12), "f"(w) : "memory");
      }
      cluster_arrive_after(warp == 0);
      cluster_wait();
      m = s_part[side][0].m;
      for (int i = 1; i < split; ++i) m = fmaxf(m, s_part[side][i].m);
      s = a = 0.f;
      for (int i = 0; i < split; ++i) {
        const KlPart o = s_part[side][i];
        s += o.m == -CUDART_INF_F ? o.s : o.s * exp2_unit((o.m - m) * c);
        a += o.w == 0.f ? o.a : o.a + o.w * ((m - (o.m == -CUDART_INF_F ? 0.f : o.m)) * inv_tau);
      }
    }
    // p = e / sum e, or e itself beside the teacher's own normaliser
    const float norm = p.lse != nullptr || !some ? 1.f : __fdividef(1.f, mass);
    const float whole = p.lse != nullptr ? mass : 1.f;     // sum p
    if (rank == 0 && threadIdx.x == 0) {
      p.row_loss[row] = some ? a * norm - (p.lse != nullptr ? 0.f : logf(mass)) + whole * logf(s) : 0.f;
      p.stats[row] = make_float2(m, s);
    }
    const uint4* from = rn.vectors() + first;
    if (p.grad == nullptr) {
      for (int i = threadIdx.x; i < nn; i += THREADS) fetch(from, i);
    } else {
      const float share = __fdividef(whole, s);
      T* gr = static_cast<T*>(p.grad) + row * p.ldg;
      T* to = gr + r.head + first * N;
      const bool wide = ((reinterpret_cast<uintptr_t>(r.at) ^ reinterpret_cast<uintptr_t>(gr)) & 15) == 0;
      if (rank == 0 && static_cast<int>(threadIdx.x) < p.V - r.nv * N)
        gr[r.single(threadIdx.x)] = from_f32<T>(some ? exp2_unit((single - m) * c) * (share * scale) : 0.f);
      if (wide && some) {
        const F2 less = f2(-m, -m), by2 = f2(share * scale, share * scale);
#pragma unroll 2
        for (int i = threadIdx.x; i < n; i += THREADS) {
          float f[N];
          Vec16<T>::unpack(s_row[i], f);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            float2 o = f2_mul(f2_add(f2(f[2 * j], f[2 * j + 1]), less), c2);
            o = (f2_mul(f2(exp2_unit(o.x), exp2_unit(o.y)), by2));
            f[2 * j] = o.x;
            f[2 * j + 1] = o.y;
          }
          reinterpret_cast<uint4*>(to)[i] = Vec16<T>::pack(f);
          if (i < nn) fetch(from, i);                      // the vector has been used: its place is free
        }
      } else {                                             // a row without slots that count, or rows that lie differently in
        for (int i = threadIdx.x; i < n; i += THREADS) {   // the gradient: single values
          float f[N];
          Vec16<T>::unpack(s_row[i], f);
#pragma unroll
          for (int j = 0; j < N; ++j) to[i * N + j] = from_f32<T>(some ? exp2_unit((f[j] - m) * c) * (share * scale) : 0.f);
          if (i < nn) fetch(from, i);
        }
      }
      // a row of odd length may have one vector more than the one before it
      for (int i = threadIdx.x + (n > static_cast<int>(threadIdx.x) ? (n - threadIdx.x + THREADS - 1) / THREADS * THREADS : 0); i < nn; i += THREADS)
        fetch(from, i);
      if (some) {
        __syncthreads();                                   // the kept logits' own part goes over what has just been written
        if (mine) {
          float want = e;
          if (twice) {                                     // each of its slots writes the same sum, taken in slot order
            want = 0.f;
            for (int j = 0; j < p.K; ++j) want += s_at[j] == at ? s_e[j] : 0.f;
          }
          gr[at] = from_f32<T>((exp2_unit((xk - m) * c) * share - want * norm) * scale);
        }
      }
    }
    single = next_single;
    row = next;
    next = s_given[side].x;
  }
  if (p.loss != nullptr) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (s_last) {                                          // the last CTA adds the rows in a fixed order
      __threadfence();
      float v = 0.f;
      for (long long i = threadIdx.x; i < p.rows; i += THREADS) v += __ldcg(p.row_loss + i);
      v = block_sum(v, scratch);
      if (threadIdx.x == 0) *p.loss = v / counted;
    }
  }
}

// Clusters of `split` CTAs with `smem` bytes each that the device holds together; 0 where the kernel does not run. (A second
// wave of a walk over all rows would double its time: of 74 clusters of 4 that 148 SMs have room for by numbers, 71 fit.)
template <typename T, typename TT, int THREADS> int kl_fit(int split, size_t smem) {
  auto kernel = kl_topk_row_kernel<T, TT, THREADS>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count() / split * split);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int got = 0;
  if (cudaOccupancyMaxActiveClusters(&got, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return got;
}

template <typename T, typename TT, int THREADS> int kl_row_launch(const KlParams& p, int split, int per_cta, cudaStream_t stream) {
  auto kernel = kl_topk_row_kernel<T, TT, THREADS>;
  static bool opted[64] = {};
  int dev = 0;
  const size_t smem = sizeof(uint4) * per_cta;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!opted[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KL_ROW_MOST) != cudaSuccess) return -3;
    opted[dev] = true;
  }
  const long long fit = kl_fit<T, TT, THREADS>(split, smem);
  if (fit < 1) return -3;
  const long long groups = p.rows < fit ? p.rows : fit;
  const dim3 grid(static_cast<unsigned>(groups * split));
  const cudaError_t e = split == 1 ? launch_pdl(kernel, grid, dim3(THREADS), smem, stream, p, split, per_cta)
                                   : launch_cluster(kernel, grid, dim3(THREADS), smem, split, stream, p, split, per_cta);
  return e == cudaSuccess ? 0 : -3;
}

template <typename T, typename TT>
int kl_run(KlParams p, bool fwd, int* ws, bool mean, const int* count, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(p.K) * 16;
  cudaError_t e = cudaSuccess;
  if (fwd) {
    p.ticket = ws + WS_TICKET;
    p.taken = ws + WS_TAKEN;
  }
  if (fwd && mean && count == nullptr) {
    const long long need = (p.rows + 8 * KL_COUNT_ROWS - 1) / (8 * KL_COUNT_ROWS);
    p.n_parts = static_cast<int>(need < KL_COUNT_BLOCKS ? need : KL_COUNT_BLOCKS);
    p.parts = ws;
    e = launch_pdl(kl_topk_count_kernel<TT>, dim3(p.n_parts), dim3(256), 0, stream, static_cast<const TT*>(p.values), p.index, ws,
                   p.rows, p.V, p.K);
    if (e != cudaSuccess) return -3;
  } else if (fwd && cudaMemsetAsync(ws, 0, WS_PARTS * sizeof(int), stream) != cudaSuccess) {
    return -3;
  }
  if (mean) p.count = count;
  if (fwd) {
    // the fewest CTAs (1, 2, 4 or 8) that hold a row, more while SMs would be left without one; a row beyond 512 KB takes
    // eight with up to 192 KB each
    constexpr int N = Vec16<T>::N, MOST = KL_ROW_BYTES / 16, TOP = KL_ROW_MOST / 16;
    const int vectors = p.V / N > 0 ? p.V / N : 1;
    int split = 1;
    while (split < 8 && (vectors + split - 1) / split > MOST) split *= 2;
    while (split < 8 && p.rows * split < sm_count() && vectors / split > 4 * KL_ROW_THREADS) split *= 2;
    const int per_cta = (vectors + split - 1) / split;
    // Many rows of up to 32 KB: half the threads for each and up to six of them at a time. With gradient, bf16, 64 kept:
    // 38910 x 2056 in 166 us against 279 with 256 threads, 9765 x 8192 76 / 98, 4882 x 16384 69 / 76; but 1200 x 12160 26 / 24.
    if (p.rows > 12LL * sm_count() && p.K <= KL_ROW_THREADS / 2 && per_cta <= MOST / 2)
      return kl_row_launch<T, TT, KL_ROW_THREADS / 2>(p, split, per_cta, stream);
    if (p.K <= KL_ROW_THREADS && per_cta <= TOP) return kl_row_launch<T, TT, KL_ROW_THREADS>(p, split, per_cta, stream);
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
                               float* row_loss, float* stats, void* grad, long long ldg, const int* count, int* ws, int ws_ints,
                               float* loss, long long rows, int V, int K, float tau, int mean, int dtype, int t_dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || K <= 0 || K > FMB_KL_MAX_KEEP || !(tau > 0.f) || ws == nullptr || ws_ints < FMB_KL_SCRATCH) return -2;
  if (rows > 0x7fff0000LL) return -2;                      // rows are given out by a counter of 32 bits
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
  if (V <= 0 || K <= 0 || K > FMB_KL_MAX_KEEP || !(tau > 0.f) || upstream == nullptr || rows > 0x7fff0000LL) return -2;
  KlParams p = {};
  p.student = student; p.ld = ld; p.values = values; p.index = index; p.lse = lse;
  p.stats = const_cast<float2*>(reinterpret_cast<const float2*>(stats)); p.grad = grad; p.ldg = ldg; p.upstream = upstream;
  p.upstream_rows = upstream_rows; p.skip_one = skip_one; p.rows = rows; p.V = V; p.K = K; p.tau = tau;
  return kl_dispatch(p, dtype, t_dtype, false, nullptr, count != nullptr, count, stream);
}

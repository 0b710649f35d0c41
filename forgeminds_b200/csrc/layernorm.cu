// LayerNorm of rows, forward (with the residual add in front of it when asked) and backward.
//
//   mean = sum x / d,  var = sum (x - mean)^2 / d,  r = 1 / sqrt(var + eps),  xh = (x - mean) r,  y = xh w + b
//   g = dy w,  dx = r (g - sum g / d - xh sum (g xh) / d) (+ dres),  dw = sum over rows dy xh,  db = sum over rows dy
//
// Bound by HBM bandwidth: about ten operations per element. A row lives in the registers of the threads that
// share it (16-byte chunks), so that mean and variance are two exact passes and memory is read once. Sums,
// statistics and the weight's gradients are fp32. Forward with residual, 16384 x 4096 bf16: 86 us, 6.3 TB/s.
#include "fmb_api.h"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "rows.cuh"

namespace fmb {

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// Rows of a block's ring in the backward pass: 1024 chunks of three tensors are 48 KB each.
template <int CHUNKS> struct BwdStages { static constexpr int N = CHUNKS <= 512 ? 3 : 2; };

// How a thread of a row's TPR threads sees it: chunk i of N values. VEC: 16 contiguous bytes; otherwise N single
// values TPR apart (widths, pitches or addresses that are no multiple of 16 bytes), still coalesced.
template <typename T, int TPR, bool VEC> struct RowMap {
  static constexpr int N = Vec16<T>::N;
  static __device__ __forceinline__ int col(int i, int j, int t) {
    return VEC ? (i * TPR + t) * N + j : (i * N + j) * TPR + t;
  }
  static __device__ __forceinline__ uint4 load(const T* row, int i, int t, int d) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if constexpr (VEC) {
      if (col(i, 0, t) < d) u = *reinterpret_cast<const uint4*>(row + col(i, 0, t));
    } else if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int a = col(i, 2 * j, t), b = col(i, 2 * j + 1, t);
        const uint32_t lo = a < d ? reinterpret_cast<const unsigned short*>(row)[a] : 0;
        const uint32_t hi = b < d ? reinterpret_cast<const unsigned short*>(row)[b] : 0;
        w[j] = lo | hi << 16;
      }
      u = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = col(i, j, t) < d ? reinterpret_cast<const uint32_t*>(row)[col(i, j, t)] : 0;
      u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return u;
  }
  static __device__ __forceinline__ void store(T* row, const float (&f)[N], int i, int t, int d) {
    if constexpr (VEC) {
      if (col(i, 0, t) < d) *reinterpret_cast<uint4*>(row + col(i, 0, t)) = Vec16<T>::pack(f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (col(i, j, t) < d) row[col(i, j, t)] = from_f32<T>(f[j]);
    }
  }
  template <typename WT> static __device__ __forceinline__ void weights(const WT* w, float (&f)[N], int i, int t, int d, float none) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = none;
    if (w == nullptr) return;
    if constexpr (VEC) {
      if (col(i, 0, t) < d) load_f32<WT, N>(w + col(i, 0, t), f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (col(i, j, t) < d) f[j] = to_f32(w[col(i, j, t)]);
    }
  }
};

// Sum over the TPR threads of a row of two values at once. `scratch`: two floats per warp, a buffer of its own for
// each call until every thread has passed the next barrier (callers alternate between two).
template <int TPR> __device__ __forceinline__ float2 row_sum2(float a, float b, float2* scratch) {
  a = lanes_sum<32>(a);
  b = lanes_sum<32>(b);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[warp] = make_float2(a, b);
    __syncthreads();
    constexpr int W = TPR / 32;
    const int first = warp / W * W;
    const float2 s = scratch[first + (threadIdx.x & 31) % W];
    a = lanes_sum<(W < 32 ? W : 32)>(s.x);
    b = lanes_sum<(W < 32 ? W : 32)>(s.y);
  }
  return make_float2(a, b);
}
template <int TPR> __device__ __forceinline__ float row_sum1(float a, float* scratch) {
  a = lanes_sum<32>(a);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[warp] = a;
    __syncthreads();
    constexpr int W = TPR / 32;
    a = lanes_sum<(W < 32 ? W : 32)>(scratch[warp / W * W + (threadIdx.x & 31) % W]);
  }
  return a;
}

// ------------------------------------------------------------------ forward
template <typename T, typename WT, int TPR, int VPL, bool VEC, bool ADD>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
layernorm_fwd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ delta, long long ldd,
                     const WT* __restrict__ w, const WT* __restrict__ b, T* __restrict__ xsum, T* __restrict__ y,
                     float2* __restrict__ stats, long long rows, int d, float inv_d, float eps) {
  using M = RowMap<T, TPR, VEC>;
  constexpr int N = M::N, THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
  __shared__ float s_a[THREADS / 32], s_b[THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x % TPR;
  const long long row = static_cast<long long>(blockIdx.x) * RPB + threadIdx.x / TPR;
  const int width = row < rows ? d : 0;                   // threads without a row take part in the sums with nothing
  const long long at = row < rows ? row : 0;
  float v[VPL][N];
#pragma unroll
  for (int i = 0; i < VPL; ++i) Vec16<T>::unpack(M::load(x + at * ldx, i, t, width), v[i]);
  if constexpr (ADD) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      float e[N];
      Vec16<T>::unpack(M::load(delta + at * ldd, i, t, width), e);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i][j] = to_f32(from_f32<T>(v[i][j] + e[j]));     // the norm is that of the stored sum
      M::store(xsum + at * d, v[i], i, t, width);
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) s += v[i][j];
  const float mean = row_sum1<TPR>(s, s_a) * inv_d;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[i][j] -= mean;
      if (M::col(i, j, t) < width) q += v[i][j] * v[i][j];
    }
  const float r = rsqrtf(row_sum1<TPR>(q, s_b) * inv_d + eps);
  if (width > 0 && t == 0 && stats != nullptr) stats[row] = make_float2(mean, r);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float wv[N], bv[N];
    M::weights(w, wv, i, t, width, 1.f);
    M::weights(b, bv, i, t, width, 0.f);
#pragma unroll
    for (int j = 0; j < N; ++j) v[i][j] = v[i][j] * r * wv[j] + bv[j];
    M::store(y + at * d, v[i], i, t, width);
  }
}

// Rows too wide for registers: one block per row, which is read again from the caches for the variance and the result.
template <typename T, typename WT, bool ADD>
__global__ void __launch_bounds__(1024)
layernorm_fwd_wide_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ delta, long long ldd,
                          const WT* __restrict__ w, const WT* __restrict__ b, T* __restrict__ xsum, T* __restrict__ y,
                          float2* __restrict__ stats, int d, float inv_d, float eps) {
  __shared__ float s_a[32], s_b[32];
  const long long row = blockIdx.x;
  const T* xr = x + row * ldx;
  T* sr = ADD ? xsum + row * d : nullptr;
  float s = 0.f;
  for (int c = threadIdx.x; c < d; c += 1024) {
    float v = to_f32(xr[c]);
    if constexpr (ADD) {
      const T sum = from_f32<T>(v + to_f32(delta[row * ldd + c]));
      sr[c] = sum;                                        // read back below by the thread that wrote it
      v = to_f32(sum);
    }
    s += v;
  }
  const float mean = row_sum1<1024>(s, s_a) * inv_d;
  const T* vr = ADD ? sr : xr;
  float q = 0.f;
  for (int c = threadIdx.x; c < d; c += 1024) {
    const float v = to_f32(vr[c]) - mean;
    q += v * v;
  }
  const float r = rsqrtf(row_sum1<1024>(q, s_b) * inv_d + eps);
  if (threadIdx.x == 0 && stats != nullptr) stats[row] = make_float2(mean, r);
  for (int c = threadIdx.x; c < d; c += 1024)
    y[row * d + c] = from_f32<T>((to_f32(vr[c]) - mean) * r * (w != nullptr ? to_f32(w[c]) : 1.f) + (b != nullptr ? to_f32(b[c]) : 0.f));
}

// ------------------------------------------------------------------ backward
// Blocks walk over the rows. A thread keeps its columns' sums of dy xh and dy in registers; a block leaves them as
// one row of `partial` [blocks, 2, d], which the column kernel below adds in a fixed order. With 16-byte chunks the rows
// come through a ring of shared memory, copied STAGES - 1 rows ahead, each thread its own chunks (no barrier guards them):
// with loads into registers a block waited out the memory's latency at every row. Two chunks per thread from 65 on: what a
// row costs beside its columns (two sums over its threads, statistics, addresses) is as much as 130 instructions a thread.
// dx, dw and db of bf16 rows with dres, the column sums included: 16384 x 4096 in 94 us (5.7 TB/s; with one chunk per
// thread 112, from registers 125), 65536 x 1024 in 88 us (6.1 TB/s; one chunk 96).
template <typename T, typename WT, int TPR, int VPL, bool VEC>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, TPR > 256 ? 1 : VPL > 1 ? 2 : 4)
layernorm_bwd_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ x, long long ldx,
                     const WT* __restrict__ w, const float2* __restrict__ stats, const T* __restrict__ dres, long long ldr,
                     T* __restrict__ dx, float* __restrict__ partial, long long rows, int d, float inv_d) {
  using M = RowMap<T, TPR, VEC>;
  constexpr int N = M::N, THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
  constexpr int STAGES = BwdStages<VPL * THREADS>::N;
  __shared__ float2 scratch[2][THREADS / 32];
  extern __shared__ uint4 s_ring[];                       // [stage][dy, x, dres][chunk][thread]; the fold below takes its place
  float* s_fold = reinterpret_cast<float*>(s_ring);       // [2, d], when several rows share a block
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int tensors = dres != nullptr ? 3 : 2;
  constexpr int H = N / 2;
  F2 wv[VPL][H], dwa[VPL][H], dba[VPL][H];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float f[N];
    M::weights(w, f, i, t, d, 1.f);
#pragma unroll
    for (int j = 0; j < H; ++j) { wv[i][j] = f2(f[2 * j], f[2 * j + 1]); dwa[i][j] = dba[i][j] = f2(0.f, 0.f); }
  }
  // Everything a row needs moves on by one step: pointers, not products, and rows in 31 bits.
  const int n_rows = static_cast<int>(rows), step = gridDim.x * RPB, start = blockIdx.x * RPB + sub;
  const int row_bytes = tensors * VPL * THREADS * 16;
  const char* ring = reinterpret_cast<const char*>(s_ring + threadIdx.x);
  const uint32_t ring_at = smem_at(ring);
  const long long step_dy = step * ldy, step_x = step * ldx, step_res = step * ldr, step_out = static_cast<long long>(step) * d;
  const int own = VEC ? M::col(0, 0, t) : 0;              // this thread's first column, where its chunks are contiguous
  const T *next_dy = dy + start * ldy + own, *next_x = x + start * ldx + own, *next_res = dres + start * ldr + own;
  T* out = dx + static_cast<long long>(start) * d;
  int next_row = start;
  int put = 0, get = 0;                                   // bytes from the ring's start
  auto copy = [&](const T* from, int tensor) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (M::col(i, 0, t) < d)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring_at + put + (tensor * VPL + i) * THREADS * 16),
                     "l"(from + i * TPR * N) : "memory");
  };
  auto fetch = [&]() {                                    // one group for each row, an empty one behind the last
    if (next_row < n_rows) {
      copy(next_dy, 0);
      copy(next_x, 1);
      if (dres != nullptr) copy(next_res, 2);
      next_dy += step_dy;
      next_x += step_x;
      next_res += step_res;
      next_row += step;                                   // stays within 31 bits: it was below the number of rows
    }
    put = put == (STAGES - 1) * row_bytes ? 0 : put + row_bytes;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto held = [&](int tensor, int i) { return *reinterpret_cast<const uint4*>(ring + get + (tensor * VPL + i) * THREADS * 16); };
  auto pairs = [](const uint4& u, F2 (&v)[H]) {
    float f[N];
    Vec16<T>::unpack(u, f);
#pragma unroll
    for (int j = 0; j < H; ++j) v[j] = f2(f[2 * j], f[2 * j + 1]);
  };
  if constexpr (VEC) {
#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) fetch();
  }
  int turn = 0;
  float2 st = stats[min(start, n_rows - 1)];
  for (int base = blockIdx.x * RPB; base < n_rows; base += step, out += step_out) {
    const int row = base + sub;
    const int width = RPB == 1 || row < n_rows ? d : 0;   // rows beyond the last take part in the sums with nothing
    const float2 next_st = stats[min(row + step, n_rows - 1)];
    const F2 mean2 = f2(-st.x, -st.x), r2 = f2(st.y, st.y);
    if constexpr (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    F2 s1 = f2(0.f, 0.f), s2 = s1;
    uint4 rg[VEC ? 1 : VPL], rx[VEC ? 1 : VPL], rr[VEC ? 1 : VPL];
    if constexpr (!VEC) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        rg[i] = M::load(dy + row * ldy, i, t, width);
        rx[i] = M::load(x + row * ldx, i, t, width);
        if (dres != nullptr) rr[i] = M::load(dres + row * ldr, i, t, width);
      }
    }
    // both halves of the row's work take the chunk from the ring: held in registers it would cost the second block of an SM
    auto take = [&](int tensor, int i) {
      if constexpr (VEC) return M::col(i, 0, t) < width ? held(tensor, i) : make_uint4(0, 0, 0, 0);
      else return tensor == 0 ? rg[i] : tensor == 1 ? rx[i] : rr[i];
    };
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      F2 g[H], xh[H];
      pairs(take(0, i), g);
      pairs(take(1, i), xh);
#pragma unroll
      for (int j = 0; j < H; ++j) {                       // where there is no column dy is 0 and nothing is added
        xh[j] = f2_mul(f2_add(xh[j], mean2), r2);
        dwa[i][j] = f2_fma(g[j], xh[j], dwa[i][j]);
        dba[i][j] = f2_add(dba[i][j], g[j]);
        g[j] = f2_mul(g[j], wv[i][j]);
        s1 = f2_add(s1, g[j]);
        s2 = f2_fma(g[j], xh[j], s2);
      }
    }
    if constexpr (VEC) fetch();                           // into the place of the row before
    const float2 sums = row_sum2<TPR>(s1.x + s1.y, s2.x + s2.y, scratch[turn]);
    turn ^= 1;
    const F2 c1 = f2(-sums.x * inv_d, -sums.x * inv_d), c2 = f2(-sums.y * inv_d, -sums.y * inv_d);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      F2 g[H], xh[H], add[H];
      pairs(take(0, i), g);
      pairs(take(1, i), xh);
      if (dres != nullptr) pairs(take(2, i), add);
      float o[N];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        xh[j] = f2_mul(f2_add(xh[j], mean2), r2);
        const F2 inner = f2_add(f2_fma(xh[j], c2, f2_mul(g[j], wv[i][j])), c1);
        const float2 v = (dres != nullptr ? f2_fma(inner, r2, add[j]) : f2_mul(inner, r2));
        o[2 * j] = v.x;
        o[2 * j + 1] = v.y;
      }
      M::store(out, o, i, t, width);
    }
    if constexpr (VEC) get = get == (STAGES - 1) * row_bytes ? 0 : get + row_bytes;
    st = next_st;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (partial == nullptr) return;
  float* mine = partial + static_cast<long long>(blockIdx.x) * 2 * d;
  if constexpr (RPB > 1) {
    for (int who = 0; who < RPB; ++who) {                 // the block's row groups one after another: a fixed order
      __syncthreads();
      if (sub == who) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const int c = M::col(i, j, t);
            const float2 a = dwa[i][j / 2], b = dba[i][j / 2];
            if (c < d) {
              s_fold[c] = (who ? s_fold[c] : 0.f) + (j % 2 ? a.y : a.x);
              s_fold[d + c] = (who ? s_fold[d + c] : 0.f) + (j % 2 ? b.y : b.x);
            }
          }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * d; c += THREADS) mine[c] = s_fold[c];
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = M::col(i, j, t);
        const float2 a = dwa[i][j / 2], b = dba[i][j / 2];
        if (c < d) {
          mine[c] = j % 2 ? a.y : a.x;
          mine[d + c] = j % 2 ? b.y : b.x;
        }
      }
  }
}

// Rows of more than 1024 chunks: a cluster of blocks shares each, `width` columns (at most 512 chunks) for a block, and
// exchanges the two sums. The blocks do not wait for one another: between a row's exchange and its result each takes the
// sums of the next row, so three rows are in the ring, one of them on its way. bf16, no dres, with the column sums: 3024 x
// 12088 in 73 us (launched while the previous kernel still ran half as long again; one block per row that reads it twice, and
// the columns once more, twice as long), 4096 x 16384 in 110. 8192 x 8192, which 512 threads hold, takes 93 there and a sixth
// more on clusters of two.
// A block's sums lie in one of three slots of each peer. A peer writes a slot again three rows later, and by then the reads of
// the slot are ordered before it: they stand before the __syncthreads of the next row's own sums, and so before the fence and
// the arrival that warp 0 makes behind that. With two slots only a relaxed arrival of the reading warps stood in between.
constexpr int CLUSTER_STAGES = 3, CLUSTER_SLOTS = 3;
template <typename T, typename WT, bool VEC>
__global__ void __launch_bounds__(256, 2)
layernorm_bwd_cluster_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ x, long long ldx, const WT* __restrict__ w,
                             const float2* __restrict__ stats, const T* __restrict__ dres, long long ldr, T* __restrict__ dx,
                             float* __restrict__ partial, long long rows, const int whole, float inv_d, const int split, const int width) {
  using M = RowMap<T, 256, VEC>;
  constexpr int N = M::N, H = N / 2, VPL = 2;
  __shared__ float2 scratch[2][8], s_peers[CLUSTER_SLOTS][8];
  extern __shared__ uint4 s_ring[];                       // [stage][dy, x, dres][chunk][thread]
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x, rank = static_cast<int>(cluster_ctarank()), group = blockIdx.x / split, step = gridDim.x / split;
  const int n_rows = static_cast<int>(rows), from_col = rank * width, d = max(0, min(width, whole - from_col));
  const int tensors = dres != nullptr ? 3 : 2;
  F2 wv[VPL][H], dwa[VPL][H], dba[VPL][H];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float f[N];
    M::weights(w != nullptr ? w + from_col : w, f, i, t, d, 1.f);
#pragma unroll
    for (int j = 0; j < H; ++j) { wv[i][j] = f2(f[2 * j], f[2 * j + 1]); dwa[i][j] = dba[i][j] = f2(0.f, 0.f); }
  }
  // Everything a row needs moves on by one step: pointers and bytes from the ring's start.
  const int row_bytes = tensors * VPL * 256 * 16;
  const char* ring = reinterpret_cast<const char*>(s_ring + t);
  const uint32_t ring_at = smem_at(ring);
  const long long step_dy = step * ldy, step_x = step * ldx, step_res = step * ldr, step_out = static_cast<long long>(step) * whole;
  const int own = from_col + (VEC ? M::col(0, 0, t) : 0);
  const T *next_dy = dy + group * ldy + own, *next_x = x + group * ldx + own, *next_res = dres + group * ldr + own;
  T* out = dx + static_cast<long long>(group) * whole + from_col;
  int next_row = group, put = 0;
  auto copy = [&](const T* from, int tensor) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (M::col(i, 0, t) < d)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring_at + put + (tensor * VPL + i) * 256 * 16),
                     "l"(from + i * 256 * N) : "memory");
  };
  auto fetch = [&]() {                                    // one group for each row, an empty one behind the last
    if (next_row < n_rows) {
      copy(next_dy, 0);
      copy(next_x, 1);
      if (dres != nullptr) copy(next_res, 2);
      next_dy += step_dy;
      next_x += step_x;
      next_res += step_res;
      next_row += step;
    }
    put = put == (CLUSTER_STAGES - 1) * row_bytes ? 0 : put + row_bytes;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto take = [&](int row, int at, int tensor, int i, F2 (&v)[H]) {
    uint4 u;
    if constexpr (VEC) {
      u = M::col(i, 0, t) < d ? *reinterpret_cast<const uint4*>(ring + at + (tensor * VPL + i) * 256 * 16) : make_uint4(0, 0, 0, 0);
    } else {
      u = M::load((tensor == 0 ? dy + row * ldy : tensor == 1 ? x + row * ldx : dres + row * ldr) + from_col, i, t, d);
    }
    float f[N];
    Vec16<T>::unpack(u, f);
#pragma unroll
    for (int j = 0; j < H; ++j) v[j] = f2(f[2 * j], f[2 * j + 1]);
  };
  if constexpr (VEC) {
#pragma unroll
    for (int n = 0; n < CLUSTER_STAGES; ++n) fetch();
  }
  cluster_sync_all();                                     // every block of the row runs before one writes to another
  int turn = 0, here = 0, before = 0;                     // bytes of this row's and the last one's place in the ring
  int slot = 0, slot_before = 0;                          // of this row's and the last one's sums
  float2 st = stats[min(group, n_rows - 1)], st_before = st;
  // one step beyond the last row, for its result
  for (int row = group; row < n_rows + step; row += step) {
    const bool more = row < n_rows, had = row != group;   // the same in all blocks of the cluster
    float2 sums = make_float2(0.f, 0.f), next_st = st;
    if (more) {
      next_st = stats[min(row + step, n_rows - 1)];
      const F2 mean2 = f2(-st.x, -st.x), r2 = f2(st.y, st.y);
      if constexpr (VEC) asm volatile("cp.async.wait_group 1;" ::: "memory");
      F2 s1 = f2(0.f, 0.f), s2 = s1;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        F2 g[H], xh[H];
        take(row, here, 0, i, g);
        take(row, here, 1, i, xh);
#pragma unroll
        for (int j = 0; j < H; ++j) {                     // where there is no column dy is 0 and nothing is added
          xh[j] = f2_mul(f2_add(xh[j], mean2), r2);
          dwa[i][j] = f2_fma(g[j], xh[j], dwa[i][j]);
          dba[i][j] = f2_add(dba[i][j], g[j]);
          g[j] = f2_mul(g[j], wv[i][j]);
          s1 = f2_add(s1, g[j]);
          s2 = f2_fma(g[j], xh[j], s2);
        }
      }
      sums = row_sum2<256>(s1.x + s1.y, s2.x + s2.y, scratch[turn]);
    }
    float2 whole_sums = make_float2(0.f, 0.f);
    if (had) {
      cluster_wait();
      for (int i = 0; i < split; ++i) {
        const float2 o = s_peers[slot_before][i];
        whole_sums.x += o.x;
        whole_sums.y += o.y;
      }
    }
    if (more) {
      if (t < split) {
        const uint32_t to = mapa_shared(smem_at(&s_peers[slot][rank]), t);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(sums.x) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(sums.y) : "memory");
      }
      cluster_arrive_after(t < 32);                       // waited for in the next step
    }
    if (had) {
      const int done = row - step;
      const F2 mean2 = f2(-st_before.x, -st_before.x), r2 = f2(st_before.y, st_before.y);
      const F2 c1 = f2(-whole_sums.x * inv_d, -whole_sums.x * inv_d), c2 = f2(-whole_sums.y * inv_d, -whole_sums.y * inv_d);
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        F2 g[H], xh[H], add[H];
        take(done, before, 0, i, g);
        take(done, before, 1, i, xh);
        if (dres != nullptr) take(done, before, 2, i, add);
        float o[N];
#pragma unroll
        for (int j = 0; j < H; ++j) {
          xh[j] = f2_mul(f2_add(xh[j], mean2), r2);
          const F2 inner = f2_add(f2_fma(xh[j], c2, f2_mul(g[j], wv[i][j])), c1);
          const float2 v = (dres != nullptr ? f2_fma(inner, r2, add[j]) : f2_mul(inner, r2));
          o[2 * j] = v.x;
          o[2 * j + 1] = v.y;
        }
        M::store(out, o, i, t, d);
      }
      out += step_out;
      if constexpr (VEC) fetch();                         // into the place of the row that is done
    }
    before = here;
    here = here == (CLUSTER_STAGES - 1) * row_bytes ? 0 : here + row_bytes;
    turn ^= 1;
    slot_before = slot;
    slot = slot == CLUSTER_SLOTS - 1 ? 0 : slot + 1;
    st_before = st;
    st = next_st;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (partial == nullptr) return;
  float* mine = partial + static_cast<long long>(group) * 2 * whole + from_col;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = M::col(i, j, t);
      const float2 a = dwa[i][j / 2], b = dba[i][j / 2];
      if (c < d) {
        mine[c] = j % 2 ? a.y : a.x;
        mine[whole + c] = j % 2 ? b.y : b.x;
      }
    }
}

// Rows too wide for the accumulators: dx by one block per row, and the weight's gradients by blocks of 256 columns
// that read dy and x once more (they need the rows' statistics only).
template <typename T, typename WT>
__global__ void __launch_bounds__(1024)
layernorm_bwd_wide_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ x, long long ldx,
                          const WT* __restrict__ w, const float2* __restrict__ stats, const T* __restrict__ dres, long long ldr,
                          T* __restrict__ dx, int d, float inv_d) {
  __shared__ float2 scratch[32];
  const long long row = blockIdx.x;
  const float2 st = stats[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < d; c += 1024) {
    const float g = to_f32(dy[row * ldy + c]) * (w != nullptr ? to_f32(w[c]) : 1.f);
    s1 += g;
    s2 += g * ((to_f32(x[row * ldx + c]) - st.x) * st.y);
  }
  const float2 sums = row_sum2<1024>(s1, s2, scratch);
  const float c1 = sums.x * inv_d, c2 = sums.y * inv_d;
  for (int c = threadIdx.x; c < d; c += 1024) {
    const float g = to_f32(dy[row * ldy + c]) * (w != nullptr ? to_f32(w[c]) : 1.f);
    float o = st.y * (g - c1 - (to_f32(x[row * ldx + c]) - st.x) * st.y * c2);
    if (dres != nullptr) o += to_f32(dres[row * ldr + c]);
    dx[row * d + c] = from_f32<T>(o);
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
layernorm_bwd_cols_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ x, long long ldx,
                          const float2* __restrict__ stats, float* __restrict__ partial, long long rows, int d) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= d) return;
  float a = 0.f, b = 0.f;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float2 st = stats[row];
    const float g = to_f32(dy[row * ldy + c]);
    a += g * ((to_f32(x[row * ldx + c]) - st.x) * st.y);
    b += g;
  }
  float* mine = partial + static_cast<long long>(blockIdx.y) * 2 * d;
  mine[c] = a;
  mine[d + c] = b;
}

// Sums of the columns of partial [n, 2d] in a fixed order: 32 columns (a line of 128 bytes) x GROUPS groups of rows per block.
template <typename WT, int GROUPS>
__global__ void __launch_bounds__(32 * GROUPS)
layernorm_cols_kernel(const float* __restrict__ partial, WT* __restrict__ dw, WT* __restrict__ db, int n, int d) {
  __shared__ float red[GROUPS][33];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * d) {
#pragma unroll 8
    for (int r = group; r < n; r += GROUPS) s += partial[static_cast<long long>(r) * 2 * d + c];
  }
  red[group][lane] = s;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 32 / GROUPS; ++k) {                 // a warp adds 32 / GROUPS columns
    const int col = group + k * GROUPS;
    const float sum = lanes_sum<32>(lane < GROUPS ? red[lane][col] : 0.f);
    const int out = blockIdx.x * 32 + col;
    if (lane == 0 && out < 2 * d) {
      WT* to = out < d ? dw : db;
      if (to != nullptr) to[out < d ? out : out - d] = from_f32<WT>(sum);
    }
  }
}

// ------------------------------------------------------------------ launches
constexpr int FWD_CHUNKS = 4096;     // most chunks of a row that the forward kernel holds in registers (1024 threads x 4)
constexpr int BWD_CHUNKS = 1024;     // and the backward kernel (512 x 2), beyond that clusters of
constexpr int BWD_SPLIT = 8;         // at most so many blocks of 256 x 2
inline int bwd_split(int chunks) { return (chunks + 511) / 512; }

template <typename T, typename WT, bool VEC, bool ADD>
cudaError_t fwd_launch(const T* x, long long ldx, const T* delta, long long ldd, const WT* w, const WT* b, T* xsum, T* y,
                       float2* stats, long long rows, int d, float eps, cudaStream_t stream) {
  const int chunks = (d + Vec16<T>::N - 1) / Vec16<T>::N;
  const float inv_d = 1.f / static_cast<float>(d);
#define FMB_LN_FWD(TPR, VPL)                                                                                            \
  do {                                                                                                                  \
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;                                                                      \
    return launch_pdl(layernorm_fwd_kernel<T, WT, TPR, VPL, VEC, ADD>, dim3(static_cast<unsigned>((rows + RPB - 1) / RPB)), \
                      dim3(TPR > 256 ? TPR : 256), 0, stream, x, ldx, delta, ldd, w, b, xsum, y, stats, rows, d, inv_d, eps); \
  } while (0)
  if (chunks <= 32) FMB_LN_FWD(32, 1);
  if (chunks <= 64) FMB_LN_FWD(32, 2);
  if (chunks <= 128) FMB_LN_FWD(32, 4);
  if (chunks <= 256) FMB_LN_FWD(128, 2);
  if (chunks <= 512) FMB_LN_FWD(256, 2);
  if (chunks <= 1024) FMB_LN_FWD(256, 4);
  if (chunks <= 2048) FMB_LN_FWD(512, 4);
  if (chunks <= FWD_CHUNKS) FMB_LN_FWD(1024, 4);
#undef FMB_LN_FWD
  layernorm_fwd_wide_kernel<T, WT, ADD><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(x, ldx, delta, ldd, w, b, xsum, y,
                                                                                         stats, d, inv_d, eps);
  return cudaGetLastError();
}

template <typename T, typename WT>
int fwd_run(const void* x, long long ldx, const void* delta, long long ldd, const void* w, const void* b, void* xsum, void* y,
            float* stats, long long rows, int d, float eps, cudaStream_t stream) {
  constexpr int N = Vec16<T>::N;
  const bool vec = d % N == 0 && ldx % N == 0 && ldd % N == 0 && aligned16(x) && aligned16(delta) && aligned16(w) &&
                   aligned16(b) && aligned16(y) && aligned16(xsum);
  const T *xp = static_cast<const T*>(x), *dp = static_cast<const T*>(delta);
  const WT *wp = static_cast<const WT*>(w), *bp = static_cast<const WT*>(b);
  T *sp = static_cast<T*>(xsum), *yp = static_cast<T*>(y);
  float2* st = reinterpret_cast<float2*>(stats);
  cudaError_t e;
  if (delta != nullptr)
    e = vec ? fwd_launch<T, WT, true, true>(xp, ldx, dp, ldd, wp, bp, sp, yp, st, rows, d, eps, stream)
            : fwd_launch<T, WT, false, true>(xp, ldx, dp, ldd, wp, bp, sp, yp, st, rows, d, eps, stream);
  else
    e = vec ? fwd_launch<T, WT, true, false>(xp, ldx, dp, ldd, wp, bp, sp, yp, st, rows, d, eps, stream)
            : fwd_launch<T, WT, false, false>(xp, ldx, dp, ldd, wp, bp, sp, yp, st, rows, d, eps, stream);
  return e == cudaSuccess ? 0 : -3;
}

// Opts a kernel in to 100 KB of shared memory (beyond 48 KB with the static part; the call costs a tenth of a microsecond).
inline bool more_shared(const void* kernel) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024) == cudaSuccess;
}

template <typename T, typename WT, bool VEC>
cudaError_t bwd_launch(const T* dy, long long ldy, const T* x, long long ldx, const WT* w, const float2* stats, const T* dres,
                       long long ldr, T* dx, float* partial, long long rows, int d, int nblocks, cudaStream_t stream) {
  const int chunks = (d + Vec16<T>::N - 1) / Vec16<T>::N;
  const float inv_d = 1.f / static_cast<float>(d);
#define FMB_LN_BWD(TPR, VPL)                                                                                             \
  do {                                                                                                                   \
    constexpr int THREADS = TPR > 256 ? TPR : 256;                                                                       \
    const size_t ring = VEC ? sizeof(uint4) * BwdStages<VPL * THREADS>::N * (dres != nullptr ? 3 : 2) * VPL * THREADS : 0;         \
    const size_t fold = TPR < 256 && partial != nullptr ? 2 * d * sizeof(float) : 0;                                     \
    const size_t smem = ring > fold ? ring : fold;                                                                       \
    auto kernel = layernorm_bwd_kernel<T, WT, TPR, VPL, VEC>;                                                            \
    if (smem > 46 * 1024 && !more_shared(reinterpret_cast<const void*>(kernel))) return cudaErrorInvalidValue;           \
    return launch_pdl(kernel, dim3(nblocks), dim3(THREADS), smem, stream, dy, ldy, x, ldx, w, stats, dres, ldr, dx,      \
                      partial, rows, d, inv_d);                                                                          \
  } while (0)
  if (chunks <= 32) FMB_LN_BWD(32, 1);
  if (chunks <= 64) FMB_LN_BWD(64, 1);
  if (chunks <= 128) FMB_LN_BWD(64, 2);
  if (chunks <= 256) FMB_LN_BWD(128, 2);
  if (chunks <= 512) FMB_LN_BWD(256, 2);
  if (chunks <= BWD_CHUNKS) FMB_LN_BWD(512, 2);
#undef FMB_LN_BWD
  if (chunks <= BWD_CHUNKS * BWD_SPLIT / 2) {
    constexpr int N = Vec16<T>::N;
    const int split = bwd_split(chunks), width = (chunks + split - 1) / split * N;
    const size_t smem = VEC ? sizeof(uint4) * CLUSTER_STAGES * (dres != nullptr ? 3 : 2) * 512 : 0;
    auto kernel = layernorm_bwd_cluster_kernel<T, WT, VEC>;
    if (smem > 46 * 1024 && !more_shared(reinterpret_cast<const void*>(kernel))) return cudaErrorInvalidValue;
    return launch_cluster(kernel, dim3(nblocks * split), dim3(256), smem, split, stream, dy, ldy, x, ldx, w, stats, dres, ldr, dx, partial,
                           rows, d, inv_d, split, width);
  }
  layernorm_bwd_wide_kernel<T, WT><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(dy, ldy, x, ldx, w, stats, dres, ldr, dx,
                                                                                    d, inv_d);
  if (partial != nullptr)
    layernorm_bwd_cols_kernel<T><<<dim3((d + 255) / 256, nblocks), 256, 0, stream>>>(dy, ldy, x, ldx, stats, partial, rows, d);
  return cudaGetLastError();
}

template <typename T, typename WT>
int bwd_run(const void* dy, long long ldy, const void* x, long long ldx, const void* w, const float* stats, const void* dres,
            long long ldr, void* dx, float* partial, void* dw, void* db, long long rows, int d, int nblocks,
            cudaStream_t stream) {
  constexpr int N = Vec16<T>::N;
  const bool vec = d % N == 0 && ldx % N == 0 && ldy % N == 0 && ldr % N == 0 && aligned16(x) && aligned16(dy) &&
                   aligned16(dres) && aligned16(w) && aligned16(dx);
  const float2* st = reinterpret_cast<const float2*>(stats);
  const T *gp = static_cast<const T*>(dy), *xp = static_cast<const T*>(x), *rp = static_cast<const T*>(dres);
  const WT* wp = static_cast<const WT*>(w);
  T* op = static_cast<T*>(dx);
  cudaError_t e = vec ? bwd_launch<T, WT, true>(gp, ldy, xp, ldx, wp, st, rp, ldr, op, partial, rows, d, nblocks, stream)
                      : bwd_launch<T, WT, false>(gp, ldy, xp, ldx, wp, st, rp, ldr, op, partial, rows, d, nblocks, stream);
  if (e == cudaSuccess && partial != nullptr)
    e = nblocks > 96 ? launch_pdl(layernorm_cols_kernel<WT, 32>, dim3((2 * d + 31) / 32), dim3(1024), 0, stream, partial,
                                  static_cast<WT*>(dw), static_cast<WT*>(db), nblocks, d)
                     : launch_pdl(layernorm_cols_kernel<WT, 8>, dim3((2 * d + 31) / 32), dim3(256), 0, stream, partial,
                                  static_cast<WT*>(dw), static_cast<WT*>(db), nblocks, d);
  return e == cudaSuccess ? 0 : -3;
}

}  // namespace fmb

using namespace fmb;

extern "C" int fmb_layernorm_fwd(const void* x, long long ldx, const void* delta, long long ldd, const void* w, const void* b,
                                 void* xsum, void* y, float* stats, long long rows, int d, float eps, int dtype, int w_dtype,
                                 cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (d <= 0 || rows > 0x7fffffffLL) return -2;
  if (dtype == FMB_BF16 && w_dtype == FMB_BF16)
    return fwd_run<__nv_bfloat16, __nv_bfloat16>(x, ldx, delta, ldd, w, b, xsum, y, stats, rows, d, eps, stream);
  if (dtype == FMB_BF16 && w_dtype == FMB_F32)
    return fwd_run<__nv_bfloat16, float>(x, ldx, delta, ldd, w, b, xsum, y, stats, rows, d, eps, stream);
  if (dtype == FMB_F32 && w_dtype == FMB_F32)
    return fwd_run<float, float>(x, ldx, delta, ldd, w, b, xsum, y, stats, rows, d, eps, stream);
  return -1;
}

// Clusters of `split` blocks that the device holds together (SMs come in groups that need not be whole clusters; a second
// wave of a walk over the rows would double its time). Asked once per device and size.
static int cluster_fit(int split) {
  static int known[64][BWD_SPLIT + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 16;
  if (known[dev][split] == 0) {
    auto kernel = layernorm_bwd_cluster_kernel<__nv_bfloat16, float, true>;
    const size_t smem = sizeof(uint4) * CLUSTER_STAGES * 3 * 512;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sm_count() / split * split);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (!more_shared(reinterpret_cast<const void*>(kernel)) || cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 16;
    }
    known[dev][split] = n;
  }
  return known[dev][split];
}

extern "C" int fmb_layernorm_bwd_blocks(long long rows, int d, int dtype) {
  const int n = dtype == FMB_BF16 ? 8 : 4;
  const int chunks = (d + n - 1) / n;
  if (chunks > BWD_CHUNKS * BWD_SPLIT / 2) return static_cast<int>(rows < 32 ? (rows < 1 ? 1 : rows) : 32);
  if (chunks > BWD_CHUNKS) {
    const long long most = cluster_fit(bwd_split(chunks));
    return static_cast<int>(rows < 1 ? 1 : rows < most ? rows : most);
  }
  const int per_row = chunks <= 32 ? 32 : chunks <= 128 ? 64 : chunks <= 256 ? 128 : 256;
  const long long need = (rows + 256 / per_row - 1) / (256 / per_row);
  const long long most = static_cast<long long>(sm_count()) * (chunks <= 64 ? 4 : chunks <= 512 ? 2 : 1);      // as many as are resident
  return static_cast<int>(need < 1 ? 1 : need < most ? need : most);
}

extern "C" int fmb_layernorm_bwd(const void* dy, long long ldy, const void* x, long long ldx, const void* w, const float* stats,
                                 const void* dres, long long ldr, void* dx, float* partial, void* dw, void* db, long long rows,
                                 int d, int dtype, int w_dtype, int nblocks, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (d <= 0 || rows > 0x7fff0000LL || nblocks < 1) return -2;      // steps over the rows stay within 31 bits
  if (dtype == FMB_BF16 && w_dtype == FMB_BF16)
    return bwd_run<__nv_bfloat16, __nv_bfloat16>(dy, ldy, x, ldx, w, stats, dres, ldr, dx, partial, dw, db, rows, d, nblocks, stream);
  if (dtype == FMB_BF16 && w_dtype == FMB_F32)
    return bwd_run<__nv_bfloat16, float>(dy, ldy, x, ldx, w, stats, dres, ldr, dx, partial, dw, db, rows, d, nblocks, stream);
  if (dtype == FMB_F32 && w_dtype == FMB_F32)
    return bwd_run<float, float>(dy, ldy, x, ldx, w, stats, dres, ldr, dx, partial, dw, db, rows, d, nblocks, stream);
  return -1;
}

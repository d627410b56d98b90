// LayerNorm of the rows of a float32, bfloat16 or float16 matrix of any width
// (the row norms of block_ops.cu and jk_norm.cu are float32 and at most 1024
// and 2048 wide).  With d columns, weight w and bias b:
//   mean = <x>,  var = <(x - mean)^2>,  rstd = (var + eps)^-1/2
//   xh = (x - mean) rstd,  y = xh w + b
// and with the upstream gradient g, u = g w:
//   grad_x = rstd (u - <u> - xh <u xh>)
//   grad_w = sum_rows g xh,  grad_b = sum_rows g
// Statistics, products and sums are float32 whatever the element type; y and
// the gradients are rounded once.
//
// The variance is formed from differences.  The mean m is a float32 number, which
// for a row of level l leaves l 2^-24 rstd and more in xh: nothing beside the other
// roundings where l is of the spread's size, but all digits of a row whose level is
// far above its spread.  Such a row (far_level) takes one more sum, delta = <e> with
// e = x - m, which is exact where x is near m:
//   var = <e^2> - delta^2,  xh = (e - delta) rstd
// The backward forms delta again from the m that it is given.  A row that is not far
// pays a comparison; the sum for every row took 3 to 6% more time (24492 x 2560
// float32: 83 + 121 us, 81 + 115 without; 103 + 138 where every row is far).
//
// Both passes are bound by memory: a row is read once into registers, the
// statistics are formed there, and the result is written.  A thread holds the same
// columns of every row that it meets, so weight, bias and the two sums of the
// backward stay in registers over all rows of a persistent block, which writes
// one partial sum of the parameter gradients at its end; a second kernel adds
// the partial sums in block order.  x and g are thus read once for all three
// gradients, and nothing is added atomically.
#include <atomic>

#include "class_rows.cuh"

namespace cign {
namespace {

constexpr int kLnGroupThreads = 256;  // block of the kernels with several rows per block
constexpr int kLnBlockThreads = 512;  // of a block that holds one row; the widest rows take twice that
constexpr int kLnMaxBlocks = 1776;    // partial sums of the parameter gradients (148 SMs x 12)
// Wider rows leave the parameter gradients to a kernel of their own.
constexpr int64_t kLnBlockColumns = 16 * kLnBlockThreads;
constexpr int kLnWideThreads = 256;
constexpr int kLnWideWarps = kLnWideThreads / 32;
constexpr int64_t kLnMaxColumns = 65535ll * kLnWideThreads;  // the grid's second dimension

// How a row lies in a block.  LANES lanes hold it, load i of lane l covering
// columns (l + LANES i) V ...; LANES == 0: the block's threads, known at launch.
// BLOCK != 0: the block holds one row (of at most BLOCK * kLnBlockThreads
// threads); else a group of LANES <= 32 lanes does, and the block
// kLnGroupThreads / LANES rows.  With LANES known, the addresses of a lane's
// loads differ by constants, which halves the instructions of the kernels that
// load single elements.
template <int LANES, int BLOCK>
struct LnLanes {
  __device__ __forceinline__ static int count() { return LANES ? LANES : blockDim.x; }
  __device__ __forceinline__ static int lane() {
    return BLOCK ? threadIdx.x : threadIdx.x & (LANES - 1);
  }
  __device__ __forceinline__ static int group() { return BLOCK ? 0 : threadIdx.x / (LANES | !LANES); }
  static constexpr int kRows = BLOCK ? 1 : kLnGroupThreads / (LANES | !LANES);
};

// Sums over the lanes of a row.  `slot` alternates between two sets of partial
// sums in shared memory, so that one barrier per sum is enough: a set is
// written again only after the barrier of the next sum.
template <int LANES, int BLOCK>
__device__ __forceinline__ float row_sum(float v, float* part, int& slot) {
  if constexpr (BLOCK == 0) {
    return group_sum<LANES>(v);
  } else {
    v = warp_sum(v);
    float* p = part + slot * 32;
    slot ^= 1;
    if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll (LANES ? 8 : 1)
    for (int w = 0; w < LnLanes<LANES, BLOCK>::count() / 32; w += 4) {  // the rest of p is 0
      const float4 q = *reinterpret_cast<const float4*>(p + w);
      s += (q.x + q.y) + (q.z + q.w);
    }
    return s;
  }
}
// Two sums at once, one barrier.
template <int LANES, int BLOCK>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2* part, int& slot) {
  if constexpr (BLOCK == 0) {
    a = group_sum<LANES>(a);
    b = group_sum<LANES>(b);
  } else {
    a = warp_sum(a);
    b = warp_sum(b);
    float2* p = part + slot * 32;
    slot ^= 1;
    if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll (LANES ? 16 : 1)
    for (int w = 0; w < LnLanes<LANES, BLOCK>::count() / 32; w += 2) {
      const float4 q = *reinterpret_cast<const float4*>(p + w);
      a += q.x + q.z;
      b += q.y + q.w;
    }
  }
}

// This lane's loads of the row at r (the lane's first).  `loads`: how many of
// them lie in the row; all but the last SLACK do.  No load depends on a
// branch, so all are in flight together, and the callers ask for a row while
// they work on the one before.
template <typename T, int V, int NV, int SLACK>
__device__ __forceinline__ void load_row(Pack<T, V> (&q)[NV], const T* r, int loads, int lanes) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    q[i] = load_pack<T, V>(r + (i < NV - SLACK ? i : (i < loads ? i : loads - 1)) * lanes * V);
}

// Whether the level of a row is above twice its spread; below, the mean's
// roundings leave no more than twice their relative size in xh.
__device__ __forceinline__ bool far_level(float mu, float rs) { return fabsf(mu * rs) > 2.0f; }
// The same for any row of a warp, whose rows' sums are formed together.
template <int BLOCK>
__device__ __forceinline__ bool any_far(bool far) {
  return BLOCK != 0 ? far : __any_sync(kFullMask, far);
}
// delta of a row, 0 if it is not far: from the lanes' e where a warp holds rows, and
// from the row at xr, read again, where a block does, whose kernels would need more
// registers for every row otherwise.
template <typename T, int V, int NV, int SLACK, int LANES, int BLOCK>
__device__ __forceinline__ float row_delta(const float (&e)[NV][V], int own, const T* xr, int d,
                                           float mu, bool far, float* part, int& slot) {
  float s = 0.0f;
  if constexpr (BLOCK == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += i < NV - SLACK || i < own ? e[i][j] : 0.0f;
  } else {
#pragma unroll 1
    for (int i = LnLanes<LANES, BLOCK>::lane(); i < d / V; i += LnLanes<LANES, BLOCK>::count()) {
      const Pack<T, V> q = load_pack<T, V>(xr + i * V);
#pragma unroll
      for (int j = 0; j < V; ++j) s += to_f(q.e[j]) - mu;
    }
  }
  s = row_sum<LANES, BLOCK>(s, part, slot) * (1.0f / static_cast<float>(d));
  return far ? s : 0.0f;
}
// The variance from <e^2> and delta, not below 0 (NaN stays).
__device__ __forceinline__ float variance(float sq, float delta) {
  const float v = fmaf(-delta, delta, sq);
  return v < 0.0f ? 0.0f : v;
}

// y, and m and rstd for the backward.  24492 x 2560 float32: 81 us, 6.2 TB/s,
// bound by memory.  131072 x 1024 bf16: 97 us, 5.5 TB/s, and 200003 x 301 fp16,
// whose rows start anywhere and are read by elements: 69 us, 3.5 TB/s; both
// bound by the instructions they issue and by the latency that the resident
// warps leave open.  (16-byte loads shifted into place were slower than the
// loads of elements.)
// At most 80 registers: left alone, the compiler gives the 16-element bf16 row
// 98 and fewer blocks are resident (131072 x 1024: 110 us, 96 us with 80; 64
// spill, 111 us).  72 for a block's rows of 12 elements per thread, which take no
// more but for the far rows (40000 x 1301 float32: 73 us, 77 with 80).
template <typename T, int V, int NV, int SLACK, int LANES, int BLOCK>
__global__ void __maxnreg__(BLOCK == 2 ? 64 : V == 1 && NV == 12 && BLOCK == 1 ? 72 : 80)
layer_norm_fwd_kernel(int64_t n, int d, const T* __restrict__ x, int64_t ldx,
                      const void* __restrict__ w, const void* __restrict__ b, int32_t param_type,
                      float eps, T* __restrict__ y, float* __restrict__ mean,
                      float* __restrict__ rstd) {
  using L = LnLanes<LANES, BLOCK>;
  __shared__ __align__(16) float part[64];
  if (BLOCK != 0 && threadIdx.x < 32) part[threadIdx.x] = part[32 + threadIdx.x] = 0.0f;
  if (BLOCK != 0) __syncthreads();
  int slot = 0;
  const int lane = L::lane(), lanes = L::count();
  const int nvec = d / V;
  // a lane of a row narrower than the lanes has no load of its own; it repeats the last one
  const int own = nvec > lane ? (nvec - lane + lanes - 1) / lanes : 0;
  const int at_lane = own > 0 ? lane : nvec - 1, loads = own > 0 ? own : 1;
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int f = (lane + lanes * i) * V + e;
      wv[i][e] = i < own ? load_param(w, param_type, f, 1.0f) : 0.0f;
      bv[i][e] = i < own ? load_param(b, param_type, f, 0.0f) : 0.0f;
    }
  const float inv_d = 1.0f / static_cast<float>(d);
  const int64_t step = static_cast<int64_t>(gridDim.x) * L::kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * L::kRows + L::group();
  const T* xp = x + (row < n ? row : n - 1) * ldx + at_lane * V;
  T* yp = y + row * d + lane * V;
  Pack<T, V> next[NV];
  load_row<T, V, NV, SLACK>(next, xp, loads, lanes);
  // every group of a block goes on until the last of them is done, as all lanes take part in the sums
  for (; row - L::group() < n; row += step, yp += step * d) {
    const bool live = BLOCK != 0 || row < n;
    float xv[NV][V];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float a = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xv[i][e] = to_f(next[i].e[e]);
        a += xv[i][e];
      }
      s += i < NV - SLACK || i < own ? a : 0.0f;
    }
    if (row + step < n) xp += step * ldx;
    load_row<T, V, NV, SLACK>(next, xp, loads, lanes);
    float mu = row_sum<LANES, BLOCK>(s, part, slot) * inv_d;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float a = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xv[i][e] -= mu;
        a = fmaf(xv[i][e], xv[i][e], a);
      }
      v += i < NV - SLACK || i < own ? a : 0.0f;
    }
    v = row_sum<LANES, BLOCK>(v, part, slot) * inv_d;
    float rs = rsqrtf(v + eps), shift = 0.0f;
    if (any_far<BLOCK>(far_level(mu, rs))) {
      const float delta = row_delta<T, V, NV, SLACK, LANES, BLOCK>(
          xv, own, x + row * ldx, d, mu, far_level(mu, rs), part, slot);
      rs = rsqrtf(variance(v, delta) + eps);
      shift = -delta * rs;
      mu += delta;
    }
    if (live && lane == 0 && mean != nullptr) {
      mean[row] = mu;
      rstd[row] = rs;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pack<T, V> q;
#pragma unroll
      for (int e = 0; e < V; ++e)
        q.e[e] = from_f<T>(fmaf(fmaf(xv[i][e], rs, shift), wv[i][e], bv[i][e]));
      if (live && (i < NV - SLACK || i < own)) store_pack<T, V>(yp + i * lanes * V, q);
    }
  }
}

// grad x; partial: [gridDim.x, 2, d] sums of g xh and g over the block's rows, or
// NULL; deltas (BLOCK 2): those of the rows, or NULL.  The weights and both sums of
// a thread's columns are in registers, so that x and g are read once for all three
// gradients: 24492 x 2560 float32 115 us, 6.5 TB/s, bound by memory; 131072 x 1024
// bf16 148 us, 5.4 TB/s, bound by latency (24% of the warps are resident at 121
// registers a thread).
// Rows that take more than kLnBlockThreads threads (BLOCK 2) leave these to a
// kernel of their own: with them a thread would need more than the 64 registers
// that a block of 1024 has (5093 x 10080 fp16: 92 us, and 52 for the other; bound by
// the latency of a row's loads and two barriers with one block to an SM).
template <typename T, int V, int NV, int SLACK, int LANES, int BLOCK>
__global__ void __launch_bounds__(BLOCK ? BLOCK * kLnBlockThreads : kLnGroupThreads)
layer_norm_bwd_kernel(int64_t n, int d, const T* __restrict__ gy, int64_t ldg,
                      const T* __restrict__ x, int64_t ldx, const void* __restrict__ w,
                      int32_t param_type, const float* __restrict__ mean,
                      const float* __restrict__ rstd, T* __restrict__ gx,
                      float* __restrict__ partial, float* __restrict__ deltas) {
  using L = LnLanes<LANES, BLOCK>;
  __shared__ __align__(16) float2 part[64];
  // row_delta's: between two uses of one set lies a barrier of its own or row_sum2's
  __shared__ __align__(16) float part1[64];
  if (BLOCK != 0 && threadIdx.x < 32) {
    part[threadIdx.x] = part[32 + threadIdx.x] = make_float2(0.0f, 0.0f);
    part1[threadIdx.x] = part1[32 + threadIdx.x] = 0.0f;
  }
  if (BLOCK != 0) __syncthreads();
  extern __shared__ float columns[];  // BLOCK == 0: [rows of the block, LANES * NV * V]
  int slot = 0;
  const int lane = L::lane(), lanes = L::count();
  const int nvec = d / V;
  const int own = nvec > lane ? (nvec - lane + lanes - 1) / lanes : 0;
  const int at_lane = own > 0 ? lane : nvec - 1, loads = own > 0 ? own : 1;
  float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      wv[i][e] = i < own ? load_param(w, param_type, (lane + lanes * i) * V + e, 1.0f) : 0.0f;
      aw[i][e] = ab[i][e] = 0.0f;
    }
  const float inv_d = 1.0f / static_cast<float>(d);
  const int64_t step = static_cast<int64_t>(gridDim.x) * L::kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * L::kRows + L::group();
  int64_t loaded = row < n ? row : n - 1;
  const T* xp = x + loaded * ldx + at_lane * V;
  const T* gp = gy + loaded * ldg + at_lane * V;
  T* op = gx + row * d + lane * V;
  // (the widest rows have no registers for the next one)
  constexpr bool kAhead = BLOCK != 2;
  Pack<T, V> xn[NV], gn[NV];
  float mu_next = 0.0f, rs_next = 0.0f;
  const auto ask = [&]() {
    load_row<T, V, NV, SLACK>(xn, xp, loads, lanes);
    load_row<T, V, NV, SLACK>(gn, gp, loads, lanes);
    mu_next = mean[loaded];
    rs_next = rstd[loaded];
  };
  if (kAhead) ask();
  for (; row - L::group() < n; row += step, op += step * d) {
    const bool live = BLOCK != 0 || row < n;
    if (!kAhead) ask();
    const float mu = mu_next, rs = rs_next;
    // with e = x - m - delta and h = g rstd: u = g w, u xh = rstd u e, g xh = h e and
    // grad_x = h w - rstd <u> - e rstd^3 <u e>.  Loads behind the last repeat it:
    // they have w = 0 and their sums are dropped.
    float ev[NV][V], hv[NV][V];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) ev[i][e] = to_f(xn[i].e[e]) - mu;
    float delta = 0.0f;
    if (any_far<BLOCK>(far_level(mu, rs))) {
      delta = row_delta<T, V, NV, SLACK, LANES, BLOCK>(ev, own, x + row * ldx, d, mu,
                                                       far_level(mu, rs), part1, slot);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) ev[i][e] -= delta;
    }
    if (BLOCK == 2 && lane == 0 && deltas != nullptr) deltas[row] = delta;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = to_f(gn[i].e[e]);
        hv[i][e] = g * rs;
        const float u = g * wv[i][e];
        s1 += u;
        s2 = fmaf(u, ev[i][e], s2);
        if (BLOCK != 2 && live) {
          aw[i][e] = fmaf(hv[i][e], ev[i][e], aw[i][e]);
          ab[i][e] += g;
        }
      }
    if (row + step < n) {
      xp += step * ldx;
      gp += step * ldg;
      loaded = row + step;
    }
    if (kAhead) ask();
    if (gx != nullptr) {
      row_sum2<LANES, BLOCK>(s1, s2, part, slot);
      s1 *= -rs * inv_d;
      s2 = (s2 * rs * inv_d) * (-rs * rs);  // rstd^3 may be out of float32's range
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Pack<T, V> q;
#pragma unroll
        for (int e = 0; e < V; ++e)
          q.e[e] = from_f<T>(fmaf(ev[i][e], s2, fmaf(hv[i][e], wv[i][e], s1)));
        if (live && (i < NV - SLACK || i < own)) store_pack<T, V>(op + i * lanes * V, q);
      }
    }
  }
  if (BLOCK == 2 || partial == nullptr) return;
  float* pw = partial + static_cast<int64_t>(blockIdx.x) * 2 * d;
  if constexpr (BLOCK != 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int f = (lane + lanes * i) * V + e;
        if (i < own) {
          pw[f] = aw[i][e];
          pw[d + f] = ab[i][e];
        }
      }
  } else {
    // the rows' groups in order
    constexpr int kCols = LANES * NV * V;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e)
          columns[L::group() * kCols + (lane + LANES * i) * V + e] =
              which == 0 ? aw[i][e] : ab[i][e];
      __syncthreads();
      for (int j = threadIdx.x; j < d; j += kLnGroupThreads) {
        float v = 0.0f;
#pragma unroll 8
        for (int k = 0; k < L::kRows; ++k) v += columns[k * kCols + j];
        pw[which * d + j] = v;
      }
    }
  }
}

// out[j] = sum over blocks of partial[block, which, j]: a block of 16 warps
// covers 32 columns, warp w adds its share of the blocks in order, then the
// warps are added in order.  444 partial sums of 2560 columns: 4.4 us, from L2.
constexpr int kLnSumWarps = 16;
template <typename P>
__global__ void __launch_bounds__(kLnSumWarps * 32)
layer_norm_param_sum_kernel(int blocks, int64_t d, const float* __restrict__ partial,
                            P* __restrict__ gw, P* __restrict__ gb) {
  __shared__ float part[kLnSumWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  P* out = blockIdx.y == 0 ? gw : gb;
  if (out == nullptr) return;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int share = (blocks + kLnSumWarps - 1) / kLnSumWarps;
  const int b0 = warp * share, b1 = b0 + share < blocks ? b0 + share : blocks;
  float s = 0.0f;
  if (j < d && b0 < b1) s = ordered_sum<1>(partial + blockIdx.y * d + j, 2 * d, b0, b1);
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && j < d) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < kLnSumWarps; ++k) t += part[k][lane];
    out[j] = from_f<P>(t);
  }
}

// delta of the block's row.
template <typename T>
__device__ __forceinline__ float wide_delta(const T* xr, int64_t d, float mu, float* part) {
  float s = 0.0f;
  for (int64_t j = threadIdx.x; j < d; j += kLnWideThreads) s += to_f(xr[j]) - mu;
  return block_sum<kLnWideWarps>(s, part) * (1.0f / static_cast<float>(d));
}

// Rows that do not fit the registers of one block: a block per row, which
// reads the row again for each of its sums (from L2).  2000 x 40000 float32: 315 us,
// 2.0 TB/s of the bytes that must move, bound by the latency of single loads; the
// backward 354 us, 2.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(kLnWideThreads)
layer_norm_wide_fwd_kernel(int64_t n, int64_t d, const T* __restrict__ x, int64_t ldx,
                           const void* __restrict__ w, const void* __restrict__ b,
                           int32_t param_type, float eps, T* __restrict__ y,
                           float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float part[kLnWideWarps];
  const float inv_d = 1.0f / static_cast<float>(d);
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  float s = 0.0f;
  for (int64_t j = threadIdx.x; j < d; j += kLnWideThreads) s += to_f(xr[j]);
  const float mu = block_sum<kLnWideWarps>(s, part) * inv_d;
  float v = 0.0f;
  for (int64_t j = threadIdx.x; j < d; j += kLnWideThreads) {
    const float a = to_f(xr[j]) - mu;
    v = fmaf(a, a, v);
  }
  v = block_sum<kLnWideWarps>(v, part) * inv_d;
  float rs = rsqrtf(v + eps), delta = 0.0f;
  if (far_level(mu, rs)) {
    delta = wide_delta(xr, d, mu, part);
    rs = rsqrtf(variance(v, delta) + eps);
  }
  if (threadIdx.x == 0 && mean != nullptr) {
    mean[row] = mu + delta;
    rstd[row] = rs;
  }
  const float shift = -delta * rs;
  for (int64_t j = threadIdx.x; j < d; j += kLnWideThreads) {
    const float xh = fmaf(to_f(xr[j]) - mu, rs, shift);
    y[row * d + j] = from_f<T>(fmaf(xh, load_param(w, param_type, j, 1.0f),
                                    load_param(b, param_type, j, 0.0f)));
  }
}

// grad x and the rows' deltas; either may be NULL.
template <typename T>
__global__ void __launch_bounds__(kLnWideThreads)
layer_norm_wide_bwd_kernel(int64_t n, int64_t d, const T* __restrict__ gy, int64_t ldg,
                           const T* __restrict__ x, int64_t ldx, const void* __restrict__ w,
                           int32_t param_type, const float* __restrict__ mean,
                           const float* __restrict__ rstd, T* __restrict__ gx,
                           float* __restrict__ deltas) {
  __shared__ float part[kLnWideWarps];
  const float inv_d = 1.0f / static_cast<float>(d);
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  const T* gr = gy + row * ldg;
  const float mu = mean[row], rs = rstd[row];
  const float delta = far_level(mu, rs) ? wide_delta(xr, d, mu, part) : 0.0f;
  if (threadIdx.x == 0 && deltas != nullptr) deltas[row] = delta;
  if (gx == nullptr) return;
  const float shift = -delta * rs;
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t j = threadIdx.x; j < d; j += kLnWideThreads) {
    const float u = to_f(gr[j]) * load_param(w, param_type, j, 1.0f);
    s1 += u;
    s2 = fmaf(u, fmaf(to_f(xr[j]) - mu, rs, shift), s2);
  }
  s1 = block_sum<kLnWideWarps>(s1, part) * inv_d;
  s2 = block_sum<kLnWideWarps>(s2, part) * inv_d;
  for (int64_t j = threadIdx.x; j < d; j += kLnWideThreads) {
    const float u = to_f(gr[j]) * load_param(w, param_type, j, 1.0f);
    const float xh = fmaf(to_f(xr[j]) - mu, rs, shift);
    gx[row * d + j] = from_f<T>(rs * (u - s1 - xh * s2));
  }
}

// Partial sums of the parameter gradients over a chunk of rows, rows in order;
// a thread has V neighbouring columns.  It reads x and g once more: 5093 x 10080
// fp16 52 us, 4.0 TB/s; 2000 x 40000 float32 107 us, 6.0 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(kLnWideThreads)
layer_norm_wide_param_kernel(int64_t n, int64_t d, int64_t chunk, const T* __restrict__ gy,
                             int64_t ldg, const T* __restrict__ x, int64_t ldx,
                             const float* __restrict__ mean, const float* __restrict__ rstd,
                             const float* __restrict__ deltas, float* __restrict__ partial) {
  const int64_t j = (static_cast<int64_t>(blockIdx.y) * kLnWideThreads + threadIdx.x) * V;
  if (j >= d) return;
  const int64_t r0 = blockIdx.x * chunk;
  const int64_t r1 = r0 + chunk < n ? r0 + chunk : n;
  float aw[V], ab[V];
#pragma unroll
  for (int e = 0; e < V; ++e) aw[e] = ab[e] = 0.0f;
  constexpr int kG = V == 1 ? 8 : 4;  // rows whose loads are in flight together
  for (int64_t rb = r0; rb < r1; rb += kG) {
    Pack<T, V> g[kG], v[kG];
    float mu[kG], rs[kG], delta[kG];
#pragma unroll
    for (int u = 0; u < kG; ++u) {
      const int64_t r = rb + u < r1 ? rb + u : r1 - 1;
      g[u] = load_pack<T, V>(gy + r * ldg + j);
      v[u] = load_pack<T, V>(x + r * ldx + j);
      mu[u] = mean[r];
      rs[u] = rstd[r];
      delta[u] = deltas[r];
    }
#pragma unroll
    for (int u = 0; u < kG; ++u)
      if (rb + u < r1) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float ge = to_f(g[u].e[e]);
          aw[e] = fmaf(ge, (to_f(v[u].e[e]) - mu[u] - delta[u]) * rs[u], aw[e]);
          ab[e] += ge;
        }
      }
  }
  float* pw = partial + static_cast<int64_t>(blockIdx.x) * 2 * d;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    pw[j + e] = aw[e];
    pw[d + j + e] = ab[e];
  }
}

// How a row of nvec loads is spread: over a group of lanes (4 to 32) or the
// threads of a block, and how many loads a thread makes, at most 16 elements.
struct LnShape {
  bool fits = false, block = false;
  int lanes = 0, nv = 0;
};
// Loads of 16 bytes.
LnShape ln_shape(int64_t nvec, int max_nv) {
  LnShape s;
  for (int g = 4; g <= 32; g *= 2)
    if (nvec <= static_cast<int64_t>(g) * max_nv) {
      s.fits = true;
      s.lanes = g;
      s.nv = static_cast<int>((nvec + g - 1) / g);
      return s;
    }
  // the work of a row: its loads, the idle ones among them, and what every
  // thread of the row pays once (its share of the sum and the barrier), which
  // takes about as long as one load's elements
  int64_t best = 0;
  for (int nv = max_nv; nv >= 1; --nv) {
    const int64_t t = ((nvec + nv - 1) / nv + 31) / 32 * 32;
    if (t > (nv == max_nv ? 2 : 1) * kLnBlockThreads) continue;
    const int64_t full = (nvec + t - 1) / t;  // at most nv; t is whole warps
    const int64_t cost = t * (full + 1);
    if (!s.fits || cost < best) {
      best = cost;
      s.fits = s.block = true;
      s.lanes = static_cast<int>(t);
      s.nv = static_cast<int>(full);
    }
  }
  return s;
}
// Loads of one element: the fewest lanes that hold the row.
LnShape ln_shape_elements(int64_t d) {
  LnShape s;
  for (int g = 8; g <= 2 * kLnBlockThreads; g *= 2)
    if (d <= static_cast<int64_t>(g) * (g < 32 ? 4 : 16)) {
      s.fits = true;
      s.block = g > 32;
      s.lanes = g;
      s.nv = static_cast<int>((d + g - 1) / g);
      return s;
    }
  return s;
}

struct LnPlan {
  bool wide;  // loads of 16 bytes: every row of every matrix starts on 16 bytes
  LnShape shape;
  int threads;
  int64_t blocks;  // that the rows need
};

template <typename T>
LnPlan ln_plan(int64_t n, int64_t d, const void* const* ptrs, const int64_t* lds, int count) {
  constexpr int V = 16 / sizeof(T);
  LnPlan p;
  p.wide = d % V == 0;
  for (int i = 0; i < count; ++i)
    if (ptrs[i] != nullptr && (!aligned16(ptrs[i]) || (lds[i] * sizeof(T)) % 16 != 0))
      p.wide = false;
  p.shape = p.wide ? ln_shape(d / V, 16 / V) : ln_shape_elements(d);
  p.threads = p.shape.block ? p.shape.lanes : kLnGroupThreads;
  const int rows = p.shape.block || !p.shape.fits ? 1 : p.threads / p.shape.lanes;
  p.blocks = (n + rows - 1) / rows;
  return p;
}

#define CIGN_LN_CASE(V_, NV_, SLACK_, LANES_, BLOCK_, ...)                               \
  {                                                                                      \
    constexpr int V = V_, NV = NV_, SLACK = SLACK_, LANES = LANES_, BLOCK = BLOCK_;      \
    __VA_ARGS__;                                                                         \
  }
#define CIGN_LN_GROUP(LANES_, ...)                                                       \
  {                                                                                      \
    if (nv_ <= 1) CIGN_LN_CASE(kV, 1, 1, LANES_, 0, __VA_ARGS__)                         \
    else if (nv_ <= 2) CIGN_LN_CASE(kV, 2, 1, LANES_, 0, __VA_ARGS__)                    \
    else if (nv_ <= 3) CIGN_LN_CASE(kV, (kMost < 3 ? kMost : 3), 1, LANES_, 0, __VA_ARGS__) \
    else CIGN_LN_CASE(kV, kMost, 1, LANES_, 0, __VA_ARGS__)                              \
  }
#define CIGN_LN_ELEMENTS(LANES_, BLOCK_, ...)                                            \
  {                                                                                      \
    if (nv_ <= 12) CIGN_LN_CASE(1, 12, 4, LANES_, BLOCK_, __VA_ARGS__)                   \
    else CIGN_LN_CASE(1, 16, 4, LANES_, BLOCK_, __VA_ARGS__)                             \
  }
// CALL with V, NV (loads per thread, rounded up), SLACK (how many of them may
// lie behind the row), LANES and BLOCK bound to the plan's.
#define CIGN_LN_DISPATCH(T, plan, ...)                                                   \
  do {                                                                                   \
    constexpr int kV = 16 / sizeof(T), kMost = 16 / kV;                                  \
    const int nv_ = (plan).shape.nv, lanes_ = (plan).shape.lanes;                        \
    if ((plan).wide && !(plan).shape.block) {                                            \
      if (lanes_ == 4) CIGN_LN_GROUP(4, __VA_ARGS__)                                     \
      else if (lanes_ == 8) CIGN_LN_GROUP(8, __VA_ARGS__)                                \
      else if (lanes_ == 16) CIGN_LN_GROUP(16, __VA_ARGS__)                              \
      else CIGN_LN_GROUP(32, __VA_ARGS__)                                                \
    } else if ((plan).wide) {                                                            \
      if (lanes_ > kLnBlockThreads) CIGN_LN_CASE(kV, kMost, 1, 0, 2, __VA_ARGS__)        \
      else if (nv_ <= 1) CIGN_LN_CASE(kV, 1, 1, 0, 1, __VA_ARGS__)                       \
      else if (nv_ <= 2) CIGN_LN_CASE(kV, 2, 1, 0, 1, __VA_ARGS__)                       \
      else if (nv_ <= 3) CIGN_LN_CASE(kV, (kMost < 3 ? kMost : 3), 1, 0, 1, __VA_ARGS__) \
      else CIGN_LN_CASE(kV, kMost, 1, 0, 1, __VA_ARGS__)                                 \
    } else if (lanes_ <= 8) CIGN_LN_CASE(1, 4, 4, 8, 0, __VA_ARGS__)                     \
    else if (lanes_ <= 16) CIGN_LN_CASE(1, 4, 4, 16, 0, __VA_ARGS__)                     \
    else if (lanes_ <= 32) {                                                             \
      if (nv_ <= 4) CIGN_LN_CASE(1, 4, 4, 32, 0, __VA_ARGS__)                            \
      else if (nv_ <= 6) CIGN_LN_CASE(1, 6, 2, 32, 0, __VA_ARGS__)                       \
      else if (nv_ <= 8) CIGN_LN_CASE(1, 8, 2, 32, 0, __VA_ARGS__)                       \
      else if (nv_ <= 10) CIGN_LN_CASE(1, 10, 2, 32, 0, __VA_ARGS__)                     \
      else CIGN_LN_ELEMENTS(32, 0, __VA_ARGS__)                                          \
    }                                                                                    \
    else if (lanes_ <= 64) CIGN_LN_ELEMENTS(64, 1, __VA_ARGS__)                          \
    else if (lanes_ <= 128) CIGN_LN_ELEMENTS(128, 1, __VA_ARGS__)                        \
    else if (lanes_ <= 256) CIGN_LN_ELEMENTS(256, 1, __VA_ARGS__)                        \
    else if (lanes_ <= 512) CIGN_LN_ELEMENTS(512, 1, __VA_ARGS__)                        \
    else CIGN_LN_CASE(1, 16, 8, 1024, 2, __VA_ARGS__)                                    \
  } while (0)

// Blocks of `kernel` that the device holds at once: the grid of a persistent
// kernel.  Asked once per kernel and block size.
template <auto kernel>
int64_t resident_blocks(int threads, size_t smem) {
  static std::atomic<int> known[2 * kLnBlockThreads / 32 + 1];
  std::atomic<int>& k = known[threads / 32];
  int per_sm = k.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem) !=
            cudaSuccess || per_sm < 1)
      per_sm = 1;
    k.store(per_sm, std::memory_order_relaxed);
  }
  return static_cast<int64_t>(per_sm) * sm_count();
}

// Of the widest rows' workspace, a multiple of 16 bytes.
int64_t delta_floats(int64_t n) { return (n + 3) / 4 * 4; }

int64_t ln_wide_chunk(int64_t n) {
  const int64_t c = (n + kLnMaxBlocks - 1) / kLnMaxBlocks;
  return c < 16 ? 16 : c;
}
int64_t ln_wide_sums(int64_t n) {
  const int64_t chunk = ln_wide_chunk(n);
  return (n + chunk - 1) / chunk;
}

int ln_check(int64_t n, int64_t d, int32_t x_type, int32_t param_type, const char* name) {
  CIGN_REQUIRE(n >= 0 && d > 0, CIGN_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
  CIGN_REQUIRE(known_type(x_type) && known_type(param_type), CIGN_ERR_INVALID_ARGUMENT,
               "%s: unknown element type", name);
  CIGN_REQUIRE(n < (1ll << 31) && d <= kLnMaxColumns, CIGN_ERR_UNSUPPORTED,
               "%s: at most 2^31 - 1 rows of at most %lld columns", name,
               static_cast<long long>(kLnMaxColumns));
  return CIGN_OK;
}

template <typename T>
int ln_fwd(int64_t n, int64_t d, const T* x, int64_t ldx, const void* w, const void* b,
           int32_t param_type, float eps, T* y, float* mean, float* rstd, cudaStream_t s) {
  const void* ptrs[] = {x, y};
  const int64_t lds[] = {ldx, d};
  const LnPlan plan = ln_plan<T>(n, d, ptrs, lds, 2);
  if (!plan.shape.fits) {
    layer_norm_wide_fwd_kernel<T><<<static_cast<unsigned>(n), kLnWideThreads, 0, s>>>(
        n, d, x, ldx, w, b, param_type, eps, y, mean, rstd);
    CIGN_CHECK_LAUNCH("layer_norm_wide_fwd_kernel");
    return CIGN_OK;
  }
  CIGN_LN_DISPATCH(T, plan, {
    constexpr auto kernel = layer_norm_fwd_kernel<T, V, NV, SLACK, LANES, BLOCK>;
    const int64_t resident = resident_blocks<kernel>(plan.threads, 0);
    kernel<<<static_cast<unsigned>(plan.blocks < resident ? plan.blocks : resident), plan.threads,
             0, s>>>(n, static_cast<int>(d), x, ldx, w, b, param_type, eps, y, mean, rstd);
  });
  CIGN_CHECK_LAUNCH("layer_norm_fwd_kernel");
  return CIGN_OK;
}

template <typename T>
int ln_bwd(int64_t n, int64_t d, const T* gy, int64_t ldg, const T* x, int64_t ldx, const void* w,
           int32_t param_type, const float* mean, const float* rstd, T* gx, void* gw, void* gb,
           float* ws, cudaStream_t s) {
  const void* ptrs[] = {x, gy, gx};
  const int64_t lds[] = {ldx, ldg, d};
  const LnPlan plan = ln_plan<T>(n, d, ptrs, lds, 3);
  const bool params = gw != nullptr || gb != nullptr;
  // the parameter gradients of the widest rows, by columns
  const bool apart = d > kLnBlockColumns;  // where ln_plan takes more than kLnBlockThreads, or none
  // the workspace: the rows' deltas where the parameter gradients read them, then partial sums
  float* deltas = params && apart ? ws : nullptr;
  float* partial = params && apart ? ws + delta_floats(n) : ws;
  int sums = 0;
  if (!plan.shape.fits || (apart && gx == nullptr)) {
    if (gx || params) {
      layer_norm_wide_bwd_kernel<T><<<static_cast<unsigned>(n), kLnWideThreads, 0, s>>>(
          n, d, gy, ldg, x, ldx, w, param_type, mean, rstd, gx, deltas);
      CIGN_CHECK_LAUNCH("layer_norm_wide_bwd_kernel");
    }
  } else if (gx || params) {
    CIGN_LN_DISPATCH(T, plan, {
      constexpr auto kernel = layer_norm_bwd_kernel<T, V, NV, SLACK, LANES, BLOCK>;
      const size_t smem = BLOCK != 0 ? 0 : kLnGroupThreads * NV * V * sizeof(float);
      int64_t resident = resident_blocks<kernel>(plan.threads, smem);
      if (resident > kLnMaxBlocks) resident = kLnMaxBlocks;
      sums = static_cast<int>(plan.blocks < resident ? plan.blocks : resident);
      kernel<<<sums, plan.threads, smem, s>>>(n, static_cast<int>(d), gy, ldg, x, ldx, w,
                                              param_type, mean, rstd, gx,
                                              params && !apart ? partial : nullptr, deltas);
    });
    CIGN_CHECK_LAUNCH("layer_norm_bwd_kernel");
  }
  if (params && apart) {
    const int64_t chunk = ln_wide_chunk(n);
    sums = static_cast<int>(ln_wide_sums(n));
    const int64_t loads = plan.wide ? d / (16 / sizeof(T)) : d;
    const unsigned cols = static_cast<unsigned>((loads + kLnWideThreads - 1) / kLnWideThreads);
    if (plan.wide)
      layer_norm_wide_param_kernel<T, 16 / sizeof(T)>
          <<<dim3(sums, cols), kLnWideThreads, 0, s>>>(n, d, chunk, gy, ldg, x, ldx, mean, rstd,
                                                       deltas, partial);
    else
      layer_norm_wide_param_kernel<T, 1><<<dim3(sums, cols), kLnWideThreads, 0, s>>>(
          n, d, chunk, gy, ldg, x, ldx, mean, rstd, deltas, partial);
    CIGN_CHECK_LAUNCH("layer_norm_wide_param_kernel");
  }
  if (params) {
    const dim3 grid(static_cast<unsigned>((d + 31) / 32), 2);
    CIGN_TYPE_DISPATCH(param_type, P,
        (layer_norm_param_sum_kernel<P><<<grid, kLnSumWarps * 32, 0, s>>>(
            sums, d, partial, static_cast<P*>(gw), static_cast<P*>(gb))));
    CIGN_CHECK_LAUNCH("layer_norm_param_sum_kernel");
  }
  return CIGN_OK;
}

}  // namespace
}  // namespace cign

using namespace cign;

extern "C" {

int cign_layer_norm_fwd(int64_t n, int64_t d, int32_t x_type, int32_t param_type, const void* x,
                        int64_t ldx, const void* w, const void* b, float eps, void* y,
                        float* mean, float* rstd, cign_stream_t stream) {
  int rc = ln_check(n, d, x_type, param_type, "layer_norm_fwd");
  if (rc) return rc;
  CIGN_REQUIRE(ldx >= d, CIGN_ERR_INVALID_ARGUMENT, "layer_norm_fwd: row stride below the width");
  CIGN_REQUIRE(eps >= 0.0f, CIGN_ERR_INVALID_ARGUMENT, "layer_norm_fwd: eps must not be negative");
  if (n == 0) return CIGN_OK;
  CIGN_REQUIRE(x && y && (mean == nullptr) == (rstd == nullptr), CIGN_ERR_NULL_POINTER,
               "layer_norm_fwd: NULL argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CIGN_TYPE_DISPATCH(x_type, T,
      return ln_fwd<T>(n, d, static_cast<const T*>(x), ldx, w, b, param_type, eps,
                       static_cast<T*>(y), mean, rstd, s));
}

size_t cign_layer_norm_bwd_workspace_bytes(int64_t n, int64_t d) {
  if (n <= 0 || d <= 0) return 0;
  // grad w and grad b of every partial sum: one per persistent block, or per chunk of rows
  const bool apart = d > kLnBlockColumns;
  const int64_t sums = apart ? ln_wide_sums(n) : n < kLnMaxBlocks ? n : kLnMaxBlocks;
  return (2 * static_cast<size_t>(sums) * d + (apart ? delta_floats(n) : 0)) * sizeof(float);
}

int cign_layer_norm_bwd(int64_t n, int64_t d, int32_t x_type, int32_t param_type, const void* gy,
                        int64_t ldg, const void* x, int64_t ldx, const void* w, const float* mean,
                        const float* rstd, void* gx, void* gw, void* gb, void* ws,
                        size_t ws_bytes, cign_stream_t stream) {
  int rc = ln_check(n, d, x_type, param_type, "layer_norm_bwd");
  if (rc) return rc;
  CIGN_REQUIRE(ldx >= d && ldg >= d, CIGN_ERR_INVALID_ARGUMENT,
               "layer_norm_bwd: row stride below the width");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t psize = type_size(param_type);
  if (n == 0) {
    if (gw) CIGN_CHECK_CUDA(cudaMemsetAsync(gw, 0, d * psize, s), "layer_norm_bwd: memset");
    if (gb) CIGN_CHECK_CUDA(cudaMemsetAsync(gb, 0, d * psize, s), "layer_norm_bwd: memset");
    return CIGN_OK;
  }
  CIGN_REQUIRE(gy && x && mean && rstd, CIGN_ERR_NULL_POINTER, "layer_norm_bwd: NULL argument");
  if (gw != nullptr || gb != nullptr) {
    const size_t need = cign_layer_norm_bwd_workspace_bytes(n, d);
    CIGN_REQUIRE(ws != nullptr && ws_bytes >= need, CIGN_ERR_INVALID_ARGUMENT,
                 "layer_norm_bwd: workspace too small (%zu < %zu bytes)", ws_bytes, need);
    CIGN_REQUIRE(aligned16(ws), CIGN_ERR_ALIGNMENT,
                 "layer_norm_bwd: ws must be 16-byte aligned");
  }
  CIGN_TYPE_DISPATCH(x_type, T,
      return ln_bwd<T>(n, d, static_cast<const T*>(gy), ldg, static_cast<const T*>(x), ldx, w,
                       param_type, mean, rstd, static_cast<T*>(gx), gw, gb,
                       static_cast<float*>(ws), s));
}

}  // extern "C"

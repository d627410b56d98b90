// Divergence of a student's class distribution from a teacher's kept classes,
// and the gradient of the student's logits.  Row: logits x over c classes,
// kept entries (class c_i, value v_i), temperature T, p = softmax(x / T).
//   tail "drop":   q = softmax(v / T) over the entries, r = 0
//   tail "bucket": q_i = e^(v_i), r = max(0, 1 - sum q); the classes that are
//                  not kept form one class of probability p_rest
//   loss   = T^2 (sum_i q_i (log q_i - log p_{c_i}) + r (log r - log p_rest))
//   grad_j = T g (W p_j - q_j)               kept classes,  W = sum q + r
//   grad_j = T g p_j (W - r / p_rest)        others
// The loss of two near distributions is a small difference of such terms, so
// it is formed as a sum of terms that are not negative,
//   loss / T^2 = sum_i q_i (e^-d_i - 1 + d_i) + (the same of the rest) + (W - 1)
// with d_i = log q_i - log p_{c_i}: the added sum p - sum q is W - 1 exactly,
// because sum over kept p + p_rest = 1, and an error of the row's log sum
// cancels in first order.  W p_j - q_j is q_j (expm1(-d_j) + (W - 1) e^-d_j).
// d and r are formed in 64 bits from the float32 values.
#include "class_rows.cuh"

namespace cign {
namespace {

constexpr int kDsThreads = 256;
constexpr int kDsWarps = kDsThreads / 32;
constexpr int kDsMaxKept = 256;
constexpr int kDsStats = 8;
constexpr int64_t kDsMaxClasses = 1 << 20;  // one bit each in shared memory

template <int WARPS>
__device__ __forceinline__ double block_sum_f64(double v, double* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) s += part[w];
  return s;
}

struct Teacher {
  const void* values;
  const void* index;
  int64_t ld_values, ld_index;
  int32_t k;
  int32_t value_type;
  int32_t wide_index;  // int64 (else int32)
};

__device__ __forceinline__ float teacher_value(const Teacher& t, int64_t row, int i) {
  const int64_t at = row * t.ld_values + i;
  if (t.value_type == CIGN_F32) return static_cast<const float*>(t.values)[at];
  if (t.value_type == CIGN_BF16) return to_f(static_cast<const __nv_bfloat16*>(t.values)[at]);
  return to_f(static_cast<const __half*>(t.values)[at]);
}
__device__ __forceinline__ int64_t teacher_index(const Teacher& t, int64_t row, int i) {
  const int64_t at = row * t.ld_index + i;
  return t.wide_index ? static_cast<const int64_t*>(t.index)[at]
                      : static_cast<int64_t>(static_cast<const int32_t*>(t.index)[at]);
}

// 1 / T as a float and what it leaves, so d / T = d * hi + d * lo.
struct InvT {
  float hi, lo;
  double full;
};

__device__ __forceinline__ float scaled(float d, const InvT& it) {
  return fmaf(d, it.hi, d == -INFINITY ? 0.0f : d * it.lo);
}

// Running sum of e^((x - m) / T) - 1, as RowStat without t.
__device__ __forceinline__ void stat_add_t(RowStat& a, float x, const InvT& it) {
  if (x > a.m) {
    a.s = (1.0f + a.s) * expf(scaled(a.m - x, it));
    a.m = x;
  } else if (x == a.m) {
    a.s += 1.0f;
  } else {
    a.s += expf(scaled(x - a.m, it));
  }
}
__device__ __forceinline__ RowStat stat_merge_t(const RowStat& a, const RowStat& b,
                                                const InvT& it) {
  const bool ge = a.m >= b.m;
  const RowStat hi = ge ? a : b, lo = ge ? b : a;
  RowStat r;
  r.m = hi.m;
  r.s = hi.s + (1.0f + lo.s) * (a.m == b.m ? 1.0f : expf(scaled(lo.m - hi.m, it)));
  return r;
}
__device__ __forceinline__ RowStat block_stat_t(RowStat a, RowStat* part, const InvT& it) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = stat_merge_t(a, stat_shfl_xor(a, o), it);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  a = part[0];
#pragma unroll
  for (int w = 1; w < kDsWarps; ++w) a = stat_merge_t(a, part[w], it);
  return a;
}

// q (e^-d - 1 + d), which is not negative; by its series where d is small.
__device__ __forceinline__ float divergence_term(float q, float d) {
  if (fabsf(d) < 0.125f) {
    const float h = fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.0f / 720.0f, -1.0f / 120.0f), 1.0f / 24.0f),
                                 -1.0f / 6.0f), 0.5f);
    return q * (d * d) * h;
  }
  return q * (expm1f(-d) + d);
}

// What the forward keeps of a row for the backward.
struct DistillRow {
  float m;       // maximum of the logits
  float logs;    // log sum e^((x - m) / T)
  float spread;  // W - r / p_rest: the factor of p outside the kept classes
  float w1;      // W - 1
  float tmax;    // tail "drop": maximum and log sum of the teacher's values
  float tlog;
  float dup;     // 1 where a class is kept twice
  float none;    // 1 where the row has no kept class
};

__device__ __forceinline__ double log_q(float v, const DistillRow& r, bool bucket,
                                        const InvT& it) {
  if (bucket) return v;
  return (static_cast<double>(v) - r.tmax) * it.full - static_cast<double>(r.tlog);
}

// W p - q of a kept class: q the sum of its entries.
__device__ __forceinline__ float kept_gradient(const Teacher& te, int64_t row, int64_t c,
                                               int64_t idx, float v, double lp,
                                               const DistillRow& r, bool bucket, const InvT& it) {
  const double lq = log_q(v, r, bucket, it);
  if (r.dup == 0.0f) {
    const float d = static_cast<float>(lq - lp);
    return expf(static_cast<float>(lq)) *
           (expm1f(-d) + (r.w1 != 0.0f ? r.w1 * expf(-d) : 0.0f));
  }
  float q = 0.0f;
  for (int i = 0; i < te.k; ++i) {
    const float w = teacher_value(te, row, i);
    if (teacher_index(te, row, i) == idx && w != -INFINITY)
      q += expf(static_cast<float>(log_q(w, r, bucket, it)));
  }
  return (1.0f + r.w1) * expf(static_cast<float>(lp)) - q;
}

__device__ __forceinline__ DistillRow load_row(const float* stats) {
  const float4 a = reinterpret_cast<const float4*>(stats)[0];
  const float4 b = reinterpret_cast<const float4*>(stats)[1];
  return DistillRow{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// The row's loss and statistics from the sum over its entries.
__device__ __forceinline__ void finish_row(DistillRow r, float sum, float mass_r, float p_rest,
                                           bool none, bool bad, bool dup, float temperature,
                                           float* loss, float* stats) {
  if (mass_r != 0.0f)
    sum += p_rest > 0.0f ? divergence_term(mass_r, logf(mass_r) - logf(p_rest)) : INFINITY;
  else
    sum += p_rest;
  float l = temperature * temperature * (sum + r.w1);
  r.spread = (1.0f + r.w1) - (mass_r != 0.0f && p_rest > 0.0f ? mass_r / p_rest : 0.0f);
  r.dup = dup ? 1.0f : 0.0f;
  r.none = none ? 1.0f : 0.0f;
  if (r.m == -INFINITY && r.logs == r.logs) l = INFINITY;  // the student has no class left
  if (none) l = 0.0f;
  if (bad) {
    l = r.logs = r.spread = __int_as_float(0x7fffffff);
    r.none = 0.0f;
  }
  *loss = l;
  if (stats) {
    reinterpret_cast<float4*>(stats)[0] = make_float4(r.m, r.logs, r.spread, r.w1);
    reinterpret_cast<float4*>(stats)[1] = make_float4(r.tmax, r.tlog, r.dup, r.none);
  }
}

template <typename T>
__global__ void __launch_bounds__(kDsThreads)
distill_fwd_kernel(int64_t n, int64_t c, const T* __restrict__ logits, int64_t ld, Teacher te,
                   float temperature, InvT it, int bucket, float* __restrict__ loss,
                   float* __restrict__ stats) {
  extern __shared__ uint32_t kept_bits[];
  __shared__ RowStat part[kDsWarps];
  __shared__ float fpart[kDsWarps];
  __shared__ double dpart[kDsWarps];
  __shared__ int64_t kidx[kDsMaxKept];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T* x = logits + row * ld;
  for (int64_t i = tid; i < (c + 31) / 32; i += kDsThreads) kept_bits[i] = 0;
  // the teacher's entries, one per thread
  int64_t idx = -1;
  float v = -INFINITY;
  if (tid < te.k) {
    idx = teacher_index(te, row, tid);
    v = teacher_value(te, row, tid);
    if (v == -INFINITY) idx = -1;
    kidx[tid] = idx;
  }
  const bool bad = idx >= c;
  const bool valid = idx >= 0 && !bad;
  __syncthreads();
  bool first = false;
  if (valid) first = !((atomicOr(&kept_bits[idx >> 5], 1u << (idx & 31)) >> (idx & 31)) & 1u);
  const int any_bad = __syncthreads_or(bad);
  const int any_dup = __syncthreads_or(valid && !first);
  const int distinct = __syncthreads_count(first);
  if (any_dup) {  // the first of equal entries by its place, not by the race above
    first = valid;
    for (int i = 0; i < tid && first; ++i) first = kidx[i] != idx;
  }
  // student: classes that are not kept, then kept ones
  RowStat rest;
  for (int64_t j = tid; j < c; j += kDsThreads)
    if (!((kept_bits[j >> 5] >> (j & 31)) & 1u)) stat_add_t(rest, to_f(x[j]), it);
  rest = block_stat_t(rest, part, it);
  RowStat all;
  const float xi = valid ? to_f(x[idx]) : 0.0f;
  if (first) stat_add_t(all, xi, it);
  all = stat_merge_t(block_stat_t(all, part, it), rest, it);
  DistillRow r;
  r.m = all.m;
  r.logs = all.m == INFINITY ? __int_as_float(0x7fffffff) : log1pf(all.s);
  const float p_rest = (1.0f + rest.s) *
                       (rest.m == all.m ? 1.0f : expf(scaled(rest.m - all.m, it))) /
                       (1.0f + all.s);
  // teacher
  RowStat ts;
  if (valid) stat_add_t(ts, v, it);
  ts = block_stat_t(ts, part, it);
  r.tmax = ts.m;
  r.tlog = log1pf(ts.s);
  const float lq = valid ? static_cast<float>(log_q(v, r, bucket, it)) : -INFINITY;
  const float q = expf(lq);
  float mass_r = 0.0f;
  r.w1 = 0.0f;
  if (bucket) {
    // a small difference where the teacher is sure of its kept classes: 64 bits
    const float raw = static_cast<float>(
        1.0 - block_sum_f64<kDsWarps>(valid ? exp(static_cast<double>(v)) : 0.0, dpart));
    if (raw == raw && raw < 0.0f) r.w1 = -raw;
    else mass_r = raw;
    if (distinct == c) {  // no class is left to take the rest
      r.w1 = -raw;
      mass_r = 0.0f;
    }
  }
  float term = 0.0f;
  if (valid) {
    const double lp = (static_cast<double>(xi) - all.m) * it.full - static_cast<double>(r.logs);
    const float d = static_cast<float>(log_q(v, r, bucket, it) - lp);
    term = first ? divergence_term(q, d) : q * (d - 1.0f);
  }
  const float sum = block_sum<kDsWarps>(term, fpart);
  if (tid == 0)
    finish_row(r, sum, mass_r, p_rest, distinct == 0, any_bad, any_dup, temperature, loss + row,
               stats ? stats + row * kDsStats : nullptr);
}

template <typename T>
__global__ void __launch_bounds__(kDsThreads)
distill_bwd_kernel(int64_t n, int64_t c, const T* __restrict__ logits, int64_t ld, Teacher te,
                   float temperature, InvT it, int bucket, const float* __restrict__ stats,
                   const float* __restrict__ g_loss, int64_t g_stride, T* __restrict__ grad) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T* x = logits + row * ld;
  T* out = grad + row * c;
  const DistillRow r = load_row(stats + row * kDsStats);
  const float g = g_loss[row * g_stride] * temperature;
  if (r.none != 0.0f || g == 0.0f || (r.m == -INFINITY && r.logs == r.logs)) {
    for (int64_t j = tid; j < c; j += kDsThreads) out[j] = from_f<T>(0.0f);
    return;
  }
  const float f = g * r.spread;
  for (int64_t j = tid; j < c; j += kDsThreads) {
    const float p = expf(scaled(to_f(x[j]) - r.m, it) - r.logs);
    out[j] = from_f<T>(p * f);
  }
  __syncthreads();  // orders the writes above before those below
  if (tid < te.k) {
    const int64_t idx = teacher_index(te, row, tid);
    const float v = teacher_value(te, row, tid);
    if (idx >= 0 && idx < c && v != -INFINITY) {
      const double lp = (static_cast<double>(to_f(x[idx])) - r.m) * it.full -
                        static_cast<double>(r.logs);
      out[idx] = from_f<T>(g * kept_gradient(te, row, c, idx, v, lp, r, bucket, it));
    }
  }
}

// Rows of at most E G classes, a group of G lanes per row (class_rows.cuh).
// The kept classes of a row are bits in shared memory; lane l takes the
// teacher's entries l, l + G, ...
template <typename T, int G, int E>
__global__ void __launch_bounds__(kNarrowThreads)
distill_narrow_fwd_kernel(int64_t n, int c, const T* __restrict__ logits, int64_t ld, Teacher te,
                          float temperature, InvT it, int bucket, float* __restrict__ loss,
                          float* __restrict__ stats) {
  constexpr int kWords = (G * E + 31) / 32;
  __shared__ uint32_t all_bits[kNarrowThreads / G * kWords];
  const int lane = threadIdx.x & (G - 1);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (kNarrowThreads / G) + threadIdx.x / G;
  const bool live = at < n;
  const int64_t row = live ? at : n - 1;  // the last warp's idle groups follow along
  const T* x = logits + row * ld;
  uint32_t* bits = all_bits + threadIdx.x / G * kWords;
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    v[i] = lane + G * i < c ? to_f(x[lane + G * i]) : -INFINITY;
  for (int i = lane; i < kWords; i += G) bits[i] = 0;
  __syncwarp();
  // teacher: kept classes, maximum, log sum, sum of probabilities
  bool bad = false, dup = false;
  float tmax = -INFINITY, nan = 0.0f;
  float distinct = 0.0f;
  for (int e = lane; e < te.k; e += G) {
    const int64_t idx = teacher_index(te, row, e);
    const float tv = teacher_value(te, row, e);
    if (idx < 0 || tv == -INFINITY) continue;
    if (idx >= c) {
      bad = true;
      continue;
    }
    const uint32_t bit = 1u << (idx & 31);
    const bool first = !(atomicOr(bits + (idx >> 5), bit) & bit);
    dup |= !first;
    distinct += first ? 1.0f : 0.0f;
    tmax = fmaxf(tmax, tv);
    if (tv != tv) nan = tv;
  }
  const unsigned mine = group_mask<G>();
  bad = __ballot_sync(kFullMask, bad) & mine;
  dup = __ballot_sync(kFullMask, dup) & mine;
  __syncwarp();
  distinct = group_sum<G>(distinct);
  DistillRow r;
  r.tmax = group_max<G>(tmax);
  float tsum = 0.0f, tcnt = 0.0f;
  double mass = 0.0;
  for (int e = lane; e < te.k; e += G) {
    const int64_t idx = teacher_index(te, row, e);
    const float tv = teacher_value(te, row, e);
    if (idx < 0 || idx >= c || tv == -INFINITY) continue;
    if (bucket) mass += exp(static_cast<double>(tv));
    else if (tv == r.tmax) tcnt += 1.0f;
    else tsum += expf(scaled(tv - r.tmax, it));
  }
  r.tlog = log1pf(group_sum<G>(tsum + nan) + (group_sum<G>(tcnt) - 1.0f));
  // student: the sums over the classes that are not kept and over the kept ones
  float m = v[0];
#pragma unroll
  for (int i = 1; i < E; ++i) m = fmaxf(m, v[i]);
  m = group_max<G>(m);
  if (m != m) m = -INFINITY;
  float s_rest = 0.0f, c_rest = 0.0f, s_kept = 0.0f, c_kept = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int j = lane + G * i;
    const bool kept = (bits[j >> 5] >> (j & 31)) & 1u;
    const float one = j < c && v[i] == m ? 1.0f : 0.0f;
    const float e = v[i] == m ? 0.0f : expf(scaled(v[i] - m, it));
    s_kept += kept ? e : 0.0f;
    c_kept += kept ? one : 0.0f;
    s_rest += kept ? 0.0f : e;
    c_rest += kept ? 0.0f : one;
  }
  s_rest = group_sum<G>(s_rest);
  c_rest = group_sum<G>(c_rest);
  const float s = s_rest + group_sum<G>(s_kept) + (group_sum<G>(c_kept) + c_rest - 1.0f);
  r.m = m;
  r.logs = m == INFINITY ? __int_as_float(0x7fffffff) : log1pf(s);
  const float p_rest = (s_rest + c_rest) / (1.0f + s);
  float mass_r = 0.0f;
  r.w1 = 0.0f;
  if (bucket) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) mass += __shfl_xor_sync(kFullMask, mass, o);
    // a small difference where the teacher is sure of its kept classes: 64 bits
    const float raw = static_cast<float>(1.0 - mass);
    if (raw == raw && raw < 0.0f) r.w1 = -raw;
    else mass_r = raw;
    if (distinct == static_cast<float>(c)) {  // no class is left to take the rest
      r.w1 = -raw;
      mass_r = 0.0f;
    }
  }
  float sum = 0.0f;
  for (int e = lane; e < te.k; e += G) {
    const int64_t idx = teacher_index(te, row, e);
    const float tv = teacher_value(te, row, e);
    if (idx < 0 || idx >= c || tv == -INFINITY) continue;
    bool first = true;
    if (dup)  // the first of equal entries by its place
      for (int q = 0; q < e && first; ++q)
        first = teacher_index(te, row, q) != idx || teacher_value(te, row, q) == -INFINITY;
    const double lq = log_q(tv, r, bucket, it);
    const double lp = (static_cast<double>(to_f(x[idx])) - m) * it.full -
                      static_cast<double>(r.logs);
    const float q = expf(static_cast<float>(lq));
    const float d = static_cast<float>(lq - lp);
    sum += first ? divergence_term(q, d) : q * (d - 1.0f);
  }
  sum = group_sum<G>(sum);
  if (live && lane == 0) finish_row(r, sum, mass_r, p_rest, distinct == 0.0f, bad, dup,
                                    temperature, loss + row,
                                    stats ? stats + row * kDsStats : nullptr);
}

template <typename T, int G, int E>
__global__ void __launch_bounds__(kNarrowThreads)
distill_narrow_bwd_kernel(int64_t n, int c, const T* __restrict__ logits, int64_t ld, Teacher te,
                          float temperature, InvT it, int bucket,
                          const float* __restrict__ stats, const float* __restrict__ g_loss,
                          int64_t g_stride, T* __restrict__ grad) {
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kNarrowThreads / G) + threadIdx.x / G;
  const unsigned mine = group_mask<G>();
  if (row >= n) return;
  const T* x = logits + row * ld;
  T* out = grad + row * c;
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    v[i] = lane + G * i < c ? to_f(x[lane + G * i]) : -INFINITY;
  const DistillRow r = load_row(stats + row * kDsStats);
  const float g = g_loss[row * g_stride] * temperature;
  const bool zero = r.none != 0.0f || g == 0.0f || (r.m == -INFINITY && r.logs == r.logs);
  const float f = g * r.spread;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (lane + G * i < c)
      out[lane + G * i] =
          from_f<T>(zero ? 0.0f : f * expf(scaled(v[i] - r.m, it) - r.logs));
  if (zero) return;
  __syncwarp(mine);  // orders the writes above before those below
  for (int e = lane; e < te.k; e += G) {
    const int64_t idx = teacher_index(te, row, e);
    const float tv = teacher_value(te, row, e);
    if (idx < 0 || idx >= c || tv == -INFINITY) continue;
    const double lp = (static_cast<double>(to_f(x[idx])) - r.m) * it.full -
                      static_cast<double>(r.logs);
    out[idx] = from_f<T>(g * kept_gradient(te, row, c, idx, tv, lp, r, bucket, it));
  }
}

int ds_check(int64_t n, int64_t c, int32_t x_type, int64_t ld, int32_t k, int32_t value_type,
             int64_t ld_values, int32_t index_type, int64_t ld_index, float temperature,
             int32_t tail, const char* name) {
  CIGN_REQUIRE(n >= 0 && c > 0, CIGN_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
  CIGN_REQUIRE(known_type(x_type) && known_type(value_type), CIGN_ERR_INVALID_ARGUMENT,
               "%s: unknown element type", name);
  CIGN_REQUIRE(index_type == 0 || index_type == 1, CIGN_ERR_INVALID_ARGUMENT,
               "%s: index type must be 0 (int32) or 1 (int64)", name);
  CIGN_REQUIRE(ld >= c, CIGN_ERR_INVALID_ARGUMENT, "%s: row stride below the class count", name);
  CIGN_REQUIRE(k >= 1, CIGN_ERR_INVALID_ARGUMENT, "%s: no kept classes", name);
  CIGN_REQUIRE(ld_values >= k && ld_index >= k, CIGN_ERR_INVALID_ARGUMENT,
               "%s: row stride of the teacher's entries below their number", name);
  CIGN_REQUIRE(temperature > 0.0f && temperature <= 3.402823466e38f, CIGN_ERR_INVALID_ARGUMENT,
               "%s: temperature must be positive and finite", name);
  CIGN_REQUIRE(tail == 0 || tail == 1, CIGN_ERR_INVALID_ARGUMENT,
               "%s: tail must be 0 (drop) or 1 (bucket)", name);
  CIGN_REQUIRE(k <= kDsMaxKept, CIGN_ERR_UNSUPPORTED, "%s: at most %d kept classes", name,
               kDsMaxKept);
  CIGN_REQUIRE(n < (1ll << 31) && c <= kDsMaxClasses, CIGN_ERR_UNSUPPORTED,
               "%s: at most 2^31 - 1 rows of at most 2^20 classes", name);
  return CIGN_OK;
}

InvT inverse(float temperature) {
  InvT it;
  it.full = 1.0 / static_cast<double>(temperature);
  it.hi = static_cast<float>(it.full);
  it.lo = static_cast<float>(it.full - static_cast<double>(it.hi));
  return it;
}

}  // namespace
}  // namespace cign

using namespace cign;

extern "C" {

int cign_distill_fwd(int64_t n, int64_t c, int32_t x_type, const void* logits, int64_t ld,
                     int32_t k, int32_t value_type, const void* values, int64_t ld_values,
                     int32_t index_type, const void* index, int64_t ld_index, float temperature,
                     int32_t tail, float* loss, float* stats, cign_stream_t stream) {
  int rc = ds_check(n, c, x_type, ld, k, value_type, ld_values, index_type, ld_index, temperature,
                    tail, "distill_fwd");
  if (rc) return rc;
  if (n == 0) return CIGN_OK;
  CIGN_REQUIRE(logits && values && index && loss, CIGN_ERR_NULL_POINTER,
               "distill_fwd: NULL argument");
  CIGN_REQUIRE(aligned16(stats), CIGN_ERR_ALIGNMENT, "distill_fwd: stats must be 16-byte aligned");
  const Teacher te{values, index, ld_values, ld_index, k, value_type, index_type};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c <= kNarrowMax) {
    CIGN_TYPE_DISPATCH(x_type, T, CIGN_GROUP_DISPATCH(c,
        distill_narrow_fwd_kernel<T, G, E><<<narrow_grid(n, G), kNarrowThreads, 0, s>>>(
            n, static_cast<int>(c), static_cast<const T*>(logits), ld, te, temperature,
            inverse(temperature), tail, loss, stats)));
    CIGN_CHECK_LAUNCH("distill_narrow_fwd_kernel");
    return CIGN_OK;
  }
  const size_t smem = static_cast<size_t>((c + 31) / 32) * 4;
  CIGN_TYPE_DISPATCH(x_type, T, {
    if (smem > 32768)
      CIGN_CHECK_CUDA(cudaFuncSetAttribute(distill_fwd_kernel<T>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(kDsMaxClasses / 8)),
                      "distill_fwd: shared memory");
    distill_fwd_kernel<T><<<static_cast<unsigned>(n), kDsThreads, smem, s>>>(
        n, c, static_cast<const T*>(logits), ld, te, temperature, inverse(temperature), tail, loss,
        stats);
  });
  CIGN_CHECK_LAUNCH("distill_fwd_kernel");
  return CIGN_OK;
}

int cign_distill_bwd(int64_t n, int64_t c, int32_t x_type, const void* logits, int64_t ld,
                     int32_t k, int32_t value_type, const void* values, int64_t ld_values,
                     int32_t index_type, const void* index, int64_t ld_index, float temperature,
                     int32_t tail, const float* stats, const float* grad_loss,
                     int64_t grad_loss_stride, void* grad_logits, cign_stream_t stream) {
  int rc = ds_check(n, c, x_type, ld, k, value_type, ld_values, index_type, ld_index, temperature,
                    tail, "distill_bwd");
  if (rc) return rc;
  if (n == 0) return CIGN_OK;
  CIGN_REQUIRE(logits && values && index && stats && grad_loss && grad_logits,
               CIGN_ERR_NULL_POINTER, "distill_bwd: NULL argument");
  CIGN_REQUIRE(aligned16(stats), CIGN_ERR_ALIGNMENT, "distill_bwd: stats must be 16-byte aligned");
  const Teacher te{values, index, ld_values, ld_index, k, value_type, index_type};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c <= kNarrowMax) {
    CIGN_TYPE_DISPATCH(x_type, T, CIGN_GROUP_DISPATCH_WRITE(c,
        distill_narrow_bwd_kernel<T, G, E><<<narrow_grid(n, G), kNarrowThreads, 0, s>>>(
            n, static_cast<int>(c), static_cast<const T*>(logits), ld, te, temperature,
            inverse(temperature), tail, stats, grad_loss, grad_loss_stride,
            static_cast<T*>(grad_logits))));
    CIGN_CHECK_LAUNCH("distill_narrow_bwd_kernel");
    return CIGN_OK;
  }
  CIGN_TYPE_DISPATCH(x_type, T,
      distill_bwd_kernel<T><<<static_cast<unsigned>(n), kDsThreads, 0, s>>>(
          n, c, static_cast<const T*>(logits), ld, te, temperature, inverse(temperature), tail,
          stats, grad_loss, grad_loss_stride, static_cast<T*>(grad_logits)));
  CIGN_CHECK_LAUNCH("distill_bwd_kernel");
  return CIGN_OK;
}

}  // extern "C"

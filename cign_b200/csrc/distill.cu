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
// d and r are formed in 64 bits from the float32 values.  Where d is far below 0
// the terms are formed as p - q + q d and W p - q: e^-d alone may overflow.
#include <cooperative_groups.h>

#include "class_rows.cuh"

namespace cign {
namespace {

constexpr int kDsMaxKept = 256;
constexpr int kDsStats = 8;
constexpr int64_t kDsMaxClasses = 1 << 20;  // one bit each in shared memory

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

// q (e^-d - 1 + d), which is not negative; by its series where d is small.
__device__ __forceinline__ float divergence_term(float q, float d) {
  if (fabsf(d) < 0.125f) {
    const float h = fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.0f / 720.0f, -1.0f / 120.0f), 1.0f / 24.0f),
                                 -1.0f / 6.0f), 0.5f);
    return q * (d * d) * h;
  }
  return q * (expm1f(-d) + d);
}

// The student's probability is e^8 times the teacher's and more: e^-d, which may
// be no float32 number while q is 0, is left out, and p - q loses nothing.
constexpr float kFarBelow = -8.0f;

// A class that the student all but masks: in 64 bits, so that q = 0 is a
// probability that no product with d = -log p makes visible.
__device__ __noinline__ float far_above_term(double lq, double lp, bool first, float scale) {
  const double q = exp(lq), p = first ? exp(lp) : 0.0;
  return static_cast<float>(scale * (p - q + (q > 0.0 ? q * (lq - lp) : 0.0)));
}

// An entry's part of the loss, p - q + q d with q = e^lq, p = e^lp, d = lq - lp,
// times `scale`; p counts with the first entry of a class.
__device__ __forceinline__ float entry_term(double lq, double lp, bool first, float scale) {
  const float q = expf(static_cast<float>(lq));
  const float d = static_cast<float>(lq - lp);
  if (d < kFarBelow)
    return scale * ((first ? expf(static_cast<float>(lp)) - q : -q) + (q > 0.0f ? q * d : 0.0f));
  if (!(d < 1e4f)) return far_above_term(lq, lp, first, scale);  // NaN too
  return scale * (first ? divergence_term(q, d) : q * (d - 1.0f));
}

// What the forward keeps of a row for the backward.  Outside the kept classes
// the gradient is T g p_j (W - r / p_rest).  Where r / p_rest is above e it is
// formed as T g r (W p_rest / r - 1) (p_j / p_rest), the last of which needs the
// distance to the rest's own maximum only, however far that is below the row's.
struct DistillRow {
  float m;       // maximum of the logits
  float logs;    // log sum e^((x - m) / T)
  float spread;  // the gradient of the other classes is T g spread e^((x - base) / T - base_log)
  float w1;      // W - 1
  float tmax;    // tail "drop": maximum and log sum of the teacher's values
  float tlog;
  float kind;    // 0; 1: a class is kept twice; 2: the row has no kept class
  __device__ __forceinline__ float base(bool bucket) const { return bucket ? tmax : m; }
  __device__ __forceinline__ float base_log(bool bucket) const { return bucket ? tlog : logs; }
};

__device__ __forceinline__ double log_q(float v, const DistillRow& r, bool bucket,
                                        const InvT& it) {
  if (bucket) return v;
  return (static_cast<double>(v) - r.tmax) * it.full - static_cast<double>(r.tlog);
}

// W p - q of a kept class: q the sum of its entries.
__device__ __forceinline__ float kept_gradient(const Teacher& te, int64_t row, int64_t idx,
                                               float v, double lp, const DistillRow& r,
                                               bool bucket, const InvT& it) {
  const double lq = log_q(v, r, bucket, it);
  if (r.kind == 0.0f) {
    const float d = static_cast<float>(lq - lp);
    if (d < kFarBelow)
      return (1.0f + r.w1) * expf(static_cast<float>(lp)) - expf(static_cast<float>(lq));
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
  return DistillRow{a.x, a.y, a.z, a.w, b.x, b.y, b.z};
}

// T^2 as a factor of a row's terms and one of their sum: below 1 the terms have
// it, so that a far one of them, up to 10^42 before, stays a float32 number.
__device__ __forceinline__ float term_scale(float temperature) {
  return temperature < 1.0f ? temperature * temperature : 1.0f;
}
__device__ __forceinline__ float sum_scale(float temperature) {
  return temperature < 1.0f ? 1.0f : temperature * temperature;
}

// The row's loss and statistics from the sum over its entries, whose terms have
// term_scale; rest_m and rest_log are the maximum and log sum of the rest alone.
__device__ __forceinline__ void finish_row(DistillRow r, float sum, float mass_r, float rest_m,
                                           float rest_log, const InvT& it, bool bucket, bool none,
                                           bool bad, bool dup, float temperature, float* loss,
                                           float* stats) {
  const float w = 1.0f + r.w1, ts = term_scale(temperature);
  // log p_rest
  const float log_rest = rest_m == -INFINITY ? -INFINITY
                         : rest_m == r.m     ? rest_log - r.logs
                                             : rest_log + scaled(rest_m - r.m, it) - r.logs;
  r.spread = w;
  if (bucket) {
    r.tmax = r.m;
    r.tlog = r.logs;
  }
  if (mass_r != 0.0f) {
    const float d = logf(mass_r) - log_rest;
    if (!(d >= 1e30f) || rest_m == -INFINITY) {
      sum += ts * divergence_term(mass_r, d);
    } else {
      sum += static_cast<float>(
          ts * (mass_r * ((static_cast<double>(r.m) - static_cast<double>(rest_m)) * it.full)));
    }
    if (d < 1.0f) {
      r.spread = w - expf(d);
    } else if (rest_m > -INFINITY) {
      r.spread = (w * expf(-d) - 1.0f) * mass_r;
      r.tmax = rest_m;
      r.tlog = rest_log;
    }
  } else {
    sum += ts * expf(log_rest);
  }
  float l = sum_scale(temperature) * fmaf(ts, r.w1, sum);
  if (r.m == -INFINITY && r.logs == r.logs) l = INFINITY;  // the student has no class left
  if (none) l = 0.0f;
  if (bad) l = r.logs = r.spread = __int_as_float(0x7fffffff);
  r.kind = none && !bad ? 2.0f : dup ? 1.0f : 0.0f;
  *loss = l;
  if (stats) {
    reinterpret_cast<float4*>(stats)[0] = make_float4(r.m, r.logs, r.spread, r.w1);
    reinterpret_cast<float4*>(stats)[1] = make_float4(r.tmax, r.tlog, r.kind, 0.0f);
  }
}

// What tail "bucket" leaves to the other classes (r) and W - 1, from the
// teacher's summed probabilities; no class is left to take it where all are kept.
__device__ __forceinline__ float rest_mass(double mass, bool all_kept, float& w1) {
  // a small difference where the teacher is sure of its kept classes
  const float raw = static_cast<float>(1.0 - mass);
  w1 = 0.0f;
  if (all_kept || raw < 0.0f) w1 = -raw;
  return all_kept || raw < 0.0f ? 0.0f : raw;
}

// Rows of more than kNarrowMax classes: a team of W warps per row, with W = 8 a
// cluster of blocks where rows are few.  The kept classes are bits in shared
// memory, at their places in the row's frame, so that a thread finds those of
// its 16 bytes in one byte or half of one.  4096 x 32768 bf16, 64 kept: 93 us, 2.9
// TB/s, bound by issue (67% of the slots), as the forward of node_log_probs.cu with
// a read of the bits per 16 bytes; 777 x 10007 fp16: 14 us, and 16 x 1000 float32:
// 5.8 us, latency: the row, then one warp's arithmetic on the entries.
template <int W>
struct alignas(16) DistillShared {
  int64_t index[kDsMaxKept];  // -1: absent
  float value[kDsMaxKept];
  float x[kDsMaxKept];
  Sums part[W];
  Sums sums;
  int bad, dup, distinct;
};

template <typename T, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 8 ? 4 : 8)
distill_wide_fwd_kernel(int64_t n, int64_t c, const T* __restrict__ logits, int64_t ld, Teacher te,
                        float temperature, InvT it, int bucket, int split, int words,
                        float* __restrict__ loss, float* __restrict__ stats) {
  constexpr int V = RowFrame<T>::V;
  constexpr int L = kWideLoads<T>;
  constexpr int kTeams = W == 1 ? 4 : 1;
  constexpr int kThreads = 32 * W;
  // the ring of the loads, then the teams' bits
  extern __shared__ __align__(16) unsigned char dynamic[];
  uint32_t* all_bits = reinterpret_cast<uint32_t*>(dynamic + ring_bytes<T>(kTeams * kThreads));
  __shared__ DistillShared<W> all[kTeams];
  const int team = W == 1 ? threadIdx.x >> 5 : 0;
  const int tid = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int lane = threadIdx.x & 31;
  DistillShared<W>& sh = all[team];
  uint32_t* bits = all_bits + team * words;
  const int rank = W == 8 ? blockIdx.x % split : 0;
  const int64_t row = W == 8 ? blockIdx.x / split : static_cast<int64_t>(blockIdx.x) * kTeams + team;
  if (row >= n) return;  // a whole team
  const T* x = logits + row * ld;
  const RowFrame<T> frame(x, c, rank, W == 8 ? split : 1);
  const int rounds = frame.template rounds<L>(kThreads);
  const float scale = kLog2e * it.hi;

  Pack<T, V> q[L];
  Ring<T, kThreads> ring(frame, dynamic + team * ring_bytes<T>(kThreads), tid);
  for (int i = tid; i < words; i += kThreads) bits[i] = 0;
  if (tid == 0) sh.bad = sh.dup = sh.distinct = 0;
  team_sync<W>();
  for (int e = tid; e < te.k; e += kThreads) {
    int64_t idx = teacher_index(te, row, e);
    const float v = teacher_value(te, row, e);
    if (idx < 0 || v == -INFINITY) idx = -1;
    if (idx >= c) {
      atomicOr(&sh.bad, 1);
      idx = -1;
    }
    sh.index[e] = idx;
    sh.value[e] = v;
    if (idx >= 0) {
      const int f = static_cast<int>(idx) + frame.shift;
      const uint32_t bit = 1u << (f & 31);
      if (atomicOr(bits + (f >> 5), bit) & bit) atomicOr(&sh.dup, 1);
      else atomicAdd(&sh.distinct, 1);
      sh.x[e] = to_f(x[idx]);
    }
  }
  team_sync<W>();
  // the values of a granule that is not whole or of a whole one, kept classes as -inf
  F2 v[V / 2];
  const auto drop_kept = [&](int g) {
    const uint32_t mine = (bits[(g * V) >> 5] >> ((g * V) & 31)) & ((1u << V) - 1u);
    if (mine != 0) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if ((mine >> (2 * i)) & 1u) v[i].x = -INFINITY;
        if ((mine >> (2 * i + 1)) & 1u) v[i].y = -INFINITY;
      }
    }
  };
  const int edge = tid == 0 ? frame.head : tid == 1 ? frame.tail : -1;
  const Pack<T, V> ends = frame.edge(edge, -INFINITY);
  float most = -INFINITY;
  ring.template read<kRingRounds - 2>(q, frame.g0 + tid, -INFINITY);
#pragma unroll
  for (int u = 0; u < L; ++u) {
    const int g = frame.g0 + tid + kThreads * u;
    unpack(q[u], v);
    if (g < frame.g1) drop_kept(g);
    most = max_nan(most, max_of(v));
  }
  unpack(ends, v);
  if (edge >= 0) drop_kept(edge);
  const float ends_top = max_of(v);
  float start = warp_max(max_nan(most, ends_top));  // skips NaN
  if (start != start) start = -INFINITY;
  if (W > 1) {
    if (lane == 0) sh.part[tid >> 5].m = start;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) start = fmaxf(start, sh.part[w].m);
  }
  Stream<T, false> sums(start, scale);
  sums.add(v, ends_top, scale);
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    ring.next();
    ring.template read<kRingRounds - 1>(q, frame.g0 + tid + kThreads * L * k, -INFINITY);
    ring.advance();
#pragma unroll
    for (int u = 0; u < L; ++u) {
      const int g = frame.g0 + tid + kThreads * (k * L + u);
      unpack(q[u], v);
      if (g < frame.g1) drop_kept(g);
      sums.add(v, max_of(v), scale);
    }
  }
  Sums rest{sums.m, sums.total_s(scale), sums.cnt, 0.0f};
  rest = join_warp<T>(rest, scale);
  if (W > 1) {
    __syncthreads();  // part was read above
    if (lane == 0) sh.part[tid >> 5] = rest;
    __syncthreads();
    if (tid < 32)
      rest = join_warp<T>(lane < W ? sh.part[lane] : Sums{-INFINITY, 0.0f, 0.0f, 0.0f}, scale);
  }
  if (W == 8 && split > 1) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) sh.sums = rest;
    cluster.sync();
    if (rank == 0 && tid < 32)
      rest = join_warp<T>(lane < split ? cluster.map_shared_rank(&sh, lane)->sums
                                       : Sums{-INFINITY, 0.0f, 0.0f, 0.0f}, scale);
    cluster.sync();  // the others' shared memory is read above
    if (rank != 0) return;
  }
  if (tid >= 32) return;
  // one warp finishes the row: the kept classes of the student, the teacher
  const bool dup = sh.dup != 0;
  const auto first_of = [&](int e) {  // of the entries of a class, by its place
    if (!dup) return true;
    for (int i = 0; i < e; ++i)
      if (sh.index[i] == sh.index[e]) return false;
    return true;
  };
  Sums kept{-INFINITY, 0.0f, 0.0f, 0.0f};
  float tmax = -INFINITY, xmax = -INFINITY;
  for (int e = lane; e < te.k; e += 32) {
    if (sh.index[e] < 0) continue;
    xmax = fmaxf(xmax, sh.x[e]);
    tmax = fmaxf(tmax, sh.value[e]);
  }
  DistillRow r;
  r.tmax = warp_max(tmax);
  kept.m = warp_max(xmax);
  float tsum = 0.0f, tcnt = 0.0f;
  double mass = 0.0;
  for (int e = lane; e < te.k; e += 32) {
    if (sh.index[e] < 0) continue;
    if (first_of(e)) {
      if (sh.x[e] == kept.m) kept.cnt += 1.0f;
      else kept.s += expf(scaled(sh.x[e] - kept.m, it));
    }
    const float tv = sh.value[e];
    if (bucket) mass += exp(static_cast<double>(tv));
    else if (tv == r.tmax) tcnt += 1.0f;
    else tsum += expf(scaled(tv - r.tmax, it));
  }
  kept.s = warp_sum(kept.s);
  kept.cnt = warp_sum(kept.cnt);
  r.tlog = log1pf(warp_sum(tsum) + (warp_sum(tcnt) - 1.0f));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(kFullMask, mass, o);
  const RowStat st =
      row_stat(join_warp<T>(lane == 0 ? rest : lane == 1 ? kept : Sums{-INFINITY, 0.0f, 0.0f, 0.0f},
                            scale));
  r.m = st.m;
  r.logs = st.m == INFINITY ? __int_as_float(0x7fffffff) : log1pf(st.s);
  rest.m = __shfl_sync(kFullMask, rest.m, 0);
  const float rest_log = log1pf(rest.s + (rest.cnt - 1.0f));
  const float mass_r = bucket ? rest_mass(mass, sh.distinct == c, r.w1) : (r.w1 = 0.0f);
  const float ts = term_scale(temperature);
  float sum = 0.0f;
  for (int e = lane; e < te.k; e += 32) {
    if (sh.index[e] < 0) continue;
    const double lq = log_q(sh.value[e], r, bucket, it);
    const double lp = (static_cast<double>(sh.x[e]) - r.m) * it.full - static_cast<double>(r.logs);
    sum += entry_term(lq, lp, first_of(e), ts);
  }
  sum = warp_sum(sum);
  if (lane == 0)
    finish_row(r, sum, mass_r, rest.m, rest_log, it, bucket, sh.distinct == 0, sh.bad != 0, dup,
               temperature, loss + row, stats ? stats + row * kDsStats : nullptr);
}

// Rows of more than kNarrowMax classes, a warp per share of a row.  4096 x 32768
// bf16, 64 kept: 119 us, 4.5 TB/s, 104 with 5; bound by latency and by the kept
// classes' arithmetic in 64 bits.
template <typename T>
__global__ void __launch_bounds__(kMapThreads, 4)
distill_wide_bwd_kernel(int64_t n, int64_t c, const T* __restrict__ logits, int64_t ld, Teacher te,
                        float temperature, InvT it, int bucket, const float* __restrict__ stats,
                        const float* __restrict__ g_loss, int64_t g_stride, int split, int warps,
                        T* __restrict__ grad) {
  static_assert(kDsMaxKept <= 256, "entries are bytes");
  __shared__ uint8_t entries[kMapThreads / 32][kDsMaxKept];
  const MapPlace at(warps);
  if (at.row >= n || at.rank >= split) return;  // a whole warp
  const int64_t row = at.row;
  const T* x = logits + row * ld;
  T* out = grad + row * c;
  const RowShare<T> share(x, out, c, at.rank, split);
  // the kept classes of this share, gathered so that few lanes' worth of arithmetic
  // in 64 bits is issued once; before the row, as these loads wait no longer than
  // those of its statistics (30000 x 2000 float32, 100 kept: 113 us, 120 behind it)
  uint8_t* mine = entries[threadIdx.x >> 5];
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int e0 = 0; e0 < te.k; e0 += 32) {
    const bool here = e0 + lane < te.k && share.holds(teacher_index(te, row, e0 + lane)) &&
                      teacher_value(te, row, e0 + lane) != -INFINITY;
    const unsigned who = __ballot_sync(kFullMask, here);
    if (here) mine[count + __popc(who & ((1u << lane) - 1u))] = static_cast<uint8_t>(e0 + lane);
    count += __popc(who);
  }
  __syncwarp();
  const DistillRow r = load_row(stats + row * kDsStats);
  const float g = g_loss[row * g_stride] * temperature;
  if (r.kind == 2.0f || g == 0.0f || (r.m == -INFINITY && r.logs == r.logs)) {
    share.template run<false>([](auto& v) {
#pragma unroll
      for (auto& p : v) p = both(0.0f);
    });
    return;
  }
  const F2 f = both(g * r.spread);
  const float base = r.base(bucket), base_log = r.base_log(bucket);
  const OneStep one(base, base_log, kLog2e * it.hi);
  if (sizeof(T) == 2 && one.near()) {
    const F2 scale = both(kLog2e * it.hi), shift = both(one.shift);
    const F2 f2 = both(f.x * exp2_hw(one.left));
    share.template run<true>([&](auto& v) {
#pragma unroll
      for (auto& p : v) {
        const F2 a = fma2(p, scale, shift);
        p = mul2(F2{exp2_hw(a.x), exp2_hw(a.y)}, f2);
      }
    });
  } else {
    share.template run<true>([&](auto& v) {
#pragma unroll
      for (auto& p : v) {
        const F2 d = add2(p, both(-base));
        F2 a{scaled(d.x, it) - base_log, scaled(d.y, it) - base_log};
        a = F2{max_nan(a.x, kExpFloor), max_nan(a.y, kExpFloor)};
        p = mul2(exp_neg2<T>(a, kLog2e), f);
      }
    });
  }
  __syncwarp();  // orders the writes above before those below
  for (int i = lane; i < count; i += 32) {
    const int idx0 = static_cast<int>(teacher_index(te, row, mine[i]));
    const float v0 = teacher_value(te, row, mine[i]);
    const double lp = (static_cast<double>(to_f(x[idx0])) - r.m) * it.full - static_cast<double>(r.logs);
    out[idx0] = from_f<T>(g * kept_gradient(te, row, idx0, v0, lp, r, bucket, it));
  }
}

// Rows of at most E G classes, a group of G lanes per row (class_rows.cuh).
// The kept classes of a row are bits in shared memory; lane l takes the
// teacher's entries l, l + G, ...  169343 x 47 float32, 5 kept: 33 us, 1.5 TB/s,
// bound by issue (71% of the slots): the 64-bit arithmetic and the logarithms of
// 5 entries and a row weigh as much as its 47 classes.
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
  const int own = c - lane;
  const float scale = kLog2e * it.hi, floor = exp_floor(scale);
  F2 v[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    v[i].x = 2 * i * G < own ? to_f(x[lane + 2 * i * G]) : -INFINITY;
    v[i].y = (2 * i + 1) * G < own ? to_f(x[lane + (2 * i + 1) * G]) : -INFINITY;
  }
  // The lane's entries, the first two of them held: class (-1: absent, -2: wrong),
  // value and logit.
  struct Entry {
    int idx;
    float v, x;
  };
  const auto load_entry = [&](int e) {
    Entry t{-1, -INFINITY, 0.0f};
    if (e < te.k) {
      const int64_t idx = teacher_index(te, row, e);
      t.v = teacher_value(te, row, e);
      t.idx = idx < 0 || t.v == -INFINITY ? -1 : idx >= c ? -2 : static_cast<int>(idx);
      if (t.idx >= 0) t.x = to_f(x[t.idx]);
    }
    return t;
  };
  const Entry first_entry = load_entry(lane), second_entry = load_entry(lane + G);
  const auto entry = [&](int e) {
    return e == lane ? first_entry : e == lane + G ? second_entry : load_entry(e);
  };
  for (int i = lane; i < kWords; i += G) bits[i] = 0;
  __syncwarp();
  // teacher: kept classes, maximum
  bool bad = false, dup = false;
  float tmax = -INFINITY;
  float distinct = 0.0f;
  for (int e = lane; e < te.k; e += G) {
    const Entry t = entry(e);
    bad |= t.idx == -2;
    if (t.idx < 0) continue;
    const uint32_t bit = 1u << (t.idx & 31);
    const bool first = !(atomicOr(bits + (t.idx >> 5), bit) & bit);
    dup |= !first;
    distinct += first ? 1.0f : 0.0f;
    tmax = fmaxf(tmax, t.v);
  }
  const unsigned mine = group_mask<G>();
  bad = __ballot_sync(kFullMask, bad) & mine;
  dup = __ballot_sync(kFullMask, dup) & mine;
  __syncwarp();
  distinct = group_sum<G>(distinct);
  DistillRow r;
  r.tmax = group_max<G>(tmax);
  // log sum, or the sum of probabilities
  float tsum = 0.0f, tcnt = 0.0f;
  double mass = 0.0;
  for (int e = lane; e < te.k; e += G) {
    const Entry t = entry(e);
    if (t.idx < 0) continue;
    if (bucket) mass += exp(static_cast<double>(t.v));
    else if (t.v == r.tmax) tcnt += 1.0f;
    else tsum += expf(scaled(t.v - r.tmax, it));
  }
  r.tlog = log1pf(group_sum<G>(tsum) + (group_sum<G>(tcnt) - 1.0f));
  // student: the sums over the classes that are not kept and over the kept ones,
  // relative to their own maxima: that of the rest may be far below the row's
  float m = -INFINITY, m_rest = -INFINITY;
  uint32_t kept_here = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float vi = i % 2 == 0 ? v[i / 2].x : v[i / 2].y;
    const int j = lane + G * i;
    m = fmaxf(m, vi);
    if ((bits[j >> 5] >> (j & 31)) & 1u) kept_here |= 1u << i;
    else m_rest = fmaxf(m_rest, vi);
  }
  m = group_max<G>(m);
  m_rest = group_max<G>(m_rest);
  float s_rest = 0.0f, c_rest = 0.0f, s_kept = 0.0f, c_kept = 0.0f;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const bool kx = (kept_here >> (2 * i)) & 1u, ky = (kept_here >> (2 * i + 1)) & 1u;
    const float rx = kx ? m : m_rest, ry = ky ? m : m_rest;
    const bool px = v[i].x == rx, py = v[i].y == ry;  // a maximum's e^0 is counted, not added
    F2 d = add2(v[i], F2{-rx, -ry});
    d = F2{px ? 0.0f : max_nan(d.x, floor), py ? 0.0f : max_nan(d.y, floor)};
    const F2 e = exp_neg2<T>(d, scale);
    const float ex = px ? 0.0f : e.x, ey = py ? 0.0f : e.y;
    const float ox = px && 2 * i * G < own ? 1.0f : 0.0f;
    const float oy = py && (2 * i + 1) * G < own ? 1.0f : 0.0f;
    s_kept += (kx ? ex : 0.0f) + (ky ? ey : 0.0f);
    c_kept += (kx ? ox : 0.0f) + (ky ? oy : 0.0f);
    s_rest += (kx ? 0.0f : ex) + (ky ? 0.0f : ey);
    c_rest += (kx ? 0.0f : ox) + (ky ? 0.0f : oy);
  }
  s_rest = group_sum<G>(s_rest);
  c_rest = group_sum<G>(c_rest);
  s_kept = group_sum<G>(s_kept);
  c_kept = group_sum<G>(c_kept);
  r.m = m;
  // the sum of both relative to m, without one of its maxima
  const bool low = m_rest < m;
  const float fall = low ? scaled(m_rest - m, it) : 0.0f;
  const float s = low ? s_kept + (c_kept - 1.0f) + (s_rest + c_rest) * expf(fall)
                      : s_kept + s_rest + (c_kept + c_rest - 1.0f);
  r.logs = m == INFINITY ? __int_as_float(0x7fffffff) : log1pf(s);
  const float rest_log = log1pf(s_rest + (c_rest - 1.0f));
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) mass += __shfl_xor_sync(kFullMask, mass, o);
  const float mass_r =
      bucket ? rest_mass(mass, distinct == static_cast<float>(c), r.w1) : (r.w1 = 0.0f);
  const float ts = term_scale(temperature);
  float sum = 0.0f;
  for (int e = lane; e < te.k; e += G) {
    const Entry t = entry(e);
    if (t.idx < 0) continue;
    bool first = true;
    if (dup)  // the first of equal entries by its place
      for (int q = 0; q < e && first; ++q)
        first = teacher_index(te, row, q) != t.idx || teacher_value(te, row, q) == -INFINITY;
    const double lq = log_q(t.v, r, bucket, it);
    const double lp = (static_cast<double>(t.x) - m) * it.full - static_cast<double>(r.logs);
    sum += entry_term(lq, lp, first, ts);
  }
  sum = group_sum<G>(sum);
  if (live && lane == 0) finish_row(r, sum, mass_r, m_rest, rest_log, it, bucket,
                                    distinct == 0.0f, bad, dup, temperature, loss + row,
                                    stats ? stats + row * kDsStats : nullptr);
}

// 169343 x 47 float32, 5 kept: 21 us, 4.0 TB/s from L2 and DRAM, bound by issue and
// the latency of the entries.
template <typename T, int G, int E>
__global__ void __launch_bounds__(kNarrowThreads)
distill_narrow_bwd_kernel(int64_t n, int c, const T* __restrict__ logits, int64_t ld, Teacher te,
                          float temperature, InvT it, int bucket,
                          const float* __restrict__ stats, const float* __restrict__ g_loss,
                          int64_t g_stride, T* __restrict__ grad) {
  __shared__ __align__(16) T piece[E * kNarrowThreads];
  constexpr int kRows = kNarrowThreads / G;
  const int lane = threadIdx.x & (G - 1);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  const int64_t row = first + threadIdx.x / G < n ? first + threadIdx.x / G : n - 1;
  const T* x = logits + row * ld;
  T* out = piece + threadIdx.x / G * c;
  const int own = c - lane;
  F2 v[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    v[i].x = 2 * i * G < own ? to_f(x[lane + 2 * i * G]) : 0.0f;
    v[i].y = (2 * i + 1) * G < own ? to_f(x[lane + (2 * i + 1) * G]) : 0.0f;
  }
  const DistillRow r = load_row(stats + row * kDsStats);
  const float g = g_loss[row * g_stride] * temperature;
  const bool zero = r.kind == 2.0f || g == 0.0f || (r.m == -INFINITY && r.logs == r.logs);
  const F2 f = both(g * r.spread), shift = both(-r.base_log(bucket));
  const float base = r.base(bucket);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const F2 d = add2(v[i], both(-base));
    F2 a = add2(F2{scaled(d.x, it), scaled(d.y, it)}, shift);
    a = F2{max_nan(a.x, kExpFloor), max_nan(a.y, kExpFloor)};
    const F2 w = mul2(exp_neg2<T>(a, kLog2e), f);
    if (2 * i * G < own) out[lane + 2 * i * G] = from_f<T>(zero ? 0.0f : w.x);
    if ((2 * i + 1) * G < own) out[lane + (2 * i + 1) * G] = from_f<T>(zero ? 0.0f : w.y);
  }
  __syncwarp();  // orders the writes above before those below
  if (!zero) {
    for (int e = lane; e < te.k; e += G) {
      const int64_t idx = teacher_index(te, row, e);
      const float tv = teacher_value(te, row, e);
      if (idx < 0 || idx >= c || tv == -INFINITY) continue;
      const double lp = (static_cast<double>(to_f(x[idx])) - r.m) * it.full -
                        static_cast<double>(r.logs);
      out[idx] = from_f<T>(g * kept_gradient(te, row, idx, tv, lp, r, bucket, it));
    }
  }
  write_piece(grad + first * c, piece, (n - first < kRows ? n - first : kRows) * c);
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
  CIGN_REQUIRE(temperature >= 1e-3f && temperature <= 1e6f, CIGN_ERR_INVALID_ARGUMENT,
               "%s: temperature must be between 1e-3 and 1e6", name);
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
  const int words = static_cast<int>((c + 15) / 32 + 1);  // a bit per element of the frame
  const int64_t granules = c * type_size(x_type) / 16;
  int warps = wide_warps(n, granules);
  if (warps == 1 && c > 8192) warps = 4;  // four rows' bits would crowd out blocks
  CIGN_TYPE_DISPATCH(x_type, T, {
    const T* x = static_cast<const T*>(logits);
    const auto kernel = warps == 1   ? distill_wide_fwd_kernel<T, 1>
                        : warps == 4 ? distill_wide_fwd_kernel<T, 4>
                                     : distill_wide_fwd_kernel<T, 8>;
    const size_t smem = ring_bytes<T>(warps == 8 ? 256 : 128) +
                        static_cast<size_t>(words) * 4 * (warps == 1 ? 4 : 1);
    if (smem > 40960)  // more than a kernel has by default, beside its own 5 KB
      CIGN_CHECK_CUDA(
          cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(ring_bytes<T>(256) + kDsMaxClasses / 8 + 64)),
          "distill_fwd: shared memory");
    const int split = warps == 8 ? wide_split(n, granules, 256) : 1;
    return launch_cluster(kernel, static_cast<unsigned>(warps == 1 ? (n + 3) / 4 : n * split),
                          warps == 8 ? 256 : 128, smem, split, s, "distill_wide_fwd_kernel", n, c,
                          x, ld, te, temperature, inverse(temperature), tail, split, words, loss,
                          stats);
  });
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
    CIGN_TYPE_DISPATCH(x_type, T, CIGN_GROUP_DISPATCH(c,
        distill_narrow_bwd_kernel<T, G, E><<<narrow_grid(n, G), kNarrowThreads, 0, s>>>(
            n, static_cast<int>(c), static_cast<const T*>(logits), ld, te, temperature,
            inverse(temperature), tail, stats, grad_loss, grad_loss_stride,
            static_cast<T*>(grad_logits))));
    CIGN_CHECK_LAUNCH("distill_narrow_bwd_kernel");
    return CIGN_OK;
  }
  const MapGrid m = map_grid(n, c * type_size(x_type) / 16 + 2);
  CIGN_TYPE_DISPATCH(x_type, T,
      distill_wide_bwd_kernel<T><<<m.grid, kMapThreads, 0, s>>>(
          n, c, static_cast<const T*>(logits), ld, te, temperature, inverse(temperature), tail,
          stats, grad_loss, grad_loss_stride, m.split, m.warps, static_cast<T*>(grad_logits)));
  CIGN_CHECK_LAUNCH("distill_wide_bwd_kernel");
  return CIGN_OK;
}

}  // extern "C"

// Log probabilities of given classes, entropy and best classes of the rows of
// a logit matrix, and the gradient of the logits.  With m the row's maximum,
// s = sum e^(x - m) - 1 and t = sum e^(x - m) (x - m) (class_rows.cuh):
//   log p_j = (x_j - m) - log1p(s),   H = log1p(s) - t / (1 + s)
// and with the upstream gradients gl (label y), gh (entropy) and gt_i (best
// class idx_i), G = gl + sum_i gt_i and a_j = gl [j = y] + sum_i gt_i [j = idx_i]:
//   grad_j = a_j - p_j G - gh p_j (log p_j + H)
// Where a_j is not zero, a_j - p_j G is formed as (a_j - G) - G expm1(log p_j),
// which keeps its digits for p_j near 1.
#include <cooperative_groups.h>

#include "class_rows.cuh"

namespace cign {
namespace {

constexpr int kLpMaxTop = 64;

struct LogProbOut {
  float* log_prob;
  float* entropy;
  float* stats;  // [n, 2]: m, log1p(s)
  float* top_log_probs;
  int64_t* top_index;
};

// log1p(s); NaN for a row that holds +inf, as it has no distribution.
__device__ __forceinline__ float stat_log(const RowStat& a) {
  return a.m == INFINITY ? __int_as_float(0x7fffffff) : log1pf(a.s);
}
// Every class of the row is masked (-inf): nothing is left to distribute.
__device__ __forceinline__ bool stat_nothing(const RowStat& a) {
  return a.m == -INFINITY && a.s == a.s;
}
__device__ __forceinline__ float log_prob_of(float x, float m, float logs) {
  return m == -INFINITY ? (logs == logs ? -INFINITY : logs) : (x - m) - logs;
}

__device__ __forceinline__ void write_row(const LogProbOut& out, int64_t row, const RowStat& a,
                                          int64_t y, float xy, int64_t c) {
  const float logs = stat_log(a);
  if (out.stats) *reinterpret_cast<float2*>(out.stats + 2 * row) = make_float2(a.m, logs);
  if (out.entropy) out.entropy[row] = stat_nothing(a) ? 0.0f : logs - a.t / (1.0f + a.s);
  if (out.log_prob) {
    float lp = 0.0f;
    if (y >= c) lp = __int_as_float(0x7fffffff);
    else if (y >= 0) lp = log_prob_of(xy, a.m, logs);
    out.log_prob[row] = lp;
  }
}

// Team of W warps per row; with W = 8 a cluster of blocks may share a row.
constexpr int kLpKept = 128;  // classes that a warp keeps at most before it sorts them out
constexpr int kLpSlots = 16;  // shares of a thread's part of the row
template <int W>
struct alignas(16) WideShared {
  static constexpr int kThreads = 32 * W;
  static constexpr int kSets = W == 1 ? 128 : kThreads;
  uint32_t most[kSets];             // value keys of maxima
  float slot[kLpSlots][kThreads];   // the maximum of each thread's shares
  alignas(16) uint64_t kept[W][kLpKept];  // a warp's classes that may be among the best, in no order
  uint64_t sorted[kLpMaxTop];
  int count[W];
  uint32_t floor;  // value key that top_k classes at least reach
  Sums part[W];
  Sums sums;
};
static_assert(offsetof(WideShared<1>, kept) % 16 == 0 && offsetof(WideShared<4>, kept) % 16 == 0 &&
              offsetof(WideShared<8>, kept) % 16 == 0 && kLpKept % 2 == 0, "read in pairs");

// Reduces a warp's `count` keys to the best top_k, in order.  A key's place is
// the number of larger ones.
__device__ __noinline__ void reduce_kept(uint64_t* list, int count, int top_k) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  uint64_t k[kLpKept / 32];
  int place[kLpKept / 32];
#pragma unroll
  for (int i = 0; i < kLpKept / 32; ++i) {
    k[i] = 32 * i + lane < count ? list[32 * i + lane] : 0;
    place[i] = 0;
  }
  for (int j = 0; j < count; ++j) {
    const uint64_t o = list[j];
#pragma unroll
    for (int i = 0; i < kLpKept / 32; ++i) place[i] += o > k[i] ? 1 : 0;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kLpKept / 32; ++i)
    if (32 * i + lane < count && place[i] < top_k) list[place[i]] = k[i];
  __syncwarp();
}

// A warp's classes that may be among the best: keys above `last`.
struct Kept {
  uint64_t* list;
  uint64_t last;
  int count;
  __device__ __forceinline__ void add(uint64_t key, bool valid, int top_k) {
    const int lane = threadIdx.x & 31;
    const bool take = valid && key > last;
    const unsigned who = __ballot_sync(kFullMask, take);
    if (take) list[count + __popc(who & ((1u << lane) - 1u))] = key;
    count += __popc(who);
    if (count > kLpKept - 32) {
      reduce_kept(list, count, top_k);
      if (count >= top_k) {
        count = top_k;
        last = list[top_k - 1];
      }
    }
  }
};

// The top_k largest of the warps' kept keys, sorted.
template <int W>
__device__ __forceinline__ void sort_best(WideShared<W>& sh, int count, int top_k, int tid) {
  const int lane = threadIdx.x & 31, warp = tid >> 5;
  uint64_t* list = sh.kept[warp];
  if (lane == 0) {
    sh.count[warp] = count;
    if (count % 2 == 1) list[count] = 0;  // read in pairs
  }
  team_sync<W>();
  for (int i = lane; i < count; i += 32) {
    const uint64_t k = list[i];
    int place = 0;
    for (int w = 0; w < W; ++w) {
      const int others = sh.count[w];
      for (int j = 0; j < others; j += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.kept[w][j]);
        place += (o.x > k ? 1 : 0) + (o.y > k ? 1 : 0);
      }
    }
    if (place < top_k) sh.sorted[place] = k;
  }
}

// The floor of the best classes: the top_k-th largest maximum of disjoint sets
// of classes is reached by top_k classes.  With B the number of sets, about
// top_k (1 + top_k / 2 B) classes reach it, so B is at least twice top_k where
// that is to be had: the sets are those of the threads joined (their threads
// share the comparisons), or with one warp parts of the threads' sets.
template <int W>
__device__ __forceinline__ void find_floor(WideShared<W>& sh, float most, int slots, int top_k,
                                           int tid) {
  constexpr int kThreads = 32 * W;
  if (W > 1 || top_k <= 16) {
    uint32_t mine = value_key(most);
    int sets = kThreads;
    while (sets > 32 && sets / 2 >= 2 * top_k) sets /= 2;
    const int join = kThreads / sets;  // at most 8 neighbouring lanes
    for (int o = 1; o < join; o <<= 1) mine = max(mine, __shfl_xor_sync(kFullMask, mine, o));
    if (tid % join == 0) sh.most[tid / join] = mine;
    team_sync<W>();
    const int share = sets / join;
    int above = 0;
    for (int j = tid % join * share; j < (tid % join + 1) * share; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(sh.most + j);
      above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
    }
    for (int o = 1; o < join; o <<= 1) above += __shfl_xor_sync(kFullMask, above, o);
    if (above < top_k && tid % join == 0) atomicMin(&sh.floor, mine);
  } else {
    constexpr int kParts = WideShared<W>::kSets / kThreads;
    uint32_t mine[kParts];
    int above[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      float m = -INFINITY;
      for (int i = p; i < slots; i += kParts) m = max_nan(m, sh.slot[i][tid]);
      mine[p] = value_key(m);
      above[p] = 0;
      sh.most[p * kThreads + tid] = mine[p];
    }
    team_sync<W>();
    for (int j = 0; j < WideShared<W>::kSets; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(sh.most + j);
#pragma unroll
      for (int p = 0; p < kParts; ++p)
        above[p] += (o.x > mine[p]) + (o.y > mine[p]) + (o.z > mine[p]) + (o.w > mine[p]);
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      if (above[p] < top_k) atomicMin(&sh.floor, mine[p]);
  }
  team_sync<W>();
}

// 4096 x 32768 bf16: 71 us, 3.8 TB/s; 2048 x 32768 float32: 65 us, 4.1 TB/s;
// 2048 x 65537 bf16 with 20 best classes: 88 us, 3.1 TB/s.  Bound by issue (65%
// of the slots, DRAM 38-46%): per pair of logits two conversions, one fma for the
// exponents, two exponentials, an add and an fma for the sums, and the compares
// of the maximum.  3 x 100003 float32 with 8 best classes, eight blocks to a row:
// 12 us, latency.
// One pass over the row.  The first loads of all threads give the team's
// maximum, from which the sums start.  A thread also notes the maxima of up to
// 16 shares of what it reads; after the pass these give a floor for the best
// classes, and only the few shares that reach it are read again.
template <typename T, int W, bool TOP>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 8 ? 4 : 8)
log_probs_wide_fwd_kernel(int64_t n, int64_t c, const T* __restrict__ logits, int64_t ld,
                          const int64_t* __restrict__ labels, int top_k, int split,
                          LogProbOut out) {
  constexpr int V = RowFrame<T>::V;
  constexpr int L = kWideLoads<T>;
  constexpr int kTeams = W == 1 ? 4 : 1;
  constexpr int kThreads = 32 * W;
  extern __shared__ __align__(16) unsigned char ring_slots[];
  __shared__ WideShared<W> all[kTeams];
  const int team = W == 1 ? threadIdx.x >> 5 : 0;
  const int tid = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int lane = threadIdx.x & 31;
  WideShared<W>& sh = all[team];
  const int rank = W == 8 ? blockIdx.x % split : 0;
  const int64_t row = W == 8 ? blockIdx.x / split : static_cast<int64_t>(blockIdx.x) * kTeams + team;
  if (row >= n) return;  // a whole team
  const T* x = logits + row * ld;
  const RowFrame<T> frame(x, c, rank, W == 8 ? split : 1);
  const int rounds = frame.template rounds<L>(kThreads);

  Pack<T, V> q[L];
  F2 v[V / 2];
  Ring<T, kThreads> ring(frame, ring_slots + team * ring_bytes<T>(kThreads), tid);
  // the two ends of the row, by the first two threads
  const int edge = tid == 0 ? frame.head : tid == 1 ? frame.tail : -1;
  const Pack<T, V> ends = frame.edge(edge, -INFINITY);
  float most = -INFINITY;
  ring.template read<kRingRounds - 2>(q, frame.g0 + tid, -INFINITY);
#pragma unroll
  for (int u = 0; u < L; ++u) {
    unpack(q[u], v);
    most = max_nan(most, max_of(v));
  }
  unpack(ends, v);
  const float ends_top = max_of(v);
  most = max_nan(most, ends_top);
  float start = warp_max(most);  // skips NaN
  if (start != start) start = -INFINITY;
  if (TOP && tid == 0) sh.floor = 0xffffffffu;
  if (W > 1) {
    if (lane == 0) sh.part[tid >> 5].m = start;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) start = fmaxf(start, sh.part[w].m);
  }

  Stream<T, true> sums(start, kLog2e);
  sums.add(v, ends_top, kLog2e);
  const int per_slot = (rounds + kLpSlots - 1) / kLpSlots;  // rounds of a share
  float share = -INFINITY;
  int slots = 0, rest = per_slot;
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    ring.next();
    ring.template read<kRingRounds - 1>(q, frame.g0 + tid + kThreads * L * k, -INFINITY);
    ring.advance();
#pragma unroll
    for (int u = 0; u < L; ++u) {
      unpack(q[u], v);
      const float top = max_of(v);
      sums.add(v, top, kLog2e);
      if (TOP) share = max_nan(share, top);
    }
    if (TOP && (--rest == 0 || k + 1 == rounds)) {
      sh.slot[slots++][tid] = share;
      most = max_nan(most, share);
      share = -INFINITY;
      rest = per_slot;
    }
  }

  Sums a{sums.m, sums.total_s(kLog2e), sums.cnt, sums.total_t(kLog2e)};
  a = join_warp<T>(a, kLog2e);
  if (W > 1) {
    __syncthreads();  // part was read above
    if (lane == 0) sh.part[tid >> 5] = a;
    __syncthreads();
    // the first warp goes on with the sums
    if (tid < 32)
      a = join_warp<T>(lane < W ? sh.part[lane] : Sums{-INFINITY, 0.0f, 0.0f, 0.0f}, kLog2e);
  }
  if (TOP) {
    find_floor<W>(sh, most, slots, top_k, tid);
    const uint32_t floor_key = *const_cast<volatile uint32_t*>(&sh.floor);
    const float floor = key_value(floor_key);
    Kept kept{sh.kept[tid >> 5], floor_key ? (static_cast<uint64_t>(floor_key) << 32) - 1 : 0, 0};
    if (tid < 32) {  // the ends
      const int f = (lane < V ? frame.head : frame.tail) * V + lane % V;
      const bool in = lane < 2 * V && f >= 0 && frame.inside(f);
      kept.add(in ? class_key(to_f(frame.base[f]), f - frame.shift) : 0, in, top_k);
    }
    for (int i = 0; i < slots; ++i) {
      unsigned who = __ballot_sync(kFullMask, !(sh.slot[i][tid] < floor));
      while (who) {
        const int from = (tid & ~31) + __ffs(who) - 1;
        who &= who - 1;
        for (int k = i * per_slot; k < (i + 1) * per_slot && k < rounds; ++k) {
          const int g = frame.g0 + from + kThreads * (k * L + lane / V);
          const bool in = lane < L * V && g < frame.g1;
          const int f = in ? g * V + lane % V : frame.shift;  // behind the row it could pass 32 bits
          kept.add(in ? class_key(to_f(frame.base[f]), f - frame.shift) : 0, in, top_k);
        }
      }
    }
    sort_best<W>(sh, kept.count, top_k, tid);
  }
  if (W == 8 && split > 1) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) sh.sums = a;
    cluster.sync();
    if (rank == 0) {
      if (tid < 32)
        a = join_warp<T>(lane < split ? cluster.map_shared_rank(&sh, lane)->sums
                                      : Sums{-INFINITY, 0.0f, 0.0f, 0.0f}, kLog2e);
      if (TOP) {  // warp r takes what block r found
        const int r = tid >> 5;
        __syncthreads();
        for (int i = lane; i < top_k && r < split; i += 32)
          sh.kept[r][i] = cluster.map_shared_rank(&sh, r)->sorted[i];
        __syncthreads();
        sort_best<W>(sh, r < split ? top_k : 0, top_k, tid);
      }
    }
    cluster.sync();  // the others' shared memory is read above
    if (rank != 0) return;
  }
  const RowStat st = row_stat(a);
  if (tid == 0) {
    const int64_t y = out.log_prob ? labels[row] : -1;
    write_row(out, row, st, y, y >= 0 && y < c ? to_f(x[y]) : 0.0f, c);
  }
  if (TOP) {
    if (tid == 0) sh.sums = Sums{st.m, stat_log(st), 0.0f, 0.0f};
    team_sync<W>();
    for (int i = tid; i < top_k; i += kThreads) {
      const uint64_t k = sh.sorted[i];
      out.top_index[row * top_k + i] = key_index(k);
      out.top_log_probs[row * top_k + i] =
          log_prob_of(key_value(static_cast<uint32_t>(k >> 32)), sh.sums.m, sh.sums.s);
    }
  }
}

// The best top_k classes of a narrow row by their keys (0: no class), for more
// than a few.  The top_k-th largest key is found by bisection, counting the
// larger ones of the group; it starts at the least of the maxima of top_k sets of
// classes at least, and ends early where exactly top_k keys are above.  Those
// classes go to `list`, and a class's place is the number of larger ones.  About
// as long as 4 rounds over the registers where a warp has one row, 5 with two and
// 10 with four, whose bisections go on until the last is done; with eight and more
// the rounds are faster up to top_k = 20 and as fast at 40 (40M float32 logits,
// select and rounds in us: 512 classes, 5 best 118 and 124, 64 best 184 and 943;
// 200, 10 best 170 and 238; 100, 10 best 235 and 233, 20 best 290 and 402; 47, 20
// best 336 and 334, 40 best 512 and 614; 30, 10 best 319 and 189).
constexpr bool narrow_selects(int G) { return G >= 8; }
constexpr int narrow_rounds(int G) { return 80 / G > 4 ? 80 / G : 4; }
template <int G, int E>
struct NarrowBest {
  static constexpr int kMost = G * E < kLpMaxTop ? G * E : kLpMaxTop;
  static constexpr int kStride = kMost + 1;  // groups read from other banks
  static constexpr int kOwn = kMost / G;     // entries of a lane
  // f(place, key) for the lane's entries of the best
  template <typename F>
  __device__ __forceinline__ static void run(const uint32_t (&key)[E], uint32_t most, int top_k,
                                             uint64_t* list, F&& f) {
    const int lane = threadIdx.x & (G - 1);
    constexpr uint32_t kNone = 0x007ffffeu;  // below the key of -inf
    uint32_t sets[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < E; ++i) sets[i * 4 / E] = max(sets[i * 4 / E], key[i]);
    uint32_t lo = 0;
    if (top_k <= G) {
      lo = max(max(sets[0], sets[1]), max(sets[2], sets[3]));
    } else if (top_k <= 2 * G) {
      lo = min(max(sets[0], sets[1]), max(sets[2], sets[3]));
    } else if (top_k <= 4 * G) {
      lo = min(min(sets[0], sets[1]), min(sets[2], sets[3]));
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) lo = min(lo, __shfl_xor_sync(kFullMask, lo, o));
    lo = max(lo, kNone + 1) - 1;
    // more than or exactly top_k keys are above lo, `above` < top_k above hi
    uint32_t hi = most;
    int above = 0;
    while (__any_sync(kFullMask, hi - lo > 1)) {
      const uint32_t mid = lo + (hi - lo) / 2;
      int count = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) count += key[i] > mid ? 1 : 0;
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) count += __shfl_xor_sync(kFullMask, count, o);
      if (hi - lo > 1) {
        if (count > top_k) {
          lo = mid;
        } else {
          hi = mid;
          above = count;
          if (count == top_k) lo = mid;  // found
        }
      }
    }
    // the classes above hi, then those at it by their index until top_k are there
    const unsigned group = group_mask<G>(), before = group & ((1u << (threadIdx.x & 31)) - 1u);
    int larger = 0, equal = above;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool gt = key[i] > hi, eq = key[i] == hi;
      const unsigned who_gt = __ballot_sync(kFullMask, gt), who_eq = __ballot_sync(kFullMask, eq);
      const int at = gt ? larger + __popc(who_gt & before) : equal + __popc(who_eq & before);
      if ((gt || eq) && at < top_k)
        list[at] = (static_cast<uint64_t>(key[i]) << 32) | static_cast<uint32_t>(~(lane + G * i));
      larger += __popc(who_gt & group);
      equal += __popc(who_eq & group);
    }
    __syncwarp();
    uint64_t mine[kOwn];
    int place[kOwn];
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      mine[r] = r * G + lane < top_k ? list[r * G + lane] : 0;
      place[r] = 0;
    }
    for (int j = 0; j < top_k; ++j) {
      const uint64_t o = list[j];
#pragma unroll
      for (int r = 0; r < kOwn; ++r)
        if (r * G < top_k) place[r] += o > mine[r] ? 1 : 0;
    }
#pragma unroll
    for (int r = 0; r < kOwn; ++r)
      if (r * G + lane < top_k) f(place[r], mine[r]);
  }
};

// Rows of at most E G classes, a group of G lanes per row (class_rows.cuh).
// 2.45M x 47 float32: 117 us, 4.4 TB/s, bound by issue and the latency of the loads,
// which a prefetching persistent grid did not change.
// One best class is where the maximum is; a few go by rounds over the registers,
// each E compares and 2 log2 G shuffles, and more by NarrowBest.  A kernel of its
// own for each, as together they take 64 registers (100000 x 400, none: 48 us
// with 32 registers, 55 with 48; one best: 58 us by the maximum, 88 by a round).
enum Best { kNoBest, kOneBest, kRounds, kSelect };
template <typename T, int G, int E, Best BEST>
__global__ void __launch_bounds__(kNarrowThreads)
log_probs_narrow_fwd_kernel(int64_t n, int c, const T* __restrict__ logits, int64_t ld,
                            const int64_t* __restrict__ labels, int top_k, LogProbOut out) {
  const int lane = threadIdx.x & (G - 1);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (kNarrowThreads / G) + threadIdx.x / G;
  const bool live = at < n;
  const int64_t row = live ? at : n - 1;  // the last warp's idle groups follow along
  const T* x = logits + row * ld;
  const int own = c - lane;  // this lane has every G-th of so many classes
  F2 v[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    v[i].x = 2 * i * G < own ? to_f(x[lane + 2 * i * G]) : -INFINITY;
    v[i].y = (2 * i + 1) * G < own ? to_f(x[lane + (2 * i + 1) * G]) : -INFINITY;
  }
  const int64_t y = out.log_prob ? labels[row] : -1;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) m = fmaxf(m, fmaxf(v[i].x, v[i].y));
  m = group_max<G>(m);
  F2 s2{0.0f, 0.0f}, cnt2{0.0f, 0.0f}, t2{0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    F2 d = add2(v[i], both(-m));  // NaN where all are -inf; t is not used there
    d = F2{max_nan(d.x, kExpFloor), max_nan(d.y, kExpFloor)};
    const F2 e = exp_neg2<T>(d, kLog2e);
    // the maximum's e^0 is counted, not added
    cnt2 = add2(cnt2, F2{v[i].x == m ? 1.0f : 0.0f, v[i].y == m ? 1.0f : 0.0f});
    s2 = add2(s2, F2{v[i].x == m ? 0.0f : e.x, v[i].y == m ? 0.0f : e.y});
    t2 = fma2(e, d, t2);
  }
  RowStat a;
  a.m = m;
  a.s = group_sum<G>(s2.x + s2.y) + (group_sum<G>(cnt2.x + cnt2.y) - 1.0f);
  a.t = group_sum<G>(t2.x + t2.y);
  if (live && lane == 0) write_row(out, row, a, y, y >= 0 && y < c ? to_f(x[y]) : 0.0f, c);
  if constexpr (BEST == kNoBest) return;
  const float logs = stat_log(a);
  const bool has_nan = a.s != a.s;  // which m skips
  if constexpr (BEST == kOneBest) {
    // the best class is where the maximum is, or the first NaN
    uint32_t j = 0xffffffffu;
#pragma unroll
    for (int i = E - 1; i >= 0; --i)
      if ((i % 2 == 0 ? v[i / 2].x : v[i / 2].y) == m) j = lane + G * i;
    if (has_nan) {  // rarely: not worth registers
      j = 0xffffffffu;
#pragma unroll 1
      for (int i = E - 1; i >= 0; --i) {
        const float xi = i * G < own ? to_f(x[lane + i * G]) : 0.0f;
        if (xi != xi) j = lane + G * i;
      }
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) j = min(j, __shfl_xor_sync(kFullMask, j, o));
    if (live && lane == 0) {
      out.top_index[row] = j;
      out.top_log_probs[row] = has_nan ? logs : log_prob_of(m, m, logs);
    }
    return;
  }
  uint32_t key[E];  // 0 = not there or taken
#pragma unroll
  for (int i = 0; i < E; ++i)
    key[i] = i * G < own ? value_key(i % 2 == 0 ? v[i / 2].x : v[i / 2].y) : 0u;
  if constexpr (BEST == kSelect) {
    using Select = NarrowBest<G, E>;
    __shared__ uint64_t lists[kNarrowThreads / G * Select::kStride];
    Select::run(key, has_nan ? 0xffffffffu : value_key(m), top_k,
              lists + threadIdx.x / G * Select::kStride, [&](int place, uint64_t k) {
                if (!live) return;
                out.top_index[row * top_k + place] = key_index(k);
                out.top_log_probs[row * top_k + place] =
                    log_prob_of(key_value(static_cast<uint32_t>(k >> 32)), m, logs);
              });
    return;
  }
  for (int k = 0; k < top_k; ++k) {  // the best class of what is left
    uint32_t best = 0, at_i = 0;
#pragma unroll
    for (int i = E - 1; i >= 0; --i)
      if (key[i] >= best) {
        best = key[i];
        at_i = i;
      }
    uint32_t most = best;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(kFullMask, most, o));
    uint32_t j = best == most ? lane + G * at_i : 0xffffffffu;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) j = min(j, __shfl_xor_sync(kFullMask, j, o));
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (j == static_cast<uint32_t>(lane + G * i)) key[i] = 0;
    if (live && lane == k % G) {
      out.top_index[row * top_k + k] = j;
      out.top_log_probs[row * top_k + k] = log_prob_of(key_value(most), m, logs);
    }
  }
}

struct LogProbGrads {
  const float* log_prob;  // element r at r * stride; NULL = no such gradient
  int64_t log_prob_stride;
  const float* entropy;
  int64_t entropy_stride;
  const float* top;  // [n, top_k] contiguous
};

// What reaches a row: the sum G of the gradients of its log probabilities, the
// entropy's, and whether there is any at all.
struct RowGrads {
  int64_t y;
  float gl, gh, all, H;
  bool any;
};
__device__ __forceinline__ RowGrads row_grads(const LogProbGrads& g, const int64_t* labels,
                                              const float* entropy, int top_k, int64_t row,
                                              int64_t c) {
  RowGrads r;
  // no load waits for another
  const float gl = g.log_prob ? g.log_prob[row * g.log_prob_stride] : 0.0f;
  r.y = g.log_prob ? labels[row] : -1;
  r.gl = r.y >= 0 ? (r.y < c ? gl : __int_as_float(0x7fffffff)) : 0.0f;
  r.gh = g.entropy ? g.entropy[row * g.entropy_stride] : 0.0f;
  r.H = g.entropy ? entropy[row] : 0.0f;
  r.all = r.gl;
  r.any = !(r.gl == 0.0f) || !(r.gh == 0.0f);
  if (g.top)
    for (int i = 0; i < top_k; ++i) {
      const float v = g.top[row * top_k + i];
      r.all += v;
      r.any |= !(v == 0.0f);
    }
  return r;
}
// The gradient of a class that is the label or one of the best: a - p G - spread.
template <typename T>
__device__ __forceinline__ float special_grad(const LogProbGrads& g, const RowGrads& r,
                                              const int64_t* top_index, int top_k, int64_t row,
                                              int64_t j, float lp) {
  float a = j == r.y ? r.gl : 0.0f;
  if (g.top)
    for (int i = 0; i < top_k; ++i)
      if (top_index[row * top_k + i] == j) a += g.top[row * top_k + i];
  lp = max_nan(lp, kExpFloor);
  const float p = exp_neg2<T>(both(lp), kLog2e).x;
  return (a - r.all) + r.all * one_minus_exp(lp, p) - r.gh * p * (lp + r.H);
}

// The gradient of a block's rows is formed in shared memory and written as one
// piece, as the rows' own starts are not aligned.  2.45M x 47 float32: 194 us,
// 5.1 TB/s, bound by issue and the latency of the row's statistics and logits.  Five
// blocks to an SM, 48 registers a thread (100000 x 400: 61 us, 68 with four, 63 with
// six, which spill).
template <typename T, int G, int E>
__global__ void __launch_bounds__(kNarrowThreads, 5)
log_probs_narrow_bwd_kernel(int64_t n, int c, const T* __restrict__ logits, int64_t ld,
                            const int64_t* __restrict__ labels, const float* __restrict__ stats,
                            const float* __restrict__ entropy, int top_k,
                            const int64_t* __restrict__ top_index, LogProbGrads g,
                            T* __restrict__ grad) {
  __shared__ __align__(16) T piece[E * kNarrowThreads];
  constexpr int kRows = kNarrowThreads / G;
  const int lane = threadIdx.x & (G - 1);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  const int64_t row = first + threadIdx.x / G < n ? first + threadIdx.x / G : n - 1;
  const T* x = logits + row * ld;
  T* out = piece + threadIdx.x / G * c;
  const int own = c - lane;
  // the logits are asked for before it is known whether any gradient reaches
  // the row: waiting for that costs more than the reads it would save
  F2 v[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    v[i].x = 2 * i * G < own ? to_f(x[lane + 2 * i * G]) : 0.0f;
    v[i].y = (2 * i + 1) * G < own ? to_f(x[lane + (2 * i + 1) * G]) : 0.0f;
  }
  const float2 st = *reinterpret_cast<const float2*>(stats + 2 * row);
  const RowGrads r = row_grads(g, labels, entropy, top_k, row, c);
  // no gradient reaches the row, or it has no distribution
  const bool none = !r.any || (st.x == -INFINITY && st.y == st.y);
  // -p G - gh p (lp + H) = p (A + B lp)
  const F2 A = both(-(r.all + r.gh * r.H)), B = both(-r.gh);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    F2 lp = add2(add2(v[i], both(-st.x)), both(-st.y));
    lp = F2{max_nan(lp.x, kExpFloor), max_nan(lp.y, kExpFloor)};
    const F2 w = mul2(exp_neg2<T>(lp, kLog2e), fma2(B, lp, A));
    if (2 * i * G < own) out[lane + 2 * i * G] = from_f<T>(none ? 0.0f : w.x);
    if ((2 * i + 1) * G < own) out[lane + (2 * i + 1) * G] = from_f<T>(none ? 0.0f : w.y);
  }
  if (!none) {
    // the label and the best classes, by the lanes that wrote them above
    if (r.y >= 0 && r.y < c && (r.y & (G - 1)) == lane)
      out[r.y] = from_f<T>(special_grad<T>(g, r, top_index, top_k, row, r.y,
                                           (to_f(x[r.y]) - st.x) - st.y));
    if (g.top)
      for (int i = 0; i < top_k; ++i) {
        const int64_t j = top_index[row * top_k + i];
        if ((j & (G - 1)) == lane)
          out[j] = from_f<T>(special_grad<T>(g, r, top_index, top_k, row, j,
                                             (to_f(x[j]) - st.x) - st.y));
      }
  }
  write_piece(grad + first * c, piece, (n - first < kRows ? n - first : kRows) * c);
}

// Rows of more than kNarrowMax classes, a warp per share of a row. Each logit is
// read and each gradient written once: bound by memory where the logits are float32
// (2048 x 32768: 88 us, 6.1 TB/s).  Four blocks to an SM (64 registers a thread):
// 4096 x 32768 bf16 96 us, 5.6 TB/s; 109 us with the three that the compiler
// leaves by itself; five, which spill, 153.
template <typename T>
__global__ void __launch_bounds__(kMapThreads, 4)
log_probs_wide_bwd_kernel(int64_t n, int64_t c, const T* __restrict__ logits, int64_t ld,
                          const int64_t* __restrict__ labels, const float* __restrict__ stats,
                          const float* __restrict__ entropy, int top_k,
                          const int64_t* __restrict__ top_index, LogProbGrads g, int split,
                          int warps, T* __restrict__ grad) {
  const MapPlace at(warps);
  if (at.row >= n || at.rank >= split) return;  // a whole warp
  const int64_t row = at.row;
  const T* x = logits + row * ld;
  T* out = grad + row * c;
  const RowShare<T> share(x, out, c, at.rank, split);
  const float2 st = *reinterpret_cast<const float2*>(stats + 2 * row);
  const RowGrads r = row_grads(g, labels, entropy, top_k, row, c);
  // no gradient reaches the row, or it has no distribution
  if (!r.any || (st.x == -INFINITY && st.y == st.y)) {
    share.template run<false>([](auto& v) {
#pragma unroll
      for (auto& p : v) p = both(0.0f);
    });
    return;
  }
  // -p G - gh p (lp + H) = p (A + B lp)
  const F2 A = both(-(r.all + r.gh * r.H)), B = both(-r.gh);
  const OneStep one(st.x, st.y, kLog2e);
  if (sizeof(T) == 2 && one.near()) {
    // with the exponent's a = (lp / log 2) - left: p (A + B lp) = 2^a 2^left (A + B2 (a + left))
    const float back = exp2_hw(one.left), B1 = B.x * 0.693147181f;
    const F2 scale = both(kLog2e), shift = both(one.shift);
    const F2 B2 = both(B1 * back), A2 = both(fmaf(B1, one.left, A.x) * back);
    if (r.gh == 0.0f) {
      share.template run<true>([&](auto& v) {
#pragma unroll
        for (auto& p : v) {
          const F2 a = fma2(p, scale, shift);
          p = mul2(F2{exp2_hw(a.x), exp2_hw(a.y)}, A2);
        }
      });
    } else {
      share.template run<true>([&](auto& v) {
#pragma unroll
        for (auto& p : v) {
          F2 a = fma2(p, scale, shift);
          a = F2{max_nan(a.x, -160.0f), max_nan(a.y, -160.0f)};  // -inf: p = 0
          p = mul2(F2{exp2_hw(a.x), exp2_hw(a.y)}, fma2(B2, a, A2));
        }
      });
    }
  } else {
    share.template run<true>([&](auto& v) {
#pragma unroll
      for (auto& p : v) {
        F2 lp = add2(add2(p, both(-st.x)), both(-st.y));
        lp = F2{max_nan(lp.x, kExpFloor), max_nan(lp.y, kExpFloor)};
        p = mul2(exp_neg2<T>(lp, kLog2e), fma2(B, lp, A));
      }
    });
  }
  __syncwarp();  // orders the writes above before those below
  const int lane = threadIdx.x & 31;
  if (lane == 0 && r.y >= 0 && r.y < c && share.holds(r.y))
    out[r.y] = from_f<T>(special_grad<T>(g, r, top_index, top_k, row, r.y,
                                         (to_f(x[r.y]) - st.x) - st.y));
  if (g.top)
    for (int i = lane; i < top_k; i += 32) {
      const int64_t j = top_index[row * top_k + i];
      if (share.holds(j))
        out[j] = from_f<T>(special_grad<T>(g, r, top_index, top_k, row, j,
                                           (to_f(x[j]) - st.x) - st.y));
    }
}

int lp_check(int64_t n, int64_t c, int32_t x_type, int64_t ld, int32_t top_k, const char* name) {
  CIGN_REQUIRE(n >= 0 && c > 0, CIGN_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
  CIGN_REQUIRE(known_type(x_type), CIGN_ERR_INVALID_ARGUMENT, "%s: unknown element type", name);
  CIGN_REQUIRE(ld >= c, CIGN_ERR_INVALID_ARGUMENT, "%s: row stride below the class count", name);
  CIGN_REQUIRE(top_k >= 0 && top_k <= c, CIGN_ERR_INVALID_ARGUMENT,
               "%s: top_k must be between 0 and the class count", name);
  CIGN_REQUIRE(top_k <= kLpMaxTop, CIGN_ERR_UNSUPPORTED, "%s: top_k is at most %d", name,
               kLpMaxTop);
  CIGN_REQUIRE(n < (1ll << 31) && c <= kWideMax, CIGN_ERR_UNSUPPORTED,
               "%s: at most 2^31 - 1 rows of at most 2^31 - 1024 classes", name);
  return CIGN_OK;
}

}  // namespace
}  // namespace cign

using namespace cign;

extern "C" {

int cign_node_log_probs_fwd(int64_t n, int64_t c, int32_t x_type, const void* logits, int64_t ld,
                            const int64_t* labels, int32_t top_k, float* log_prob, float* entropy,
                            float* stats, float* top_log_probs, int64_t* top_index,
                            cign_stream_t stream) {
  int rc = lp_check(n, c, x_type, ld, top_k, "node_log_probs_fwd");
  if (rc) return rc;
  if (n == 0) return CIGN_OK;
  CIGN_REQUIRE(logits != nullptr && (log_prob == nullptr || labels != nullptr) &&
                   (top_k == 0 || (top_log_probs && top_index)),
               CIGN_ERR_NULL_POINTER, "node_log_probs_fwd: NULL argument");
  CIGN_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, CIGN_ERR_ALIGNMENT,
               "node_log_probs_fwd: stats must be 8-byte aligned");
  const LogProbOut out{log_prob, entropy, stats, top_log_probs, top_index};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c <= kNarrowMax) {
    CIGN_TYPE_DISPATCH(x_type, T, CIGN_GROUP_DISPATCH(c, {
      auto kernel = top_k > 1    ? log_probs_narrow_fwd_kernel<T, G, E, kRounds>
                    : top_k == 1 ? log_probs_narrow_fwd_kernel<T, G, E, kOneBest>
                                 : log_probs_narrow_fwd_kernel<T, G, E, kNoBest>;
      if constexpr (narrow_selects(G))
        if (top_k > narrow_rounds(G)) kernel = log_probs_narrow_fwd_kernel<T, G, E, kSelect>;
      kernel<<<narrow_grid(n, G), kNarrowThreads, 0, s>>>(
          n, static_cast<int>(c), static_cast<const T*>(logits), ld, labels, top_k, out);
    }));
    CIGN_CHECK_LAUNCH("log_probs_narrow_fwd_kernel");
    return CIGN_OK;
  }
  const int64_t granules = c * type_size(x_type) / 16;
  CIGN_TYPE_DISPATCH(x_type, T, {
    const T* x = static_cast<const T*>(logits);
    const int warps = wide_warps(n, granules);
    if (warps < 8) {
      const auto kernel = warps == 1 ? (top_k ? log_probs_wide_fwd_kernel<T, 1, true>
                                              : log_probs_wide_fwd_kernel<T, 1, false>)
                                     : (top_k ? log_probs_wide_fwd_kernel<T, 4, true>
                                              : log_probs_wide_fwd_kernel<T, 4, false>);
      kernel<<<static_cast<unsigned>(warps == 1 ? (n + 3) / 4 : n), 128, ring_bytes<T>(128), s>>>(
          n, c, x, ld, labels, top_k, 1, out);
    } else {
      const int split = wide_split(n, granules, 256);
      const auto kernel = top_k ? log_probs_wide_fwd_kernel<T, 8, true>
                                : log_probs_wide_fwd_kernel<T, 8, false>;
      CIGN_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(ring_bytes<T>(256))),
                      "node_log_probs_fwd: shared memory");
      return launch_cluster(kernel, static_cast<unsigned>(n * split), 256, ring_bytes<T>(256),
                            split, s,
                            "log_probs_wide_fwd_kernel", n, c, x, ld, labels, top_k, split, out);
    }
  });
  CIGN_CHECK_LAUNCH("log_probs_wide_fwd_kernel");
  return CIGN_OK;
}

int cign_node_log_probs_bwd(int64_t n, int64_t c, int32_t x_type, const void* logits, int64_t ld,
                            const int64_t* labels, const float* stats, const float* entropy,
                            int32_t top_k, const int64_t* top_index, const float* grad_log_prob,
                            int64_t grad_log_prob_stride, const float* grad_entropy,
                            int64_t grad_entropy_stride, const float* grad_top, void* grad_logits,
                            cign_stream_t stream) {
  int rc = lp_check(n, c, x_type, ld, top_k, "node_log_probs_bwd");
  if (rc) return rc;
  if (n == 0) return CIGN_OK;
  CIGN_REQUIRE(logits && stats && grad_logits && (!grad_log_prob || labels) &&
                   (!grad_entropy || entropy) && (!grad_top || top_index),
               CIGN_ERR_NULL_POINTER, "node_log_probs_bwd: NULL argument");
  CIGN_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, CIGN_ERR_ALIGNMENT,
               "node_log_probs_bwd: stats must be 8-byte aligned");
  const LogProbGrads g{grad_log_prob, grad_log_prob_stride, grad_entropy, grad_entropy_stride,
                       top_k > 0 ? grad_top : nullptr};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c <= kNarrowMax) {
    CIGN_TYPE_DISPATCH(x_type, T, CIGN_GROUP_DISPATCH(c,
        log_probs_narrow_bwd_kernel<T, G, E><<<narrow_grid(n, G), kNarrowThreads, 0, s>>>(
            n, static_cast<int>(c), static_cast<const T*>(logits), ld, labels, stats, entropy,
            top_k, top_index, g, static_cast<T*>(grad_logits))));
    CIGN_CHECK_LAUNCH("log_probs_narrow_bwd_kernel");
    return CIGN_OK;
  }
  const MapGrid m = map_grid(n, c * type_size(x_type) / 16 + 2);
  CIGN_TYPE_DISPATCH(x_type, T,
      log_probs_wide_bwd_kernel<T><<<m.grid, kMapThreads, 0, s>>>(
          n, c, static_cast<const T*>(logits), ld, labels, stats, entropy, top_k, top_index, g,
          m.split, m.warps, static_cast<T*>(grad_logits)));
  CIGN_CHECK_LAUNCH("log_probs_wide_bwd_kernel");
  return CIGN_OK;
}

}  // extern "C"

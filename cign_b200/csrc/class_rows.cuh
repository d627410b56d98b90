// Shared device code of the row operators over float32, bfloat16 and float16
// matrices (layer_norm.cu, node_log_probs.cu, distill.cu): element types and
// conversions, block reductions, and the running softmax statistics of a row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cign {

// ---------------------------------------------------------------- types
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);  // to nearest, ties to even
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

inline bool known_type(int32_t t) { return t == CIGN_F32 || t == CIGN_BF16 || t == CIGN_F16; }
inline size_t type_size(int32_t t) { return t == CIGN_F32 ? 4 : 2; }

// CALL with `T` bound to the element type named by the run-time code `TYPE`.
#define CIGN_TYPE_DISPATCH(TYPE, T, ...)                              \
  do {                                                                \
    if ((TYPE) == CIGN_F32) { using T = float; __VA_ARGS__; }         \
    else if ((TYPE) == CIGN_BF16) { using T = __nv_bfloat16; __VA_ARGS__; } \
    else { using T = __half; __VA_ARGS__; }                           \
  } while (0)

// V neighbouring elements as one load or store: 16 bytes, or one element.
template <typename T, int V>
struct Pack {
  static_assert(V == 1 || V * sizeof(T) == 16, "one element or 16 bytes");
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V == 1) {
    r.e[0] = *p;
  } else {
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
  if constexpr (V == 1) *p = v.e[0];
  else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
}
// Element i of a parameter vector of run-time type, `none` without one.
__device__ __forceinline__ float load_param(const void* p, int32_t type, int64_t i, float none) {
  if (p == nullptr) return none;
  if (type == CIGN_F32) return static_cast<const float*>(p)[i];
  if (type == CIGN_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f(static_cast<const __half*>(p)[i]);
}

// ---------------------------------------------------------------- block sums
// Sum of v over the block, in lane order then warp order (fixed, so runs
// repeat bit for bit); every thread gets it.  `part` holds one float per warp.
template <int WARPS>
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  __syncthreads();  // part may still be read from an earlier call
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) s += part[w];
  return s;
}

// Two float32 values of one lane, worked on by one instruction each (sm_100's
// f32x2 arithmetic): the row kernels are bound by the instructions they issue.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n"
      " add.rn.f32x2 r, p, q;\n mov.b64 {%0, %1}, r;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n"
      " mul.rn.f32x2 r, p, q;\n mov.b64 {%0, %1}, r;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("{\n .reg .b64 p, q, r, s;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n"
      " mov.b64 s, {%6, %7};\n fma.rn.f32x2 r, p, q, s;\n mov.b64 {%0, %1}, r;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ F2 both(float v) { return F2{v, v}; }
// The larger of two values, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The largest and the smallest of three.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float exp2_hw(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// e^(d / T) of two values d <= 0 by the hardware's 2^x, `scale` = log2(e) / T;
// below 2^-126 zero.  d must be finite (callers raise it to exp_floor(scale),
// where the result is 0).  For 16-bit logits the argument d scale is rounded to
// float32, which leaves a relative error of about |d| 2^-23: the terms of a
// softmax sum weigh e^d, and a gradient is rounded to 16 bits.  For float32
// logits what the rounding drops is put back, so that the small probabilities
// beside a sure class keep their digits.
constexpr float kLog2e = 1.44269504f;
__device__ __forceinline__ float exp_floor(float scale) { return -160.0f / scale; }
constexpr float kExpFloor = -160.0f / kLog2e;  // T = 1
template <typename T>
__device__ __forceinline__ F2 exp_neg2(F2 d, float scale) {
  const F2 t = mul2(d, both(scale));
  F2 e{exp2_hw(t.x), exp2_hw(t.y)};
  if constexpr (sizeof(T) == 4) {
    const F2 rest = fma2(d, both(scale), F2{-t.x, -t.y});
    e = fma2(mul2(e, both(0.693147181f)), rest, e);
  }
  return e;
}

// e^((x - m) / T - logs) of 16-bit logits as 2^(x scale + shift), one operation on
// the logit: the constant part -(m scale + logs log2(e)) is rounded to `shift`, and
// 2^left is a factor of what the exponentials are multiplied with.  A shift of 8192
// is rounded by 2^-12, which would be 2^-12.5 of a probability.
struct OneStep {
  float shift, left;
  __device__ __forceinline__ OneStep(float m, float logs, float scale) {
    const double s = -(static_cast<double>(m) * scale + static_cast<double>(logs) * 1.4426950408889634);
    shift = static_cast<float>(s);
    left = static_cast<float>(s - shift);
  }
  // far ones are not finite, or their left not small
  __device__ __forceinline__ bool near() const { return fabsf(shift) <= 8192.0f; }
};

// 1 - e^x for x <= 0, with its digits where x is near 0 (the series to x^8 is
// exact to float32 for x > -1/2); p = e^x is given.
__device__ __forceinline__ float one_minus_exp(float x, float p) {
  float h = fmaf(x, 1.0f / 8.0f, 1.0f);
  h = fmaf(h * x, 1.0f / 7.0f, 1.0f);
  h = fmaf(h * x, 1.0f / 6.0f, 1.0f);
  h = fmaf(h * x, 1.0f / 5.0f, 1.0f);
  h = fmaf(h * x, 1.0f / 4.0f, 1.0f);
  h = fmaf(h * x, 1.0f / 3.0f, 1.0f);
  h = fmaf(h * x, 1.0f / 2.0f, 1.0f);
  return x > -0.5f ? -h * x : 1.0f - p;
}

// ---------------------------------------------------------------- softmax
// Running statistics of the values seen so far, relative to their maximum m:
//   s = sum e^(x - m) - 1   (without the maximum's own e^0)
//   t = sum e^(x - m) (x - m)
// so lse = m + log1p(s) and the entropy is log1p(s) - t / (1 + s), a sum of
// two terms that are not negative.  Keeping the 1 out of the sum keeps the
// digits of log1p(s) where one class has nearly all of the probability.
// Nothing seen: m = -inf, s = -1.  Values -inf count as probability 0; a NaN
// makes s NaN.
struct RowStat {
  float m = -INFINITY, s = -1.0f, t = 0.0f;
};

// ---------------------------------------------------------------- narrow rows
// Rows of at most E G classes are held by a group of G lanes (a power of two),
// class lane + G i in register i < E: a row is read once, and the 32 / G rows
// of a warp are neighbours.  A row costs a warp E of its steps, the sums over
// the group, one logarithm and what is read once per row, so few lanes and many
// classes per lane are cheapest (2.45M x 47 float32 forward: 117 us with 4
// lanes, 166 with 8, 158 with 2, whose loads are too scattered).  Up to 512
// classes this beats a warp that streams the row (200000 rows of 512: forward
// 90 us and 143 in float32, 92 and 204 in bf16; of 1000: 209 and 199, 338 and
// 207).
constexpr int kNarrowThreads = 256;
constexpr int64_t kNarrowMax = 512;

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}
// The lanes of this lane's group, as a warp mask.
template <int G>
__device__ __forceinline__ unsigned group_mask() {
  if (G == 32) return kFullMask;
  return ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) & ~(G - 1));
}

inline unsigned narrow_grid(int64_t n, int G) {
  return static_cast<unsigned>((n + kNarrowThreads / G - 1) / (kNarrowThreads / G));
}

#define CIGN_GROUP_CASE(G_, E_, ...) \
  { constexpr int G = G_, E = E_; __VA_ARGS__; }
// CALL with `G` and `E` bound to the lanes and registers of a row of
// c <= kNarrowMax classes.
#define CIGN_GROUP_DISPATCH(c, ...)                            \
  do {                                                          \
    if ((c) <= 8) CIGN_GROUP_CASE(1, 8, __VA_ARGS__)            \
    else if ((c) <= 16) CIGN_GROUP_CASE(1, 16, __VA_ARGS__)     \
    else if ((c) <= 32) CIGN_GROUP_CASE(2, 16, __VA_ARGS__)     \
    else if ((c) <= 48) CIGN_GROUP_CASE(4, 12, __VA_ARGS__)     \
    else if ((c) <= 64) CIGN_GROUP_CASE(4, 16, __VA_ARGS__)     \
    else if ((c) <= 96) CIGN_GROUP_CASE(8, 12, __VA_ARGS__)     \
    else if ((c) <= 128) CIGN_GROUP_CASE(8, 16, __VA_ARGS__)    \
    else if ((c) <= 192) CIGN_GROUP_CASE(16, 12, __VA_ARGS__)   \
    else if ((c) <= 256) CIGN_GROUP_CASE(16, 16, __VA_ARGS__)   \
    else if ((c) <= 384) CIGN_GROUP_CASE(32, 12, __VA_ARGS__)   \
    else CIGN_GROUP_CASE(32, 16, __VA_ARGS__)                   \
  } while (0)

// The rows of a block of a kernel that writes rows: formed in shared memory
// (at most E kNarrowThreads elements), then written as one piece, 16 bytes per
// thread.  A block has a multiple of 8 rows, so its piece starts on 16 bytes if the
// matrix does.
template <typename T>
__device__ __forceinline__ void write_piece(T* out, const T* piece, int64_t count) {
  __syncthreads();
  constexpr int V = 16 / sizeof(T);
  if (reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    const int whole = static_cast<int>(count / V);
    for (int i = threadIdx.x; i < whole; i += kNarrowThreads)
      reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(piece)[i];
    for (int i = whole * V + threadIdx.x; i < count; i += kNarrowThreads) out[i] = piece[i];
  } else {
    for (int i = threadIdx.x; i < count; i += kNarrowThreads) out[i] = piece[i];
  }
}

// ---------------------------------------------------------------- ordering
// Classes are ordered by value, larger first (NaN before everything, as
// torch.sort orders it), and by index, smaller first: larger keys come first.
// -0 and +0 are equal.  0 is below every key.
__device__ __forceinline__ uint32_t value_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  if (v != v) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t class_key(float v, uint32_t index) {
  return (static_cast<uint64_t>(value_key(v)) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) {
  return ~static_cast<uint32_t>(key);
}
__device__ __forceinline__ float key_value(uint32_t u) {
  if (u == 0xffffffffu) return __int_as_float(0x7fffffff);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// ---------------------------------------------------------------- wide rows
// Rows of more than kNarrowMax classes are streamed by a team of W warps, 16
// aligned bytes per thread and load.  A row may start anywhere: granule g of
// V = 16 / sizeof(T) elements covers the row's elements g V - shift ..., and the
// two granules at its ends are read by elements.
// Granules of a thread that are worked on together.
template <typename T>
constexpr int kWideLoads = 4;
// Rounds of them that a streaming thread has in its own slots of shared memory
// (cp.async, no barriers: a thread reads only what it asked for).  Held there
// instead of in registers, the round that is under way leaves 64 registers to a
// thread and room for a third more warps (2048 x 65537 bf16 with 20 best
// classes: 87 us, 109 with registers; 95 with three rounds).
constexpr int kRingRounds = 2;
template <typename T>
__host__ __device__ constexpr size_t ring_bytes(int threads) {
  return static_cast<size_t>(kRingRounds) * kWideLoads<T> * 16 * threads;
}

// Classes: positions in a row are 32-bit, and loops step past its end by less than 1024.
constexpr int64_t kWideMax = (1ll << 31) - 1024;

template <typename T>
struct RowFrame {
  static constexpr int V = 16 / sizeof(T);
  const T* base;  // aligned address of granule 0, at most V - 1 elements before the row
  int shift;      // the row begins at element `shift` of the frame
  int end;        // and ends before this one
  int g0, g1;     // the whole granules of this team's share of the row
  int head, tail; // granules of the share that are not whole, or -1
  __device__ __forceinline__ RowFrame(const T* row, int64_t c, int rank, int split) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) % 16) / sizeof(T));
    base = row - shift;
    end = shift + static_cast<int>(c);
    const int granules = (end + V - 1) / V;
    g0 = split > 1 ? static_cast<int>(static_cast<int64_t>(granules) * rank / split) : 0;
    g1 = split > 1 ? static_cast<int>(static_cast<int64_t>(granules) * (rank + 1) / split)
                   : granules;
    head = g0 == 0 && shift > 0 ? g0++ : -1;
    tail = g1 == granules && end % V != 0 && g1 > g0 ? --g1 : -1;
  }
  __device__ __forceinline__ bool inside(int f) const { return f >= shift && f < end; }
  // A granule that is not whole, elements outside of the row as `outside`.
  __device__ __forceinline__ Pack<T, V> edge(int g, float outside) const {
    Pack<T, V> q;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int f = g * V + e;
      q.e[e] = g >= 0 && inside(f) ? base[f] : from_f<T>(outside);
    }
    return q;
  }
  // Thread `tid` of `threads` has the whole granules g0 + tid + threads (k L + u), u < L.
  template <int L>
  __device__ __forceinline__ int rounds(int threads) const {
    return (g1 - g0 + threads * L - 1) / (threads * L);
  }
  template <int L>
  __device__ __forceinline__ void load(Pack<T, V> (&q)[L], int k, int tid, int threads,
                                       float outside) const {
    const int g = g0 + tid + threads * L * k;
    const T* p = base + static_cast<int64_t>(g) * V;
    if (g - tid + threads * L <= g1) {  // all threads have all of them
#pragma unroll
      for (int u = 0; u < L; ++u) q[u] = load_pack<T, V>(p + u * threads * V);
    } else {
#pragma unroll
      for (int u = 0; u < L; ++u) {
        if (g + u * threads < g1) {
          q[u] = load_pack<T, V>(p + u * threads * V);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) q[u].e[e] = from_f<T>(outside);
        }
      }
    }
  }
};

// A thread's granules of a frame, round by round through shared memory.
template <typename T, int THREADS>
struct Ring {
  static constexpr int V = RowFrame<T>::V;
  static constexpr int L = kWideLoads<T>;
  uint32_t slots;  // this thread's first slot
  const T* ask;    // the first granule of the next round to ask for
  int ask_g, ask_slot, read_slot;
  int g1;
  __device__ __forceinline__ Ring(const RowFrame<T>& f, void* smem, int tid)
      : slots(smem_u32(smem) + 16 * tid), ask(f.base + static_cast<int64_t>(f.g0 + tid) * V),
        ask_g(f.g0 + tid), ask_slot(0), read_slot(0), g1(f.g1) {
#pragma unroll
    for (int k = 0; k < kRingRounds - 1; ++k) next();
  }
  __device__ __forceinline__ void next() {
#pragma unroll
    for (int u = 0; u < L; ++u)
      if (ask_g + u * THREADS < g1)
        cp_async16_s(slots + (ask_slot + u) * 16 * THREADS, ask + u * THREADS * V);
    cp_async_commit();
    ask += L * THREADS * V;
    ask_g += L * THREADS;
    ask_slot = ask_slot + L == kRingRounds * L ? 0 : ask_slot + L;
  }
  // The round at read_slot, whose first granule of this thread is g, with AHEAD
  // rounds asked for behind it.
  template <int AHEAD>
  __device__ __forceinline__ void read(Pack<T, V> (&q)[L], int g, float outside) {
    cp_async_wait<AHEAD>();
#pragma unroll
    for (int u = 0; u < L; ++u) {
      const float4 w = lds_f4(slots + (read_slot + u) * 16 * THREADS);
      q[u] = *reinterpret_cast<const Pack<T, V>*>(&w);
      if (g + u * THREADS >= g1) {
#pragma unroll
        for (int e = 0; e < V; ++e) q[u].e[e] = from_f<T>(outside);
      }
    }
  }
  __device__ __forceinline__ void advance() {
    read_slot = read_slot + L == kRingRounds * L ? 0 : read_slot + L;
  }
};

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& q, F2 (&v)[V / 2]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) v[i] = F2{to_f(q.e[2 * i]), to_f(q.e[2 * i + 1])};
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, 2 * N> pack_of(const F2 (&v)[N]) {
  Pack<T, 2 * N> q;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q.e[2 * i] = from_f<T>(v[i].x);
    q.e[2 * i + 1] = from_f<T>(v[i].y);
  }
  return q;
}
__device__ __forceinline__ float max_of(const F2 (&v)[2]) {
  return max3_nan(max_nan(v[0].x, v[0].y), v[1].x, v[1].y);
}
__device__ __forceinline__ float max_of(const F2 (&v)[4]) {
  return max3_nan(max3_nan(v[0].x, v[0].y, v[1].x), max3_nan(v[1].y, v[2].x, v[2].y),
                  max_nan(v[3].x, v[3].y));
}
__device__ __forceinline__ float min_of(const F2 (&v)[2]) {
  return min3_nan(min3_nan(v[0].x, v[0].y, v[1].x), v[1].y, INFINITY);
}
__device__ __forceinline__ float min_of(const F2 (&v)[4]) {
  return min3_nan(min3_nan(v[0].x, v[0].y, v[1].x), min3_nan(v[1].y, v[2].x, v[2].y),
                  min3_nan(v[3].x, v[3].y, INFINITY));
}

// One warp's share of a row, the rank-th of `split`, taken through f (which
// changes pairs of values in place) from x to out, both of c elements.  Whole
// granules where x and out start at the same place within 16 bytes; elements
// otherwise.
template <typename T>
struct RowShare {
  static constexpr int V = RowFrame<T>::V;
  static constexpr int L = kWideLoads<T>;
  RowFrame<T> frame;
  T* out;
  int first, last;  // elements [first, last) of the row
  __device__ __forceinline__ RowShare(const T* x, T* out, int64_t c, int rank, int split)
      : frame(x, c, rank, split), out(out) {
    first = (frame.head >= 0 ? frame.shift : frame.g0 * V) - frame.shift;
    last = (frame.tail >= 0 ? frame.end : frame.g1 * V) - frame.shift;
  }
  __device__ __forceinline__ bool holds(int64_t j) const { return j >= first && j < last; }
  template <bool READ, typename F>
  __device__ __forceinline__ void run(F&& f) const {
    const int lane = threadIdx.x & 31;
    const T* x = frame.base + frame.shift;
    if ((reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(out)) % 16 == 0) {
      T* o = out - frame.shift;
      const int edge = lane == 0 ? frame.head : lane == 1 ? frame.tail : -1;
      F2 v[V / 2];
      if (edge >= 0) {
        if (READ) unpack(frame.edge(edge, 0.0f), v);
        f(v);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (frame.inside(edge * V + e))
            o[edge * V + e] = from_f<T>(e % 2 == 0 ? v[e / 2].x : v[e / 2].y);
      }
      const int rounds = frame.template rounds<L>(32);
      Pack<T, V> q[L];
      for (int k = 0; k < rounds; ++k) {
        if (READ) frame.load(q, k, lane, 32, 0.0f);
#pragma unroll
        for (int u = 0; u < L; ++u) {
          const int g = frame.g0 + lane + 32 * (k * L + u);
          if (READ) unpack(q[u], v);
          f(v);
          if (g < frame.g1) store_pack<T, V>(o + static_cast<int64_t>(g) * V, pack_of<T>(v));
        }
      }
    } else {
      for (int j = first + lane; j - lane < last; j += 32 * 8) {
        F2 v[4];
        if (READ) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i].x = j + 64 * i < last ? to_f(x[j + 64 * i]) : 0.0f;
            v[i].y = j + 64 * i + 32 < last ? to_f(x[j + 64 * i + 32]) : 0.0f;
          }
        }
        f(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (j + 64 * i < last) out[j + 64 * i] = from_f<T>(v[i].x);
          if (j + 64 * i + 32 < last) out[j + 64 * i + 32] = from_f<T>(v[i].y);
        }
      }
    }
  }
};

// The grid of a kernel that takes rows through warps: a block of 8 warps has
// 8 / `split` rows, or one row (with blockIdx.y its next 8 shares).
constexpr int kMapThreads = 256;
struct MapGrid {
  int split, warps;  // shares of a row; warps of a block for one row: 1, 2, 4 or 8
  dim3 grid;
};
inline MapGrid map_grid(int64_t n, int64_t granules) {
  MapGrid m;
  // 16 granules per lane amortise what every share reads of its row (more where
  // the grid's second dimension would not hold the shares)
  const int64_t share = granules > 512ll * 8 * 65535 ? granules / (8 * 65535) + 1 : 512;
  m.split = static_cast<int>((granules + share - 1) / share);
  m.warps = 1;
  while (m.warps < 8 && m.warps < m.split) m.warps *= 2;
  m.grid = dim3(static_cast<unsigned>((n * m.warps + 7) / 8),
                static_cast<unsigned>((m.split + m.warps - 1) / m.warps));
  return m;
}
struct MapPlace {
  int64_t row;
  int rank;
  __device__ __forceinline__ explicit MapPlace(int warps) {
    const int w = threadIdx.x >> 5;
    row = static_cast<int64_t>(blockIdx.x) * (8 / warps) + w / warps;
    rank = blockIdx.y * warps + w % warps;
  }
};

template <int W>
__device__ __forceinline__ void team_sync() {
  if constexpr (W == 1) __syncwarp();
  else __syncthreads();
}

// Running sums of a thread over the values it has seen, relative to m:
//   s = sum over x < m of e^((x - m) / T),  cnt = how many x equal m,
//   t = sum of e^((x - m) / T) (x - m)
// with `scale` = log2(e) / T.  m may be any value that is not below what was
// seen: a thread starts with its team's maximum and meets larger ones rarely.
//
// 16-bit logits take the exponent x scale - m scale in one operation and sum
// e 2^x's argument instead of e (x - m); what the rounding of m scale leaves,
// the same factor in every term, is put back when the sums are read.  The
// kernels are bound by issue: each operation per logit counts.
template <typename T, bool ENTROPY>
struct Stream {
  static constexpr bool kOneStep = sizeof(T) == 2;
  float m, ref, cnt;  // ref = m but where m scale would overflow to -inf
  float shift;        // kOneStep: ref scale, rounded
  float floor;        // of x - m
  F2 s[2], u[2];      // two chains each; u: kOneStep: sum of e times the argument; else t
  __device__ __forceinline__ Stream(float start, float scale) : cnt(0.0f) {
    s[0] = s[1] = u[0] = u[1] = both(0.0f);
    floor = exp_floor(scale);
    set(start, scale);
  }
  __device__ __forceinline__ void set(float to, float scale) {
    m = to;
    ref = fmaxf(to, -1e30f);
    shift = ref * scale;
  }
  template <bool CLAMP, int N>
  __device__ __forceinline__ void sum(const F2 (&v)[N], float scale) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kOneStep) {
        F2 a = fma2(v[i], both(scale), both(-shift));
        if (CLAMP) a = F2{max_nan(a.x, -160.0f), max_nan(a.y, -160.0f)};
        const F2 e{exp2_hw(a.x), exp2_hw(a.y)};
        s[i % 2] = add2(s[i % 2], e);
        if (ENTROPY) u[i % 2] = fma2(e, a, u[i % 2]);
      } else {
        F2 d = add2(v[i], both(-ref));
        if (CLAMP) d = F2{max_nan(d.x, floor), max_nan(d.y, floor)};
        const F2 e = exp_neg2<T>(d, scale);
        s[i % 2] = add2(s[i % 2], e);
        if (ENTROPY) u[i % 2] = fma2(e, d, u[i % 2]);
      }
    }
  }
  // `most` = max_of(v); NaN makes s NaN.  Changes v.
  template <int N>
  __device__ __forceinline__ void add(F2 (&v)[N], float most, float scale) {
    if (most >= m) {
      if (most > m) raise(most, scale);
#pragma unroll
      for (int i = 0; i < N; ++i) {  // the maximum's e^0 is counted, not added
        if (v[i].x == m) { cnt += 1.0f; v[i].x = -INFINITY; }
        if (v[i].y == m) { cnt += 1.0f; v[i].y = -INFINITY; }
      }
    }
    // -inf would make 0 times inf of u; the arithmetic of finite values needs no floor
    if (min_of(v) - ref < floor) sum<true>(v, scale);
    else sum<false>(v, scale);
  }
  __device__ __forceinline__ static float all(const F2 (&p)[2]) {
    return (p[0].x + p[0].y) + (p[1].x + p[1].y);
  }
  __device__ __forceinline__ float total_s(float scale) const {
    return kOneStep ? all(s) * exp2_hw(left(scale)) : all(s);
  }
  __device__ __forceinline__ float total_t(float scale) const {
    const float r = left(scale);
    return kOneStep ? exp2_hw(r) * fmaf(r, all(s), all(u)) / scale : all(u);
  }
  // What rounding ref scale has left.  Where that is large, a 16-bit logit's
  // next lower value is 2^-11 of it and more below m: every term is 0.
  __device__ __forceinline__ float left(float scale) const {
    return fabsf(shift) < 4194304.0f ? -fmaf(ref, scale, -shift) : 0.0f;
  }
  __device__ __forceinline__ void raise(float to, float scale) {
    const float d = max_nan(m - to, floor);
    const float f = exp_neg2<T>(both(d), scale).x;
    float n = (total_s(scale) + cnt) * f;
    float w = ENTROPY ? fmaf(n, d, f * total_t(scale)) : 0.0f;
    set(to, scale);
    if (kOneStep) {  // as sums whose rounding is still to be put back
      const float r = left(scale), g = exp2_hw(-r);
      n *= g;
      w = g * (w * scale) - r * n;
    }
    s[0] = F2{n, 0.0f};
    u[0] = F2{w, 0.0f};
    s[1] = u[1] = both(0.0f);
    cnt = 0.0f;
  }
};

// The same of a whole team or row.  Disjoint sets join by raising the lower ones
// to the highest maximum.
struct Sums {
  float m, s, cnt, t;
};
// Over the warp; every lane gets it.  Lanes that hold nothing have m = -inf and
// zeros.
template <typename T>
__device__ __forceinline__ Sums join_warp(const Sums& a, float scale) {
  Sums r;
  r.m = warp_max(a.m);
  const bool top = a.m == r.m;
  const float d = max_nan(a.m - r.m, exp_floor(scale));
  const float f = top ? 1.0f : exp_neg2<T>(both(d), scale).x;
  const float n = top ? a.s : (a.s + a.cnt) * f;
  r.s = warp_sum(n);
  r.cnt = warp_sum(top ? a.cnt : 0.0f);
  r.t = warp_sum(top ? a.t : fmaf(n, d, f * a.t));
  return r;
}
// As RowStat (t stays relative to the unscaled differences).
__device__ __forceinline__ RowStat row_stat(const Sums& a) {
  RowStat r;
  r.m = a.m;
  r.s = a.s + (a.cnt - 1.0f);
  r.t = a.t;
  return r;
}

// Launch `kernel` with clusters of `cluster` blocks (1 to 8).
template <typename... Params, typename... Args>
int launch_cluster(void (*kernel)(Params...), unsigned grid, int threads, size_t smem, int cluster,
                   cudaStream_t s, const char* what, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(CIGN_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  }
  count_launch();
  return CIGN_OK;
}

// Warps of a team.  What a row costs each warp at its ends (the maxima, the
// sums, the barriers) is as much as about eight rounds of loads, so a team has
// no more warps than it takes to fill the device: single warps want two rows
// per resident warp to even out, or rows of at most 16 loads per lane (1500
// rows of 1000 bf16: 5 us, 10 with teams of four), teams of four one row per
// resident team (777 rows of 10007 fp16: 14 us, 21 with teams of eight).
inline int wide_warps(int64_t n, int64_t granules) {
  const int64_t sms = sm_count();
  if (n >= 48 * sms || granules < 64) return 1;
  if (n >= 4 * sms) return granules <= 512 ? 1 : 4;
  return granules < 256 ? 4 : 8;
}

// Blocks that share a row of `granules` where there are too few rows to fill
// the device: as many as leave every thread eight loads, at most 8.
inline int wide_split(int64_t n, int64_t granules, int threads) {
  int split = 1;
  while (split < 8 && n * split * 2 <= 2 * sm_count() &&
         granules >= static_cast<int64_t>(16) * split * threads)
    split *= 2;
  return split;
}

}  // namespace cign

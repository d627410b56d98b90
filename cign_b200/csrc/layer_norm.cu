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
#include "class_rows.cuh"

namespace cign {
namespace {

constexpr int kLnThreads = 256;
constexpr int kLnWarps = kLnThreads / 32;
constexpr int kLnRowsPerChunk = 64;  // rows of one partial sum of the parameter gradients

template <typename T, typename P>
__global__ void __launch_bounds__(kLnThreads)
layer_norm_fwd_kernel(int64_t n, int64_t d, const T* __restrict__ x, int64_t ldx,
                      const P* __restrict__ w, const P* __restrict__ b, float eps,
                      T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float part[kLnWarps];
  const float inv_d = 1.0f / static_cast<float>(d);
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.0f;
    for (int64_t j = threadIdx.x; j < d; j += kLnThreads) s += to_f(xr[j]);
    const float mu = block_sum<kLnWarps>(s, part) * inv_d;
    float v = 0.0f;
    for (int64_t j = threadIdx.x; j < d; j += kLnThreads) {
      const float a = to_f(xr[j]) - mu;
      v = fmaf(a, a, v);
    }
    const float rs = rsqrtf(block_sum<kLnWarps>(v, part) * inv_d + eps);
    if (threadIdx.x == 0 && mean != nullptr) {
      mean[row] = mu;
      rstd[row] = rs;
    }
    for (int64_t j = threadIdx.x; j < d; j += kLnThreads) {
      const float xh = (to_f(xr[j]) - mu) * rs;
      y[row * d + j] = from_f<T>(fmaf(xh, w ? to_f(w[j]) : 1.0f, b ? to_f(b[j]) : 0.0f));
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kLnThreads)
layer_norm_bwd_x_kernel(int64_t n, int64_t d, const T* __restrict__ gy, int64_t ldg,
                        const T* __restrict__ x, int64_t ldx, const P* __restrict__ w,
                        const float* __restrict__ mean, const float* __restrict__ rstd,
                        T* __restrict__ gx) {
  __shared__ float part[kLnWarps];
  const float inv_d = 1.0f / static_cast<float>(d);
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const T* xr = x + row * ldx;
    const T* gr = gy + row * ldg;
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t j = threadIdx.x; j < d; j += kLnThreads) {
      const float u = to_f(gr[j]) * (w ? to_f(w[j]) : 1.0f);
      s1 += u;
      s2 = fmaf(u, (to_f(xr[j]) - mu) * rs, s2);
    }
    s1 = block_sum<kLnWarps>(s1, part) * inv_d;
    s2 = block_sum<kLnWarps>(s2, part) * inv_d;
    for (int64_t j = threadIdx.x; j < d; j += kLnThreads) {
      const float u = to_f(gr[j]) * (w ? to_f(w[j]) : 1.0f);
      const float xh = (to_f(xr[j]) - mu) * rs;
      gx[row * d + j] = from_f<T>(rs * (u - s1 - xh * s2));
    }
  }
}

// Partial sums over one chunk of rows, rows in order; one thread per column.
template <typename T>
__global__ void __launch_bounds__(kLnThreads)
layer_norm_bwd_param_kernel(int64_t n, int64_t d, const T* __restrict__ gy, int64_t ldg,
                            const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean,
                            const float* __restrict__ rstd, float* __restrict__ pw,
                            float* __restrict__ pb) {
  const int64_t j = static_cast<int64_t>(blockIdx.y) * kLnThreads + threadIdx.x;
  if (j >= d) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kLnRowsPerChunk;
  const int64_t r1 = r0 + kLnRowsPerChunk < n ? r0 + kLnRowsPerChunk : n;
  float aw = 0.0f, ab = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = to_f(gy[r * ldg + j]);
    aw = fmaf(g, (to_f(x[r * ldx + j]) - mean[r]) * rstd[r], aw);
    ab += g;
  }
  pw[static_cast<int64_t>(blockIdx.x) * d + j] = aw;
  pb[static_cast<int64_t>(blockIdx.x) * d + j] = ab;
}

template <typename P>
__global__ void __launch_bounds__(kLnThreads)
layer_norm_param_sum_kernel(int64_t chunks, int64_t d, const float* __restrict__ pw,
                            const float* __restrict__ pb, P* __restrict__ gw,
                            P* __restrict__ gb) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kLnThreads + threadIdx.x;
  if (j >= d) return;
  float aw = 0.0f, ab = 0.0f;
  for (int64_t c = 0; c < chunks; ++c) {
    aw += pw[c * d + j];
    ab += pb[c * d + j];
  }
  if (gw) gw[j] = from_f<P>(aw);
  if (gb) gb[j] = from_f<P>(ab);
}

int64_t ln_chunks(int64_t n) { return (n + kLnRowsPerChunk - 1) / kLnRowsPerChunk; }

int ln_check(int64_t n, int64_t d, int32_t x_type, int32_t param_type, const char* name) {
  CIGN_REQUIRE(n >= 0 && d > 0, CIGN_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
  CIGN_REQUIRE(known_type(x_type) && known_type(param_type), CIGN_ERR_INVALID_ARGUMENT,
               "%s: unknown element type", name);
  CIGN_REQUIRE(n < (1ll << 31) && d < (1ll << 24), CIGN_ERR_UNSUPPORTED,
               "%s: at most 2^31 - 1 rows of at most 2^24 - 1 columns", name);
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
  CIGN_TYPE_DISPATCH(x_type, T, CIGN_TYPE_DISPATCH(param_type, P,
      layer_norm_fwd_kernel<T, P><<<static_cast<unsigned>(n), kLnThreads, 0, s>>>(
          n, d, static_cast<const T*>(x), ldx, static_cast<const P*>(w),
          static_cast<const P*>(b), eps, static_cast<T*>(y), mean, rstd)));
  CIGN_CHECK_LAUNCH("layer_norm_fwd_kernel");
  return CIGN_OK;
}

size_t cign_layer_norm_bwd_workspace_bytes(int64_t n, int64_t d) {
  if (n <= 0 || d <= 0) return 0;
  return 2 * static_cast<size_t>(ln_chunks(n)) * d * sizeof(float);
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
  const bool params = gw != nullptr || gb != nullptr;
  if (params) {
    const size_t need = cign_layer_norm_bwd_workspace_bytes(n, d);
    CIGN_REQUIRE(ws != nullptr && ws_bytes >= need, CIGN_ERR_INVALID_ARGUMENT,
                 "layer_norm_bwd: workspace too small (%zu < %zu bytes)", ws_bytes, need);
    CIGN_REQUIRE(aligned16(ws), CIGN_ERR_ALIGNMENT,
                 "layer_norm_bwd: ws must be 16-byte aligned");
  }
  if (gx) {
    CIGN_TYPE_DISPATCH(x_type, T, CIGN_TYPE_DISPATCH(param_type, P,
        layer_norm_bwd_x_kernel<T, P><<<static_cast<unsigned>(n), kLnThreads, 0, s>>>(
            n, d, static_cast<const T*>(gy), ldg, static_cast<const T*>(x), ldx,
            static_cast<const P*>(w), mean, rstd, static_cast<T*>(gx))));
    CIGN_CHECK_LAUNCH("layer_norm_bwd_x_kernel");
  }
  if (params) {
    const int64_t chunks = ln_chunks(n);
    float* pw = static_cast<float*>(ws);
    float* pb = pw + chunks * d;
    const unsigned cols = static_cast<unsigned>((d + kLnThreads - 1) / kLnThreads);
    CIGN_REQUIRE(cols < 65536, CIGN_ERR_UNSUPPORTED, "layer_norm_bwd: too many columns");
    CIGN_TYPE_DISPATCH(x_type, T,
        layer_norm_bwd_param_kernel<T><<<dim3(static_cast<unsigned>(chunks), cols), kLnThreads, 0,
                                          s>>>(n, d, static_cast<const T*>(gy), ldg,
                                               static_cast<const T*>(x), ldx, mean, rstd, pw, pb));
    CIGN_CHECK_LAUNCH("layer_norm_bwd_param_kernel");
    CIGN_TYPE_DISPATCH(param_type, P,
        layer_norm_param_sum_kernel<P><<<cols, kLnThreads, 0, s>>>(
            chunks, d, pw, pb, static_cast<P*>(gw), static_cast<P*>(gb)));
    CIGN_CHECK_LAUNCH("layer_norm_param_sum_kernel");
  }
  return CIGN_OK;
}

}  // extern "C"

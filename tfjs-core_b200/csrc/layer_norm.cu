// Layer normalisation over the inner-most axis and its gradients.
//
//   y = (x - m) r g + b,   m = mean(x),   r = 1 / sqrt(mean((x - m)^2) + eps)
//   with n = (x - m) r and a = dy g:
//   dx = r (a - mean(a) - n mean(a n)),   dg = sum over rows of dy n,   db = sum over rows of dy
//
// All sums are float32 or wider; a half-stored x is widened on load and y rounded once on store.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }

// Sum over the block; every thread gets it.  The order is fixed, so equal inputs give equal bits.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) v += scratch[w];
  return v;
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kThreads) layer_norm_kernel(const TX* __restrict__ x, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, TY* __restrict__ y,
                                                             float* __restrict__ stats, int64_t rows, int64_t width,
                                                             float epsilon) {
  __shared__ float scratch[kThreads / 32];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TX* r = x + row * width;
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < width; j += kThreads) s += load_f32(r + j);
    const float mean = block_sum(s, scratch) / (float)width;
    s = 0.f;
    for (int64_t j = threadIdx.x; j < width; j += kThreads) {
      const float d = load_f32(r + j) - mean;
      s += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(s, scratch) / (float)width + epsilon);
    for (int64_t j = threadIdx.x; j < width; j += kThreads) {
      float v = (load_f32(r + j) - mean) * rstd;
      if (gamma) v *= gamma[j];
      if (beta) v += beta[j];
      store_f32(y + row * width + j, v);
    }
    if (stats && threadIdx.x == 0) {
      stats[2 * row] = mean;
      stats[2 * row + 1] = rstd;
    }
  }
}

template <typename TD, typename TX>
__global__ void __launch_bounds__(kThreads) layer_norm_dx_kernel(const TD* __restrict__ dy, const TX* __restrict__ x,
                                                                const float* __restrict__ gamma,
                                                                const float* __restrict__ stats, float* __restrict__ dx,
                                                                int64_t rows, int64_t width) {
  __shared__ float scratch[kThreads / 32];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t at = row * width;
    const float mean = stats[2 * row], rstd = stats[2 * row + 1];
    float sa = 0.f, san = 0.f;
    for (int64_t j = threadIdx.x; j < width; j += kThreads) {
      const float a = load_f32(dy + at + j) * (gamma ? gamma[j] : 1.f);
      sa += a;
      san += a * ((load_f32(x + at + j) - mean) * rstd);
    }
    const float ma = block_sum(sa, scratch) / (float)width;
    const float man = block_sum(san, scratch) / (float)width;
    for (int64_t j = threadIdx.x; j < width; j += kThreads) {
      const float a = load_f32(dy + at + j) * (gamma ? gamma[j] : 1.f);
      const float n = (load_f32(x + at + j) - mean) * rstd;
      dx[at + j] = rstd * (a - ma - n * man);
    }
  }
}

// One thread a column, rows in order.
template <typename TD, typename TX>
__global__ void __launch_bounds__(32) layer_norm_dweights_kernel(const TD* __restrict__ dy, const TX* __restrict__ x,
                                                                const float* __restrict__ stats,
                                                                float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                int64_t rows, int64_t width) {
  for (int64_t j = blockIdx.x * 32 + threadIdx.x; j < width; j += gridDim.x * 32) {
    double sg = 0.0, sb = 0.0;
    for (int64_t row = 0; row < rows; row++) {
      const float d = load_f32(dy + row * width + j);
      sb += d;
      sg += d * ((load_f32(x + row * width + j) - stats[2 * row]) * stats[2 * row + 1]);
    }
    if (dgamma) dgamma[j] = (float)sg;
    if (dbeta) dbeta[j] = (float)sb;
  }
}

template <typename TX, typename TY>
void launch_forward(tfjs_cuda_ctx* ctx, const void* x, const float* gamma, const float* beta, void* y, float* stats,
                    int64_t rows, int64_t width, float epsilon) {
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  layer_norm_kernel<TX, TY><<<(unsigned)(rows < cap ? rows : cap), kThreads, 0, ctx->stream>>>(
      (const TX*)x, gamma, beta, (TY*)y, stats, rows, width, epsilon);
}

template <typename TD, typename TX>
int launch_backward(tfjs_cuda_ctx* ctx, const void* dy, const void* x, const float* gamma, const float* stats, float* dx,
                    float* dgamma, float* dbeta, int64_t rows, int64_t width) {
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  if (dx && rows) {
    layer_norm_dx_kernel<TD, TX><<<(unsigned)(rows < cap ? rows : cap), kThreads, 0, ctx->stream>>>(
        (const TD*)dy, (const TX*)x, gamma, stats, dx, rows, width);
    const int rc = post_launch(ctx, "layerNormBackprop (dx)");
    if (rc) return rc;
  }
  if (dgamma || dbeta) {
    const int64_t blocks = ceil_div64(width, 32);
    layer_norm_dweights_kernel<TD, TX><<<(unsigned)(blocks < 65535 ? blocks : 65535), 32, 0, ctx->stream>>>(
        (const TD*)dy, (const TX*)x, stats, dgamma, dbeta, rows, width);
    return post_launch(ctx, "layerNormBackprop (weights)");
  }
  return TFJS_CUDA_OK;
}

// A float32 operand of exactly `elems` values, not quantised; null for id 0.
int optional_vector(tfjs_cuda_ctx* ctx, tfjs_tensor_id id, int64_t elems, const char* what, TensorEntry** out) {
  *out = nullptr;
  if (!id) return TFJS_CUDA_OK;
  const int rc = get_f32(ctx, id, elems, what, out);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, !(*out)->quant.quantized, "%s cannot be a quantised tensor", what);
  TFJS_REQUIRE(ctx, (*out)->size == elems, "%s holds %lld elements, %lld expected", what, (long long)(*out)->size,
               (long long)elems);
  return TFJS_CUDA_OK;
}

int exact_activation(tfjs_cuda_ctx* ctx, tfjs_tensor_id id, int64_t elems, const char* what, TensorEntry** out) {
  const int rc = get_activation(ctx, id, elems, what, out);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, (*out)->size == elems, "%s holds %lld elements, %lld expected", what, (long long)(*out)->size,
               (long long)elems);
  return TFJS_CUDA_OK;
}

int check_extent(tfjs_cuda_ctx* ctx, int64_t rows, int64_t width) {
  TFJS_REQUIRE(ctx, rows >= 0 && width >= 0, "negative extent");
  TFJS_REQUIRE(ctx, width < (1ll << 31), "layerNorm: the normalised axis is too long");
  TFJS_REQUIRE(ctx, rows <= (1ll << 60) / (width > 2 ? width : 2), "layerNorm: too many elements");
  return TFJS_CUDA_OK;
}

const float* f32_ptr(const TensorEntry* t) { return t ? (const float*)t->ptr : nullptr; }
float* f32_out(TensorEntry* t) { return t ? (float*)t->ptr : nullptr; }

}  // namespace

extern "C" int tfjs_cuda_layer_norm(tfjs_cuda_ctx* ctx, tfjs_tensor_id x_id, tfjs_tensor_id gamma_id,
                                    tfjs_tensor_id beta_id, tfjs_tensor_id y_id, tfjs_tensor_id stats_id, int64_t rows,
                                    int64_t width, float epsilon) {
  if (!ctx) return TFJS_CUDA_ERR_INVALID_ARG;
  int rc = check_extent(ctx, rows, width);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, epsilon >= 0.f && epsilon - epsilon == 0.f, "layerNorm: epsilon must be finite and not negative");
  TensorEntry *x, *gamma, *beta, *y, *stats;
  if ((rc = exact_activation(ctx, x_id, rows * width, "x", &x))) return rc;
  if ((rc = optional_vector(ctx, gamma_id, width, "gamma", &gamma))) return rc;
  if ((rc = optional_vector(ctx, beta_id, width, "beta", &beta))) return rc;
  if ((rc = exact_activation(ctx, y_id, rows * width, "layerNorm output", &y))) return rc;
  if ((rc = optional_vector(ctx, stats_id, 2 * rows, "layerNorm statistics", &stats))) return rc;
  TFJS_REQUIRE(ctx, y != x && y != gamma && y != beta && y != stats && (!stats || (stats != x && stats != gamma && stats != beta)),
               "layerNorm: an output cannot be one of the inputs or another output");
  y->version++;
  if (stats) stats->version++;
  if (rows == 0 || (width == 0 && !stats)) return TFJS_CUDA_OK;
  cudaSetDevice(ctx->device);
  const bool hx = x->dtype == TFJS_F16, hy = y->dtype == TFJS_F16;
  auto launch = hx ? (hy ? launch_forward<__half, __half> : launch_forward<__half, float>)
                   : (hy ? launch_forward<float, __half> : launch_forward<float, float>);
  launch(ctx, x->ptr, f32_ptr(gamma), f32_ptr(beta), y->ptr, f32_out(stats), rows, width, epsilon);
  return post_launch(ctx, "layerNorm");
}

extern "C" int tfjs_cuda_layer_norm_backprop(tfjs_cuda_ctx* ctx, tfjs_tensor_id dy_id, tfjs_tensor_id x_id,
                                             tfjs_tensor_id gamma_id, tfjs_tensor_id stats_id, tfjs_tensor_id dx_id,
                                             tfjs_tensor_id dgamma_id, tfjs_tensor_id dbeta_id, int64_t rows,
                                             int64_t width) {
  if (!ctx) return TFJS_CUDA_ERR_INVALID_ARG;
  int rc = check_extent(ctx, rows, width);
  if (rc) return rc;
  TensorEntry *dy, *x, *gamma, *stats, *out[3];
  if ((rc = exact_activation(ctx, dy_id, rows * width, "dy", &dy))) return rc;
  if ((rc = exact_activation(ctx, x_id, rows * width, "x", &x))) return rc;
  if ((rc = optional_vector(ctx, gamma_id, width, "gamma", &gamma))) return rc;
  TFJS_REQUIRE(ctx, stats_id != 0, "layerNormBackprop needs the statistics of the forward pass");
  if ((rc = optional_vector(ctx, stats_id, 2 * rows, "layerNorm statistics", &stats))) return rc;
  if ((rc = optional_vector(ctx, dx_id, rows * width, "dx", &out[0]))) return rc;
  if ((rc = optional_vector(ctx, dgamma_id, width, "dgamma", &out[1]))) return rc;
  if ((rc = optional_vector(ctx, dbeta_id, width, "dbeta", &out[2]))) return rc;
  for (int i = 0; i < 3; i++) {
    if (!out[i]) continue;
    TFJS_REQUIRE(ctx, out[i] != dy && out[i] != x && out[i] != gamma && out[i] != stats && out[i] != out[(i + 1) % 3],
                 "layerNormBackprop: an output cannot be one of the inputs or another output");
    out[i]->version++;
  }
  if (width == 0) return TFJS_CUDA_OK;
  cudaSetDevice(ctx->device);
  const bool hd = dy->dtype == TFJS_F16, hx = x->dtype == TFJS_F16;
  auto launch = hd ? (hx ? launch_backward<__half, __half> : launch_backward<__half, float>)
                   : (hx ? launch_backward<float, __half> : launch_backward<float, float>);
  return launch(ctx, dy->ptr, x->ptr, f32_ptr(gamma), f32_ptr(stats), f32_out(out[0]), f32_out(out[1]), f32_out(out[2]),
                rows, width);
}

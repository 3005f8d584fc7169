// Distillation loss over a teacher's top logits, and its gradient.
//
// For each row, with student logits z over all classes, temperature T and the teacher's list of K
// (class, logit) entries, of which those with a class in [0, classes) and a logit above -inf count:
//
//   q = softmax(z / T) over all classes,   p = softmax(u / T) over the counting entries
//   loss = T^2 sum_k p_k (log p_k - log q_{i_k})              (T^2 keeps the gradient's size)
//   dz_v = dloss T (q_v - sum of p_k over the entries with i_k == v)
//
// A row without a counting entry has loss 0 and gradient 0.  The forward pass leaves the two
// log-sum-exps (of z / T and of u / T; -inf for an empty list) for the backward pass.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 1024;

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) v += scratch[w];
  return v;
}
__device__ __forceinline__ float block_max(float v, float* scratch) {
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = -INFINITY;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) v = max_nan(v, scratch[w]);
  return v;
}

// u / T of a counting entry, -inf of any other.
template <typename TU>
__device__ __forceinline__ float teacher_entry(const TU* u, int32_t i, int64_t classes, float inv_t) {
  return i >= 0 && i < classes ? load_f32(u) * inv_t : -INFINITY;
}

template <typename TZ, typename TU>
__global__ void __launch_bounds__(kThreads) distillation_kernel(const TZ* __restrict__ z, const TU* __restrict__ u,
                                                               const int32_t* __restrict__ indices,
                                                               float* __restrict__ loss, float* __restrict__ stats,
                                                               int64_t rows, int64_t classes, int top, float temperature) {
  __shared__ float scratch[kThreads / 32];
  const float inv_t = 1.f / temperature;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TZ* zr = z + row * classes;
    const TU* ur = u + row * top;
    const int32_t* ir = indices + row * top;
    float m = -INFINITY;
    for (int64_t j = threadIdx.x; j < classes; j += kThreads) m = max_nan(m, load_f32(zr + j) * inv_t);
    m = block_max(m, scratch);
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < classes; j += kThreads) s += expf(load_f32(zr + j) * inv_t - m);
    const float lse = m + logf(block_sum(s, scratch));
    float um = -INFINITY;
    for (int k = threadIdx.x; k < top; k += kThreads) um = max_nan(um, teacher_entry(ur + k, ir[k], classes, inv_t));
    um = block_max(um, scratch);
    float ulse = -INFINITY, l = 0.f;
    if (um != -INFINITY) {  // the same for the whole block
      s = 0.f;
      for (int k = threadIdx.x; k < top; k += kThreads) s += expf(teacher_entry(ur + k, ir[k], classes, inv_t) - um);
      ulse = um + logf(block_sum(s, scratch));
      for (int k = threadIdx.x; k < top; k += kThreads) {
        const float lp = teacher_entry(ur + k, ir[k], classes, inv_t) - ulse, p = expf(lp);
        if (p != 0.f) l += p * (lp - (load_f32(zr + ir[k]) * inv_t - lse));
      }
      l = block_sum(l, scratch);
    }
    if (threadIdx.x == 0) {
      loss[row] = temperature * temperature * l;
      if (stats) {
        stats[2 * row] = lse;
        stats[2 * row + 1] = ulse;
      }
    }
  }
}

template <typename TZ, typename TU>
__global__ void __launch_bounds__(kThreads) distillation_backprop_kernel(
    const float* __restrict__ dloss, const TZ* __restrict__ z, const TU* __restrict__ u,
    const int32_t* __restrict__ indices, const float* __restrict__ stats, float* __restrict__ dz, int64_t rows,
    int64_t classes, int top, float temperature) {
  __shared__ int32_t s_i[kMaxTop];
  __shared__ float s_p[kMaxTop];
  const float inv_t = 1.f / temperature;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TZ* zr = z + row * classes;
    float* dr = dz + row * classes;
    const float lse = stats[2 * row], ulse = stats[2 * row + 1], c = dloss[row] * temperature;
    const bool empty = ulse == -INFINITY;
    __syncthreads();
    for (int k = threadIdx.x; k < top; k += kThreads) {
      const int32_t i = indices[row * top + k];
      const bool there = i >= 0 && i < classes && !empty;
      s_i[k] = there ? i : -1;
      s_p[k] = there ? expf(load_f32(u + row * top + k) * inv_t - ulse) : 0.f;
    }
    for (int64_t j = threadIdx.x; j < classes; j += kThreads)
      dr[j] = empty ? 0.f : c * expf(load_f32(zr + j) * inv_t - lse);
    __syncthreads();
    // the entries' own classes: the first entry of a class writes q - (all its entries' p)
    for (int k = threadIdx.x; k < top; k += kThreads) {
      const int32_t i = s_i[k];
      if (i < 0) continue;
      float p = 0.f;
      bool first = true;
      for (int j = 0; j < top; j++) {
        if (s_i[j] != i) continue;
        if (j < k) {
          first = false;
          break;
        }
        p += s_p[j];
      }
      if (first) dr[i] = c * (expf(load_f32(zr + i) * inv_t - lse) - p);
    }
  }
}

struct Operands {
  TensorEntry *z, *u, *indices;
};

int get_operands(tfjs_cuda_ctx* ctx, tfjs_tensor_id z, tfjs_tensor_id u, tfjs_tensor_id indices, int64_t rows,
                 int64_t classes, int64_t top, float temperature, Operands* o) {
  TFJS_REQUIRE(ctx, rows >= 0 && classes >= 0 && top >= 0, "negative extent");
  TFJS_REQUIRE(ctx, classes < (1ll << 31) && rows <= (1ll << 60) / (classes > kMaxTop ? classes : kMaxTop),
               "distillationLoss: too many rows or classes");
  TFJS_REQUIRE(ctx, top <= kMaxTop, "distillationLoss: a teacher's list holds at most %d entries, got %lld", kMaxTop,
               (long long)top);
  TFJS_REQUIRE(ctx, temperature > 0.f && temperature - temperature == 0.f && 1.f / temperature - 1.f / temperature == 0.f,
               "distillationLoss: the temperature must be positive and finite");
  int rc;
  if ((rc = get_activation(ctx, z, rows * classes, "logits", &o->z))) return rc;
  if ((rc = get_activation(ctx, u, rows * top, "teacherLogits", &o->u))) return rc;
  if ((rc = get_i32(ctx, indices, rows * top, "teacherIndices", &o->indices))) return rc;
  TFJS_REQUIRE(ctx, o->z->size == rows * classes && o->u->size == rows * top,
               "distillationLoss: logits must be [rows, classes] and teacherLogits [rows, top]");
  return TFJS_CUDA_OK;
}

int get_rows(tfjs_cuda_ctx* ctx, tfjs_tensor_id id, int64_t elems, const char* what, TensorEntry** out) {
  const int rc = get_f32(ctx, id, elems, what, out);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, !(*out)->quant.quantized && (*out)->size == elems, "%s must be a float32 tensor of %lld elements", what,
               (long long)elems);
  return TFJS_CUDA_OK;
}

template <typename TZ, typename TU>
void launch_forward(tfjs_cuda_ctx* ctx, const Operands& o, float* loss, float* stats, int64_t rows, int64_t classes,
                    int top, float temperature) {
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  distillation_kernel<TZ, TU><<<(unsigned)(rows < cap ? rows : cap), kThreads, 0, ctx->stream>>>(
      (const TZ*)o.z->ptr, (const TU*)o.u->ptr, (const int32_t*)o.indices->ptr, loss, stats, rows, classes, top,
      temperature);
}

template <typename TZ, typename TU>
void launch_backward(tfjs_cuda_ctx* ctx, const float* dloss, const Operands& o, const float* stats, float* dz,
                     int64_t rows, int64_t classes, int top, float temperature) {
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  distillation_backprop_kernel<TZ, TU><<<(unsigned)(rows < cap ? rows : cap), kThreads, 0, ctx->stream>>>(
      dloss, (const TZ*)o.z->ptr, (const TU*)o.u->ptr, (const int32_t*)o.indices->ptr, stats, dz, rows, classes, top,
      temperature);
}

}  // namespace

extern "C" int tfjs_cuda_distillation_loss(tfjs_cuda_ctx* ctx, tfjs_tensor_id logits_id, tfjs_tensor_id teacher_logits_id,
                                           tfjs_tensor_id teacher_indices_id, tfjs_tensor_id loss_id,
                                           tfjs_tensor_id stats_id, int64_t rows, int64_t classes, int64_t top,
                                           float temperature) {
  if (!ctx) return TFJS_CUDA_ERR_INVALID_ARG;
  Operands o;
  TensorEntry *loss, *stats = nullptr;
  int rc = get_operands(ctx, logits_id, teacher_logits_id, teacher_indices_id, rows, classes, top, temperature, &o);
  if (!rc) rc = get_rows(ctx, loss_id, rows, "distillationLoss output", &loss);
  if (!rc && stats_id) rc = get_rows(ctx, stats_id, 2 * rows, "distillationLoss statistics", &stats);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, loss != o.z && loss != o.u && loss != stats && (!stats || (stats != o.z && stats != o.u)),
               "distillationLoss: an output cannot be one of the inputs or another output");
  loss->version++;
  if (stats) stats->version++;
  if (rows == 0) return TFJS_CUDA_OK;
  cudaSetDevice(ctx->device);
  const bool hz = o.z->dtype == TFJS_F16, hu = o.u->dtype == TFJS_F16;
  auto launch = hz ? (hu ? launch_forward<__half, __half> : launch_forward<__half, float>)
                   : (hu ? launch_forward<float, __half> : launch_forward<float, float>);
  launch(ctx, o, (float*)loss->ptr, stats ? (float*)stats->ptr : nullptr, rows, classes, (int)top, temperature);
  return post_launch(ctx, "distillationLoss");
}

extern "C" int tfjs_cuda_distillation_loss_backprop(tfjs_cuda_ctx* ctx, tfjs_tensor_id dloss_id, tfjs_tensor_id logits_id,
                                                    tfjs_tensor_id teacher_logits_id, tfjs_tensor_id teacher_indices_id,
                                                    tfjs_tensor_id stats_id, tfjs_tensor_id dlogits_id, int64_t rows,
                                                    int64_t classes, int64_t top, float temperature) {
  if (!ctx) return TFJS_CUDA_ERR_INVALID_ARG;
  Operands o;
  TensorEntry *dloss, *stats, *dz;
  int rc = get_operands(ctx, logits_id, teacher_logits_id, teacher_indices_id, rows, classes, top, temperature, &o);
  if (!rc) rc = get_rows(ctx, dloss_id, rows, "dloss", &dloss);
  if (!rc) rc = get_rows(ctx, stats_id, 2 * rows, "distillationLoss statistics", &stats);
  if (!rc) rc = get_rows(ctx, dlogits_id, rows * classes, "dlogits", &dz);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, dz != o.z && dz != o.u && dz != dloss && dz != stats,
               "distillationLossBackprop: the output cannot be one of the inputs");
  dz->version++;
  if (rows * classes == 0) return TFJS_CUDA_OK;
  cudaSetDevice(ctx->device);
  const bool hz = o.z->dtype == TFJS_F16, hu = o.u->dtype == TFJS_F16;
  auto launch = hz ? (hu ? launch_backward<__half, __half> : launch_backward<__half, float>)
                   : (hu ? launch_backward<float, __half> : launch_backward<float, float>);
  launch(ctx, (const float*)dloss->ptr, o, (const float*)stats->ptr, (float*)dz->ptr, rows, classes, (int)top, temperature);
  return post_launch(ctx, "distillationLossBackprop");
}

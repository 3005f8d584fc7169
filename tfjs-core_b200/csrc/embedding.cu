// Embedding lookup with scaling, and the gradient of its table.
//
//   out[t] = scale * table[i_t],      zeros where i_t lies outside [0, vocab) (padding)
//   dtable[v] = scale * sum of dy[t] over the tokens t with i_t == v, in the order of t
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }

// A quantised table's value is the float32 that decodeWeights gives (io_utils.ts:139).
__device__ __forceinline__ float decode(const uint8_t* p, double qs, double qm) { return (float)__dadd_rn(__dmul_rn((double)*p, qs), qm); }
template <typename T>
__device__ __forceinline__ float decode(const T* p, double, double) { return load_f32(p); }

template <typename TT, typename TO>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const TT* __restrict__ table,
                                                            const int32_t* __restrict__ indices, TO* __restrict__ out,
                                                            int64_t tokens, int64_t vocab, int64_t width, float scale,
                                                            double qs, double qm) {
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int64_t v = indices[t];
    const bool there = v >= 0 && v < vocab;
    for (int64_t j = threadIdx.x; j < width; j += kThreads)
      store_f32(out + t * width + j, there ? decode(table + v * width + j, qs, qm) * scale : 0.f);
  }
}

// One warp a table row: it walks all tokens in order and adds the rows that name it.
template <typename TD>
__global__ void __launch_bounds__(kThreads) embedding_backprop_kernel(const TD* __restrict__ dy,
                                                                     const int32_t* __restrict__ indices,
                                                                     float* __restrict__ dtable, int64_t tokens,
                                                                     int64_t vocab, int64_t width, float scale) {
  const int lane = threadIdx.x & 31;
  for (int64_t v = (blockIdx.x * (int64_t)kThreads + threadIdx.x) >> 5; v < vocab; v += (int64_t)gridDim.x * (kThreads / 32)) {
    for (int64_t j0 = 0; j0 < width; j0 += 32) {
      const int64_t j = j0 + lane;
      float acc = 0.f;
      for (int64_t t0 = 0; t0 < tokens; t0 += 32) {
        const bool mine = t0 + lane < tokens && indices[t0 + lane] == v;
        unsigned hits = __ballot_sync(0xffffffffu, mine);
        while (hits) {
          const int64_t t = t0 + __ffs(hits) - 1;
          hits &= hits - 1;
          if (j < width) acc += load_f32(dy + t * width + j);
        }
      }
      if (j < width) dtable[v * width + j] = acc * scale;
    }
  }
}

int check_extent(tfjs_cuda_ctx* ctx, int64_t tokens, int64_t vocab, int64_t width) {
  TFJS_REQUIRE(ctx, tokens >= 0 && vocab >= 0 && width >= 0, "negative extent");
  TFJS_REQUIRE(ctx, tokens < (1ll << 31) && vocab < (1ll << 31) && width < (1ll << 31),
               "embeddingLookup: too many tokens, rows or columns");
  return TFJS_CUDA_OK;
}

}  // namespace

extern "C" int tfjs_cuda_embedding_lookup(tfjs_cuda_ctx* ctx, tfjs_tensor_id table_id, tfjs_tensor_id indices_id,
                                          tfjs_tensor_id out_id, int64_t tokens, int64_t vocab, int64_t width,
                                          float scale) {
  if (!ctx) return TFJS_CUDA_ERR_INVALID_ARG;
  int rc = check_extent(ctx, tokens, vocab, width);
  if (rc) return rc;
  TensorEntry *table, *indices, *o;
  table = find_tensor(ctx, table_id);
  if (table && table->quant.quantized)
    rc = get_f32(ctx, table_id, vocab * width, "table", &table);
  else
    rc = get_activation(ctx, table_id, vocab * width, "table", &table);
  if (rc) return rc;
  TFJS_REQUIRE(ctx, table->size == vocab * width, "table holds %lld elements, %lld expected", (long long)table->size,
               (long long)(vocab * width));
  if ((rc = get_i32(ctx, indices_id, tokens, "indices", &indices))) return rc;
  if ((rc = get_activation(ctx, out_id, tokens * width, "embeddingLookup output", &o))) return rc;
  TFJS_REQUIRE(ctx, o->size == tokens * width, "embeddingLookup output holds %lld elements, %lld expected",
               (long long)o->size, (long long)(tokens * width));
  TFJS_REQUIRE(ctx, o != table && o != indices, "embeddingLookup: the output cannot be one of the inputs");
  o->version++;
  if (tokens * width == 0) return TFJS_CUDA_OK;
  cudaSetDevice(ctx->device);
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  const unsigned grid = (unsigned)(tokens < cap ? tokens : cap);
  const int32_t* idx = (const int32_t*)indices->ptr;
  const double qs = table->quant.scale, qm = table->quant.min;
  const bool half_out = o->dtype == TFJS_F16;
#define TFJS_EMBED(TT, TO)                                                                                           \
  embedding_kernel<TT, TO><<<grid, kThreads, 0, ctx->stream>>>((const TT*)table->ptr, idx, (TO*)o->ptr, tokens, vocab, \
                                                               width, scale, qs, qm)
  if (table->quant.quantized) {
    if (half_out) TFJS_EMBED(uint8_t, __half);
    else TFJS_EMBED(uint8_t, float);
  } else if (table->dtype == TFJS_F16) {
    if (half_out) TFJS_EMBED(__half, __half);
    else TFJS_EMBED(__half, float);
  } else {
    if (half_out) TFJS_EMBED(float, __half);
    else TFJS_EMBED(float, float);
  }
#undef TFJS_EMBED
  return post_launch(ctx, "embeddingLookup");
}

extern "C" int tfjs_cuda_embedding_lookup_backprop(tfjs_cuda_ctx* ctx, tfjs_tensor_id dy_id, tfjs_tensor_id indices_id,
                                                   tfjs_tensor_id dtable_id, int64_t tokens, int64_t vocab,
                                                   int64_t width, float scale) {
  if (!ctx) return TFJS_CUDA_ERR_INVALID_ARG;
  int rc = check_extent(ctx, tokens, vocab, width);
  if (rc) return rc;
  TensorEntry *dy, *indices, *o;
  if ((rc = get_activation(ctx, dy_id, tokens * width, "dy", &dy))) return rc;
  if ((rc = get_i32(ctx, indices_id, tokens, "indices", &indices))) return rc;
  if ((rc = get_f32(ctx, dtable_id, vocab * width, "table gradient", &o))) return rc;
  TFJS_REQUIRE(ctx, dy->size == tokens * width, "dy holds %lld elements, %lld expected", (long long)dy->size,
               (long long)(tokens * width));
  TFJS_REQUIRE(ctx, !o->quant.quantized && o->size == vocab * width && o != dy && o != indices,
               "embeddingLookupBackprop: the table gradient must be a float32 tensor of its own, [vocab, width]");
  o->version++;
  if (vocab * width == 0) return TFJS_CUDA_OK;
  cudaSetDevice(ctx->device);
  if (tokens == 0) {
    TFJS_CHECK_CUDA(ctx, cudaMemsetAsync(o->ptr, 0, (size_t)(vocab * width) * 4, ctx->stream));
    return TFJS_CUDA_OK;
  }
  const int64_t blocks = ceil_div64(vocab, kThreads / 32), cap = (int64_t)ctx->sm_count * 16;
  const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
  const int32_t* idx = (const int32_t*)indices->ptr;
  if (dy->dtype == TFJS_F16)
    embedding_backprop_kernel<__half><<<grid, kThreads, 0, ctx->stream>>>((const __half*)dy->ptr, idx, (float*)o->ptr,
                                                                         tokens, vocab, width, scale);
  else
    embedding_backprop_kernel<float><<<grid, kThreads, 0, ctx->stream>>>((const float*)dy->ptr, idx, (float*)o->ptr,
                                                                        tokens, vocab, width, scale);
  return post_launch(ctx, "embeddingLookupBackprop");
}

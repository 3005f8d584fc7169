// Layer normalisation over the inner-most axis and its gradients.
//
//   y = (x - m) r g + b,   m = mean(x),   r = 1 / sqrt(mean((x - m)^2) + eps)
//   with n = (x - m) r and a = dy g:
//   dx = r (a - mean(a) - n mean(a n)),   dg = sum over rows of dy n,   db = sum over rows of dy
//
// All sums are float32; a half-stored x or dy is widened on load, a half-stored y rounded once on
// store.  Every sum has a fixed order, so equal inputs give equal bits.
//
// Forward.  A row is read once and stays on chip: the mean and then the centred square sum (which
// does not cancel, unlike E[x^2] - m^2) come from the same registers.  By width:
//   up to 1024     L lanes a row (4 .. 32), no shared memory (32768 x 1024: 45 us, 6.0 TB/s; a block a row 62)
//   up to 16384    one block a row (2048 x 16384: 48 us, 5.6 TB/s; clusters 66)
//   either         where rows start off the 16-byte boundaries, a warp or a block with a ring of rows in
//                  shared memory (33000 x 1001 half: 39 us; one value a load 93)
//   above          a cluster of 1 to 8 blocks a row, the row in their shared memory, sums joined over DSMEM
//                  (1000 x 33000: 76 us, 3.5 TB/s)
// The first two are bound by memory, the ring by its instructions (4-byte words instead of 16), the clusters
// by the latency of a row: load, two cluster-wide joins, store.
// Gradient.  One pass over dy and x gives dx and, per block, the weights' gradients:
//   up to 8192     persistent blocks; a ring of stages (several rows each) filled by cp.async.  First
//                  the lanes of a row sum a and a n, then every thread takes the same columns of every
//                  row: it writes dx and keeps its columns' dg, db in registers.  16384 x 1024: 38 us, 5.3 TB/s
//                  (with 8 KB rows and 512 threads, whose fixed cost a stage was 60 % of all instructions, 68);
//                  4096 x 8192: 79 us, clusters 141
//   above          a cluster of 1 to 8 blocks a row; dg, db add up in the blocks' shared memory.  1000 x 33000:
//                  186 us, bound by the latency of a row (a quarter of the DRAM rate, 36 % of the issue slots)
// and a second kernel adds the blocks' partial dg, db in order (4 us at 16384 x 1024, 2.4 MB from L2).
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace cg = cooperative_groups;

namespace {

// y = (x - mean) * rstd * gamma + beta for V columns from `col`
template <int V, typename TY>
__device__ __forceinline__ void finish_vec(const float (&x)[V], float mean, float rstd, const float* __restrict__ gamma,
                                           const float* __restrict__ beta, int64_t col, TY* y) {
  float o[V], w[V];
#pragma unroll
  for (int i = 0; i < V; i++) o[i] = (x[i] - mean) * rstd;
  if (gamma) {
    load_vec<V>(gamma + col, w);
#pragma unroll
    for (int i = 0; i < V; i++) o[i] *= w[i];
  }
  if (beta) {
    load_vec<V>(beta + col, w);
#pragma unroll
    for (int i = 0; i < V; i++) o[i] += w[i];
  }
  store_vec<V>(y, o);
}

// Sum over a block of NT threads; every thread gets it.  `scratch` holds NT / 32 floats of its own.
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = lanes_sum<32>(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_sum<NT / 32>(scratch[threadIdx.x & (NT / 32 - 1)]);
}

// ---- forward -------------------------------------------------------------------------------------
// L lanes a row, NV vectors of V values a lane: width <= L * NV * V, a multiple of V.  gamma and beta come from
// L1 when the row is finished: fetched with the row they took registers from other rows in flight (100352 x
// 256 float32 36 us so, 34 us now; 25088 x 512 half 16 and 13.5 us).
template <typename TX, typename TY, int V, int NV, int L>
__global__ void __launch_bounds__(256) layer_norm_lanes_kernel(const TX* __restrict__ x, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, TY* __restrict__ y,
                                                              float* __restrict__ stats, int64_t rows, int width,
                                                              float epsilon) {
  const int lane = threadIdx.x & (L - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const bool there = row < rows;  // lanes without a row go along, for the shuffles
  const TX* r = x + row * width;
  float v[NV][V];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = (i * L + lane) * V;
    if (there && col < width) {
      load_vec<V>(r + col, v[i]);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) v[i][k] = 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; i++)
#pragma unroll
    for (int k = 0; k < V; k++) s += v[i][k];
  const float mean = lanes_sum<L>(s) / (float)width;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; i++)
    if ((i * L + lane) * V < width) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float d = v[i][k] - mean;
        s = fmaf(d, d, s);
      }
    }
  const float rstd = 1.f / sqrtf(lanes_sum<L>(s) / (float)width + epsilon);
  if (!there) return;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = (i * L + lane) * V;
    if (col >= width) break;
    finish_vec<V>(v[i], mean, rstd, gamma, beta, col, y + row * width + col);
  }
  if (stats && lane == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(mean, rstd);
}

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The whole 16-byte units that [first, first + bytes) touches, into shared memory, by LANES threads.  The units lie
// within the tensor's buffer: its start is 16-byte aligned and its size class a multiple of 16.
template <int LANES>
__device__ __forceinline__ void stage_copy(uint8_t* dst, const uint8_t* base, int64_t first, int bytes) {
  const int off = (int)(first & 15), units = (off + bytes + 15) >> 4;
  const uint8_t* src = base + (first - off);
#pragma unroll 4
  for (int i = threadIdx.x & (LANES - 1); i < units; i += LANES) copy_async16(dst + i * 16, src + i * 16);
}

// Rows that do not start on 16-byte boundaries.  A group of G threads, a warp or the block, has a ring of two
// row slots in shared memory that cp.async fills with the row's 16-byte units, so the loads are wide whatever
// the row's offset; it takes the row from there into registers as 4-byte words, NW a thread (P values each:
// two halves or one float).  Where halves start at an odd place, the first word (and maybe the last) holds
// one value of the neighbouring row, which is left out.  For a warp's rows, gamma and beta lie beside each
// other in shared memory in the words' order, once for even and once for odd rows.
// (One value a load in place of this: 33000 x 1001 half 93 us, 9000 x 3001 half 76 us.)
constexpr int kRingThreads = 256;
template <typename TX, typename TY, int NW, int G>
__global__ void __launch_bounds__(kRingThreads) layer_norm_ring_kernel(const TX* __restrict__ x,
                                                                         const float* __restrict__ gamma,
                                                                         const float* __restrict__ beta, TY* __restrict__ y,
                                                                         float* __restrict__ stats, int64_t rows, int width,
                                                                         float epsilon, int slot_bytes) {
  constexpr int P = 4 / (int)sizeof(TX);
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kGroups = kRingThreads / G;
  __shared__ float scratch[2][kRingThreads / 32];
  const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G;
  uint8_t* ring = smem + group * 2 * slot_bytes;
  auto sync = [] {
    if (G == 32) __syncwarp();
    else __syncthreads();
  };
  auto sum = [&](float v, int turn) { return G == 32 ? lanes_sum<32>(v) : block_sum<kRingThreads>(v, scratch[turn]); };
  const int most = width / P + 1;  // words of a row, at most
  float* weights = reinterpret_cast<float*>(smem + kGroups * 2 * slot_bytes);  // [odd][most][2 P]: P of gamma, P of beta
  const int64_t step = (int64_t)gridDim.x * kGroups, first = (int64_t)blockIdx.x * kGroups + group;
  auto fill = [&](int64_t row, int slot) {
    if (row < rows)
      stage_copy<G>(ring + slot * slot_bytes, (const uint8_t*)x, row * width * (int64_t)sizeof(TX), width * (int)sizeof(TX));
    copy_commit();
  };
  fill(first, 0);
  for (int j = threadIdx.x; G == 32 && j < P * most * P; j += kRingThreads) {
    const int odd = j / (most * P), e = j - odd * most * P, col = e - odd;
    float* w = weights + (odd * most + e / P) * 2 * P + e % P;
    const bool there = col >= 0 && col < width;
    w[0] = gamma && there ? gamma[col] : 1.f;
    w[P] = beta && there ? beta[col] : 0.f;
  }
  __syncthreads();
  const float inv = 1.f / (float)width;
  int slot = 0;
  for (int64_t row = first; row < rows; row += step, slot ^= 1) {
    fill(row + step, slot ^ 1);
    copy_wait<1>();
    sync();  // the row is there for all
    const int64_t at = row * width;
    const int odd = (int)(at & (P - 1)), words = (odd + width + P - 1) / P;
    const TX* r = reinterpret_cast<const TX*>(ring + slot * slot_bytes + ((at * (int64_t)sizeof(TX)) & 15)) - odd;
    const bool cut = P == 2 && ((odd + width) & 1);  // the last word's second value is the next row's
    uint32_t q[NW];
#pragma unroll
    for (int i = 0; i < NW; i++) {
      const int w = lane + G * i;
      q[i] = w < words ? *reinterpret_cast<const uint32_t*>(r + w * P) : 0u;
      if (P == 2) {
        if (w == 0 && odd) q[i] &= 0xffff0000u;
        if (w == words - 1 && cut) q[i] &= 0x0000ffffu;
      }
    }
    sync();  // read by all: the slot may be filled again
    const TX* none = nullptr;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      float v[P];
      unpack_word(q[i], none, v);
#pragma unroll
      for (int k = 0; k < P; k++) s += v[k];
    }
    const float mean = sum(s, 0) * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      const int w = lane + G * i;
      if (w >= words) break;
      float v[P];
      unpack_word(q[i], none, v);
#pragma unroll
      for (int k = 0; k < P; k++) {
        float d = v[k] - mean;
        if (P == 2 && ((k == 0 && w == 0 && odd) || (k == 1 && w == words - 1 && cut))) d = 0.f;
        s = fmaf(d, d, s);
      }
    }
    const float rstd = 1.f / sqrtf(sum(s, 1) * inv + epsilon);
    TY* out = y + at - odd;
    const float* mine = weights + odd * most * 2 * P;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      const int w = lane + G * i;
      if (w >= words) break;
      float v[P], gb[2 * P];
      unpack_word(q[i], none, v);
      if (G == 32) {
        load_vec<2 * P>(mine + w * 2 * P, gb);
      } else {
#pragma unroll
        for (int k = 0; k < P; k++) {
          const int col = min(max(w * P + k - odd, 0), width - 1);
          gb[k] = gamma ? gamma[col] : 1.f;
          gb[P + k] = beta ? beta[col] : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < P; k++) v[k] = fmaf((v[k] - mean) * rstd, gb[k], gb[P + k]);
      const bool low = P == 2 && w == 0 && odd, high = P == 2 && w == words - 1 && cut;
      if (!low && !high) {
        store_vec<P>(out + w * P, v);
      } else {
        if (!low) {
          const float o[1] = {v[0]};
          store_vec<1>(out + w * P, o);
        }
        if (!high) {
          const float o[1] = {v[P - 1]};
          store_vec<1>(out + w * P + P - 1, o);
        }
      }
    }
    if (stats && lane == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(mean, rstd);
  }
}

// One block of NT threads a row: width <= NT * NV * V, a multiple of V.
template <typename TX, typename TY, int V, int NV, int NT>
__global__ void __launch_bounds__(NT) layer_norm_block_kernel(const TX* __restrict__ x, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, TY* __restrict__ y,
                                                             float* __restrict__ stats, int64_t rows, int width,
                                                             float epsilon) {
  __shared__ float scratch[2][32];  // one for each sum of a row: its readers are done before its next writers start
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TX* r = x + row * width;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = (i * NT + threadIdx.x) * V;
      if (col < width) {
        load_vec<V>(r + col, v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) v[i][k] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int k = 0; k < V; k++) s += v[i][k];
    const float mean = block_sum<NT>(s, scratch[0]) / (float)width;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if ((i * NT + (int)threadIdx.x) * V < width) {
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float d = v[i][k] - mean;
          s = fmaf(d, d, s);
        }
      }
    const float rstd = 1.f / sqrtf(block_sum<NT>(s, scratch[1]) / (float)width + epsilon);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = (i * NT + threadIdx.x) * V;
      if (col < width) finish_vec<V>(v[i], mean, rstd, gamma, beta, col, y + row * width + col);
    }
    if (stats && threadIdx.x == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(mean, rstd);
  }
}

constexpr int kClusterThreads = 512;

// Sums of a and b over the cluster's C blocks, in their order.  `slot` is this block's place in its own
// shared memory; two uses of the same slot must have another cluster-wide sum between them.
__device__ __forceinline__ float2 cluster_sum(float a, float b, int C, float2* slot, float2* scratch) {
  cg::cluster_group cluster = cg::this_cluster();
  a = lanes_sum<32>(a);
  b = lanes_sum<32>(b);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  const float2 v = scratch[threadIdx.x & (kClusterThreads / 32 - 1)];
  float2 t = make_float2(lanes_sum<kClusterThreads / 32>(v.x), lanes_sum<kClusterThreads / 32>(v.y));
  if (C == 1) return t;
  if (threadIdx.x == 0) *slot = t;
  cluster.sync();
  t = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (i >= C) break;
    const float2 o = *cluster.map_shared_rank(slot, i);
    t.x += o.x;
    t.y += o.y;
  }
  return t;
}

// A cluster of C blocks a row.  `cached`: the block's share of the row comes into its dynamic shared memory
// by cp.async, whatever its offset, and is read from there; else three times from global memory (L2).
template <typename TX, typename TY, int V>
__global__ void __launch_bounds__(kClusterThreads, 3) layer_norm_cluster_kernel(
    const TX* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, TY* __restrict__ y,
    float* __restrict__ stats, int64_t rows, int64_t width, float epsilon, int C, int cached) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 scratch[2][kClusterThreads / 32];
  __shared__ float2 slot[2];
  const int64_t vecs = width / V, clusters = gridDim.x / C;
  const int64_t rank = blockIdx.x % C;
  const int64_t lo = vecs * rank / C;
  const int n = (int)(vecs * (rank + 1) / C - lo);
  for (int64_t row = blockIdx.x / C; row < rows; row += clusters) {
    const TX* r = x + row * width + lo * V;
    if (cached) {
      const int64_t first = row * width + lo * V;
      __syncthreads();  // all are done with the row before
      stage_copy<kClusterThreads>(smem, (const uint8_t*)x, first * (int64_t)sizeof(TX), n * V * (int)sizeof(TX));
      copy_commit();
      copy_wait<0>();
      __syncthreads();
      r = reinterpret_cast<const TX*>(smem + ((first * (int64_t)sizeof(TX)) & 15));
    }
    float s = 0.f;
#pragma unroll 4
    for (int j = threadIdx.x; j < n; j += kClusterThreads) {
      float v[V];
      load_vec<V>(r + j * V, v);
#pragma unroll
      for (int k = 0; k < V; k++) s += v[k];
    }
    const float mean = cluster_sum(s, 0.f, C, &slot[0], scratch[0]).x / (float)width;
    s = 0.f;
#pragma unroll 4
    for (int j = threadIdx.x; j < n; j += kClusterThreads) {
      float v[V];
      load_vec<V>(r + j * V, v);
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float d = v[k] - mean;
        s = fmaf(d, d, s);
      }
    }
    const float rstd = 1.f / sqrtf(cluster_sum(s, 0.f, C, &slot[1], scratch[1]).x / (float)width + epsilon);
#pragma unroll 2
    for (int j = threadIdx.x; j < n; j += kClusterThreads) {
      float v[V];
      load_vec<V>(r + j * V, v);
      finish_vec<V>(v, mean, rstd, gamma, beta, (lo + j) * V, y + row * width + (lo + j) * V);
    }
    if (stats && rank == 0 && threadIdx.x == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(mean, rstd);
  }
  cg::this_cluster().sync();  // no block leaves while another may still read its slot
}

// ---- gradient, width <= kStagedWidth -----------------------------------------------------------------
constexpr int kStagedWidth = 8192;
constexpr int kStagedThreads = 256;
constexpr int kMaxStageRows = 256;

// Where a block (or cluster) leaves its dg and db: its row of a buffer that the join kernel adds up, or, where
// there is only one, the results themselves.  Either may be null (not wanted).
struct WeightSums {
  float *dg, *db;
  int64_t stride;  // from one block's row to the next
};

struct StagedParams {
  const float* gamma;
  const float* stats;
  float* dx;
  WeightSums sums;
  int64_t rows, items;
  int width, stage_rows;        // stage_rows: a power of two
  int x_bytes, stage_bytes;     // of the dy and the whole stage area
};

constexpr int kStages = 3;

// MC vectors of V columns a thread: width <= 256 * MC * V, a multiple of V.
// The products of dx are rounded before they are added or subtracted (no contraction): in rows of one or two
// columns the terms cancel, and a product kept unrounded on one side only would leave its rounding error,
// times rstd, where the formula gives 0.
template <typename TD, typename TX, int V, int MC>
__global__ void __launch_bounds__(kStagedThreads, 2) layer_norm_staged_kernel(const TD* __restrict__ dy,
                                                                              const TX* __restrict__ x,
                                                                              StagedParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int width = p.width, R = p.stage_rows, nc = width / V;
  const int tid = threadIdx.x;
  const float inv = 1.f / (float)width;
  uint8_t* ring = smem;
  float* s_gamma = reinterpret_cast<float*>(smem + kStages * p.stage_bytes);
  const int LR = kStagedThreads / R;             // lanes that sum a row
  const int parts = LR > 32 ? LR / 32 : 1;       // their warps' partial sums
  float2* s_part = reinterpret_cast<float2*>(s_gamma + (width + 3) / 4 * 4);

  // phase 2: thread -> columns; several row groups share the block where a row has few columns
  const int RG = nc < kStagedThreads ? kStagedThreads / nc : 1;
  const int rg = nc < kStagedThreads ? tid / nc : 0;
  const int c0 = nc < kStagedThreads ? tid - rg * nc : tid;
  const bool owner = rg < RG;
  // phase 1: LR threads a row
  const int l = tid & (LR - 1), row1 = tid / LR;
  float dg[MC][V], db[MC][V];
#pragma unroll
  for (int i = 0; i < MC; i++)
#pragma unroll
    for (int k = 0; k < V; k++) dg[i][k] = db[i][k] = 0.f;

  const int64_t step = gridDim.x;
  auto fill = [&](int64_t item, int slot) {
    if (item < p.items) {
      const int64_t row = item * R;
      const int n = (int)(p.rows - row < R ? p.rows - row : R);
      uint8_t* dst = ring + slot * p.stage_bytes;
      stage_copy<kStagedThreads>(dst, (const uint8_t*)dy, row * width * (int64_t)sizeof(TD), n * width * (int)sizeof(TD));
      stage_copy<kStagedThreads>(dst + p.x_bytes, (const uint8_t*)x, row * width * (int64_t)sizeof(TX), n * width * (int)sizeof(TX));
      float2* st = reinterpret_cast<float2*>(dst + p.stage_bytes) - R;
      if (tid < n) copy_async8(st + tid, p.stats + 2 * (row + tid));
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) fill(blockIdx.x + s * step, s);
  for (int j = tid; j < width; j += kStagedThreads) s_gamma[j] = p.gamma ? p.gamma[j] : 1.f;
  pdl_launch_dependents();  // the join kernel waits for this one's end before it reads

  int slot = 0;
  for (int64_t item = blockIdx.x; item < p.items; item += step) {
    copy_wait<kStages - 2>();
    __syncthreads();  // this stage has arrived for all; the stage before it has been read by all
    fill(item + (kStages - 1) * step, slot == 0 ? kStages - 1 : slot - 1);
    const int64_t row0 = item * R;
    const int n = (int)(p.rows - row0 < R ? p.rows - row0 : R);
    const uint8_t* st = ring + slot * p.stage_bytes;
    const TD* sd = reinterpret_cast<const TD*>(st + ((row0 * width * (int64_t)sizeof(TD)) & 15));
    const TX* sx = reinterpret_cast<const TX*>(st + p.x_bytes + ((row0 * width * (int64_t)sizeof(TX)) & 15));
    const float2* ss = reinterpret_cast<const float2*>(st + p.stage_bytes) - R;
    // ---- phase 1: sum a and a (x - m) of each row
    {
      float sa = 0.f, sn = 0.f;
      if (row1 < n) {
        const float2 mr = ss[row1];
        const TD* d1 = sd + row1 * width;
        const TX* x1 = sx + row1 * width;
#pragma unroll 4
        for (int j = l; j < nc; j += LR) {
          float d[V], v[V], g[V];
          load_vec<V>(d1 + j * V, d);
          load_vec<V>(x1 + j * V, v);
          load_vec<V>(s_gamma + j * V, g);
#pragma unroll
          for (int k = 0; k < V; k++) {
            const float a = __fmul_rn(d[k], g[k]);
            sa += a;
            sn += __fmul_rn(a, __fmul_rn(v[k] - mr.x, mr.y));
          }
        }
      }
      for (int o = (LR < 32 ? LR : 32) >> 1; o > 0; o >>= 1) {
        sa += __shfl_xor_sync(0xffffffffu, sa, o);
        sn += __shfl_xor_sync(0xffffffffu, sn, o);
      }
      if ((l & 31) == 0) s_part[row1 * parts + (l >> 5)] = make_float2(sa, sn);
    }
    __syncthreads();
    // ---- phase 2: dx, and the owned columns' dg and db
    if (owner) {
#pragma unroll 2
      for (int row = rg; row < n; row += RG) {
        const float2 mr = ss[row];
        float2 t = s_part[row * parts];
        for (int i = 1; i < parts; i++) {
          const float2 o = s_part[row * parts + i];
          t.x += o.x;
          t.y += o.y;
        }
        const float ma = t.x * inv, man = t.y * inv;
        const TD* d2 = sd + row * width;
        const TX* x2 = sx + row * width;
        float* out = p.dx + (row0 + row) * width;
#pragma unroll
        for (int i = 0; i < MC; i++) {
          const int c = c0 + i * kStagedThreads;
          if (MC > 1 && c >= nc) break;
          float d[V], v[V], g[V], o[V];
          load_vec<V>(d2 + c * V, d);
          load_vec<V>(x2 + c * V, v);
          load_vec<V>(s_gamma + c * V, g);
#pragma unroll
          for (int k = 0; k < V; k++) {
            const float nn = __fmul_rn(v[k] - mr.x, mr.y);
            o[k] = mr.y * ((__fmul_rn(d[k], g[k]) - ma) - __fmul_rn(nn, man));
            dg[i][k] = fmaf(d[k], nn, dg[i][k]);
            db[i][k] += d[k];
          }
          if (p.dx) store_vec<V>(out + c * V, o);
        }
      }
    }
    if (++slot == kStages) slot = 0;
  }
  if (!p.sums.dg && !p.sums.db) return;
  // ---- the row groups' sums, in order; then this block's
  float* to_g = p.sums.dg ? p.sums.dg + blockIdx.x * p.sums.stride : nullptr;
  float* to_b = p.sums.db ? p.sums.db + blockIdx.x * p.sums.stride : nullptr;
  if (RG > 1) {
    copy_wait<0>();
    __syncthreads();
    float* join = reinterpret_cast<float*>(ring);  // [RG][2][width]
    if (owner) {
      store_vec<V>(join + (rg * 2) * width + c0 * V, dg[0]);
      store_vec<V>(join + (rg * 2 + 1) * width + c0 * V, db[0]);
    }
    __syncthreads();
    for (int j = tid; j < 2 * width; j += kStagedThreads) {
      float s = 0.f;
      for (int g = 0; g < RG; g++) s += join[g * 2 * width + j];
      float* to = j < width ? to_g : to_b;
      if (to) to[j < width ? j : j - width] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < MC; i++) {
      const int c = c0 + i * kStagedThreads;
      if (owner && c < nc) {
        if (to_g) store_vec<V>(to_g + c * V, dg[i]);
        if (to_b) store_vec<V>(to_b + c * V, db[i]);
      }
    }
  }
}

// ---- gradient, longer rows: a cluster of C blocks a row --------------------------------------------
// RING: the block's share of dy and x comes into shared memory by cp.async, the next row's while this one is
// summed and written, and its columns' dg and db add up there over the cluster's rows; else both passes read
// global memory (the second one L2), and the cluster's row of the sums is where dg and db add up.  In both
// a thread meets its own columns only, but for the copies, which the barriers of the sums order.
struct ClusterParams {
  const float *gamma, *stats;
  float* dx;
  WeightSums sums;
  int64_t rows, width;
  int C, d_bytes, slot_bytes;  // RING: of the dy area of a slot, and of a slot
};
template <typename TD, typename TX, int V, bool RING>
__global__ void __launch_bounds__(kClusterThreads, 2) layer_norm_backprop_cluster_kernel(const TD* __restrict__ dy,
                                                                                        const TX* __restrict__ x,
                                                                                        ClusterParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 scratch[2][kClusterThreads / 32];
  __shared__ float2 slot[2];
  const int C = p.C, tid = threadIdx.x;
  const int64_t width = p.width, vecs = width / V, clusters = gridDim.x / C, cluster = blockIdx.x / C;
  const int64_t rank = blockIdx.x % C, lo = vecs * rank / C * V;
  const int n = (int)(vecs * (rank + 1) / C - vecs * rank / C);
  float* pg = p.sums.dg ? p.sums.dg + cluster * p.sums.stride + lo : nullptr;
  float* pb = p.sums.db ? p.sums.db + cluster * p.sums.stride + lo : nullptr;
  const float* gamma = p.gamma ? p.gamma + lo : nullptr;
  float* sg = reinterpret_cast<float*>(smem + 2 * p.slot_bytes);  // dg and db, V columns of each in turn
  auto fill = [&](int64_t row, int at) {
    if (row < p.rows) {
      const int64_t first = row * width + lo;
      uint8_t* dst = smem + at * p.slot_bytes;
      stage_copy<kClusterThreads>(dst, (const uint8_t*)dy, first * (int64_t)sizeof(TD), n * V * (int)sizeof(TD));
      stage_copy<kClusterThreads>(dst + p.d_bytes, (const uint8_t*)x, first * (int64_t)sizeof(TX), n * V * (int)sizeof(TX));
    }
    copy_commit();
  };
  if (RING) fill(cluster, 0);
  pdl_launch_dependents();  // the join kernel waits for this one's end before it reads
  int turn = 0;
  for (int64_t row = cluster; row < p.rows; row += clusters, turn ^= 1) {
    const int64_t first = row * width + lo;
    const TD* d0 = dy + first;
    const TX* x0 = x + first;
    if (RING) {
      __syncthreads();  // all are done with the row before this one: its slot takes the next
      fill(row + clusters, turn ^ 1);
      copy_wait<1>();
      __syncthreads();
      const uint8_t* at = smem + turn * p.slot_bytes;
      d0 = reinterpret_cast<const TD*>(at + ((first * (int64_t)sizeof(TD)) & 15));
      x0 = reinterpret_cast<const TX*>(at + p.d_bytes + ((first * (int64_t)sizeof(TX)) & 15));
    }
    const float2 mr = *reinterpret_cast<const float2*>(p.stats + 2 * row);
    float sa = 0.f, sn = 0.f;
#pragma unroll 4
    for (int j = tid; j < n; j += kClusterThreads) {
      float d[V], v[V], g[V];
      load_vec<V>(d0 + j * V, d);
      load_vec<V>(x0 + j * V, v);
      if (gamma) load_vec<V>(gamma + j * V, g);
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float a = gamma ? d[k] * g[k] : d[k];
        sa += a;
        sn = fmaf(a, v[k] - mr.x, sn);
      }
    }
    const float2 t = cluster_sum(sa, sn, C, &slot[turn], scratch[turn]);
    const float ma = t.x / (float)width, man = t.y * mr.y / (float)width;
    const bool fresh = row == cluster;                     // nothing added up yet
    const bool hand_over = !RING || row + clusters >= p.rows;  // the cluster's last row
#pragma unroll 2
    for (int j = tid; j < n; j += kClusterThreads) {
      float d[V], v[V], g[V], o[V], wg[V], wb[V];
      load_vec<V>(d0 + j * V, d);
      load_vec<V>(x0 + j * V, v);
      if (gamma) load_vec<V>(gamma + j * V, g);
#pragma unroll
      for (int k = 0; k < V; k++) wg[k] = wb[k] = 0.f;
      if (pg && !fresh) load_vec<V>(RING ? sg + 2 * j * V : pg + j * V, wg);
      if (pb && !fresh) load_vec<V>(RING ? sg + (2 * j + 1) * V : pb + j * V, wb);
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float nn = (v[k] - mr.x) * mr.y;
        o[k] = mr.y * fmaf(-nn, man, (gamma ? d[k] * g[k] : d[k]) - ma);
        wg[k] = fmaf(d[k], nn, wg[k]);
        wb[k] += d[k];
      }
      if (p.dx) store_vec<V>(p.dx + first + j * V, o);
      if (pg) store_vec<V>(hand_over ? pg + j * V : sg + 2 * j * V, wg);
      if (pb) store_vec<V>(hand_over ? pb + j * V : sg + (2 * j + 1) * V, wb);
    }
  }
  cg::this_cluster().sync();
}

// out[j] = sum over the blocks of partial[block][j]; j runs over dg and then db.  Many blocks: 32 columns a
// block, 32 threads a column take every 32nd block's row and join theirs in order.  Up to 64: a thread a column.
// (40 blocks of 20000 columns: 2 us with a thread a column, 6 with 32; 60 of 200000: 10 and 66; 100 of 8000: 6 and
// 4; 296 of 1024: 12 and 4.)
// `partial` comes without __restrict__: a load that the compiler may take for one of constant data could be moved
// ahead of pdl_wait().
constexpr int kJoinThreads = 1024, kFewBlocks = 64;
__global__ void __launch_bounds__(kJoinThreads) layer_norm_join_kernel(const float* partial,
                                                                      float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                      int blocks, int64_t width) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  pdl_wait();
  for (int64_t j0 = (int64_t)blockIdx.x * 32; j0 < 2 * width; j0 += (int64_t)gridDim.x * 32) {
    const int64_t j = j0 + lane;
    float s = 0.f;
    if (j < 2 * width) {
#pragma unroll 10
      for (int b = w; b < blocks; b += 32) s += partial[(int64_t)b * 2 * width + j];
    }
    part[w][lane] = s;
    __syncthreads();
    s = lanes_sum<32>(part[lane][w]);  // warp w joins column w
    const int64_t c = j0 + w;
    if (lane == 0 && c < 2 * width) {
      float* out = c < width ? dgamma : dbeta;
      if (out) out[c < width ? c : c - width] = s;
    }
    __syncthreads();
  }
}
__global__ void __launch_bounds__(256) layer_norm_join_few_kernel(const float* partial,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                 int blocks, int64_t width) {
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  pdl_wait();
  if (j >= 2 * width) return;
  float* out = j < width ? dgamma : dbeta;
  if (!out) return;
  float s = 0.f;
#pragma unroll 8
  for (int b = 0; b < blocks; b++) s += partial[(int64_t)b * 2 * width + j];
  out[j < width ? j : j - width] = s;
}

// ---- launchers -----------------------------------------------------------------------------------
struct ForwardArgs {
  const void* x;
  const float *gamma, *beta;
  void* y;
  float* stats;
  int64_t rows, width;
  float epsilon;
};

unsigned grid_rows(const tfjs_cuda_ctx* ctx, int64_t blocks, int per_sm) {
  const int64_t cap = (int64_t)ctx->sm_count * per_sm;
  return (unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}

template <typename TX, typename TY, int V, int NV, int L>
void lanes_form(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  layer_norm_lanes_kernel<TX, TY, V, NV, L><<<(unsigned)ceil_div64(a.rows, 256 / L), 256, 0, ctx->stream>>>(
      (const TX*)a.x, a.gamma, a.beta, (TY*)a.y, a.stats, a.rows, (int)a.width, a.epsilon);
}
// Eight blocks an SM go on to further rows: 16384 x 2048 45 us, 57 with four, 90 with two.  (A block for every row
// measures the same there and is ahead with more rows: 65536 x 1536 half 160 us, 191 with eight.)
template <typename TX, typename TY, int V, int NV, int NT>
void block_form(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  layer_norm_block_kernel<TX, TY, V, NV, NT><<<grid_rows(ctx, a.rows, 8), NT, 0, ctx->stream>>>(
      (const TX*)a.x, a.gamma, a.beta, (TY*)a.y, a.stats, a.rows, (int)a.width, a.epsilon);
}

// Clusters of C blocks with `smem` bytes of dynamic shared memory each: a launch, and how many run at once.
struct ClusterLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  ClusterLaunch(const tfjs_cuda_ctx* ctx, int64_t clusters, int C, size_t smem) {
    cfg.gridDim = dim3((unsigned)(clusters * C));
    cfg.blockDim = dim3(kClusterThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx ? ctx->stream : nullptr;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
};
template <typename Kernel>
cudaError_t clusters_at_once(Kernel kernel, int C, size_t smem, int* most) {
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  ClusterLaunch l(nullptr, 1, C, smem);
  return cudaOccupancyMaxActiveClusters(most, kernel, &l.cfg);
}
template <typename... Params, typename... Args>
cudaError_t launch_clusters(tfjs_cuda_ctx* ctx, void (*kernel)(Params...), int64_t clusters, int C, size_t smem, Args... args) {
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  ClusterLaunch l(ctx, clusters, C, smem);
  return cudaLaunchKernelEx(&l.cfg, kernel, static_cast<Params>(args)...);
}

template <typename TX, typename TY, int V>
int cluster_form(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  // Blocks a row: so many that three blocks' shares fit into an SM's shared memory (one loads while another
  // sums), and with few rows so many that the SMs have a block each.  1000 x 33000: 76 us with the two that
  // gives, 94 with one, 151 with eight; 8 x 33000: 7 us with eight, 12 with one.  Half: 1000 x 33000 45 us with one,
  // as shares of 72 or 144 KB give, 59 with two; 1000 x 65536 86 with two, 111 with one, 119 with four.
  const auto share_of = [&](int C) { return (ceil_div64(a.width / V, C) * V * (int64_t)sizeof(TX) + 31) / 16 * 16; };
  int C = 1;
  while (C < 8 && (share_of(C) > 72 * 1024 || a.rows * C < ctx->sm_count)) C *= 2;
  const int64_t share = share_of(C), cap = 1 << 24;
  const bool cached = share <= 200 * 1024;
  TFJS_CHECK_CUDA(ctx, launch_clusters(ctx, layer_norm_cluster_kernel<TX, TY, V>, a.rows < cap ? a.rows : cap, C,
                                       cached ? (size_t)share : 0, (const TX*)a.x, a.gamma, a.beta, (TY*)a.y, a.stats,
                                       a.rows, a.width, a.epsilon, C, cached ? 1 : 0));
  return post_launch(ctx, "layerNorm (clusters)");
}

// Rows on the 16-byte boundaries: V values, 16 bytes of the result, a load.
template <typename TX, typename TY, int V>
int aligned_form(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  const int64_t w = a.width;
  constexpr int NV = 32 / V;  // 32 values a thread
  if (w <= 1024) {
    if (w <= 4 * V) lanes_form<TX, TY, V, 1, 4>(ctx, a);
    else if (w <= 16 * V) lanes_form<TX, TY, V, 1, 16>(ctx, a);
    else if (w <= 256) lanes_form<TX, TY, V, 8 / V, 32>(ctx, a);
    else if (w <= 512) lanes_form<TX, TY, V, 16 / V, 32>(ctx, a);
    else lanes_form<TX, TY, V, NV, 32>(ctx, a);
    return post_launch(ctx, "layerNorm (lanes)");
  }
  if (w > 16384) return cluster_form<TX, TY, V>(ctx, a);
  if (w <= 256 * 8) block_form<TX, TY, V, NV / 4, 256>(ctx, a);
  else if (w <= 256 * 16) block_form<TX, TY, V, NV / 2, 256>(ctx, a);
  else if (w <= 256 * 32) block_form<TX, TY, V, NV, 256>(ctx, a);
  else block_form<TX, TY, V, NV, 512>(ctx, a);
  return post_launch(ctx, "layerNorm (blocks)");
}

template <typename TX, typename TY, int NW, int G>
int ring_launch(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  constexpr int P = 4 / (int)sizeof(TX), groups = kRingThreads / G;
  const int slot_bytes = ((int)a.width * (int)sizeof(TX) + 31) / 16 * 16;  // one unit more for the row's own offset
  const int smem = groups * 2 * slot_bytes + (G == 32 ? P * ((int)a.width / P + 1) * 2 * P * 4 : 0);
  auto kernel = layer_norm_ring_kernel<TX, TY, NW, G>;
  TFJS_CHECK_CUDA(ctx, allow_smem(kernel, smem));
  // as many blocks an SM as fit, up to six: 100000 x 131 half 41 us, 43 with up to four, 49 with two; 4000 x 7001 half
  // 47 and 57 with two; with three (33000 x 1001 float32, 59 us) two would be ahead, 47
  const int per_sm = smem <= 36 * 1024 ? 6 : smem <= 55 * 1024 ? 4 : smem <= 74 * 1024 ? 3 : 2;
  kernel<<<grid_rows(ctx, ceil_div64(a.rows, groups), per_sm), kRingThreads, smem, ctx->stream>>>(
      (const TX*)a.x, a.gamma, a.beta, (TY*)a.y, a.stats, a.rows, (int)a.width, a.epsilon, slot_bytes);
  return post_launch(ctx, "layerNorm (ring)");
}
// Words of a row that starts at an odd place: width / P + 1 at most.
constexpr int kRingWords = 32 * kRingThreads;
template <typename TX, typename TY>
int ring_form(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  const int64_t words = a.width / (4 / (int)sizeof(TX)) + 1;
  if (words <= 256) return ring_launch<TX, TY, 8, 32>(ctx, a);
  if (words <= 512) return ring_launch<TX, TY, 16, 32>(ctx, a);
  if (words <= 1024) return ring_launch<TX, TY, 32, 32>(ctx, a);
  if (words <= 8 * kRingThreads) return ring_launch<TX, TY, 8, kRingThreads>(ctx, a);
  if (words <= 16 * kRingThreads) return ring_launch<TX, TY, 16, kRingThreads>(ctx, a);
  return ring_launch<TX, TY, 32, kRingThreads>(ctx, a);
}

template <typename TX, typename TY>
int launch_forward(tfjs_cuda_ctx* ctx, const ForwardArgs& a) {
  constexpr int W = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;  // 16 bytes of the result
  const int64_t w = a.width;
  if (w % W == 0) return aligned_form<TX, TY, W>(ctx, a);
  if (w % 2 == 0 && w <= 128) {
    if (w <= 32) lanes_form<TX, TY, 2, 1, 16>(ctx, a);
    else lanes_form<TX, TY, 2, 2, 32>(ctx, a);
    return post_launch(ctx, "layerNorm (lanes)");
  }
  if (w <= 64) {
    if (w <= 16) lanes_form<TX, TY, 1, 1, 16>(ctx, a);
    else lanes_form<TX, TY, 1, 2, 32>(ctx, a);
    return post_launch(ctx, "layerNorm (lanes)");
  }
  if (w / (4 / (int)sizeof(TX)) + 1 <= kRingWords) return ring_form<TX, TY>(ctx, a);
  return w % 2 == 0 ? cluster_form<TX, TY, 2>(ctx, a) : cluster_form<TX, TY, 1>(ctx, a);
}

struct BackwardArgs {
  const void *dy, *x;
  const float *gamma, *stats;
  float *dx, *dgamma, *dbeta;
  int64_t rows, width;
};

// Where `blocks` blocks leave their weights' sums: *partial is a workspace for more than one, and the caller
// gives it back after join_sums.
int place_sums(tfjs_cuda_ctx* ctx, const BackwardArgs& a, int64_t blocks, WeightSums* sums, void** partial, size_t* cap) {
  *partial = nullptr;
  *cap = 0;
  *sums = {a.dgamma, a.dbeta, 0};
  if (blocks == 1 || (!a.dgamma && !a.dbeta)) return TFJS_CUDA_OK;
  const int rc = ctx_alloc(ctx, (size_t)blocks * 2 * a.width * 4, partial, cap);
  if (rc) return rc;
  *sums = {(float*)*partial, (float*)*partial + a.width, 2 * a.width};
  return TFJS_CUDA_OK;
}
int join_sums(tfjs_cuda_ctx* ctx, const BackwardArgs& a, const void* partial, int64_t blocks) {
  if (!partial) return TFJS_CUDA_OK;
  if (blocks <= kFewBlocks)
    launch_dependent(ctx, layer_norm_join_few_kernel, dim3((unsigned)ceil_div64(2 * a.width, 256)), dim3(256),
                     (const float*)partial, a.dgamma, a.dbeta, (int)blocks, a.width);
  else
    launch_dependent(ctx, layer_norm_join_kernel, dim3(grid_rows(ctx, ceil_div64(2 * a.width, 32), 2)), dim3(kJoinThreads),
                     (const float*)partial, a.dgamma, a.dbeta, (int)blocks, a.width);
  return post_launch(ctx, "layerNormBackprop (join)");
}

template <typename TD, typename TX, int V, int MC>
int staged_launch(tfjs_cuda_ctx* ctx, const BackwardArgs& a, StagedParams& p, int blocks, size_t smem) {
  auto kernel = layer_norm_staged_kernel<TD, TX, V, MC>;
  TFJS_CHECK_CUDA(ctx, allow_smem(kernel, smem));
  kernel<<<blocks, kStagedThreads, smem, ctx->stream>>>((const TD*)a.dy, (const TX*)a.x, p);
  return post_launch(ctx, "layerNormBackprop");
}

template <typename TD, typename TX, int V>
int staged_form(tfjs_cuda_ctx* ctx, const BackwardArgs& a) {
  const int width = (int)a.width, row_bytes = width * (int)(sizeof(TD) + sizeof(TX));
  // rows a stage: about 32 KB, so that two blocks with three stages each share an SM, but not so many that
  // the blocks have fewer than two stages each; and all rows where they fit (one block, and no join)
  int R = 1;
  while (R < kMaxStageRows && 2 * R * row_bytes <= 32 * 1024 && ceil_div64(a.rows, 2 * R) >= 4 * ctx->sm_count) R *= 2;
  if (a.rows <= kMaxStageRows && a.rows * row_bytes <= 32 * 1024)
    while (R < a.rows) R *= 2;
  StagedParams p = {};
  p.gamma = a.gamma;
  p.stats = a.stats;
  p.dx = a.dx;
  p.rows = a.rows;
  p.items = ceil_div64(a.rows, R);
  p.width = width;
  p.stage_rows = R;
  p.x_bytes = (R * width * (int)sizeof(TD) + 31) / 16 * 16;  // one 16-byte unit more for the rows' own offset
  p.stage_bytes = p.x_bytes + (R * width * (int)sizeof(TX) + 31) / 16 * 16 + (R + 1) / 2 * 16;
  const int join_bytes = 2 * kStagedThreads * V * 4;  // the row groups' sums reuse the ring
  if (kStages * p.stage_bytes < join_bytes) p.stage_bytes = (join_bytes / kStages + 16) / 16 * 16;
  const int parts = kStagedThreads / R > 32 ? kStagedThreads / R / 32 : 1;
  const size_t smem = (size_t)kStages * p.stage_bytes + (size_t)(width + 3) / 4 * 16 + (size_t)R * parts * 8;
  const int64_t cap = (int64_t)ctx->sm_count * (smem <= 113 * 1024 ? 2 : 1);
  const int blocks = (int)(p.items < cap ? p.items : cap);
  void* partial;
  size_t partial_cap;
  int rc = place_sums(ctx, a, blocks, &p.sums, &partial, &partial_cap);
  if (rc) return rc;
  // 4, 8, 16 or 32 columns a thread
  const int columns = (width + kStagedThreads - 1) / kStagedThreads;
  if (columns <= 4) rc = staged_launch<TD, TX, V, 4 / V>(ctx, a, p, blocks, smem);
  else if (columns <= 8) rc = staged_launch<TD, TX, V, 8 / V>(ctx, a, p, blocks, smem);
  else if (columns <= 16) rc = staged_launch<TD, TX, V, 16 / V>(ctx, a, p, blocks, smem);
  else rc = staged_launch<TD, TX, V, 32 / V>(ctx, a, p, blocks, smem);
  if (!rc) rc = join_sums(ctx, a, partial, blocks);
  ctx_free(ctx, partial, partial_cap);
  return rc;
}

template <typename TD, typename TX, int V>
int backward_cluster_form(tfjs_cuda_ctx* ctx, const BackwardArgs& a) {
  ClusterParams p = {a.gamma, a.stats, a.dx, {}, a.rows, a.width, 1, 0, 0};
  const auto bytes_of = [&](int C) {
    const int64_t share = ceil_div64(a.width / V, C) * V;
    p.C = C;
    p.d_bytes = (int)((share * (int64_t)sizeof(TD) + 31) / 16 * 16);  // one unit more for the row's own offset
    p.slot_bytes = p.d_bytes + (int)((share * (int64_t)sizeof(TX) + 31) / 16 * 16);
    return 2 * (int64_t)p.slot_bytes + share * 8;
  };
  // as for the forward pass: two blocks an SM, and with few rows a block for every SM (1000 x 20000 half 82 us with
  // shares of 112 KB, 146 with 56, 84 with 224; 1000 x 33000 float32 186, 186 and 205, but 1000 x 20000 float32 154,
  // 156 and 139)
  int C = 1;
  int64_t smem = a.width < (1 << 22) ? bytes_of(C) : INT64_MAX;
  while (C < 8 && (smem > 112 * 1024 || a.rows * C < ctx->sm_count)) {
    C *= 2;
    if (a.width < (1 << 22)) smem = bytes_of(C);
  }
  p.C = C;
  const bool ring = smem <= 224 * 1024;
  if (!ring) p.slot_bytes = 0;
  auto kernel = ring ? layer_norm_backprop_cluster_kernel<TD, TX, V, true> : layer_norm_backprop_cluster_kernel<TD, TX, V, false>;
  // as many clusters as run at once (the SMs of a cluster lie together, so it is fewer than SMs / C): one that
  // had to wait for another's end would double the time
  int64_t clusters = a.rows;
  if (clusters * C > ctx->sm_count) {
    int most = 0;
    TFJS_CHECK_CUDA(ctx, clusters_at_once(kernel, C, ring ? (size_t)smem : 0, &most));
    if (clusters > most) clusters = most > 0 ? most : 1;
  }
  void* partial;
  size_t partial_cap;
  int rc = place_sums(ctx, a, clusters, &p.sums, &partial, &partial_cap);
  if (rc) return rc;
  const cudaError_t e = launch_clusters(ctx, kernel, clusters, C, ring ? (size_t)smem : 0, (const TD*)a.dy, (const TX*)a.x, p);
  if (e != cudaSuccess) rc = set_error(ctx, TFJS_CUDA_ERR_CUDA, "layerNormBackprop failed: %s", cudaGetErrorString(e));
  if (!rc) rc = post_launch(ctx, "layerNormBackprop (clusters)");
  if (!rc) rc = join_sums(ctx, a, partial, clusters);
  ctx_free(ctx, partial, partial_cap);
  return rc;
}

template <typename TD, typename TX>
int launch_backward(tfjs_cuda_ctx* ctx, const BackwardArgs& a) {
  if (a.width <= kStagedWidth) return a.width % 4 == 0 ? staged_form<TD, TX, 4>(ctx, a) : staged_form<TD, TX, 1>(ctx, a);
  return a.width % 4 == 0 ? backward_cluster_form<TD, TX, 4>(ctx, a) : backward_cluster_form<TD, TX, 1>(ctx, a);
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
  return launch(ctx, {x->ptr, f32_ptr(gamma), f32_ptr(beta), y->ptr, f32_out(stats), rows, width, epsilon});
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
  if (rows == 0) {  // the sum of no rows
    for (int i = 1; i < 3; i++)
      if (out[i]) TFJS_CHECK_CUDA(ctx, cudaMemsetAsync(out[i]->ptr, 0, (size_t)width * 4, ctx->stream));
    return TFJS_CUDA_OK;
  }
  if (!out[0] && !out[1] && !out[2]) return TFJS_CUDA_OK;
  const bool hd = dy->dtype == TFJS_F16, hx = x->dtype == TFJS_F16;
  auto launch = hd ? (hx ? launch_backward<__half, __half> : launch_backward<__half, float>)
                   : (hx ? launch_backward<float, __half> : launch_backward<float, float>);
  return launch(ctx, {dy->ptr, x->ptr, f32_ptr(gamma), f32_ptr(stats), f32_out(out[0]), f32_out(out[1]), f32_out(out[2]),
                      rows, width});
}

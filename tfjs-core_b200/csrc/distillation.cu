// Distillation loss over a teacher's top logits, and its gradient.
//
// For each row, with student logits z over all classes, temperature T and the teacher's list of K
// (class, logit) entries, of which those with a class in [0, classes) and a logit above -inf count:
//
//   q = softmax(z / T) over all classes,   p = softmax(u / T) over the counting entries
//   loss = T^2 sum_k p_k (log p_k - log q_{i_k})              (T^2 keeps the gradient's size)
//   dz_v = dloss T (q_v - sum of p_k over the entries with i_k == v)
//
// A row without a counting entry has loss 0 and gradient 0.
//
// Both softmaxes are taken relative to their largest logit, in raw units: exp2((z - max) * k) with
// k = log2(e) / T, so that a row of the type's lowest values is still a uniform row.  The forward
// pass leaves (max z, log2 of z's sum, max u, log2 of u's sum) of each row for the backward pass,
// apart, because the logarithm would be lost beside a large maximum.  max u is -inf for an empty list.
//
// Both passes stream the logits once.  A row starts anywhere, so its elements before the first 16-byte
// boundary and behind the last one are taken one by one and all others in 16-byte loads; the float32
// gradient has the same element offsets, so its stores are aligned too.
// The gradient is bound by memory: 8192 x 32000 half with 64 entries 239 us, 1.57 GB at 6.6 TB/s; with 16-byte
// loads of halves, whose gradients are then two stores a lane that do not lie side by side, 296 us; with four
// units a thread in place of eight 264 us.  The loss of the same rows takes 112 us, 524 MB at 4.7 TB/s, and fills
// nothing (DRAM 50 % of nominal, the exp2 unit 51 %, issue slots 56 %): every row ends in three joins of its
// block, during which that block loads nothing.  Single-value arithmetic instead of the packed one 172 us, two
// blocks of 512 threads an SM instead of five of 256 129 us.
// Exponentials are the hardware's approximation (ex2.approx, 2 ulp), in p, in q and in the sums.
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace cg = cooperative_groups;

namespace {

// The loss keeps a list in registers.  The gradient looks every listed class of a tile up in the whole list, top^2 / 4
// reads of shared memory a row at worst: 2048 x 32000 half 55 us with 1 entry, 66 with 64, 80 with 128, 135 with 256,
// 467 with 512, 1806 with 1024.
constexpr int kMaxTop = 1024;
constexpr int kThreads = 256;      // of a block of the loss
constexpr int kGradThreads = 256;  // of a block of the gradient
constexpr int kBatch = 8;          // 16-byte loads in flight a thread of the loss
constexpr int kGradBatch = 8;      // and of the gradient
constexpr float kLn2 = 0.693147180559945f;
constexpr float kLog2e = 1.44269504088896f;

// 2^v by the hardware's approximation (2 ulp); below 2^-126 it gives 0
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const __half* p) { return __half2float(*p); }

// Two float32 values in one register pair, for the packed instructions (one issue slot for two values).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 bytes of logits as they are stored: P pairs.
template <typename T>
struct Unit {
  static constexpr int P = 8 / (int)sizeof(T);
  uint4 q;
  __device__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
  __device__ void fill_low() {  // -inf
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xfc00fc00u;
    q = make_uint4(w, w, w, w);
  }
  __device__ float2 get(int i) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
};
// Four of them.
template <typename T>
struct alignas(4 * sizeof(T)) Raw4 {
  T v[4];
  __device__ float2 get(int i) const { return make_float2(load_one(&v[2 * i]), load_one(&v[2 * i + 1])); }
};
// Largest value of N units, NaN if there is one (halves are compared two at a time, as halves).
template <int N>
__device__ __forceinline__ float units_max(const Unit<float> (&u)[N]) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float2 f = u[i].get(j);
      m = max_nan(m, max_nan(f.x, f.y));
    }
  return m;
}
template <int N>
__device__ __forceinline__ float units_max(const Unit<__half> (&u)[N]) {
  uint32_t low = 0xfc00fc00u;
  __half2 m = *reinterpret_cast<__half2*>(&low);
#pragma unroll
  for (int i = 0; i < N; i++) {
    const uint32_t w[4] = {u[i].q.x, u[i].q.y, u[i].q.z, u[i].q.w};
#pragma unroll
    for (int j = 0; j < 4; j++) m = __hmax2_nan(m, *reinterpret_cast<const __half2*>(&w[j]));
  }
  const float2 f = __half22float2(m);
  return max_nan(f.x, f.y);
}

// The exponent (z - m) k - l of a value z is taken as fma(z, k, shift), shift = -(m k + l): one packed
// instruction for two values.  What the rounding of `shift` loses is the same for all of them, so it
// goes into a factor for the whole: 2^((z - m) k - l) = 2^fma(z, k, shift) * factor.  Where m k + l is too
// large for that (a row of the type's lowest values), `exact` is set and the difference comes first.
struct Shift {
  float shift, factor;
  bool exact;
  __device__ Shift(float m, float k, float l) {
    const float hi = m * k, lo = fmaf(m, k, -hi);
    const float sum = hi + l, back = sum - hi;
    const float lost = (hi - (sum - back)) + (l - back) + lo;
    shift = -sum;
    factor = 1.f - lost * kLn2;  // |lost| <= 2^-13: 2^-lost to 4e-9
    exact = !(fabsf(sum) < 2048.f);
  }
};

// NaN-keeping maximum, or sum, of two values over G threads: a warp, or the whole block of G (`scratch`:
// G / 32 pairs that no other call uses).
template <int G, bool MAX>
__device__ __forceinline__ float2 group_reduce(float a, float b, float2* scratch) {
  auto join = [](float p, float q) { return MAX ? max_nan(p, q) : p + q; };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
    b = join(b, __shfl_xor_sync(0xffffffffu, b, o));
  }
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const float2 v = scratch[threadIdx.x & (G / 32 - 1)];
    a = v.x;
    b = v.y;
#pragma unroll
    for (int o = G / 64; o > 0; o >>= 1) {
      a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
      b = join(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
  }
  return make_float2(a, b);
}

// Where a row's 16-byte units lie: `head` elements before them, `vecs` units, `tail` elements behind.
template <int V>
struct RowSplit {
  int head, vecs, tail;
  __device__ RowSplit(int64_t first, int classes) {
    head = (int)(-first & (V - 1));
    if (head > classes) head = classes;
    vecs = (classes - head) / V;
    tail = classes - head - vecs * V;
  }
  // element of the i-th of the head + tail ones
  __device__ int loose(int i) const { return i < head ? i : i + vecs * V; }
};

// 2^((z - m) k) of a value (or a part's maximum) z relative to the maximum m, 0 where all is -inf
__device__ __forceinline__ float shifted(float z, float m, float k) { return exp2_approx((z - (m == -INFINITY ? 0.f : m)) * k); }

// G threads a row (a warp, or a block), C blocks a row (only with whole blocks).  NK: teacher entries a
// thread, G * NK >= top.
template <typename TZ, typename TU, int G, int NK>
__global__ void __launch_bounds__(G > 32 ? kThreads : 256) distillation_kernel(
    const TZ* __restrict__ z, const TU* __restrict__ u, const int32_t* __restrict__ indices, float* __restrict__ loss,
    float* __restrict__ stats, int64_t rows, int classes, int top, float temperature, int C) {
  constexpr int V = 16 / (int)sizeof(TZ);
  __shared__ float2 scratch[3][kThreads / 32];
  __shared__ float2 slot;
  const int t = threadIdx.x & (G - 1);
  const int rank = G > 32 ? (int)(blockIdx.x % C) : 0;
  const int64_t row = G > 32 ? blockIdx.x / C : (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (G == 32 && row >= rows) return;  // whole warps
  const float inv_t = 1.f / temperature, k2 = kLog2e * inv_t;
  const int64_t first = row * classes;
  const TZ* zr = z + first;
  const RowSplit<V> split(first, classes);

  // the teacher's entries, fetched ahead of the row (by the row's first block; the others have none)
  float tu[NK], tz[NK];
#pragma unroll
  for (int i = 0; i < NK; i++) {
    const int e = t + i * G;
    tu[i] = -INFINITY;
    tz[i] = 0.f;
    if (rank == 0 && e < top) {
      const int32_t at = indices[row * top + e];
      if (at >= 0 && at < classes) {
        tu[i] = load_one(u + row * top + e);
        tz[i] = load_one(zr + at);
      }
    }
  }

  // ---- one pass over the row: running maximum and sum
  float m = -INFINITY, s = 0.f;
  if (rank == 0 && t < split.head + split.tail) {
    m = load_one(zr + split.loose(t));
    s = shifted(m, m, k2);
  }
  {
    const TZ* body = zr + split.head;
    const int lo = (int)((int64_t)split.vecs * rank / C), hi = (int)((int64_t)split.vecs * (rank + 1) / C);
    const uint64_t kk = pair(k2, k2);
    for (int j = lo + t; j < hi; j += G * kBatch) {
      Unit<TZ> q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        if (j + i * G < hi) q[i].load(body + (int64_t)(j + i * G) * V);
        else q[i].fill_low();
      }
      const float b = max_nan(m, units_max(q));
      const float at = b == -INFINITY ? 0.f : b;
      const Shift sh(at, k2, 0.f);
      s *= exp2_approx((m - at) * k2);  // m = -inf: 0 * s = 0
      if (!sh.exact) {
        const uint64_t shift2 = pair(sh.shift, sh.shift);
        uint64_t sum = 0;
#pragma unroll
        for (int i = 0; i < kBatch; i++)
#pragma unroll
          for (int k = 0; k < Unit<TZ>::P; k++) {
            const float2 f = q[i].get(k), e = unpair(fma_pair(pair(f.x, f.y), kk, shift2));
            sum = add_pair(sum, pair(exp2_approx(e.x), exp2_approx(e.y)));
          }
        const float2 f = unpair(sum);
        s = fmaf(f.x + f.y, sh.factor, s);
      } else {
#pragma unroll
        for (int i = 0; i < kBatch; i++)
#pragma unroll
          for (int k = 0; k < Unit<TZ>::P; k++) {
            const float2 f = q[i].get(k);
            s += exp2_approx((f.x - at) * k2) + exp2_approx((f.y - at) * k2);
          }
      }
      m = b;
    }
  }
  float um = -INFINITY;
#pragma unroll
  for (int i = 0; i < NK; i++) um = max_nan(um, tu[i]);
  const float2 big = group_reduce<G, true>(m, um, scratch[0]);
  float all = big.x;
  um = big.y;
  const float ut = um == -INFINITY ? 0.f : um;
  float e = 0.f;
#pragma unroll
  for (int i = 0; i < NK; i++) e += exp2_approx((tu[i] - ut) * k2);
  const float2 sums = group_reduce<G, false>(s * shifted(m, all, k2), e, scratch[1]);
  s = sums.x;
  if (G > 32 && C > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) slot = make_float2(all, s);
    cluster.sync();
    if (rank == 0) {
      float most = -INFINITY, sum = 0.f;
      for (int i = 0; i < C; i++) most = max_nan(most, cluster.map_shared_rank(&slot, i)->x);
      for (int i = 0; i < C; i++) {
        const float2 o = *cluster.map_shared_rank(&slot, i);
        sum += o.y * shifted(o.x, most, k2);
      }
      all = most;
      s = sum;
    }
    cluster.sync();  // the other blocks' slots have been read
    if (rank != 0) return;
  }
  // ---- the loss
  const float ls = log2f(s);
  float uls = 0.f, l = 0.f;
  if (um != -INFINITY) {  // the same for all threads of the row
    uls = log2f(sums.y);
#pragma unroll
    for (int i = 0; i < NK; i++) {
      const float lp = (tu[i] - um) * k2 - uls, p = exp2_approx(lp);
      if (p != 0.f) l += p * (lp - ((tz[i] - all) * k2 - ls));
    }
    l = group_reduce<G, false>(l, 0.f, scratch[2]).x * kLn2;
  }
  if (t == 0) {
    loss[row] = temperature * (temperature * l);  // the square alone may leave the range that the loss is in
    if (stats) *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(all, ls, um, uls);
  }
}

template <int G>
__device__ __forceinline__ void group_sync() {
  if (G > 32) __syncthreads();
  else __syncwarp();
}

// G threads take a tile of G * kGradBatch units of a row (the first tile also the loose elements): all
// classes get c q_v, then the tile's listed classes are written again with their p taken off, by the
// first entry that names the class.  `room`: entries of shared memory a group.
template <typename TZ, typename TU, int G>
__global__ void __launch_bounds__(kGradThreads) distillation_backprop_kernel(
    const float* __restrict__ dloss, const TZ* __restrict__ z, const TU* __restrict__ u,
    const int32_t* __restrict__ indices, const float* __restrict__ stats, float* __restrict__ dz, int64_t rows,
    int classes, int top, float temperature, int tiles, int room) {
  constexpr int V = 4;  // values a unit: their float32 gradient is one 16-byte store, side by side over the lanes
  extern __shared__ __align__(16) uint8_t smem[];
  const int t = threadIdx.x & (G - 1), group = threadIdx.x / G;
  const int64_t item = (int64_t)blockIdx.x * (kGradThreads / G) + group;
  const int64_t row = item / tiles;
  if (row >= rows) return;  // whole groups
  const int tile = (int)(item - row * tiles);
  int32_t* s_i = reinterpret_cast<int32_t*>(smem) + group * 2 * room;
  float* s_p = reinterpret_cast<float*>(s_i) + room;
  const float k2 = kLog2e * (1.f / temperature);
  const int64_t first = row * classes;
  const TZ* zr = z + first;
  float* dr = dz + first;
  const RowSplit<V> split(first, classes);
  const int v0 = tile * G * kGradBatch;

  Raw4<TZ> q[kGradBatch];
#pragma unroll
  for (int i = 0; i < kGradBatch; i++)
    if (v0 + i * G + t < split.vecs) q[i] = *reinterpret_cast<const Raw4<TZ>*>(zr + split.head + (int64_t)(v0 + i * G + t) * V);
  const float4 st = *reinterpret_cast<const float4*>(stats + 4 * row);
  const float c = dloss[row] * temperature;
  const bool empty = st.z == -INFINITY;
  for (int e = t; e < room; e += G) {
    int32_t at = -1;
    float p = 0.f;
    if (e < top) {
      at = indices[row * top + e];
      p = exp2_approx((load_one(u + row * top + e) - st.z) * k2 - st.w);
      if (at < 0 || at >= classes) at = -1;
    }
    s_i[e] = at;
    s_p[e] = p;
  }
  const Shift sh(st.x, k2, st.y);
  const uint64_t kk = pair(k2, k2), shift2 = pair(sh.shift, sh.shift);
  const uint64_t c2 = pair(c * sh.factor, c * sh.factor);
#pragma unroll
  for (int i = 0; i < kGradBatch; i++) {
    if (v0 + i * G + t >= split.vecs) continue;
    float o[V];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float2 f = q[i].get(h);
      float2 e;
      if (!sh.exact) {
        e = unpair(fma_pair(pair(f.x, f.y), kk, shift2));
        e = unpair(mul_pair(pair(exp2_approx(e.x), exp2_approx(e.y)), c2));
      } else {
        e = make_float2(c * exp2_approx((f.x - st.x) * k2 - st.y), c * exp2_approx((f.y - st.x) * k2 - st.y));
      }
      o[2 * h] = empty ? 0.f : e.x;
      o[2 * h + 1] = empty ? 0.f : e.y;
    }
    store_vec<V>(dr + split.head + (int64_t)(v0 + i * G + t) * V, o);
  }
  if (tile == 0 && t < split.head + split.tail) {
    const int at = split.loose(t);
    dr[at] = empty ? 0.f : c * exp2_approx((load_one(zr + at) - st.x) * k2 - st.y);
  }
  if (empty) return;  // the whole group
  group_sync<G>();    // the list is there, and the classes are written before they are written again
  const int lo = split.head + v0 * V, hi = split.head + min(v0 + G * kGradBatch, split.vecs) * V;
  for (int e = t; e < top; e += G) {
    const int32_t at = s_i[e];
    if (at < 0) continue;
    const bool loose = at < split.head || at >= split.head + split.vecs * V;
    if (loose ? tile != 0 : (at < lo || at >= hi)) continue;
    float p = 0.f;
    bool is_first = true;
    for (int j = 0; j < top; j += 4) {  // room is a multiple of 4; the entries behind top hold -1
      const int4 q = *reinterpret_cast<const int4*>(s_i + j);
      if (q.x == at) is_first &= j >= e, p += s_p[j];
      if (q.y == at) is_first &= j + 1 >= e, p += s_p[j + 1];
      if (q.z == at) is_first &= j + 2 >= e, p += s_p[j + 2];
      if (q.w == at) is_first &= j + 3 >= e, p += s_p[j + 3];
    }
    if (is_first) dr[at] = c * (exp2_approx((load_one(zr + at) - st.x) * k2 - st.y) - p);
  }
}

struct Operands {
  TensorEntry *z, *u, *indices;
};

int get_operands(tfjs_cuda_ctx* ctx, tfjs_tensor_id z, tfjs_tensor_id u, tfjs_tensor_id indices, int64_t rows,
                 int64_t classes, int64_t top, float temperature, Operands* o) {
  TFJS_REQUIRE(ctx, rows >= 0 && classes >= 0 && top >= 0, "negative extent");
  TFJS_REQUIRE(ctx, classes < (1ll << 31) - 65536 && rows < (1ll << 27) && rows <= (1ll << 60) / (classes > kMaxTop ? classes : kMaxTop),
               "distillationLoss: too many rows or classes");
  TFJS_REQUIRE(ctx, top <= kMaxTop, "distillationLoss: a teacher's list holds at most %d entries, got %lld", kMaxTop,
               (long long)top);
  const float k2 = kLog2e * (1.f / temperature);
  TFJS_REQUIRE(ctx, temperature > 0.f && temperature - temperature == 0.f && k2 - k2 == 0.f,
               "distillationLoss: the temperature and its reciprocal must be positive and finite");
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
int launch_forward(tfjs_cuda_ctx* ctx, const Operands& o, float* loss, float* stats, int64_t rows, int64_t classes,
                   int top, float temperature) {
  const TZ* z = (const TZ*)o.z->ptr;
  const TU* u = (const TU*)o.u->ptr;
  const int32_t* indices = (const int32_t*)o.indices->ptr;
  // A warp a row, for short rows and, where the rows fill the SMs with warps, for longer ones: a block's three
  // joins cost it 5 us whatever the row holds.  8192 rows of 1000 classes: 10 us, 49 with blocks; of 8000 (half)
  // 38 and 72; of 16000 the block is ahead (4096 rows: 61 and 55), and so it is with 100 rows of 4000 (6 and 4).
  if (top <= 128 && (classes <= 1024 || (classes <= 8192 && rows >= 8 * ctx->sm_count))) {
    distillation_kernel<TZ, TU, 32, 4><<<(unsigned)ceil_div64(rows, 8), 256, 0, ctx->stream>>>(
        z, u, indices, loss, stats, rows, (int)classes, top, temperature, 1);
    return post_launch(ctx, "distillationLoss (warps)");
  }
  // few rows: up to 8 blocks share one, while each still has 8192 classes or more (7 rows of 131101: 6 us, 12
  // with a block each)
  int C = 1;
  while (C < 8 && rows * C * 2 <= 2 * ctx->sm_count && classes / (2 * C) >= 8192) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TFJS_CHECK_CUDA(ctx, cudaLaunchKernelEx(&cfg, distillation_kernel<TZ, TU, kThreads, kMaxTop / kThreads>, z, u, indices, loss, stats, rows,
                                          (int)classes, top, temperature, C));
  return post_launch(ctx, "distillationLoss");
}

template <typename TZ, typename TU>
int launch_backward(tfjs_cuda_ctx* ctx, const float* dloss, const Operands& o, const float* stats, float* dz,
                    int64_t rows, int64_t classes, int top, float temperature) {
  constexpr int V = 4;
  // a warp takes up to four tiles of 1024 classes: a block's tile is 8192 (8192 rows of 1000 classes: 11 us, 31
  // with blocks; of 4000 40 and 50; of 8000 half 87 and 74)
  const bool warps = classes <= 4 * 32 * kGradBatch * V && top <= 128;
  const int G = warps ? 32 : kGradThreads, groups = kGradThreads / G;
  const int64_t tiles = classes <= G * kGradBatch * V ? 1 : ceil_div64(classes, (int64_t)G * kGradBatch * V);
  const int64_t blocks = ceil_div64(rows * tiles, groups);
  TFJS_REQUIRE(ctx, blocks < (1ll << 31), "distillationLossBackprop: too many rows times classes");
  const int room = (top + 3) / 4 * 4;
  auto kernel = warps ? distillation_backprop_kernel<TZ, TU, 32> : distillation_backprop_kernel<TZ, TU, kGradThreads>;
  kernel<<<(unsigned)blocks, kGradThreads, (size_t)groups * room * 8, ctx->stream>>>(
      dloss, (const TZ*)o.z->ptr, (const TU*)o.u->ptr, (const int32_t*)o.indices->ptr, stats, dz, rows, (int)classes, top,
      temperature, (int)tiles, room);
  return post_launch(ctx, "distillationLossBackprop");
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
  if (!rc && stats_id) rc = get_rows(ctx, stats_id, 4 * rows, "distillationLoss statistics", &stats);
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
  return launch(ctx, o, (float*)loss->ptr, stats ? (float*)stats->ptr : nullptr, rows, classes, (int)top, temperature);
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
  if (!rc) rc = get_rows(ctx, stats_id, 4 * rows, "distillationLoss statistics", &stats);
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
  return launch(ctx, (const float*)dloss->ptr, o, (const float*)stats->ptr, (float*)dz->ptr, rows, classes, (int)top,
                temperature);
}

// Embedding lookup with scaling, and the gradient of its table.
//
//   out[t] = scale * table[i_t],      zeros where i_t lies outside [0, vocab) (padding)
//   dtable[v] = scale * sum of dy[t] over the tokens t with i_t == v, in the order of t
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;

// ---- lookup ----------------------------------------------------------------------------------------
// A quantised table's value is the float32 that decodeWeights gives (io_utils.ts:139): a float64
// product and sum, rounded once.
struct Decode {
  double scale, min;
};
template <int V>
__device__ __forceinline__ void load_row(const uint8_t* p, Decode q, float (&v)[V]) {
  uint32_t word = 0;
  if constexpr (V == 4) word = *reinterpret_cast<const uint32_t*>(p);
  else word = *p;
#pragma unroll
  for (int i = 0; i < V; i++)
    v[i] = (float)__dadd_rn(__dmul_rn((double)((word >> (8 * i)) & 255u), q.scale), q.min);
}
template <int V, typename T>
__device__ __forceinline__ void load_row(const T* p, Decode, float (&v)[V]) {
  load_vec<V>(p, v);
}

// L lanes a token, V columns a lane and step.
template <typename TT, typename TO, int V, int L>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const TT* __restrict__ table,
                                                            const int32_t* __restrict__ indices, TO* __restrict__ out,
                                                            int64_t tokens, int64_t vocab, int width, float scale,
                                                            Decode q) {
  const int lane = threadIdx.x & (L - 1), vecs = width / V;
  const int64_t step = (int64_t)gridDim.x * (kThreads / L);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L; t < tokens; t += step) {
    const int64_t v = indices[t];
    const bool there = v >= 0 && v < vocab;
    const TT* row = table + (there ? v : 0) * width;
    TO* o = out + t * width;
#pragma unroll 4
    for (int j = lane; j < vecs; j += L) {
      float r[V];
      if (there) {
        load_row<V>(row + j * V, q, r);
#pragma unroll
        for (int i = 0; i < V; i++) r[i] *= scale;
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) r[i] = 0.f;
      }
      store_vec<V>(o + j * V, r);
    }
  }
}

// ---- gradient: tokens sorted by table row --------------------------------------------------------------
// Stable least-significant-digit radix sort of (table row, token) pairs; a token outside the table
// gets the key `vocab`, behind all others.  Within a block each warp owns a run of keys: it counts
// their digits into its own counters (the lanes of equal digits agree through match_any, one of them
// adds), the counters are summed over the warps and blocks, and the same walk then gives each key its
// place.  No atomics: equal inputs give the same order, ascending tokens within each table row.
constexpr int kSortThreads = 1024, kSortWarps = 32;
constexpr int kSortKeys = 8192;  // of one block
constexpr int kMaxBins = 512;

struct Digits {
  int passes, bits;
};
Digits digits_of(int64_t vocab) {
  int total = 1;
  while (total < 32 && (vocab >> total)) total++;
  const int passes = (total + 8) / 9;
  return {passes, (total + passes - 1) / passes};
}

// One walk over the block's keys.  PLACE false: counts[warp][digit]; true: place(key, token, place within
// the block's own keys of that digit), from the exclusive prefix over the warps that counts then holds.
template <bool PLACE, typename F>
__device__ __forceinline__ void walk_keys(const uint32_t* keys, const uint32_t* tokens, int n, int per_warp, int shift,
                                          int bins, uint16_t* counts, F place) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* mine = counts + warp * bins;
  for (int i = 0; i < per_warp; i += 32) {
    const int at = warp * per_warp + i + lane;
    const bool there = at < n;
    if (!__any_sync(0xffffffffu, there)) break;
    const uint32_t key = there ? keys[at] : 0;
    const uint32_t digit = there ? (key >> shift) & (uint32_t)(bins - 1) : 0xffffffffu;
    const uint32_t peers = __match_any_sync(0xffffffffu, digit);
    const int before = __popc(peers & ((1u << lane) - 1));
    uint32_t base = 0;
    if (there) base = mine[digit];
    __syncwarp();
    if (there && before == 0) mine[digit] = (uint16_t)(base + __popc(peers));
    __syncwarp();
    if (PLACE && there) place(key, tokens[at], digit, base + before);
  }
}

// counts[warp][digit] -> exclusive prefix over the warps; returns the block's total of digit threadIdx.x.
__device__ __forceinline__ uint32_t prefix_over_warps(uint16_t* counts, int bins) {
  uint32_t sum = 0;
  if ((int)threadIdx.x < bins)
    for (int w = 0; w < kSortWarps; w++) {
      const uint32_t c = counts[w * bins + threadIdx.x];
      counts[w * bins + threadIdx.x] = (uint16_t)sum;
      sum += c;
    }
  return sum;
}

// Exclusive sum over the threads of the block; `warps` holds 32 values.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* warps) {
  const int lane = threadIdx.x & 31;
  uint32_t s = v;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warps[threadIdx.x >> 5] = s;
  __syncthreads();
  uint32_t w = warps[lane];
  uint32_t before = 0;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  before = __shfl_sync(0xffffffffu, w, (threadIdx.x >> 5) ? (threadIdx.x >> 5) - 1 : 0);
  return (threadIdx.x >> 5 ? before : 0u) + s - v;
}

struct SortShared {
  uint32_t keys[2][kSortKeys], tokens[2][kSortKeys];
  uint16_t counts[kSortWarps * kMaxBins];
  uint32_t totals[kMaxBins], base[kMaxBins], warps[32];
};

// Up to 8 * 8192 tokens: the first cluster sorts them in its blocks' shared memory, the other blocks
// write the table gradient's zeros meanwhile.
__global__ void __launch_bounds__(kSortThreads, 1) embedding_sort_kernel(
    const int32_t* __restrict__ indices, int tokens, uint32_t vocab, int passes, int bits, uint32_t* __restrict__ sorted_keys,
    uint32_t* __restrict__ sorted_tokens, float* __restrict__ dtable, int64_t values) {
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks();
  if ((int)blockIdx.x >= blocks) {
    const int64_t stride = (int64_t)(gridDim.x - blocks) * kSortThreads;
    const int64_t first = (int64_t)(blockIdx.x - blocks) * kSortThreads + threadIdx.x;
    float4* quads = reinterpret_cast<float4*>(dtable);
    for (int64_t i = first; i < values / 4; i += stride) quads[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (first < (values & 3)) dtable[(values & ~3ll) + first] = 0.f;
    return;
  }
  extern __shared__ __align__(16) uint8_t raw[];
  SortShared& s = *reinterpret_cast<SortShared*>(raw);
  const int rank = (int)cluster.block_rank();
  const int share = ((tokens + blocks - 1) / blocks + kSortThreads - 1) / kSortThreads * kSortThreads;
  const int n = max(0, min(share, tokens - rank * share));
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    const int32_t v = indices[rank * share + i];
    s.keys[0][i] = (uint32_t)v < vocab ? (uint32_t)v : vocab;
    s.tokens[0][i] = (uint32_t)(rank * share + i);
  }
  for (int pass = 0; pass < passes; pass++) {
    const int from = pass & 1, shift = pass * bits;
    for (int i = threadIdx.x; i < kSortWarps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(s.counts)[i] = 0;
    __syncthreads();
    walk_keys<false>(s.keys[from], s.tokens[from], n, share / kSortWarps, shift, bins, s.counts,
                     [](uint32_t, uint32_t, uint32_t, uint32_t) {});
    __syncthreads();
    const uint32_t total = prefix_over_warps(s.counts, bins);
    if ((int)threadIdx.x < bins) s.totals[threadIdx.x] = total;
    cluster.sync();
    uint32_t all = 0, before = 0;
    if ((int)threadIdx.x < bins)
      for (int r = 0; r < blocks; r++) {
        const uint32_t c = cluster.map_shared_rank(s.totals, r)[threadIdx.x];
        all += c;
        if (r < rank) before += c;
      }
    const uint32_t smaller = block_exclusive(all, s.warps);
    if ((int)threadIdx.x < bins) s.base[threadIdx.x] = smaller + before;
    __syncthreads();
    const bool last = pass + 1 == passes;
    walk_keys<true>(s.keys[from], s.tokens[from], n, share / kSortWarps, shift, bins, s.counts,
                    [&](uint32_t key, uint32_t token, uint32_t digit, uint32_t place) {
                      const int g = (int)(s.base[digit] + place);
                      if (last) {
                        sorted_keys[g] = key;
                        sorted_tokens[g] = token;
                      } else {
                        const int to = g / share, slot = g - to * share;
                        cluster.map_shared_rank(s.keys[from ^ 1], to)[slot] = key;
                        cluster.map_shared_rank(s.tokens[from ^ 1], to)[slot] = token;
                      }
                    });
    cluster.sync();  // the pass's writes have arrived; nobody reads this block's totals any more
  }
}

// More tokens: three launches a pass, over tiles of 8192 keys.
__device__ __forceinline__ int load_tile(const int32_t* indices, const uint32_t* keys_in, const uint32_t* tokens_in,
                                         int64_t tokens, uint32_t vocab, SortShared& s) {
  const int64_t first = (int64_t)blockIdx.x * kSortKeys;
  const int n = (int)(tokens - first < kSortKeys ? tokens - first : kSortKeys);
  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    if (indices) {
      const int32_t v = indices[first + i];
      s.keys[0][i] = (uint32_t)v < vocab ? (uint32_t)v : vocab;
      s.tokens[0][i] = (uint32_t)(first + i);
    } else {
      s.keys[0][i] = keys_in[first + i];
      s.tokens[0][i] = tokens_in[first + i];
    }
  }
  return n;
}
// counts[digit][tile]
__global__ void __launch_bounds__(kSortThreads, 1) embedding_count_kernel(const int32_t* indices, const uint32_t* keys_in,
                                                                         const uint32_t* tokens_in, int64_t tokens,
                                                                         uint32_t vocab, int shift, int bits,
                                                                         uint32_t* counts) {
  extern __shared__ __align__(16) uint8_t raw[];
  SortShared& s = *reinterpret_cast<SortShared*>(raw);
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < kSortWarps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(s.counts)[i] = 0;
  const int n = load_tile(indices, keys_in, tokens_in, tokens, vocab, s);
  __syncthreads();
  walk_keys<false>(s.keys[0], s.tokens[0], n, kSortKeys / kSortWarps, shift, bins, s.counts,
                   [](uint32_t, uint32_t, uint32_t, uint32_t) {});
  __syncthreads();
  const uint32_t total = prefix_over_warps(s.counts, bins);
  if ((int)threadIdx.x < bins) counts[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = total;
}
// Exclusive sum in place, by one block.
__global__ void __launch_bounds__(kSortThreads, 1) embedding_scan_kernel(uint32_t* counts, int64_t n) {
  __shared__ uint32_t warps[32];
  __shared__ uint32_t carry_out;
  uint32_t carry = 0;
  for (int64_t first = 0; first < n; first += kSortThreads) {
    const int64_t i = first + threadIdx.x;
    const uint32_t v = i < n ? counts[i] : 0;
    const uint32_t before = block_exclusive(v, warps) + carry;
    if (i < n) counts[i] = before;
    if (threadIdx.x == kSortThreads - 1) carry_out = before + v;
    __syncthreads();
    carry = carry_out;
    __syncthreads();
  }
}
__global__ void __launch_bounds__(kSortThreads, 1) embedding_scatter_kernel(
    const int32_t* indices, const uint32_t* keys_in, const uint32_t* tokens_in, int64_t tokens, uint32_t vocab, int shift,
    int bits, const uint32_t* counts, uint32_t* keys_out, uint32_t* tokens_out) {
  extern __shared__ __align__(16) uint8_t raw[];
  SortShared& s = *reinterpret_cast<SortShared*>(raw);
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < kSortWarps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(s.counts)[i] = 0;
  const int n = load_tile(indices, keys_in, tokens_in, tokens, vocab, s);
  __syncthreads();
  walk_keys<false>(s.keys[0], s.tokens[0], n, kSortKeys / kSortWarps, shift, bins, s.counts,
                   [](uint32_t, uint32_t, uint32_t, uint32_t) {});
  __syncthreads();
  prefix_over_warps(s.counts, bins);
  if ((int)threadIdx.x < bins) s.base[threadIdx.x] = counts[(int64_t)threadIdx.x * gridDim.x + blockIdx.x];
  __syncthreads();
  walk_keys<true>(s.keys[0], s.tokens[0], n, kSortKeys / kSortWarps, shift, bins, s.counts,
                  [&](uint32_t key, uint32_t token, uint32_t digit, uint32_t place) {
                    const uint32_t g = s.base[digit] + place;
                    keys_out[g] = key;
                    tokens_out[g] = token;
                  });
}

// ---- gradient: sums over the sorted tokens -----------------------------------------------------------------
// A warp takes 32 sorted tokens and 32 V columns.  A table row whose tokens all lie in this chunk is
// finished here.  One that began in an earlier chunk leaves this chunk's share in partial[chunk][0], one
// that begins here and goes on in partial[chunk][1].
constexpr int kChunk = 32;
constexpr int kBatch = 8;  // rows of dy in flight a warp

template <typename TD, int V>
__global__ void __launch_bounds__(kThreads) embedding_sum_kernel(const TD* __restrict__ dy,
                                                                const uint32_t* __restrict__ keys,
                                                                const uint32_t* __restrict__ order,
                                                                float* __restrict__ dtable, float* __restrict__ partial,
                                                                int64_t tokens, uint32_t vocab, int64_t width, float scale,
                                                                int64_t tiles, int64_t items) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (item >= items) return;
  const int64_t chunk = item / tiles, col = ((item - chunk * tiles) * 32 + lane) * V;
  const int64_t p0 = chunk * kChunk;
  const uint32_t key = p0 + lane < tokens ? keys[p0 + lane] : vocab;
  const uint32_t token = p0 + lane < tokens ? order[p0 + lane] : 0;
  uint32_t edge = vocab;  // lane 0: the key before the chunk, lane 1: the key behind it
  if (lane == 0 && p0 > 0) edge = keys[p0 - 1];
  if (lane == 1 && p0 + kChunk < tokens) edge = keys[p0 + kChunk];
  const uint32_t before = p0 > 0 ? __shfl_sync(0xffffffffu, edge, 0) : 0xffffffffu;
  const uint32_t behind = __shfl_sync(0xffffffffu, edge, 1);
  const uint32_t below = __shfl_down_sync(0xffffffffu, key, 1);
  const uint32_t next = lane == 31 ? behind : below;
  const uint32_t first_key = __shfl_sync(0xffffffffu, key, 0);
  const int n = __popc(__ballot_sync(0xffffffffu, key < vocab));  // keys ascend: the real ones come first
  const uint32_t ends = __ballot_sync(0xffffffffu, key != next || lane == 31);
  const bool column = col < width;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; k++) acc[k] = 0.f;
  for (int b = 0; b < n; b += kBatch) {
    float v[kBatch][V];
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const uint32_t t = __shfl_sync(0xffffffffu, token, (b + i) & 31);
      if (b + i < n && column) {
        load_vec<V>(dy + (int64_t)t * width + col, v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) v[i][k] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const int at = b + i;
      if (at >= n) break;
#pragma unroll
      for (int k = 0; k < V; k++) acc[k] += v[i][k];
      if (!(ends >> at & 1)) continue;
      const uint32_t row = __shfl_sync(0xffffffffu, key, at);
      const bool came = row == first_key && row == before;
      const bool goes = at == 31 && row == behind;
      if (column) {
        if (came || goes) {
          store_vec<V>(partial + (chunk * 2 + (came ? 0 : 1)) * width + col, acc);
        } else {
#pragma unroll
          for (int k = 0; k < V; k++) acc[k] *= scale;
          store_vec<V>(dtable + (int64_t)row * width + col, acc);
        }
      }
#pragma unroll
      for (int k = 0; k < V; k++) acc[k] = 0.f;
    }
  }
}

// The table rows that begin in chunk blockIdx.x and go on: the sum of the chunks' shares.  Each of the 8
// warps adds a run of chunks, then the runs are added in order.
template <int V>
__global__ void __launch_bounds__(kThreads) embedding_join_kernel(const uint32_t* __restrict__ keys,
                                                                 const float* __restrict__ partial,
                                                                 float* __restrict__ dtable, int64_t tokens,
                                                                 uint32_t vocab, int64_t width, float scale) {
  __shared__ __align__(16) float join[kThreads / 32][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chunk = blockIdx.x, end = (chunk + 1) * kChunk;
  if (end >= tokens) return;
  const uint32_t row = keys[end - 1];
  if (row >= vocab || keys[end] != row || (chunk > 0 && keys[end - kChunk - 1] == row)) return;
  // chunks that go on with this row: those whose first key it is
  const int64_t chunks = (tokens + kChunk - 1) / kChunk;
  int64_t more = 0;
  for (;;) {
    const int64_t c = chunk + 1 + more + threadIdx.x;
    const int hit = __syncthreads_count(c < chunks && keys[c * kChunk] == row);
    more += hit;
    if (hit < kThreads) break;
  }
  const int64_t per = (more + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t lo = chunk + 1 + warp * per, hi = min(lo + per, chunk + 1 + more);
  for (int64_t j0 = (int64_t)blockIdx.y * 32 * V; j0 < width; j0 += (int64_t)gridDim.y * 32 * V) {
    const int64_t col = j0 + lane * V;
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; k++) acc[k] = 0.f;
    if (col < width) {
      if (warp == 0) load_vec<V>(partial + (chunk * 2 + 1) * width + col, acc);
#pragma unroll 4
      for (int64_t c = lo; c < hi; c++) {
        float v[V];
        load_vec<V>(partial + c * 2 * width + col, v);
#pragma unroll
        for (int k = 0; k < V; k++) acc[k] += v[k];
      }
    }
    store_vec<V>(&join[warp][lane * V], acc);
    __syncthreads();
    if (warp == 0 && col < width) {
#pragma unroll
      for (int w = 1; w < kThreads / 32; w++) {
        float v[V];
        load_vec<V>(&join[w][lane * V], v);
#pragma unroll
        for (int k = 0; k < V; k++) acc[k] += v[k];
      }
#pragma unroll
      for (int k = 0; k < V; k++) acc[k] *= scale;
      store_vec<V>(dtable + (int64_t)row * width + col, acc);
    }
    __syncthreads();
  }
}

// ---- launchers ---------------------------------------------------------------------------------------------
struct LookupArgs {
  const void* table;
  const int32_t* indices;
  void* out;
  int64_t tokens, vocab;
  int width;
  float scale;
  Decode q;
};

template <typename TT, typename TO, int V, int L>
void lookup_lanes(tfjs_cuda_ctx* ctx, const LookupArgs& a) {
  const int64_t blocks = ceil_div64(a.tokens, kThreads / L);
  embedding_kernel<TT, TO, V, L><<<(unsigned)(blocks < (1 << 30) ? blocks : (1 << 30)), kThreads, 0, ctx->stream>>>(
      (const TT*)a.table, a.indices, (TO*)a.out, a.tokens, a.vocab, a.width, a.scale, a.q);
}
template <typename TT, typename TO, int V>
void lookup_width(tfjs_cuda_ctx* ctx, const LookupArgs& a) {
  if (a.width <= 8 * V) lookup_lanes<TT, TO, V, 8>(ctx, a);
  else lookup_lanes<TT, TO, V, 32>(ctx, a);
}
// 16 bytes of the result a lane where the width allows it (bytes: 4, which are 16 of the result)
template <typename TT, typename TO>
int launch_lookup(tfjs_cuda_ctx* ctx, const LookupArgs& a) {
  constexpr int W = sizeof(TT) == 2 && sizeof(TO) == 2 ? 8 : 4;
  if (a.width % W == 0) lookup_width<TT, TO, W>(ctx, a);
  else if (sizeof(TT) != 1 && a.width % 2 == 0) lookup_width<TT, TO, sizeof(TT) != 1 ? 2 : 1>(ctx, a);
  else lookup_width<TT, TO, 1>(ctx, a);
  return post_launch(ctx, "embeddingLookup");
}

struct GradientArgs {
  const void* dy;
  const int32_t* indices;
  float* dtable;
  int64_t tokens, vocab, width;
  float scale;
};

// Sorted keys and tokens in `work` (4 arrays of `tokens`, the counts behind them); *keys and *order
// point at the sorted ones.  Writes dtable's zeros too.
int sort_tokens(tfjs_cuda_ctx* ctx, const GradientArgs& a, uint32_t* work, int64_t tiles, const uint32_t** keys,
                const uint32_t** order) {
  const Digits d = digits_of(a.vocab);
  const int smem = (int)sizeof(SortShared);
  uint32_t* k[2] = {work, work + 2 * a.tokens};
  uint32_t* t[2] = {work + a.tokens, work + 3 * a.tokens};
  if (tiles <= 8) {
    TFJS_CHECK_CUDA(ctx, cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    // 1024 keys a block and more: below that a block's passes cost more than they share out
    int blocks = 1;
    while (blocks < 8 && blocks * 1024 < a.tokens) blocks *= 2;
    const int64_t zero_blocks = ceil_div64(a.vocab * a.width, 4 * kSortThreads);
    int64_t grid = blocks + ceil_div64(zero_blocks, blocks) * blocks;
    const int64_t cap = (int64_t)ctx->sm_count / blocks * blocks;
    if (grid > cap) grid = cap;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TFJS_CHECK_CUDA(ctx, cudaLaunchKernelEx(&cfg, embedding_sort_kernel, a.indices, (int)a.tokens, (uint32_t)a.vocab,
                                            d.passes, d.bits, k[0], t[0], a.dtable, a.vocab * a.width));
    *keys = k[0];
    *order = t[0];
    return post_launch(ctx, "embeddingLookupBackprop (sort)");
  }
  TFJS_CHECK_CUDA(ctx, cudaFuncSetAttribute(embedding_count_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  TFJS_CHECK_CUDA(ctx, cudaFuncSetAttribute(embedding_scatter_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  TFJS_CHECK_CUDA(ctx, cudaMemsetAsync(a.dtable, 0, (size_t)(a.vocab * a.width) * 4, ctx->stream));
  uint32_t* counts = work + 4 * a.tokens;
  for (int pass = 0; pass < d.passes; pass++) {
    const int32_t* idx = pass == 0 ? a.indices : nullptr;
    const int from = (pass + 1) & 1, to = pass & 1, shift = pass * d.bits;
    int rc;
    embedding_count_kernel<<<(unsigned)tiles, kSortThreads, smem, ctx->stream>>>(idx, k[from], t[from], a.tokens,
                                                                                 (uint32_t)a.vocab, shift, d.bits, counts);
    if ((rc = post_launch(ctx, "embeddingLookupBackprop (count)"))) return rc;
    embedding_scan_kernel<<<1, kSortThreads, 0, ctx->stream>>>(counts, tiles << d.bits);
    if ((rc = post_launch(ctx, "embeddingLookupBackprop (scan)"))) return rc;
    embedding_scatter_kernel<<<(unsigned)tiles, kSortThreads, smem, ctx->stream>>>(
        idx, k[from], t[from], a.tokens, (uint32_t)a.vocab, shift, d.bits, counts, k[to], t[to]);
    if ((rc = post_launch(ctx, "embeddingLookupBackprop (scatter)"))) return rc;
    *keys = k[to];
    *order = t[to];
  }
  return TFJS_CUDA_OK;
}

template <typename TD, int V>
int sum_tokens(tfjs_cuda_ctx* ctx, const GradientArgs& a, const uint32_t* keys, const uint32_t* order, float* partial) {
  const int64_t chunks = ceil_div64(a.tokens, kChunk), tiles = ceil_div64(a.width, 32 * V), items = chunks * tiles;
  TFJS_REQUIRE(ctx, items < (1ll << 33), "embeddingLookupBackprop: too many tokens times columns");
  embedding_sum_kernel<TD, V><<<(unsigned)ceil_div64(items, kThreads / 32), kThreads, 0, ctx->stream>>>(
      (const TD*)a.dy, keys, order, a.dtable, partial, a.tokens, (uint32_t)a.vocab, a.width, a.scale, tiles, items);
  const int rc = post_launch(ctx, "embeddingLookupBackprop (sum)");
  if (rc || chunks < 2) return rc;
  embedding_join_kernel<V><<<dim3((unsigned)(chunks - 1), (unsigned)(tiles < 64 ? tiles : 64)), kThreads, 0, ctx->stream>>>(
      keys, partial, a.dtable, a.tokens, (uint32_t)a.vocab, a.width, a.scale);
  return post_launch(ctx, "embeddingLookupBackprop (join)");
}

template <typename TD>
int launch_gradient(tfjs_cuda_ctx* ctx, const GradientArgs& a) {
  const int64_t tiles = ceil_div64(a.tokens, kSortKeys), chunks = ceil_div64(a.tokens, kChunk);
  // sorted pairs (twice where the passes go through global memory), counts, partial sums
  const int64_t words = 4 * a.tokens + (tiles > 8 ? tiles * kMaxBins : 0), at = (words + 3) / 4 * 4;
  void* work;
  size_t cap;
  int rc = ctx_alloc(ctx, (size_t)(at + chunks * 2 * a.width) * 4, &work, &cap);
  if (rc) return rc;
  const uint32_t *keys, *order;
  rc = sort_tokens(ctx, a, (uint32_t*)work, tiles, &keys, &order);
  float* partial = (float*)work + at;
  if (!rc) rc = a.width % 4 == 0 ? sum_tokens<TD, 4>(ctx, a, keys, order, partial) : sum_tokens<TD, 1>(ctx, a, keys, order, partial);
  ctx_free(ctx, work, cap);
  return rc;
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
  const LookupArgs a = {table->ptr, (const int32_t*)indices->ptr, o->ptr, tokens, vocab, (int)width, scale,
                        {table->quant.scale, table->quant.min}};
  const bool half_out = o->dtype == TFJS_F16;
  if (table->quant.quantized) return half_out ? launch_lookup<uint8_t, __half>(ctx, a) : launch_lookup<uint8_t, float>(ctx, a);
  if (table->dtype == TFJS_F16) return half_out ? launch_lookup<__half, __half>(ctx, a) : launch_lookup<__half, float>(ctx, a);
  return half_out ? launch_lookup<float, __half>(ctx, a) : launch_lookup<float, float>(ctx, a);
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
  const GradientArgs a = {dy->ptr, (const int32_t*)indices->ptr, (float*)o->ptr, tokens, vocab, width, scale};
  return dy->dtype == TFJS_F16 ? launch_gradient<__half>(ctx, a) : launch_gradient<float>(ctx, a);
}

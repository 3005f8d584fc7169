// Embedding lookup with scaling, and the gradient of its table.
//
//   out[t] = scale * table[i_t],      zeros where i_t lies outside [0, vocab) (padding)
//   dtable[v] = scale * sum of dy[t] over the tokens t with i_t == v
//
// The lookup is bound by the bytes of the result.  The gradient writes the whole table and reads dy; adding
// rows with atomics would make the result's last bits depend on their order, so the tokens are sorted by table
// row first and each table row has its rows of dy added in a fixed order: three launches,
//   sort   one cluster sorts up to 65536 (row, token) pairs in shared memory while all other blocks write the
//          table's zeros (32000 x 768, 16384 tokens: 18 us; the zeros alone need 16, the sort alone 11)
//   sum    a warp adds 16 or 32 sorted tokens over 128 columns and writes the rows that end within them
//          (12 us: 50 MB of dy, latency as much as bandwidth)
//   join   rows that go on over several warps' tokens have their shares added, in order (6 us)
// Above 65536 tokens the table's zeros, then a count, a scan and a placing for each digit: 100000 x 256 of 50000 rows
// 47 us for the sort, 22 for the sums, 8 for the join.
// Sums are float32; the scale multiplies each finished sum.
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;

// ---- lookup ----------------------------------------------------------------------------------------
// V values of a table row as they are stored.
template <typename T, int V>
struct alignas(sizeof(T) * V) Raw {
  T v[V];
};
// A quantised table's value is the float32 that decodeWeights gives (io_utils.ts:139): a float64
// product and sum, rounded once.
struct Decode {
  double scale, min;
};
__device__ __forceinline__ float widen(float v, Decode) { return v; }
__device__ __forceinline__ float widen(__half v, Decode) { return __half2float(v); }
__device__ __forceinline__ float widen(uint8_t v, Decode q) { return (float)__dadd_rn(__dmul_rn((double)v, q.scale), q.min); }

// L lanes a token; blockIdx.y takes U * L * V columns.  Bound by the bytes written; the U loads of a lane
// are issued before its first store, and a block ends with its tokens (blocks that go on to further ones
// measured 8 % slower: 32768 x 1024 from bytes 28.9 us, this form 26.7; a decoded-value table in shared
// memory instead of the float64 arithmetic changes nothing).  `stream`: the result exceeds L2 by far, so
// its lines may leave first (24.7 us).
template <typename TT, typename TO, int V, int L, int U>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const TT* __restrict__ table,
                                                            const int32_t* __restrict__ indices, TO* __restrict__ out,
                                                            int64_t tokens, int64_t vocab, int width, float scale,
                                                            Decode q, bool stream) {
  const int lane = threadIdx.x & (L - 1), vecs = width / V;
  const int64_t t = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (t >= tokens) return;
  const int32_t v = indices[t];
  const bool there = v >= 0 && v < vocab;
  const Raw<TT, V>* row = reinterpret_cast<const Raw<TT, V>*>(table + (int64_t)(there ? v : 0) * width);
  for (int j = blockIdx.y * U * L + lane; j < vecs; j += gridDim.y * U * L) {
    Raw<TT, V> r[U];
    if (there) {
#pragma unroll
      for (int i = 0; i < U; i++)
        if (j + i * L < vecs) r[i] = row[j + i * L];
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (j + i * L >= vecs) break;
      float f[V];
#pragma unroll
      for (int k = 0; k < V; k++) f[k] = there ? widen(r[i].v[k], q) * scale : 0.f;
      TO* o = out + t * width + (int64_t)(j + i * L) * V;
      if (stream) store_vec_stream<V>(o, f);
      else store_vec<V>(o, f);
    }
  }
}

// ---- gradient: tokens sorted by table row --------------------------------------------------------------
// Stable least-significant-digit radix sort of (table row, token) pairs; a token outside the table
// gets the key `vocab`, behind all others.  Within a block each warp owns a run of keys: it counts
// their digits into its own counters (the lanes of equal digits find each other by votes, one of them
// adds), the counters are summed over the warps and blocks, and the same walk then gives each key its
// place.  No atomics: equal inputs give the same order, ascending tokens within each table row.
constexpr int kSortThreads = 1024, kSortWarps = 32;
constexpr int kSortKeys = 8192;  // of one block, at most
constexpr int kMaxBins = 512;
constexpr int kZeroQuads = 8 * kSortThreads;  // 128 KB of zeros a block

struct Digits {
  int passes, bits;
};
Digits digits_of(int64_t vocab) {
  int total = 1;
  while (total < 32 && (vocab >> total)) total++;
  const int passes = (total + 8) / 9;
  return {passes, (total + passes - 1) / passes};
}

// Each thread's keys (at most 8): their digits, and their places among the keys of that digit that the
// warp owns; counts[warp][digit] is the number of them.  A place beyond the block's n keys has digit ~0.
constexpr int kKeysPerThread = kSortKeys / kSortThreads;
__device__ __forceinline__ void rank_keys(const uint2* pairs, int n, int per_warp, int shift, int bins, uint16_t* counts,
                                          uint32_t (&digit)[kKeysPerThread], uint32_t (&place)[kKeysPerThread]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* mine = counts + warp * bins;
#pragma unroll
  for (int i = 0; i < kKeysPerThread; i++) {
    digit[i] = ~0u;
    place[i] = 0;
    const int at = warp * per_warp + i * 32 + lane;
    const bool there = i * 32 < per_warp && at < n;
    if (!__any_sync(0xffffffffu, there)) continue;
    if (there) digit[i] = (pairs[at].x >> shift) & (uint32_t)(bins - 1);
    // the lanes of the same digit, by a vote on each of its bits
    uint32_t peers = __ballot_sync(0xffffffffu, there);
    for (int bit = 0; (bins >> bit) > 1; bit++) {
      const bool set = digit[i] >> bit & 1;
      const uint32_t votes = __ballot_sync(0xffffffffu, set);
      peers &= set ? votes : ~votes;
    }
    const int before = __popc(peers & ((1u << lane) - 1));
    uint32_t base = 0;
    if (there) base = mine[digit[i]];
    __syncwarp();
    if (there && before == 0) mine[digit[i]] = (uint16_t)(base + __popc(peers));
    __syncwarp();
    place[i] = base + before;
  }
}

// counts[warp][digit] -> exclusive prefix over the warps; returns the block's total of digit threadIdx.x.
__device__ __forceinline__ uint32_t prefix_over_warps(uint16_t* counts, int bins) {
  uint32_t sum = 0;
  if ((int)threadIdx.x < bins) {
    uint32_t c[kSortWarps];
#pragma unroll
    for (int w = 0; w < kSortWarps; w++) c[w] = counts[w * bins + threadIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; w++) {
      counts[w * bins + threadIdx.x] = (uint16_t)sum;
      sum += c[w];
    }
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

// A sorting block's dynamic shared memory, of a size that goes with its share of the keys: `buffers` arrays
// of (key, token) pairs, the digits' totals and first places, and the warps' counters.
struct SortView {
  uint2* pairs[2];
  uint32_t *totals, *base, *warps;
  uint16_t* counts;
  __device__ SortView(uint8_t* raw, int share, int buffers, int bins) {
    pairs[0] = reinterpret_cast<uint2*>(raw);
    pairs[1] = pairs[0] + (buffers - 1) * share;
    totals = reinterpret_cast<uint32_t*>(pairs[1] + share);
    base = totals + bins;
    warps = base + bins;
    counts = reinterpret_cast<uint16_t*>(warps + 32);
  }
  static size_t bytes(int share, int buffers, int bins) {
    return (size_t)share * buffers * 8 + (size_t)bins * 8 + 32 * 4 + (size_t)kSortWarps * bins * 2;
  }
};

// Up to 8 * 8192 tokens: the first cluster sorts them in its blocks' shared memory, the other blocks
// write the table gradient's zeros meanwhile.  `share`: keys a block, a multiple of 1024.
__global__ void __launch_bounds__(kSortThreads, 1) embedding_sort_kernel(const int32_t* __restrict__ indices, int tokens,
                                                                        int share, uint32_t vocab, int passes, int bits,
                                                                        uint2* __restrict__ sorted,
                                                                        float* __restrict__ dtable, int64_t values) {
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks();
  pdl_launch_dependents();  // the sums wait for this kernel's end before they read
  if ((int)blockIdx.x >= blocks) {
    // a piece of kZeroQuads float4 each, and out: blocks that stayed for a fixed share of the table made the
    // clusters that do not fit at first double the kernel's time (32000 x 768 with 16384 tokens: 26 us)
    const int64_t first = (int64_t)(blockIdx.x - blocks) * kZeroQuads + threadIdx.x, quads = values / 4;
    float4* table = reinterpret_cast<float4*>(dtable);
#pragma unroll
    for (int i = 0; i < kZeroQuads / kSortThreads; i++)
      if (first + i * kSortThreads < quads) table[first + i * kSortThreads] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (first < (values & 3)) dtable[(values & ~3ll) + first] = 0.f;
    return;
  }
  extern __shared__ __align__(16) uint8_t raw[];
  const int bins = 1 << bits;
  SortView s(raw, share, 2, bins);
  const int rank = (int)cluster.block_rank();
  const int n = max(0, min(share, tokens - rank * share));
  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    const int32_t v = indices[rank * share + i];
    s.pairs[0][i] = make_uint2((uint32_t)v < vocab ? (uint32_t)v : vocab, (uint32_t)(rank * share + i));
  }
  const int per_warp = share / kSortWarps, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int pass = 0; pass < passes; pass++) {
    const int from = pass & 1, shift = pass * bits;
    for (int i = threadIdx.x; i < kSortWarps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(s.counts)[i] = 0;
    __syncthreads();
    uint32_t digit[kKeysPerThread], place[kKeysPerThread];
    rank_keys(s.pairs[from], n, per_warp, shift, bins, s.counts, digit, place);
    __syncthreads();
    const uint32_t total = prefix_over_warps(s.counts, bins);
    if ((int)threadIdx.x < bins) s.totals[threadIdx.x] = total;
    cluster.sync();
    uint32_t all = 0, before = 0;
    if ((int)threadIdx.x < bins) {
#pragma unroll
      for (int r = 0; r < 8; r++) {
        const uint32_t c = r < blocks ? cluster.map_shared_rank(s.totals, r)[threadIdx.x] : 0;
        all += c;
        if (r < rank) before += c;
      }
    }
    const bool last = pass + 1 == passes;
    const uint32_t smaller = block_exclusive(all, s.warps);
    if ((int)threadIdx.x < bins) s.base[threadIdx.x] = smaller + before;
    __syncthreads();
    // The last pass writes to global memory only: its barrier, which keeps the blocks until the others have
    // read their totals, is entered here, so that it does not wait for those writes (they queue behind the
    // other blocks' zeros).  The totals that this block read have been used by now.
    if (last) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kKeysPerThread; i++) {
      if (digit[i] == ~0u) continue;
      const uint2 pair = s.pairs[from][warp * per_warp + i * 32 + lane];
      const int g = (int)(s.base[digit[i]] + s.counts[warp * bins + digit[i]] + place[i]);
      if (last) {
        sorted[g] = pair;
      } else {
        const int to = g / share;
        cluster.map_shared_rank(s.pairs[from ^ 1], to)[g - to * share] = pair;
      }
    }
    if (!last) cluster.sync();  // the pass's writes have arrived; nobody reads this block's totals any more
  }
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// More tokens: three launches a pass, over tiles of `share` keys.
__device__ __forceinline__ int load_tile(const int32_t* indices, const uint2* in, int64_t tokens, int share, uint32_t vocab,
                                         uint2* pairs) {
  const int64_t first = (int64_t)blockIdx.x * share;
  const int n = (int)(tokens - first < share ? tokens - first : share);
  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    if (indices) {
      const int32_t v = indices[first + i];
      pairs[i] = make_uint2((uint32_t)v < vocab ? (uint32_t)v : vocab, (uint32_t)(first + i));
    } else {
      pairs[i] = in[first + i];
    }
  }
  return n;
}
// PLACE false: counts[digit][tile]; true: the keys to their places, from the counts' exclusive sum.
template <bool PLACE>
__global__ void __launch_bounds__(kSortThreads, 1) embedding_tile_kernel(const int32_t* __restrict__ indices,
                                                                        const uint2* __restrict__ in, int64_t tokens,
                                                                        int share, uint32_t vocab, int shift, int bits,
                                                                        uint32_t* __restrict__ counts,
                                                                        uint2* __restrict__ out) {
  extern __shared__ __align__(16) uint8_t raw[];
  const int bins = 1 << bits;
  SortView s(raw, share, 1, bins);
  for (int i = threadIdx.x; i < kSortWarps * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(s.counts)[i] = 0;
  const int n = load_tile(indices, in, tokens, share, vocab, s.pairs[0]);
  __syncthreads();
  uint32_t digit[kKeysPerThread], place[kKeysPerThread];
  const int per_warp = share / kSortWarps, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  rank_keys(s.pairs[0], n, per_warp, shift, bins, s.counts, digit, place);
  __syncthreads();
  const uint32_t total = prefix_over_warps(s.counts, bins);
  uint32_t* count = counts + (int64_t)threadIdx.x * gridDim.x + blockIdx.x;
  if (!PLACE) {
    if ((int)threadIdx.x < bins) *count = total;
    return;
  }
  if ((int)threadIdx.x < bins) s.base[threadIdx.x] = *count;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kKeysPerThread; i++)
    if (digit[i] != ~0u)
      out[s.base[digit[i]] + s.counts[warp * bins + digit[i]] + place[i]] = s.pairs[0][warp * per_warp + i * 32 + lane];
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

// ---- gradient: sums over the sorted tokens -----------------------------------------------------------------
// A warp takes CH sorted tokens (16 or 32) and 32 V columns.  A table row whose tokens all lie in this chunk is
// finished here.  One that began in an earlier chunk leaves this chunk's share in partial[chunk][0], one
// that begins here and goes on in partial[chunk][1].
constexpr int kBatch = 4;  // rows of dy in flight a warp
constexpr int kSumThreads = 128;
// In this kernel and the next, what the kernel before wrote is read through pointers without __restrict__: a load
// that the compiler may take for one of constant data could be moved ahead of pdl_wait().

template <typename TD, int V, int CH>
__global__ void __launch_bounds__(kSumThreads) embedding_sum_kernel(const TD* __restrict__ dy,
                                                                const uint2* sorted,
                                                                float* __restrict__ dtable, float* __restrict__ partial,
                                                                int64_t tokens, uint32_t vocab, int64_t width, float scale,
                                                                int64_t tiles, int64_t items) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (kSumThreads / 32) + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();  // the join waits for this kernel's end
  if (item >= items) return;
  const int64_t chunk = item / tiles, col = ((item - chunk * tiles) * 32 + lane) * V;
  const int64_t p0 = chunk * CH;
  const bool held = lane < CH && p0 + lane < tokens;
  const uint2 pair = held ? sorted[p0 + lane] : make_uint2(vocab, 0);
  const uint32_t key = pair.x, token = pair.y;
  uint32_t edge = vocab;  // lane 0: the key before the chunk, lane 1: the key behind it
  if (lane == 0 && p0 > 0) edge = sorted[p0 - 1].x;
  if (lane == 1 && p0 + CH < tokens) edge = sorted[p0 + CH].x;
  const uint32_t before = p0 > 0 ? __shfl_sync(0xffffffffu, edge, 0) : 0xffffffffu;
  const uint32_t behind = __shfl_sync(0xffffffffu, edge, 1);
  const uint32_t next = __shfl_down_sync(0xffffffffu, key, 1);
  const uint32_t first_key = __shfl_sync(0xffffffffu, key, 0);
  const int n = __popc(__ballot_sync(0xffffffffu, key < vocab));  // keys ascend: the real ones come first
  const uint32_t ends = __ballot_sync(0xffffffffu, key != next || lane == CH - 1);
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
      const bool goes = at == CH - 1 && row == behind;
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

// The table rows that begin in one chunk and go on in others: the sum of the chunks' shares.  A warp takes a
// chunk and 32 V columns, and up to 31 further chunks by itself; the longer runs (a token of hundreds of
// places) the block's 8 warps then share out one after the other, each adding a run of chunks, in order.
constexpr int kJoinWarps = kThreads / 32;
template <int V>
__device__ __forceinline__ void add_shares(const float* partial, int64_t lo, int64_t hi, int64_t width, int64_t col,
                                           float (&acc)[V]) {
#pragma unroll 8
  for (int64_t c = lo; c < hi; c++) {
    float v[V];
    load_vec<V>(partial + c * 2 * width + col, v);
#pragma unroll
    for (int k = 0; k < V; k++) acc[k] += v[k];
  }
}
template <int V, int CH>
__global__ void __launch_bounds__(kThreads) embedding_join_kernel(const uint2* sorted,
                                                                 const float* partial,
                                                                 float* __restrict__ dtable, int64_t tokens,
                                                                 uint32_t vocab, int64_t width, float scale,
                                                                 int64_t chunks) {
  __shared__ __align__(16) float join[kJoinWarps][32 * V];
  __shared__ uint32_t long_row[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = (int64_t)blockIdx.x * kJoinWarps, chunk = first + warp, end = (chunk + 1) * CH;
  pdl_wait();
  uint32_t row = vocab, behind = vocab, before = vocab, head = vocab;
  if (end < tokens) {
    row = sorted[end - 1].x;
    behind = sorted[end].x;
    if (chunk > 0) before = sorted[end - CH - 1].x;
    if (chunk + 1 + lane < chunks) head = sorted[(chunk + 1 + lane) * CH].x;
  }
  const bool mine = row < vocab && behind == row && before != row;
  const int more = mine ? __popc(__ballot_sync(0xffffffffu, head == row)) : 0;  // heads ascend: a run of ones
  if (lane == 0) long_row[warp] = more == 32 ? row : vocab;
  for (int64_t j0 = (int64_t)blockIdx.y * 32 * V; j0 < width; j0 += (int64_t)gridDim.y * 32 * V) {
    const int64_t col = j0 + lane * V;
    if (more > 0 && more < 32 && col < width) {
      float acc[V];
      load_vec<V>(partial + (chunk * 2 + 1) * width + col, acc);
      add_shares<V>(partial, chunk + 1, chunk + 1 + more, width, col, acc);
#pragma unroll
      for (int k = 0; k < V; k++) acc[k] *= scale;
      store_vec<V>(dtable + (int64_t)row * width + col, acc);
    }
  }
  __syncthreads();
  for (int w = 0; w < kJoinWarps; w++) {
    const uint32_t long_key = long_row[w];
    if (long_key >= vocab) continue;  // the same for the whole block
    int64_t run = 0;
    for (;;) {
      const int64_t c = first + w + 1 + run + threadIdx.x;
      const int hit = __syncthreads_count(c < chunks && sorted[c * CH].x == long_key);
      run += hit;
      if (hit < kThreads) break;
    }
    const int64_t per = (run + kJoinWarps - 1) / kJoinWarps;
    const int64_t lo = first + w + 1 + warp * per, hi = min(lo + per, first + w + 1 + run);
    for (int64_t j0 = (int64_t)blockIdx.y * 32 * V; j0 < width; j0 += (int64_t)gridDim.y * 32 * V) {
      const int64_t col = j0 + lane * V;
      float acc[V];
#pragma unroll
      for (int k = 0; k < V; k++) acc[k] = 0.f;
      if (col < width) {
        if (warp == 0) load_vec<V>(partial + ((first + w) * 2 + 1) * width + col, acc);
        add_shares<V>(partial, lo, hi, width, col, acc);
      }
      store_vec<V>(&join[warp][lane * V], acc);
      __syncthreads();
      if (warp == 0 && col < width) {
#pragma unroll
        for (int o = 1; o < kJoinWarps; o++) {
          float v[V];
          load_vec<V>(&join[o][lane * V], v);
#pragma unroll
          for (int k = 0; k < V; k++) acc[k] += v[k];
        }
#pragma unroll
        for (int k = 0; k < V; k++) acc[k] *= scale;
        store_vec<V>(dtable + (int64_t)long_key * width + col, acc);
      }
      __syncthreads();
    }
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

template <typename TT, typename TO, int V, int L, int U>
void lookup_lanes(tfjs_cuda_ctx* ctx, const LookupArgs& a) {
  const int64_t parts = ceil_div64(a.width / V, U * L);
  const bool stream = a.tokens * a.width * (int64_t)sizeof(TO) > kStreamBytes;
  embedding_kernel<TT, TO, V, L, U><<<dim3((unsigned)ceil_div64(a.tokens, kThreads / L), (unsigned)(parts < 64 ? parts : 64)),
                                      kThreads, 0, ctx->stream>>>((const TT*)a.table, a.indices, (TO*)a.out, a.tokens, a.vocab,
                                                                  a.width, a.scale, a.q, stream);
}
template <typename TT, typename TO, int V>
void lookup_width(tfjs_cuda_ctx* ctx, const LookupArgs& a) {
  constexpr int U = sizeof(TT) == 1 ? 8 : 4;
  // narrow rows share a warp: 500000 tokens x 16 columns 22 us, 58 with a warp each
  if (a.width <= 8 * V) lookup_lanes<TT, TO, V, 8, 1>(ctx, a);
  else if (a.width <= 64 * V) lookup_lanes<TT, TO, V, 32, 2>(ctx, a);
  else lookup_lanes<TT, TO, V, 32, U>(ctx, a);
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

// Sorts the (table row, token) pairs into *sorted, one of `buffers`, and writes dtable's zeros.  `counts`:
// 512 for each tile of `share` keys, where there are more than 8 blocks can hold.
int sort_tokens(tfjs_cuda_ctx* ctx, const GradientArgs& a, uint2* const* buffers, uint32_t* counts, int share, int64_t tiles,
                const uint2** sorted) {
  const Digits d = digits_of(a.vocab);
  const int bins = 1 << d.bits;
  if (!counts) {
    const int blocks = (int)tiles;
    const int smem = (int)SortView::bytes(share, 2, bins);
    TFJS_CHECK_CUDA(ctx, allow_smem(embedding_sort_kernel, smem));
    const int64_t zero_blocks = ceil_div64(a.vocab * a.width, 4 * kZeroQuads);
    const int64_t grid = blocks + ceil_div64(zero_blocks, blocks) * blocks;
    TFJS_REQUIRE(ctx, grid < (1ll << 31), "embeddingLookupBackprop: the table is too large");
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
    TFJS_CHECK_CUDA(ctx, cudaLaunchKernelEx(&cfg, embedding_sort_kernel, a.indices, (int)a.tokens, share, (uint32_t)a.vocab,
                                            d.passes, d.bits, buffers[0], a.dtable, a.vocab * a.width));
    *sorted = buffers[0];
    return post_launch(ctx, "embeddingLookupBackprop (sort)");
  }
  const int smem = (int)SortView::bytes(share, 1, bins);
  auto count = embedding_tile_kernel<false>, place = embedding_tile_kernel<true>;
  TFJS_CHECK_CUDA(ctx, allow_smem(count, smem));
  TFJS_CHECK_CUDA(ctx, allow_smem(place, smem));
  TFJS_CHECK_CUDA(ctx, cudaMemsetAsync(a.dtable, 0, (size_t)(a.vocab * a.width) * 4, ctx->stream));
  for (int pass = 0; pass < d.passes; pass++) {
    const int32_t* indices = pass == 0 ? a.indices : nullptr;
    const uint2* in = buffers[(pass + 1) & 1];
    uint2* out = buffers[pass & 1];
    int rc;
    count<<<(unsigned)tiles, kSortThreads, smem, ctx->stream>>>(indices, in, a.tokens, share, (uint32_t)a.vocab,
                                                                pass * d.bits, d.bits, counts, nullptr);
    if ((rc = post_launch(ctx, "embeddingLookupBackprop (count)"))) return rc;
    embedding_scan_kernel<<<1, kSortThreads, 0, ctx->stream>>>(counts, tiles << d.bits);
    if ((rc = post_launch(ctx, "embeddingLookupBackprop (scan)"))) return rc;
    place<<<(unsigned)tiles, kSortThreads, smem, ctx->stream>>>(indices, in, a.tokens, share, (uint32_t)a.vocab,
                                                                pass * d.bits, d.bits, counts, out);
    if ((rc = post_launch(ctx, "embeddingLookupBackprop (place)"))) return rc;
    *sorted = out;
  }
  return TFJS_CUDA_OK;
}

template <typename TD, int V, int CH>
int sum_tokens(tfjs_cuda_ctx* ctx, const GradientArgs& a, const uint2* sorted, float* partial) {
  const int64_t chunks = ceil_div64(a.tokens, CH), tiles = ceil_div64(a.width, 32 * V), items = chunks * tiles;
  TFJS_REQUIRE(ctx, items < (1ll << 32), "embeddingLookupBackprop: too many tokens times columns");
  launch_dependent(ctx, embedding_sum_kernel<TD, V, CH>, dim3((unsigned)ceil_div64(items, kSumThreads / 32)), dim3(kSumThreads),
                   (const TD*)a.dy, sorted, a.dtable, partial, a.tokens, (uint32_t)a.vocab, a.width, a.scale, tiles, items);
  const int rc = post_launch(ctx, "embeddingLookupBackprop (sum)");
  if (rc || chunks < 2) return rc;
  launch_dependent(ctx, embedding_join_kernel<V, CH>, dim3((unsigned)ceil_div64(chunks - 1, kJoinWarps), (unsigned)(tiles < 64 ? tiles : 64)),
                   dim3(kThreads), sorted, (const float*)partial, a.dtable, a.tokens, (uint32_t)a.vocab, a.width, a.scale, chunks);
  return post_launch(ctx, "embeddingLookupBackprop (join)");
}

template <typename TD>
int launch_gradient(tfjs_cuda_ctx* ctx, const GradientArgs& a) {
  // One cluster, up to 1024 keys a block (4000 keys: 10 us with four blocks, 14 with one; 8000: 10 with eight,
  // 20), as long as eight blocks hold them (65536 keys: 26 us beside the zeros, where tiles take 50 after them).
  // Else tiles of 2048 keys, of 8192 where there are so many that their counts would grow past the keys.
  const bool cluster = a.tokens <= 8 * kSortKeys;
  int64_t tiles = 1;
  int share = a.tokens > (1 << 20) ? kSortKeys : 2048;
  if (cluster) {
    while (tiles < 8 && tiles * 1024 < a.tokens) tiles *= 2;
    share = (int)ceil_div64(ceil_div64(a.tokens, tiles), kSortThreads) * kSortThreads;
  } else {
    tiles = ceil_div64(a.tokens, share);
  }
  // 32 tokens a warp leave fewer shares to join (65536 tokens x 768: the join 14 us, 25 with 16 tokens a warp),
  // 16 make more warps (1021 tokens x 130: the sums 5 us, 10 with 32); at 16384 tokens both take the same
  const bool long_chunks = a.tokens >= 32768;
  const int64_t chunks = ceil_div64(a.tokens, long_chunks ? 32 : 16);
  const size_t pair_bytes = (size_t)(a.tokens + 1) / 2 * 16, partial_bytes = (size_t)(chunks * 2 * a.width) * 4;
  const size_t count_bytes = cluster ? 0 : (size_t)tiles * kMaxBins * 4;
  uint8_t* work;
  size_t cap;
  int rc = ctx_alloc(ctx, (cluster ? 1 : 2) * pair_bytes + count_bytes + partial_bytes + 16, (void**)&work, &cap);
  if (rc) return rc;
  uint2* buffers[2] = {(uint2*)work, (uint2*)(work + pair_bytes)};
  uint8_t* behind = work + (cluster ? 1 : 2) * pair_bytes;
  const uint2* sorted;
  rc = sort_tokens(ctx, a, buffers, cluster ? nullptr : (uint32_t*)behind, share, tiles, &sorted);
  float* partial = (float*)(behind + count_bytes);
  if (!rc) {
    if (a.width % 4 == 0) rc = long_chunks ? sum_tokens<TD, 4, 32>(ctx, a, sorted, partial) : sum_tokens<TD, 4, 16>(ctx, a, sorted, partial);
    else rc = long_chunks ? sum_tokens<TD, 1, 32>(ctx, a, sorted, partial) : sum_tokens<TD, 1, 16>(ctx, a, sorted, partial);
  }
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

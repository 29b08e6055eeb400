// Token-embedding lookup with a scale, and its gradient by sorted tokens.
//
//   fwd : out[t, :] = scale * W[id[t], :]
//   bwd : dW[v, :] (+)= scale * sum_{t : id[t] = v, v != padding} dy[t, :]
//
// Tables and activations are fp32, bf16 or fp16, sums and dW fp32.  An id outside the table
// sets kStatusBadShape, gives a row of zeros and adds nothing to dW.
//
// Backward.  Adding rows with atomics makes the result depend on the order in which they
// arrive; here the tokens are sorted by id (stable, so each row's terms lie in token order), a row's
// terms are added in an order that their positions fix (parts of 8, then across the warps of a chunk,
// then across chunks) and every dW element is written once: equal inputs give equal bits.
//
//  1. embed_sort_kernel: 2^c bins, each of the ids with the same low c bits (frequent tokens, which
//     vocabularies number low, spread over the bins).  A cluster of four CTAs per bin (two or one where
//     the table has more than 32768 or 65536 rows) reads all n ids, a part each, counts those of earlier bins (the bin's offset in the sorted order, with no
//     exchange between clusters) and places its own by a counting sort: the CTAs' counts meet over
//     distributed shared memory, and within a CTA up to 16 warps take consecutive parts of its tokens,
//     so that the order within an id is the token order.
//  2. embed_reduce_kernel: one CTA per (chunk of sorted tokens, slab of columns).  Each warp adds
//     the rows of its part of the chunk run by run in registers and writes the runs that lie
//     inside; runs that cross warps meet in shared memory, and runs that cross chunks leave one
//     piece per chunk in the workspace.  Without accumulation, further CTAs write zeros to the rows
//     that no token names.
//  3. embed_join_kernel: adds the pieces of each run that crosses chunks, in chunk order.
//
// What bounds them, and what they take at 32768 tokens x 1024 columns (B200, 30522 rows, a quarter of
// the tokens padding): the lookup of fp32 rows into bf16 20 us, L2 and DRAM (201 MB with the repeated
// rows); the sort 10 us, latency (two sweeps of dependent loads, shared-memory counters, a scan); the
// join 5.6 us, latency.  The reduce takes 28 us when adding (101 MB of dy, 29 MB of named rows read and
// written: 5.6 TB/s; DRAM moves 133 MB, 4.7 TB/s) and 41 us when writing every row (101 MB of dy, 125 MB of
// dW: 5.5 TB/s): what bounds it is the bytes in flight.  All rows of a warp (8 tokens x 1 KB) are loaded
// before the first is added: 20 warps per SM keep 160 KB in flight; 16 tokens per warp left 12 warps and
// took 38 us, 8 of 32 tokens at a time 46 us.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "common.cuh"
#include "host.h"
#include "vec.cuh"

namespace revpp {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kFwdUnroll = 4;      // vectors per lane and row slab
constexpr int kFwdBlocksPerSm = 4;
constexpr int kSortWarps = 32;
constexpr int kSortPer = 1024;     // tokens a warp lists at most before they are placed
constexpr int kSortCtas = 128;     // at most one CTA per SM, unless the table is very long
constexpr int kSortCluster = 4;    // CTAs that share a bin of ids, each with a part of the tokens; fewer for long tables
constexpr int kSortLogRange = 10;  // ids per bin: 1024 at most, one per thread
constexpr int kRankers = 16;       // warps that place tokens
constexpr int kWarps = 4;          // of a reduce CTA
constexpr int kWarpTokens = 8;    // sorted tokens a reduce warp adds: all their rows are in flight at once
constexpr int kChunk = kWarps * kWarpTokens;
constexpr int kLaneColumns = 8;    // columns of a reduce lane
constexpr int kSlab = 32 * kLaneColumns;
constexpr int kZeroRows = 8;       // dW rows per zero-writing warp

// ------------------------------------------------------------------ forward
// L lanes (a power of two) per (row, slab of L * V * kFwdUnroll columns).  A group walks over its
// pieces with the next one's id already on its way, so that a row costs one trip to memory, not two.
template <typename TI, typename TW, typename TO, int V>
__global__ void __launch_bounds__(kThreads, kFwdBlocksPerSm)
    embed_fwd_kernel(const TI* __restrict__ ids, const TW* __restrict__ w, long long ldw, TO* __restrict__ out,
                     long long ldo, long long n, long long vocab, int H, int log_l, int slabs, float scale,
                     int* __restrict__ status) {
  pdl_wait();
  pdl_trigger();
  constexpr int P = V * sizeof(TW) <= 16 ? V : 16 / sizeof(TW), Q = V * sizeof(TO) <= 16 ? V : 16 / sizeof(TO);
  const long long pieces = n * slabs, groups = (static_cast<long long>(gridDim.x) * kThreads) >> log_l;
  long long piece = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> log_l;
  const int sub = threadIdx.x & ((1 << log_l) - 1);
  long long row = piece / slabs;
  long long next_id = piece < pieces ? static_cast<long long>(ids[row]) : 0;
  while (piece < pieces) {
    const int slab = static_cast<int>(piece - row * slabs);
    const long long id = next_id;
    const bool ok = id >= 0 && id < vocab;
    if (!ok && sub == 0 && slab == 0) atomicOr(status, kStatusBadShape);
    const TW* src = w + (ok ? id : 0) * ldw;
    TO* dst = out + row * ldo;
    piece += groups;
    row = piece / slabs;
    if (piece < pieces) next_id = static_cast<long long>(ids[row]);
    const int c0 = ((slab * kFwdUnroll << log_l) + sub) * V;
    Pack<TW, P> x[kFwdUnroll][V / P];
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      const int c = c0 + ((u * V) << log_l);
#pragma unroll
      for (int i = 0; i < V / P; ++i)
        if (c < H && ok) x[u][i] = Pack<TW, P>::load_ro(src + c + i * P);
    }
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      const int c = c0 + ((u * V) << log_l);
      if (c >= H) continue;
      float f[V];
#pragma unroll
      for (int i = 0; i < V / P; ++i) {
        float g[P];
        x[u][i].get(g);
#pragma unroll
        for (int j = 0; j < P; ++j) f[i * P + j] = ok ? g[j] * scale : 0.f;
      }
#pragma unroll
      for (int i = 0; i < V / Q; ++i) {
        float g[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) g[j] = f[i * Q + j];
        Pack<TO, Q> y;
        y.set(g);
        y.store(dst + c + i * Q);
      }
    }
  }
}

// ------------------------------------------------------------------ backward: sort
// An id's place in the sorted order follows from its slot: its bin, then the rest.
struct EmbedWs {
  int* start;     // [slots + 1] first sorted position of each slot
  int* order;     // [n] token of each sorted position
  int* key;       // [n] slot of each sorted position
  float* part;    // [2][chunks][H] pieces of runs that cross chunks: from before, and into the next
  int log_c, log_r;
  __device__ __forceinline__ int slots() const { return 1 << (log_c + log_r); }
  __device__ __forceinline__ int slot_of(int id) const { return ((id & ((1 << log_c) - 1)) << log_r) | (id >> log_c); }
  __device__ __forceinline__ int id_of(int slot) const { return ((slot & ((1 << log_r) - 1)) << log_c) | (slot >> log_r); }
};

// The low 32 bits of an id inside the table, or ~0 for one outside.
__device__ __forceinline__ unsigned checked(int64_t id, unsigned vocab) {
  const unsigned lo = static_cast<unsigned>(id), hi = static_cast<unsigned>(static_cast<uint64_t>(id) >> 32);
  return hi == 0 && lo < vocab ? lo : 0xffffffffu;
}
__device__ __forceinline__ unsigned checked(int32_t id, unsigned vocab) {
  const unsigned lo = static_cast<unsigned>(id);
  return lo < vocab ? lo : 0xffffffffu;
}

// The tokens [beg, end) of one warp whose ids belong to `bin` go to `list` in token order, as
// (token - seg) << kSortLogRange | local id, and are counted per local id; returns how many.  `less`
// counts the ids of earlier bins.  A lane reads two neighbouring ids per access (`wide`: the address allows it).
template <typename TI>
__device__ __forceinline__ int sweep(const TI* __restrict__ ids, int seg, int beg, int end, bool wide, unsigned vocab,
                                     unsigned padding, unsigned bin, int log_c, int lane, int* list, int* count, int& less,
                                     bool& bad) {
  constexpr int kPairs = 8;
  const unsigned low = (1u << log_c) - 1, before = (1u << lane) - 1;
  int len = 0;
  for (int t0 = beg; t0 < end; t0 += kPairs * 64) {
    unsigned id[kPairs][2];
#pragma unroll
    for (int u = 0; u < kPairs; ++u) {
      const int t = t0 + 64 * u + 2 * lane;
      if (wide && t0 + 64 * u + 64 <= end) {
        using Raw = typename RawOf<2 * sizeof(TI)>::type;
        const Raw raw = __ldg(reinterpret_cast<const Raw*>(ids + t));
        id[u][0] = checked(reinterpret_cast<const TI*>(&raw)[0], vocab);
        id[u][1] = checked(reinterpret_cast<const TI*>(&raw)[1], vocab);
        if (bin == 0) bad |= id[u][0] == 0xffffffffu || id[u][1] == 0xffffffffu;
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          id[u][e] = 0xffffffffu;
          if (t + e < end) {
            id[u][e] = checked(__ldg(ids + t + e), vocab);
            bad |= id[u][e] == 0xffffffffu;
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kPairs; ++u) {
      if (t0 + 64 * u >= end) break;
      bool in[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const unsigned k = id[u][e];
        const unsigned c = k == padding || k == 0xffffffffu ? 0xffffffffu : k & low;
        less += c < bin;
        in[e] = c == bin;
      }
      if (!__any_sync(0xffffffffu, in[0] || in[1])) continue;
      const unsigned m0 = __ballot_sync(0xffffffffu, in[0]), m1 = __ballot_sync(0xffffffffu, in[1]);
      int at = len + __popc(m0 & before) + __popc(m1 & before);
      const int t = t0 - seg + 64 * u + 2 * lane;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (in[e]) {
          const int local = static_cast<int>(id[u][e] >> log_c);
          list[at++] = (t + e) << kSortLogRange | local;
          atomicAdd(count + local, 1);
        }
      len += __popc(m0) + __popc(m1);
    }
  }
  return len;
}

__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

template <typename TI, int C>
__global__ void __cluster_dims__(C, 1, 1) __launch_bounds__(kSortWarps * 32, 1)
    embed_sort_kernel(const TI* __restrict__ ids, int n, int per, unsigned vocab, unsigned padding, EmbedWs ws,
                      int* __restrict__ status) {
  // [kSortWarps][per] tokens of each warp, [kRankers][range] next positions of each ranking warp
  extern __shared__ int sm[];
  __shared__ int s_count[1 << kSortLogRange];  // tokens of each local id: of all segments, then of one
  __shared__ int s_next[1 << kSortLogRange];   // position of the next token of each local id
  __shared__ int s_less[kSortWarps], s_len[kSortWarps], s_sum[kSortWarps], s_off[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int range = 1 << ws.log_r;
  const int rank = static_cast<int>(cluster.block_rank());
  const int bin = blockIdx.x / C;
  const int share = kSortWarps * per;           // tokens of a CTA whose lists fit into shared memory
  const int segment = C * share;
  const int slot = threadIdx.x;                 // the thread's local id, where slot < range
  int* list = sm + warp * per;
  int* hist = sm + kSortWarps * per;
  s_count[slot] = 0;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const bool wide = reinterpret_cast<uintptr_t>(ids) % (2 * sizeof(TI)) == 0;
  int len = 0, less = 0;
  bool bad = false;
  auto take = [&](int seg) {  // this warp's part of a segment
    const long long from = static_cast<long long>(seg) + rank * share + warp * per;
    const int beg = static_cast<int>(min(from, static_cast<long long>(n)));
    const int end = static_cast<int>(min(from + per, static_cast<long long>(n)));
    len = sweep(ids, seg, beg, end, wide, vocab, padding, bin, ws.log_c, lane, list, s_count, less, bad);
  };
  // sum of every CTA's count of the thread's local id, and of the CTAs before this one
  auto gather = [&](int& earlier) {
    int total = 0;
    earlier = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const int c = cluster.map_shared_rank(s_count, r)[slot];
      total += c;
      earlier += r < rank ? c : 0;
    }
    return total;
  };
  for (long long seg = 0; seg < n; seg += segment) take(static_cast<int>(seg));
  if (bin == 0 && bad) atomicOr(status, kStatusBadShape);
  less = warp_sum(less);
  if (lane == 0) s_less[warp] = less;
  cluster.sync();
  // first position of each local id: the tokens of earlier bins, and of smaller local ids
  int earlier;
  const int total = gather(earlier);
  int base = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) base += cluster.map_shared_rank(s_less, r)[lane];
  base = warp_sum(base);
  const int incl = warp_scan(total, lane);
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  const int first = base + warp_sum(lane < warp ? s_sum[lane] : 0) + incl - total;
  const bool many = n > segment;
  s_next[slot] = first + (many ? 0 : earlier);
  if (rank == 0 && slot < range) {
    ws.start[bin * range + slot] = first;
    if (blockIdx.x + C >= gridDim.x && slot == range - 1) ws.start[ws.slots()] = first + total;
  }
  for (long long seg = 0; seg < n; seg += segment) {
    int of_segment = 0;
    if (many) {  // the lists hold the last segment only
      cluster.sync();  // all have read the counts
      s_count[slot] = 0;
      __syncthreads();
      take(static_cast<int>(seg));
      cluster.sync();
      of_segment = gather(earlier);
      of_segment -= earlier;  // of this CTA and those behind it
      s_next[slot] += earlier;
    }
    if (lane == 0) s_len[warp] = len;
    __syncthreads();
    // `rankers` warps share the CTA's tokens, 64 or more each, in token order
    const int mine = s_len[lane];
    const int ends = warp_scan(mine, lane);
    const int m = __shfl_sync(0xffffffffu, ends, 31);
    const int rankers = max(1, min(kRankers, (m + 63) / 64));
    const int each = ((m + rankers - 1) / rankers + 31) & ~31;
    if (warp == 0) s_off[lane] = ends - mine;
    if (rankers > 1)
      for (int i = threadIdx.x; i < rankers * range; i += kSortWarps * 32) hist[i] = 0;
    __syncthreads();
    // item i lies in the last list that starts at or before i
    auto item_at = [&](int i) {
      int w = 0;
#pragma unroll
      for (int o = kSortWarps / 2; o > 0; o >>= 1)
        if (s_off[w + o] <= i) w += o;
      return sm[w * per + i - s_off[w]];
    };
    const int i0 = min(m, warp * each), i1 = min(m, i0 + each);
    int* my = s_next;
    constexpr int kLocal = (1 << kSortLogRange) - 1;
    if (rankers > 1) {
      my = hist + min(warp, kRankers - 1) * range;  // the warps behind the rankers have no tokens
      for (int i = i0 + lane; i < i1; i += 32) atomicAdd(my + (item_at(i) & kLocal), 1);
      __syncthreads();
      if (slot < range) {
        int at = s_next[slot];
        for (int w = 0; w < rankers; ++w) {
          const int c = hist[w * range + slot];
          hist[w * range + slot] = at;
          at += c;
        }
        s_next[slot] = at;
      }
      __syncthreads();
    }
    for (int i = i0; i < i1; i += 32) {
      const bool on = i + lane < i1;
      const int item = on ? item_at(i + lane) : 0;
      const int k = on ? item & kLocal : -1;
      const unsigned same = __match_any_sync(0xffffffffu, k);
      const int before = __popc(same & ((1u << lane) - 1));
      if (on) {
        const int at = my[k] + before;
        ws.order[at] = static_cast<int>(seg) + (static_cast<unsigned>(item) >> kSortLogRange);
        ws.key[at] = bin * range + k;
      }
      __syncwarp();
      if (on && before == 0) my[k] += __popc(same);
      __syncwarp();
    }
    if (many) {
      // s_next stands behind this CTA's tokens: the next segment begins behind those of the others too
      __syncthreads();
      s_next[slot] += of_segment - s_count[slot];
    }
  }
  cluster.sync();  // the others may still read this CTA's counts
}

// ------------------------------------------------------------------ backward: reduce
template <int V>
__device__ __forceinline__ void emit_row(float* __restrict__ dst, const float (&acc)[V], float scale, int accumulate) {
  float o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = acc[j] * scale;
  if (!accumulate) {
    store_f32<V>(dst, o);
    return;
  }
  // One addition per element and call, so the order of the atomics does not matter, and calls on several
  // streams may add to one dW.  The global atomic takes a subnormal operand or result (below 2^-126) as
  // zero: dW is off by less than 2^-125 there.  Keeping such numbers costs more than they are worth: a
  // load, an addition and a store take 62 us for 32768 x 1024 instead of 44; compare-and-swap for terms
  // below 2^-101 only, 12 to 15 % more where a tenth of dy is zero (dropout), up to 30 % where half of it is.
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4)
      atomicAdd(reinterpret_cast<float4*>(dst + j), make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) atomicAdd(dst + j, o[j]);
  }
}

// A lane holds J vectors of V elements, 32 V columns apart: V J = kLaneColumns.
template <typename T, int V, int J>
__global__ void __launch_bounds__(kWarps * 32, 5)
    embed_reduce_kernel(const T* __restrict__ dy, long long ldy, float* __restrict__ dw, long long ldw, EmbedWs ws, int n,
                        long long chunks, int slabs, int vocab, int H, float scale, int accumulate) {
  __shared__ __align__(16) float s_head[kWarps][kSlab], s_tail[kWarps][kSlab];
  __shared__ int s_flags[kWarps], s_id[kWarps];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long chunk_ctas = chunks * slabs;
  if (blockIdx.x >= chunk_ctas) {  // rows that no token names
    const long long r0 = ((blockIdx.x - chunk_ctas) * kWarps + warp) * kZeroRows;
    if (r0 >= vocab) return;
    const int rows = static_cast<int>(min(static_cast<long long>(kZeroRows), vocab - r0));
    bool empty = false;
    if (lane < rows) {
      const int slot = ws.slot_of(static_cast<int>(r0) + lane);
      empty = ws.start[slot] == ws.start[slot + 1];
    }
    const unsigned m = __ballot_sync(0xffffffffu, empty);
    constexpr int C = V < 4 ? V : 4;
    const float z[C] = {};
    for (int r = 0; r < rows; ++r)
      if (m >> r & 1)
        for (int c = lane * C; c < H; c += 32 * C) store_f32<C>(dw + (r0 + r) * ldw + c, z);
    return;
  }
  const int chunk = static_cast<int>(blockIdx.x / slabs);
  const int slab = static_cast<int>(blockIdx.x - static_cast<long long>(chunk) * slabs);
  const int p0 = chunk * kChunk + warp * kWarpTokens;
  const int col0 = slab * kSlab;
  const int col = col0 + lane * V;
  bool on[J];
#pragma unroll
  for (int q = 0; q < J; ++q) on[q] = col + 32 * V * q < H;
  // positions behind `valid` hold nothing: they are read with the rest and masked
  const int valid = ws.start[ws.slots()];
  int tok = 0, key = -1, before = -1, after = -1;
  if (lane < kWarpTokens && p0 + lane < n) {
    tok = ws.order[p0 + lane];
    key = ws.key[p0 + lane];
  }
  if (p0 > 0 && p0 - 1 < n) before = ws.key[p0 - 1];
  if (p0 + kWarpTokens < n) after = ws.key[p0 + kWarpTokens];
  if (chunk * kChunk >= valid) return;  // the whole CTA
  const int m = min(kWarpTokens, valid - p0);
  if (p0 + kWarpTokens >= valid) after = -1;
  int flags = 0, head_id = 0;  // 1: a run comes from before, 2: a run goes on behind, 4: it is one run
  if (m > 0) {
    Pack<T, V> x[kWarpTokens][J];
#pragma unroll
    for (int u = 0; u < kWarpTokens; ++u) {
      const long long t = __shfl_sync(0xffffffffu, tok, u);
      if (u < m) {
        const T* row = dy + t * ldy + col;
#pragma unroll
        for (int q = 0; q < J; ++q)
          if (on[q]) x[u][q] = Pack<T, V>::load(row + 32 * V * q);
      }
    }
    const int key0 = __shfl_sync(0xffffffffu, key, 0), key1 = __shfl_sync(0xffffffffu, key, m - 1);
    const bool head = before == key0, tail = after == key1;
    flags = (head ? 1 : 0) | (tail ? 2 : 0) | (head && tail && key0 == key1 ? 4 : 0);
    head_id = ws.id_of(key0);
    // bit i: token i begins another run
    const int up = __shfl_up_sync(0xffffffffu, key, 1);
    const unsigned begins = __ballot_sync(0xffffffffu, lane > 0 && lane < m && key != up);
    const int id = ws.id_of(key);
    float acc[J][V];
    auto clear = [&] {
#pragma unroll
      for (int q = 0; q < J; ++q)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[q][j] = 0.f;
    };
    clear();
    auto keep = [&](float* dst) {
#pragma unroll
      for (int q = 0; q < J; ++q) store_f32<V>(dst + (lane + 32 * q) * V, acc[q]);
    };
    bool first = head;
    auto close = [&](int i) {  // the run that ends at token i
      const long long r = __shfl_sync(0xffffffffu, id, i);
      if (first) {
        keep(s_head[warp]);
      } else {
        float* row = dw + r * ldw + col;
#pragma unroll
        for (int q = 0; q < J; ++q)
          if (on[q]) emit_row<V>(row + 32 * V * q, acc[q], scale, accumulate);
      }
      first = false;
    };
#pragma unroll
    for (int u = 0; u < kWarpTokens; ++u) {
      if (u >= m) break;
      if (begins >> u & 1) {
        close(u - 1);
        clear();
      }
#pragma unroll
      for (int q = 0; q < J; ++q)
        if (on[q]) {
          float f[V];
          x[u][q].get(f);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[q][j] += f[j];
        }
    }
    if (!first && tail) keep(s_tail[warp]);
    else close(m - 1);
  }
  if (lane == 0) {
    s_flags[warp] = flags;
    s_id[warp] = head_id;
  }
  __syncthreads();
  // Runs that cross warps: the threads of a column follow the one that is open.  What crosses the
  // chunk's ends goes to the workspace.
  for (int c = threadIdx.x; c < kSlab; c += kWarps * 32) {
    if (col0 + c >= H) break;
    float carry = 0.f;
    bool from_before = s_flags[0] & 1, open = false;
    for (int w = 0; w < kWarps; ++w) {
      const int f = s_flags[w];
      if (f & 1) {
        carry += s_head[w][c];
        open = f & 4;
        if (!open) {
          if (from_before) {
            ws.part[static_cast<long long>(chunk) * H + col0 + c] = carry;
          } else {
            const float one[1] = {carry};
            emit_row<1>(dw + s_id[w] * ldw + col0 + c, one, scale, accumulate);
          }
          from_before = false;
        }
      }
      if ((f & 2) && !(f & 4)) {
        carry = s_tail[w][c];
        open = true;
        from_before = false;
      }
    }
    if (open) ws.part[((from_before ? 0 : chunks) + chunk) * H + col0 + c] = carry;
  }
}

// Runs that cross chunks: a warp looks at one chunk's end and, where a run that began in the chunk
// goes on, adds its pieces, one per chunk, in order.  The pieces of long runs (more than kOwnPieces)
// are added by all of the CTA's warps: warp w takes every eighth, then the warps in turn.
constexpr int kJoinWarps = kThreads / 32, kOwnPieces = 4;
__global__ void __launch_bounds__(kThreads)
    embed_join_kernel(float* __restrict__ dw, long long ldw, EmbedWs ws, long long chunks, int slabs, int H, float scale,
                      int accumulate) {
  constexpr int B = 4;  // pieces in flight
  static_assert(kThreads == kSlab, "a thread per column");
  __shared__ float sum[kJoinWarps][kSlab];
  __shared__ int s_pieces[kJoinWarps], s_id[kJoinWarps];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk0 = static_cast<int>(blockIdx.x / slabs) * kJoinWarps;
  const int col0 = static_cast<int>(blockIdx.x % slabs) * kSlab;
  // acc = pieces first, first + step, ... of the m that begin in chunk c
  float acc[kLaneColumns];
  auto add = [&](int c, int m, int first, int step) {
#pragma unroll
    for (int j = 0; j < kLaneColumns; ++j) acc[j] = 0.f;
    for (int i0 = first; i0 < m; i0 += B * step) {
      float x[B][kLaneColumns];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int i = i0 + u * step;
        const float* p = ws.part + ((i == 0 ? chunks : 0) + c + i) * H + col0 + lane;  // the first lies in slot 1
#pragma unroll
        for (int j = 0; j < kLaneColumns; ++j) x[u][j] = i < m && col0 + lane + 32 * j < H ? p[32 * j] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < B; ++u)
#pragma unroll
        for (int j = 0; j < kLaneColumns; ++j) acc[j] += x[u][j];
    }
  };
  const int chunk = chunk0 + warp, next = (chunk + 1) * kChunk;
  int pieces = 0, slot = 0;
  if (chunk + 1 < chunks) {
    const int valid = ws.start[ws.slots()], last = ws.key[next - 1];
    slot = ws.key[next];
    if (next < valid && last == slot && ws.start[slot] >= next - kChunk)
      pieces = (ws.start[slot + 1] - 1) / kChunk - chunk + 1;
  }
  const int id = pieces > 0 ? ws.id_of(slot) : 0;
  if (pieces > 0 && pieces <= kOwnPieces) {
    add(chunk, pieces, 0, 1);
#pragma unroll
    for (int j = 0; j < kLaneColumns; ++j) {
      const int c = col0 + lane + 32 * j;
      const float one[1] = {acc[j]};
      if (c < H) emit_row<1>(dw + id * ldw + c, one, scale, accumulate);
    }
  }
  if (lane == 0) {
    s_pieces[warp] = pieces > kOwnPieces ? pieces : 0;
    s_id[warp] = id;
  }
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) {
    const int m = s_pieces[w];
    if (m == 0) continue;
    add(chunk0 + w, m, warp, kJoinWarps);
#pragma unroll
    for (int j = 0; j < kLaneColumns; ++j) sum[warp][lane + 32 * j] = acc[j];
    __syncthreads();
    const int c = col0 + threadIdx.x;
    if (c < H) {
      float one[1] = {0.f};
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) one[0] += sum[i][threadIdx.x];
      emit_row<1>(dw + s_id[w] * ldw + c, one, scale, accumulate);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ backward: few tokens
// Up to kSmallTokens tokens in one launch (the three above take longer to launch than to run: at 128
// tokens 8.3 us, this one 5.8): every
// CTA has 64 columns and sorts the tokens itself, a token's place being the number of tokens with a
// smaller id, or the same id and an earlier place.  Its 32 warps add consecutive parts of the sorted
// tokens, and runs that cross warps meet in shared memory.  Further CTAs write the zeros.
constexpr int kSmallTokens = 256, kSmallWarps = 32, kSmallSlab = 64;
constexpr int kSmallPer = kSmallTokens / kSmallWarps;  // sorted tokens per warp at most

template <typename TI, typename T, int V>
__global__ void __launch_bounds__(kSmallWarps * 32, 1)
    embed_small_kernel(const TI* __restrict__ ids, int n, unsigned vocab, unsigned padding, const T* __restrict__ dy,
                       long long ldy, float* __restrict__ dw, long long ldw, int slabs, int H, float scale, int accumulate,
                       int zero_rows, int quads, int* __restrict__ status) {
  constexpr int J = 2 / V;  // vectors per lane
  __shared__ __align__(16) int s_id[kSmallTokens];
  __shared__ int s_order[kSmallTokens], s_key[kSmallTokens];
  __shared__ __align__(16) float s_head[kSmallWarps][kSmallSlab], s_tail[kSmallWarps][kSmallSlab];
  __shared__ int s_flags[kSmallWarps];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kNone = 0x7fffffff;
  int mine = kNone;
  if (threadIdx.x < n) {
    const unsigned id = checked(__ldg(ids + threadIdx.x), vocab);
    if (id == 0xffffffffu) {
      if (blockIdx.x == 0) atomicOr(status, kStatusBadShape);
    } else if (id != padding) {
      mine = static_cast<int>(id);
    }
  }
  if (static_cast<int>(blockIdx.x) >= slabs) {  // rows that no token names
    const long long r0 = static_cast<long long>(blockIdx.x - slabs) * zero_rows;
    if (threadIdx.x < kSmallTokens) s_id[threadIdx.x] = 0;
    __syncthreads();
    if (mine >= r0 && mine < r0 + zero_rows) s_id[mine - r0] = 1;
    __syncthreads();
    const int rows = static_cast<int>(min(static_cast<long long>(zero_rows), vocab - r0));
    const float z[4] = {}, z1[1] = {};
    for (int r = warp; r < rows; r += kSmallWarps) {
      if (s_id[r] != 0) continue;
      float* row = dw + (r0 + r) * ldw;
      if (quads)
        for (int c = lane * 4; c < H; c += 32 * 4) store_f32<4>(row + c, z);
      else
        for (int c = lane; c < H; c += 32) store_f32<1>(row + c, z1);
    }
    return;
  }
  if (threadIdx.x < kSmallTokens) s_id[threadIdx.x] = mine;
  const int valid = __syncthreads_count(mine != kNone);
  // four threads per token, each with every fourth four ids
  static_assert(kSmallWarps * 32 == 4 * kSmallTokens, "four threads per token");
  const int token = threadIdx.x >> 2;
  const int id = s_id[token];
  int place = 0;
  for (int j = (threadIdx.x & 3) * 4; j < n; j += 16) {
    const int4 k = *reinterpret_cast<const int4*>(s_id + j);
    place += k.x < id || (k.x == id && j < token);
    place += k.y < id || (k.y == id && j + 1 < token);
    place += k.z < id || (k.z == id && j + 2 < token);
    place += k.w < id || (k.w == id && j + 3 < token);
  }
  place += __shfl_xor_sync(0xffffffffu, place, 1);
  place += __shfl_xor_sync(0xffffffffu, place, 2);
  if ((threadIdx.x & 3) == 0 && id != kNone) {
    s_order[place] = token;
    s_key[place] = id;
  }
  __syncthreads();
  const int per = (valid + kSmallWarps - 1) / kSmallWarps;
  const int p0 = min(valid, warp * per), m = min(per, valid - p0);
  const int col0 = static_cast<int>(blockIdx.x) * kSmallSlab;
  const int col = col0 + lane * V;
  bool on[J];
#pragma unroll
  for (int q = 0; q < J; ++q) on[q] = col + 32 * V * q < H;
  int flags = 0;  // 1: a run comes from before, 2: a run goes on behind, 4: it is one run
  if (m > 0) {
    Pack<T, V> x[kSmallPer][J];
#pragma unroll
    for (int u = 0; u < kSmallPer; ++u)
      if (u < m) {
        const T* row = dy + s_order[p0 + u] * ldy + col;
#pragma unroll
        for (int q = 0; q < J; ++q)
          if (on[q]) x[u][q] = Pack<T, V>::load(row + 32 * V * q);
      }
    const int key0 = s_key[p0], key1 = s_key[p0 + m - 1];
    const bool head = p0 > 0 && s_key[p0 - 1] == key0, tail = p0 + m < valid && s_key[p0 + m] == key1;
    flags = (head ? 1 : 0) | (tail ? 2 : 0) | (head && tail && key0 == key1 ? 4 : 0);
    float acc[J][V] = {};
    auto keep = [&](float* dst) {
#pragma unroll
      for (int q = 0; q < J; ++q) store_f32<V>(dst + (lane + 32 * q) * V, acc[q]);
    };
    bool first = head;
    auto close = [&](int key) {
      if (first) {
        keep(s_head[warp]);
      } else {
        float* row = dw + key * ldw + col;
#pragma unroll
        for (int q = 0; q < J; ++q)
          if (on[q]) emit_row<V>(row + 32 * V * q, acc[q], scale, accumulate);
      }
      first = false;
    };
    int cur = key0;
#pragma unroll
    for (int u = 0; u < kSmallPer; ++u) {
      if (u >= m) break;
      const int key = s_key[p0 + u];
      if (key != cur) {
        close(cur);
        cur = key;
#pragma unroll
        for (int q = 0; q < J; ++q)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[q][j] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < J; ++q)
        if (on[q]) {
          float f[V];
          x[u][q].get(f);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[q][j] += f[j];
        }
    }
    if (!first && tail) keep(s_tail[warp]);
    else close(cur);
  }
  if (lane == 0) s_flags[warp] = flags;
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= kSmallSlab || col0 + c >= H) return;
  float carry[1] = {0.f};
  for (int w = 0; w < kSmallWarps; ++w) {
    const int f = s_flags[w];
    if (f & 1) {
      carry[0] += s_head[w][c];
      if (!(f & 4)) emit_row<1>(dw + s_key[w * per] * ldw + col0 + c, carry, scale, accumulate);
    }
    if ((f & 2) && !(f & 4)) carry[0] = s_tail[w][c];
  }
}

// ------------------------------------------------------------------ host
bool float_type(const torch::Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
}
bool id_type(const torch::Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

// Whether rows of t, `stride` elements apart, allow accesses of `elems` elements.
bool rows_allow(const torch::Tensor& t, long long stride, long long rows, int elems) {
  const long long bytes = static_cast<long long>(elems) * t.element_size();
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0 &&
         (rows <= 1 || (stride * static_cast<long long>(t.element_size())) % bytes == 0);
}

void check_rows(const torch::Tensor& t, const char* name) {
  REVPP_CHECK(t.dim() == 2, name, " must be 2-D");
  REVPP_CHECK(float_type(t), name, " must be float32, bfloat16 or float16");
  REVPP_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must be contiguous along its last dimension");
}
void check_written_rows(const torch::Tensor& t, const char* name) {
  REVPP_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " has rows that overlap");
}
void check_same_device(const torch::Tensor& a, const torch::Tensor& b, const char* names) {
  REVPP_CHECK(a.is_cuda() && b.is_cuda(), names, " must be CUDA tensors");
  REVPP_CHECK(a.device() == b.device(), names, " must be on the same device");
}

// A written tensor must lie apart from what is read.
void check_apart(const torch::Tensor& written, const torch::Tensor& read, const char* names) {
  auto end = [](const torch::Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) + ((t.size(0) - 1) * t.stride(0) + t.size(1)) * t.element_size();
  };
  REVPP_CHECK(end(written) <= reinterpret_cast<uintptr_t>(read.data_ptr()) ||
                  end(read) <= reinterpret_cast<uintptr_t>(written.data_ptr()),
              names, " must not overlap");
}

template <typename F>
void by_float(at::ScalarType t, F&& f) {
  if (t == at::kFloat)
    f(float{});
  else if (t == at::kBFloat16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

long long align256(long long b) { return (b + 255) / 256 * 256; }

struct Plan {
  int v, slabs, log_c, log_r, cluster;
  long long chunks, off_order, off_key, off_part, bytes;
};
Plan plan_bwd(long long n, long long vocab, int H, int v) {
  Plan p;
  p.v = v;
  p.slabs = (H + kSlab - 1) / kSlab;
  p.log_c = p.log_r = 0;
  while ((kSortCluster << p.log_c) < kSortCtas && (1LL << p.log_c) < vocab) ++p.log_c;
  while ((1LL << (p.log_c + p.log_r)) < vocab) ++(p.log_r < kSortLogRange ? p.log_r : p.log_c);
  p.cluster = kSortCluster;
  while (p.cluster > 1 && (static_cast<long long>(p.cluster) << p.log_c) > kSortCtas) p.cluster /= 2;
  p.chunks = (n + kChunk - 1) / kChunk;
  p.off_order = align256(((1LL << (p.log_c + p.log_r)) + 1) * 4);
  p.off_key = p.off_order + align256(n * 4);
  p.off_part = p.off_key + align256(n * 4);
  p.bytes = p.off_part + align256(2 * p.chunks * H * 4);
  return p;
}

}  // namespace

void embedding_fwd(const torch::Tensor& ids, const torch::Tensor& w, torch::Tensor out, double scale) {
  REVPP_CHECK(id_type(ids) && ids.is_contiguous(), "ids must be contiguous int64 or int32");
  check_rows(w, "w");
  check_rows(out, "out");
  check_written_rows(out, "out");
  const long long n = ids.numel(), vocab = w.size(0);
  REVPP_CHECK(out.size(0) == n && out.size(1) == w.size(1), "out must be [", n, ", ", w.size(1), "], got [", out.size(0),
              ", ", out.size(1), "]");
  REVPP_CHECK(w.size(1) <= (1 << 30), "rows too wide");
  if (n == 0 || w.size(1) == 0) return;
  REVPP_CHECK(vocab > 0, "the table is empty");
  check_apart(out, w, "out and w");
  check_same_device(ids, w, "ids and w");
  check_same_device(w, out, "w and out");
  c10::cuda::CUDAGuard guard(w.device());
  const int H = static_cast<int>(w.size(1));
  // the narrower type in 16-byte accesses, the other in one or two
  const int w_most = 16 / static_cast<int>(w.element_size()), out_most = 16 / static_cast<int>(out.element_size());
  int v = std::max(w_most, out_most);
  while (v > 1 && !(H % v == 0 && rows_allow(w, w.stride(0), vocab, std::min(v, w_most)) &&
                    rows_allow(out, out.stride(0), n, std::min(v, out_most))))
    v /= 2;
  int log_l = 0;
  while (log_l < 5 && (kFwdUnroll << log_l) * v < H) ++log_l;  // narrow rows: several per warp, all lanes loading
  const int per_slab = (kFwdUnroll << log_l) * v;
  const int slabs = (H + per_slab - 1) / per_slab;
  const long long threads = (n * slabs) << log_l;
  const long long blocks = std::min<long long>((threads + kThreads - 1) / kThreads, kFwdBlocksPerSm * num_sms());
  int* status = status_device_ptr();
  by_float(w.scalar_type(), [&](auto tw) {
    using TW = decltype(tw);
    by_float(out.scalar_type(), [&](auto to) {
      using TO = decltype(to);
      auto go = [&](auto ti, auto vc) {
        using TI = decltype(ti);
        constexpr int V = decltype(vc)::value;
        if constexpr (V * std::min(sizeof(TW), sizeof(TO)) <= 16)
          launch_pdl(embed_fwd_kernel<TI, TW, TO, V>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, cur_stream(),
                     static_cast<const TI*>(ids.data_ptr()), static_cast<const TW*>(w.data_ptr()),
                     static_cast<long long>(w.stride(0)), static_cast<TO*>(out.data_ptr()),
                     static_cast<long long>(out.stride(0)), n, vocab, H, log_l, slabs, static_cast<float>(scale), status);
      };
      auto by_v = [&](auto ti) {
        if (v == 8) go(ti, std::integral_constant<int, 8>{});
        else if (v == 4) go(ti, std::integral_constant<int, 4>{});
        else if (v == 2) go(ti, std::integral_constant<int, 2>{});
        else go(ti, std::integral_constant<int, 1>{});
      };
      if (ids.scalar_type() == at::kLong) by_v(int64_t{});
      else by_v(int32_t{});
    });
  });
  REVPP_CHECK_LAUNCH();
}

void embedding_bwd(const torch::Tensor& dy, const torch::Tensor& ids, torch::Tensor dw, double scale, int64_t padding_idx,
                   bool accumulate) {
  REVPP_CHECK(id_type(ids) && ids.is_contiguous(), "ids must be contiguous int64 or int32");
  check_rows(dy, "dy");
  check_rows(dw, "dw");
  REVPP_CHECK(dw.scalar_type() == at::kFloat, "dw must be float32");
  check_written_rows(dw, "dw");
  const long long n = ids.numel(), vocab = dw.size(0);
  REVPP_CHECK(dy.size(0) == n && dy.size(1) == dw.size(1), "dy must be [", n, ", ", dw.size(1), "], got [", dy.size(0),
              ", ", dy.size(1), "]");
  REVPP_CHECK(n < (1LL << 26) && vocab < (1LL << 30) && dw.size(1) < (1LL << 30), "too many tokens, rows or columns");
  if (vocab == 0 || dw.size(1) == 0 || (n == 0 && accumulate)) return;
  if (n > 0) check_apart(dw, dy, "dw and dy");
  check_same_device(dy, dw, "dy and dw");
  check_same_device(ids, dw, "ids and dw");
  c10::cuda::CUDAGuard guard(dw.device());
  const int H = static_cast<int>(dw.size(1));
  int v = 16 / static_cast<int>(dy.element_size());
  // rows of the workspace are H floats: a vector of v floats in it needs H % v == 0 too
  while (v > 1 && !(H % v == 0 && rows_allow(dy, dy.stride(0), n, v) && rows_allow(dw, dw.stride(0), vocab, std::min(v, 4))))
    v /= 2;
  // One launch up to 256 tokens, at any width: 256 tokens added to a table of 30522 rows take 7.7 us
  // against 9.4 in three launches at 128 columns, 7.7 against 9.8 at 1024, 7.9 against 12.7 at 4096, written
  // 7.2 against 10.5, 24.4 against 26.2 and 80.4 against 85.6 (replayed from a graph).  At 512 tokens
  // the sorting in every CTA makes it 16 us against 12.8.
  if (n <= kSmallTokens) {
    const unsigned padding = padding_idx >= 0 && padding_idx < vocab ? static_cast<unsigned>(padding_idx) : 0xffffffffu;
    const int slabs = (H + kSmallSlab - 1) / kSmallSlab;
    // two zero-writing CTAs per SM where the table has the rows: 32 (one per warp) to 256 each
    const int zero_rows = static_cast<int>(std::min<long long>(
        kSmallTokens, std::max<long long>(kSmallWarps, (vocab + 2 * num_sms() - 1) / (2 * num_sms()))));
    const long long blocks = slabs + (accumulate ? 0 : (vocab + zero_rows - 1) / zero_rows);
    REVPP_CHECK(blocks < (1LL << 31), "too many rows");
    const int quads = H % 4 == 0 && rows_allow(dw, dw.stride(0), vocab, 4);
    int* status = status_device_ptr();
    by_float(dy.scalar_type(), [&](auto t) {
      using T = decltype(t);
      auto go = [&](auto ti, auto vc) {
        using TI = decltype(ti);
        launch_pdl(embed_small_kernel<TI, T, decltype(vc)::value>, dim3(static_cast<unsigned>(blocks)), dim3(kSmallWarps * 32),
                   0, cur_stream(), static_cast<const TI*>(ids.data_ptr()), static_cast<int>(n), static_cast<unsigned>(vocab),
                   padding, static_cast<const T*>(dy.data_ptr()), static_cast<long long>(dy.stride(0)), dw.data_ptr<float>(),
                   static_cast<long long>(dw.stride(0)), slabs, H, static_cast<float>(scale), accumulate ? 1 : 0, zero_rows, quads,
                   status);
      };
      auto by_v = [&](auto ti) {
        if (v >= 2) go(ti, std::integral_constant<int, 2>{});
        else go(ti, std::integral_constant<int, 1>{});
      };
      if (ids.scalar_type() == at::kLong) by_v(int64_t{});
      else by_v(int32_t{});
    });
    REVPP_CHECK_LAUNCH();
    return;
  }
  const Plan p = plan_bwd(n, vocab, H, v);
  torch::Tensor buf = torch::empty({p.bytes}, dw.options().dtype(at::kByte));
  char* base = static_cast<char*>(buf.data_ptr());
  EmbedWs ws{reinterpret_cast<int*>(base), reinterpret_cast<int*>(base + p.off_order),
             reinterpret_cast<int*>(base + p.off_key), reinterpret_cast<float*>(base + p.off_part), p.log_c, p.log_r};
  int* status = status_device_ptr();
  // the cluster's warps list all tokens, in segments where there are more than kSortPer for each
  const int lists = p.cluster * kSortWarps * 64;
  const int per = static_cast<int>(std::min<long long>(kSortPer, (n + lists - 1) / lists * 64));
  const size_t smem = (static_cast<size_t>(kRankers << p.log_r) + kSortWarps * per) * 4;
  const unsigned padding = padding_idx >= 0 && padding_idx < vocab ? static_cast<unsigned>(padding_idx) : 0xffffffffu;
  auto sort = [&](auto ti, auto cluster) {
    using TI = decltype(ti);
    constexpr auto kernel = &embed_sort_kernel<TI, decltype(cluster)::value>;
    static std::atomic<uint64_t> ready{0};  // devices that know the kernel's shared memory
    const uint64_t bit = 1ull << (dw.get_device() & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
      REVPP_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            ((kRankers << kSortLogRange) + kSortWarps * kSortPer) * 4));
      ready.fetch_or(bit, std::memory_order_relaxed);
    }
    launch_pdl(kernel, dim3(static_cast<unsigned>(p.cluster) << p.log_c), dim3(kSortWarps * 32), smem, cur_stream(),
               static_cast<const TI*>(ids.data_ptr()), static_cast<int>(n), per, static_cast<unsigned>(vocab), padding, ws, status);
  };
  auto by_cluster = [&](auto ti) {
    if (p.cluster == 4) sort(ti, std::integral_constant<int, 4>{});
    else if (p.cluster == 2) sort(ti, std::integral_constant<int, 2>{});
    else sort(ti, std::integral_constant<int, 1>{});
  };
  if (ids.scalar_type() == at::kLong) by_cluster(int64_t{});
  else by_cluster(int32_t{});
  REVPP_CHECK_LAUNCH();
  const long long zero_rows = kWarps * kZeroRows;
  const long long blocks = p.chunks * p.slabs + (accumulate ? 0 : (vocab + zero_rows - 1) / zero_rows);
  REVPP_CHECK(blocks < (1LL << 31), "too many tokens");
  by_float(dy.scalar_type(), [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vc) {
      constexpr int V = decltype(vc)::value;
      if constexpr (V * sizeof(T) <= 16)
        launch_pdl(embed_reduce_kernel<T, V, kLaneColumns / V>, dim3(static_cast<unsigned>(blocks)), dim3(kWarps * 32), 0,
                   cur_stream(), static_cast<const T*>(dy.data_ptr()), static_cast<long long>(dy.stride(0)),
                   dw.data_ptr<float>(), static_cast<long long>(dw.stride(0)), ws, static_cast<int>(n), p.chunks, p.slabs,
                   static_cast<int>(vocab), H,
                   static_cast<float>(scale), accumulate ? 1 : 0);
    };
    if (v == 8) go(std::integral_constant<int, 8>{});
    else if (v == 4) go(std::integral_constant<int, 4>{});
    else if (v == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
  });
  REVPP_CHECK_LAUNCH();
  if (p.chunks < 2) return;  // no run crosses chunks
  const long long joins = (p.chunks - 1 + kJoinWarps - 1) / kJoinWarps * p.slabs;
  launch_pdl(embed_join_kernel, dim3(static_cast<unsigned>(joins)), dim3(kThreads), 0, cur_stream(),
             dw.data_ptr<float>(), static_cast<long long>(dw.stride(0)), ws, p.chunks, p.slabs, H,
             static_cast<float>(scale), accumulate ? 1 : 0);
  REVPP_CHECK_LAUNCH();
}

}  // namespace revpp

// Token-embedding lookup with a scale, and its gradient by sorted tokens.
//
//   fwd : out[t, :] = scale * W[id[t], :]
//   bwd : dW[v, :] (+)= scale * sum_{t : id[t] = v, v != padding} dy[t, :]
//
// Tables and activations are fp32, bf16 or fp16, sums and dW fp32.  An id outside the table
// sets kStatusBadShape, gives a row of zeros and adds nothing to dW.
//
// Backward.  Adding rows with atomics makes the result depend on the order in which they
// arrive; here the tokens are sorted by id (stable, so each row's terms come in token order)
// and every dW row is written once, so equal inputs give equal bits.
//
//  1. embed_sort_kernel: each CTA owns a range of ids, reads all n ids, counts those below
//     its range (its offset in the sorted order, with no exchange between CTAs) and places its
//     own by a counting sort.  Warp w reads the w-th part of the tokens and keeps its own
//     counters, so that the order within an id is the token order.
//  2. embed_reduce_kernel: one warp per (32 sorted tokens, slab of columns) adds the rows of
//     each run of equal ids in registers.  A run inside the 32 goes straight to dW; a run
//     that crosses into neighbouring chunks leaves its pieces in the workspace, and the warp
//     that delivers the last piece adds them in chunk order (in groups of 32 for long runs).
//     Without accumulation, further warps write zeros to the rows that no token names.
#include <algorithm>

#include "common.cuh"
#include "host.h"
#include "vec.cuh"

namespace revpp {

namespace {

constexpr int kThreads = 256;
constexpr int kFwdUnroll = 4;      // vectors per lane and row slab
constexpr int kSortWarps = 32;
constexpr int kSortList = 256;     // matches a warp keeps between the two sweeps
constexpr int kSortRange = 512;    // ids per CTA at most
constexpr int kChunk = 32;         // sorted tokens per reduce task
constexpr int kZeroRows = 8;       // dW rows per zero-writing warp

// ------------------------------------------------------------------ forward
// L lanes (a power of two) per (row, slab of L * V * kFwdUnroll columns).
template <typename TI, typename TW, typename TO, int V>
__global__ void __launch_bounds__(kThreads)
    embed_fwd_kernel(const TI* __restrict__ ids, const TW* __restrict__ w, long long ldw, TO* __restrict__ out,
                     long long ldo, long long n, long long vocab, int H, int log_l, int slabs, float scale,
                     int* __restrict__ status) {
  pdl_wait();
  pdl_trigger();
  const long long group = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> log_l;
  const int sub = threadIdx.x & ((1 << log_l) - 1);
  const long long row = group / slabs;
  if (row >= n) return;
  const int slab = static_cast<int>(group - row * slabs);
  const long long id = static_cast<long long>(ids[row]);
  const bool ok = id >= 0 && id < vocab;
  if (!ok && sub == 0 && slab == 0) atomicOr(status, kStatusBadShape);
  const TW* src = w + (ok ? id : 0) * ldw;
  TO* dst = out + row * ldo;
  const int c0 = ((slab * kFwdUnroll << log_l) + sub) * V;
  Pack<TW, V> x[kFwdUnroll];
#pragma unroll
  for (int u = 0; u < kFwdUnroll; ++u) {
    const int c = c0 + ((u * V) << log_l);
    if (c < H && ok) x[u] = Pack<TW, V>::load_ro(src + c);
  }
#pragma unroll
  for (int u = 0; u < kFwdUnroll; ++u) {
    const int c = c0 + ((u * V) << log_l);
    if (c >= H) continue;
    float f[V];
    x[u].get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = ok ? f[j] * scale : 0.f;
    Pack<TO, V> y;
    y.set(f);
    y.store(dst + c);
  }
}

// ------------------------------------------------------------------ backward: sort
struct EmbedWs {
  int* start;     // [vocab + 1] first sorted position of each id
  int* order;     // [n] token of each sorted position
  int* key;       // [n] id of each sorted position
  int* count;     // [3][slabs][chunks] pieces delivered
  float* part;    // [2][chunks][H] pieces of runs that cross chunks
};

// The tokens of one warp whose id lies in [lo, lo + range), in token order, 32 at a time at
// most: fn(token, local id, active).  Returns through `less` the number of ids below lo.
template <typename TI, typename F>
__device__ __forceinline__ void sweep(const TI* __restrict__ ids, int beg, int end, long long vocab, long long padding,
                                      int lo, int range, int lane, int* list_tok, int* list_id, int& len, int& less,
                                      bool& bad, bool& spilled, F&& fn) {
  len = 0;
  for (int t0 = beg; t0 < end; t0 += 8 * 32) {
    int k[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = t0 + 32 * u + lane;
      long long id = -1;
      if (t < end) {
        id = static_cast<long long>(ids[t]);
        bad |= id < 0 || id >= vocab;
      }
      k[u] = (id >= 0 && id < vocab && id != padding) ? static_cast<int>(id) : 0x7fffffff;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      less += k[u] < lo;
      const bool in = static_cast<unsigned>(k[u] - lo) < static_cast<unsigned>(range);
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (m == 0) continue;
      if (len > kSortList - 32) {
        spilled = true;
        __syncwarp();
        for (int i = 0; i < len; i += 32) fn(list_tok, list_id, i, len);
        len = 0;
        __syncwarp();
      }
      if (in) {
        const int at = len + __popc(m & ((1u << lane) - 1));
        list_tok[at] = t0 + 32 * u + lane;
        list_id[at] = k[u] - lo;
      }
      len += __popc(m);
    }
  }
  __syncwarp();
}

template <typename TI>
__global__ void __launch_bounds__(kSortWarps * 32, 1)
    embed_sort_kernel(const TI* __restrict__ ids, int n, int vocab, long long padding, int range, EmbedWs ws,
                      long long counters, int* __restrict__ status) {
  extern __shared__ int sm[];  // [kSortWarps][range] counters, [kSortWarps][2][kSortList] matches
  __shared__ int s_less[kSortWarps];
  __shared__ int s_sum[kSortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* hist = sm + warp * range;
  int* list_tok = sm + kSortWarps * range + warp * 2 * kSortList;
  int* list_id = list_tok + kSortList;
  const int lo = blockIdx.x * range;
  const int width = min(range, vocab - lo);
  for (int i = lane; i < range; i += 32) hist[i] = 0;
  pdl_wait();
  pdl_trigger();
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < counters;
       i += static_cast<long long>(gridDim.x) * blockDim.x)
    ws.count[i] = 0;
  __syncwarp();
  const int per = ((n + kSortWarps - 1) / kSortWarps + 31) & ~31;
  const int beg = static_cast<int>(min(static_cast<long long>(warp) * per, static_cast<long long>(n)));
  const int end = static_cast<int>(min(static_cast<long long>(beg) + per, static_cast<long long>(n)));
  int len = 0, less = 0;
  bool bad = false, spilled = false;
  auto count = [&](const int* tok, const int* id, int i, int m) {
    const bool on = i + lane < m;
    const int k = on ? id[i + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, k);
    if (on && (same & ((1u << lane) - 1)) == 0) hist[k] += __popc(same);
    __syncwarp();
  };
  sweep(ids, beg, end, vocab, padding, lo, width, lane, list_tok, list_id, len, less, bad, spilled, count);
  for (int i = 0; i < len; i += 32) count(list_tok, list_id, i, len);
  if (blockIdx.x == 0 && bad) atomicOr(status, kStatusBadShape);
  less = warp_sum(less);
  if (lane == 0) s_less[warp] = less;
  __syncthreads();
  // thread j: the warps' counts of id lo + j become offsets; a block scan over j gives the starts
  const int j = threadIdx.x;
  int total = 0;
  if (j < width)
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = sm[w * range + j];
      sm[w * range + j] = total;
      total += c;
    }
  int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWarps; ++w) {
    base += s_less[w];
    if (w < warp) base += s_sum[w];
  }
  const int first = base + incl - total;
  if (j < width) {
    ws.start[lo + j] = first;
    if (lo + j == vocab - 1) ws.start[vocab] = first + total;
    for (int w = 0; w < kSortWarps; ++w) sm[w * range + j] += first;
  }
  __syncthreads();
  auto place = [&](const int* tok, const int* id, int i, int m) {
    const bool on = i + lane < m;
    const int k = on ? id[i + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, k);
    if (on) {
      const int at = hist[k] + __popc(same & ((1u << lane) - 1));
      ws.order[at] = tok[i + lane];
      ws.key[at] = lo + k;
    }
    __syncwarp();
    if (on && (same & ((1u << lane) - 1)) == 0) hist[k] += __popc(same);
    __syncwarp();
  };
  if (spilled)
    sweep(ids, beg, end, vocab, padding, lo, width, lane, list_tok, list_id, len, less, bad, spilled, place);
  for (int i = 0; i < len; i += 32) place(list_tok, list_id, i, len);
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
  // one addition per element and call: the order of the atomics does not matter
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4)
      atomicAdd(reinterpret_cast<float4*>(dst + j), make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) atomicAdd(dst + j, o[j]);
  }
}

// part[slot][chunk] of `m` pieces, `step` chunks apart from chunk c0 on (the first in `slot0`,
// the others in slot 0), added in order.
template <int V>
__device__ __forceinline__ void add_pieces(const float* part, long long chunks, int H, int col, int slot0, int c0, int m,
                                           int step, float (&acc)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  constexpr int C = V < 4 ? V : 4;
  for (int i0 = 0; i0 < m; i0 += 4) {
    typename Pack<float, C>::Raw raw[4][V / C];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < m) {
        const long long c = c0 + static_cast<long long>(i0 + u) * step;
        const float* p = part + ((i0 + u == 0 ? slot0 : 0) * chunks + c) * H + col;
#pragma unroll
        for (int q = 0; q < V / C; ++q)
          raw[u][q] = __ldcg(reinterpret_cast<const typename Pack<float, C>::Raw*>(p + q * C));
      }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < m) {
#pragma unroll
        for (int q = 0; q < V / C; ++q) {
          float t[C];
          Pack<float, C>{raw[u][q]}.get(t);
#pragma unroll
          for (int j = 0; j < C; ++j) acc[q * C + j] += t[j];
        }
      }
  }
}

// One piece of the run [s, e) lies in chunk c; its sum is already in `part`.  The warp that
// delivers the run's last piece adds them all.
template <int V>
__device__ void join_run(EmbedWs ws, long long chunks, int H, int col, bool on, int lane, const int* counts_of_slab,
                         int c, int s, int e, float* dst, float scale, int accumulate) {
  int* cnt = const_cast<int*>(counts_of_slab);  // [3][chunks]
  const int c0 = s / kChunk, c1 = (e - 1) / kChunk;
  int m = c1 - c0 + 1, step = 1;
  float acc[V];
  if (m > kChunk) {  // groups of 32 pieces first
    const int g = (c - c0) / kChunk;
    const int gc = c0 + g * kChunk;
    const int in_group = min(kChunk, m - g * kChunk);
    int last = 0;
    if (lane == 0) last = atomicAdd(cnt + (g == 0 ? 2 : 1) * chunks + gc, 1) == in_group - 1;
    if (!__shfl_sync(0xffffffffu, last, 0)) return;
    __threadfence();
    __syncwarp();
    if (on) {
      add_pieces<V>(ws.part, chunks, H, col, g == 0 ? 1 : 0, gc, in_group, 1, acc);
      store_f32<V>(ws.part + ((g == 0 ? 1 : 0) * chunks + gc) * H + col, acc);
    }
    __threadfence();
    __syncwarp();
    m = (m + kChunk - 1) / kChunk;
    step = kChunk;
  }
  int last = 0;
  if (lane == 0) last = atomicAdd(cnt + c0, 1) == m - 1;
  if (!__shfl_sync(0xffffffffu, last, 0)) return;
  __threadfence();
  __syncwarp();
  if (on) {
    add_pieces<V>(ws.part, chunks, H, col, 1, c0, m, step, acc);
    emit_row<V>(dst, acc, scale, accumulate);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    embed_reduce_kernel(const T* __restrict__ dy, long long ldy, float* __restrict__ dw, long long ldw, EmbedWs ws,
                        long long chunks, int slabs, int vocab, int H, float scale, int accumulate) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  long long task = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  if (task >= chunks * slabs) {  // rows that no token names
    const long long r0 = (task - chunks * slabs) * kZeroRows;
    if (accumulate || r0 >= vocab) return;
    const int rows = static_cast<int>(min(static_cast<long long>(kZeroRows), vocab - r0));
    bool empty = false;
    if (lane < rows) empty = ws.start[r0 + lane] == ws.start[r0 + lane + 1];
    const unsigned m = __ballot_sync(0xffffffffu, empty);
    const float z[V] = {};
    for (int r = 0; r < rows; ++r)
      if (m >> r & 1)
        for (int c = lane * V; c < H; c += 32 * V) store_f32<V>(dw + (r0 + r) * ldw + c, z);
    return;
  }
  const int c = static_cast<int>(task / slabs);
  const int slab = static_cast<int>(task - static_cast<long long>(c) * slabs);
  const int valid = ws.start[vocab];
  const int p0 = c * kChunk;
  const int m = min(kChunk, valid - p0);
  if (m <= 0) return;
  const int col = (slab * 32 + lane) * V;
  const bool on = col < H;
  int tok = 0, key = -1;
  if (lane < m) {
    tok = ws.order[p0 + lane];
    key = ws.key[p0 + lane];
  }
  const int key0 = __shfl_sync(0xffffffffu, key, 0);
  const int key1 = __shfl_sync(0xffffffffu, key, m - 1);
  const int s0 = ws.start[key0], e0 = ws.start[key0 + 1];
  const int s1 = ws.start[key1], e1 = ws.start[key1 + 1];
  const bool head = s0 < p0;                          // the first run began in an earlier chunk
  const bool tail = e1 > p0 + m && !(head && key0 == key1);  // the last run begins here and goes on
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int cur = key0;
  bool first = head;
  for (int i0 = 0; i0 < m; i0 += 8) {
    Pack<T, V> x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long long t = __shfl_sync(0xffffffffu, tok, i0 + u);
      if (i0 + u < m && on) x[u] = Pack<T, V>::load(dy + t * ldy + col);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = __shfl_sync(0xffffffffu, key, i0 + u);
      if (i0 + u >= m) break;
      if (k != cur) {
        if (on) {
          if (first) {
            store_f32<V>(ws.part + static_cast<long long>(c) * H + col, acc);
          } else {
            emit_row<V>(dw + static_cast<long long>(cur) * ldw + col, acc, scale, accumulate);
          }
        }
        first = false;
        cur = k;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.f;
      }
      if (on) {
        float f[V];
        x[u].get(f);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += f[j];
      }
    }
  }
  if (on) {
    if (first)
      store_f32<V>(ws.part + static_cast<long long>(c) * H + col, acc);
    else if (tail)
      store_f32<V>(ws.part + (chunks + c) * H + col, acc);
    else
      emit_row<V>(dw + static_cast<long long>(cur) * ldw + col, acc, scale, accumulate);
  }
  if (!head && !tail) return;
  __threadfence();
  __syncwarp();
  const int* counts = ws.count + static_cast<long long>(slab) * 3 * chunks;
  if (head)
    join_run<V>(ws, chunks, H, col, on, lane, counts, c, s0, e0, dw + static_cast<long long>(key0) * ldw + col, scale,
                accumulate);
  if (tail)
    join_run<V>(ws, chunks, H, col, on, lane, counts, c, s1, e1, dw + static_cast<long long>(key1) * ldw + col, scale,
                accumulate);
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
int slab_columns(int v) { return 32 * v; }

struct Plan {
  int v, slabs;
  long long chunks, counters;
  long long off_order, off_key, off_count, off_part, bytes;
};
Plan plan_bwd(long long n, long long vocab, int H, int v) {
  Plan p;
  p.v = v;
  p.slabs = (H + slab_columns(v) - 1) / slab_columns(v);
  p.chunks = (n + kChunk - 1) / kChunk;
  p.counters = 3 * p.chunks * p.slabs;
  p.off_order = align256((vocab + 1) * 4);
  p.off_key = p.off_order + align256(n * 4);
  p.off_count = p.off_key + align256(n * 4);
  p.off_part = p.off_count + align256(p.counters * 4);
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
  check_same_device(ids, w, "ids and w");
  check_same_device(w, out, "w and out");
  c10::cuda::CUDAGuard guard(w.device());
  const int H = static_cast<int>(w.size(1));
  const int top = 16 / static_cast<int>(std::max(w.element_size(), out.element_size()));
  int v = top;
  while (v > 1 && !(H % v == 0 && rows_allow(w, w.stride(0), vocab, v) && rows_allow(out, out.stride(0), n, v))) v /= 2;
  int log_l = 0;
  while (log_l < 5 && (1 << log_l) * v < H) ++log_l;
  const int per_slab = (kFwdUnroll << log_l) * v;
  const int slabs = (H + per_slab - 1) / per_slab;
  const long long threads = (n * slabs) << log_l;
  const long long blocks = (threads + kThreads - 1) / kThreads;
  REVPP_CHECK(blocks < (1LL << 31), "too many tokens");
  int* status = status_device_ptr();
  by_float(w.scalar_type(), [&](auto tw) {
    using TW = decltype(tw);
    by_float(out.scalar_type(), [&](auto to) {
      using TO = decltype(to);
      auto go = [&](auto ti, auto vc) {
        using TI = decltype(ti);
        constexpr int V = decltype(vc)::value;
        if constexpr (V * std::max(sizeof(TW), sizeof(TO)) <= 16)
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
  REVPP_CHECK(n < (1LL << 30) && vocab < (1LL << 30) && dw.size(1) < (1LL << 30), "too many tokens, rows or columns");
  if (vocab == 0 || dw.size(1) == 0 || (n == 0 && accumulate)) return;
  check_same_device(dy, dw, "dy and dw");
  check_same_device(ids, dw, "ids and dw");
  c10::cuda::CUDAGuard guard(dw.device());
  const int H = static_cast<int>(dw.size(1));
  int v = 16 / static_cast<int>(dy.element_size());
  // rows of the workspace are H floats: a vector of v floats in it needs H % v == 0 too
  while (v > 1 && !(H % v == 0 && rows_allow(dy, dy.stride(0), n, v) && rows_allow(dw, dw.stride(0), vocab, std::min(v, 4))))
    v /= 2;
  const Plan p = plan_bwd(n, vocab, H, v);
  torch::Tensor buf = torch::empty({p.bytes}, dw.options().dtype(at::kByte));
  char* base = static_cast<char*>(buf.data_ptr());
  EmbedWs ws{reinterpret_cast<int*>(base), reinterpret_cast<int*>(base + p.off_order),
             reinterpret_cast<int*>(base + p.off_key), reinterpret_cast<int*>(base + p.off_count),
             reinterpret_cast<float*>(base + p.off_part)};
  int* status = status_device_ptr();
  const int range = static_cast<int>(
      std::min<long long>(kSortRange, std::max<long long>(1, (vocab + num_sms() - 1) / num_sms())));
  const int ctas = static_cast<int>((vocab + range - 1) / range);
  const size_t smem = static_cast<size_t>(kSortWarps) * (range + 2 * kSortList) * 4;
  auto sort = [&](auto ti) {
    using TI = decltype(ti);
    REVPP_CUDA_CHECK(cudaFuncSetAttribute(embed_sort_kernel<TI>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          kSortWarps * (kSortRange + 2 * kSortList) * 4));
    launch_pdl(embed_sort_kernel<TI>, dim3(ctas), dim3(kSortWarps * 32), smem, cur_stream(),
               static_cast<const TI*>(ids.data_ptr()), static_cast<int>(n), static_cast<int>(vocab),
               static_cast<long long>(padding_idx), range, ws, p.counters, status);
  };
  if (ids.scalar_type() == at::kLong) sort(int64_t{});
  else sort(int32_t{});
  REVPP_CHECK_LAUNCH();
  const long long tasks = p.chunks * p.slabs + (accumulate ? 0 : (vocab + kZeroRows - 1) / kZeroRows);
  const long long blocks = (tasks + kThreads / 32 - 1) / (kThreads / 32);
  REVPP_CHECK(blocks < (1LL << 31), "too many tokens");
  by_float(dy.scalar_type(), [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vc) {
      constexpr int V = decltype(vc)::value;
      if constexpr (V * sizeof(T) <= 16)
        launch_pdl(embed_reduce_kernel<T, V>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, cur_stream(),
                   static_cast<const T*>(dy.data_ptr()), static_cast<long long>(dy.stride(0)), dw.data_ptr<float>(),
                   static_cast<long long>(dw.stride(0)), ws, p.chunks, p.slabs, static_cast<int>(vocab), H,
                   static_cast<float>(scale), accumulate ? 1 : 0);
    };
    if (v == 8) go(std::integral_constant<int, 8>{});
    else if (v == 4) go(std::integral_constant<int, 4>{});
    else if (v == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
  });
  REVPP_CHECK_LAUNCH();
}

}  // namespace revpp

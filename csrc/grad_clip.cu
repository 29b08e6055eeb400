// Global norm of many gradient tensors and clipping.
//
//   norm  = sqrt(sum_i sum g_i^2)          (norm_type 2),  or  max_i max |g_i|   (norm_type inf)
//   coef  = min(1, max_norm / (norm + 1e-6))
//   out_i = g_i * coef                     (out_i may be g_i itself)
//
// Two launches for any number of tensors up to the table's size: the first reads every gradient
// and leaves one partial per block, the second adds the partials (each block by itself, in a fixed
// order) and scales.  The table of tensors travels in the kernel's parameters, so a captured graph
// keeps it and nothing is copied to the device.  Squares are summed in 64 bits: gradients from 1e-30
// to 1e30 neither vanish nor overflow, and the result does not depend on how tensors are cut.
// A NaN makes the norm and every output NaN, an infinity makes finite outputs 0, as in the formula.
#include <algorithm>
#include <vector>

#include "common.cuh"
#include "host.h"
#include "vec.cuh"

namespace revpp {

namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 8;                              // 16-byte vectors per thread and chunk
constexpr int kChunkBytes = kThreads * kVecs * 16;    // of the gradient
constexpr int kBlocksPerSm = 4;

enum Type : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

struct Entry {
  const void* src;
  void* dst;
  long long n;
  int chunk0;          // first chunk
  unsigned char src_type, dst_type, wide, pad;  // wide: both addresses allow vectors
};

template <int CAP>
struct Table {
  int count, chunks;
  Entry e[CAP];
};

template <int CAP>
__device__ __forceinline__ int entry_of(const Table<CAP>& t, int chunk) {
  int lo = 0, hi = t.count;  // the last entry whose first chunk is not behind `chunk`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.e[mid].chunk0 <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Running value of one thread: a sum of squares, or the largest |g| as bits (a NaN's are above
// every number's, so it stays).
template <bool MAX>
struct Running {
  double sum = 0.0;
  unsigned bits = 0;
  __device__ __forceinline__ void add(float g) {
    if (MAX) {
      bits = max(bits, __float_as_uint(g) & 0x7fffffffu);
    } else {
      const double d = g;
      sum = fma(d, d, sum);
    }
  }
  __device__ __forceinline__ double value() const { return MAX ? static_cast<double>(__uint_as_float(bits)) : sum; }
  __device__ __forceinline__ static double join(double a, double b) {
    if (!MAX) return a + b;
    return (a > b || a != a) ? a : b;
  }
};

// Joins the block's values in a fixed order; every thread gets the result.
template <bool MAX>
__device__ __forceinline__ double block_join(double v, double* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Running<MAX>::join(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) s[warp] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = Running<MAX>::join(v, s[w]);
  return v;
}

template <typename T, bool MAX>
__device__ __forceinline__ void norm_chunk(const Entry& e, int chunk, Running<MAX>& run) {
  constexpr int V = 16 / sizeof(T);
  const T* p = static_cast<const T*>(e.src);
  const long long first = static_cast<long long>(chunk - e.chunk0) * (kChunkBytes / static_cast<int>(sizeof(T)));
  const long long left = e.n - first;
  const int m = static_cast<int>(min(left, static_cast<long long>(kChunkBytes / sizeof(T))));
  p += first;
  if (e.wide && m == kChunkBytes / static_cast<int>(sizeof(T))) {  // a whole chunk: all loads in flight
    const T* q = p + threadIdx.x * V;
    Pack<T, V> x[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) x[u] = Pack<T, V>::load_ro(q + u * kThreads * V);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      float f[V];
      x[u].get(f);
#pragma unroll
      for (int j = 0; j < V; ++j) run.add(f[j]);
    }
    return;
  }
  const int done = e.wide ? m / V * V : 0;
#pragma unroll 1
  for (int c = threadIdx.x * V; c < done; c += kThreads * V) {
    float f[V];
    Pack<T, V>::load_ro(p + c).get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) run.add(f[j]);
  }
#pragma unroll 1
  for (int c = done + threadIdx.x; c < m; c += kThreads) run.add(to_f32(p[c]));
}

template <int CAP, bool MAX>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    grad_norm_kernel(const __grid_constant__ Table<CAP> t, double* __restrict__ part) {
  __shared__ double s[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  Running<MAX> run;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const Entry& e = t.e[entry_of(t, c)];
    if (e.src_type == kF32) norm_chunk<float, MAX>(e, c, run);
    else if (e.src_type == kBf16) norm_chunk<__nv_bfloat16, MAX>(e, c, run);
    else norm_chunk<__half, MAX>(e, c, run);
  }
  const double v = block_join<MAX>(run.value(), s);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <typename T, typename O, int V>
__device__ __forceinline__ Pack<O, V> scaled(Pack<T, V> x, float coef) {
  float f[V];
  x.get(f);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] *= coef;
  Pack<O, V> y;
  y.set(f);
  return y;
}

template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const Entry& e, int chunk, float coef) {
  constexpr int V = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
  constexpr int N = kChunkBytes / sizeof(T) / kThreads / V;  // vectors per thread
  constexpr int B = N < 8 ? N : 8;
  const long long first = static_cast<long long>(chunk - e.chunk0) * (kChunkBytes / static_cast<int>(sizeof(T)));
  const long long left = e.n - first;
  const int m = static_cast<int>(min(left, static_cast<long long>(kChunkBytes / sizeof(T))));
  const T* p = static_cast<const T*>(e.src) + first;
  O* q = static_cast<O*>(e.dst) + first;
  if (e.wide && m == kChunkBytes / static_cast<int>(sizeof(T))) {
    const T* pp = p + threadIdx.x * V;
    O* qq = q + threadIdx.x * V;
#pragma unroll 1
    for (int u0 = 0; u0 < N; u0 += B) {
      Pack<T, V> x[B];
#pragma unroll
      for (int u = 0; u < B; ++u) x[u] = Pack<T, V>::load(pp + u * kThreads * V);
#pragma unroll
      for (int u = 0; u < B; ++u) scaled<T, O, V>(x[u], coef).store(qq + u * kThreads * V);
      pp += B * kThreads * V;
      qq += B * kThreads * V;
    }
    return;
  }
  const int done = e.wide ? m / V * V : 0;
#pragma unroll 1
  for (int c = threadIdx.x * V; c < done; c += kThreads * V)
    scaled<T, O, V>(Pack<T, V>::load(p + c), coef).store(q + c);
#pragma unroll 1
  for (int c = done + threadIdx.x; c < m; c += kThreads) q[c] = from_f32<O>(to_f32(p[c]) * coef);
}

template <typename T>
__device__ __forceinline__ void scale_to(const Entry& e, int chunk, float coef) {
  if (e.dst_type == kF32) scale_chunk<T, float>(e, chunk, coef);
  else if (e.dst_type == kBf16) scale_chunk<T, __nv_bfloat16>(e, chunk, coef);
  else scale_chunk<T, __half>(e, chunk, coef);
}

template <int CAP, bool MAX>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* __restrict__ part, int parts, double max_norm,
                      float* __restrict__ norm_out) {
  __shared__ double s[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) v = Running<MAX>::join(v, part[i]);
  v = block_join<MAX>(v, s);
  const double norm = MAX ? v : sqrt(v);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  const double ratio = max_norm / (norm + 1e-6);
  const float coef = ratio > 1.0 ? 1.f : static_cast<float>(ratio);  // a NaN stays
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const Entry& e = t.e[entry_of(t, c)];
    if (coef == 1.f && e.dst == e.src) continue;
    if (e.src_type == kF32) scale_to<float>(e, c, coef);
    else if (e.src_type == kBf16) scale_to<__nv_bfloat16>(e, c, coef);
    else scale_to<__half>(e, c, coef);
  }
}

// ------------------------------------------------------------------ host
int type_of(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBf16;
    case at::kHalf: return kF16;
    default: return -1;
  }
}

// Equal sizes and equal order in memory: element k of one is element k of the other.
bool same_layout(const torch::Tensor& a, const torch::Tensor& b) {
  if (!a.sizes().equals(b.sizes())) return false;
  if (a.is_contiguous() && b.is_contiguous()) return true;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

struct Range {
  uintptr_t lo, hi;
  int64_t index;
  bool written;
};

// No output may share memory with another output or with another tensor's gradient.
void check_overlaps(const std::vector<torch::Tensor>& grads, const std::vector<torch::Tensor>& outs) {
  std::vector<Range> r;
  r.reserve(grads.size() * 2);
  for (size_t i = 0; i < grads.size(); ++i) {
    if (grads[i].numel() == 0) continue;
    const uintptr_t g = reinterpret_cast<uintptr_t>(grads[i].data_ptr()), o = reinterpret_cast<uintptr_t>(outs[i].data_ptr());
    const bool same = g == o && grads[i].scalar_type() == outs[i].scalar_type();
    r.push_back({o, o + outs[i].nbytes(), static_cast<int64_t>(i), true});
    if (!same) r.push_back({g, g + grads[i].nbytes(), static_cast<int64_t>(i), false});
  }
  auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
  if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
  // the furthest end among all ranges so far, and among the written ones
  uintptr_t any = 0, written = 0;
  int64_t any_i = -1, written_i = -1;
  for (const Range& x : r) {
    const bool clash = x.written ? x.lo < any : x.lo < written;
    REVPP_CHECK(!clash, "out ", x.written ? x.index : written_i, " shares memory with the tensors at ",
                x.written ? any_i : x.index, ": outputs must be distinct, or their own gradients");
    if (x.hi > any) any = x.hi, any_i = x.index;
    if (x.written && x.hi > written) written = x.hi, written_i = x.index;
  }
}

template <int CAP, bool MAX>
void run_clip(const std::vector<Entry>& es, double max_norm, const torch::Tensor& norm, const torch::TensorOptions& opt) {
  // tables of at most CAP tensors, each with its own launch of either kernel
  const int wave = kBlocksPerSm * num_sms();
  std::vector<Table<CAP>> tables;
  std::vector<int> blocks;
  int parts = 0;
  for (size_t i = 0; i < es.size(); i += CAP) {
    tables.emplace_back();
    Table<CAP>& t = tables.back();
    t.count = static_cast<int>(std::min<size_t>(CAP, es.size() - i));
    long long chunks = 0;
    for (int k = 0; k < t.count; ++k) {
      t.e[k] = es[i + k];
      t.e[k].chunk0 = static_cast<int>(chunks);
      const long long bytes = es[i + k].n * (es[i + k].src_type == kF32 ? 4 : 2);
      chunks += (bytes + kChunkBytes - 1) / kChunkBytes;
    }
    REVPP_CHECK(chunks < (1LL << 31), "too many gradients");
    t.chunks = static_cast<int>(chunks);
    blocks.push_back(static_cast<int>(std::min<long long>(chunks, wave)));
    parts += blocks.back();
  }
  torch::Tensor part = torch::empty({std::max(parts, 1)}, opt.dtype(at::kDouble));
  double* pp = part.data_ptr<double>();
  int at_part = 0;
  for (size_t i = 0; i < tables.size(); ++i) {
    launch_pdl(grad_norm_kernel<CAP, MAX>, dim3(blocks[i]), dim3(kThreads), 0, cur_stream(), tables[i], pp + at_part);
    REVPP_CHECK_LAUNCH();
    at_part += blocks[i];
  }
  for (size_t i = 0; i < tables.size(); ++i) {
    launch_pdl(grad_scale_kernel<CAP, MAX>, dim3(blocks[i]), dim3(kThreads), 0, cur_stream(), tables[i],
               static_cast<const double*>(pp), parts, max_norm, i == 0 ? norm.data_ptr<float>() : static_cast<float*>(nullptr));
    REVPP_CHECK_LAUNCH();
  }
}

}  // namespace

torch::Tensor clip_grads(const std::vector<torch::Tensor>& grads, double max_norm,
                         const c10::optional<std::vector<torch::Tensor>>& out, bool max_type) {
  REVPP_CHECK(!grads.empty(), "grads must not be empty");
  REVPP_CHECK(max_norm >= 0.0, "max_norm must not be negative or NaN");
  const std::vector<torch::Tensor>& outs = out.has_value() ? *out : grads;
  REVPP_CHECK(outs.size() == grads.size(), "out must have one tensor per gradient: ", outs.size(), " for ", grads.size());
  std::vector<Entry> es;
  es.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const torch::Tensor &g = grads[i], &o = outs[i];
    const int gt = type_of(g), ot = type_of(o);
    REVPP_CHECK(gt >= 0 && ot >= 0, "tensor ", i, " must be float32, bfloat16 or float16");
    REVPP_CHECK(g.layout() == at::kStrided && o.layout() == at::kStrided, "tensor ", i, " must be dense");
    REVPP_CHECK(g.is_non_overlapping_and_dense(), "gradient ", i, " has gaps or repeats in memory: make it contiguous");
    REVPP_CHECK(same_layout(g, o), "out ", i, " must have its gradient's sizes and strides");
  }
  for (size_t i = 0; i < grads.size(); ++i) {
    const torch::Tensor &g = grads[i], &o = outs[i];
    REVPP_CHECK(g.is_cuda(), "gradient ", i, " must be a CUDA tensor");
    REVPP_CHECK(g.device() == grads[0].device() && o.device() == g.device(), "all tensors must be on one device");
    if (g.numel() == 0) continue;
    const int gt = type_of(g), ot = type_of(o);
    const bool wide = reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(o.data_ptr()) % 16 == 0;
    es.push_back({g.data_ptr(), o.data_ptr(), g.numel(), 0, static_cast<unsigned char>(gt), static_cast<unsigned char>(ot),
                  static_cast<unsigned char>(wide), 0});
  }
  check_overlaps(grads, outs);
  c10::cuda::CUDAGuard guard(grads[0].device());
  torch::Tensor norm = torch::empty({}, grads[0].options().dtype(at::kFloat));
  if (es.empty()) return norm.zero_();
  auto go = [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    if (max_type) run_clip<CAP, true>(es, max_norm, norm, grads[0].options());
    else run_clip<CAP, false>(es, max_norm, norm, grads[0].options());
  };
  if (es.size() <= 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 512>{});
  return norm;
}

}  // namespace revpp

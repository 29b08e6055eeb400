// Global norm of many gradient tensors and clipping.
//
//   norm  = sqrt(sum_i sum g_i^2)          (norm_type 2),  or  max_i max |g_i|   (norm_type inf)
//   coef  = min(1, max_norm / (norm + 1e-6))
//   out_i = g_i * coef                     (out_i may be g_i itself)
//
// Two launches for any number of tensors up to the table's size: the first reads every gradient
// and leaves one partial per block, the second adds the partials (each block by itself, in a fixed
// order) and scales, from the last chunk to the first: what was read last is still in L2.  The table of tensors travels in the kernel's parameters, so a captured graph
// keeps it and nothing is copied to the device.  Squares are summed in 64 bits: gradients from 1e-30
// to 1e30 neither vanish nor overflow, and the result does not depend on how tensors are cut.
// DRAM bounds both passes: 334 M fp32 gradients in 297 tensors (B200) take 217 us to read (6.2 TB/s)
// and 443 us to read and write (6.0 TB/s); small models take their launches.
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
  for (int c = t.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
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
  int index;
};

// No output may share memory with another output or with another tensor's gradient.
void check_overlaps(const std::vector<Entry>& es, const std::vector<int>& indexes) {
  auto size = [](int type) { return type == kF32 ? 4 : 2; };
  std::vector<Range> outs(es.size());
  uintptr_t grads_lo = ~uintptr_t(0), grads_hi = 0;  // of the gradients that are not their own outputs
  for (size_t i = 0; i < es.size(); ++i) {
    const uintptr_t o = reinterpret_cast<uintptr_t>(es[i].dst), g = reinterpret_cast<uintptr_t>(es[i].src);
    outs[i] = {o, o + es[i].n * size(es[i].dst_type), static_cast<int>(i)};
    if (o != g || es[i].dst_type != es[i].src_type) {
      grads_lo = std::min(grads_lo, g);
      grads_hi = std::max<uintptr_t>(grads_hi, g + es[i].n * size(es[i].src_type));
    }
  }
  auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
  if (!std::is_sorted(outs.begin(), outs.end(), before)) std::sort(outs.begin(), outs.end(), before);
  for (size_t i = 1; i < outs.size(); ++i)
    REVPP_CHECK(outs[i].lo >= outs[i - 1].hi, "out ", indexes[outs[i].index], " shares memory with out ",
                indexes[outs[i - 1].index], ": outputs must be distinct");
  if (grads_lo >= outs.back().hi || grads_hi <= outs.front().lo) return;
  for (size_t i = 0; i < es.size(); ++i) {
    const uintptr_t g = reinterpret_cast<uintptr_t>(es[i].src), end = g + es[i].n * size(es[i].src_type);
    // the last output that starts before the gradient's end
    auto it = std::lower_bound(outs.begin(), outs.end(), end, [](const Range& r, uintptr_t v) { return r.lo < v; });
    for (; it != outs.begin() && (it - 1)->hi > g; --it) {
      const Range& r = *(it - 1);
      const bool own = r.index == static_cast<int>(i) && r.lo == g && es[i].dst_type == es[i].src_type;
      REVPP_CHECK(own, "out ", indexes[r.index], " shares memory with gradient ", indexes[i],
                  ": an output must be its own gradient, or lie apart from all of them");
    }
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

// `grads` and `out` are Python lists (taken as they are: a list of hundreds of tensors is called once
// per training step, and converting it would cost more than the checks).
torch::Tensor clip_grads(const py::list& grads, double max_norm, const c10::optional<py::list>& out, bool max_type) {
  const Py_ssize_t n = PyList_GET_SIZE(grads.ptr());
  REVPP_CHECK(n > 0, "grads must not be empty");
  REVPP_CHECK(max_norm >= 0.0, "max_norm must not be negative or NaN");
  PyObject* outs = out.has_value() ? out->ptr() : grads.ptr();
  REVPP_CHECK(PyList_GET_SIZE(outs) == n, "out must have one tensor per gradient: ", PyList_GET_SIZE(outs), " for ", n);
  auto tensor = [](PyObject* list, Py_ssize_t i, const char* name) -> const torch::Tensor& {
    PyObject* o = PyList_GET_ITEM(list, i);
    REVPP_CHECK(THPVariable_Check(o), name, " ", i, " is not a tensor");
    return THPVariable_Unpack(o);
  };
  std::vector<Entry> es;
  std::vector<int> indexes;
  es.reserve(n);
  indexes.reserve(n);
  const torch::Tensor& front = tensor(grads.ptr(), 0, "gradient");
  const at::Device device = front.device();
  for (Py_ssize_t i = 0; i < n; ++i) {
    const torch::Tensor &g = tensor(grads.ptr(), i, "gradient"), &o = tensor(outs, i, "out");
    const int gt = type_of(g), ot = type_of(o);
    REVPP_CHECK(gt >= 0 && ot >= 0, "tensor ", i, " must be float32, bfloat16 or float16");
    REVPP_CHECK(g.layout() == at::kStrided && o.layout() == at::kStrided, "tensor ", i, " must be dense");
    REVPP_CHECK(g.is_contiguous() || g.is_non_overlapping_and_dense(), "gradient ", i,
                " has gaps or repeats in memory: make it contiguous");
    REVPP_CHECK(g.is_same(o) || same_layout(g, o), "out ", i, " must have its gradient's sizes and strides");
    REVPP_CHECK(g.is_cuda(), "gradient ", i, " must be a CUDA tensor");
    REVPP_CHECK(g.device() == device && o.device() == device, "all tensors must be on one device");
    const int64_t count = g.numel();
    if (count == 0) continue;
    const void* src = g.const_data_ptr();
    void* dst = o.data_ptr();
    const bool wide = (reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) % 16 == 0;
    es.push_back({src, dst, count, 0, static_cast<unsigned char>(gt), static_cast<unsigned char>(ot),
                  static_cast<unsigned char>(wide), 0});
    indexes.push_back(static_cast<int>(i));
  }
  c10::cuda::CUDAGuard guard(front.device());
  torch::Tensor norm = torch::empty({}, front.options().dtype(at::kFloat));
  if (es.empty()) return norm.zero_();
  check_overlaps(es, indexes);
  auto go = [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    if (max_type) run_clip<CAP, true>(es, max_norm, norm, front.options());
    else run_clip<CAP, false>(es, max_norm, norm, front.options());
  };
  if (es.size() <= 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 512>{});
  return norm;
}

}  // namespace revpp

// Per-head RMS norm of queries and keys with the position rotation in the same pass, over the
// packed [rows, (heads + 2 kv_heads) * d] projection that the attention kernels read.
//
//   fwd : r = 1 / sqrt(mean(x^2) + eps),  z = x r w,  y = R(p) z
//         R(p) turns the pairs (i, i + rot/2), or (2i, 2i+1) when interleaved, of the first rot
//         columns by the angle whose cosine and sine stand in row p of the tables
//   bwd : dz = R(p)^T dy,  dw (+)= sum dz x r,  g = dz w,  dx = r (g - x r mean(g x r))
//
// Value heads are copied when the output is another buffer and left alone when it is the input
// itself.  Statistics, rotation and sums are fp32; the result is rounded once.  A position outside
// the tables sets kStatusBadShape and leaves the row unrotated.
//
// A head belongs to G lanes (a power of two).  Each lane owns "units" of two vectors of V
// elements: in the rotated part the two vectors that hold the two members of V pairs, so that the
// rotation needs no exchange between lanes, and behind it two neighbouring vectors.  A lane keeps
// its head and walks over the rows: norm weights and, in the backward pass, their gradients stay
// in registers.
#include <algorithm>

#include "common.cuh"
#include "host.h"
#include "vec.cuh"

namespace revpp {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

struct QkArgs {
  long long ldx, ldy, lddx;  // row strides (elements)
  const float* wq;
  const float* wk;
  const float* cos;
  const float* sin;
  long long ldt;             // row stride of the tables
  const void* pos;           // positions, or null: row % seq
  int pos64;
  int seq;
  int table_rows;
  int rows, heads, kv_heads, all_heads, dim, rot;
  int units, log_g;          // units per head, lanes per head
  float eps, inv_dim;
  int* status;
};

// Columns of the two vectors of unit u (b < 0: none), whether they rotate, and the first pair.
template <int V, bool NEIGHBOURS>
__device__ __forceinline__ void unit_at(int u, int dim, int rot, int& a, int& b, bool& turn, int& pair) {
  const int half = rot >> 1;
  if (NEIGHBOURS && V > 1) {  // pairs inside a vector: vectors 2u and 2u + 1
    a = 2 * u * V;
    b = a + V;
    pair = a >> 1;
    turn = a < rot;
    if (b >= dim) b = -1;
    return;
  }
  const int turning = half / V;
  turn = u < turning;
  if (turn) {
    pair = u * V;
    a = NEIGHBOURS ? 2 * u : u * V;
    b = NEIGHBOURS ? 2 * u + 1 : half + u * V;
  } else {
    pair = 0;
    a = rot + 2 * (u - turning) * V;
    b = a + V;
    if (b >= dim) b = -1;
  }
}

__device__ __forceinline__ long long position_of(const QkArgs& a, int row) {
  if (a.pos == nullptr) return static_cast<unsigned>(row) % static_cast<unsigned>(a.seq);
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[row] : static_cast<const int32_t*>(a.pos)[row];
}

// Rotates the unit (xa, xb) by +angle (SIGN 1) or -angle (SIGN -1).
template <int V, bool NEIGHBOURS, int SIGN>
__device__ __forceinline__ void rotate(float (&xa)[V], float (&xb)[V], const float* __restrict__ cos,
                                       const float* __restrict__ sin, int pair, int b, int rot) {
  if constexpr (NEIGHBOURS && V > 1) {
    constexpr int P = V / 2;
    float c[P], s[P];
    load_f32<P>(cos + pair, c);
    load_f32<P>(sin + pair, s);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float p = xa[2 * j], q = xa[2 * j + 1], n = SIGN * s[j];
      xa[2 * j] = p * c[j] - q * n;
      xa[2 * j + 1] = p * n + q * c[j];
    }
    if (b >= 0 && b < rot) {
      load_f32<P>(cos + pair + P, c);
      load_f32<P>(sin + pair + P, s);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float p = xb[2 * j], q = xb[2 * j + 1], n = SIGN * s[j];
        xb[2 * j] = p * c[j] - q * n;
        xb[2 * j + 1] = p * n + q * c[j];
      }
    }
  } else {
    float c[V], s[V];
    load_f32<V>(cos + pair, c);
    load_f32<V>(sin + pair, s);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float p = xa[j], q = xb[j], n = SIGN * s[j];
      xa[j] = p * c[j] - q * n;
      xb[j] = p * n + q * c[j];
    }
  }
}

// The lane's place: its head, first row and row stride (rows advance by whole sets of heads).
struct Place {
  int head, row, stride, lane;
};
__device__ __forceinline__ Place place_of(const QkArgs& a) {
  const unsigned slot = (blockIdx.x * kThreads + threadIdx.x) >> a.log_g;
  const unsigned slots = (gridDim.x * kThreads) >> a.log_g;
  const unsigned stride = slots / a.all_heads;
  Place p;
  p.row = slot / a.all_heads;
  p.head = slot - p.row * a.all_heads;
  p.stride = stride;
  if (p.row >= static_cast<int>(stride)) p.row = a.rows;  // a remainder that makes no whole set
  p.lane = threadIdx.x & ((1 << a.log_g) - 1);
  return p;
}

__device__ __forceinline__ float group_sum(float v, int log_g) {
  for (int o = (1 << log_g) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int V, int U, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads)
    qk_norm_rope_fwd_kernel(const T* x, T* y, QkArgs a) {
  pdl_wait();
  pdl_trigger();
  const Place p = place_of(a);
  const int G = 1 << a.log_g;
  const bool norm = p.head < a.heads + a.kv_heads;
  const float* w = p.head < a.heads ? a.wq : a.wk;
  int ca[U], cb[U], pair[U];
  bool turn[U];
  float wa[U][V], wb[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int unit = p.lane + u * G;
    unit_at<V, NEIGHBOURS>(unit, a.dim, a.rot, ca[u], cb[u], turn[u], pair[u]);
    if (unit >= a.units) ca[u] = cb[u] = -1;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wa[u][j] = norm && w != nullptr && ca[u] >= 0 ? __ldg(w + ca[u] + j) : 1.f;
      wb[u][j] = norm && w != nullptr && cb[u] >= 0 ? __ldg(w + cb[u] + j) : 1.f;
    }
  }
  const int trips = (a.rows + p.stride - 1) / p.stride;
  for (int t = 0; t < trips; ++t) {
    const int row = p.row + t * p.stride;
    const bool on = row < a.rows;
    const T* xr = x + static_cast<long long>(row) * a.ldx + p.head * a.dim;
    T* yr = y + static_cast<long long>(row) * a.ldy + p.head * a.dim;
    Pack<T, V> ra[U], rb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (on && ca[u] >= 0) ra[u] = Pack<T, V>::load(xr + ca[u]);
      if (on && cb[u] >= 0) rb[u] = Pack<T, V>::load(xr + cb[u]);
    }
    long long pos = -1;
    if (on && norm && a.rot > 0) {
      pos = position_of(a, row);
      if (pos < 0 || pos >= a.table_rows) {
        atomicOr(a.status, kStatusBadShape);
        pos = -1;
      }
    }
    float fa[U][V], fb[U][V], ss = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (on && ca[u] >= 0) {
        ra[u].get(fa[u]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) fa[u][j] = 0.f;
      }
      if (on && cb[u] >= 0) {
        rb[u].get(fb[u]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) fb[u][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ss += fa[u][j] * fa[u][j] + fb[u][j] * fb[u][j];
    }
    const float r = rsqrtf(group_sum(ss, a.log_g) * a.inv_dim + a.eps);
    if (!on) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ca[u] < 0) continue;
      if (norm) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          fa[u][j] *= r * wa[u][j];
          fb[u][j] *= r * wb[u][j];
        }
        if (turn[u] && pos >= 0)
          rotate<V, NEIGHBOURS, 1>(fa[u], fb[u], a.cos + pos * a.ldt, a.sin + pos * a.ldt, pair[u], cb[u], a.rot);
        ra[u].set(fa[u]);
        rb[u].set(fb[u]);
      }
      ra[u].store(yr + ca[u]);
      if (cb[u] >= 0) rb[u].store(yr + cb[u]);
    }
  }
}

// part: [gridDim.x][2][dim] sums of dz x r over the block's query heads and key heads, added up
// by qk_weight_grad_kernel in block order.
template <typename T, int V, int U, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads)
    qk_norm_rope_bwd_kernel(const T* dy, const T* __restrict__ x, T* dx, QkArgs a, float* __restrict__ part) {
  extern __shared__ float sums[];  // [kThreads / G][dim]
  pdl_wait();
  pdl_trigger();
  const Place p = place_of(a);
  const int G = 1 << a.log_g;
  const bool norm = p.head < a.heads + a.kv_heads;
  const float* w = p.head < a.heads ? a.wq : a.wk;
  int ca[U], cb[U], pair[U];
  bool turn[U];
  float wa[U][V], wb[U][V], da[U][V], db[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int unit = p.lane + u * G;
    unit_at<V, NEIGHBOURS>(unit, a.dim, a.rot, ca[u], cb[u], turn[u], pair[u]);
    if (unit >= a.units) ca[u] = cb[u] = -1;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wa[u][j] = norm && w != nullptr && ca[u] >= 0 ? __ldg(w + ca[u] + j) : 1.f;
      wb[u][j] = norm && w != nullptr && cb[u] >= 0 ? __ldg(w + cb[u] + j) : 1.f;
      da[u][j] = db[u][j] = 0.f;
    }
  }
  const int trips = (a.rows + p.stride - 1) / p.stride;
  for (int t = 0; t < trips; ++t) {
    const int row = p.row + t * p.stride;
    const bool on = row < a.rows;
    const bool work = on && norm;
    const T* xr = x + static_cast<long long>(row) * a.ldx + p.head * a.dim;
    const T* gr = dy + static_cast<long long>(row) * a.ldy + p.head * a.dim;
    T* dr = dx + static_cast<long long>(row) * a.lddx + p.head * a.dim;
    Pack<T, V> ra[U], rb[U], ga[U], gb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (on && ca[u] >= 0) ga[u] = Pack<T, V>::load(gr + ca[u]);
      if (on && cb[u] >= 0) gb[u] = Pack<T, V>::load(gr + cb[u]);
      if (work && ca[u] >= 0) ra[u] = Pack<T, V>::load(xr + ca[u]);
      if (work && cb[u] >= 0) rb[u] = Pack<T, V>::load(xr + cb[u]);
    }
    long long pos = -1;
    if (work && a.rot > 0) {
      pos = position_of(a, row);
      if (pos < 0 || pos >= a.table_rows) {
        atomicOr(a.status, kStatusBadShape);
        pos = -1;
      }
    }
    float xa[U][V], xb[U][V], za[U][V], zb[U][V], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) xa[u][j] = xb[u][j] = za[u][j] = zb[u][j] = 0.f;
      if (work && ca[u] >= 0) {
        ra[u].get(xa[u]);
        ga[u].get(za[u]);
      }
      if (work && cb[u] >= 0) {
        rb[u].get(xb[u]);
        gb[u].get(zb[u]);
      }
      if (turn[u] && pos >= 0 && ca[u] >= 0)
        rotate<V, NEIGHBOURS, -1>(za[u], zb[u], a.cos + pos * a.ldt, a.sin + pos * a.ldt, pair[u], cb[u], a.rot);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss += xa[u][j] * xa[u][j] + xb[u][j] * xb[u][j];
        dot += za[u][j] * wa[u][j] * xa[u][j] + zb[u][j] * wb[u][j] * xb[u][j];
      }
    }
    const float r = rsqrtf(group_sum(ss, a.log_g) * a.inv_dim + a.eps);
    dot = group_sum(dot, a.log_g) * a.inv_dim * r * r;  // mean(g x r) r
    if (!on) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ca[u] < 0) continue;
      if (norm) {
        float oa[V], ob[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          da[u][j] += za[u][j] * (xa[u][j] * r);
          db[u][j] += zb[u][j] * (xb[u][j] * r);
          oa[j] = r * (za[u][j] * wa[u][j] - xa[u][j] * dot);
          ob[j] = r * (zb[u][j] * wb[u][j] - xb[u][j] * dot);
        }
        ga[u].set(oa);
        gb[u].set(ob);
      }
      ga[u].store(dr + ca[u]);
      if (cb[u] >= 0) gb[u].store(dr + cb[u]);
    }
  }
  if (part == nullptr) return;
  const int groups = kThreads >> a.log_g;
  float* mine = sums + (threadIdx.x >> a.log_g) * a.dim;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (ca[u] >= 0) mine[ca[u] + j] = da[u][j];
      if (cb[u] >= 0) mine[cb[u] + j] = db[u][j];
    }
  __syncthreads();
  const unsigned slot0 = (blockIdx.x * kThreads) >> a.log_g;
  for (int c = threadIdx.x; c < 2 * a.dim; c += kThreads) {
    const bool keys = c >= a.dim;
    const int col = keys ? c - a.dim : c;
    float s = 0.f;
    for (int g = 0; g < groups; ++g) {
      const int head = (slot0 + g) % a.all_heads;
      const bool use = keys ? head >= a.heads && head < a.heads + a.kv_heads : head < a.heads;
      if (use) s += sums[g * a.dim + col];
    }
    part[static_cast<long long>(blockIdx.x) * 2 * a.dim + c] = s;
  }
}

// dw (+)= sums of part over the blocks, in a fixed order: 32 columns per block, 32 slices.
__global__ void __launch_bounds__(1024)
    qk_weight_grad_kernel(const float* __restrict__ part, int blocks, int dim, float* __restrict__ dwq,
                          float* __restrict__ dwk, int accumulate) {
  __shared__ float s[32][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < 2 * dim)
    for (int b = slice; b < blocks; b += 32) v += part[static_cast<long long>(b) * 2 * dim + c];
  s[slice][lane] = v;
  __syncthreads();
  if (slice != 0 || c >= 2 * dim) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) v += s[i][lane];
  float* d = c < dim ? dwq : dwk;
  if (d == nullptr) return;
  const int col = c < dim ? c : c - dim;
  d[col] = accumulate ? d[col] + v : v;
}

// ------------------------------------------------------------------ host
using OptTensor = c10::optional<torch::Tensor>;
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

struct Span {
  uintptr_t lo, hi;
};
Span span_of(const torch::Tensor& t) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(t.data_ptr());
  const long long last = (t.size(0) - 1) * t.stride(0) + t.size(1);
  return {lo, lo + static_cast<uintptr_t>(last * t.element_size())};
}
// `out` may be `in` itself (same start, same row stride), or lie apart from it.
void check_in_place(const torch::Tensor& in, const torch::Tensor& out, const char* names) {
  if (in.data_ptr() == out.data_ptr() && in.stride(0) == out.stride(0)) return;
  const Span a = span_of(in), b = span_of(out);
  REVPP_CHECK(a.hi <= b.lo || b.hi <= a.lo, names, " must be the same tensor or not overlap");
}

void check_packed(const torch::Tensor& t, const char* name, int64_t rows, int64_t width, at::ScalarType type,
                  bool written) {
  REVPP_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == width, name, " must be [", rows, ", ", width, "]");
  REVPP_CHECK(t.scalar_type() == type, name, " must have qkv's type");
  REVPP_CHECK(t.stride(1) == 1 || width == 1, name, " must be contiguous along its last dimension");
  if (written) REVPP_CHECK(rows <= 1 || t.stride(0) >= width, name, " has rows that overlap");
}

struct Problem {
  QkArgs a;
  int v;
};

// Checks that need no device, then fills in the arguments.
Problem make_problem(const torch::Tensor& qkv, int64_t heads, int64_t kv_heads, const OptTensor& wq, const OptTensor& wk,
                     double eps, const OptTensor& cos, const OptTensor& sin, const OptTensor& positions,
                     const c10::optional<int64_t>& seq, bool interleaved) {
  REVPP_CHECK(qkv.dim() == 2, "qkv must be [rows, (heads + 2 kv_heads) * dim]");
  const at::ScalarType type = qkv.scalar_type();
  REVPP_CHECK(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf,
              "qkv must be float32, bfloat16 or float16");
  REVPP_CHECK(heads >= 1 && kv_heads >= 1 && heads <= 4096 && kv_heads <= 4096, "heads and kv_heads must be 1 to 4096");
  const int64_t all = heads + 2 * kv_heads;
  REVPP_CHECK(qkv.size(1) % all == 0, "the width ", qkv.size(1), " is not a multiple of heads + 2 kv_heads = ", all);
  const int64_t dim = qkv.size(1) / all, rows = qkv.size(0);
  REVPP_CHECK(dim >= 1 && dim <= kMaxDim, "the head dimension must be 1 to ", kMaxDim, ", got ", dim);
  REVPP_CHECK(rows < (1LL << 30), "too many rows");
  REVPP_CHECK(eps >= 0.0, "eps must not be negative");
  check_packed(qkv, "qkv", rows, qkv.size(1), type, false);
  for (const auto* w : {&wq, &wk})
    if (given(*w))
      REVPP_CHECK((*w)->scalar_type() == at::kFloat && (*w)->dim() == 1 && (*w)->size(0) == dim && (*w)->is_contiguous(),
                  "wq and wk must be contiguous float32 [", dim, "]");
  REVPP_CHECK(given(cos) == given(sin), "cos and sin go together");
  Problem p{};
  QkArgs& a = p.a;
  if (given(cos)) {
    for (const auto* t : {&cos, &sin})
      REVPP_CHECK((*t)->scalar_type() == at::kFloat && (*t)->dim() == 2 && (*t)->size(1) == cos->size(1) &&
                      (*t)->size(0) == cos->size(0) && (*t)->stride(0) == cos->stride(0) &&
                      ((*t)->size(1) <= 1 || (*t)->stride(1) == 1),
                  "cos and sin must be float32 [positions, rot / 2] of one shape and layout, contiguous along the last "
                  "dimension");
    a.rot = static_cast<int>(2 * cos->size(1));
    REVPP_CHECK(a.rot >= 2 && a.rot <= dim, "cos and sin have ", cos->size(1), " columns: a head of ", dim,
                " has room for 1 to ", dim / 2);
    REVPP_CHECK(cos->size(0) >= 1 && cos->size(0) < (1LL << 30), "cos and sin must have 1 to 2^30 rows");
    REVPP_CHECK(given(positions) != (seq.has_value()), "give positions or S, and not both");
    if (given(positions)) {
      REVPP_CHECK(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt,
                  "positions must be int64 or int32");
      REVPP_CHECK(positions->numel() == rows && positions->is_contiguous(), "positions must be contiguous, one per row");
    } else {
      REVPP_CHECK(*seq >= 1 && *seq <= cos->size(0), "S must be 1 to the tables' ", cos->size(0), " rows, got ", *seq);
    }
  }
  a.rows = static_cast<int>(rows);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.dim = static_cast<int>(dim);
  a.eps = static_cast<float>(eps);
  a.inv_dim = 1.f / static_cast<float>(dim);
  a.ldx = qkv.stride(0);
  return p;
}

void check_devices(const torch::Tensor& qkv, std::initializer_list<const torch::Tensor*> ts) {
  REVPP_CHECK(qkv.is_cuda(), "qkv must be a CUDA tensor");
  for (const auto* t : ts)
    if (t != nullptr && t->defined()) REVPP_CHECK(t->device() == qkv.device(), "all tensors must be on qkv's device");
}
const torch::Tensor* ptr_of(const OptTensor& t) { return given(t) ? &*t : nullptr; }

// Pointers, and the widest vector that columns, strides and addresses allow.
void finish(Problem& p, std::initializer_list<const torch::Tensor*> packed, const OptTensor& wq, const OptTensor& wk,
            const OptTensor& cos, const OptTensor& sin, const OptTensor& positions, const c10::optional<int64_t>& seq,
            bool interleaved) {
  QkArgs& a = p.a;
  const int size = static_cast<int>((*packed.begin())->element_size());
  auto allowed = [&](int v) {
    if (v == 1) return true;
    if (a.dim % v != 0) return false;
    for (const auto* t : packed)
      if (reinterpret_cast<uintptr_t>(t->data_ptr()) % (v * size) != 0 || (t->size(0) > 1 && t->stride(0) % v != 0))
        return false;
    if (a.rot == 0) return true;
    if (interleaved ? a.rot % v != 0 : (a.rot / 2) % v != 0) return false;
    const int c = std::min(4, interleaved ? v / 2 : v);  // floats per table access
    return reinterpret_cast<uintptr_t>(cos->data_ptr()) % (4 * c) == 0 &&
           reinterpret_cast<uintptr_t>(sin->data_ptr()) % (4 * c) == 0 && (cos->size(0) <= 1 || cos->stride(0) % c == 0);
  };
  p.v = 16 / size;
  while (!allowed(p.v)) p.v /= 2;
  const int v = p.v, half = a.rot / 2;
  if (interleaved && v > 1)
    a.units = (a.dim / v + 1) / 2;
  else
    a.units = half / v + ((a.dim - a.rot) / v + 1) / 2;
  while (a.log_g < 5 && (1 << a.log_g) < a.units) ++a.log_g;
  a.wq = given(wq) ? wq->data_ptr<float>() : nullptr;
  a.wk = given(wk) ? wk->data_ptr<float>() : nullptr;
  if (a.rot > 0) {
    a.cos = cos->data_ptr<float>();
    a.sin = sin->data_ptr<float>();
    a.ldt = cos->stride(0);
    a.table_rows = static_cast<int>(cos->size(0));
    if (given(positions)) {
      a.pos = positions->data_ptr();
      a.pos64 = positions->scalar_type() == at::kLong;
    } else {
      a.seq = static_cast<int>(*seq);
    }
  }
  a.status = status_device_ptr();
}

// Blocks for one resident wave, or fewer when the rows need fewer.
template <typename K>
int blocks_for(K kernel, const QkArgs& a, size_t smem) {
  int per_sm = 0;
  REVPP_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, smem));
  const long long need = ((static_cast<long long>(a.rows) * a.all_heads << a.log_g) + kThreads - 1) / kThreads;
  const long long least = ((static_cast<long long>(a.all_heads) << a.log_g) + kThreads - 1) / kThreads;
  const long long wave = static_cast<long long>(std::max(1, per_sm)) * num_sms();
  return static_cast<int>(std::max(least, std::min(need, wave)));
}

template <typename F>
void by_type(const Problem& p, at::ScalarType t, bool interleaved, F&& f) {
  auto by_v = [&](auto e, auto nb) {
    using T = decltype(e);
    if constexpr (sizeof(T) == 2) {
      if (p.v == 8) return f(e, std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{}, nb);
    }
    if (p.v == 4) f(e, std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{}, nb);
    else if (p.v == 2) f(e, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{}, nb);
    else f(e, std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{}, nb);
  };
  auto by_pairs = [&](auto e) {
    if (interleaved) by_v(e, std::true_type{});
    else by_v(e, std::false_type{});
  };
  if (t == at::kFloat) by_pairs(float{});
  else if (t == at::kBFloat16) by_pairs(__nv_bfloat16{});
  else by_pairs(__half{});
}

}  // namespace

void qk_norm_rope_fwd(const torch::Tensor& qkv, torch::Tensor out, int64_t heads, int64_t kv_heads, const OptTensor& wq,
                      const OptTensor& wk, double eps, const OptTensor& cos, const OptTensor& sin,
                      const OptTensor& positions, const c10::optional<int64_t>& S, bool interleaved) {
  Problem p = make_problem(qkv, heads, kv_heads, wq, wk, eps, cos, sin, positions, S, interleaved);
  check_packed(out, "out", qkv.size(0), qkv.size(1), qkv.scalar_type(), true);
  if (p.a.rows == 0) return;
  check_in_place(qkv, out, "qkv and out");
  check_devices(qkv, {&out, ptr_of(wq), ptr_of(wk), ptr_of(cos), ptr_of(sin), ptr_of(positions)});
  c10::cuda::CUDAGuard guard(qkv.device());
  finish(p, {&qkv, &out}, wq, wk, cos, sin, positions, S, interleaved);
  QkArgs& a = p.a;
  a.ldy = out.stride(0);
  a.all_heads = a.heads + a.kv_heads * (qkv.data_ptr() == out.data_ptr() ? 1 : 2);
  by_type(p, qkv.scalar_type(), interleaved, [&](auto e, auto v, auto u, auto nb) {
    using T = decltype(e);
    auto kernel = qk_norm_rope_fwd_kernel<T, decltype(v)::value, decltype(u)::value, decltype(nb)::value>;
    launch_pdl(kernel, dim3(blocks_for(kernel, a, 0)), dim3(kThreads), 0, cur_stream(),
               static_cast<const T*>(qkv.data_ptr()), static_cast<T*>(out.data_ptr()), a);
  });
  REVPP_CHECK_LAUNCH();
}

void qk_norm_rope_bwd(const torch::Tensor& dout, const torch::Tensor& qkv, torch::Tensor dqkv, int64_t heads,
                      int64_t kv_heads, const OptTensor& wq, const OptTensor& wk, const OptTensor& dwq,
                      const OptTensor& dwk, double eps, const OptTensor& cos, const OptTensor& sin,
                      const OptTensor& positions, const c10::optional<int64_t>& S, bool interleaved, bool accumulate) {
  Problem p = make_problem(qkv, heads, kv_heads, wq, wk, eps, cos, sin, positions, S, interleaved);
  QkArgs& a = p.a;
  check_packed(dout, "dout", qkv.size(0), qkv.size(1), qkv.scalar_type(), false);
  check_packed(dqkv, "dqkv", qkv.size(0), qkv.size(1), qkv.scalar_type(), true);
  for (const auto* d : {&dwq, &dwk})
    if (given(*d))
      REVPP_CHECK((*d)->scalar_type() == at::kFloat && (*d)->dim() == 1 && (*d)->size(0) == a.dim && (*d)->is_contiguous(),
                  "dwq and dwk must be contiguous float32 [", a.dim, "]");
  if (given(dwq) && given(dwk)) {
    const float *dq = dwq->data_ptr<float>(), *dk = dwk->data_ptr<float>();
    REVPP_CHECK(dq + a.dim <= dk || dk + a.dim <= dq, "dwq and dwk must not overlap");
  }
  const bool weights = given(dwq) || given(dwk);
  if (a.rows == 0 && (accumulate || !weights)) return;
  if (a.rows > 0) {
    check_in_place(dout, dqkv, "dout and dqkv");
    const Span s = span_of(qkv), d = span_of(dqkv);
    REVPP_CHECK(s.hi <= d.lo || d.hi <= s.lo, "dqkv must not overlap qkv");
  }
  check_devices(qkv, {&dout, &dqkv, ptr_of(wq), ptr_of(wk), ptr_of(dwq), ptr_of(dwk), ptr_of(cos), ptr_of(sin),
                      ptr_of(positions)});
  c10::cuda::CUDAGuard guard(qkv.device());
  int blocks = 0;
  torch::Tensor part;
  if (a.rows > 0) {
    finish(p, {&qkv, &dout, &dqkv}, wq, wk, cos, sin, positions, S, interleaved);
    a.ldy = dout.stride(0);
    a.lddx = dqkv.stride(0);
    a.all_heads = a.heads + a.kv_heads * (dout.data_ptr() == dqkv.data_ptr() ? 1 : 2);
    const size_t smem = weights ? static_cast<size_t>(kThreads >> a.log_g) * a.dim * 4 : 0;
    by_type(p, qkv.scalar_type(), interleaved, [&](auto e, auto v, auto u, auto nb) {
      using T = decltype(e);
      auto kernel = qk_norm_rope_bwd_kernel<T, decltype(v)::value, decltype(u)::value, decltype(nb)::value>;
      blocks = blocks_for(kernel, a, smem);
      if (weights) part = torch::empty({static_cast<int64_t>(blocks) * 2 * a.dim}, qkv.options().dtype(at::kFloat));
      launch_pdl(kernel, dim3(blocks), dim3(kThreads), smem, cur_stream(), static_cast<const T*>(dout.data_ptr()),
                 static_cast<const T*>(qkv.data_ptr()), static_cast<T*>(dqkv.data_ptr()), a,
                 weights ? part.data_ptr<float>() : static_cast<float*>(nullptr));
    });
    REVPP_CHECK_LAUNCH();
  }
  if (!weights) return;
  launch_pdl(qk_weight_grad_kernel, dim3((2 * a.dim + 31) / 32), dim3(1024), 0, cur_stream(),
             blocks > 0 ? const_cast<const float*>(part.data_ptr<float>()) : static_cast<const float*>(nullptr), blocks, a.dim,
             given(dwq) ? dwq->data_ptr<float>() : static_cast<float*>(nullptr),
             given(dwk) ? dwk->data_ptr<float>() : static_cast<float*>(nullptr), accumulate ? 1 : 0);
  REVPP_CHECK_LAUNCH();
}

}  // namespace revpp

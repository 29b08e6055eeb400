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
// A head belongs to G lanes.  Each lane owns U "units" of two vectors of V elements: in the
// rotated part the two vectors that hold the two members of V pairs, so that the rotation needs no
// exchange between lanes, and behind it two neighbouring vectors.  A lane keeps its head or heads and
// walks over the rows: norm weights and, in the backward pass, their gradients stay in registers.
// Arithmetic runs on packed fp32 pairs.  What bounds both passes is the number of bytes in flight:
//  - fwd: a lane takes H heads of one kind (queries, keys or values) of a row, all loaded at once,
//    with one set of angles;
//  - bwd: one head, its vectors copied into shared memory two rows ahead (cp.async, every lane its
//    own, so no barrier), since the registers are taken by weights and their gradients.
// Value heads have no arithmetic; as lanes of their own they would be through early and leave warps
// idle, so all lanes copy them at the end.  32768 rows of 16 heads x 64 bf16 (B200, out of place): fwd
// 67 us, 403 MB at 0.91 of the copy rate (one head at a time with the next row prefetched 83 us); bwd
// 103 us, 537 MB at 0.79 (two heads at once 128 us: registers for 12 warps per SM only; value heads as
// lanes of their own 120 us).
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host.h"
#include "vec.cuh"

namespace revpp {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kFwdHeads = 4;                  // heads that a lane of the forward pass has in flight

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
  int rows, heads, kv_heads, dim, rot;
  int q_sets, sets;          // sets of heads that a lane takes together: of queries, and of keys behind them
  int copies;                // the value heads go to another buffer
  int units, group, groups;  // units per head, lanes per head, heads per warp
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

// Packed arithmetic on neighbouring elements of arrays (V = 1: plain).
template <int V>
__device__ __forceinline__ void mul(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      f32x2_split(mul_f32x2(f32x2(a[j], a[j + 1]), f32x2(b[j], b[j + 1])), d[j], d[j + 1]);
  } else {
    d[0] = a[0] * b[0];
  }
}
template <int V>
__device__ __forceinline__ void scale(float (&d)[V], float s) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2) f32x2_split(mul_f32x2(f32x2(d[j], d[j + 1]), f32x2_splat(s)), d[j], d[j + 1]);
  } else {
    d[0] *= s;
  }
}
// d = a b + c
template <int V>
__device__ __forceinline__ void mad(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      f32x2_split(fma_f32x2(f32x2(a[j], a[j + 1]), f32x2(b[j], b[j + 1]), f32x2(c[j], c[j + 1])), d[j], d[j + 1]);
  } else {
    d[0] = fmaf(a[0], b[0], c[0]);
  }
}
// d = a s + c
template <int V>
__device__ __forceinline__ void mad(float (&d)[V], const float (&a)[V], float s, const float (&c)[V]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      f32x2_split(fma_f32x2(f32x2(a[j], a[j + 1]), f32x2_splat(s), f32x2(c[j], c[j + 1])), d[j], d[j + 1]);
  } else {
    d[0] = fmaf(a[0], s, c[0]);
  }
}
// sum += a b, in two running halves
template <int V>
__device__ __forceinline__ void dot(float (&sum)[2], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      f32x2_split(fma_f32x2(f32x2(a[j], a[j + 1]), f32x2(b[j], b[j + 1]), f32x2(sum[0], sum[1])), sum[0], sum[1]);
  } else {
    sum[0] = fmaf(a[0], b[0], sum[0]);
  }
}
template <int V>
__device__ __forceinline__ void zero(float (&d)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) d[j] = 0.f;
}

// Cosines and sines of a unit's pairs: V of each, for the pairs inside its two vectors V / 2 and V / 2.
template <int V, bool NEIGHBOURS>
__device__ __forceinline__ void load_angles(const float* __restrict__ cos, const float* __restrict__ sin, int pair, bool second,
                                            float (&c)[V], float (&s)[V]) {
  if constexpr (NEIGHBOURS && V > 1) {
    constexpr int P = V / 2;
    float t[P];
    load_f32<P>(cos + pair, t);
#pragma unroll
    for (int j = 0; j < P; ++j) c[j] = t[j];
    load_f32<P>(sin + pair, t);
#pragma unroll
    for (int j = 0; j < P; ++j) s[j] = t[j];
    if (second) load_f32<P>(cos + pair + P, t);
#pragma unroll
    for (int j = 0; j < P; ++j) c[P + j] = second ? t[j] : 1.f;  // the second vector may lie behind rot
    if (second) load_f32<P>(sin + pair + P, t);
#pragma unroll
    for (int j = 0; j < P; ++j) s[P + j] = second ? t[j] : 0.f;
  } else {
    load_f32<V>(cos + pair, c);
    load_f32<V>(sin + pair, s);
  }
}

// Rotates the unit (xa, xb) by +angle (SIGN 1) or -angle (SIGN -1).
template <int V, bool NEIGHBOURS, int SIGN>
__device__ __forceinline__ void rotate(float (&xa)[V], float (&xb)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (NEIGHBOURS && V > 1) {
    constexpr int P = V / 2;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float p = xa[2 * j], q = xa[2 * j + 1], n = SIGN * s[j];
      xa[2 * j] = p * c[j] - q * n;
      xa[2 * j + 1] = p * n + q * c[j];
      const float pb = xb[2 * j], qb = xb[2 * j + 1], nb = SIGN * s[P + j];
      xb[2 * j] = pb * c[P + j] - qb * nb;
      xb[2 * j + 1] = pb * nb + qb * c[P + j];
    }
  } else {
    float ya[V], yb[V], m[V], n[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      m[j] = -SIGN * s[j];
      n[j] = SIGN * s[j];
    }
    mul<V>(ya, xa, c);
    mul<V>(yb, xb, c);
    mad<V>(ya, xb, m, ya);
    mad<V>(yb, xa, n, yb);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      xa[j] = ya[j];
      xb[j] = yb[j];
    }
  }
}

// The lane's place: its heads, first row and row stride (rows advance by whole sets of heads).  Row
// counters are unsigned: those of a lane with nothing to do start at `rows` (below 2^30) and advance with
// the others, two strides ahead of the last trip, which passes 2^31.
struct Place {
  bool keys;
  int head, count;        // the first of `count` heads, among all of the row
  int row, stride, lane;  // row >= rows: nothing to do
};
template <int H>
__device__ __forceinline__ Place place_of(const QkArgs& a) {
  const int lane = threadIdx.x & 31, sub = lane / a.group;
  const unsigned warps = gridDim.x * (kThreads / 32);
  const unsigned warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  Place p;
  const unsigned slot = warp * a.groups + sub;
  p.stride = warps * a.groups / a.sets;
  p.row = slot / a.sets;
  const int set = slot - p.row * a.sets;
  // lanes behind the last whole group, and slots that make no whole set of heads
  if (sub >= a.groups || p.row >= p.stride) p.row = a.rows;
  p.lane = lane - sub * a.group;
  p.keys = set >= a.q_sets;
  const int first = (p.keys ? set - a.q_sets : set) * H;
  p.head = first + (p.keys ? a.heads : 0);
  p.count = min(H, (p.keys ? a.kv_heads : a.heads) - first);
  return p;
}

// Sum over a head's lanes, in every one of them; the whole warp takes part.  FULL: the lanes are a
// power of two.
template <bool FULL>
__device__ __forceinline__ float group_sum(float v, const QkArgs& a, const Place& p) {
  if constexpr (FULL) {
    for (int o = a.group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  } else {
    for (int n = a.group; n > 1;) {
      const int half = (n + 1) >> 1;
      const float up = __shfl_down_sync(0xffffffffu, v, half);
      if (p.lane + half < n) v += up;
      n = half;
    }
    return __shfl_sync(0xffffffffu, v, (threadIdx.x & 31) - p.lane);
  }
}

// What a lane keeps: its units' columns, norm weights and first pairs.
template <int V, int U, bool NEIGHBOURS, bool FULL>
struct Lane {
  int ca[U], cb[U], pair[U];
  bool turn[U], second[U];
  float wa[U][V], wb[U][V];
  __device__ __forceinline__ bool has_a(int u) const { return FULL || ca[u] >= 0; }
  __device__ __forceinline__ bool has_b(int u) const { return FULL || cb[u] >= 0; }
  __device__ __forceinline__ Lane(const QkArgs& a, const Place& p, const float* w) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int unit = p.lane + u * a.group;
      unit_at<V, NEIGHBOURS>(unit, a.dim, a.rot, ca[u], cb[u], turn[u], pair[u]);
      if (!FULL && unit >= a.units) {
        ca[u] = cb[u] = -1;
        turn[u] = false;
      }
      second[u] = cb[u] >= 0 && cb[u] < a.rot;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        wa[u][j] = w != nullptr && has_a(u) ? __ldg(w + ca[u] + j) : 1.f;
        wb[u][j] = w != nullptr && has_b(u) ? __ldg(w + cb[u] + j) : 1.f;
      }
    }
  }
};

// A row's position: the table row, or -1 where there is none.
struct Positions {
  int at, step;
  __device__ __forceinline__ Positions(const QkArgs& a, const Place& p) {
    at = step = 0;
    if (a.rot > 0 && a.pos == nullptr) {
      at = static_cast<unsigned>(p.row) % static_cast<unsigned>(a.seq);
      step = static_cast<unsigned>(p.stride) % static_cast<unsigned>(a.seq);
    }
  }
  // of `row`; rows come in order
  __device__ __forceinline__ long long next(const QkArgs& a, unsigned row) {
    if (a.pos != nullptr)
      return a.pos64 ? static_cast<const int64_t*>(a.pos)[row] : static_cast<const int32_t*>(a.pos)[row];
    const int now = at;
    at += step;
    if (at >= a.seq) at -= a.seq;
    return now;
  }
};

// The position, or -1 (and the status word set) for one outside the tables.
__device__ __forceinline__ long long checked(const QkArgs& a, long long pos) {
  if (pos >= 0 && pos < a.table_rows) return pos;
  atomicOr(a.status, kStatusBadShape);
  return -1;
}

struct WeightGrads {
  float *q, *k;
  int accumulate;
};

template <typename T, int V, int U>
struct Vectors {
  Pack<T, V> a[U], b[U];
  template <typename L>
  __device__ __forceinline__ void load(const T* p, const L& l) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l.has_a(u)) a[u] = Pack<T, V>::load(p + l.ca[u]);
      if (l.has_b(u)) b[u] = Pack<T, V>::load(p + l.cb[u]);
    }
  }
  template <typename L>
  __device__ __forceinline__ void store(T* p, const L& l) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l.has_a(u)) a[u].store(p + l.ca[u]);
      if (l.has_b(u)) b[u].store(p + l.cb[u]);
    }
  }
  template <typename L>
  __device__ __forceinline__ void get(float (&fa)[U][V], float (&fb)[U][V], const L& l) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l.has_a(u)) a[u].get(fa[u]);
      else zero<V>(fa[u]);
      if (l.has_b(u)) b[u].get(fb[u]);
      else zero<V>(fb[u]);
    }
  }
};

// The value heads, once the lanes are through with queries and keys: a warp per row, four vectors of
// every lane in flight.
template <typename T, int V>
__device__ __forceinline__ void copy_values(const T* src, long long ld_src, T* dst, long long ld_dst, const QkArgs& a) {
  constexpr int B = 4;
  const int first = (a.heads + a.kv_heads) * a.dim, width = a.kv_heads * a.dim;
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kThreads / 32);
  for (int row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); row < a.rows; row += warps) {
    const T* s = src + row * ld_src + first;
    T* d = dst + row * ld_dst + first;
    for (int c0 = lane * V; c0 < width; c0 += 32 * V * B) {
      Pack<T, V> v[B];
#pragma unroll
      for (int i = 0; i < B; ++i)
        if (c0 + 32 * V * i < width) v[i] = Pack<T, V>::load(s + c0 + 32 * V * i);
#pragma unroll
      for (int i = 0; i < B; ++i)
        if (c0 + 32 * V * i < width) v[i].store(d + c0 + 32 * V * i);
    }
  }
}

template <typename T, int V, int U, int H, bool NEIGHBOURS, bool FULL>
__global__ void __launch_bounds__(kThreads, 2)
    qk_norm_rope_fwd_kernel(const T* x, T* y, QkArgs a) {
  pdl_wait();
  pdl_trigger();
  const Place p = place_of<H>(a);
  const Lane<V, U, NEIGHBOURS, FULL> l(a, p, p.keys ? a.wk : a.wq);
  Positions where(a, p);
  const T* xr = x + static_cast<long long>(p.row) * a.ldx + p.head * a.dim;
  T* yr = y + static_cast<long long>(p.row) * a.ldy + p.head * a.dim;
  const long long step_x = static_cast<long long>(p.stride) * a.ldx, step_y = static_cast<long long>(p.stride) * a.ldy;
  const unsigned rows = a.rows, trips = (rows + p.stride - 1) / p.stride;
  unsigned row = p.row;
  for (unsigned t = 0; t < trips; ++t, row += p.stride, xr += step_x, yr += step_y) {
    const bool on = row < rows;
    Vectors<T, V, U> v[H];
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (on && h < p.count) v[h].load(xr + h * a.dim, l);
    const long long pos = on && a.rot > 0 ? checked(a, where.next(a, row)) : -1;
    float c[U][V], s[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (pos >= 0 && l.turn[u])
        load_angles<V, NEIGHBOURS>(a.cos + pos * a.ldt, a.sin + pos * a.ldt, l.pair[u], l.second[u], c[u], s[u]);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const bool here = on && h < p.count;
      float fa[U][V], fb[U][V], ss[2] = {0.f, 0.f};
      v[h].get(fa, fb, l);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        dot<V>(ss, fa[u], fa[u]);
        dot<V>(ss, fb[u], fb[u]);
      }
      const float r = rsqrtf(group_sum<FULL>(here ? ss[0] + ss[1] : 0.f, a, p) * a.inv_dim + a.eps);
      if (!here) continue;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        mul<V>(fa[u], fa[u], l.wa[u]);
        mul<V>(fb[u], fb[u], l.wb[u]);
        scale<V>(fa[u], r);
        scale<V>(fb[u], r);
        if (pos >= 0 && l.turn[u]) rotate<V, NEIGHBOURS, 1>(fa[u], fb[u], c[u], s[u]);
        v[h].a[u].set(fa[u]);
        v[h].b[u].set(fb[u]);
      }
      v[h].store(yr + h * a.dim, l);
    }
  }
  if (a.copies) copy_values<T, V>(x, a.ldx, y, a.ldy, a);
}

// BYTES of global memory to shared memory, in the background from 4 bytes on.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  } else if constexpr (BYTES >= 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
  } else {
    *static_cast<unsigned short*>(dst) = *static_cast<const unsigned short*>(src);
  }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's own ring of kStages rows: the vectors of dy and of x.
constexpr int kStages = 3;
template <typename T, int V, int U>
struct Ring {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T)), kVectors = 4 * U;
  static constexpr int kSize = kStages * kVectors * kThreads * kBytes;
  char* base;
  __device__ __forceinline__ T* at(int stage, int k) const {
    return reinterpret_cast<T*>(base + ((stage * kVectors + k) * kThreads + threadIdx.x) * kBytes);
  }
  template <typename L>
  __device__ __forceinline__ void fetch(int stage, int k0, const T* p, const L& l) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l.has_a(u)) copy_async<kBytes>(at(stage, k0 + 2 * u), p + l.ca[u]);
      if (l.has_b(u)) copy_async<kBytes>(at(stage, k0 + 2 * u + 1), p + l.cb[u]);
    }
  }
  template <typename L>
  __device__ __forceinline__ void read(Vectors<T, V, U>& v, int stage, int k0, const L& l) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l.has_a(u)) v.a[u] = Pack<T, V>::load(at(stage, k0 + 2 * u));
      if (l.has_b(u)) v.b[u] = Pack<T, V>::load(at(stage, k0 + 2 * u + 1));
    }
  }
};

// part: [gridDim.x][2][dim] sums of dz x r over the block's query heads and key heads, added up
// by qk_weight_grad_kernel in block order.  A single block writes dwq and dwk itself.
template <typename T, int V, int U, bool NEIGHBOURS, bool FULL>
__global__ void __launch_bounds__(kThreads, 2)
    qk_norm_rope_bwd_kernel(const T* dy, const T* __restrict__ x, T* dx, QkArgs a, float* __restrict__ part,
                            WeightGrads dw) {
  extern __shared__ __align__(16) char shared[];  // the rings, then [sets in the block][dim] sums
  pdl_wait();
  pdl_trigger();
  const Place p = place_of<1>(a);
  const Lane<V, U, NEIGHBOURS, FULL> l(a, p, p.keys ? a.wk : a.wq);
  Positions where(a, p);
  const int col = p.head * a.dim;
  const T* xr = x + static_cast<long long>(p.row) * a.ldx + col;
  const T* gr = dy + static_cast<long long>(p.row) * a.ldy + col;
  T* dr = dx + static_cast<long long>(p.row) * a.lddx + col;
  const long long step_x = static_cast<long long>(p.stride) * a.ldx, step_g = static_cast<long long>(p.stride) * a.ldy,
                  step_d = static_cast<long long>(p.stride) * a.lddx;
  float da[U][V], db[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    zero<V>(da[u]);
    zero<V>(db[u]);
  }
  {
    const Ring<T, V, U> ring{shared};
    const unsigned rows = a.rows, trips = (rows + p.stride - 1) / p.stride;
    unsigned row = p.row, ahead = row;  // the row that is fetched next
    auto fetch = [&](int stage) {
      if (ahead < rows) {
        ring.fetch(stage, 0, gr, l);
        ring.fetch(stage, 2 * U, xr, l);
      }
      copy_commit();
      ahead += p.stride;
      gr += step_g;
      xr += step_x;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i);
    int stage = 0;
    long long next_pos = a.rot > 0 && row < rows ? where.next(a, row) : -1;
    for (unsigned t = 0; t < trips; ++t, row += p.stride, dr += step_d) {
      const bool on = row < rows;
      fetch(stage == 0 ? kStages - 1 : stage - 1);
      const long long pos = on && a.rot > 0 ? checked(a, next_pos) : -1;
      if (a.rot > 0 && row + p.stride < rows) next_pos = where.next(a, row + p.stride);
      float c[U][V], s[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (pos >= 0 && l.turn[u])
          load_angles<V, NEIGHBOURS>(a.cos + pos * a.ldt, a.sin + pos * a.ldt, l.pair[u], l.second[u], c[u], s[u]);
      copy_wait<kStages - 1>();  // the row's own copies; each lane reads only what it fetched
      Vectors<T, V, U> vx, vg;
      if (on) {
        ring.read(vg, stage, 0, l);
        ring.read(vx, stage, 2 * U, l);
      }
      stage = stage == kStages - 1 ? 0 : stage + 1;
      float xa[U][V], xb[U][V], za[U][V], zb[U][V], ss[2] = {0.f, 0.f}, gx[2] = {0.f, 0.f};
      vx.get(xa, xb, l);
      vg.get(za, zb, l);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (pos >= 0 && l.turn[u]) rotate<V, NEIGHBOURS, -1>(za[u], zb[u], c[u], s[u]);
        dot<V>(ss, xa[u], xa[u]);
        dot<V>(ss, xb[u], xb[u]);
        float w_[V];
        mul<V>(w_, xa[u], l.wa[u]);
        dot<V>(gx, za[u], w_);
        mul<V>(w_, xb[u], l.wb[u]);
        dot<V>(gx, zb[u], w_);
      }
      const float r = rsqrtf(group_sum<FULL>(on ? ss[0] + ss[1] : 0.f, a, p) * a.inv_dim + a.eps);
      const float mean = group_sum<FULL>(on ? gx[0] + gx[1] : 0.f, a, p) * a.inv_dim * r * r;  // mean(g x r) r
      if (!on) continue;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float w_[V];
        // dw += dz (x r);  dx = r (dz w - x mean)
        mul<V>(w_, za[u], xa[u]);
        mad<V>(da[u], w_, r, da[u]);
        mul<V>(w_, zb[u], xb[u]);
        mad<V>(db[u], w_, r, db[u]);
        mul<V>(za[u], za[u], l.wa[u]);
        mul<V>(zb[u], zb[u], l.wb[u]);
        mad<V>(za[u], xa[u], -mean, za[u]);
        mad<V>(zb[u], xb[u], -mean, zb[u]);
        scale<V>(za[u], r);
        scale<V>(zb[u], r);
        vg.a[u].set(za[u]);
        vg.b[u].set(zb[u]);
      }
      vg.store(dr, l);
    }
  }
  copy_wait<0>();
  if (a.copies) copy_values<T, V>(dy, a.ldy, dx, a.lddx, a);
  if (part == nullptr && dw.q == nullptr && dw.k == nullptr) return;
  __syncthreads();  // the rings give way to the sums
  float* sums = reinterpret_cast<float*>(shared);
  const int sets = a.groups * (kThreads / 32);  // of the block
  const int sub = (threadIdx.x & 31) / a.group;
  if (sub < a.groups) {
    float* mine = sums + ((threadIdx.x >> 5) * a.groups + sub) * a.dim;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (l.has_a(u)) mine[l.ca[u] + j] = da[u][j];
        if (l.has_b(u)) mine[l.cb[u] + j] = db[u][j];
      }
  }
  __syncthreads();
  const unsigned slot0 = blockIdx.x * sets;
  for (int c = threadIdx.x; c < 2 * a.dim; c += kThreads) {
    const bool keys = c >= a.dim;
    const int column = keys ? c - a.dim : c;
    float v = 0.f;
    int set = slot0 % a.sets;
    for (int g = 0; g < sets; ++g) {
      if ((set >= a.q_sets) == keys) v += sums[g * a.dim + column];
      if (++set == a.sets) set = 0;
    }
    if (part != nullptr) {
      part[static_cast<long long>(blockIdx.x) * 2 * a.dim + c] = v;
    } else if (float* d = keys ? dw.k : dw.q; d != nullptr) {
      d[column] = dw.accumulate ? d[column] + v : v;
    }
  }
}

// dw (+)= sums of part over the blocks, in a fixed order: 32 columns per block, 32 slices.
__global__ void __launch_bounds__(1024)
    qk_weight_grad_kernel(const float* __restrict__ part, int blocks, int dim, WeightGrads dw) {
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
  float* d = c < dim ? dw.q : dw.k;
  if (d == nullptr) return;
  const int col = c < dim ? c : c - dim;
  d[col] = dw.accumulate ? d[col] + v : v;
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
  int v, u;
  bool full;
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
  // One unit per lane, or (narrow vectors) as many as leave fewer lanes idle; heads do not cross warps.
  // 12 + 6 heads of 72 columns, 36 of them rotated, fp32, backward: 18 units on 18 lanes of a warp take
  // 61 us, two units each on 9 lanes, three heads to a warp, 32 us.
  auto lanes = [&](int u) { return (a.units + u - 1) / u; };
  p.u = v == 2 ? 2 : v == 1 ? 4 : 1;
  if (lanes(1) <= 32 && (p.u == 1 || (32 / lanes(1)) * p.u >= 32 / lanes(p.u))) p.u = 1;
  a.group = lanes(p.u);
  a.groups = 32 / a.group;
  p.full = v * size == 16 && 2 * v * a.units == a.dim && (a.group & (a.group - 1)) == 0;
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

// Shared memory of the backward kernels: the rings (48 KB at most).  The weight gradients' sums
// that take their place need 8 warps x 2 V U x 32 columns at most, a third of that.
template <typename T, int V, int U>
constexpr int kBwdSmem = std::max(Ring<T, V, U>::kSize, kThreads / 32 * 64 * V * U * 4);

// Blocks of a kernel that fit on an SM of the current device.
template <auto Kernel, int Smem>
int resident(int device) {
  static std::atomic<int> known[64];
  std::atomic<int>& k = known[device & 63];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    REVPP_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, kThreads, Smem));
    n = std::max(1, n);
    k.store(n, std::memory_order_relaxed);
  }
  return n;
}

// Blocks for one resident wave, or fewer when the rows need fewer; one where `single` would do.
template <auto Kernel, int Smem>
int blocks_for(const QkArgs& a, int device, int single) {
  const int per_block = a.groups * (kThreads / 32);
  const long long need = (static_cast<long long>(a.rows) * a.sets + per_block - 1) / per_block;
  const long long least = (a.sets + per_block - 1) / per_block;
  if (least == 1 && need <= single) return 1;
  const long long wave = static_cast<long long>(resident<Kernel, Smem>(device)) * num_sms();
  return static_cast<int>(std::max(least, std::min(need, wave)));
}

// Sets of h query or key heads.
void make_sets(QkArgs& a, int h) {
  a.q_sets = (a.heads + h - 1) / h;
  a.sets = a.q_sets + (a.kv_heads + h - 1) / h;
}

template <typename F>
void by_type(const Problem& p, at::ScalarType t, bool interleaved, F&& f) {
  using std::integral_constant;
  auto by_v = [&](auto e, auto nb) {
    using T = decltype(e);
    constexpr int W = 16 / sizeof(T);
    if (p.v == W && p.full) return f(e, integral_constant<int, W>{}, integral_constant<int, 1>{}, nb, std::true_type{});
    if (p.v == W) return f(e, integral_constant<int, W>{}, integral_constant<int, 1>{}, nb, std::false_type{});
    if constexpr (W > 4) {
      if (p.v == 4) return f(e, integral_constant<int, 4>{}, integral_constant<int, 1>{}, nb, std::false_type{});
    }
    if (p.v == 2 && p.u == 1) return f(e, integral_constant<int, 2>{}, integral_constant<int, 1>{}, nb, std::false_type{});
    if (p.v == 2) return f(e, integral_constant<int, 2>{}, integral_constant<int, 2>{}, nb, std::false_type{});
    if (p.u == 1) return f(e, integral_constant<int, 1>{}, integral_constant<int, 1>{}, nb, std::false_type{});
    f(e, integral_constant<int, 1>{}, integral_constant<int, 4>{}, nb, std::false_type{});
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
  make_sets(a, kFwdHeads);
  a.copies = qkv.data_ptr() != out.data_ptr();
  by_type(p, qkv.scalar_type(), interleaved, [&](auto e, auto v, auto u, auto nb, auto full) {
    using T = decltype(e);
    constexpr auto kernel =
        &qk_norm_rope_fwd_kernel<T, decltype(v)::value, decltype(u)::value, kFwdHeads, decltype(nb)::value, decltype(full)::value>;
    launch_pdl(kernel, dim3(blocks_for<kernel, 0>(a, qkv.get_device(), 1)), dim3(kThreads), 0, cur_stream(),
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
  const WeightGrads dw{given(dwq) ? dwq->data_ptr<float>() : nullptr, given(dwk) ? dwk->data_ptr<float>() : nullptr,
                       accumulate ? 1 : 0};
  int blocks = 0;
  torch::Tensor part;
  if (a.rows > 0) {
    finish(p, {&qkv, &dout, &dqkv}, wq, wk, cos, sin, positions, S, interleaved);
    a.ldy = dout.stride(0);
    a.lddx = dqkv.stride(0);
    make_sets(a, 1);
    a.copies = dout.data_ptr() != dqkv.data_ptr();
    by_type(p, qkv.scalar_type(), interleaved, [&](auto e, auto v, auto u, auto nb, auto full) {
      using T = decltype(e);
      constexpr auto kernel =
          &qk_norm_rope_bwd_kernel<T, decltype(v)::value, decltype(u)::value, decltype(nb)::value, decltype(full)::value>;
      constexpr int smem = kBwdSmem<T, decltype(v)::value, decltype(u)::value>;
      // work for two blocks goes to one that needs no second launch for the weight gradients
      blocks = blocks_for<kernel, smem>(a, qkv.get_device(), weights ? 2 : 1);
      if (weights && blocks > 1) part = torch::empty({static_cast<int64_t>(blocks) * 2 * a.dim}, qkv.options().dtype(at::kFloat));
      launch_pdl(kernel, dim3(blocks), dim3(kThreads), smem, cur_stream(), static_cast<const T*>(dout.data_ptr()),
                 static_cast<const T*>(qkv.data_ptr()), static_cast<T*>(dqkv.data_ptr()), a,
                 weights && blocks > 1 ? part.data_ptr<float>() : static_cast<float*>(nullptr), dw);
    });
    REVPP_CHECK_LAUNCH();
  }
  if (!weights || blocks == 1) return;
  launch_pdl(qk_weight_grad_kernel, dim3((2 * a.dim + 31) / 32), dim3(1024), 0, cur_stream(),
             blocks > 0 ? const_cast<const float*>(part.data_ptr<float>()) : static_cast<const float*>(nullptr), blocks, a.dim,
             dw);
  REVPP_CHECK_LAUNCH();
}

}  // namespace revpp

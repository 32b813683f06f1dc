// A block's result onto the residual stream, and the norm before the next block (tc_residual_norm_*).
//
//   u = f r, r = (mean f^2 + eps)^-1/2      h = s x + g (u post)      n = h q pre, q = (mean h^2 + eps)^-1/2
//
// and backward, at h as it was stored, with v = h q and means over a row:
//
//   dh' = dh + q (dn pre - v mean(dn pre v))    dx = s dh'     dp = dh' g     df = r (dp post - u mean(dp post u))
//   dg = dh' u post    dpost = sum dp u    dpre = sum dn v
//
// where tokens share the gate (or have none) both of the first come from one sum S = sum dh' u: dg = post S, dpost = g S.
//
// Both directions read every row once: a group of warps holds it in registers, eight elements a thread and piece.  A group takes
// row after row; where rows are aligned the next ones are already on their way to shared memory (cp.async, each thread its own
// elements, so that nothing has to be waited for together), else its threads read neighbouring elements one by one.  Backward the sums
// over tokens of a thread's columns stay in registers too; a block's groups add theirs up, and blocks' are joined in order by a second
// launch, so that results do not depend on which ran when.  Rows of more than 16384 elements (backward 8192, of single
// precision 4096) are read again for each of the steps between row sums.
//
// Bound by bytes.
#include <algorithm>

#include "tc_elem.cuh"
#include "tc_inst.cuh"
#include "tc_op.h"

namespace {
using namespace tck;

constexpr int kMostWarps = 16;

struct NormArgs {
  const void *x, *f, *gate, *post, *pre;
  const void *dh, *dn;     // backward: either may be null
  void *h, *n;             // backward: h is read; dx, df and dgate (by token) are written where they are asked for
  void *dx, *df, *dgate;
  int64_t ld_x, ld_f, ld_gate, ld_h, ld_n, ld_dh, ld_dn, ld_dx, ld_df, ld_dgate, tokens;
  float* part;             // [2][slots][pitch]: sums of dh' u (times the token's own gate) and of dn v
  uint32_t slots, pitch;
  uint32_t dim;
  int warps;               // that hold a row
  int gate_kind, wide;     // wide: weights are fp32
  float residual, inverse_dim;
  double eps;
};

// ---- sums over a group of warps ----
struct Group {
  int warps, lane, warp, id, thread;  // warp: in the group; id: the group in its block
  __device__ __forceinline__ explicit Group(int w) : warps(w) {
    lane = threadIdx.x & 31;
    warp = (int)(threadIdx.x >> 5) % w;
    id = (int)(threadIdx.x >> 5) / w;
    thread = warp * 32 + lane;
  }
  __device__ __forceinline__ void wait() const {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;\n" ::"r"(id + 1), "r"(warps * 32) : "memory");
  }
};
// `turn` alternates between two places that share no byte, so that one wait a sum is enough.
constexpr int kMostSums = 3;
template <int N, class S>
__device__ __forceinline__ void group_sum(const Group& g, S (&v)[N], double* shared, int turn) {
  static_assert(N <= kMostSums, "place");
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (g.warps == 1) return;
  S* mine = reinterpret_cast<S*>(shared + turn * kMostWarps * kMostSums) + g.id * g.warps * N;
  if (g.lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) mine[g.warp * N + i] = v[i];
  g.wait();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0;
    for (int w = 0; w < g.warps; ++w) v[i] += mine[w * N + i];
  }
}
// Sums of squares that left 32 bits on either side are taken again in 64.
__device__ __forceinline__ bool out_of_range(float s) { return !(s > 1e-30f && s < INFINITY); }
__device__ __forceinline__ float inverse_root(float sum, const NormArgs& a) { return 1.f / sqrtf(fmaf(sum, a.inverse_dim, (float)a.eps)); }
__device__ __forceinline__ float inverse_root(double sum, const NormArgs& a) { return (float)(1.0 / sqrt(sum / a.dim + a.eps)); }
template <class Again>
__device__ __forceinline__ float root_of(const Group& g, const NormArgs& a, float sum, double* shared, int turn, Again again) {
  float s[1] = {sum};
  group_sum(g, s, shared, turn);
  if (!out_of_range(s[0])) return inverse_root(s[0], a);
  g.wait();
  double d[1] = {again()};
  group_sum(g, d, shared, turn);
  g.wait();
  return inverse_root(d[0], a);
}
__device__ __forceinline__ double squares8(const float* f) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s = fmaf(f[k], f[k], s);
  if (!out_of_range(s)) return (double)s;
  double d = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) d = fma((double)f[k], (double)f[k], d);
  return d;
}

// ---- eight elements of a thread ----
// Neighbours where 16-byte accesses reach them, else `step` apart, so that neighbouring threads touch neighbours.  None from `dim` on: zeros.
template <bool Vec>
struct Where {
  uint32_t col, step, dim;
  __device__ __forceinline__ bool there(int k) const { return Vec ? col < dim : col + k * step < dim; }
};
template <class T, bool Vec>
__device__ __forceinline__ Raw<T> get8(const T* p, const Where<Vec>& at, bool any = true) {
  if constexpr (Vec) {
    return load8<T, true>(p + at.col, any && at.col < at.dim ? 8 : 0);
  } else {
    Raw<T> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 8; ++k) r.w[k] = any && at.there(k) ? __float_as_uint(p[at.col + k * at.step]) : 0u;
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + at.col;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r.w[k] = (any && at.there(2 * k) ? (uint32_t)q[2 * k * at.step] : 0u) | (any && at.there(2 * k + 1) ? (uint32_t)q[(2 * k + 1) * at.step] << 16 : 0u);
    }
    return r;
  }
}
template <class T, bool Vec>
__device__ __forceinline__ void put8(T* p, const Where<Vec>& at, const float* f) {
  const Raw<T> r = pack8<T>(f);
  if constexpr (Vec) {
    store8<T, true>(p + at.col, r, at.col < at.dim ? 8 : 0);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at.there(k)) p[at.col + k * at.step] = __uint_as_float(r.w[k]);
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p) + at.col;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at.there(k)) q[k * at.step] = (uint16_t)(r.w[k >> 1] >> (16 * (k & 1)));
  }
}
template <class T, bool Vec>
__device__ __forceinline__ void weight8(const void* w, const Where<Vec>& at, bool wide, float* f) {
  if (!w) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 1.f;
  } else if (wide) {
    unpack8<float>(get8<float, Vec>(static_cast<const float*>(w), at), f);
  } else {
    unpack8<T>(get8<T, Vec>(static_cast<const T*>(w), at), f);
  }
}
template <class T, bool Vec>
__device__ __forceinline__ Raw<T> row8(const void* p, int64_t ld, int64_t row, const Where<Vec>& at) {
  return get8<T, Vec>(static_cast<const T*>(p) + row * ld, at, p != nullptr);
}
template <class T, bool Vec>
__device__ __forceinline__ void put_row8(void* p, int64_t ld, int64_t row, const Where<Vec>& at, const float* f) {
  put8<T, Vec>(static_cast<T*>(p) + row * ld, at, f);
}
// A gate that is the same for all tokens, or none; a token's own comes with its row.
template <class T, bool Vec>
__device__ __forceinline__ void gate8(const NormArgs& a, int64_t row, const Where<Vec>& at, float* f) {
  if (a.gate_kind == TC_GATE_TOKEN) unpack8<T>(row8<T, Vec>(a.gate, a.ld_gate, row, at), f);
  else weight8<T, Vec>(a.gate, at, false, f);
}

// N matrices whose rows a group takes one after another: a thread's own elements, Stages rows ahead in shared memory where Vec.
template <class T, bool Vec, int V, int N>
struct Ahead {
  static constexpr int kBytes = V * N * 8 * (int)sizeof(T);                          // of a thread and row
  static constexpr int kStages = !Vec ? 0 : kBytes <= 32 ? 4 : kBytes <= 64 ? 2 : 1;  // at most 128 KB a multiprocessor, and L1 for the weights
  static constexpr int kPieces = 8 * (int)sizeof(T) / 16;
  const void* from[N];
  int64_t ld[N];
  uint32_t place, stride;  // of the thread's first 16 bytes; between one thread's pieces
  int64_t tokens, slots;
  uint32_t dim, first, step;
  __device__ __forceinline__ void start(unsigned char* ring, const NormArgs& a, const Group& g, int64_t row) {
    place = Vec ? smem_u32(ring) + threadIdx.x * 16 : 0u;
    stride = blockDim.x * 16;
    tokens = a.tokens;
    slots = a.slots;
    dim = a.dim;
    first = g.thread * 8;
    step = a.warps * 32 * 8;
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(s, row + s * slots);
  }
  __device__ __forceinline__ void fetch(int stage, int64_t row) const {
    if constexpr (Vec) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int p = 0; p < V; ++p)
#pragma unroll
          for (int q = 0; q < kPieces; ++q) {
            const uint32_t col = first + p * step;
            const bool there = from[i] && row < tokens && col < dim;
            const unsigned char* src = static_cast<const unsigned char*>(from[i]) + ((there ? row * ld[i] + col : 0) * (int64_t)sizeof(T) + (there ? q * 16 : 0));
            if (there) cp_async16(place + (((stage * N + i) * V + p) * kPieces + q) * stride, src, true);
          }
      cp_async_commit();
    }
  }
  // The group's row number n (of this loop), row `row` of the matrices.
  __device__ __forceinline__ void take(int n, int64_t row, const Where<Vec> (&at)[V], Raw<T> (&raw)[N][V]) const {
    if constexpr (Vec) {
      cp_async_wait<kStages - 1>();
      const int stage = kStages == 1 ? 0 : n % kStages;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int p = 0; p < V; ++p) {
          const bool there = from[i] && at[p].col < dim;
#pragma unroll
          for (int q = 0; q < kPieces; ++q) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (there) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                    : "r"(place + (((stage * N + i) * V + p) * kPieces + q) * stride) : "memory");
            raw[i][p].w[4 * q] = v.x; raw[i][p].w[4 * q + 1] = v.y; raw[i][p].w[4 * q + 2] = v.z; raw[i][p].w[4 * q + 3] = v.w;
          }
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int p = 0; p < V; ++p) raw[i][p] = row8<T, Vec>(from[i], ld[i], row, at[p]);
    }
  }
  // Once the row's elements have been used: the one that takes its place.
  __device__ __forceinline__ void next(int n, int64_t row) const {
    if constexpr (Vec) fetch(kStages == 1 ? 0 : n % kStages, row + kStages * slots);
  }
};
template <bool Vec, int V>
__device__ __forceinline__ void places(const NormArgs& a, const Group& g, Where<Vec> (&at)[V]) {
#pragma unroll
  for (int p = 0; p < V; ++p) {
    const uint32_t threads = a.warps * 32;
    at[p] = Vec ? Where<Vec>{(p * threads + g.thread) * 8, 1u, a.dim} : Where<Vec>{p * threads * 8 + g.thread, threads, a.dim};
  }
}

// ---- forward ----
// ByToken: a gate of its own for each token.
template <class T, bool Vec, int V, bool ByToken>
__global__ void __launch_bounds__(32 * kMostWarps, V == 1 ? 2 : 1) norm_kernel(const __grid_constant__ NormArgs a) {
  constexpr int N = ByToken ? 3 : 2;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(a.warps);
  const int64_t first = (int64_t)blockIdx.x * (blockDim.x / (32 * a.warps)) + g.id;
  Where<Vec> at[V];
  places(a, g, at);
  Ahead<T, Vec, V, N> rows{};
  rows.from[0] = a.f; rows.ld[0] = a.ld_f;
  rows.from[1] = a.x; rows.ld[1] = a.ld_x;
  if constexpr (ByToken) { rows.from[N - 1] = a.gate; rows.ld[N - 1] = a.ld_gate; }
  chain_wait();
  rows.start(ring, a, g, first);
  int turn = 0;
  for (int64_t row = first; row < a.tokens; row += a.slots, ++turn) {
    Raw<T> raw[N][V];
    rows.take(turn, row, at, raw);
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float f[8];
      unpack8<T>(raw[0][p], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(f[k], f[k], s);
    }
    const float r = root_of(g, a, s, shared, 0, [&]() {
      double d = 0;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        float f[8];
        unpack8<T>(raw[0][p], f);
        d += squares8(f);
      }
      return d;
    });
    float h[V][8];
    s = 0.f;
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float f[8], w[8];
      unpack8<T>(raw[1][p], h[p]);
      unpack8<T>(raw[0][p], f);
      weight8<T, Vec>(a.post, at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = f[k] * r * w[k];
      if constexpr (ByToken) unpack8<T>(raw[N - 1][p], w);
      else weight8<T, Vec>(a.gate, at[p], false, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        h[p][k] = fmaf(w[k], f[k], a.residual * h[p][k]);
        s = fmaf(h[p][k], h[p][k], s);
      }
      put_row8<T, Vec>(a.h, a.ld_h, row, at[p], h[p]);
    }
    rows.next(turn, row);
    if (!a.n) {
      g.wait();  // the sums' place is free again
      continue;
    }
    const float q = root_of(g, a, s, shared, 1, [&]() {
      double d = 0;
#pragma unroll
      for (int p = 0; p < V; ++p) d += squares8(h[p]);
      return d;
    });
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float w[8];
      weight8<T, Vec>(a.pre, at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) h[p][k] = h[p][k] * q * w[k];
      put_row8<T, Vec>(a.n, a.ld_n, row, at[p], h[p]);
    }
  }
}

// The places of a long row: 8 * kLongThreads columns at a time.
constexpr uint32_t kLongThreads = 32 * kMostWarps, kLongStep = kLongThreads * 8;
template <bool Vec>
__device__ __forceinline__ Where<Vec> long_place(const NormArgs& a, uint32_t base) {
  return Vec ? Where<Vec>{base + threadIdx.x * 8, 1u, a.dim} : Where<Vec>{base + threadIdx.x, kLongThreads, a.dim};
}

// Rows too long for registers: h is computed a second time for n.
template <class T, bool Vec>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(kMostWarps);
  const int64_t row = blockIdx.x;
  chain_wait();
  double s[1] = {0};
  for (uint32_t base = 0; base < a.dim; base += kLongStep) {
    float f[8];
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, long_place<Vec>(a, base)), f);
    s[0] += squares8(f);
  }
  group_sum(g, s, shared, 0);
  const float r = inverse_root(s[0], a);
  auto residual = [&](const Where<Vec>& at, float* h) {
    float f[8], w[8];
    unpack8<T>(row8<T, Vec>(a.x, a.ld_x, row, at), h);
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, at), f);
    weight8<T, Vec>(a.post, at, a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = f[k] * r * w[k];
    gate8<T, Vec>(a, row, at, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = fmaf(w[k], f[k], a.residual * h[k]);
  };
  s[0] = 0;
  for (uint32_t base = 0; base < a.dim; base += kLongStep) {
    const Where<Vec> at = long_place<Vec>(a, base);
    float h[8];
    residual(at, h);
    put_row8<T, Vec>(a.h, a.ld_h, row, at, h);
    s[0] += squares8(h);
  }
  if (!a.n) return;
  group_sum(g, s, shared, 1);
  const float q = inverse_root(s[0], a);
  for (uint32_t base = 0; base < a.dim; base += kLongStep) {
    const Where<Vec> at = long_place<Vec>(a, base);
    float h[8], w[8];
    residual(at, h);
    weight8<T, Vec>(a.pre, at, a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = h[k] * q * w[k];
    put_row8<T, Vec>(a.n, a.ld_n, row, at, h);
  }
}

// ---- backward ----
// Eight columns of a row once its sums are known; adds to the columns' own sums.
struct RowSums {
  float r, q, c2, c1;  // c2: mean(dn pre v), c1: mean(dp post u)
};
// dh' of eight columns, and v.
template <class T>
__device__ __forceinline__ void stream8(const Raw<T>& rh, const Raw<T>& rdh, const float* dnw, const RowSums& t, float* dh, float* v) {
  unpack8<T>(rh, v);
  unpack8<T>(rdh, dh);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    v[k] *= t.q;
    dh[k] = fmaf(t.q, fmaf(-v[k], t.c2, dnw[k]), dh[k]);
  }
}

template <class T, bool Vec, int V, bool ByToken>
__global__ void __launch_bounds__(32 * kMostWarps) norm_grad_kernel(const __grid_constant__ NormArgs a) {
  constexpr int N = ByToken ? 5 : 4;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(a.warps);
  const uint32_t groups = blockDim.x / (32 * a.warps);
  const int64_t first = (int64_t)blockIdx.x * groups + g.id;
  float stream[V][8] = {}, dpre[V][8] = {};
  Where<Vec> at[V];
  places(a, g, at);
  Ahead<T, Vec, V, N> rows{};
  rows.from[0] = a.f; rows.ld[0] = a.ld_f;
  rows.from[1] = a.h; rows.ld[1] = a.ld_h;
  rows.from[2] = a.dn; rows.ld[2] = a.ld_dn;
  rows.from[3] = a.dh; rows.ld[3] = a.ld_dh;
  if constexpr (ByToken) { rows.from[N - 1] = a.gate; rows.ld[N - 1] = a.ld_gate; }
  chain_wait();
  rows.start(ring, a, g, first);
  int turn = 0;
  for (int64_t row = first; row < a.tokens; row += a.slots, ++turn) {
    Raw<T> raw[N][V];
    rows.take(turn, row, at, raw);
    auto sums = [&](auto* s) {  // f^2, h^2, dn pre h
      using S = std::remove_reference_t<decltype(*s)>;
      s[0] = s[1] = s[2] = 0;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        float f[8], h[8], dn[8], w[8];
        unpack8<T>(raw[0][p], f);
        unpack8<T>(raw[1][p], h);
        unpack8<T>(raw[2][p], dn);
        weight8<T, Vec>(a.pre, at[p], a.wide, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          s[0] = fma((S)f[k], (S)f[k], s[0]);
          s[1] = fma((S)h[k], (S)h[k], s[1]);
          s[2] = fma((S)dn[k] * (S)w[k], (S)h[k], s[2]);
        }
      }
    };
    float s[3];
    sums(s);
    group_sum(g, s, shared, 0);
    RowSums t;
    t.r = inverse_root(s[0], a);
    t.q = inverse_root(s[1], a);
    t.c2 = t.q * s[2] * a.inverse_dim;
    if (out_of_range(s[0]) || out_of_range(s[1])) {
      g.wait();
      double d[3];
      sums(d);
      group_sum(g, d, shared, 0);
      g.wait();
      t.r = inverse_root(d[0], a);
      t.q = inverse_root(d[1], a);
      t.c2 = (float)(t.q * d[2] * a.inverse_dim);
    }
    rows.next(turn, row);
    float c1[1] = {0.f};
    float dpw[V][8];
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float dn[8], w[8], dh[8], v[8], u[8], gate[8];
      unpack8<T>(raw[2][p], dn);
      weight8<T, Vec>(a.pre, at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] *= dn[k];
      stream8<T>(raw[1][p], raw[3][p], w, t, dh, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) dpre[p][k] = fmaf(dn[k], v[k], dpre[p][k]);
      unpack8<T>(raw[0][p], u);
      if constexpr (ByToken) unpack8<T>(raw[N - 1][p], gate);
      else weight8<T, Vec>(a.gate, at[p], false, gate);
      weight8<T, Vec>(a.post, at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        u[k] *= t.r;
        stream[p][k] = fmaf(ByToken ? dh[k] * gate[k] : dh[k], u[k], stream[p][k]);
        dpw[p][k] = dh[k] * gate[k] * w[k];
        c1[0] = fmaf(dpw[p][k], u[k], c1[0]);
        if constexpr (ByToken) gate[k] = dh[k] * u[k] * w[k];
        dh[k] *= a.residual;
      }
      if (a.dx) put_row8<T, Vec>(a.dx, a.ld_dx, row, at[p], dh);
      if (ByToken && a.dgate) put_row8<T, Vec>(a.dgate, a.ld_dgate, row, at[p], gate);
    }
    group_sum(g, c1, shared, 1);
    if (!a.df) continue;
    const float mean = c1[0] * a.inverse_dim;
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float u[8];
      unpack8<T>(raw[0][p], u);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = t.r * fmaf(-u[k] * t.r, mean, dpw[p][k]);
      put_row8<T, Vec>(a.df, a.ld_df, row, at[p], u);
    }
  }
  if (!a.part) return;
  // The block's groups in order, each sum through the shared memory that the rows came by; then the block's slot.
  cp_async_wait<0>();
  float* sums = reinterpret_cast<float*>(ring);
  const uint32_t threads = a.warps * 32, width = V * threads * 8;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (groups > 1) {
      __syncthreads();
#pragma unroll
      for (int p = 0; p < V; ++p)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          sums[g.id * width + (p * 8 + k) * threads + g.thread] = which == 0 ? stream[p][k] : dpre[p][k];
      __syncthreads();
      if (g.id > 0) continue;
    }
    float* to = a.part + ((size_t)which * gridDim.x + blockIdx.x) * a.pitch;
#pragma unroll
    for (int p = 0; p < V; ++p)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float v = which == 0 ? stream[p][k] : dpre[p][k];
        for (uint32_t i = 1; i < groups; ++i) v += sums[i * width + (p * 8 + k) * threads + g.thread];
        if (at[p].there(k)) to[at[p].col + k * at[p].step] = v;
      }
  }
}

// Rows too long for registers: their sums first ...
template <class T, bool Vec>
__global__ void __launch_bounds__(kLongThreads) norm_long_sums_kernel(const __grid_constant__ NormArgs a, RowSums* out) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(kMostWarps);
  const int64_t row = blockIdx.x;
  chain_wait();
  double s[3] = {0, 0, 0};
  auto scaled = [&](const Where<Vec>& at, float* dnw) {
    float w[8];
    unpack8<T>(row8<T, Vec>(a.dn, a.ld_dn, row, at), dnw);
    weight8<T, Vec>(a.pre, at, a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) dnw[k] *= w[k];
  };
  for (uint32_t base = 0; base < a.dim; base += kLongStep) {
    const Where<Vec> at = long_place<Vec>(a, base);
    float f[8], h[8], dnw[8];
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, at), f);
    unpack8<T>(row8<T, Vec>(a.h, a.ld_h, row, at), h);
    scaled(at, dnw);
    s[0] += squares8(f);
    s[1] += squares8(h);
#pragma unroll
    for (int k = 0; k < 8; ++k) s[2] = fma((double)dnw[k], (double)h[k], s[2]);
  }
  group_sum(g, s, shared, 0);
  RowSums t;
  t.r = inverse_root(s[0], a);
  t.q = inverse_root(s[1], a);
  t.c2 = (float)(t.q * s[2] * a.inverse_dim);
  double c1[1] = {0};
  for (uint32_t base = 0; base < a.dim; base += kLongStep) {
    const Where<Vec> at = long_place<Vec>(a, base);
    float dnw[8], dh[8], v[8], u[8], w[8], gate[8];
    scaled(at, dnw);
    stream8<T>(row8<T, Vec>(a.h, a.ld_h, row, at), row8<T, Vec>(a.dh, a.ld_dh, row, at), dnw, t, dh, v);
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, at), u);
    weight8<T, Vec>(a.post, at, a.wide, w);
    gate8<T, Vec>(a, row, at, gate);
    float e = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) e = fmaf(dh[k] * gate[k] * w[k], u[k] * t.r, e);
    c1[0] += (double)e;
  }
  group_sum(g, c1, shared, 1);
  t.c1 = (float)(c1[0] * a.inverse_dim);
  if (g.thread == 0) out[row] = t;
}
// ... then 1024 columns a block, every slots-th row.
template <class T, bool Vec>
__global__ void __launch_bounds__(128) norm_long_grad_kernel(const __grid_constant__ NormArgs a, const RowSums* in) {
  const Where<Vec> at = Vec ? Where<Vec>{blockIdx.x * 1024 + threadIdx.x * 8, 1u, a.dim} : Where<Vec>{blockIdx.x * 1024 + threadIdx.x, 128u, a.dim};
  chain_wait();
  if (at.col >= a.dim) return;
  float stream[8] = {}, dpre[8] = {}, post[8], pre[8];
  weight8<T, Vec>(a.post, at, a.wide, post);
  weight8<T, Vec>(a.pre, at, a.wide, pre);
  for (int64_t row = blockIdx.y; row < a.tokens; row += a.slots) {
    const RowSums t = in[row];
    float dn[8], dnw[8], dh[8], v[8], u[8], gate[8], dg[8];
    unpack8<T>(row8<T, Vec>(a.dn, a.ld_dn, row, at), dn);
#pragma unroll
    for (int k = 0; k < 8; ++k) dnw[k] = dn[k] * pre[k];
    stream8<T>(row8<T, Vec>(a.h, a.ld_h, row, at), row8<T, Vec>(a.dh, a.ld_dh, row, at), dnw, t, dh, v);
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, at), u);
    gate8<T, Vec>(a, row, at, gate);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u[k] *= t.r;
      const float dp = dh[k] * gate[k];
      dpre[k] = fmaf(dn[k], v[k], dpre[k]);
      stream[k] = fmaf(a.gate_kind == TC_GATE_TOKEN ? dp : dh[k], u[k], stream[k]);
      dg[k] = dh[k] * u[k] * post[k];
      u[k] = t.r * fmaf(-u[k], t.c1, dp * post[k]);
      dh[k] *= a.residual;
    }
    if (a.dx) put_row8<T, Vec>(a.dx, a.ld_dx, row, at, dh);
    if (a.df) put_row8<T, Vec>(a.df, a.ld_df, row, at, u);
    if (a.dgate && a.gate_kind == TC_GATE_TOKEN) put_row8<T, Vec>(a.dgate, a.ld_dgate, row, at, dg);
  }
  if (!a.part) return;
  float* to = a.part + (size_t)blockIdx.y * a.pitch;
  const size_t next = (size_t)gridDim.y * a.pitch;
  put8<float, Vec>(to, at, stream);
  put8<float, Vec>(to + next, at, dpre);
}

// Sums over tokens: 32 columns a block, every 32nd slot a warp, warps in order.  blockIdx.y 0: the gradients by post and a gate that tokens
// share, 1: by pre.
struct JoinArgs {
  const float* part;
  const void *gate, *post;
  void *dpost, *dgate, *dpre;
  int wide, channel;
  uint32_t slots, pitch, dim;
};
template <class T>
__global__ void __launch_bounds__(1024) norm_join_kernel(const __grid_constant__ JoinArgs a) {
  __shared__ float sums[32][33];
  const uint32_t lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane, warp = threadIdx.x >> 5;
  chain_wait();
  if (blockIdx.y == 0 ? !a.dpost && !a.dgate : !a.dpre) return;
  const float* from = a.part + (size_t)blockIdx.y * a.slots * a.pitch + col;
  float s = 0.f;
  if (col < a.dim)
#pragma unroll 8
    for (uint32_t i = warp; i < a.slots; i += 32) s += from[(size_t)i * a.pitch];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp > 0 || col >= a.dim) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) s += sums[i][lane];
  auto put = [&](void* out, float v) {
    if (a.wide) static_cast<float*>(out)[col] = v;
    else static_cast<T*>(out)[col] = Elem<T>::put(v);
  };
  if (blockIdx.y == 1) {
    put(a.dpre, s);
    return;
  }
  if (a.dpost) put(a.dpost, a.channel ? s * Elem<T>::get(static_cast<const T*>(a.gate)[col]) : s);
  if (a.dgate) {
    const float w = !a.post ? 1.f : a.wide ? static_cast<const float*>(a.post)[col] : Elem<T>::get(static_cast<const T*>(a.post)[col]);
    static_cast<T*>(a.dgate)[col] = Elem<T>::put(s * w);
  }
}

// ---- launches ----
constexpr int64_t kForward = 16384;  // longest rows that stay in registers
int64_t longest_backward(const TcOpShape& p) { return p.dtype == TC_F32 ? 4096 : 8192; }

int warps_of(int64_t dim, int pieces) {  // that hold a row of `pieces` pieces a thread
  int w = 1;
  while (w < kMostWarps && (int64_t)w * 256 * pieces < dim) w *= 2;
  return w;
}
// Backward, 16-bit rows of 2049 to 4096 elements in blocks of 256 threads, of which two share a multiprocessor.
int pieces_of(const TcOpShape& p, bool backward) {
  return p.dim <= (backward && p.dtype != TC_F32 ? 2048 : 4096) ? 1 : p.dim <= 8192 ? 2 : 4;
}
int groups_of(int warps) { return warps >= 8 ? 1 : 8 / warps; }
uint32_t pitch_of(const TcOpShape& p) { return (uint32_t)((p.dim + 7) / 8 * 8); }
// Blocks that take row after row: as many as a multiprocessor holds, by their registers.
int64_t most_blocks(const TcOpShape& p, bool backward) {
  const int v = pieces_of(p, backward), w = warps_of(p.dim, v);
  return (int64_t)p.sms * (backward ? (w == 16 ? 1 : v == 2 ? 2 : p.dtype == TC_F32 ? 2 : 3) : w < 16 ? 4 : v > 1 ? 1 : 2);
}
// Most blocks that sum columns of their own.
int64_t most_slots(const TcOpShape& p) {
  return p.dim <= longest_backward(p) ? most_blocks(p, true) : std::min<int64_t>(p.tokens, std::max<int64_t>(1, 16 * (int64_t)p.sms / ((p.dim + 1023) / 1024)));
}

struct Buffers {
  float* part;
  RowSums* sums;
};
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  TcCarver c{base};
  b->part = c.take<float>((size_t)2 * most_slots(p) * pitch_of(p));
  b->sums = c.take<RowSums>(p.dim > longest_backward(p) ? (size_t)p.tokens : 0);
  return c.used;
}

typedef void (*Kernel)(NormArgs);
struct Built {
  Kernel kernel;
  int per_thread;  // bytes of shared memory
};
template <class T, bool Vec, int V, bool ByToken>
Built built(bool backward) {
  if constexpr (V == 1 || (V == 2 && sizeof(T) == 2)) {
    if (backward) {
      using A = Ahead<T, Vec, V, ByToken ? 5 : 4>;
      return Built{norm_grad_kernel<T, Vec, V, ByToken>, std::max(A::kStages * A::kBytes, V * 32)};  // or a column's sum
    }
  }
  using A = Ahead<T, Vec, V, ByToken ? 3 : 2>;
  return Built{norm_kernel<T, Vec, V, ByToken>, A::kStages * A::kBytes};
}
template <class T, bool Vec, bool ByToken>
Built built(bool backward, int v) {
  return v == 1 ? built<T, Vec, 1, ByToken>(backward) : v == 2 ? built<T, Vec, 2, ByToken>(backward) : built<T, Vec, 4, ByToken>(backward);
}
template <class T>
Built built(bool backward, int v, bool vec, bool by_token) {
  return vec ? (by_token ? built<T, true, true>(backward, v) : built<T, true, false>(backward, v))
             : (by_token ? built<T, false, true>(backward, v) : built<T, false, false>(backward, v));
}
template <class T>
int prepare() {
  for (bool backward : {false, true})
    for (int v : {1, 2, 4})
      for (bool vec : {false, true})
        for (bool by_token : {false, true}) {
          const Built b = built<T>(backward, v, vec, by_token);
          TC_CUDA_OK(cudaFuncSetAttribute(b.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, b.per_thread * 32 * kMostWarps));
        }
  return TC_OK;
}
template <class T>
int launch(const TcOpShape& p, NormArgs a, bool backward, bool vec, int64_t* blocks, cudaStream_t stream) {
  const int v = pieces_of(p, backward);
  a.warps = warps_of(p.dim, v);
  const int groups = groups_of(a.warps);
  a.slots = (uint32_t)(*blocks * groups);
  const Built b = built<T>(backward, v, vec, p.gate == TC_GATE_TOKEN);
  const unsigned threads = 32u * a.warps * groups;
  TC_CUDA_OK(launch_chained(true, b.kernel, dim3((unsigned)*blocks), threads, (size_t)b.per_thread * threads, stream, a));
  return TC_OK;
}

template <class T>
int forward(const TcOpShape& p, NormArgs a, bool vec, cudaStream_t stream) {
  if (p.dim > kForward) {
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_kernel<T, true> : norm_long_kernel<T, false>, dim3((unsigned)a.tokens), kLongThreads, 0, stream, a));
    return TC_OK;
  }
  const int groups = groups_of(warps_of(p.dim, pieces_of(p, false)));
  int64_t blocks = std::min<int64_t>(most_blocks(p, false), (a.tokens + groups - 1) / groups);
  return launch<T>(p, a, false, vec, &blocks, stream);
}

template <class T>
int backward(const TcOpShape& p, NormArgs a, const Buffers& b, bool vec, void* dpost, void* dpre, cudaStream_t stream) {
  void* shared_gate = p.gate == TC_GATE_CHANNEL ? a.dgate : nullptr;
  const bool sums = dpost || dpre || shared_gate;
  a.pitch = pitch_of(p);
  a.part = sums ? b.part : nullptr;
  int64_t slots = most_slots(p);
  if (p.dim > longest_backward(p)) {
    slots = std::min<int64_t>(slots, a.tokens);
    a.slots = (uint32_t)slots;
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_sums_kernel<T, true> : norm_long_sums_kernel<T, false>, dim3((unsigned)a.tokens), kLongThreads, 0, stream, a, b.sums));
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_grad_kernel<T, true> : norm_long_grad_kernel<T, false>, dim3((unsigned)((p.dim + 1023) / 1024), a.slots), 128u, 0, stream, a,
                              b.sums));
  } else {
    const int groups = groups_of(warps_of(p.dim, pieces_of(p, true)));
    slots = std::min<int64_t>(slots, (a.tokens + groups - 1) / groups);
    const int st = launch<T>(p, a, true, vec, &slots, stream);
    if (st != TC_OK) return st;
  }
  if (!sums) return TC_OK;
  const JoinArgs j{b.part, a.gate, a.post, dpost, shared_gate, dpre, p.weight_dtype == TC_F32, p.gate == TC_GATE_CHANNEL, (uint32_t)slots, a.pitch, a.dim};
  TC_CUDA_OK(launch_chained(true, norm_join_kernel<T>, dim3((unsigned)((p.dim + 31) / 32), 2u), 1024u, 0, stream, j));
  return TC_OK;
}

// One argument: a matrix of rows of `cols` elements.
struct Rows {
  const void* ptr;
  int64_t ld;
  bool written;
};
int check(const tc_op_plan* p, int64_t tokens, const Rows* rows, int count, const void* const* weights, int n_weights, bool* vec) {
  const int es = tc_elem_bytes(p->dtype), wes = tc_elem_bytes(p->weight_dtype);
  *vec = true;
  for (int i = 0; i < count; ++i) {
    if (!rows[i].ptr) continue;
    if (rows[i].ld < (rows[i].written ? p->dim : 0)) return TC_ERR_EXTENT;
    if (tc_odd_address(rows[i].ptr, es)) return TC_ERR_ALIGNMENT;
    *vec = *vec && tc_vec8(rows[i].ptr, tokens > 1 ? rows[i].ld : p->dim, p->dim, es);
  }
  for (int i = 0; i < n_weights; ++i) {
    if (tc_odd_address(weights[i], wes)) return TC_ERR_ALIGNMENT;
    *vec = *vec && !tc_odd_address(weights[i], 16);
  }
  return TC_OK;
}

NormArgs base_args(const tc_op_plan& p, int64_t tokens) {
  NormArgs a{};
  a.tokens = tokens;
  a.dim = (uint32_t)p.dim;
  a.gate_kind = p.gate;
  a.wide = p.weight_dtype == TC_F32 && p.dtype != TC_F32;
  a.residual = (float)p.scale;
  a.inverse_dim = (float)(1.0 / (double)p.dim);
  a.eps = p.eps;
  return a;
}

}  // namespace

size_t tc_norm_workspace(const TcOpShape& p) {
  Buffers b;
  return carve(p, nullptr, &b);
}

int tc_norm_prepare() {
  for (int st : {prepare<float>(), prepare<__nv_bfloat16>(), prepare<__half>()})
    if (st != TC_OK) return st;
  return TC_OK;
}

std::string tc_norm_json(const TcOpShape& p) {
  static const char* const gates[] = {"none", "channel", "token"};
  return "{\"operator\":\"residual_norm\",\"dtype\":\"" + tc_type_name(p.dtype) + "\",\"tokens\":" + std::to_string(p.tokens) + ",\"dim\":" + std::to_string(p.dim) +
         ",\"gate\":\"" + gates[p.gate] + "\",\"workspace_bytes\":" + std::to_string(tc_norm_workspace(p)) + "}";
}

extern "C" int tc_residual_norm_execute(tc_op_plan* p, void* h, int64_t ld_h, void* n, int64_t ld_n, const void* x, int64_t ld_x, const void* f, int64_t ld_f, const void* post,
                                        const void* pre, const void* gate, int64_t ld_gate, int64_t tokens, void* stream) {
  if (!p || p->kind != TC_OP_RESIDUAL_NORM || (tokens && (!h || !x || !f)) || (p->gate != TC_GATE_NONE) != (gate != nullptr)) return TC_ERR_INVALID_ARG;
  if (tokens < 0 || tokens > p->tokens) return TC_ERR_EXTENT;
  const Rows rows[] = {{h, ld_h, true}, {n, ld_n, true}, {x, ld_x, false}, {f, ld_f, false}, {gate, p->gate == TC_GATE_TOKEN ? ld_gate : p->dim, false}};
  const void* const weights[] = {post, pre};
  bool vec;
  int st = check(p, tokens, rows, 5, weights, 2, &vec);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (st == TC_OK) st = tc_op_ready(p, s);
  if (st != TC_OK || tokens == 0) return st;
  NormArgs a = base_args(*p, tokens);
  a.h = h; a.ld_h = ld_h;
  a.n = n; a.ld_n = ld_n;
  a.x = x; a.ld_x = ld_x;
  a.f = f; a.ld_f = ld_f;
  a.post = post; a.pre = pre;
  a.gate = gate; a.ld_gate = ld_gate;
  switch (p->dtype) {
    case TC_F32: return forward<float>(*p, a, vec, s);
    case TC_BF16: return forward<__nv_bfloat16>(*p, a, vec, s);
    default: return forward<__half>(*p, a, vec, s);
  }
}

extern "C" int tc_residual_norm_execute_grad(tc_op_plan* p, void* dx, int64_t ld_dx, void* df, int64_t ld_df, void* dgate, int64_t ld_dgate, void* dpost, void* dpre,
                                             const void* dh, int64_t ld_dh, const void* dn, int64_t ld_dn, const void* h, int64_t ld_h, const void* f, int64_t ld_f,
                                             const void* post, const void* pre, const void* gate, int64_t ld_gate, int64_t tokens, void* workspace, size_t workspace_bytes,
                                             void* stream) {
  if (!p || p->kind != TC_OP_RESIDUAL_NORM || (tokens && (!h || !f || (!dh && !dn))) || (p->gate != TC_GATE_NONE) != (gate != nullptr)) return TC_ERR_INVALID_ARG;
  if ((!dx && !df && !dgate && !dpost && !dpre) || (dgate && p->gate == TC_GATE_NONE)) return TC_ERR_INVALID_ARG;
  if (tokens < 0 || tokens > p->tokens) return TC_ERR_EXTENT;
  const bool by_token = p->gate == TC_GATE_TOKEN;
  const Rows rows[] = {{dx, ld_dx, true}, {df, ld_df, true}, {dgate, by_token ? ld_dgate : p->dim, true}, {dh, ld_dh, false}, {dn, ld_dn, false}, {h, ld_h, false},
                       {f, ld_f, false}, {gate, by_token ? ld_gate : p->dim, false}};
  const void* const weights[] = {post, pre, dpost, dpre};
  bool vec;
  int st = check(p, tokens, rows, 8, weights, 4, &vec);
  if (st != TC_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  TcScratch scratch;
  st = scratch.open(p, TC_OP_RESIDUAL_NORM, workspace, workspace_bytes, s);
  if (st != TC_OK) return st;
  if (tokens == 0) {  // no tokens: sums over them are zeros
    const size_t wes = (size_t)tc_elem_bytes(p->weight_dtype) * p->dim;
    if (dpost) TC_CUDA_OK(cudaMemsetAsync(dpost, 0, wes, s));
    if (dpre) TC_CUDA_OK(cudaMemsetAsync(dpre, 0, wes, s));
    if (dgate && !by_token) TC_CUDA_OK(cudaMemsetAsync(dgate, 0, (size_t)tc_elem_bytes(p->dtype) * p->dim, s));
    return TC_OK;
  }
  Buffers b;
  carve(*p, scratch.base, &b);
  NormArgs a = base_args(*p, tokens);
  a.dx = dx; a.ld_dx = ld_dx;
  a.df = df; a.ld_df = ld_df;
  a.dgate = dgate; a.ld_dgate = ld_dgate;
  a.dh = dh; a.ld_dh = ld_dh;
  a.dn = dn; a.ld_dn = ld_dn;
  a.h = const_cast<void*>(h); a.ld_h = ld_h;
  a.f = f; a.ld_f = ld_f;
  a.post = post; a.pre = pre;
  a.gate = gate; a.ld_gate = ld_gate;
  switch (p->dtype) {
    case TC_F32: return scratch.close(backward<float>(*p, a, b, vec, dpost, dpre, s));
    case TC_BF16: return scratch.close(backward<__nv_bfloat16>(*p, a, b, vec, dpost, dpre, s));
    default: return scratch.close(backward<__half>(*p, a, b, vec, dpost, dpre, s));
  }
}

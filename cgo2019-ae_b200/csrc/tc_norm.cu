// A block's result onto the residual stream, and the norm before the next block (tc_residual_norm_*).
//
//   u = f r, r = (mean f^2 + eps)^-1/2      h = s x + g (u post)      n = h q pre, q = (mean h^2 + eps)^-1/2
//
// and backward, at h as it was stored, with v = h q and means over a row:
//
//   dh' = dh + q (dn pre - v mean(dn pre v))    dx = s dh'     dp = dh' g     df = r (dp post - u mean(dp post u))
//   dg = dh' u post (summed over tokens where they share the gate)    dpost = sum dp u    dpre = sum dn v
//
// Both directions read every row once: a group of warps holds it in registers, eight neighbouring elements a thread and piece.
// Backward a group takes row after row and keeps the sums over tokens of its columns in registers too; groups' sums are joined in
// order by a second launch, so that results do not depend on which group ran when.  Rows of more than 8192 (backward) or 16384
// elements are read again for each of the steps between row sums.
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
  float* part;             // [3][slots][pitch]: dpost, dpre, dgate of tokens that share it
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
__device__ __forceinline__ double squares8(const float* f, int valid) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < valid) s = fmaf(f[k], f[k], s);
  if (!out_of_range(s)) return (double)s;
  double d = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < valid) d = fma((double)f[k], (double)f[k], d);
  return d;
}

// ---- what a row is multiplied by ----
template <class T, bool Vec>
__device__ __forceinline__ void weight8(const void* w, uint32_t col, int valid, bool wide, float* f) {
  if (!w) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 1.f;
  } else if (wide) {
    unpack8<float>(load8<float, Vec>(static_cast<const float*>(w) + col, valid), f);
  } else {
    unpack8<T>(load8<T, Vec>(static_cast<const T*>(w) + col, valid), f);
  }
}
template <class T, bool Vec>
__device__ __forceinline__ void gate8(const NormArgs& a, int64_t row, uint32_t col, int valid, float* f) {
  if (a.gate_kind == TC_GATE_NONE) weight8<T, Vec>(nullptr, col, valid, false, f);
  else unpack8<T>(load8<T, Vec>(static_cast<const T*>(a.gate) + (a.gate_kind == TC_GATE_TOKEN ? row * a.ld_gate : 0) + col, valid), f);
}
template <class T, bool Vec>
__device__ __forceinline__ Raw<T> row8(const void* p, int64_t ld, int64_t row, uint32_t col, int valid) {
  return load8<T, Vec>(static_cast<const T*>(p) + row * ld + col, valid);
}
template <class T, bool Vec>
__device__ __forceinline__ void put8(void* p, int64_t ld, int64_t row, uint32_t col, int valid, const float* f) {
  store8<T, Vec>(static_cast<T*>(p) + row * ld + col, pack8<T>(f), valid);
}

// ---- forward ----
template <class T, bool Vec, int V>
__global__ void __launch_bounds__(32 * kMostWarps) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(a.warps);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / (32 * a.warps)) + g.id;
  chain_wait();
  if (row >= a.tokens) return;  // the whole group
  Raw<T> rx[V], rf[V];
  uint32_t col[V];
  int valid[V];
#pragma unroll
  for (int p = 0; p < V; ++p) {
    col[p] = (uint32_t)(p * a.warps * 32 + g.thread) * 8;
    valid[p] = (int)a.dim - (int)col[p];
    rf[p] = row8<T, Vec>(a.f, a.ld_f, row, col[p], valid[p]);
  }
#pragma unroll
  for (int p = 0; p < V; ++p) rx[p] = row8<T, Vec>(a.x, a.ld_x, row, col[p], valid[p]);
  auto squares = [&]() {
    double d = 0;
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float f[8];
      unpack8<T>(rf[p], f);
      d += squares8(f, 8);
    }
    return d;
  };
  float s = 0.f;
#pragma unroll
  for (int p = 0; p < V; ++p) {
    float f[8];
    unpack8<T>(rf[p], f);
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(f[k], f[k], s);
  }
  const float r = root_of(g, a, s, shared, 0, squares);
  float h[V][8];
  s = 0.f;
#pragma unroll
  for (int p = 0; p < V; ++p) {
    float f[8], w[8];
    unpack8<T>(rx[p], h[p]);
    unpack8<T>(rf[p], f);
    weight8<T, Vec>(a.post, col[p], valid[p], a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = f[k] * r * w[k];
    gate8<T, Vec>(a, row, col[p], valid[p], w);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      h[p][k] = fmaf(w[k], f[k], a.residual * h[p][k]);
      if (k < valid[p]) s = fmaf(h[p][k], h[p][k], s);  // what lies behind the row is no number of it
    }
    put8<T, Vec>(a.h, a.ld_h, row, col[p], valid[p], h[p]);
  }
  if (!a.n) return;
  const float q = root_of(g, a, s, shared, 1, [&]() {
    double d = 0;
#pragma unroll
    for (int p = 0; p < V; ++p) d += squares8(h[p], valid[p]);
    return d;
  });
#pragma unroll
  for (int p = 0; p < V; ++p) {
    float w[8];
    weight8<T, Vec>(a.pre, col[p], valid[p], a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[p][k] = h[p][k] * q * w[k];
    put8<T, Vec>(a.n, a.ld_n, row, col[p], valid[p], h[p]);
  }
}

// Rows too long for registers: h is computed a second time for n.
template <class T, bool Vec>
__global__ void __launch_bounds__(32 * kMostWarps) norm_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(kMostWarps);
  const int64_t row = blockIdx.x;
  chain_wait();
  double s[1] = {0};
  for (uint32_t col = g.thread * 8; col < a.dim; col += 32 * kMostWarps * 8) {
    float f[8];
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, col, (int)(a.dim - col)), f);
    s[0] += squares8(f, 8);
  }
  group_sum(g, s, shared, 0);
  const float r = inverse_root(s[0], a);
  auto residual = [&](uint32_t col, int valid, float* h) {
    float f[8], w[8];
    unpack8<T>(row8<T, Vec>(a.x, a.ld_x, row, col, valid), h);
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, col, valid), f);
    weight8<T, Vec>(a.post, col, valid, a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = f[k] * r * w[k];
    gate8<T, Vec>(a, row, col, valid, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = fmaf(w[k], f[k], a.residual * h[k]);
  };
  s[0] = 0;
  for (uint32_t col = g.thread * 8; col < a.dim; col += 32 * kMostWarps * 8) {
    const int valid = (int)(a.dim - col);
    float h[8];
    residual(col, valid, h);
    put8<T, Vec>(a.h, a.ld_h, row, col, valid, h);
    s[0] += squares8(h, valid);
  }
  if (!a.n) return;
  group_sum(g, s, shared, 1);
  const float q = inverse_root(s[0], a);
  for (uint32_t col = g.thread * 8; col < a.dim; col += 32 * kMostWarps * 8) {
    const int valid = (int)(a.dim - col);
    float h[8], w[8];
    residual(col, valid, h);
    weight8<T, Vec>(a.pre, col, valid, a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = h[k] * q * w[k];
    put8<T, Vec>(a.n, a.ld_n, row, col, valid, h);
  }
}

// ---- backward ----
// Eight columns of a row once its sums are known; adds to the columns' own sums.
struct RowSums {
  float r, q, c2, c1;  // c2: mean(dn pre v), c1: mean(dp post u)
};
// dh' of eight columns, and v.
template <class T, bool Vec>
__device__ __forceinline__ void stream8(const NormArgs& a, const Raw<T>& rh, const Raw<T>& rdh, const float* dnw, const RowSums& t, float* dh, float* v) {
  unpack8<T>(rh, v);
  unpack8<T>(rdh, dh);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    v[k] *= t.q;
    dh[k] = fmaf(t.q, fmaf(-v[k], t.c2, dnw[k]), dh[k]);
  }
}

template <class T, bool Vec, int V>
__global__ void __launch_bounds__(32 * kMostWarps) norm_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(a.warps);
  const uint32_t groups = blockDim.x / (32 * a.warps), slot = blockIdx.x * groups + g.id;
  float dpost[V][8] = {}, dpre[V][8] = {}, dgate[V][8] = {};
  chain_wait();
  for (int64_t row = slot; row < a.tokens; row += a.slots) {
    Raw<T> rf[V], rh[V], rdn[V], rdh[V];
    uint32_t col[V];
    int valid[V];
#pragma unroll
    for (int p = 0; p < V; ++p) {
      col[p] = (uint32_t)(p * a.warps * 32 + g.thread) * 8;
      valid[p] = (int)a.dim - (int)col[p];
      rf[p] = row8<T, Vec>(a.f, a.ld_f, row, col[p], valid[p]);
      rh[p] = row8<T, Vec>(a.h, a.ld_h, row, col[p], valid[p]);
      rdn[p] = row8<T, Vec>(a.dn, a.ld_dn, row, col[p], a.dn ? valid[p] : 0);
      rdh[p] = row8<T, Vec>(a.dh, a.ld_dh, row, col[p], a.dh ? valid[p] : 0);
    }
    auto sums = [&](auto* s) {  // f^2, h^2, dn pre h
      using S = std::remove_reference_t<decltype(*s)>;
      s[0] = s[1] = s[2] = 0;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        float f[8], h[8], dn[8], w[8];
        unpack8<T>(rf[p], f);
        unpack8<T>(rh[p], h);
        unpack8<T>(rdn[p], dn);
        weight8<T, Vec>(a.pre, col[p], valid[p], a.wide, w);
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
    float c1[1] = {0.f};
    Raw<T> rgate[V];
    float dpw[V][8];
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float dn[8], w[8], dh[8], v[8], u[8], gate[8];
      unpack8<T>(rdn[p], dn);
      weight8<T, Vec>(a.pre, col[p], valid[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] *= dn[k];
      stream8<T, Vec>(a, rh[p], rdh[p], w, t, dh, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) dpre[p][k] = fmaf(dn[k], v[k], dpre[p][k]);
      unpack8<T>(rf[p], u);
      gate8<T, Vec>(a, row, col[p], valid[p], gate);
      weight8<T, Vec>(a.post, col[p], valid[p], a.wide, w);
      float dg[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        u[k] *= t.r;
        const float dp = dh[k] * gate[k];
        dpost[p][k] = fmaf(dp, u[k], dpost[p][k]);
        dg[k] = dh[k] * u[k] * w[k];
        dgate[p][k] += dg[k];
        dpw[p][k] = dp * w[k];
        if (k < valid[p]) c1[0] = fmaf(dpw[p][k], u[k], c1[0]);
        dh[k] *= a.residual;
      }
      if (a.dx) put8<T, Vec>(a.dx, a.ld_dx, row, col[p], valid[p], dh);
      if (a.dgate && a.gate_kind == TC_GATE_TOKEN) put8<T, Vec>(a.dgate, a.ld_dgate, row, col[p], valid[p], dg);
    }
    if (!a.df) continue;
    group_sum(g, c1, shared, 1);
    const float mean = c1[0] * a.inverse_dim;
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float u[8];
      unpack8<T>(rf[p], u);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = t.r * fmaf(-u[k] * t.r, mean, dpw[p][k]);
      put8<T, Vec>(a.df, a.ld_df, row, col[p], valid[p], u);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int p = 0; p < V; ++p) {
    const uint32_t col = (uint32_t)(p * a.warps * 32 + g.thread) * 8;
    if (col >= a.dim) continue;  // rows of the sums are filled up to a multiple of eight
    float* to = a.part + (size_t)slot * a.pitch + col;
    const size_t next = (size_t)a.slots * a.pitch;
    store8<float, true>(to, pack8<float>(dpost[p]), 8);
    store8<float, true>(to + next, pack8<float>(dpre[p]), 8);
    store8<float, true>(to + 2 * next, pack8<float>(dgate[p]), 8);
  }
}

// Rows too long for registers: their sums first ...
template <class T, bool Vec>
__global__ void __launch_bounds__(32 * kMostWarps) norm_long_sums_kernel(const __grid_constant__ NormArgs a, RowSums* out) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const Group g(kMostWarps);
  const int64_t row = blockIdx.x;
  constexpr uint32_t kStep = 32 * kMostWarps * 8;
  chain_wait();
  double s[3] = {0, 0, 0};
  auto scaled = [&](uint32_t col, int valid, float* dnw) {
    float w[8];
    unpack8<T>(row8<T, Vec>(a.dn, a.ld_dn, row, col, a.dn ? valid : 0), dnw);
    weight8<T, Vec>(a.pre, col, valid, a.wide, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) dnw[k] *= w[k];
  };
  for (uint32_t col = g.thread * 8; col < a.dim; col += kStep) {
    const int valid = (int)(a.dim - col);
    float f[8], h[8], dnw[8];
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, col, valid), f);
    unpack8<T>(row8<T, Vec>(a.h, a.ld_h, row, col, valid), h);
    scaled(col, valid, dnw);
    s[0] += squares8(f, 8);
    s[1] += squares8(h, 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) s[2] = fma((double)dnw[k], (double)h[k], s[2]);
  }
  group_sum(g, s, shared, 0);
  RowSums t;
  t.r = inverse_root(s[0], a);
  t.q = inverse_root(s[1], a);
  t.c2 = (float)(t.q * s[2] * a.inverse_dim);
  double c1[1] = {0};
  for (uint32_t col = g.thread * 8; col < a.dim; col += kStep) {
    const int valid = (int)(a.dim - col);
    float dnw[8], dh[8], v[8], u[8], w[8], gate[8];
    scaled(col, valid, dnw);
    stream8<T, Vec>(a, row8<T, Vec>(a.h, a.ld_h, row, col, valid), row8<T, Vec>(a.dh, a.ld_dh, row, col, a.dh ? valid : 0), dnw, t, dh, v);
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, col, valid), u);
    weight8<T, Vec>(a.post, col, valid, a.wide, w);
    gate8<T, Vec>(a, row, col, valid, gate);
    float e = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < valid) e = fmaf(dh[k] * gate[k] * w[k], u[k] * t.r, e);
    c1[0] += (double)e;
  }
  group_sum(g, c1, shared, 1);
  t.c1 = (float)(c1[0] * a.inverse_dim);
  if (g.thread == 0) out[row] = t;
}
// ... then 1024 columns a block, every slots-th row.
template <class T, bool Vec>
__global__ void __launch_bounds__(128) norm_long_grad_kernel(const __grid_constant__ NormArgs a, const RowSums* in) {
  const uint32_t col = blockIdx.x * 1024 + threadIdx.x * 8;
  const int valid = (int)(a.dim - col);
  chain_wait();
  if (col >= a.dim) return;
  float dpost[8] = {}, dpre[8] = {}, dgate[8] = {}, post[8], pre[8];
  weight8<T, Vec>(a.post, col, valid, a.wide, post);
  weight8<T, Vec>(a.pre, col, valid, a.wide, pre);
  for (int64_t row = blockIdx.y; row < a.tokens; row += a.slots) {
    const RowSums t = in[row];
    float dn[8], dnw[8], dh[8], v[8], u[8], gate[8], dg[8];
    unpack8<T>(row8<T, Vec>(a.dn, a.ld_dn, row, col, a.dn ? valid : 0), dn);
#pragma unroll
    for (int k = 0; k < 8; ++k) dnw[k] = dn[k] * pre[k];
    stream8<T, Vec>(a, row8<T, Vec>(a.h, a.ld_h, row, col, valid), row8<T, Vec>(a.dh, a.ld_dh, row, col, a.dh ? valid : 0), dnw, t, dh, v);
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, col, valid), u);
    gate8<T, Vec>(a, row, col, valid, gate);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u[k] *= t.r;
      const float dp = dh[k] * gate[k];
      dpre[k] = fmaf(dn[k], v[k], dpre[k]);
      dpost[k] = fmaf(dp, u[k], dpost[k]);
      dg[k] = dh[k] * u[k] * post[k];
      dgate[k] += dg[k];
      u[k] = t.r * fmaf(-u[k], t.c1, dp * post[k]);
      dh[k] *= a.residual;
    }
    if (a.dx) put8<T, Vec>(a.dx, a.ld_dx, row, col, valid, dh);
    if (a.df) put8<T, Vec>(a.df, a.ld_df, row, col, valid, u);
    if (a.dgate && a.gate_kind == TC_GATE_TOKEN) put8<T, Vec>(a.dgate, a.ld_dgate, row, col, valid, dg);
  }
  if (!a.part) return;
  float* to = a.part + (size_t)blockIdx.y * a.pitch + col;
  const size_t next = (size_t)a.slots * a.pitch;
  store8<float, true>(to, pack8<float>(dpost), 8);
  store8<float, true>(to + next, pack8<float>(dpre), 8);
  store8<float, true>(to + 2 * next, pack8<float>(dgate), 8);
}

// Sums over tokens: 32 columns a block, each eighth slot a warp, warps in order.  blockIdx.y: dpost, dpre, dgate.
struct JoinArgs {
  const float* part;
  void* out[3];
  int wide[3];
  uint32_t slots, pitch, dim;
};
template <class T>
__global__ void __launch_bounds__(256) norm_join_kernel(const __grid_constant__ JoinArgs a) {
  __shared__ float sums[8][32];
  const uint32_t col = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  chain_wait();
  if (!a.out[blockIdx.y]) return;
  const float* from = a.part + (size_t)blockIdx.y * a.slots * a.pitch + col;
  float s = 0.f;
  if (col < a.dim)
    for (uint32_t i = warp; i < a.slots; i += 8) s += from[(size_t)i * a.pitch];
  sums[warp][threadIdx.x & 31] = s;
  __syncthreads();
  if (warp > 0 || col >= a.dim) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
  if (a.wide[blockIdx.y]) static_cast<float*>(a.out[blockIdx.y])[col] = s;
  else static_cast<T*>(a.out[blockIdx.y])[col] = Elem<T>::put(s);
}

// ---- launches ----
constexpr int64_t kForward = 16384, kBackward = 8192;  // longest rows that stay in registers

int warps_of(int64_t dim, int pieces) {  // that hold a row of `pieces` pieces a thread
  int w = 1;
  while (w < kMostWarps && (int64_t)w * 256 * pieces < dim) w *= 2;
  return w;
}
int pieces_of(int64_t dim) { return dim <= 4096 ? 1 : dim <= 8192 ? 2 : 4; }
int groups_of(int warps) { return warps >= 8 ? 1 : 8 / warps; }
uint32_t pitch_of(const TcOpShape& p) { return (uint32_t)((p.dim + 7) / 8 * 8); }
// Most groups that sum columns of their own.
int64_t most_slots(const TcOpShape& p) {
  if (p.dim > kBackward) return std::min<int64_t>(p.tokens, std::max<int64_t>(1, 16 * (int64_t)p.sms / ((p.dim + 1023) / 1024)));
  const int w = warps_of(p.dim, pieces_of(p.dim));
  return (int64_t)p.sms * (w >= 16 ? 2 : w == 8 ? 4 : 4) * groups_of(w);
}

struct Buffers {
  float* part;
  RowSums* sums;
};
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  TcCarver c{base};
  b->part = c.take<float>((size_t)3 * most_slots(p) * pitch_of(p));
  b->sums = c.take<RowSums>(p.dim > kBackward ? (size_t)p.tokens : 0);
  return c.used;
}

template <class T>
int forward(const TcOpShape& p, NormArgs a, bool vec, cudaStream_t stream) {
  if (p.dim > kForward) {
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_kernel<T, true> : norm_long_kernel<T, false>, dim3((unsigned)a.tokens), 32u * kMostWarps, 0, stream, a));
    return TC_OK;
  }
  const int v = pieces_of(p.dim);
  a.warps = warps_of(p.dim, v);
  const int groups = groups_of(a.warps);
  auto kernel = v == 1 ? (vec ? norm_kernel<T, true, 1> : norm_kernel<T, false, 1>)
                : v == 2 ? (vec ? norm_kernel<T, true, 2> : norm_kernel<T, false, 2>) : (vec ? norm_kernel<T, true, 4> : norm_kernel<T, false, 4>);
  TC_CUDA_OK(launch_chained(true, kernel, dim3((unsigned)((a.tokens + groups - 1) / groups)), 32u * a.warps * groups, 0, stream, a));
  return TC_OK;
}

template <class T>
int backward(const TcOpShape& p, NormArgs a, const Buffers& b, bool vec, void* dpost, void* dpre, cudaStream_t stream) {
  void* shared_gate = p.gate == TC_GATE_CHANNEL ? a.dgate : nullptr;
  const bool sums = dpost || dpre || shared_gate;
  a.pitch = pitch_of(p);
  a.part = sums ? b.part : nullptr;
  const int64_t most = most_slots(p);
  if (p.dim > kBackward) {
    a.slots = (uint32_t)std::min<int64_t>(most, a.tokens);
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_sums_kernel<T, true> : norm_long_sums_kernel<T, false>, dim3((unsigned)a.tokens), 32u * kMostWarps, 0, stream, a, b.sums));
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_grad_kernel<T, true> : norm_long_grad_kernel<T, false>, dim3((unsigned)((p.dim + 1023) / 1024), a.slots), 128u, 0, stream, a,
                              b.sums));
  } else {
    const int v = pieces_of(p.dim);
    a.warps = warps_of(p.dim, v);
    const int groups = groups_of(a.warps);
    const int64_t blocks = std::min<int64_t>(most / groups, (a.tokens + groups - 1) / groups);
    a.slots = (uint32_t)(blocks * groups);
    auto kernel = v == 1 ? (vec ? norm_grad_kernel<T, true, 1> : norm_grad_kernel<T, false, 1>) : (vec ? norm_grad_kernel<T, true, 2> : norm_grad_kernel<T, false, 2>);
    TC_CUDA_OK(launch_chained(true, kernel, dim3((unsigned)blocks), 32u * a.warps * groups, 0, stream, a));
  }
  if (!sums) return TC_OK;
  const int wide = p.weight_dtype == TC_F32;
  const JoinArgs j{b.part, {dpost, dpre, shared_gate}, {wide, wide, 0}, a.slots, a.pitch, a.dim};
  TC_CUDA_OK(launch_chained(true, norm_join_kernel<T>, dim3((unsigned)((p.dim + 31) / 32), 3u), 256u, 0, stream, j));
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

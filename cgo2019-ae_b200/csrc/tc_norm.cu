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
// Both directions read every row once.  A block takes row after row, eight elements a thread and piece, while the next rows are on
// their way to shared memory (cp.async).  Where rows are aligned each thread fetches its own elements, which nobody waits for together,
// and reads them anew for each step; else the row's 16-byte pieces are fetched as they lie, and threads take neighbouring elements one by
// one.  Backward the sums over tokens of a thread's columns stay in registers; blocks' sums are joined in order by a second launch, so
// that results do not depend on which ran when.  Rows of more than 16384 elements (backward 8192, of single precision 4096) are read
// again for each of the steps between row sums.
//
// Arithmetic is two floats at a time (fma.rn.f32x2).
//
// Bound by bytes and by what is issued for them.  One B200, 8192 rows of 4096 bf16, a gate by channel: forward 49 to 51 us (5.5 TB/s), backward 89 (4.5);
// with a gate for each token 58 to 60 and 115.  Rows in registers instead, a thread's eight elements each: 79 and 133; the next row fetched only when
// this one is done 98 and 200.  One row 6.4 us, the host's call.
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
  uint32_t slots, pitch;   // slots: of long rows, else the grid's blocks
  uint32_t dim;
  int gate_kind, wide;     // wide: weights are fp32
  float residual, inverse_dim;
  double eps;
};

// ---- sums over a block's warps ----
// `turn` alternates between two places that share no byte, so that one wait a sum is enough.
constexpr int kMostSums = 3;
template <int N, class S>
__device__ __forceinline__ void block_sum(S (&v)[N], double* shared, int turn) {
  static_assert(N <= kMostSums && kMostWarps == 16, "place, lanes");
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (warps == 1) return;
  S* place = reinterpret_cast<S*>(shared + turn * kMostWarps * kMostSums);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) place[(threadIdx.x >> 5) * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = (lane & 15) < warps ? place[(lane & 15) * N + i] : S(0);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}
// Sums of squares or products that left 32 bits on either side are taken again in 64.
__device__ __forceinline__ bool out_of_range(float s) { return !(s > 1e-30f && s < INFINITY); }
__device__ __forceinline__ float inverse_root(float sum, const NormArgs& a) {
  const float m = fmaf(sum, a.inverse_dim, (float)a.eps), r = rsqrtf(m);
  return fmaf(r, fmaf(-0.5f * m * r, r, 0.5f), r);  // one Newton step
}
__device__ __forceinline__ float inverse_root(double sum, const NormArgs& a) { return (float)(1.0 / sqrt(sum / a.dim + a.eps)); }
template <class Again>
__device__ __forceinline__ float root_of(const NormArgs& a, float sum, double* shared, int turn, Again again) {
  float s[1] = {sum};
  block_sum(s, shared, turn);
  if (!out_of_range(s[0])) return inverse_root(s[0], a);
  __syncthreads();
  double d[1] = {again()};
  block_sum(d, shared, turn);
  __syncthreads();
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
  uint32_t col, step;
  int count;  // how many there are
  __device__ __forceinline__ Where() {}
  __device__ __forceinline__ Where(uint32_t col_, uint32_t step_, uint32_t dim)
      : col(col_), step(step_), count(col_ >= dim ? 0 : Vec ? 8 : (int)min(8u, (dim - col_ + step_ - 1) / step_)) {}
};
// f(k) for each that there is; most threads have all, and a condition on each costs more than the access.
template <bool Vec, class F>
__device__ __forceinline__ void each8(const Where<Vec>& at, F f) {
  if (at.count == 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f(k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < at.count) f(k);
  }
}
template <class T>
__device__ __forceinline__ Raw<T> raw_of(const uint32_t (&w)[8]) {  // an element each
  Raw<T> r;
#pragma unroll
  for (int k = 0; k < Elem<T>::kWords; ++k) r.w[k] = sizeof(T) == 4 ? w[k] : w[2 * k & 7] | w[(2 * k + 1) & 7] << 16;
  return r;
}
template <class T, bool Vec>
__device__ __forceinline__ Raw<T> get8(const T* p, const Where<Vec>& at, bool any = true) {
  if constexpr (Vec) {
    return load8<T, true>(p + at.col, any ? at.count : 0);
  } else {
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (any) {
      if constexpr (sizeof(T) == 4) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p) + at.col;
        each8(at, [&](int k) { w[k] = q[k * at.step]; });
      } else {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + at.col;
        each8(at, [&](int k) { w[k] = q[k * at.step]; });
      }
    }
    return raw_of<T>(w);
  }
}
template <class T, bool Vec, class F>
__device__ __forceinline__ void put8(T* p, const Where<Vec>& at, const F& f) {
  const Raw<T> r = pack8<T>(f);
  if constexpr (Vec) {
    store8<T, true>(p + at.col, r, at.count);
  } else if constexpr (sizeof(T) == 4) {
    uint32_t* q = reinterpret_cast<uint32_t*>(p) + at.col;
    each8(at, [&](int k) { q[k * at.step] = r.w[k]; });
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p) + at.col;
    each8(at, [&](int k) { q[k * at.step] = (uint16_t)(r.w[k >> 1] >> (16 * (k & 1))); });
  }
}
__device__ __forceinline__ void ones8(float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = 1.f;
}
__device__ __forceinline__ void ones8(F2 (&f)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = f2(1.f);
}
// Plain: there are weights, of the rows' type.
template <class T, bool Vec, bool Plain = false, class F>
__device__ __forceinline__ void weight8(const void* w, const Where<Vec>& at, bool wide, F& f) {
  if constexpr (Plain) {
    unpack8<T>(get8<T, Vec>(static_cast<const T*>(w), at), f);
  } else if (!w) {
    ones8(f);
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
template <class T, bool Vec, class F>
__device__ __forceinline__ void put_row8(void* p, int64_t ld, int64_t row, const Where<Vec>& at, const F& f) {
  put8<T, Vec>(static_cast<T*>(p) + row * ld, at, f);
}
// A gate that is the same for all tokens, or none; a token's own comes with its row.
template <class T, bool Vec>
__device__ __forceinline__ void gate8(const NormArgs& a, int64_t row, const Where<Vec>& at, float (&f)[8]) {
  if (a.gate_kind == TC_GATE_TOKEN) unpack8<T>(row8<T, Vec>(a.gate, a.ld_gate, row, at), f);
  else weight8<T, Vec>(a.gate, at, false, f);
}

// N matrices whose rows a block takes one after another, the next ones on their way to shared memory.  Vec: each thread fetches its own
// elements, up to four rows ahead.  Else the row's whole 16-byte pieces, as they lie in memory, and the elements before and behind
// those through a register; the block waits together before it reads.
template <class T, bool Vec, int V, int N>
struct Ahead {
  static constexpr int kBytes = V * N * 8 * (int)sizeof(T);                            // of a thread and row
  static constexpr int kStages = !Vec ? 1 : kBytes <= 32 ? 4 : kBytes <= (N >= 4 ? 128 : 64) ? 2 : 1;  // where there are several at most 128 KB a multiprocessor, and L1 for the weights; one of three matrices, V = 4, of floats takes 192
  static constexpr int kPieces = 8 * (int)sizeof(T) / 16;
  static constexpr int kEdge = 16 / (int)sizeof(T);  // most elements of a 16-byte piece that are the row's
  const void* from[N];
  int64_t ld[N];
  Where<Vec> at[V];
  uint32_t place, stride;  // of the thread's first 16 bytes, between one thread's pieces; or of the first row, between those of a matrix each
  uint32_t edge[Vec ? 1 : N];
  Raw<T> held[Vec ? 1 : N][Vec ? 1 : V];
  int64_t tokens;
  uint32_t dim;

  static __host__ __device__ uint32_t row_bytes(int64_t dim) { return (uint32_t)((dim * (int)sizeof(T) + 30) / 16 * 16); }  // anywhere in 16-byte pieces
  __device__ __forceinline__ void start(unsigned char* ring, const NormArgs& a) {
    tokens = a.tokens;
    dim = a.dim;
#pragma unroll
    for (int p = 0; p < V; ++p)
      at[p] = Vec ? Where<Vec>((p * blockDim.x + threadIdx.x) * 8, 1u, a.dim) : Where<Vec>(p * blockDim.x * 8 + threadIdx.x, blockDim.x, a.dim);
    place = smem_u32(ring) + (Vec ? threadIdx.x * 16 : 0u);
    stride = Vec ? blockDim.x * 16 : row_bytes(dim);
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(s, (int64_t)blockIdx.x + s * (int64_t)gridDim.x);
  }
  __device__ __forceinline__ const unsigned char* row_of(int i, int64_t row) const { return static_cast<const unsigned char*>(from[i]) + row * ld[i] * (int64_t)sizeof(T); }
  // The element of the row that this thread carries through a register, or -1: the first threads those before the first whole piece, the
  // next those behind the last.
  __device__ __forceinline__ int64_t carried(uint32_t shift) const {
    const uint32_t end = shift + dim * (uint32_t)sizeof(T), head = shift == 0 ? 0u : min(dim, (16u - shift) / (uint32_t)sizeof(T));
    if (threadIdx.x < head) return threadIdx.x;
    const uint32_t tail = end / 16 == 0 && shift != 0 ? 0u : end % 16 / (uint32_t)sizeof(T), k = threadIdx.x - kEdge;
    return threadIdx.x >= (uint32_t)kEdge && k < tail ? (int64_t)dim - tail + k : -1;
  }
  __device__ __forceinline__ void fetch(int stage, int64_t row) {
    if (row < tokens) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!from[i]) continue;
        const unsigned char* src = row_of(i, row);
        if constexpr (Vec) {
#pragma unroll
          for (int p = 0; p < V; ++p)
            if (at[p].count)
#pragma unroll
              for (int q = 0; q < kPieces; ++q) cp_async16(place + (((stage * N + i) * V + p) * kPieces + q) * stride, src + at[p].col * (uint32_t)sizeof(T) + q * 16, true);
        } else {
          const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(src) & 15u;
          const uint32_t whole = (shift + dim * (uint32_t)sizeof(T)) / 16;  // pieces that end inside the row; the first begins there if nothing is shifted
          for (uint32_t c = threadIdx.x + (shift ? 1u : 0u); c < whole; c += blockDim.x) cp_async16(place + i * stride + c * 16, src - shift + c * 16, true);
          const int64_t e = carried(shift);
          if (e >= 0) edge[i] = sizeof(T) == 4 ? reinterpret_cast<const uint32_t*>(src)[e] : reinterpret_cast<const uint16_t*>(src)[e];
        }
      }
    }
    cp_async_commit();
  }
  // The block's row number n, row `row` of the matrices, is there.
  __device__ __forceinline__ void take(int64_t row) {
    if constexpr (Vec) {
      cp_async_wait<kStages - 1>();
    } else {
      uint32_t shift[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        shift[i] = (uint32_t)reinterpret_cast<uintptr_t>(row_of(i, row)) & 15u;
        const int64_t e = from[i] ? carried(shift[i]) : -1;
        if (e >= 0) {
          const uint32_t to = place + i * stride + shift[i] + (uint32_t)e * (uint32_t)sizeof(T);
          if constexpr (sizeof(T) == 4) asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(to), "r"(edge[i]) : "memory");
          else asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(to), "h"((uint16_t)edge[i]) : "memory");
        }
      }
      cp_async_wait<0>();
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int p = 0; p < V; ++p) {
          const uint32_t base = place + i * stride + shift[i] + at[p].col * (uint32_t)sizeof(T);
          uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          if (from[i])
            each8(at[p], [&](int k) {
              if constexpr (sizeof(T) == 4) {
                asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(w[k]) : "r"(base + k * at[p].step * 4) : "memory");
              } else {
                uint16_t h;
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(h) : "r"(base + k * at[p].step * 2) : "memory");
                w[k] = h;
              }
            });
          held[i][p] = raw_of<T>(w);
        }
    }
  }
  // Piece p of matrix i's row in stage `stage`, by take's order.
  __device__ __forceinline__ Raw<T> get(int i, int p, int stage) const {
    if constexpr (Vec) {
      Raw<T> r;
      const bool there = from[i] && at[p].count;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                : "r"(place + (((stage * N + i) * V + p) * kPieces + q) * stride) : "memory");
        r.w[4 * q] = v.x; r.w[4 * q + 1] = v.y; r.w[4 * q + 2] = v.z; r.w[4 * q + 3] = v.w;
      }
      return r;
    } else {
      return held[i][p];
    }
  }
  // The row that takes this one's place.  Not Vec: once the whole block has taken it.
  __device__ __forceinline__ void next(int stage, int64_t row) { fetch(stage, row + kStages * (int64_t)gridDim.x); }
};

// ByToken: a gate of its own for each token.  Plain: both weights and a gate are given, of the rows' type.
template <class T, bool Vec, int V, bool ByToken, bool Plain>
__global__ void __launch_bounds__(32 * kMostWarps) norm_kernel(const __grid_constant__ NormArgs a) {
  constexpr int N = ByToken ? 3 : 2;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ double shared[2 * kMostWarps * kMostSums];
  Ahead<T, Vec, V, N> rows;
  rows.from[0] = a.f; rows.ld[0] = a.ld_f;
  rows.from[1] = a.x; rows.ld[1] = a.ld_x;
  if constexpr (ByToken) { rows.from[N - 1] = a.gate; rows.ld[N - 1] = a.ld_gate; }
  chain_wait();
  rows.start(ring, a);
  int stage = 0;
  for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x) {
    rows.take(row);
    F2 part = f2(0.f);
#pragma unroll
    for (int p = 0; p < V; ++p) {
      F2 f[4];
      unpack8<T>(rows.get(0, p, stage), f);
#pragma unroll
      for (int k = 0; k < 4; ++k) part = fma2(f[k], f[k], part);
    }
    const float r = root_of(a, sum2(part), shared, 0, [&]() {
      double d = 0;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        float f[8];
        unpack8<T>(rows.get(0, p, stage), f);
        d += squares8(f);
      }
      return d;
    });
    F2 h[V][4];
    part = f2(0.f);
#pragma unroll
    for (int p = 0; p < V; ++p) {
      F2 f[4], w[4];
      unpack8<T>(rows.get(0, p, stage), f);
      weight8<T, Vec, Plain>(a.post, rows.at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = mul2(mul2(f[k], f2(r)), w[k]);
      if constexpr (ByToken) unpack8<T>(rows.get(N - 1, p, stage), w);
      else weight8<T, Vec, Plain>(a.gate, rows.at[p], false, w);
      unpack8<T>(rows.get(1, p, stage), h[p]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[p][k] = fma2(w[k], f[k], mul2(f2(a.residual), h[p][k]));
        part = fma2(h[p][k], h[p][k], part);
      }
      put_row8<T, Vec>(a.h, a.ld_h, row, rows.at[p], h[p]);
    }
    rows.next(stage, row);
    stage = stage + 1 == Ahead<T, Vec, V, N>::kStages ? 0 : stage + 1;
    if (!a.n) {
      __syncthreads();  // the sums' place is free again
      continue;
    }
    const float q = root_of(a, sum2(part), shared, 1, [&]() {
      double d = 0;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 t = of2(h[p][k]);
          v[2 * k] = t.x;
          v[2 * k + 1] = t.y;
        }
        d += squares8(v);
      }
      return d;
    });
#pragma unroll
    for (int p = 0; p < V; ++p) {
      F2 w[4];
      weight8<T, Vec, Plain>(a.pre, rows.at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) h[p][k] = mul2(mul2(h[p][k], f2(q)), w[k]);
      put_row8<T, Vec>(a.n, a.ld_n, row, rows.at[p], h[p]);
    }
  }
}

// The places of a long row: 8 * kLongThreads columns at a time.
constexpr uint32_t kLongThreads = 32 * kMostWarps, kLongStep = kLongThreads * 8;
template <bool Vec>
__device__ __forceinline__ Where<Vec> long_place(const NormArgs& a, uint32_t base) {
  return Vec ? Where<Vec>(base + threadIdx.x * 8, 1u, a.dim) : Where<Vec>(base + threadIdx.x, kLongThreads, a.dim);
}

// Rows too long for registers: h is computed a second time for n.
template <class T, bool Vec>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const int64_t row = blockIdx.x;
  chain_wait();
  double s[1] = {0};
  for (uint32_t base = 0; base < a.dim; base += kLongStep) {
    float f[8];
    unpack8<T>(row8<T, Vec>(a.f, a.ld_f, row, long_place<Vec>(a, base)), f);
    s[0] += squares8(f);
  }
  block_sum(s, shared, 0);
  const float r = inverse_root(s[0], a);
  auto residual = [&](const Where<Vec>& at, float (&h)[8]) {
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
  block_sum(s, shared, 1);
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

template <class T, bool Vec, int V, bool ByToken, bool Plain>
__global__ void __launch_bounds__(32 * kMostWarps) norm_grad_kernel(const __grid_constant__ NormArgs a) {
  constexpr int N = ByToken ? 5 : 4;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ double shared[2 * kMostWarps * kMostSums];
  F2 stream[V][4], dpre[V][4];
#pragma unroll
  for (int p = 0; p < V; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) stream[p][k] = dpre[p][k] = f2(0.f);
  Ahead<T, Vec, V, N> rows;
  rows.from[0] = a.f; rows.ld[0] = a.ld_f;
  rows.from[1] = a.h; rows.ld[1] = a.ld_h;
  rows.from[2] = a.dn; rows.ld[2] = a.ld_dn;
  rows.from[3] = a.dh; rows.ld[3] = a.ld_dh;
  if constexpr (ByToken) { rows.from[N - 1] = a.gate; rows.ld[N - 1] = a.ld_gate; }
  chain_wait();
  rows.start(ring, a);
  int stage = 0;
  for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x) {
    rows.take(row);
    float s[3];  // f^2, h^2, dn pre h
    {
      F2 ff = f2(0.f), hh = f2(0.f), nh = f2(0.f);
#pragma unroll
      for (int p = 0; p < V; ++p) {
        F2 f[4], h[4], dn[4], w[4];
        unpack8<T>(rows.get(0, p, stage), f);
        unpack8<T>(rows.get(1, p, stage), h);
        unpack8<T>(rows.get(2, p, stage), dn);
        weight8<T, Vec, Plain>(a.pre, rows.at[p], a.wide, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          ff = fma2(f[k], f[k], ff);
          hh = fma2(h[k], h[k], hh);
          nh = fma2(mul2(dn[k], w[k]), h[k], nh);
        }
      }
      s[0] = sum2(ff);
      s[1] = sum2(hh);
      s[2] = sum2(nh);
    }
    block_sum(s, shared, 0);
    RowSums t;
    t.r = inverse_root(s[0], a);
    t.q = inverse_root(s[1], a);
    t.c2 = t.q * s[2] * a.inverse_dim;
    // products of dn and h may leave 32 bits where neither's squares do; a dn of zeros then has the same norms as none
    const bool squares = out_of_range(s[0]) || out_of_range(s[1]);
    if (squares || (a.dn && out_of_range(fabsf(s[2])))) {
      __syncthreads();
      double d[3] = {0, 0, 0};
#pragma unroll
      for (int p = 0; p < V; ++p) {
        float f[8], h[8], dn[8], w[8];
        unpack8<T>(rows.get(0, p, stage), f);
        unpack8<T>(rows.get(1, p, stage), h);
        unpack8<T>(rows.get(2, p, stage), dn);
        weight8<T, Vec, Plain>(a.pre, rows.at[p], a.wide, w);
        d[0] += squares8(f);
        d[1] += squares8(h);
        for (int k = 0; k < 8; ++k) d[2] = fma((double)dn[k] * (double)w[k], (double)h[k], d[2]);
      }
      block_sum(d, shared, 0);
      __syncthreads();
      if (squares) {
        t.r = inverse_root(d[0], a);
        t.q = inverse_root(d[1], a);
      }
      t.c2 = (float)(t.q * d[2] * a.inverse_dim);
    }
    if constexpr (!Vec) rows.next(stage, row);
    F2 dpw[V][4], parts = f2(0.f);
#pragma unroll
    for (int p = 0; p < V; ++p) {
      F2 dn[4], w[4], dh[4], v[4], u[4];
      unpack8<T>(rows.get(2, p, stage), dn);
      weight8<T, Vec, Plain>(a.pre, rows.at[p], a.wide, w);
      unpack8<T>(rows.get(1, p, stage), v);
      unpack8<T>(rows.get(3, p, stage), dh);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = mul2(v[k], f2(t.q));
        dh[k] = fma2(f2(t.q), fma2(v[k], f2(-t.c2), mul2(dn[k], w[k])), dh[k]);
        dpre[p][k] = fma2(dn[k], v[k], dpre[p][k]);
      }
      unpack8<T>(rows.get(0, p, stage), u);
      if constexpr (ByToken) unpack8<T>(rows.get(N - 1, p, stage), v);
      else weight8<T, Vec, Plain>(a.gate, rows.at[p], false, v);
      weight8<T, Vec, Plain>(a.post, rows.at[p], a.wide, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        u[k] = mul2(u[k], f2(t.r));
        const F2 dp = mul2(dh[k], v[k]);
        stream[p][k] = fma2(ByToken ? dp : dh[k], u[k], stream[p][k]);
        dpw[p][k] = mul2(dp, w[k]);
        parts = fma2(dpw[p][k], u[k], parts);
        if constexpr (ByToken) v[k] = mul2(mul2(dh[k], u[k]), w[k]);
        dh[k] = mul2(dh[k], f2(a.residual));
      }
      if (a.dx) put_row8<T, Vec>(a.dx, a.ld_dx, row, rows.at[p], dh);
      if (ByToken && a.dgate) put_row8<T, Vec>(a.dgate, a.ld_dgate, row, rows.at[p], v);
    }
    float c1[1] = {sum2(parts)};
    block_sum(c1, shared, 1);
    if (a.df) {
      const float mean = c1[0] * a.inverse_dim;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        F2 u[4];
        unpack8<T>(rows.get(0, p, stage), u);
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = mul2(f2(t.r), fma2(mul2(u[k], f2(t.r)), f2(-mean), dpw[p][k]));
        put_row8<T, Vec>(a.df, a.ld_df, row, rows.at[p], u);
      }
    }
    if constexpr (Vec) rows.next(stage, row);
    stage = stage + 1 == Ahead<T, Vec, V, N>::kStages ? 0 : stage + 1;
  }
  if (!a.part) return;
  float* to = a.part + (size_t)blockIdx.x * a.pitch;
#pragma unroll
  for (int p = 0; p < V; ++p) {
    put8<float, Vec>(to, rows.at[p], stream[p]);
    put8<float, Vec>(to + (size_t)gridDim.x * a.pitch, rows.at[p], dpre[p]);
  }
}

// Rows too long for registers: their sums first ...
template <class T, bool Vec>
__global__ void __launch_bounds__(kLongThreads) norm_long_sums_kernel(const __grid_constant__ NormArgs a, RowSums* out) {
  __shared__ double shared[2 * kMostWarps * kMostSums];
  const int64_t row = blockIdx.x;
  chain_wait();
  double s[3] = {0, 0, 0};
  auto scaled = [&](const Where<Vec>& at, float (&dnw)[8]) {
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
  block_sum(s, shared, 0);
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
  block_sum(c1, shared, 1);
  t.c1 = (float)(c1[0] * a.inverse_dim);
  if (threadIdx.x == 0) out[row] = t;
}
// ... then 1024 columns a block, every slots-th row.
template <class T, bool Vec>
__global__ void __launch_bounds__(128) norm_long_grad_kernel(const __grid_constant__ NormArgs a, const RowSums* in) {
  const Where<Vec> at = Vec ? Where<Vec>(blockIdx.x * 1024 + threadIdx.x * 8, 1u, a.dim) : Where<Vec>(blockIdx.x * 1024 + threadIdx.x, 128u, a.dim);
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
constexpr int64_t kForward = 16384;  // longest rows that blocks hold
int64_t longest_backward(const TcOpShape& p) { return p.dtype == TC_F32 ? 4096 : 8192; }
uint32_t pitch_of(const TcOpShape& p) { return (uint32_t)((p.dim + 7) / 8 * 8); }

// Pieces of eight elements a thread.  Many, since what a row costs beside its elements -- two sums over the block, addresses -- is each
// warp's; as many as registers hold.  One where there are too few rows to fill the device.  Before the loops lost their choice of weights 8192 x 4096
// bf16 took forward 53 us with four and 63 with one, backward 98 with two and 102 with one (now 51 and 90); 4099 x 2051 fp16, unaligned, forward 36 with two
// and 75 with one, backward 86 and 207 (now 36 and 78).
int pieces_of(const TcOpShape& p, bool backward, bool vec, int64_t tokens) {
  const int most = backward ? (p.dtype == TC_F32 ? 1 : 2) : p.dtype == TC_F32 || !vec ? 2 : 4;
  int v = tokens <= 2 * p.sms ? 1 : most;
  while (v > 1 && 128 * v >= p.dim) v /= 2;
  while (4096 * v < p.dim) v *= 2;
  return v;
}
int warps_of(int64_t dim, int pieces) { return (int)((dim + 256 * pieces - 1) / (256 * pieces)); }
// Blocks that take row after row: what a multiprocessor holds, by warps that its registers allow.
int64_t most_blocks(const TcOpShape& p, int warps, int pieces) { return (int64_t)p.sms * std::min(32, std::max(1, warps / warps_of(p.dim, pieces))); }
int64_t blocks_of(const TcOpShape& p, bool backward, bool vec, int pieces, int64_t tokens) {
  const int warps = backward && !(vec && pieces == 1) ? 16 : vec ? (pieces == 4 ? 24 : 32) : 20;
  return std::min(tokens, most_blocks(p, warps, pieces));
}
// Most blocks that sum columns of their own.
int64_t most_slots(const TcOpShape& p) {
  if (p.dim > longest_backward(p)) return std::min<int64_t>(p.tokens, std::max<int64_t>(1, 16 * (int64_t)p.sms / ((p.dim + 1023) / 1024)));
  return std::min<int64_t>(p.tokens, std::max(p.dim <= 4096 ? most_blocks(p, 32, 1) : 0, most_blocks(p, 16, 2)));
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
  int per_thread, rows;  // shared memory: bytes for each thread, or rows
};
template <class T, bool Vec, int V, bool ByToken, bool Plain>
Built built(bool backward) {
  if constexpr (V == 1 || (V == 2 && sizeof(T) == 2)) {
    if (backward) {
      using A = Ahead<T, Vec, V, ByToken ? 5 : 4>;
      return Built{norm_grad_kernel<T, Vec, V, ByToken, Plain>, Vec ? A::kStages * A::kBytes : 0, Vec ? 0 : (ByToken ? 5 : 4)};
    }
  }
  using A = Ahead<T, Vec, V, ByToken ? 3 : 2>;
  return Built{norm_kernel<T, Vec, V, ByToken, Plain>, Vec ? A::kStages * A::kBytes : 0, Vec ? 0 : (ByToken ? 3 : 2)};
}
template <class T, bool Vec, bool ByToken, bool Plain>
Built built(bool backward, int v) {
  return v == 1 ? built<T, Vec, 1, ByToken, Plain>(backward) : v == 2 ? built<T, Vec, 2, ByToken, Plain>(backward) : built<T, Vec, 4, ByToken, Plain>(backward);
}
template <class T, bool Vec, bool ByToken>
Built built(bool backward, int v, bool plain) {
  if constexpr (Vec)
    if (plain) return built<T, Vec, ByToken, true>(backward, v);
  return built<T, Vec, ByToken, false>(backward, v);
}
template <class T>
Built built(bool backward, int v, bool vec, bool by_token, bool plain) {
  return vec ? (by_token ? built<T, true, true>(backward, v, plain) : built<T, true, false>(backward, v, plain))
             : (by_token ? built<T, false, true>(backward, v, plain) : built<T, false, false>(backward, v, plain));
}
constexpr int kMostShared = 200 * 1024;  // three rows of 16383 floats
template <class T>
int prepare() {
  for (int i = 0; i < 48; ++i) {
    const Built b = built<T>(i & 1, 1 << (i >> 4), i & 2, i & 4, i & 8);
    TC_CUDA_OK(cudaFuncSetAttribute(b.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
  }
  return TC_OK;
}
// Returns the number of blocks in *blocks.
template <class T>
int launch(const TcOpShape& p, const NormArgs& a, bool backward, bool vec, int64_t* blocks, cudaStream_t stream) {
  const int v = pieces_of(p, backward, vec, a.tokens);
  const unsigned threads = 32u * warps_of(p.dim, v);
  *blocks = blocks_of(p, backward, vec, v, a.tokens);
  const Built b = built<T>(backward, v, vec, p.gate == TC_GATE_TOKEN, a.post && a.pre && a.gate && !a.wide);
  const size_t shared = b.rows ? (size_t)b.rows * Ahead<T, false, 1, 1>::row_bytes(p.dim) : (size_t)b.per_thread * threads;
  TC_CUDA_OK(launch_chained(true, b.kernel, dim3((unsigned)*blocks), threads, shared, stream, a));
  return TC_OK;
}

template <class T>
int forward(const TcOpShape& p, NormArgs a, bool vec, cudaStream_t stream) {
  if (p.dim > kForward) {
    TC_CUDA_OK(launch_chained(true, vec ? norm_long_kernel<T, true> : norm_long_kernel<T, false>, dim3((unsigned)a.tokens), kLongThreads, 0, stream, a));
    return TC_OK;
  }
  int64_t blocks;
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
  bool written, gate;
};
struct Vector {
  const void* ptr;
  bool written;
};
template <int N, int M>
int check(const tc_op_plan* p, int64_t tokens, const Rows (&rows)[N], const Vector (&weights)[M], bool by_token, bool* vec) {
  const int es = tc_elem_bytes(p->dtype), wes = tc_elem_bytes(p->weight_dtype);
  *vec = true;
  for (int i = 0; i < N; ++i) {
    if (!rows[i].ptr) continue;
    if (rows[i].ld < (rows[i].written ? p->dim : 0)) return TC_ERR_EXTENT;
    if (tc_odd_address(rows[i].ptr, es)) return TC_ERR_ALIGNMENT;
    *vec = *vec && tc_vec8(rows[i].ptr, tokens > 1 ? rows[i].ld : p->dim, p->dim, es);
  }
  for (const Vector& w : weights) {
    if (tc_odd_address(w.ptr, wes)) return TC_ERR_ALIGNMENT;
    *vec = *vec && !tc_odd_address(w.ptr, 16);
  }
  // Long rows are read again after their result was written, sums over tokens are scaled by weights behind it: a result over an argument would be
  // wrong there, and is refused at every size.
  TcSpan spans[N + M];
  for (int i = 0; i < N; ++i) {
    const bool vector = rows[i].gate && !by_token;
    spans[i] = TcSpan{rows[i].ptr, rows[i].ld * es, p->dim * es, vector ? 1 : tokens, rows[i].written};
  }
  for (int i = 0; i < M; ++i) spans[N + i] = TcSpan{weights[i].ptr, 0, p->dim * wes, 1, weights[i].written};
  return tc_results_overlap(spans) ? TC_ERR_INVALID_ARG : TC_OK;
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
  const bool by_token = p->gate == TC_GATE_TOKEN;
  const Rows rows[] = {{h, ld_h, true, false}, {n, ld_n, true, false}, {x, ld_x, false, false}, {f, ld_f, false, false}, {gate, by_token ? ld_gate : p->dim, false, true}};
  const Vector weights[] = {{post, false}, {pre, false}};
  bool vec;
  int st = check(p, tokens, rows, weights, by_token, &vec);
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
  const Rows rows[] = {{dx, ld_dx, true, false}, {df, ld_df, true, false}, {dgate, by_token ? ld_dgate : p->dim, true, true}, {dh, ld_dh, false, false},
                       {dn, ld_dn, false, false}, {h, ld_h, false, false}, {f, ld_f, false, false}, {gate, by_token ? ld_gate : p->dim, false, true}};
  const Vector weights[] = {{post, false}, {pre, false}, {dpost, true}, {dpre, true}};
  bool vec;
  int st = check(p, tokens, rows, weights, by_token, &vec);
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

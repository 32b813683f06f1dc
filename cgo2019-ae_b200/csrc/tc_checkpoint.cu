// An activation function whose input is kept in 8 bits for the backward pass (tc_checkpoint_*).
//
//   x^ = q 2^e, e as in tc_elem.cuh over 32 neighbours of a row with e4m3 elements;   y = f(x),  gated: x = [a | b], y = f(a) b
//   dx = dy f'(x^),  gated: da = dy b^ f'(a^), db = dy f(a^);       dW[o, i] = sum_t dy[t, o] f(x^)[t, i]
//
// The result comes from the input itself, gradients from what was kept.  Codes lie along rows, each half's columns filled up with
// zeros to a multiple of 32; scales as bytes e + 127, a row's blocks one after another.
//
// Elementwise kernels: eight elements a lane, four lanes a block.  Bound by bytes without a function (8192 x 4096 bf16 kept in 28 us with a copy,
// 6.0 TB/s), with a gated silu 48 and its gradient 45 us (5.6 and 6.0 TB/s), by instructions with gelu (41 and 42; by the library's normal integral 83 and
// 94).  The weight gradient takes f(x^) from the workspace into the 16-bit product of tc_wm_kernel.cuh, as the sum of two numbers of dy's type (x^
// itself is one): rounded to one it gave bf16 results errors of 0.0020 against 64 bits in place of their own rounding's 0.0017, and nearly all of the
// error of fp32 results.  That costs the product twice its operations: 8192 tokens, 2048 x 4096 silu 218 to 220 us (one term 118), of which f(x^) 35
// (26) and the product 183 (92, 1490 TFLOP/s); without a function 107 to 126.
#include <algorithm>

#include "tc_elem.cuh"
#include "tc_inst.cuh"
#include "tc_op.h"
#include "tc_wm.h"

namespace {
using namespace tck;

constexpr int kThreads = 256;
enum { kNone = TC_ACT_NONE, kSilu = TC_ACT_SILU, kGelu = TC_ACT_GELU };

// 2^-(2 (hi - lo)) for hi >= 0 and lo far below the last place of what the result needs of hi: the square of 2^-hi, since the half never leaves the
// range in which the device's function needs no help.
__device__ __forceinline__ F2 power_of(F2 hi, F2 lo) {
  const float2 h = of2(hi);
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e.x) : "f"(-h.x));
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e.y) : "f"(-h.y));
  const F2 half = f2(e.x, e.y), v = mul2(half, half);
  return fma2(v, mul2(lo, f2(2.f * 0.693147181f)), v);
}
__device__ __forceinline__ F2 inverse_of(F2 v) {  // of numbers from 1 on
  const float2 t = of2(v);
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r.x) : "f"(t.x));
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r.y) : "f"(t.y));
  return f2(r.x, r.y);
}
__device__ __forceinline__ F2 size_of(float2 a, float most) { return f2(fminf(fabsf(a.x), most), fminf(fabsf(a.y), most)); }
__device__ __forceinline__ F2 by_sign(float2 a, F2 negative, F2 positive) {
  const float2 n = of2(negative), p = of2(positive);
  return f2(a.x < 0.f ? n.x : p.x, a.y < 0.f ? n.y : p.y);
}
// f(a) and its derivative of two numbers, to a few units of fp32's last place of their terms; one exponential and one reciprocal each.
//   silu   the logistic function and its complement both from exp(-|a|): neither is a difference.
//   gelu   P(a) = the normal distribution's integral.  With z = |a|, exp(z^2 / 2) P(-z) (z + k) is smooth on all of [0, oo) as a function of
//          u = (z - k) / (z + k) (Shepherd and Laframboise's transformation for the complementary error function); k = 2.5, and a
//          polynomial of degree 9 by least squares reweighted towards the largest relative error: 1.5e-8 up to z = 15, where the
//          exponential is zero in fp32, and with its coefficients in fp32 6.6e-8.  Exponents are split, since a rounding of z^2 is worth z^2 / 2 roundings of the result.
template <int Act>
__device__ __forceinline__ void activate(F2 a, F2* f, F2* slope) {
  constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.92596299e-8f;  // their sum is log2(e) to twice the bits
  const float2 v = of2(a);
  if constexpr (Act == kSilu) {
    const F2 z = size_of(v, 120.f), hi = mul2(z, f2(0.5f * kLog2e));  // exp(-120) is zero in fp32
    const F2 t = power_of(hi, fma2(z, f2(-0.5f * kLog2eRest), fma2(z, f2(-0.5f * kLog2e), hi)));
    const F2 big = inverse_of(fma2(t, f2(1.f), f2(1.f))), small = mul2(t, big);
    const F2 s = by_sign(v, small, big);
    *f = mul2(a, s);
    *slope = fma2(*f, by_sign(v, big, small), s);
  } else if constexpr (Act == kGelu) {
    const F2 z = size_of(v, 15.f), q = inverse_of(fma2(z, f2(1.f), f2(2.5f))), u = fma2(q, f2(-5.f), f2(1.f));
    constexpr float kTerms[10] = {0.706656635f,    -0.433692008f, 0.131986976f,    0.00923587568f,    -0.0163861867f,
                                  -0.00160083012f, 0.0025239361f, 0.000684414175f, -0.000311626092f, -0.000157704548f};
    F2 r = f2(kTerms[9]);
#pragma unroll
    for (int i = 8; i >= 0; --i) r = fma2(r, u, f2(kTerms[i]));
    const F2 square = mul2(z, z), rest = fma2(z, z, mul2(square, f2(-1.f))), hi = mul2(square, f2(0.25f * kLog2e));
    const F2 off = fma2(square, f2(-0.25f * kLog2e), hi);
    const F2 e = power_of(hi, fma2(rest, f2(-0.25f * kLog2e), fma2(square, f2(-0.25f * kLog2eRest), off)));
    const F2 far = mul2(mul2(r, q), e), s = by_sign(v, far, fma2(far, f2(-1.f), f2(1.f)));
    *f = mul2(a, s);
    *slope = fma2(a, mul2(e, f2(0.39894228f)), s);
  } else {
    *f = a;
    *slope = f2(1.f);
  }
}

struct ActArgs {
  unsigned char *codes, *scales;
  const void* in;         // x, or dy
  void* out;              // y, or dx; may be null where x is kept
  void* rest;             // kTerms: what `out` leaves of f(x^), rows as far apart
  int64_t ld_in, ld_out, rows;
  uint32_t pieces;        // units of 128 columns of a row
  uint32_t dim, padded;
};
// 16 lanes take 128 columns of R rows, eight each, four a block.
template <int R>
struct ActPlace {
  int lane, rows, valid;  // rows: that there are; valid: columns from the unit's first to the row's end
  int64_t row0;
  uint32_t col;           // the unit's first
  bool kept;              // the lane's columns have codes
  __device__ __forceinline__ explicit ActPlace(const ActArgs& a) {
    lane = threadIdx.x & 15;
    const uint64_t unit = (uint64_t)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4), group = unit < UINT32_MAX ? (uint32_t)unit / a.pieces : unit / a.pieces;
    col = (uint32_t)(unit - group * a.pieces) * 128;
    row0 = (int64_t)group * R;
    rows = (int)max((int64_t)0, min((int64_t)R, a.rows - row0));
    valid = (int)a.dim - (int)col;
    kept = col + lane * 8 < a.padded;
  }
};

template <class T, bool Vec, int Act, bool Gated, int R>
__global__ void __launch_bounds__(kThreads) keep_kernel(const __grid_constant__ ActArgs a) {
  constexpr int kParts = Gated ? 2 : 1;
  __shared__ __align__(16) T staged[Vec ? 1 : kThreads * 8];
  T* stage = staged + (Vec ? 0 : (threadIdx.x >> 4) * 128);
  const ActPlace<R> p(a);
  const T* x = static_cast<const T*>(a.in) + p.row0 * a.ld_in + p.col;
  const size_t per_row = (size_t)a.padded * kParts, at0 = p.row0 * per_row + p.col + p.lane * 8;
  chain_wait();
  Raw<T> raw[R][kParts];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int h = 0; h < kParts; ++h) raw[i][h] = unit_load<T, Vec>(x + i * a.ld_in + h * a.dim, p.lane, i < p.rows ? p.valid : 0, stage);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    F2 v[kParts][4];
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      unpack8<T>(raw[i][h], v[h]);
      const uint32_t byte = micro8_scale(block_max(magnitude_of<T>(raw[i][h])));
      const F2 inverse = f2(micro_inverse(byte));
      float scaled[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 t = of2(mul2(v[h][k], inverse));
        scaled[2 * k] = t.x;
        scaled[2 * k + 1] = t.y;
      }
      const uint2 code = byte == 255u ? make_uint2(0, 0) : to_e4m3(scaled);
      const size_t at = at0 + i * per_row + h * a.padded;
      if (p.kept && i < p.rows) {
        *reinterpret_cast<uint2*>(a.codes + at) = code;
        if ((p.lane & 3) == 0) a.scales[at >> 5] = (unsigned char)byte;
      }
    }
    if (a.out) {
      F2 y[4], slope;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        activate<Act>(v[0][k], y + k, &slope);
        if constexpr (Gated) y[k] = mul2(y[k], v[1][k]);
      }
      unit_store<T, Vec>(static_cast<T*>(a.out) + (p.row0 + i) * a.ld_out + p.col, pack8<T>(y), p.lane, i < p.rows ? p.valid : 0, stage);
    }
  }
}

enum Pass { kKeep, kRestore, kGrad, kTerms };

// f = hi + lo in numbers of type T, off by half of the last place of what hi leaves (2^-16 of f in bf16, 2^-22 in fp16, in whose subnormal range
// half of the smallest).  hi stays finite: beyond T's range lo is the rest of it, infinite where f is beyond twice that.
template <class T>
__device__ __forceinline__ void two_terms(const F2 (&f)[4], Raw<T>* hi, Raw<T>* lo) {
  constexpr float most = Elem<T>::kMost;
  auto in_range = [](float v) { return v > most ? most : v < -most ? -most : v; };  // NaN stays
  F2 part[4], rest[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 v = of2(f[k]);
    part[k] = f2(in_range(v.x), in_range(v.y));
  }
  *hi = pack8<T>(part);
  unpack8<T>(*hi, part);
#pragma unroll
  for (int k = 0; k < 4; ++k) rest[k] = fma2(part[k], f2(-1.f), f[k]);
  *lo = pack8<T>(rest);
}

// f(x^), once rounded or as two terms, or the gradient by x from dy.
template <class T, bool Vec, int Act, bool Gated, int R, Pass P>
__global__ void __launch_bounds__(kThreads) kept_kernel(const __grid_constant__ ActArgs a) {
  constexpr int kParts = Gated ? 2 : 1;
  constexpr bool Grad = P == kGrad;
  __shared__ __align__(16) T staged[Vec ? 1 : kThreads * 8];
  T* stage = staged + (Vec ? 0 : (threadIdx.x >> 4) * 128);
  const ActPlace<R> p(a);
  const size_t per_row = (size_t)a.padded * kParts, at0 = p.row0 * per_row + p.col + p.lane * 8;
  chain_wait();
  uint2 code[R][kParts];
  uint32_t scale[R][kParts];
  Raw<T> raw[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool there = p.kept && i < p.rows;
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      const size_t at = at0 + i * per_row + h * a.padded;
      code[i][h] = there ? *reinterpret_cast<const uint2*>(a.codes + at) : make_uint2(0, 0);
      scale[i][h] = there ? a.scales[at >> 5] : 0u;
    }
    if constexpr (Grad) raw[i] = unit_load<T, Vec>(static_cast<const T*>(a.in) + (p.row0 + i) * a.ld_in + p.col, p.lane, i < p.rows ? p.valid : 0, stage);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    F2 x[kParts][4], dy[4];
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      float v[8];
      from_e4m3(code[i][h], v);
      rescale8<T>(v, scale[i][h]);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[h][k] = f2(v[2 * k], v[2 * k + 1]);
    }
    if constexpr (Grad) unpack8<T>(raw[i], dy);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      F2 f, slope;
      activate<Act>(x[0][k], &f, &slope);
      if constexpr (Grad && Gated) {
        x[0][k] = mul2(dy[k], mul2(x[1][k], slope));
        x[1][k] = mul2(dy[k], f);
      } else if constexpr (Grad) {
        x[0][k] = mul2(dy[k], slope);
      } else if constexpr (Gated) {
        x[0][k] = mul2(f, x[1][k]);
      } else {
        x[0][k] = f;
      }
    }
    T* out = static_cast<T*>(a.out) + (p.row0 + i) * a.ld_out + p.col;
    if constexpr (P == kTerms) {
      Raw<T> hi, lo;
      two_terms<T>(x[0], &hi, &lo);
      unit_store<T, Vec>(out, hi, p.lane, i < p.rows ? p.valid : 0, stage);
      unit_store<T, Vec>(static_cast<T*>(a.rest) + (p.row0 + i) * a.ld_out + p.col, lo, p.lane, i < p.rows ? p.valid : 0, stage);
      continue;
    }
#pragma unroll
    for (int h = 0; h < (Grad ? kParts : 1); ++h) unit_store<T, Vec>(out + h * a.dim, pack8<T>(x[h]), p.lane, i < p.rows ? p.valid : 0, stage);
  }
}

template <class T, bool Vec, int Act, bool Gated, int R>
void (*kernel_of(Pass pass))(ActArgs) {
  // terms: of functions, to the workspace
  if constexpr (Vec && sizeof(T) == 2 && (Act != kNone || Gated))
    if (pass == kTerms) return kept_kernel<T, Vec, Act, Gated, R, kTerms>;
  return pass == kKeep ? keep_kernel<T, Vec, Act, Gated, R> : pass == kGrad ? kept_kernel<T, Vec, Act, Gated, R, kGrad> : kept_kernel<T, Vec, Act, Gated, R, kRestore>;
}
template <class T, int Act, bool Gated>
int launch(Pass pass, const ActArgs& a, bool vec, int sms, cudaStream_t stream) {
  // several rows a thread where that leaves a few blocks for each multiprocessor
  constexpr int kRows = Gated ? 2 : 4;
  const bool many = a.rows * a.pieces >= 16 * 16 * (int64_t)sms;
  const int64_t grid = ((many ? (a.rows + kRows - 1) / kRows : a.rows) * a.pieces + kThreads / 16 - 1) / (kThreads / 16);
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  auto kernel = many ? (vec ? kernel_of<T, true, Act, Gated, kRows>(pass) : kernel_of<T, false, Act, Gated, kRows>(pass))
                     : (vec ? kernel_of<T, true, Act, Gated, 1>(pass) : kernel_of<T, false, Act, Gated, 1>(pass));
  TC_CUDA_OK(launch_chained(true, kernel, dim3((unsigned)grid), (unsigned)kThreads, 0, stream, a));
  return TC_OK;
}
template <class T>
int launch(Pass pass, const TcOpShape& p, const ActArgs& a, bool vec, cudaStream_t stream) {
  switch (p.activation * 2 + (p.gated ? 1 : 0)) {
    case kSilu * 2: return launch<T, kSilu, false>(pass, a, vec, p.sms, stream);
    case kSilu * 2 + 1: return launch<T, kSilu, true>(pass, a, vec, p.sms, stream);
    case kGelu * 2: return launch<T, kGelu, false>(pass, a, vec, p.sms, stream);
    case kGelu * 2 + 1: return launch<T, kGelu, true>(pass, a, vec, p.sms, stream);
    case kNone * 2 + 1: return launch<T, kNone, true>(pass, a, vec, p.sms, stream);
    default: return launch<T, kNone, false>(pass, a, vec, p.sms, stream);
  }
}

int64_t padded_of(const TcOpShape& p) { return (p.dim + 31) / 32 * 32; }
// Numbers of the plan's type that f(x^) is the sum of in the product: x^ itself is one.
int terms_of(const TcOpShape& p) { return p.activation == kNone && !p.gated ? 1 : 2; }

int run(Pass pass, const TcOpShape& p, void* out, int64_t ld_out, unsigned char* codes, unsigned char* scales, const void* in, int64_t ld_in, int64_t tokens, int64_t cols,
        cudaStream_t stream, void* rest = nullptr) {
  const int64_t padded = padded_of(p);
  const int es = tc_elem_bytes(p.dtype);
  const ActArgs a{codes, scales, in, out, rest, ld_in, ld_out, tokens, (uint32_t)((padded + 127) / 128), (uint32_t)cols, (uint32_t)padded};
  const bool vec = (!in || tc_vec8(in, ld_in, cols, es)) && (!out || tc_vec8(out, ld_out, cols, es));
  switch (p.dtype) {
    case TC_F32: return launch<float>(pass, p, a, vec, stream);
    case TC_BF16: return launch<__nv_bfloat16>(pass, p, a, vec, stream);
    default: return launch<__half>(pass, p, a, vec, stream);
  }
}

// ---- the weight gradient ----
// Where the rows of dy are not aligned its columns are copied, as many at a time as take 32 MB, at least 1024 and at most 65536: each time is a product of
// its own (208 tokens, 1384 x 2193, with the call before it 26 us with 1024 at a time, 16 with all).
int64_t panel_of(const TcOpShape& p) { return std::min<int64_t>(65536, std::max<int64_t>(1024, (int64_t(16) << 20) / p.tokens / 64 * 64)); }
constexpr int kMostSlices = 16;
// Steps of 64 tokens and a term.  Fewer than 16 are never sliced: by the model below those of a whole tile on a CTA take 3.0 us, as much as slices cost
// besides, and where tiles take a second round there are too many to be sliced so finely.
int64_t steps_of(const TcOpShape& p, int64_t tokens) { return (tokens + 63) / 64 * terms_of(p); }
constexpr int64_t kLeastSteps = 16;

struct Buffers {
  uint16_t *kept, *panel;  // kept: one matrix a term
  float* slab;  // fp32 slices: of at most one tile a multiprocessor (a pair's for two)
};
size_t slab_floats(const TcOpShape& p) { return (size_t)p.sms * 128 * 256; }
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  TcCarver c{base};
  b->kept = c.take<uint16_t>(p.products ? (size_t)p.tokens * padded_of(p) * terms_of(p) : 0);
  b->panel = c.take<uint16_t>(p.products ? (size_t)p.tokens * panel_of(p) : 0);
  b->slab = c.take<float>(p.products && steps_of(p, p.tokens) >= kLeastSteps ? slab_floats(p) : 0);
  return c.used;
}

__global__ void __launch_bounds__(256) panel_kernel(uint16_t* to, int64_t pitch, const uint16_t* from, int64_t ld, int64_t tokens, uint32_t cols) {
  chain_wait();
  for (uint32_t col = (blockIdx.y * 256 + threadIdx.x) * 4; col < cols; col += gridDim.y * 1024)
    for (int64_t row = blockIdx.x; row < tokens; row += gridDim.x) {
      uint16_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = col + k < cols ? from[row * ld + col + k] : (uint16_t)0;
      *reinterpret_cast<uint2*>(to + row * pitch + col) = make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
    }
}

struct JoinArgs {
  const float* slab;
  void* out;
  int64_t ld, n, slice_stride;
  uint32_t dim, slices;
  int32_t add;
};
template <class T>
__global__ void __launch_bounds__(256) weight_join_kernel(const __grid_constant__ JoinArgs a) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  chain_wait();
  if (at >= a.n) return;
  float s = 0.f;
  for (uint32_t i = 0; i < a.slices; ++i) s += a.slab[i * a.slice_stride + at];
  T* to = static_cast<T*>(a.out) + at / a.dim * a.ld + at % a.dim;
  *to = Elem<T>::put(a.add ? Elem<T>::get(*to) + s : s);
}

// Tile and slices of the tokens that take the least time by a model (us): rounds of tiles, each its stages of 64 tokens and what a tile
// costs besides; slices add a launch and their fp32 results, written and read.  By it 1024 x 1024 by 1024 tokens stays whole (8.5 us with f(x^); two
// slices 14.1), 512 x 512 by 4096 is sliced (10.7; whole 16.6), 1024 x 2048 by 8192 takes single CTAs (38; two slices on pairs 44).
void choose(const TcOpShape& p, int64_t outputs, int64_t tokens, int* tile, int* slices) {
  const int64_t blocks = steps_of(p, tokens);
  const int most = blocks >= kLeastSteps ? kMostSlices : 1;
  double least = 0;
  *tile = WM_PAIR_256;
  *slices = 1;
  for (int t : {WM_PAIR_256, WM_128}) {
    const bool pair = t == WM_PAIR_256;
    const int64_t bk = wm_weight_stage(tokens, t), stages = (tokens + bk - 1) / bk * terms_of(p);
    const int64_t tiles = ((p.dim + wm_tile_m(t) - 1) / wm_tile_m(t)) * ((outputs + wm_tile_n(t) - 1) / wm_tile_n(t)), workers = std::max(1, pair ? p.sms / 2 : p.sms);
    for (int s = 1; s <= most && s <= stages && (s == 1 || tiles * s <= workers); ++s) {
      const double cost = (double)((tiles * s + workers - 1) / workers) * ((pair ? 0.29 : 0.2) * ((blocks + s - 1) / s) + (pair ? 0.5 : 0.35)) +
                          (s > 1 ? 3.0 + 2e-6 * s * (double)p.dim * outputs : 0.0);
      if (least == 0 || cost < least) {
        least = cost;
        *tile = t;
        *slices = s;
      }
    }
  }
}

int weight(const tc_op_plan& p, const Buffers& b, void* dw, int64_t ld_dw, int type, const uint16_t* dy, int64_t ld_dy, unsigned char* codes, unsigned char* scales, int64_t outputs,
           int64_t tokens, int accumulate, cudaStream_t stream) {
  const int64_t padded = padded_of(p), panel = panel_of(p);
  const int terms = terms_of(p);
  int st = run(terms == 2 ? kTerms : kRestore, p, b.kept, padded, codes, scales, nullptr, 0, tokens, padded, stream, b.kept + tokens * padded);
  const bool boxes = wm_boxable(dy, ld_dy, 0, 2);
  for (int64_t first = 0; st == TC_OK && first < outputs; first += boxes ? outputs : panel) {
    const int64_t n = boxes ? outputs : std::min(panel, outputs - first), pitch = (n + 7) / 8 * 8;
    if (!boxes)
      TC_CUDA_OK(launch_chained(true, panel_kernel, dim3((unsigned)std::min<int64_t>(tokens, 8 * p.sms), (unsigned)std::min<int64_t>((n + 1023) / 1024, 64)), 256u, 0, stream, b.panel,
                                pitch, dy + first, ld_dy, tokens, (uint32_t)n));
    int tile, slices;
    choose(p, n, tokens, &tile, &slices);
    WmArgs m{};
    m.M = (uint32_t)p.dim;
    m.N = (uint32_t)n;
    m.K = (uint32_t)tokens;
    m.batch = 1;
    m.slices = (uint32_t)slices;
    m.bf16 = p.dtype == TC_BF16;
    m.status = p.status;
    m.spin_limit = p.test_fault ? 1u << 14 : TC_SPIN_LIMIT;
    m.test_fault = p.test_fault;
    char* to = static_cast<char*>(dw) + first * ld_dw * tc_elem_bytes(type);
    m.weight = slices > 1 ? WmWeightArgs{b.slab, p.dim, n * p.dim, TC_F32, 0, terms} : WmWeightArgs{to, ld_dw, 0, type, accumulate != 0, terms};
    st = wm_launch(WM_WEIGHT, tile, m, WmOperand{b.kept, padded, tokens * padded}, boxes ? WmOperand{dy, ld_dy, 0} : WmOperand{b.panel, pitch, 0}, p.sms, stream);
    if (st != TC_OK || slices == 1) continue;
    const JoinArgs j{b.slab, to, ld_dw, n * p.dim, n * p.dim, (uint32_t)p.dim, (uint32_t)slices, accumulate != 0};
    auto join = type == TC_F32 ? weight_join_kernel<float> : type == TC_BF16 ? weight_join_kernel<__nv_bfloat16> : weight_join_kernel<__half>;
    TC_CUDA_OK(launch_chained(true, join, dim3((unsigned)((j.n + 255) / 256)), 256u, 0, stream, j));
  }
  return st;
}

int check(const tc_op_plan* p, const void* codes, const void* scales, int64_t tokens) {
  if (!p || p->kind != TC_OP_CHECKPOINT || (tokens && (!codes || !scales))) return TC_ERR_INVALID_ARG;
  if (tokens < 0 || tokens > p->tokens) return TC_ERR_EXTENT;
  if (tc_odd_address(codes, 16)) return TC_ERR_ALIGNMENT;
  return TC_OK;
}

// What is kept of some rows, each array without a gap.
TcSpan codes_of(const tc_op_plan* p, const void* codes, int64_t tokens, bool written) {
  return TcSpan{codes, 0, padded_of(*p) * (p->gated ? 2 : 1) * tokens, 1, written};
}
TcSpan scales_of(const tc_op_plan* p, const void* scales, int64_t tokens, bool written) {
  return TcSpan{scales, 0, padded_of(*p) / 32 * (p->gated ? 2 : 1) * tokens, 1, written};
}
TcSpan rows_of(const tc_op_plan* p, const void* ptr, int64_t ld, int64_t cols, int64_t rows, bool written) {
  const int es = tc_elem_bytes(p->dtype);
  return TcSpan{ptr, ld * es, cols * es, rows, written};
}

}  // namespace

std::string tc_checkpoint_json(const TcOpShape& p) {
  const int64_t padded = padded_of(p) * (p.gated ? 2 : 1);
  static const char* const names[] = {"none", "silu", "gelu"};
  return "{\"operator\":\"checkpoint\",\"dtype\":\"" + tc_type_name(p.dtype) + "\",\"tokens\":" + std::to_string(p.tokens) + ",\"dim\":" + std::to_string(p.dim) +
         ",\"activation\":\"" + names[p.activation] + "\",\"gated\":" + (p.gated ? "true" : "false") + ",\"bytes_per_row\":" + std::to_string(padded) +
         ",\"scales_per_row\":" + std::to_string(padded / 32) + ",\"workspace_bytes\":" + std::to_string(tc_checkpoint_workspace(p)) + "}";
}

size_t tc_checkpoint_workspace(const TcOpShape& p) {
  Buffers b;
  return carve(p, nullptr, &b);
}

int tc_checkpoint_prepare() { return wm_prepare(WM_WEIGHT); }

extern "C" int tc_checkpoint_execute(tc_op_plan* p, void* y, int64_t ld_y, void* codes, void* scales, const void* x, int64_t ld_x, int64_t tokens, void* stream) {
  int st = check(p, codes, scales, tokens);
  if (st != TC_OK) return st;
  if (tokens && !x) return TC_ERR_INVALID_ARG;
  if (ld_x < 0 || (y && ld_y < p->dim)) return TC_ERR_EXTENT;
  const int es = tc_elem_bytes(p->dtype);
  if (tc_odd_address(x, es) || tc_odd_address(y, es)) return TC_ERR_ALIGNMENT;
  const TcSpan spans[] = {rows_of(p, y, ld_y, p->dim, tokens, true), codes_of(p, codes, tokens, true), scales_of(p, scales, tokens, true),
                          rows_of(p, x, ld_x, p->dim * (p->gated ? 2 : 1), tokens, false)};
  if (tc_results_overlap(spans)) return TC_ERR_INVALID_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = tc_op_ready(p, s);
  if (st != TC_OK || tokens == 0) return st;
  return run(kKeep, *p, y, ld_y, static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), x, ld_x, tokens, p->dim, s);
}

extern "C" int tc_checkpoint_restore(tc_op_plan* p, void* y, int64_t ld_y, const void* codes, const void* scales, int64_t tokens, void* stream) {
  int st = check(p, codes, scales, tokens);
  if (st != TC_OK) return st;
  if (tokens && !y) return TC_ERR_INVALID_ARG;
  if (ld_y < p->dim) return TC_ERR_EXTENT;
  if (tc_odd_address(y, tc_elem_bytes(p->dtype))) return TC_ERR_ALIGNMENT;
  const TcSpan spans[] = {rows_of(p, y, ld_y, p->dim, tokens, true), codes_of(p, codes, tokens, false), scales_of(p, scales, tokens, false)};
  if (tc_results_overlap(spans)) return TC_ERR_INVALID_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = tc_op_ready(p, s);
  if (st != TC_OK || tokens == 0) return st;
  return run(kRestore, *p, y, ld_y, const_cast<unsigned char*>(static_cast<const unsigned char*>(codes)), const_cast<unsigned char*>(static_cast<const unsigned char*>(scales)), nullptr, 0,
             tokens, p->dim, s);
}

extern "C" int tc_checkpoint_execute_grad(tc_op_plan* p, void* dx, int64_t ld_dx, const void* dy, int64_t ld_dy, const void* codes, const void* scales, int64_t tokens,
                                          void* stream) {
  int st = check(p, codes, scales, tokens);
  if (st != TC_OK) return st;
  if (tokens && (!dx || !dy)) return TC_ERR_INVALID_ARG;
  if (ld_dx < p->dim * (p->gated ? 2 : 1) || ld_dy < 0) return TC_ERR_EXTENT;
  const int es = tc_elem_bytes(p->dtype);
  if (tc_odd_address(dx, es) || tc_odd_address(dy, es)) return TC_ERR_ALIGNMENT;
  const TcSpan spans[] = {rows_of(p, dx, ld_dx, p->dim * (p->gated ? 2 : 1), tokens, true), rows_of(p, dy, ld_dy, p->dim, tokens, false), codes_of(p, codes, tokens, false),
                          scales_of(p, scales, tokens, false)};
  if (tc_results_overlap(spans)) return TC_ERR_INVALID_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = tc_op_ready(p, s);
  if (st != TC_OK || tokens == 0) return st;
  return run(kGrad, *p, dx, ld_dx, const_cast<unsigned char*>(static_cast<const unsigned char*>(codes)), const_cast<unsigned char*>(static_cast<const unsigned char*>(scales)), dy, ld_dy,
             tokens, p->dim, s);
}

extern "C" int tc_checkpoint_execute_product(tc_op_plan* p, void* dweight, int64_t ld_dweight, int dweight_dtype, const void* dy, int64_t ld_dy, const void* codes, const void* scales,
                                             int64_t outputs, int64_t tokens, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check(p, codes, scales, tokens);
  if (st != TC_OK) return st;
  if (!dweight || (tokens && !dy) || (dweight_dtype != TC_F32 && dweight_dtype != p->dtype)) return TC_ERR_INVALID_ARG;
  if (!p->products) return TC_ERR_UNSUPPORTED;
  if (outputs < 1 || ld_dweight < p->dim || ld_dy < 0) return TC_ERR_EXTENT;
  if (outputs > int64_t(1) << 30) return TC_ERR_UNSUPPORTED;
  const int es = tc_elem_bytes(dweight_dtype);
  if (tc_odd_address(dweight, es) || tc_odd_address(dy, 2)) return TC_ERR_ALIGNMENT;
  const TcSpan spans[] = {{dweight, ld_dweight * es, p->dim * es, outputs, true}, rows_of(p, dy, ld_dy, outputs, tokens, false), codes_of(p, codes, tokens, false),
                          scales_of(p, scales, tokens, false)};
  if (tc_results_overlap(spans)) return TC_ERR_INVALID_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  TcScratch scratch;
  st = scratch.open(p, TC_OP_CHECKPOINT, workspace, workspace_bytes, s);
  if (st != TC_OK) return st;
  if (tokens == 0) {  // no tokens: the gradient is zero
    if (!accumulate) TC_CUDA_OK(cudaMemset2DAsync(dweight, (size_t)ld_dweight * es, 0, (size_t)p->dim * es, (size_t)outputs, s));
    return TC_OK;
  }
  Buffers b;
  carve(*p, scratch.base, &b);
  return scratch.close(weight(*p, b, dweight, ld_dweight, dweight_dtype, static_cast<const uint16_t*>(dy), ld_dy, const_cast<unsigned char*>(static_cast<const unsigned char*>(codes)),
                              const_cast<unsigned char*>(static_cast<const unsigned char*>(scales)), outputs, tokens, accumulate, s));
}

// An activation function whose input is kept in 8 bits for the backward pass (tc_checkpoint_*).
//
//   x^ = q 2^e, e as in tc_elem.cuh over 32 neighbours of a row with e4m3 elements;   y = f(x),  gated: x = [a | b], y = f(a) b
//   dx = dy f'(x^),  gated: da = dy b^ f'(a^), db = dy f(a^);       dW[o, i] = sum_t dy[t, o] f(x^)[t, i]
//
// The result comes from the input itself, gradients from what was kept.  Codes lie along rows, each half's columns filled up with
// zeros to a multiple of 32; scales as bytes e + 127, a row's blocks one after another.
//
// Elementwise kernels: eight elements a lane, four lanes a block; bound by bytes.  The weight gradient takes f(x^), rounded to the
// type of dy (without a function: as it is), from the workspace into the 16-bit product of tc_wm_kernel.cuh.
#include <algorithm>

#include "tc_elem.cuh"
#include "tc_inst.cuh"
#include "tc_op.h"
#include "tc_wm.h"

namespace {
using namespace tck;

constexpr int kThreads = 256;
enum { kNone = TC_ACT_NONE, kSilu = TC_ACT_SILU, kGelu = TC_ACT_GELU };

// f(a) and its derivative.  The logistic function and its complement both from exp(-|a|): neither is a difference.
template <int Act>
__device__ __forceinline__ void activate(float a, float* f, float* slope) {
  if constexpr (Act == kSilu) {
    const float t = expf(-fabsf(a)), big = 1.f / (1.f + t), small = t * big;
    const float s = a < 0.f ? small : big;
    *f = a * s;
    *slope = fmaf(*f, a < 0.f ? big : small, s);
  } else if constexpr (Act == kGelu) {
    const float s = normcdff(a);
    *f = a * s;
    *slope = fmaf(a, 0.3989422804014327f * expf(-0.5f * a * a), s);
  } else {
    *f = a;
    *slope = 1.f;
  }
}

struct ActArgs {
  unsigned char *codes, *scales;
  const void* in;         // x, or dy
  void* out;              // y, or dx; may be null where x is kept
  int64_t ld_in, ld_out, units;
  uint32_t per_row;       // units of a row: of eight columns
  uint32_t dim, padded;
};
struct ActPlace {
  int64_t row;
  uint32_t col;
  int valid;              // columns from here to the row's end; none behind the last row
};
__device__ __forceinline__ ActPlace act_place(const ActArgs& a, int64_t unit) {
  ActPlace p;
  p.row = unit < UINT32_MAX ? (int64_t)((uint32_t)unit / a.per_row) : unit / a.per_row;
  p.col = (uint32_t)(unit - p.row * a.per_row) * 8;
  p.valid = unit < a.units ? (int)a.dim - (int)p.col : 0;
  return p;
}

// Eight elements to their codes and, by one of the block's four lanes, its scale.
__device__ __forceinline__ void keep8(const float* x, unsigned char* codes, unsigned char* scales, size_t at, bool there) {
  const uint32_t byte = micro8_scale(block_max(magnitude8(x)));
  uint2 code = make_uint2(0, 0);
  if (byte != 255u) {
    const float inverse = micro_inverse(byte);
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = x[k] * inverse;
    code = to_e4m3(f);
  }
  if (there) {
    *reinterpret_cast<uint2*>(codes + at) = code;
    if ((at & 31) == 0) scales[at >> 5] = (unsigned char)byte;
  }
}
template <class T>
__device__ __forceinline__ void kept8(uint2 code, uint32_t byte, float* x) {
  from_e4m3(code, x);
  rescale8<T>(x, micro_power(byte));
}

template <class T, bool Vec, int Act, bool Gated, int N>
__global__ void __launch_bounds__(kThreads) keep_kernel(const __grid_constant__ ActArgs a) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * N) + threadIdx.x;
  constexpr int kParts = Gated ? 2 : 1;
  chain_wait();
  Raw<T> raw[N][kParts];
  ActPlace p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = act_place(a, first + i * kThreads);
    const T* x = static_cast<const T*>(a.in) + p[i].row * a.ld_in + p[i].col;
#pragma unroll
    for (int h = 0; h < kParts; ++h) raw[i][h] = load8<T, Vec>(x + h * a.dim, p[i].valid);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float x[kParts][8];
    const bool there = first + i * kThreads < a.units;
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      unpack8<T>(raw[i][h], x[h]);
      keep8(x[h], a.codes, a.scales, ((size_t)p[i].row * kParts + h) * a.padded + p[i].col, there);
    }
    if (a.out && p[i].valid > 0) {
      float y[8], slope;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        activate<Act>(x[0][k], y + k, &slope);
        if constexpr (Gated) y[k] *= x[1][k];
      }
      store8<T, Vec>(static_cast<T*>(a.out) + p[i].row * a.ld_out + p[i].col, pack8<T>(y), p[i].valid);
    }
  }
}

// f(x^), or the gradient by x from dy.
template <class T, bool Vec, int Act, bool Gated, bool Grad, int N>
__global__ void __launch_bounds__(kThreads) kept_kernel(const __grid_constant__ ActArgs a) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * N) + threadIdx.x;
  constexpr int kParts = Gated ? 2 : 1;
  chain_wait();
  uint2 code[N][kParts];
  uint32_t scale[N][kParts];
  Raw<T> raw[N];
  ActPlace p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = act_place(a, first + i * kThreads);
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      const size_t at = ((size_t)p[i].row * kParts + h) * a.padded + p[i].col;
      code[i][h] = make_uint2(0, 0);
      scale[i][h] = 0;
      if (p[i].valid > 0) {
        code[i][h] = *reinterpret_cast<const uint2*>(a.codes + at);
        scale[i][h] = a.scales[at >> 5];
      }
    }
    if constexpr (Grad) raw[i] = load8<T, Vec>(static_cast<const T*>(a.in) + p[i].row * a.ld_in + p[i].col, p[i].valid);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (p[i].valid <= 0) continue;
    float x[kParts][8], dy[8];
#pragma unroll
    for (int h = 0; h < kParts; ++h) kept8<T>(code[i][h], scale[i][h], x[h]);
    if constexpr (Grad) unpack8<T>(raw[i], dy);
    T* out = static_cast<T*>(a.out) + p[i].row * a.ld_out + p[i].col;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float f, slope;
      activate<Act>(x[0][k], &f, &slope);
      if constexpr (Grad && Gated) {
        x[0][k] = dy[k] * (x[1][k] * slope);
        x[1][k] = dy[k] * f;
      } else if constexpr (Grad) {
        x[0][k] = dy[k] * slope;
      } else if constexpr (Gated) {
        x[0][k] = f * x[1][k];
      } else {
        x[0][k] = f;
      }
    }
#pragma unroll
    for (int h = 0; h < (Grad ? kParts : 1); ++h) store8<T, Vec>(out + h * a.dim, pack8<T>(x[h]), p[i].valid);
  }
}

enum Pass { kKeep, kRestore, kGrad };

template <class T, bool Vec, int Act, bool Gated, int N>
void (*kernel_of(Pass pass))(ActArgs) {
  return pass == kKeep ? keep_kernel<T, Vec, Act, Gated, N> : pass == kGrad ? kept_kernel<T, Vec, Act, Gated, true, N> : kept_kernel<T, Vec, Act, Gated, false, N>;
}
template <class T, int Act, bool Gated>
int launch(Pass pass, const ActArgs& a, bool vec, int sms, cudaStream_t stream) {
  const bool many = a.units >= (int64_t)kThreads * 2 * 4 * sms;
  const int64_t grid = (a.units + kThreads * (many ? 2 : 1) - 1) / (kThreads * (many ? 2 : 1));
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  auto kernel = many ? (vec ? kernel_of<T, true, Act, Gated, 2>(pass) : kernel_of<T, false, Act, Gated, 2>(pass))
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

int run(Pass pass, const TcOpShape& p, void* out, int64_t ld_out, unsigned char* codes, unsigned char* scales, const void* in, int64_t ld_in, int64_t tokens, int64_t cols,
        cudaStream_t stream) {
  const int64_t padded = padded_of(p);
  const int es = tc_elem_bytes(p.dtype);
  const ActArgs a{codes, scales, in, out, ld_in, ld_out, tokens * (padded / 8), (uint32_t)(padded / 8), (uint32_t)cols, (uint32_t)padded};
  const bool vec = (!in || tc_vec8(in, ld_in, cols, es)) && (!out || tc_vec8(out, ld_out, cols, es));
  switch (p.dtype) {
    case TC_F32: return launch<float>(pass, p, a, vec, stream);
    case TC_BF16: return launch<__nv_bfloat16>(pass, p, a, vec, stream);
    default: return launch<__half>(pass, p, a, vec, stream);
  }
}

// ---- the weight gradient ----
constexpr int64_t kPanel = 1024;  // columns of dy that are copied at a time where its rows are not aligned
constexpr int kMostSlices = 16;

struct Buffers {
  uint16_t *kept, *panel;
  float* slab;  // fp32 slices: of at most one tile a multiprocessor (a pair's for two)
};
size_t slab_floats(const TcOpShape& p) { return (size_t)p.sms * 128 * 256; }
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  TcCarver c{base};
  b->kept = c.take<uint16_t>(p.products ? (size_t)p.tokens * padded_of(p) : 0);
  b->panel = c.take<uint16_t>(p.products ? (size_t)p.tokens * kPanel : 0);
  b->slab = c.take<float>(p.products ? slab_floats(p) : 0);
  return c.used;
}

__global__ void __launch_bounds__(256) panel_kernel(uint16_t* to, const uint16_t* from, int64_t ld, int64_t tokens, uint32_t cols) {
  const uint32_t col = threadIdx.x * 4;
  chain_wait();
  if (col >= cols) return;
  for (int64_t row = blockIdx.x; row < tokens; row += gridDim.x) {
    uint16_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = col + k < cols ? from[row * ld + col + k] : (uint16_t)0;
    *reinterpret_cast<uint2*>(to + row * kPanel + col) = make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
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

int weight(const tc_op_plan& p, const Buffers& b, void* dw, int64_t ld_dw, int type, const uint16_t* dy, int64_t ld_dy, unsigned char* codes, unsigned char* scales, int64_t outputs,
           int64_t tokens, int accumulate, cudaStream_t stream) {
  const int64_t padded = padded_of(p);
  int st = run(kRestore, p, b.kept, padded, codes, scales, nullptr, 0, tokens, padded, stream);
  const bool boxes = wm_boxable(dy, ld_dy, 0, 2);
  for (int64_t first = 0; st == TC_OK && first < outputs; first += boxes ? outputs : kPanel) {
    const int64_t n = boxes ? outputs : std::min(kPanel, outputs - first);
    if (!boxes) TC_CUDA_OK(launch_chained(true, panel_kernel, dim3((unsigned)std::min<int64_t>(tokens, 8 * p.sms)), 256u, 0, stream, b.panel, dy + first, ld_dy, tokens, (uint32_t)n));
    int tile, slices;
    wm_choose(WM_WEIGHT, p.dim, n, tokens, 1, kMostSlices, p.sms, &tile, &slices);
    const int64_t tiles = ((p.dim + wm_tile_m(tile) - 1) / wm_tile_m(tile)) * ((n + wm_tile_n(tile) - 1) / wm_tile_n(tile));
    slices = (int)std::max<int64_t>(1, std::min<int64_t>(slices, (tile == WM_PAIR_256 ? p.sms / 2 : p.sms) / tiles));
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
    m.weight = slices > 1 ? WmWeightArgs{b.slab, p.dim, n * p.dim, TC_F32, 0} : WmWeightArgs{to, ld_dw, 0, type, accumulate != 0};
    st = wm_launch(WM_WEIGHT, tile, m, WmOperand{b.kept, padded, 0}, boxes ? WmOperand{dy, ld_dy, 0} : WmOperand{b.panel, kPanel, 0}, p.sms, stream);
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

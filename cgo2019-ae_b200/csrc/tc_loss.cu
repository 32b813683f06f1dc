// Softmax cross entropy over a vocabulary and its gradients, without the logits (tc_vocab_loss_execute*).
//
//   z_tv = h_t . w_v      lse_t = log sum_v exp(z_tv)      loss_t = lse_t - z_t,target(t)
//   G_tv = g_t (exp(z_tv - lse_t) - [v = target(t)])       dH = G W      dW = G^T H
//
// Few tokens of up to 2560 columns: passes over the table without tensor cores (see there).  Otherwise:
// Forward: one product whose epilogue keeps a maximum and a sum per row and half tile of columns; 2 T D V operations.
// Gradients: per piece of the vocabulary the logits once more, turned into G in the epilogue (rounded once to the operands'
// type, the other rounding being the result's own), then both products with G in one launch: 8 T D V operations in all for loss and
// gradients, where a program that holds T x V logits needs 6.
// Bound by the products: loss and gradients of 7782 tokens, K = 2048, 131072 rows take 13.4 to 14.4 ms (16.7e12 operations: 1160 to 1250
// TFLOP/s, under the power cap), of 2048, K = 1024, 32768 rows 476 to 506 us; 1023 x 777 x 50001 in fp16 400 to 418 us, of which 51 copy the
// table to aligned rows (in both directions together) and 25 pack the tokens' rows; the loss alone of 16 tokens, 32000 rows of 512 15.4 to
// 15.9 us: the product (two rounds of mostly empty tiles, 12.6 by itself) and the join (5.6), a launch each, for 5 us of traffic.
// Tokens without a target take no part: the others' rows are packed first, so masked rows cost nothing and whatever they
// hold (infinities, NaN) reaches no sum.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc_inst.cuh"
#include "tc_op.h"
#include "tc_wm.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowsPerBlock = 8;         // packing: one row per warp
// Tokens up to which a packing block counts the ones before its own itself.  The loss of 64 columns, 1000 rows, us with counts from a launch
// and by each block: 4096 tokens 15.9, 14.8; 8192 21.3, 20.8; 12000 28.2, 29.1; 32768 61.9, 87.5.
constexpr int64_t kCountedDirectly = 8192;
constexpr int kCountChunk = 2048;
// ... and up to which it finds the largest weight itself.  Loss and gradients of that size, us with a launch and without: 1023 tokens 34.8, 32.8;
// 2048 38.8, 37.6; 4096 54.1, 54.5; 16384 154, 171.
constexpr int64_t kScaledDirectly = 2048;
constexpr int64_t kStatsRows = 16384;       // rows whose statistics are kept at a time
constexpr int64_t kUnpacked = 256;          // tokens up to which the forward pass takes the rows where they are

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Eight 16-bit elements from `from` on, of which `left` belong to the row: out of the aligned 16-byte words that hold them where
// those lie between `begin` and `end` (the first and last byte of all rows), else element by element, zeros behind the row.
__device__ __forceinline__ uint4 eight_of_row(const uint16_t* from, int left, uintptr_t begin, uintptr_t end) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(from), word = at & ~uintptr_t(15);
  uint32_t w[8];
  if (word >= begin && word + 32 <= end) {
    const uint4 a = *reinterpret_cast<const uint4*>(word), b = *reinterpret_cast<const uint4*>(word + 16);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    const uint32_t shift = (uint32_t)(at & 15), bits = (shift & 2) * 8;  // bytes, even
#pragma unroll
    for (int k = 0; k < 7; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], bits);
    w[7] >>= bits;
    if (shift & 8) { w[0] = w[2]; w[1] = w[3]; w[2] = w[4]; w[3] = w[5]; w[4] = w[6]; }
    if (shift & 4) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = w[4]; }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (2 * k < left ? (uint32_t)from[2 * k] : 0u) | (2 * k + 1 < left ? (uint32_t)from[2 * k + 1] << 16 : 0u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct PackArgs {
  const void* targets;
  int64_t tokens, vocab;
  int wide;                  // targets are 64-bit
  const int* chunk_counts;   // per kCountChunk tokens, or null: counted here
  const uint16_t* hidden;    // 16-bit values, moved as they are
  int64_t ld_hidden;
  int dim, pitch, vec;       // packed rows' pitch; 16-byte copies are possible
  int pad;                   // zeros up to a multiple of so many rows
  uint16_t* packed;
  int64_t* target;           // per packed row
  int* source;               // packed row -> token
  int* packed_of;            // token -> packed row or -1
  int* count;
  float *loss, *lse;         // forward: zeros for tokens without a target
  // gradient: rows of WmRow from the forward's lse and the caller's weights
  const float *lse_in, *weight;
  float* weight_scale;
  float range;               // > 0: every block finds the scale itself, the first writes it down
  WmRow* rows;
  int* lift;                 // per packed row: lift_of() its weight, which is multiplied by 2 to it; null: left as they are
  float* most;               // per block: the largest of its rows' elements, each divided by 2^lift; null: not wanted
};

// What weights are multiplied by, and what the products with G are: relative to the largest weight.  Where all are equal, as for a
// mean, G's entries at the targets are then -1 and a little, not all rounded the same way from 1 / n; `range` is 2^14 in fp16, so
// that probabilities down to 2^-28 keep all their bits.
__device__ __forceinline__ float2 scale_for(float most, float range) {
  if (!(most > 1e-30f && most < 1e30f)) most = 1.f;
  return make_float2(range / most, most / range);
}

// fp16 has no room for small weights beside small probabilities (a millionth of 2^14 leaves a probability of 1e-4 five bits), so there the
// weight's power of two moves from G to the other operand.  G is rounded relative to each token's own weight:
//   dH_t = 2^-lift_t scale (2^lift_t G_t) W        dW = sum_t (2^lift_t G_t) (2^-lift_t H_t) scale
// where powers of two round nothing, and 2^-lift_t H_t, lifted together until the largest element is near 2^14, keeps all bits of
// what is above 2^-28 of that (lift_kernel).
__device__ __forceinline__ int lift_of(float weight) {  // a weight of at most 2^14 to above 2^13
  const float size = fabsf(weight);
  if (!(size > 0.f && size < 16384.f)) return 0;
  int e;
  frexpf(size, &e);
  return min(14 - e, 100);
}

// Tokens with a target per chunk of kCountChunk.
__global__ void __launch_bounds__(256) count_kernel(const void* targets, int wide, int64_t tokens, int64_t vocab, int* counts) {
  tck::chain_wait();
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kCountChunk, end = min(tokens, first + kCountChunk);
  int n = 0;
  for (int64_t i = first + threadIdx.x; i < end; i += 256) {
    const int64_t t = index_at(targets, i, wide);
    n += t >= 0 && t < vocab;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) atomicAdd(&total, n);  // whole numbers: any order
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}

// Packs the rows of the tokens that take part, in order.  One warp per token; a block first counts the tokens before its own.
__global__ void __launch_bounds__(32 * kRowsPerBlock) pack_kernel(const PackArgs p) {
  tck::chain_wait();
  __shared__ int before, has[kRowsPerBlock];
  __shared__ uint32_t most;  // largest weight's bits
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t first = (int64_t)blockIdx.x * kRowsPerBlock;
  if (tid == 0) before = most = 0;
  __syncthreads();
  auto takes_part = [&](int64_t i) {
    const int64_t t = index_at(p.targets, i, p.wide);
    return t >= 0 && t < p.vocab;
  };
  int n = 0;
  int64_t from = 0;
  if (p.chunk_counts) {
    const int64_t chunks = first / kCountChunk;
    for (int64_t c = tid; c < chunks; c += blockDim.x) n += p.chunk_counts[c];
    from = chunks * kCountChunk;
  }
  for (int64_t i = from + tid; i < first; i += blockDim.x) n += takes_part(i);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) atomicAdd(&before, n);
  if (p.range > 0.f) {
    float m = 0.f;
    for (int64_t i = tid; i < p.tokens; i += blockDim.x)
      if (takes_part(i)) m = fmaxf(m, fabsf(p.weight[i]));
    atomicMax(&most, __reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // not negative: bits are ordered as values are
  }
  const int64_t token = first + warp;
  const bool mine = token < p.tokens && takes_part(token);
  if (lane == 0) has[warp] = mine;
  __syncthreads();
  int row = before;
  for (int w = 0; w < warp; ++w) row += has[w];
  float scale = 1.f;
  if (p.rows) {
    const float2 both = p.range > 0.f ? scale_for(__uint_as_float(most), p.range) : make_float2(p.weight_scale[0], p.weight_scale[1]);
    scale = both.x;
    if (p.range > 0.f && blockIdx.x == 0 && tid == 0) {
      p.weight_scale[0] = both.x;
      p.weight_scale[1] = both.y;
    }
  }
  uint32_t largest = 0;  // two elements' bits without their signs
  if (token < p.tokens) {
    if (lane == 0) {
      if (p.packed_of) p.packed_of[token] = mine ? row : -1;
      if (mine) {
        const int64_t t = index_at(p.targets, token, p.wide);
        if (p.target) p.target[row] = t;
        if (p.source) p.source[row] = (int)token;
        if (p.rows) {
          float weight = p.weight[token] * scale;
          if (p.lift) {
            p.lift[row] = lift_of(weight);
            weight = ldexpf(weight, lift_of(weight));
          }
          p.rows[row] = WmRow{p.lse_in[token] * kLog2e, weight, t};
        }
      } else if (p.loss) {
        p.loss[token] = 0.f;
        p.lse[token] = 0.f;
      }
    }
    if (mine) {
      const uint16_t* src = p.hidden + token * p.ld_hidden;
      uint16_t* dst = p.packed + (int64_t)row * p.pitch;
      auto put = [&](int c, uint4 v) {
        *reinterpret_cast<uint4*>(dst + c) = v;
        if (!p.most) return;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int left = p.dim - c - 2 * k;
          largest = __vmaxu2(largest, w[k] & (left > 1 ? 0x7FFF7FFFu : left > 0 ? 0x7FFFu : 0u));
        }
      };
      if (p.vec) {
#pragma unroll 4
        for (int c = 8 * lane; c < p.dim; c += 256) put(c, *reinterpret_cast<const uint4*>(src + c));
      } else {
        const uintptr_t begin = reinterpret_cast<uintptr_t>(p.hidden), end = reinterpret_cast<uintptr_t>(p.hidden + (p.tokens - 1) * p.ld_hidden + p.dim);
#pragma unroll 4
        for (int c = 8 * lane; c < p.dim; c += 256) put(c, eight_of_row(src + c, p.dim - c, begin, end));
      }
    }
  }
  if (p.most) {
    __shared__ float row_most[kRowsPerBlock];
    largest = __reduce_max_sync(0xffffffffu, max(largest & 0xFFFFu, largest >> 16));
    if (lane == 0) row_most[warp] = mine ? ldexpf(__half2float(__ushort_as_half((uint16_t)largest)), -lift_of(p.weight[token] * scale)) : 0.f;
    __syncthreads();
    if (tid == 0) {
      float m = 0.f;
      for (int w = 0; w < kRowsPerBlock; ++w) m = fmaxf(m, row_most[w]);
      p.most[blockIdx.x] = m;
    }
  }
  if (blockIdx.x == gridDim.x - 1) {
    int total = before;
    for (int w = 0; w < kRowsPerBlock; ++w) total += has[w];
    if (tid == 0) *p.count = total;
    if (p.pad == 0) return;
    // k of a product
    const int pad = (total + p.pad - 1) / p.pad * p.pad - total;
    uint4* to = reinterpret_cast<uint4*>(p.packed + (int64_t)total * p.pitch);
    for (int64_t i = tid; i < (int64_t)pad * p.pitch / 8; i += blockDim.x) to[i] = make_uint4(0, 0, 0, 0);
  }
}

// Packed fp16 rows times 2^(s - lift), s such that the largest element of all comes to between 2^13 and 2^14 (or stays, where it is larger);
// zeros up to a multiple of `pad` rows.  scale[2]: what the product with them is multiplied by.
__global__ void __launch_bounds__(256) lift_kernel(const uint16_t* packed, const int* lift, const float* most, int parts, const int* count, int pitch, int pad, uint16_t* out,
                                                   float* scale) {
  tck::chain_wait();
  __shared__ uint32_t top;
  if (threadIdx.x == 0) top = 0;
  __syncthreads();
  float m = 0.f;
  for (int i = threadIdx.x; i < parts; i += 256) m = fmaxf(m, most[i]);
  atomicMax(&top, __reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // not negative: bits are ordered as values are
  __syncthreads();
  const int s = lift_of(__uint_as_float(top));
  if (blockIdx.x == 0 && threadIdx.x == 0) scale[2] = ldexpf(scale[1], -s);
  const int n = *count, rows = (n + pad - 1) / pad * pad, lane = threadIdx.x & 31;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
    const float factor = r < n ? ldexpf(1.f, s - lift[r]) : 0.f;
#pragma unroll 4
    for (int c = 8 * lane; c < pitch; c += 256) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < n) {
        v = *reinterpret_cast<const uint4*>(packed + (int64_t)r * pitch + c);
        __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = __half22float2(h[k]);
          h[k] = __floats2half2_rn(f.x * factor, f.y * factor);
        }
      }
      *reinterpret_cast<uint4*>(out + (int64_t)r * pitch + c) = v;
    }
  }
}

// Rows whose 16-byte alignment the copy engine needs (a piece of the table).
__global__ void __launch_bounds__(256) align_kernel(const uint16_t* src, int64_t ld, int rows, int dim, int pitch, uint16_t* dst) {
  tck::chain_wait();
  const uint32_t per = (uint32_t)(dim + 7) / 8;
  const int64_t total = (int64_t)rows * per, stride = (int64_t)gridDim.x * 256;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(src), end = reinterpret_cast<uintptr_t>(src + (rows - 1) * ld + dim);
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
    const int64_t r = total <= UINT32_MAX ? (uint32_t)i / per : i / per;
    const int c = (int)(i - r * per) * 8;
    *reinterpret_cast<uint4*>(dst + r * pitch + c) = eight_of_row(src + r * ld + c, dim - c, begin, end);
  }
}

// Parts of a row's statistics -> logsumexp and loss.  Rows per block; the block's other threads take the parts in turn, four at
// a time under way: 8 rows where there are many (neighbouring rows' parts lie next to each other), one where there are few.  count: of
// all rows, of which these begin at `first`.  source and count null: rows are tokens, those without a target among them.
template <int Rows>
__global__ void __launch_bounds__(256) combine_kernel(const float2* part, int parts, uint32_t pitch, const float* hit, const int* source, const int* count,
                                                      int first, const void* targets, int wide, int tokens, int64_t vocab, float* loss, float* lse) {
  tck::chain_wait();
  constexpr int Turns = 256 / Rows;
  __shared__ float2 all[Turns][Rows];
  const int r = threadIdx.x % Rows, turn = threadIdx.x / Rows;
  const int row = blockIdx.x * Rows + r, n = count ? min(*count - first, tokens) : tokens;
  if ((int)blockIdx.x * Rows >= n) return;
  auto join = [](float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x);
    const float shift = top == -INFINITY ? 0.f : top;
    return make_float2(top, a.y * exp2f((a.x - shift) * kLog2e) + b.y * exp2f((b.x - shift) * kLog2e));
  };
  float2 got = make_float2(-INFINITY, 0.f);
  if (row < n)
    for (int i = turn; i < parts; i += 4 * Turns) {
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = i + u * Turns < parts ? part[(size_t)(i + u * Turns) * pitch + row] : make_float2(-INFINITY, 0.f);
      got = join(got, join(join(v[0], v[1]), join(v[2], v[3])));
    }
  all[turn][r] = got;
  __syncthreads();
  for (int half = Turns / 2; half; half /= 2) {
    if (turn < half) all[turn][r] = join(all[turn][r], all[turn + half][r]);
    __syncthreads();
  }
  if (turn != 0 || row >= n) return;
  got = all[0][r];
  const float l = got.x + logf(got.y);
  if (source) {
    lse[source[row]] = l;
    loss[source[row]] = l - hit[row];
  } else {
    const int64_t t = index_at(targets, row, wide);
    const bool part_of_it = t >= 0 && t < vocab;
    lse[row] = part_of_it ? l : 0.f;
    loss[row] = part_of_it ? l - hit[row] : 0.f;
  }
}

// The scale of scale_for() over many tokens, which packing blocks do not look for themselves.
__global__ void __launch_bounds__(1024) weight_scale_kernel(const void* targets, int wide, int64_t tokens, int64_t vocab, const float* weight, float range, float* scale) {
  tck::chain_wait();
  __shared__ uint32_t most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  float m = 0.f;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < tokens; i += 1024) {
    const int64_t t = index_at(targets, i, wide);
    if (t >= 0 && t < vocab) m = fmaxf(m, fabsf(weight[i]));
  }
  atomicMax(&most, __reduce_max_sync(0xffffffffu, __float_as_uint(m)));
  __syncthreads();
  if (threadIdx.x) return;
  const float2 both = scale_for(__uint_as_float(most), range);
  scale[0] = both.x;
  scale[1] = both.y;
}

// Sum of the slices' partial gradients, scaled and rounded once, to each token's row; zeros for the others.
__global__ void __launch_bounds__(256) hidden_grad_kernel(const float* slab, int slices, int64_t slab_rows, int pitch, const int* packed_of, int64_t tokens, int dim,
                                                          const float* scale, const int* lift, int bf, int vec, uint16_t* out, int64_t ld) {
  tck::chain_wait();
  auto pack = [&](float a, float b) {
    if (bf) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
      return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  const uint32_t per = (uint32_t)(dim + 3) / 4;
  const int64_t total = tokens * per, stride = (int64_t)gridDim.x * 256;
  for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < total; j += stride) {
    const int64_t t = total <= UINT32_MAX ? (uint32_t)j / per : j / per;
    const int c = (int)(j - t * per) * 4, row = packed_of[t];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float s = scale[1];
    if (row >= 0) {
      if (lift) s = ldexpf(s, -lift[row]);
#pragma unroll 8
      for (int i = 0; i < slices; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(slab + ((int64_t)i * slab_rows + row) * pitch + c);
        v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
      }
    }
    const uint32_t lo = pack(v.x * s, v.y * s), hi = pack(v.z * s, v.w * s);
    uint16_t* dst = out + t * ld + c;
    if (vec) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    } else {
      dst[0] = (uint16_t)lo;
      if (c + 1 < dim) dst[1] = (uint16_t)(lo >> 16);
      if (c + 2 < dim) dst[2] = (uint16_t)hi;
      if (c + 3 < dim) dst[3] = (uint16_t)(hi >> 16);
    }
  }
}

// ---- few tokens ----
// Up to kFew tokens (of as many columns as kFewBytes hold: 2560) everything is a pass over the table: its rows are read as they lie, whatever their alignment, products are fp32
// multiply-adds, and nothing is padded to tiles.  Bound by the table's bytes under way and by the launches.  Measured against the
// products on tensor cores, us: loss of one token, 31703 x 77 16.5 -> 11.3, of four, 9000 x 999 26.7 -> 15.9, 131072 x 2048 131 -> 127;
// loss and gradients of four, 9000 x 999 91 -> 67, of three, 41621 x 1731 417 -> 353 (there two passes are copies to aligned rows), of two,
// 32000 x 512 62 -> 56.  Gradients of three and four tokens over aligned rows take longer this way (6456 x 1576 55 -> 70, 20000 x 712
// 69 -> 79), but keep G in fp32: a gradient by the table is then off by its own rounding alone, where with so few tokens to
// average over G's rounding would add as much again (3 x 1920 x 115943 in fp16 3.0e-4 off instead of 2.1e-4).
constexpr int kFew = 4, kFewSlices = 1024;  // most tokens; most blocks along the table
constexpr int64_t kFewBytes = 40960;        // of the tokens' rows in shared memory, fp32

template <bool Bf>
__device__ __forceinline__ float few_value(uint32_t bits) {
  return Bf ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((uint16_t)bits));
}
template <bool Bf>
__device__ __forceinline__ uint16_t few_bits(float v) {
  return Bf ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
template <bool Bf, int Vec>
__device__ __forceinline__ void few_load(const uint16_t* p, float (&f)[Vec]) {
  if constexpr (Vec == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = few_value<Bf>(w[k / 2] >> (16 * (k & 1)) & 0xFFFFu);
  } else {
    f[0] = few_value<Bf>(*p);
  }
}

struct FewArgs {
  const uint16_t *hidden, *weight;
  int64_t ld_hidden, ld_weight, vocab;
  int dim, tokens;         // rows of hidden; with `count`, those from it on do not take part
  const int* count;
  // statistics
  const void* targets;
  int wide;
  float* hit;
  float2* part;            // [8 per block][pitch]
  uint32_t pitch;
  // gradients
  const WmRow* rows;
  float* probs;            // [vocab][kFew]: the loss's gradient by each logit
  uint16_t* dweight;
  int64_t ld_dweight;
  float* slab;             // [slices][slab_rows][slab_pitch]
  int64_t slab_rows, slab_pitch;
  const float* scale;      // scale[1]: what the rows' weights have to be multiplied by
};

// Logits of Few tokens, four rows of the table per warp at a time, the tokens' rows in shared memory: their statistics (Prob false)
// or the gradients by them.
template <bool Bf, int Vec, int Few, bool Prob>
__global__ void __launch_bounds__(256) few_logits_kernel(const FewArgs p) {
  tck::chain_wait();
  extern __shared__ float few_smem[];  // [Few][dim rounded up to 8]
  constexpr int R = 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, pitch = (p.dim + 7) / 8 * 8;
  const int n = p.count ? min(*p.count, p.tokens) : p.tokens;
  for (int i = tid; i < Few * pitch; i += 256) {
    const int t = i / pitch, c = i - t * pitch;
    few_smem[i] = t < n && c < p.dim ? few_value<Bf>(p.hidden[t * p.ld_hidden + c]) : 0.f;
  }
  __syncthreads();
  // lane t of the first Few: token t
  int64_t target = -1;
  float lse2 = 0.f, weight = 0.f, top = -INFINITY, sum = 0.f;
  if (lane < n) {
    if constexpr (Prob) {
      const WmRow r = p.rows[lane];
      target = r.target;
      lse2 = r.lse2;
      weight = r.weight * p.scale[1];
    } else {
      target = index_at(p.targets, lane, p.wide);
    }
  }
  for (int64_t v0 = ((int64_t)blockIdx.x * 8 + warp) * R; v0 < p.vocab; v0 += (int64_t)gridDim.x * 8 * R) {
    float acc[R][Few] = {};
    const uint16_t* row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) row[r] = p.weight + min(v0 + r, p.vocab - 1) * p.ld_weight;
#pragma unroll 4
    for (int c = lane * Vec; c < p.dim; c += 32 * Vec) {
      float w[R][Vec];
#pragma unroll
      for (int r = 0; r < R; ++r) few_load<Bf, Vec>(row[r] + c, w[r]);
#pragma unroll
      for (int t = 0; t < Few; ++t) {
        const float* h = few_smem + t * pitch + c;
#pragma unroll
        for (int k = 0; k < Vec; k += 4) {
          if constexpr (Vec == 8) {
            const float4 q = *reinterpret_cast<const float4*>(h + k);
#pragma unroll
            for (int r = 0; r < R; ++r)
              acc[r][t] = fmaf(q.w, w[r][k + 3], fmaf(q.z, w[r][k + 2], fmaf(q.y, w[r][k + 1], fmaf(q.x, w[r][k], acc[r][t]))));
          } else {
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][t] = fmaf(h[0], w[r][0], acc[r][t]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mine = 0.f;
#pragma unroll
      for (int t = 0; t < Few; ++t) {
        float z = acc[r][t];
#pragma unroll
        for (int d = 16; d; d >>= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
        if (lane == t) mine = z;
      }
      const int64_t v = v0 + r;
      if (v >= p.vocab) break;
      if constexpr (Prob) {
        if (lane < kFew) p.probs[v * kFew + lane] = lane < n ? (exp2f(fmaf(mine, kLog2e, -lse2)) - (v == target ? 1.f : 0.f)) * weight : 0.f;
      } else if (lane < n) {
        if (v == target) p.hit[lane] = mine;
        const float m = fmaxf(top, mine), shift = m == -INFINITY ? 0.f : m * kLog2e;
        sum = sum * exp2f(fmaf(top, kLog2e, -shift)) + exp2f(fmaf(mine, kLog2e, -shift));
        top = m;
      }
    }
  }
  if (!Prob && lane < n) p.part[(size_t)(blockIdx.x * 8 + warp) * p.pitch + lane] = make_float2(top, sum);
}

// Both gradients from the gradients by the logits: block x a slice of the table's rows, block y columns.  `groups` rows at a time
// where a row takes less than the block's threads.
template <bool Bf, int Vec, int Few>
__global__ void __launch_bounds__(256) few_grads_kernel(const FewArgs p, int columns, int want_hidden) {
  tck::chain_wait();
  extern __shared__ float few_smem[];  // [groups][Few][columns]
  const int tid = threadIdx.x, lanes = columns / Vec, groups = 256 / lanes, group = tid / lanes, at = (tid - group * lanes) * Vec;
  const int c = blockIdx.y * columns + at, n = min(*p.count, p.tokens);
  const bool mine = group < groups && c < p.dim;
  float h[Few][Vec], acc[Few][Vec] = {};
#pragma unroll
  for (int t = 0; t < Few; ++t) {
#pragma unroll
    for (int k = 0; k < Vec; ++k) h[t][k] = 0.f;
    if (mine && t < n) few_load<Bf, Vec>(p.hidden + t * p.ld_hidden + c, h[t]);
  }
  const int64_t from = p.vocab * blockIdx.x / gridDim.x, to = p.vocab * (blockIdx.x + 1) / gridDim.x;
  constexpr int U = Vec == 1 ? 8 : 4;  // rows under way: all are read before one is written
  if (mine)
    for (int64_t v0 = from + group; v0 < to; v0 += U * groups) {
      float4 g[U];
      float w[U][Vec];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t v = min(v0 + u * groups, to - 1);
        g[u] = *reinterpret_cast<const float4*>(p.probs + v * kFew);
        if (want_hidden) few_load<Bf, Vec>(p.weight + v * p.ld_weight + c, w[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t v = v0 + u * groups;
        if (v >= to) break;
        const float gs[4] = {g[u].x, g[u].y, g[u].z, g[u].w};
        if (want_hidden) {
#pragma unroll
          for (int t = 0; t < Few; ++t)
#pragma unroll
            for (int k = 0; k < Vec; ++k) acc[t][k] = fmaf(gs[t], w[u][k], acc[t][k]);
        }
        if (!p.dweight) continue;
        float d[Vec] = {};
#pragma unroll
        for (int t = 0; t < Few; ++t)
#pragma unroll
          for (int k = 0; k < Vec; ++k) d[k] = fmaf(gs[t], h[t][k], d[k]);
        uint16_t* dst = p.dweight + v * p.ld_dweight + c;
        if constexpr (Vec == 8) {
          uint32_t b[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) b[k] = (uint32_t)few_bits<Bf>(d[2 * k]) | (uint32_t)few_bits<Bf>(d[2 * k + 1]) << 16;
          *reinterpret_cast<uint4*>(dst) = make_uint4(b[0], b[1], b[2], b[3]);
        } else {
          *dst = few_bits<Bf>(d[0]);
        }
      }
    }
  if (!want_hidden) return;
  if (mine) {
#pragma unroll
    for (int t = 0; t < Few; ++t)
#pragma unroll
      for (int k = 0; k < Vec; ++k) few_smem[(group * Few + t) * columns + at + k] = acc[t][k];
  }
  __syncthreads();
  for (int i = tid; i < Few * columns; i += 256) {
    const int t = i / columns, a = i - t * columns, col = blockIdx.y * columns + a;
    if (col >= p.dim || t >= p.tokens) continue;
    float s = 0.f;
    for (int g = 0; g < groups; ++g) s += few_smem[(g * Few + t) * columns + a];
    p.slab[(blockIdx.x * p.slab_rows + t) * p.slab_pitch + col] = s;
  }
}

// Sum of the slices' partial gradients of few tokens: 32 columns of a token per block, eight warps take the slices in turn.
__global__ void __launch_bounds__(256) few_hidden_kernel(const float* slab, int slices, int64_t slab_rows, int64_t pitch, const int* packed_of, int dim, int bf, uint16_t* out,
                                                         int64_t ld) {
  tck::chain_wait();
  __shared__ float part[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, t = blockIdx.y, row = packed_of[t];
  float s = 0.f;
  if (row >= 0 && c < dim)
#pragma unroll 8
    for (int i = warp; i < slices; i += 8) s += slab[(i * slab_rows + row) * pitch + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= dim) return;
  for (int w = 1; w < 8; ++w) s += part[w][lane];
  out[t * ld + c] = bf ? __bfloat16_as_ushort(__float2bfloat16_rn(s)) : __half_as_ushort(__float2half_rn(s));
}

// ---- sizes ----
constexpr int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
bool few_fits(int64_t pitch) { return kFew * pitch * 4 <= kFewBytes; }
struct Sizes {
  int64_t rows, pitch, slab_pitch;
  int64_t piece;     // rows of the table whose G is held at a time ...
  int64_t laid_out;  // ... and that are copied at a time where the copy engine cannot address them
  int64_t pieces, parts;
  int slices_most;
  bool only_few;     // every call is a pass over the table
};
// The table in pieces of at most `most` rows, as equal as whole tiles allow.
int64_t piece_of(int64_t vocab, int64_t most) {
  const int64_t pieces = (vocab + most - 1) / most;
  return std::min<int64_t>(up(vocab, 8), up((vocab + pieces - 1) / pieces, 256));
}
Sizes sizes_of(const TcOpShape& p) {
  Sizes s;
  s.rows = up(p.tokens, 128);
  s.pitch = up(p.dim, 8);
  s.slab_pitch = up(p.dim, 4);
  s.only_few = p.tokens <= kFew && few_fits(s.pitch);
  // A piece's G takes at most 256 MB, a piece of the table that has to be laid out as much.
  s.piece = piece_of(p.vocab, std::max<int64_t>(256, (int64_t(1) << 27) / s.rows / 256 * 256));
  s.pieces = (p.vocab + s.piece - 1) / s.piece;
  s.laid_out = std::min(s.piece, piece_of(p.vocab, std::max<int64_t>(256, (int64_t(1) << 27) / s.pitch / 256 * 256)));
  s.parts = std::max((2 * ((p.vocab + 127) / 128) + 2 * ((p.vocab + s.laid_out - 1) / s.laid_out)) * std::min(s.rows, kStatsRows), int64_t(8) * kFew * 4 * p.sms);
  // ... and the partial gradients 256 MB where one slice takes less
  s.slices_most = (int)std::max<int64_t>(1, std::min<int64_t>(64, (int64_t(1) << 26) / (s.rows * s.slab_pitch)));
  return s;
}

struct Buffers {
  uint16_t *packed, *lifted, *piece, *grads;
  int64_t* target;
  int *source, *packed_of, *count, *chunks, *lift;
  float2* part;
  float *hit, *scale, *slab, *probs, *most;
  WmRow* rows;
};
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  const Sizes s = sizes_of(p);
  TcCarver c{base};
  b->packed = c.take<uint16_t>(s.rows * s.pitch);
  const bool lifts = p.dtype == TC_F16 && !s.only_few;
  b->lifted = c.take<uint16_t>(lifts ? s.rows * s.pitch : 0);
  b->lift = c.take<int>(lifts ? s.rows : 0);
  b->most = c.take<float>(lifts ? s.rows / kRowsPerBlock : 0);
  b->piece = c.take<uint16_t>(s.only_few ? 0 : s.laid_out * s.pitch);
  b->grads = c.take<uint16_t>(s.only_few ? 0 : s.rows * up(s.piece, 8));
  b->target = c.take<int64_t>(s.rows);
  b->source = c.take<int>(s.rows);
  b->packed_of = c.take<int>(s.rows);
  b->chunks = c.take<int>((p.tokens + kCountChunk - 1) / kCountChunk);
  b->count = c.take<int>(1);
  b->part = c.take<float2>(s.parts);
  b->hit = c.take<float>(s.rows);
  b->scale = c.take<float>(3);
  const int64_t few_rows = few_fits(s.pitch) ? std::min<int64_t>(p.tokens, kFew) : 0;
  b->slab = c.take<float>(std::max<size_t>(s.only_few ? 0 : (size_t)s.slices_most * s.rows * s.slab_pitch, (size_t)kFewSlices * few_rows * s.slab_pitch));
  b->probs = c.take<float>(p.vocab * kFew);
  b->rows = c.take<WmRow>(s.rows);
  return c.used;
}

struct Call {
  const tc_op_plan& p;
  Sizes s;
  Buffers b;
  int64_t tokens;
  const void* targets;
  int wide;
  cudaStream_t stream;
};

int launch_pack(const Call& c, PackArgs a, const void* hidden, int64_t ld) {
  a.targets = c.targets;
  a.tokens = c.tokens;
  a.vocab = c.p.vocab;
  a.wide = c.wide;
  a.chunk_counts = nullptr;
  if (c.tokens > kCountedDirectly) {
    const unsigned n = (unsigned)((c.tokens + kCountChunk - 1) / kCountChunk);
    TC_CUDA_OK(tck::launch_chained(true, count_kernel, dim3(n), 256u, 0, c.stream, c.targets, c.wide, c.tokens, c.p.vocab, c.b.chunks));
    a.chunk_counts = c.b.chunks;
  }
  a.hidden = static_cast<const uint16_t*>(hidden);
  a.ld_hidden = ld;
  a.dim = (int)c.p.dim;
  a.pitch = (int)c.s.pitch;
  a.vec = c.p.dim % 8 == 0 && ld % 8 == 0 && !(reinterpret_cast<uintptr_t>(hidden) & 15);
  a.packed = c.b.packed;
  a.count = c.b.count;
  const unsigned blocks = (unsigned)((c.tokens + kRowsPerBlock - 1) / kRowsPerBlock);
  TC_CUDA_OK(tck::launch_chained(true, pack_kernel, dim3(blocks), 32u * kRowsPerBlock, 0, c.stream, a));
  return TC_OK;
}

// The table's rows v0 .. v0 + n as an operand: in place, or copied where the copy engine cannot address them.
int piece_operand(const Call& c, const void* weight, int64_t ld, int64_t v0, int64_t n, WmOperand* out) {
  const uint16_t* w = static_cast<const uint16_t*>(weight) + v0 * ld;
  *out = WmOperand{w, ld, 0};
  if (wm_boxable(weight, ld, 0, 2)) return TC_OK;
  TC_CUDA_OK(tck::launch_chained(true, align_kernel, dim3((unsigned)std::min<int64_t>((n * c.s.pitch / 8 + 255) / 256, 8 * c.p.sms)), 256u, 0, c.stream, w, ld, (int)n, (int)c.p.dim,
                                 (int)c.s.pitch, c.b.piece));
  *out = WmOperand{c.b.piece, c.s.pitch, 0};
  return TC_OK;
}

WmArgs base_args(const Call& c) {
  WmArgs a{};
  a.batch = a.slices = 1;
  a.count = c.b.count;
  a.bf16 = c.p.dtype == TC_BF16;
  a.status = c.p.status;
  a.spin_limit = c.p.test_fault ? 1u << 14 : TC_SPIN_LIMIT;
  a.test_fault = c.p.test_fault;
  return a;
}

bool few(const Call& c) { return c.tokens <= kFew && few_fits(c.s.pitch); }
// 16-byte pieces of rows
bool whole_pieces(const void* p, int64_t ld, int64_t dim) { return dim % 8 == 0 && ld % 8 == 0 && !(reinterpret_cast<uintptr_t>(p) & 15); }

template <bool Bf, int Few, bool Prob>
int launch_few_logits(const Call& c, const FewArgs& a, int blocks) {
  const bool vec = whole_pieces(a.weight, a.ld_weight, c.p.dim);
  TC_CUDA_OK(tck::launch_chained(true, vec ? few_logits_kernel<Bf, 8, Few, Prob> : few_logits_kernel<Bf, 1, Few, Prob>, dim3((unsigned)blocks), 256u,
                                 (size_t)(Few * c.s.pitch * 4), c.stream, a));
  return TC_OK;
}
template <bool Prob>
int few_logits(const Call& c, const FewArgs& a, int blocks) {
  const bool bf = c.p.dtype == TC_BF16;
  if (c.tokens <= 2) return bf ? launch_few_logits<true, 2, Prob>(c, a, blocks) : launch_few_logits<false, 2, Prob>(c, a, blocks);
  return bf ? launch_few_logits<true, 4, Prob>(c, a, blocks) : launch_few_logits<false, 4, Prob>(c, a, blocks);
}
template <bool Bf, int Few>
int launch_few_grads(const Call& c, const FewArgs& a, bool want_hidden, int* slices) {
  const bool vec = whole_pieces(a.weight, a.ld_weight, c.p.dim) && (!a.dweight || whole_pieces(a.dweight, a.ld_dweight, c.p.dim));
  const int unit = vec ? 8 : 1;
  int columns = 256 * unit;  // of a block: fewer where the row has fewer
  while (columns / 2 >= c.p.dim && columns / unit > 32) columns /= 2;
  const int64_t across = (c.p.dim + columns - 1) / columns, groups = 256 * unit / columns;
  *slices = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kFewSlices, ((vec ? 2 : 6) * c.p.sms + across - 1) / across), c.p.vocab / (8 * groups)));
  const size_t smem = want_hidden ? (size_t)(groups * Few * columns * 4) : 0;
  TC_CUDA_OK(tck::launch_chained(true, vec ? few_grads_kernel<Bf, 8, Few> : few_grads_kernel<Bf, 1, Few>, dim3((unsigned)*slices, (unsigned)across), 256u, smem, c.stream, a,
                                 columns, (int)want_hidden));
  return TC_OK;
}

int few_blocks(const Call& c, int64_t rows) { return (int)std::min<int64_t>(4 * c.p.sms, (rows + 31) / 32); }

int few_forward(const Call& c, float* loss, float* lse, const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight) {
  FewArgs a{};
  a.hidden = static_cast<const uint16_t*>(hidden);
  a.weight = static_cast<const uint16_t*>(weight);
  a.ld_hidden = ld_hidden;
  a.ld_weight = ld_weight;
  a.vocab = c.p.vocab;
  a.dim = (int)c.p.dim;
  a.tokens = (int)c.tokens;
  a.targets = c.targets;
  a.wide = c.wide;
  a.hit = c.b.hit;
  a.part = c.b.part;
  a.pitch = kFew;
  const int blocks = few_blocks(c, c.p.vocab);
  const int st = few_logits<false>(c, a, blocks);
  if (st != TC_OK) return st;
  TC_CUDA_OK(tck::launch_chained(true, combine_kernel<1>, dim3((unsigned)c.tokens), 256u, 0, c.stream, c.b.part, 8 * blocks, (uint32_t)kFew, c.b.hit,
                                 static_cast<const int*>(nullptr), static_cast<const int*>(nullptr), 0, c.targets, c.wide, (int)c.tokens, c.p.vocab, loss, lse));
  return TC_OK;
}

// After packing.
int few_backward(const Call& c, bool want_hidden, void* dweight, int64_t ld_dweight, const void* weight, int64_t ld_weight, int* slices) {
  const bool bf = c.p.dtype == TC_BF16;
  FewArgs a{};
  a.hidden = c.b.packed;
  a.weight = static_cast<const uint16_t*>(weight);
  a.ld_hidden = c.s.pitch;
  a.ld_weight = ld_weight;
  a.vocab = c.p.vocab;
  a.dim = (int)c.p.dim;
  a.tokens = (int)c.tokens;
  a.count = c.b.count;
  a.rows = c.b.rows;
  a.probs = c.b.probs;
  a.dweight = static_cast<uint16_t*>(dweight);
  a.ld_dweight = ld_dweight;
  a.slab = c.b.slab;
  a.slab_rows = c.tokens;
  a.slab_pitch = c.s.slab_pitch;
  a.scale = c.b.scale;
  const int st = few_logits<true>(c, a, few_blocks(c, c.p.vocab));
  if (st != TC_OK) return st;
  if (c.tokens <= 2) return bf ? launch_few_grads<true, 2>(c, a, want_hidden, slices) : launch_few_grads<false, 2>(c, a, want_hidden, slices);
  return bf ? launch_few_grads<true, 4>(c, a, want_hidden, slices) : launch_few_grads<false, 4>(c, a, want_hidden, slices);
}

int forward(const Call& c, float* loss, float* lse, const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight) {
  if (few(c)) return few_forward(c, loss, lse, hidden, ld_hidden, weight, ld_weight);
  // Few tokens are one tile of rows with or without those that take no part: their rows are left where they are, and statistics
  // of rows without a target go nowhere.
  const bool packed = c.tokens > kUnpacked || !wm_boxable(hidden, ld_hidden, 0, 2);
  int st = TC_OK;
  if (packed) {
    PackArgs a{};
    a.target = c.b.target;
    a.source = c.b.source;
    a.loss = loss;
    a.lse = lse;
    st = launch_pack(c, a, hidden, ld_hidden);
    if (st != TC_OK) return st;
  }
  const bool in_place = wm_boxable(weight, ld_weight, 0, 2);
  const int64_t step = in_place ? c.p.vocab : c.s.laid_out;
  // Blocks of rows, so that statistics take a bounded place: each goes through the table once.
  for (int64_t r0 = 0; r0 < c.tokens; r0 += kStatsRows) {
    const int64_t rows = std::min(kStatsRows, c.tokens - r0), pitch = up(rows, 64);
    int64_t parts = 0;
    for (int64_t v0 = 0; v0 < c.p.vocab; v0 += step) {
      const int64_t n = std::min(step, c.p.vocab - v0);
      WmOperand w;
      st = piece_operand(c, weight, ld_weight, v0, n, &w);
      if (st != TC_OK) return st;
      int tile, slices;
      wm_choose(WM_STATS, rows, n, c.p.dim, 1, 1, c.p.sms, &tile, &slices);
      WmArgs m = base_args(c);
      m.M = (uint32_t)rows;
      m.N = (uint32_t)n;
      m.K = (uint32_t)c.p.dim;
      m.count_first = (int32_t)r0;
      if (!packed) m.count = nullptr;
      m.stats = WmStatsArgs{packed ? static_cast<const void*>(c.b.target + r0) : c.targets, packed ? 1 : c.wide, c.b.hit + r0, c.b.part, (uint32_t)pitch,
                            (uint32_t)parts, v0};
      st = wm_launch(WM_STATS, tile, m, packed ? WmOperand{c.b.packed + r0 * c.s.pitch, c.s.pitch, 0} : WmOperand{hidden, ld_hidden, 0}, w, c.p.sms, c.stream);
      if (st != TC_OK) return st;
      parts += 2 * ((n + wm_tile_n(tile) - 1) / wm_tile_n(tile));
    }
    const bool many = rows > 64;
    TC_CUDA_OK(tck::launch_chained(true, many ? combine_kernel<8> : combine_kernel<1>, dim3((unsigned)(many ? (rows + 7) / 8 : rows)), 256u, 0, c.stream, c.b.part,
                                   (int)parts, (uint32_t)pitch, c.b.hit + r0, packed ? c.b.source + r0 : nullptr, packed ? c.b.count : nullptr, (int)r0, c.targets, c.wide,
                                   (int)rows, c.p.vocab, loss, lse));
  }
  return TC_OK;
}

int backward(const Call& c, void* dhidden, int64_t ld_dhidden, void* dweight, int64_t ld_dweight, const void* hidden, int64_t ld_hidden, const void* weight,
             int64_t ld_weight, const float* lse, const float* grad) {
  const bool bf = c.p.dtype == TC_BF16;
  float* scale = c.b.scale;
  const float range = bf ? 1.f : 16384.f;
  if (c.tokens > kScaledDirectly)
    TC_CUDA_OK(tck::launch_chained(true, weight_scale_kernel, dim3(1), 1024u, 0, c.stream, c.targets, c.wide, c.tokens, c.p.vocab, grad, range, scale));
  const int64_t piece = wm_boxable(weight, ld_weight, 0, 2) ? c.s.piece : c.s.laid_out, pieces = (c.p.vocab + piece - 1) / piece;
  int grads_tile = 0, slices = 1;
  wm_choose_grads(dhidden ? c.tokens : 0, c.p.dim, piece, dweight ? piece : 0, c.p.dim, c.tokens, c.s.slices_most, c.p.sms, &grads_tile, &slices);
  const int64_t krows = up(c.tokens, 128);
  auto stage = [&](int64_t n) { return wm_grads_stage(n, krows, grads_tile); };
  const int pad = std::max(stage(std::min(piece, c.p.vocab)), stage(c.p.vocab - (pieces - 1) * piece));  // of all pieces
  PackArgs a{};
  a.packed_of = c.b.packed_of;
  a.pad = pad;
  a.lse_in = lse;
  a.weight = grad;
  a.weight_scale = scale;
  a.range = c.tokens > kScaledDirectly ? 0.f : range;
  a.rows = c.b.rows;
  const bool by_few = few(c);
  if (by_few) a.pad = 0;
  const bool lifts = !bf && !by_few;
  a.lift = lifts ? c.b.lift : nullptr;
  a.most = lifts && dweight ? c.b.most : nullptr;
  int st = launch_pack(c, a, hidden, ld_hidden);
  if (st != TC_OK) return st;
  const WmOperand h{c.b.packed, c.s.pitch, 0}, h2{lifts ? c.b.lifted : c.b.packed, c.s.pitch, 0};
  if (a.most) {
    const int64_t blocks = (c.tokens + kRowsPerBlock - 1) / kRowsPerBlock;
    TC_CUDA_OK(tck::launch_chained(true, lift_kernel, dim3((unsigned)std::min<int64_t>((c.tokens + pad + 7) / 8, 4 * c.p.sms)), 256u, 0, c.stream, c.b.packed, c.b.lift, c.b.most, (int)blocks,
                                   c.b.count, (int)c.s.pitch, pad, c.b.lifted, scale));
  }
  const int64_t gpitch = up(piece, 8), slab_rows = by_few ? c.tokens : c.s.rows;
  if (by_few) {
    st = few_backward(c, dhidden != nullptr, dweight, ld_dweight, weight, ld_weight, &slices);
    if (st != TC_OK) return st;
  }
  for (int64_t v0 = by_few ? c.p.vocab : 0; v0 < c.p.vocab; v0 += piece) {
    const int64_t n = std::min(piece, c.p.vocab - v0);
    WmOperand w;
    st = piece_operand(c, weight, ld_weight, v0, n, &w);
    if (st != TC_OK) return st;
    int tile, one;
    WmArgs m = base_args(c);
    m.M = (uint32_t)c.tokens;
    m.N = (uint32_t)n;
    m.K = (uint32_t)c.p.dim;
    m.out = WmOut{c.b.grads, gpitch, 1, 0, 1, bf, 1};
    m.prob = WmProbArgs{c.b.rows, v0, (uint32_t)c.s.rows, (uint32_t)pad};
    wm_choose(WM_PROB, c.tokens, n, c.p.dim, 1, 1, c.p.sms, &tile, &one);
    st = wm_launch(WM_PROB, tile, m, h, w, c.p.sms, c.stream);
    if (st != TC_OK) return st;
    const WmOperand g{c.b.grads, gpitch, 0};
    m = base_args(c);
    m.M = dhidden ? (uint32_t)c.tokens : 0;
    m.N = (uint32_t)c.p.dim;
    m.K = (uint32_t)n;
    m.slices = (uint32_t)slices;
    m.grads = WmGradsArgs{v0 > 0, scale + (lifts ? 2 : 1)};
    if (dweight) {
      m.second.M = (uint32_t)n;
      m.second.N = (uint32_t)c.p.dim;
      m.second.K = (uint32_t)krows;
      m.out = WmOut{static_cast<uint16_t*>(dweight) + v0 * ld_dweight, ld_dweight, 1, 0, wm_box_output(dweight, c.p.dim, ld_dweight, 0), bf, 1};
    }
    st = wm_launch_grads(grads_tile, m, g, w, c.b.slab, slab_rows, g, h2, c.p.sms, c.stream);
    if (st != TC_OK) return st;
  }
  if (dhidden && by_few) {
    TC_CUDA_OK(tck::launch_chained(true, few_hidden_kernel, dim3((unsigned)((c.p.dim + 31) / 32), (unsigned)c.tokens), 256u, 0, c.stream, c.b.slab, slices, slab_rows,
                                   c.s.slab_pitch, c.b.packed_of, (int)c.p.dim, (int)bf, static_cast<uint16_t*>(dhidden), ld_dhidden));
  } else if (dhidden) {
    const int vec = c.p.dim % 4 == 0 && ld_dhidden % 4 == 0 && !(reinterpret_cast<uintptr_t>(dhidden) & 7);
    TC_CUDA_OK(tck::launch_chained(true, hidden_grad_kernel, dim3((unsigned)std::min<int64_t>((c.tokens * ((c.p.dim + 3) / 4) + 255) / 256, 32 * c.p.sms)), 256u, 0, c.stream, c.b.slab, slices,
                                   slab_rows, (int)c.s.slab_pitch, c.b.packed_of, c.tokens, (int)c.p.dim, scale, a.lift, (int)bf, vec, static_cast<uint16_t*>(dhidden),
                                   ld_dhidden));
  }
  return TC_OK;
}

bool odd_address(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

int check(const tc_op_plan* p, int64_t tokens, const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, const void* targets,
          int index_dtype) {
  if (!p || p->kind != TC_OP_VOCAB_LOSS || !weight || (tokens && (!hidden || !targets)) || (index_dtype != TC_I32 && index_dtype != TC_I64)) return TC_ERR_INVALID_ARG;
  if (tokens < 0 || tokens > p->tokens || ld_hidden < 0 || ld_weight < 0) return TC_ERR_EXTENT;
  if (odd_address(hidden, 2) || odd_address(weight, 2) || odd_address(targets, index_dtype == TC_I64 ? 8 : 4)) return TC_ERR_ALIGNMENT;
  return TC_OK;
}

}  // namespace

size_t tc_loss_workspace(const TcOpShape& p) {
  Buffers b;
  return carve(p, nullptr, &b);
}

int tc_loss_prepare() {
  for (WmKind k : {WM_STATS, WM_PROB, WM_GRADS}) {
    const int st = wm_prepare(k);
    if (st != TC_OK) return st;
  }
  return TC_OK;
}

std::string tc_loss_json(const TcOpShape& p) {
  const Sizes s = sizes_of(p);
  const double product = 2.0 * p.tokens * p.dim * p.vocab;
  return "{\"operator\":\"vocab_loss\",\"dtype\":\"" + std::string(p.dtype == TC_BF16 ? "bf16" : "f16") + "\",\"tokens\":" + std::to_string(p.tokens) +
         ",\"dim\":" + std::to_string(p.dim) + ",\"vocab\":" + std::to_string(p.vocab) + ",\"piece\":" + std::to_string(s.piece) +
         ",\"pieces\":" + std::to_string(s.pieces) + ",\"flops_loss\":" + std::to_string(product) + ",\"flops_grad\":" + std::to_string(3 * product) +
         ",\"workspace_bytes\":" + std::to_string(tc_loss_workspace(p)) + "}";
}

extern "C" int tc_vocab_loss_execute(tc_op_plan* p, float* loss, float* lse, const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight,
                                     const void* targets, int index_dtype, int64_t tokens, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check(p, tokens, hidden, ld_hidden, weight, ld_weight, targets, index_dtype);
  if (st != TC_OK) return st;
  if (tokens && (!loss || !lse)) return TC_ERR_INVALID_ARG;
  if (odd_address(loss, 4) || odd_address(lse, 4)) return TC_ERR_ALIGNMENT;
  TcScratch scratch;
  st = scratch.open(p, TC_OP_VOCAB_LOSS, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  if (st != TC_OK || tokens == 0) return st;
  Call c{*p, sizes_of(*p), {}, tokens, targets, index_dtype == TC_I64, static_cast<cudaStream_t>(stream)};
  carve(*p, scratch.base, &c.b);
  return scratch.close(forward(c, loss, lse, hidden, ld_hidden, weight, ld_weight));
}

extern "C" int tc_vocab_loss_execute_grad(tc_op_plan* p, void* dhidden, int64_t ld_dhidden, void* dweight, int64_t ld_dweight, const void* hidden,
                                          int64_t ld_hidden, const void* weight, int64_t ld_weight, const void* targets, int index_dtype, const float* lse,
                                          const float* grad, int64_t tokens, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check(p, tokens, hidden, ld_hidden, weight, ld_weight, targets, index_dtype);
  if (st != TC_OK) return st;
  if (tokens && (!lse || !grad || (!dhidden && !dweight))) return TC_ERR_INVALID_ARG;
  if ((dhidden && ld_dhidden < p->dim) || (dweight && ld_dweight < p->dim)) return TC_ERR_EXTENT;
  if (odd_address(lse, 4) || odd_address(grad, 4) || odd_address(dhidden, 2) || odd_address(dweight, 2)) return TC_ERR_ALIGNMENT;
  TcScratch scratch;
  st = scratch.open(p, TC_OP_VOCAB_LOSS, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  if (st != TC_OK) return st;
  if (tokens == 0) {  // no tokens: the table's gradient is zero
    if (dweight)
      TC_CUDA_OK(cudaMemset2DAsync(dweight, (size_t)ld_dweight * 2, 0, (size_t)p->dim * 2, (size_t)p->vocab, static_cast<cudaStream_t>(stream)));
    return TC_OK;
  }
  Call c{*p, sizes_of(*p), {}, tokens, targets, index_dtype == TC_I64, static_cast<cudaStream_t>(stream)};
  carve(*p, scratch.base, &c.b);
  return scratch.close(backward(c, dhidden, ld_dhidden, dweight, ld_dweight, hidden, ld_hidden, weight, ld_weight, lse, grad));
}

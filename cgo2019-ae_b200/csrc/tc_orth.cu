// Orthogonalised updates by the Newton-Schulz iteration (tc_orthogonal_execute).
//
//   X <- X / (|X|_F + eps);  then per step   A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// on the orientation with fewer rows than columns: an odd polynomial of each singular value, which the coefficients drive
// towards one.  m x n, m <= n: m m n + m m m + 2 m m n operations per step with the symmetric products' other halves stored
// as mirror images of the computed tiles.
//
// Between the products matrices are held in fp16, 11 bits, not in bf16's 8, at the same rate: singular values stay near one
// at most, so the range is known.  X is held 2^6 times as large (entries of a 4096 x 4096 X start around 2^-12, below which
// fp16 soon loses bits); the input's own norm goes into the first products' fp32 results, so a 16-bit input enters them as it is.
// Sums are fp32 in the tensor core's accumulators, a X + B X is rounded once.  Where the result is fp16, operands are sums of two
// fp16 numbers, 22 bits, and products three (high by high, low by high, high by low).
//
// Up to 128 rows: one launch (the cluster kernel).  Otherwise three products per step, each a launch that begins under the last one's
// end.  5 steps, one B200: 4096 x 4096 1287 us (1.37e12 operations: 1070 TFLOP/s; four rounds of tiles for 3.46 of
// work in X X^T and A A), four 1024 x 4096 376 to 390 us, 1000 x 1333 in two terms 400 us.  There the ten symmetric products take 33 us
// each: 36 tiles on 148 multiprocessors, each over the whole k three times; their sums are not split.  (The others take 32, each launch
// beginning under the end of the one before; four 1024 x 4096: 20 and 37.)  All steps in one kernel whose CTAs wait for one another was slower (160 x 392 92 -> 113 us, 4 of 1024 x 4096 388 -> 465).
#include <algorithm>

#include "tc_inst.cuh"
#include "tc_op.h"
#include "tc_orth_cluster.cuh"
#include "tc_wm.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace {

// The last two of four steps or more, where singular values are near one and A near the identity, work with E = A - 1 instead of A:
//   a X + (b A + c A A) X = (a + b + c) X + ((b + 2 c) E + c E E) X
// A's diagonal, rounded to 11 bits, would be off by 2^-12 and weighed by coefficients that all but cancel; E is small.  A 64 x 128
// result is 9.4e-4 off so, 1.5e-3 without, a 1000 x 1333 one 1.2e-3 and 1.3e-3 (before its own rounding, simulated in 64 bits).
float shift_of(int step, int steps) { return steps >= 4 && step >= steps - 2 ? 1.f : 0.f; }

constexpr int kGuard = 6;        // X is held times 2^kGuard
constexpr int kNormBlocks = 256;  // partial sums of squares per matrix, at most

struct InputArgs {
  const void* x;
  int64_t batch_stride, row_stride, col_stride;  // of the orientation with fewer rows
  int rows, cols, dtype, turn, vec;              // turn: rows lie next to each other, not columns; vec: 16-byte pieces along that index
  double* partial;                               // [batch][kNormBlocks]
};

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
  if (dtype == TC_F32) return static_cast<const float*>(p)[i];
  if (dtype == TC_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
// Eight neighbouring values, 16-byte aligned.
__device__ __forceinline__ void load8(const void* p, int64_t i, int dtype, float* f) {
  if (dtype == TC_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i), b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    return;
  }
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 two = dtype == TC_BF16 ? make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u))
                                        : __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    f[2 * k] = two.x;
    f[2 * k + 1] = two.y;
  }
}
__device__ __forceinline__ const void* matrix(const InputArgs& p, int z) {
  return static_cast<const char*>(p.x) + z * p.batch_stride * (p.dtype == TC_F32 ? 4 : 2);
}
__device__ __forceinline__ double block_sum(double v, double* shared) {  // 256 threads, always in the same order
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < 8; ++w) v += shared[w];
  __syncthreads();
  return v;
}

// Sums of squares: fp32 over eight values where their range allows it, fp64 from there on.
__global__ void __launch_bounds__(256) norm_kernel(const InputArgs p) {
  tck::chain_wait();
  __shared__ double shared[8];
  const void* x = matrix(p, blockIdx.y);
  const int inner = p.turn ? p.rows : p.cols, outer = p.turn ? p.cols : p.rows;
  const int64_t step_in = p.turn ? p.row_stride : p.col_stride, step_out = p.turn ? p.col_stride : p.row_stride;
  const int64_t per = (inner + 7) / 8, total = per * outer, stride = (int64_t)gridDim.x * 256;
  double sum = 0;
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
    const int64_t o = i / per, at = (i - o * per) * 8;
    float f[8];
    if (p.vec) {
      load8(x, o * step_out + at, p.dtype, f);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = at + k < inner ? load_as_float(x, o * step_out + (at + k) * step_in, p.dtype) : 0.f;
    }
    sum += tck::wm_squares8(f);
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) p.partial[blockIdx.y * kNormBlocks + blockIdx.x] = sum;
}

// The power of two that brings a matrix's norm to [2^(kGuard - 1), 2^kGuard); and, from one block, what is left of 1 / (norm + eps).
__device__ __forceinline__ float scale_of(const InputArgs& p, int blocks, double eps, double* shared, float* scale) {
  const double norm = sqrt(block_sum((int)threadIdx.x < blocks ? p.partial[blockIdx.y * kNormBlocks + threadIdx.x] : 0.0, shared));
  int e = 0;
  const bool finite = norm < INFINITY;
  if (norm > 0 && finite) frexp(norm, &e);
  e = min(max(kGuard - e, -126), 126);
  if (blockIdx.x == 0 && threadIdx.x == 0) scale[blockIdx.y] = finite ? (float)(ldexp(1.0, -e) / (norm + eps)) : NAN;  // NaN in every result
  return ldexpf(1.f, e);
}

// The input as fp16 times that power of two, rows padded.
__global__ void __launch_bounds__(256) input_kernel(const InputArgs p, int blocks, double eps, __half* out, int64_t pitch, int64_t out_batch, int planes, float* scale) {
  tck::chain_wait();
  __shared__ float tile[32][33];
  __shared__ double shared[8];
  const float factor = scale_of(p, blocks, eps, shared, scale);
  const void* x = matrix(p, blockIdx.y);
  out += blockIdx.y * planes * out_batch;
  __half* rest = out + out_batch;  // second term, where there are two
  if (!p.turn) {
    const int64_t per = (p.cols + 7) / 8, total = per * p.rows, stride = (int64_t)gridDim.x * 256;
#pragma unroll 2
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
      const int64_t r = i / per, at = (i - r * per) * 8;
      float f[8];
      if (p.vec) {
        load8(x, r * p.row_stride + at, p.dtype, f);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = at + k < p.cols ? load_as_float(x, r * p.row_stride + (at + k) * p.col_stride, p.dtype) : 0.f;
      }
      __half2 h[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = __floats2half2_rn(f[2 * k] * factor, f[2 * k + 1] * factor);
      *reinterpret_cast<uint4*>(out + r * pitch + at) = *reinterpret_cast<const uint4*>(h);
      if (planes == 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 got = __half22float2(h[k]);
          h[k] = __floats2half2_rn(f[2 * k] * factor - got.x, f[2 * k + 1] * factor - got.y);
        }
        *reinterpret_cast<uint4*>(rest + r * pitch + at) = *reinterpret_cast<const uint4*>(h);
      }
    }
    return;
  }
  const int tr = (p.rows + 31) / 32, tc = (p.cols + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t t = blockIdx.x; t < (int64_t)tr * tc; t += gridDim.x) {
    const int r0 = (int)(t / tc) * 32, c0 = (int)(t % tc) * 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int lr = lane, lc = warp + 8 * i;
      float v = 0.f;
      if (r0 + lr < p.rows && c0 + lc < p.cols) v = load_as_float(x, (r0 + lr) * p.row_stride + (c0 + lc) * p.col_stride, p.dtype);
      tile[lr][lc] = v * factor;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int lr = warp + 8 * i;
      if (r0 + lr < p.rows && c0 + lane < p.cols) {
        const __half h = __float2half_rn(tile[lr][lane]);
        out[(int64_t)(r0 + lr) * pitch + c0 + lane] = h;
        if (planes == 2) rest[(int64_t)(r0 + lr) * pitch + c0 + lane] = __float2half_rn(tile[lr][lane] - __half2float(h));
      }
    }
    __syncthreads();
  }
}

// fp16 results keep 11 bits: with one-term operands 1.3e-3 to 2e-3 of the result were off, of which rounding it is 2e-4; with two
// terms 2.1e-4, for 1.6 to 2 times the time (4 to 6 times at 65 to 128 rows of more than 1536 columns, which do not fit the cluster
// kernel so).  bf16 results, 1.7e-3 by their own rounding, are 1.8e-3 to 2.2e-3 off with one term.
bool two_terms(const TcOpShape& p) { return p.out_dtype == TC_F16; }

constexpr int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
struct Buffers {
  __half *x[2], *a, *b;
  float* scale;
  double* partial;
};
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  const int64_t m = std::min(p.rows, p.cols), n = std::max(p.rows, p.cols);
  TcCarver c{base};
  const int64_t planes = two_terms(p) ? 2 : 1;
  for (auto& x : b->x) x = c.take<__half>(p.batch * planes * m * up(n, 8));
  b->a = c.take<__half>(p.batch * planes * m * up(m, 8));
  b->b = c.take<__half>(p.batch * planes * m * up(m, 8));
  b->scale = c.take<float>(p.batch);
  b->partial = c.take<double>(p.batch * kNormBlocks);
  return c.used;
}

int iterate(const tc_op_plan& p, const Buffers& b, void* out, const int64_t* so, const void* x, const int64_t* sx, cudaStream_t stream) {
  const bool tall = p.rows > p.cols;
  const int64_t m = std::min(p.rows, p.cols), n = std::max(p.rows, p.cols), px = up(n, 8), pa = up(m, 8);
  InputArgs in{x, sx[0], tall ? sx[2] : sx[1], tall ? sx[1] : sx[2], (int)m, (int)n, p.dtype, 0, 0, b.partial};
  in.turn = in.col_stride != 1 && in.row_stride == 1;
  const int es = tc_elem_bytes(p.dtype);
  in.vec = (in.turn ? in.row_stride : in.col_stride) == 1 && (in.turn ? m : n) % 8 == 0 && (in.turn ? in.col_stride : in.row_stride) * es % 16 == 0 &&
           in.batch_stride * es % 16 == 0 && !(reinterpret_cast<uintptr_t>(x) & 15);
  const int planes = two_terms(p) ? 2 : 1;
  const int64_t pieces = in.turn ? (m + 7) / 8 * n : (n + 7) / 8 * m, tiles = ((m + 31) / 32) * ((n + 31) / 32);
  const int64_t share = std::max<int64_t>(1, 8 * p.sms / p.batch);  // blocks per matrix that fill the device
  const unsigned norm_blocks = (unsigned)std::min<int64_t>(std::min<int64_t>(kNormBlocks, share), (pieces + 255) / 256);
  TC_CUDA_OK(tck::launch_chained(true, norm_kernel, dim3(norm_blocks, (unsigned)p.batch), 256u, 0, stream, in));
  const unsigned input_blocks = (unsigned)std::min<int64_t>(share, in.turn ? tiles : (pieces + 255) / 256);
  TC_CUDA_OK(tck::launch_chained(true, input_kernel, dim3(input_blocks, (unsigned)p.batch), 256u, 0, stream, in, (int)norm_blocks, p.eps, b.x[0], px, m * px, planes, b.scale));
  // terms of the products: the first step's X has a second term only where the input has more than 11 bits
  const bool exact = p.dtype != TC_F32;
  auto base = [&](int64_t N, int64_t K, int terms) {
    WmArgs a{};
    a.terms = planes == 2 ? terms : 0;
    a.M = (uint32_t)m;
    a.N = (uint32_t)N;
    a.K = (uint32_t)K;
    a.batch = (uint32_t)p.batch;
    a.slices = 1;
    a.status = p.status;
    a.spin_limit = p.test_fault ? 1u << 14 : TC_SPIN_LIMIT;
    a.test_fault = p.test_fault;
    return a;
  };
  const WmOut square{nullptr, pa, 1, m * pa, 1, 0, planes};
  const WmOperand A{b.a, pa, m * pa}, B{b.b, pa, m * pa};
  const float guard = (float)(1 << kGuard);
  for (int i = 0; i < p.steps; ++i) {
    const bool first = i == 0, last = i + 1 == p.steps;
    const WmOperand X{b.x[i & 1], px, m * px};
    int tile, slices, st;
    WmArgs a = base(m, n, first && exact ? 1 : 3);
    a.out = square;
    a.out.ptr = b.a;
    const float shift = shift_of(i, p.steps), ca = p.coef[i][0] + shift * (p.coef[i][1] + shift * p.coef[i][2]), cb = p.coef[i][1] + 2 * shift * p.coef[i][2];
    a.affine = WmAffineArgs{first ? 1.f : 1.f / (guard * guard), 0.f, first ? b.scale : nullptr, 2, nullptr, 0, 0, shift};
    wm_choose(WM_SYMMETRIC, m, m, n, p.batch, 1, p.sms, &tile, &slices);
    st = wm_launch(WM_SYMMETRIC, tile, a, X, X, p.sms, stream);
    if (st != TC_OK) return st;

    a = base(m, m, 3);
    a.out = square;
    a.out.ptr = b.b;
    a.affine = WmAffineArgs{p.coef[i][2], cb, nullptr, 0, b.a, pa, m * pa, 0.f};
    wm_choose(WM_SYMMETRIC, m, m, m, p.batch, 1, p.sms, &tile, &slices);
    st = wm_launch(WM_SYMMETRIC, tile, a, A, A, p.sms, stream);
    if (st != TC_OK) return st;

    a = base(n, m, first && exact ? 2 : 3);
    const float held = (first ? 1.f : 1.f / guard) * (last ? 1.f : guard);  // from how X is held to how the result is
    a.affine = WmAffineArgs{held, ca * held, first ? b.scale : nullptr, 1, X.ptr, px, m * px, 0.f};
    if (last) {
      const int64_t rs = tall ? so[2] : so[1], cs = tall ? so[1] : so[2];
      a.out = WmOut{out, rs, cs, so[0], cs == 1 && wm_box_output(out, n, rs, p.batch > 1 ? so[0] : 0), p.out_dtype == TC_BF16, 1};
    } else {
      a.out = WmOut{b.x[(i + 1) & 1], px, 1, m * px, 1, 0, planes};
    }
    wm_choose(WM_UPDATE, m, n, m, p.batch, 1, p.sms, &tile, &slices);
    st = wm_launch(WM_UPDATE, tile, a, B, X, p.sms, stream);
    if (st != TC_OK) return st;
  }
  return TC_OK;
}

// Matrices of up to 128 rows and 4096 columns (1536 of more than 64 rows with two terms), in the orientation with fewer rows: one
// launch, a cluster each.
int rows_of_images(const TcOpShape& p) { return tck::orth_rows(std::min(p.rows, p.cols)); }
int most_columns(const TcOpShape& p) { return tck::orth_most_columns(rows_of_images(p), two_terms(p)); }
bool in_clusters(const TcOpShape& p) { return std::min(p.rows, p.cols) <= 128 && std::max(p.rows, p.cols) <= 8 * most_columns(p); }
typedef void (*ClusterKernel)(tck::OrthClusterArgs);
ClusterKernel cluster_kernel(int rows, bool terms) {
  if (rows == 64) return terms ? tck::orth_cluster_kernel<true, 64> : tck::orth_cluster_kernel<false, 64>;
  return terms ? tck::orth_cluster_kernel<true, 128> : tck::orth_cluster_kernel<false, 128>;
}

struct ClusterLaunch {
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg;
  int slab;
};
void cluster_launch(const tc_op_plan& p, int ctas, ClusterLaunch* l) {
  const int64_t n = std::max(p.rows, p.cols);
  *l = ClusterLaunch{};
  l->slab = (int)up((n + ctas - 1) / ctas, 64);
  l->at[0].id = cudaLaunchAttributeClusterDimension;
  l->at[0].val.clusterDim.x = (unsigned)ctas;
  l->at[0].val.clusterDim.y = l->at[0].val.clusterDim.z = 1;
  l->at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  l->at[1].val.programmaticStreamSerializationAllowed = 1;
  l->cfg.gridDim = dim3((unsigned)(p.batch * ctas));
  l->cfg.blockDim = dim3(tck::kOrthThreads);
  l->cfg.dynamicSmemBytes = (size_t)tck::orth_cluster_smem(l->slab, rows_of_images(p), two_terms(p));
  l->cfg.attrs = l->at;
  l->cfg.numAttrs = 2;
}
// CTAs per matrix: 256 columns each measured fastest (1504 columns of 21 rows: 25 us on 8 CTAs, 36 on 3; 399 of 17: 28.7 on 2,
// 29.2 on 1), up to the portable 8; fewer where the batch's clusters do not all fit the device at once (16 of 101 x 2584: 115 us
// on 8, 64 on 6).  On commit, for the device the plan runs on.
int choose_ctas(const tc_op_plan& p, int* ctas) {
  const int64_t n = std::max(p.rows, p.cols);
  const int least = (int)((n + most_columns(p) - 1) / most_columns(p)), most = std::max(least, n <= 256 ? 1 : n <= 512 ? 2 : n <= 1024 ? 4 : 8);
  double best = 0;
  for (int c = most; c >= least; --c) {
    ClusterLaunch l;
    cluster_launch(p, c, &l);
    int fit = 0;
    TC_CUDA_OK(cudaOccupancyMaxActiveClusters(&fit, cluster_kernel(rows_of_images(p), two_terms(p)), &l.cfg));
    if (fit < 1) continue;
    const int64_t rounds = (p.batch + fit - 1) / fit;
    const double cost = (double)rounds * (l.slab + 128);
    if (best == 0 || cost < best) {
      best = cost;
      *ctas = c;
    }
    if (c == most && rounds == 1) break;
  }
  return best > 0 ? TC_OK : TC_ERR_UNSUPPORTED;
}

int iterate_in_clusters(const tc_op_plan& p, void* out, const int64_t* so, const void* x, const int64_t* sx, cudaStream_t stream) {
  const bool tall = p.rows > p.cols;
  tck::OrthClusterArgs a{};
  a.x = x;
  a.x_batch = sx[0];
  a.x_row = tall ? sx[2] : sx[1];
  a.x_col = tall ? sx[1] : sx[2];
  a.out = out;
  a.out_batch = so[0];
  a.out_row = tall ? so[2] : so[1];
  a.out_col = tall ? so[1] : so[2];
  a.rows = (int)std::min(p.rows, p.cols);
  a.cols = (int)std::max(p.rows, p.cols);
  a.dtype = p.dtype;
  a.out_bf16 = p.out_dtype == TC_BF16;
  a.steps = p.steps;
  // eight columns of a row start on 16 bytes and end inside the row; a CTA's columns start at a multiple of 64
  auto pieces = [&](const void* ptr, int64_t batch, int64_t row, int64_t col, int es) {
    return col == 1 && a.cols % 8 == 0 && row * es % 16 == 0 && (p.batch == 1 || batch * es % 16 == 0) && !(reinterpret_cast<uintptr_t>(ptr) & 15);
  };
  a.x_vec = pieces(x, a.x_batch, a.x_row, a.x_col, tc_elem_bytes(p.dtype));
  a.out_vec = pieces(out, a.out_batch, a.out_row, a.out_col, 2);
  ClusterLaunch l;
  cluster_launch(p, p.ctas, &l);
  a.slab = l.slab;
  a.tmem_cols = 128;
  while (a.tmem_cols < l.slab) a.tmem_cols *= 2;
  for (int i = 0; i < p.steps; ++i) {
    const float shift = shift_of(i, p.steps), *c = p.coef[i];
    a.coef[i] = make_float4(c[0] + shift * (c[1] + shift * c[2]), c[1] + 2 * shift * c[2], c[2], shift);
  }
  a.eps = p.eps;
  a.status = p.status;
  a.spin_limit = p.test_fault ? 1u << 14 : TC_SPIN_LIMIT;
  a.test_fault = p.test_fault;
  l.cfg.stream = stream;
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, cluster_kernel(rows_of_images(p), two_terms(p)), a);
  if (e != cudaSuccess) (void)cudaGetLastError();
  TC_CUDA_OK(e);
  return TC_OK;
}

}  // namespace

size_t tc_orth_workspace(const TcOpShape& p) {
  if (in_clusters(p)) return 0;
  Buffers b;
  return carve(p, nullptr, &b);
}

int tc_orth_plan(tc_op_plan* p) { return in_clusters(*p) ? choose_ctas(*p, &p->ctas) : TC_OK; }

int tc_orth_prepare() {
  for (int rows : {64, 128})
    for (bool terms : {false, true})
      TC_CUDA_OK(cudaFuncSetAttribute(cluster_kernel(rows, terms), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      tck::orth_cluster_smem(tck::orth_most_columns(rows, terms), rows, terms)));
  const int st = wm_prepare(WM_SYMMETRIC);
  return st != TC_OK ? st : wm_prepare(WM_UPDATE);
}

std::string tc_orth_json(const TcOpShape& p) {
  const double m = (double)std::min(p.rows, p.cols), n = (double)std::max(p.rows, p.cols);
  return "{\"operator\":\"orthogonal\",\"batch\":" + std::to_string(p.batch) + ",\"rows\":" + std::to_string(p.rows) + ",\"cols\":" + std::to_string(p.cols) +
         ",\"steps\":" + std::to_string(p.steps) + ",\"flops\":" + std::to_string(p.batch * p.steps * (3 * m * m * n + m * m * m)) +
         ",\"workspace_bytes\":" + std::to_string(tc_orth_workspace(p)) + "}";
}

extern "C" int tc_orthogonal_execute(tc_op_plan* p, void* out, const int64_t* out_strides, const void* x, const int64_t* x_strides, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (!p || p->kind != TC_OP_ORTHOGONAL || !out || !x || !out_strides || !x_strides) return TC_ERR_INVALID_ARG;
  const uintptr_t es = (uintptr_t)tc_elem_bytes(p->dtype);
  if ((reinterpret_cast<uintptr_t>(x) & (es - 1)) || (reinterpret_cast<uintptr_t>(out) & 1)) return TC_ERR_ALIGNMENT;
  const int64_t ext[3] = {p->batch, p->rows, p->cols};
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 3; ++i)
    if (x_strides[i] < 0 || out_strides[i] < 0) return TC_ERR_EXTENT;
  // no two results at one place: each index steps over all that the faster ones span
  std::sort(order, order + 3, [&](int i, int j) { return out_strides[i] < out_strides[j]; });
  int64_t span = 1;
  for (int i : order) {
    if (ext[i] == 1) continue;
    if (out_strides[i] < span) return TC_ERR_EXTENT;
    span = out_strides[i] * (ext[i] - 1) + span;
  }
  TcScratch scratch;
  const int st = scratch.open(p, TC_OP_ORTHOGONAL, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  if (st != TC_OK) return st;
  if (in_clusters(*p)) return scratch.close(iterate_in_clusters(*p, out, out_strides, x, x_strides, static_cast<cudaStream_t>(stream)));
  Buffers b;
  carve(*p, scratch.base, &b);
  return scratch.close(iterate(*p, b, out, out_strides, x, x_strides, static_cast<cudaStream_t>(stream)));
}

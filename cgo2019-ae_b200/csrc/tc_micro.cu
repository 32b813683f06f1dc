// Microscaled 4-bit numbers: quantisation along either index of a matrix, and back (tc_microscale_*).
//
//   e = min { e >= -127 : max |x| <= 6 * 2^e }   over 32 neighbours of a row,     q = e2m1(x / 2^e), ties to even
//
// Scaling by a power of two and the comparison that finds it are exact, so every code is the nearest one to the number itself.
// Codes lie along rows, 16 bytes a block; scales in pieces of 128 rows by 4 blocks (512 bytes), row 32 j + i of a piece at
// byte 16 i + 4 j: the order in which tensor memory takes them.
//
// Bound by bytes and by instructions: 154 for a thread's eight elements were 23 us on 8192 x 4096 bf16, and a fifth of them where the thread is;
// with that worked out once for four rows 17.7 us (4.8 TB/s), down columns 19.4, back 15.9.
#include "tc_elem.cuh"
#include "tc_inst.cuh"
#include "tc_op.h"

namespace {
using namespace tck;

constexpr int kThreads = 256;

__device__ __forceinline__ size_t scale_at(uint64_t row, uint32_t piece, uint32_t pieces) {
  return ((row >> 7) * pieces + piece) * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4;
}

struct RowsArgs {
  unsigned char *codes, *scales;
  const void* x;
  int64_t ld_codes, ld_x, rows;
  uint32_t pieces, cols, blocks;
};

// 16 lanes take 128 columns of R rows, eight each, four a block: where a thread is, is worked out once, and its loads are under way together.
template <class T, bool Vec, int R>
__global__ void __launch_bounds__(kThreads) quantise_kernel(const __grid_constant__ RowsArgs a) {
  __shared__ __align__(16) T staged[Vec ? 1 : kThreads * 8];
  const int lane = threadIdx.x & 15;
  T* stage = staged + (Vec ? 0 : (threadIdx.x >> 4) * 128);
  const uint64_t unit = (uint64_t)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4), group = unit < UINT32_MAX ? (uint32_t)unit / a.pieces : unit / a.pieces;
  const uint32_t piece = (uint32_t)(unit - group * a.pieces);
  const int64_t row0 = (int64_t)group * R;
  const int rows = (int)max((int64_t)0, min((int64_t)R, a.rows - row0)), valid = (int)a.cols - (int)(piece * 128);
  const T* x = static_cast<const T*>(a.x) + row0 * a.ld_x + piece * 128;
  unsigned char* codes = a.codes + row0 * a.ld_codes + piece * 64 + lane * 4;
  unsigned char* scales = a.scales + scale_at((uint64_t)row0, piece, a.pieces);  // R divides 32: the rows' scales are 16 bytes apart
  const bool there = piece * 4 + (lane >> 2) < a.blocks;
  chain_wait();
  Raw<T> raw[R];
#pragma unroll
  for (int i = 0; i < R; ++i) raw[i] = unit_load<T, Vec>(x + i * a.ld_x, lane, i < rows ? valid : 0, stage);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float f[8];
    unpack8<T>(raw[i], f);
    const uint32_t byte = micro4_scale(block_max(magnitude_of<T>(raw[i])));
    const float inverse = micro_inverse(byte);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= inverse;
    const uint32_t code = byte == 255u ? 0u : to_e2m1(f);
    uint32_t four = byte << (lane >> 2) * 8;  // the scales of the row's four blocks
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    four |= __shfl_xor_sync(0xffffffffu, four, 8);
    if (i < rows) {
      if (there) *reinterpret_cast<uint32_t*>(codes + i * a.ld_codes) = code;
      if (lane == 0) *reinterpret_cast<uint32_t*>(scales + i * 16) = four;
    }
  }
}

// x is [cols][rows]: blocks run down its columns.  128 of the blocks' index by 64 words (128 rows of 16-bit elements, 64 of 32)
// through shared memory; a thread takes 32 words of a column, lanes so that four write the 64 bytes of a row.  Words are turned by
// eight per block, which leaves neither access a bank conflict.
struct ColumnsArgs {
  unsigned char *codes, *scales;
  const void* x;
  int64_t ld_codes, ld_x, rows;
  uint32_t pieces, cols, blocks, row_tiles;
};
template <class T, bool Vec>
__global__ void __launch_bounds__(kThreads) quantise_columns_kernel(const __grid_constant__ ColumnsArgs a) {
  constexpr int kPer = 4 / sizeof(T), kRows = 64 * kPer;
  __shared__ __align__(16) uint32_t words[128 * 64];
  const uint32_t row_tile = blockIdx.x % a.row_tiles, piece = blockIdx.x / a.row_tiles;
  const int64_t row0 = (int64_t)row_tile * kRows;
  const uint32_t k0 = piece * 128, tid = threadIdx.x;
  const int rows = (int)min((int64_t)kRows, a.rows - row0);
  const T* x = static_cast<const T*>(a.x) + (int64_t)k0 * a.ld_x + row0;
  chain_wait();
  if constexpr (Vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t at = tid + i * kThreads, k = at >> 4, w = (at & 15) * 4;
      const bool there = k0 + k < a.cols && (int)(w * kPer) < rows;
      const uint4 v = there ? *reinterpret_cast<const uint4*>(x + (int64_t)k * a.ld_x + w * kPer) : make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(words + k * 64 + ((w + 8 * (k >> 5)) & 63)) = v;
    }
  } else {
    T* elems = reinterpret_cast<T*>(words);
    for (uint32_t at = tid; at < 128 * kRows; at += kThreads) {
      const uint32_t k = at / kRows, r = at % kRows;
      const T v = k0 + k < a.cols && (int)r < rows ? x[(int64_t)k * a.ld_x + r] : Elem<T>::put(0.f);
      elems[(k * 64 + ((r / kPer + 8 * (k >> 5)) & 63)) * kPer + r % kPer] = v;
    }
  }
  __syncthreads();
  const uint32_t kb = tid & 3, column = tid >> 2;
  uint32_t w[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) w[j] = words[(kb * 32 + j) * 64 + ((column + 8 * kb) & 63)];
#pragma unroll
  for (int h = 0; h < kPer; ++h) {
    auto value = [&](int j) {
      if constexpr (kPer == 1) return __uint_as_float(w[j]);
      else return Elem<T>::get(reinterpret_cast<const T*>(&w[j])[h]);
    };
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(value(j)) & 0x7FFFFFFFu);
    const uint32_t byte = micro4_scale(top);
    uint32_t code[4] = {0, 0, 0, 0};
    if (byte != 255u) {
      const float inverse = micro_inverse(byte);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = value(8 * q + j) * inverse;
        code[q] = to_e2m1(f);
      }
    }
    uint32_t four = byte << kb * 8;
    four |= __shfl_xor_sync(0xffffffffu, four, 1);
    four |= __shfl_xor_sync(0xffffffffu, four, 2);
    const int r = (int)column * kPer + h;
    if (r < rows) {
      const int64_t row = row0 + r;
      if (piece * 4 + kb < a.blocks)
        *reinterpret_cast<uint4*>(a.codes + row * a.ld_codes + (piece * 4 + kb) * 16) = make_uint4(code[0], code[1], code[2], code[3]);
      if (kb == 0) *reinterpret_cast<uint32_t*>(a.scales + scale_at((uint64_t)row, piece, a.pieces)) = four;
    }
  }
}

struct RestoreArgs {
  const unsigned char *codes, *scales;
  void* x;
  int64_t ld_codes, ld_x, rows;
  uint32_t pieces, cols;
};
template <class T, bool Vec, int R>
__global__ void __launch_bounds__(kThreads) restore_kernel(const __grid_constant__ RestoreArgs a) {
  __shared__ __align__(16) T staged[Vec ? 1 : kThreads * 8];
  const int lane = threadIdx.x & 15;
  T* stage = staged + (Vec ? 0 : (threadIdx.x >> 4) * 128);
  const uint64_t unit = (uint64_t)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4), group = unit < UINT32_MAX ? (uint32_t)unit / a.pieces : unit / a.pieces;
  const uint32_t piece = (uint32_t)(unit - group * a.pieces);
  const int64_t row0 = (int64_t)group * R;
  const int rows = (int)max((int64_t)0, min((int64_t)R, a.rows - row0)), valid = (int)a.cols - (int)(piece * 128);
  const unsigned char* codes = a.codes + row0 * a.ld_codes + piece * 64 + lane * 4;
  const unsigned char* scales = a.scales + scale_at((uint64_t)row0, piece, a.pieces) + (lane >> 2);
  T* x = static_cast<T*>(a.x) + row0 * a.ld_x + piece * 128;
  chain_wait();
  uint32_t code[R], scale[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool there = i < rows && lane * 8 < valid;
    code[i] = there ? *reinterpret_cast<const uint32_t*>(codes + i * a.ld_codes) : 0u;
    scale[i] = there ? scales[i * 16] : 0u;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float f[8];
    from_e2m1(code[i], f);
    rescale8<T>(f, scale[i]);
    unit_store<T, Vec>(x + i * a.ld_x, pack8<T>(f), lane, i < rows ? valid : 0, stage);
  }
}

// Four rows a thread where that leaves a few blocks for each multiprocessor, so that small matrices are spread over all of them.
constexpr int64_t kManyUnits = 16;
int64_t blocks_for(int64_t rows, int64_t pieces, bool many) { return ((many ? (rows + 3) / 4 : rows) * pieces + kThreads / 16 - 1) / (kThreads / 16); }

template <class T>
int quantise(const tc_op_plan& p, unsigned char* codes, int64_t ld_codes, unsigned char* scales, const void* x, int64_t ld_x, bool transposed, int64_t rows,
             cudaStream_t stream) {
  const uint32_t blocks = (uint32_t)((p.dim + 31) / 32), pieces = (blocks + 3) / 4;
  if (transposed) {
    const int64_t tiles = (rows + 64 * (4 / (int)sizeof(T)) - 1) / (64 * (4 / (int)sizeof(T)));
    if (tiles * pieces > INT32_MAX) return TC_ERR_UNSUPPORTED;
    const ColumnsArgs a{codes, scales, x, ld_codes, ld_x, rows, pieces, (uint32_t)p.dim, blocks, (uint32_t)tiles};
    const bool vec = tc_vec8(x, ld_x, rows, sizeof(T));
    TC_CUDA_OK(launch_chained(true, vec ? quantise_columns_kernel<T, true> : quantise_columns_kernel<T, false>, dim3((unsigned)(tiles * pieces)), (unsigned)kThreads, 0, stream, a));
    return TC_OK;
  }
  const RowsArgs a{codes, scales, x, ld_codes, ld_x, rows, pieces, (uint32_t)p.dim, blocks};
  const bool vec = tc_vec8(x, ld_x, p.dim, sizeof(T)), many = rows * pieces >= 16 * kManyUnits * (int64_t)p.sms;
  const int64_t grid = blocks_for(rows, pieces, many);
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  auto kernel = many ? (vec ? quantise_kernel<T, true, 4> : quantise_kernel<T, false, 4>) : (vec ? quantise_kernel<T, true, 1> : quantise_kernel<T, false, 1>);
  TC_CUDA_OK(launch_chained(true, kernel, dim3((unsigned)grid), (unsigned)kThreads, 0, stream, a));
  return TC_OK;
}

template <class T>
int restore(const tc_op_plan& p, void* x, int64_t ld_x, const unsigned char* codes, int64_t ld_codes, const unsigned char* scales, int64_t rows, cudaStream_t stream) {
  const uint32_t pieces = (uint32_t)((p.dim + 127) / 128);
  const RestoreArgs a{codes, scales, x, ld_codes, ld_x, rows, pieces, (uint32_t)p.dim};
  const bool vec = tc_vec8(x, ld_x, p.dim, sizeof(T)), many = rows * pieces >= 16 * kManyUnits * (int64_t)p.sms;
  const int64_t grid = blocks_for(rows, pieces, many);
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  auto kernel = many ? (vec ? restore_kernel<T, true, 4> : restore_kernel<T, false, 4>) : (vec ? restore_kernel<T, true, 1> : restore_kernel<T, false, 1>);
  TC_CUDA_OK(launch_chained(true, kernel, dim3((unsigned)grid), (unsigned)kThreads, 0, stream, a));
  return TC_OK;
}

// x: [rows][cols], or [cols][rows] where transposed.  back: x is the result.
int check(const tc_op_plan* p, const void* codes, int64_t ld_codes, const void* scales, const void* x, int64_t ld_x, int transposed, int64_t rows, bool back) {
  if (!p || p->kind != TC_OP_MICROSCALE || (rows && (!codes || !scales || !x))) return TC_ERR_INVALID_ARG;
  if (rows < 0 || rows > p->tokens || ld_codes < (p->dim + 31) / 32 * 16 || ld_x < 0) return TC_ERR_EXTENT;
  const int es = tc_elem_bytes(p->dtype);
  if (tc_odd_address(codes, 16) || tc_odd_address(scales, 16) || ld_codes % 16 || tc_odd_address(x, es)) return TC_ERR_ALIGNMENT;
  if (back && ld_x < p->dim) return TC_ERR_EXTENT;
  if (!rows) return TC_OK;
  const int64_t x_cols = transposed ? rows : p->dim, x_rows = transposed ? p->dim : rows;
  const TcSpan spans[] = {{codes, ld_codes, (p->dim + 31) / 32 * 16, rows, !back}, {scales, 0, tc_micro_scale_bytes(rows, p->dim), 1, !back}, {x, ld_x * es, x_cols * es, x_rows, back}};
  return tc_results_overlap(spans) ? TC_ERR_INVALID_ARG : TC_OK;
}

}  // namespace

std::string tc_micro_json(const TcOpShape& p) {
  const int64_t blocks = (p.dim + 31) / 32;
  return "{\"operator\":\"microscale\",\"dtype\":\"" + tc_type_name(p.dtype) + "\",\"rows\":" + std::to_string(p.tokens) + ",\"cols\":" + std::to_string(p.dim) +
         ",\"bytes_per_row\":" + std::to_string(16 * blocks) + ",\"scale_pieces\":[" + std::to_string((p.tokens + 127) / 128) + "," + std::to_string((blocks + 3) / 4) + "]}";
}

extern "C" int tc_microscale_execute(tc_op_plan* p, void* codes, int64_t ld_codes, void* scales, const void* x, int64_t ld_x, int transposed, int64_t rows, void* stream) {
  int st = check(p, codes, ld_codes, scales, x, ld_x, transposed, rows, false);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (st == TC_OK) st = tc_op_ready(p, s);
  if (st != TC_OK || rows == 0) return st;
  unsigned char *c = static_cast<unsigned char*>(codes), *e = static_cast<unsigned char*>(scales);
  switch (p->dtype) {
    case TC_F32: return quantise<float>(*p, c, ld_codes, e, x, ld_x, transposed != 0, rows, s);
    case TC_BF16: return quantise<__nv_bfloat16>(*p, c, ld_codes, e, x, ld_x, transposed != 0, rows, s);
    default: return quantise<__half>(*p, c, ld_codes, e, x, ld_x, transposed != 0, rows, s);
  }
}

extern "C" int tc_microscale_restore(tc_op_plan* p, void* x, int64_t ld_x, const void* codes, int64_t ld_codes, const void* scales, int64_t rows, void* stream) {
  int st = check(p, codes, ld_codes, scales, x, ld_x, 0, rows, true);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (st == TC_OK) st = tc_op_ready(p, s);
  if (st != TC_OK || rows == 0) return st;
  const unsigned char *c = static_cast<const unsigned char*>(codes), *e = static_cast<const unsigned char*>(scales);
  switch (p->dtype) {
    case TC_F32: return restore<float>(*p, x, ld_x, c, ld_codes, e, rows, s);
    case TC_BF16: return restore<__nv_bfloat16>(*p, x, ld_x, c, ld_codes, e, rows, s);
    default: return restore<__half>(*p, x, ld_x, c, ld_codes, e, rows, s);
  }
}

// Rows of a table by token, scaled, and their gradient by sorted tokens (tc_embedding_execute*).
//
//   out_t = s E[id_t]            dE[v] = s sum over {t : id_t = v} of G_t
//
// Tokens outside [0, vocab) stand for none: zeros out, no share in the gradient.
//
// The gradient sums each row's tokens in the order they come in, whatever runs when: tokens are sorted (stably) by row, the sorted
// list is cut into chunks of equal length, a block sums a chunk's runs of equal rows in fp32, and runs that pass a chunk's
// end leave partial sums that one block per run adds up in order.  A token that appears thousands of times is spread over as
// many blocks as it has chunks.  The rows without a token, most of a large table, are zeroed by blocks of their own beside
// those that sort (a share of the table, whatever is in it) and those that sum (the rest, but for the rows of tokens).
//
// Bound by bytes.  One B200: 16384 tokens' rows of 2048 bf16 out of 131072 21.7 us (6.2 TB/s), their gradient 132 us (537 MB written, 67 read:
// 4.6 TB/s, the four sorting kernels' latencies among it); 8 tokens 7 us, the host's call; the gradient of 3001 fp32 rows of 301 18 us,
// three launches.
#include <algorithm>

#include "tc_inst.cuh"
#include "tc_op.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace {

constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 1024, kSortWarps = 32;
constexpr int kOneBlockItems = 4;                               // tokens per thread of the one-block sort
constexpr int64_t kOneBlock = kSortThreads * kOneBlockItems;    // most tokens it sorts
// What of a table each sorting kernel zeroes while it sorts (four times that where there is one).  bf16 gradients, us with 6, 12 and 24e6: 16384
// tokens, 131072 rows of 2048 132, 132, 137; 65536 of 1024 58, 59, 64; 12000, 262144 of 2048 200, 201, 204; 3000, 131072 of 1024 61, 58, 53;
// 1000, 28424 of 960 25.3, 23.9, 23.8; 40000, 131072 of 512 88, 89, 89.
constexpr double kEarlyBytes = 12e6;
constexpr int64_t kShortPasses = 65536;                         // tokens up to which a block of the sort by passes takes one per thread, else four

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// ---- 16 bytes of a type ----
template <class T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  __device__ static void get(uint4 v, float* f) { f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w); }
  __device__ static uint4 put(const float* f) { return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])); }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void get(uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
  }
  __device__ static uint4 put(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&v); }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Piece<__half> {
  static constexpr int N = 8;
  __device__ static void get(uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v2 = __half22float2(*reinterpret_cast<const __half2*>(&w[i])); f[2 * i] = v2.x; f[2 * i + 1] = v2.y; }
  }
  __device__ static uint4 put(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&v); }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N neighbouring values from `p`: one access where rows are 16-byte aligned (Vec), else element by element within `left`.
template <class T, bool Vec>
__device__ __forceinline__ void get_values(const T* p, int left, float* f) {
  if constexpr (Vec) {
    Piece<T>::get(*reinterpret_cast<const uint4*>(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) f[i] = i < left ? to_float(p[i]) : 0.f;
  }
}
template <class T, bool Vec>
__device__ __forceinline__ void put_values(T* p, int left, const float* f) {
  if constexpr (Vec) {
    *reinterpret_cast<uint4*>(p) = Piece<T>::put(f);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (i < left) p[i] = from_float<T>(f[i]);
  }
}

// ---- lookup ----
// A thread takes 16 bytes (or one element) of a row at a time, four of them in flight.  Elements cost several times as much, a division and
// two accesses each: 16384 rows of 2047 bf16 108 us, of 2048 24.5; of 1023 fp32 62, of 1024 23.6.
template <class T, bool Vec>
__global__ void __launch_bounds__(256) lookup_kernel(T* out, int64_t ld_out, const T* table, int64_t ld_table, const void* ids, int wide, int64_t tokens, int64_t vocab,
                                                     int dim, float scale) {
  tck::chain_wait();
  constexpr int N = Vec ? Piece<T>::N : 1, U = 4;
  const uint32_t per_row = (uint32_t)((dim + N - 1) / N);
  const int64_t total = tokens * per_row, stride = (int64_t)gridDim.x * 256;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < total; i0 += U * stride) {
    int64_t row[U], id[U];
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * stride;
      row[u] = i < total ? i / per_row : -1;
      at[u] = i < total ? (uint32_t)(i - row[u] * per_row) * N : 0u;
      id[u] = row[u] >= 0 ? index_at(ids, row[u], wide) : -1;
    }
    if constexpr (Vec) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = id[u] >= 0 && id[u] < vocab ? *reinterpret_cast<const uint4*>(table + id[u] * ld_table + at[u]) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[u] < 0) continue;
        if (scale != 1.f) {
          float f[N];
          Piece<T>::get(v[u], f);
#pragma unroll
          for (int k = 0; k < N; ++k) f[k] *= scale;
          v[u] = id[u] >= 0 && id[u] < vocab ? Piece<T>::put(f) : make_uint4(0, 0, 0, 0);
        }
        *reinterpret_cast<uint4*>(out + row[u] * ld_out + at[u]) = v[u];
      }
    } else {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = id[u] >= 0 && id[u] < vocab ? to_float(table[id[u] * ld_table + at[u]]) * scale : 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row[u] >= 0) out[row[u] * ld_out + at[u]] = from_float<T>(v[u]);
    }
  }
}

// ---- gradient: zeros ----
struct FillArgs {
  char* table;                            // null: nothing to zero
  int64_t rows, pitch_bytes, row_bytes;   // rows of the table, the distance between them, what is zeroed of each
  int64_t early;                          // rows that the sorting kernels zero
};
// `bytes` from p on (both even), by `threads` threads of which this is number `me`: 16 bytes each, next to one another, between the
// first and the last 16-byte boundary (a warp's own stretch each was slower: 143 against 133 us for a gradient of 537 MB).
__device__ __forceinline__ void zero_bytes(char* p, int64_t bytes, int64_t me, int64_t threads) {
  const int64_t head = min(bytes, (int64_t)(-reinterpret_cast<uintptr_t>(p) & 15)), body = (bytes - head) / 16, tail = bytes - head - 16 * body;
  if (2 * me < head) *reinterpret_cast<uint16_t*>(p + 2 * me) = 0;
  uint4* q = reinterpret_cast<uint4*>(p + head);
#pragma unroll 4
  for (int64_t i = me; i < body; i += threads) q[i] = make_uint4(0, 0, 0, 0);
  if (2 * me < tail) *reinterpret_cast<uint16_t*>(p + head + 16 * body + 2 * me) = 0;
}
// Part `part` of `parts` of the early rows, by block `block` of `blocks`.
__device__ void zero_early(const FillArgs& f, int block, int blocks, int part, int parts) {
  const int64_t from = f.early * part / parts, to = f.early * (part + 1) / parts;
  if (f.pitch_bytes == f.row_bytes) {
    zero_bytes(f.table + from * f.row_bytes, (to - from) * f.row_bytes, (int64_t)block * blockDim.x + threadIdx.x, (int64_t)blocks * blockDim.x);
  } else {
    const int64_t warps = (int64_t)blocks * (blockDim.x >> 5);
    for (int64_t r = from + (int64_t)block * (blockDim.x >> 5) + (threadIdx.x >> 5); r < to; r += warps)
      zero_bytes(f.table + r * f.pitch_bytes, f.row_bytes, threadIdx.x & 31, 32);
  }
}

// ---- gradient: tokens sorted by row ----
struct SortArgs {
  const void* ids;
  int wide;
  int64_t tokens, vocab;
  int passes;
  uint32_t *key[2], *pos[2];  // by passes: from key[0], pos[0] to key[1], pos[1] and back; the last pass writes sorted_*
  uint32_t *sorted_key, *sorted_pos;
  uint32_t* hist;             // [blocks][kDigits]
  uint32_t* touched;          // a bit per row of the table: has a token
  FillArgs fill;
};
__device__ __forceinline__ uint32_t key_of(const SortArgs& p, int64_t i) {  // tokens that stand for none come last
  const int64_t id = index_at(p.ids, i, p.wide);
  return id >= 0 && id < p.vocab ? (uint32_t)id : (uint32_t)p.vocab;
}

__device__ __forceinline__ void clear_touched(const SortArgs& p, int64_t me, int64_t threads) {
  for (int64_t i = me; i < (p.vocab + 31) / 32; i += threads) p.touched[i] = 0;
}
__device__ __forceinline__ void touch(const SortArgs& p, uint32_t key) {
  if (key < p.vocab) atomicOr(p.touched + key / 32, 1u << (key % 32));
}

// Stable places of a block's items by a digit.  Warp w holds the items w * 32 * Items .. in order (item j of lane l: j * 32 + l).
// base[d]: first place of the block's items of digit d.  count: [kSortWarps][kDigits] in shared memory.
template <int Items>
__device__ void places(const uint32_t (&digit)[Items], const bool (&live)[Items], uint16_t* count, const uint32_t* base, uint32_t (&place)[Items]) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kSortWarps * kDigits / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(count)[i] = 0;
  __syncthreads();
  uint16_t* mine = count + warp * kDigits;
#pragma unroll
  for (int j = 0; j < Items; ++j) {
    const uint32_t d = live[j] ? digit[j] : (uint32_t)kDigits;
    const uint32_t same = __match_any_sync(0xffffffffu, d);
    const uint32_t before = __popc(same & ((1u << lane) - 1u));
    if (live[j]) place[j] = mine[d] + before;
    __syncwarp();
    if (live[j] && before == 0) mine[d] = (uint16_t)(mine[d] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  if (tid < kDigits) {
    uint32_t run = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t n = count[w * kDigits + tid];
      count[w * kDigits + tid] = (uint16_t)run;
      run += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < Items; ++j)
    if (live[j]) place[j] += mine[digit[j]] + base[digit[j]];
}

// Exclusive prefix sums of kDigits numbers by the first kDigits threads; all threads call.
__device__ __forceinline__ uint32_t digit_prefix(uint32_t v, uint32_t* warps) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t sum = v;
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (tid < kDigits && lane == 31) warps[tid >> 5] = sum;
  __syncthreads();
  uint32_t before = 0;
  if (tid < kDigits)
    for (int w = 0; w < tid >> 5; ++w) before += warps[w];
  __syncthreads();
  return before + sum - v;
}

// Up to kOneBlock tokens, Items per thread at most: block 0 sorts them in shared memory while the others zero the early rows.
constexpr size_t one_block_smem(int items) { return (size_t)kSortThreads * items * 8 + kSortWarps * kDigits * 2 + kDigits * 4 + 64; }
template <int Items>
__global__ void __launch_bounds__(kSortThreads, 1) sort_one_kernel(const SortArgs p) {
  tck::chain_wait();
  if (blockIdx.x > 0) {
    zero_early(p.fill, blockIdx.x - 1, gridDim.x - 1, 0, 1);
    return;
  }
  extern __shared__ __align__(16) unsigned char smem[];
  uint32_t* key = reinterpret_cast<uint32_t*>(smem);
  uint32_t* pos = key + kSortThreads * Items;
  uint16_t* count = reinterpret_cast<uint16_t*>(pos + kSortThreads * Items);
  uint32_t* base = reinterpret_cast<uint32_t*>(count + kSortWarps * kDigits);
  uint32_t* warps = base + kDigits;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = (int)p.tokens;
  clear_touched(p, tid, kSortThreads);
  // items per thread that this many tokens need; each warp's items follow one another
  const int items = (n + kSortThreads - 1) / kSortThreads;
  for (int i = tid; i < n; i += kSortThreads) { key[i] = key_of(p, i); pos[i] = (uint32_t)i; }
  __syncthreads();
  for (int pass = 0; pass < p.passes; ++pass) {
    uint32_t k[Items], o[Items], digit[Items], place[Items];
    bool live[Items];
    if (tid < kDigits) base[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < Items; ++j) {
      const int i = warp * 32 * items + j * 32 + lane;
      live[j] = j < items && i < n;
      k[j] = live[j] ? key[i] : 0u;
      o[j] = live[j] ? pos[i] : 0u;
      digit[j] = (k[j] >> (pass * kDigitBits)) & (kDigits - 1);
      if (live[j]) atomicAdd(base + digit[j], 1u);  // counts: any order
    }
    __syncthreads();
    const uint32_t first = digit_prefix(tid < kDigits ? base[tid] : 0u, warps);
    if (tid < kDigits) base[tid] = first;
    __syncthreads();
    places<Items>(digit, live, count, base, place);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < Items; ++j)
      if (live[j]) { key[place[j]] = k[j]; pos[place[j]] = o[j]; }
    __syncthreads();
  }
  for (int i = tid; i < n; i += kSortThreads) {
    p.sorted_key[i] = key[i];
    p.sorted_pos[i] = pos[i];
    if (i == 0 || key[i] != key[i - 1]) touch(p, key[i]);
  }
}

// More tokens, by passes of one digit: counts of each block's tokens, then stable places.  Both kernels zero their part of the early rows.
template <int Items>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs p, int pass, int blocks, int part, int parts) {
  tck::chain_wait();
  if ((int)blockIdx.x >= blocks) {
    zero_early(p.fill, blockIdx.x - blocks, gridDim.x - blocks, part, parts);
    return;
  }
  __shared__ uint32_t count[kDigits];
  if (pass == 0) clear_touched(p, (int64_t)blockIdx.x * kSortThreads + threadIdx.x, (int64_t)blocks * kSortThreads);
  if (threadIdx.x < kDigits) count[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t* from = pass ? p.key[(pass - 1) & 1] : nullptr;
#pragma unroll
  for (int j = 0; j < Items; ++j) {
    const int64_t i = (int64_t)blockIdx.x * (kSortThreads * Items) + j * kSortThreads + threadIdx.x;
    if (i < p.tokens) atomicAdd(count + (((from ? from[i] : key_of(p, i)) >> (pass * kDigitBits)) & (kDigits - 1)), 1u);
  }
  __syncthreads();
  if (threadIdx.x < kDigits) p.hist[(int64_t)blockIdx.x * kDigits + threadIdx.x] = count[threadIdx.x];
}
template <int Items>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const SortArgs p, int pass, int blocks, int part, int parts) {
  tck::chain_wait();
  if ((int)blockIdx.x >= blocks) {
    zero_early(p.fill, blockIdx.x - blocks, gridDim.x - blocks, part, parts);
    return;
  }
  __shared__ uint16_t count[kSortWarps * kDigits];
  __shared__ uint32_t base[kDigits], warps[kDigits / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t all = 0, before = 0;
  if (tid < kDigits)
#pragma unroll 16
    for (int b = 0; b < blocks; ++b) {
      const uint32_t c = p.hist[(int64_t)b * kDigits + tid];
      if (b < (int)blockIdx.x) before += c;
      all += c;
    }
  const uint32_t first = digit_prefix(all, warps);
  if (tid < kDigits) base[tid] = first + before;
  __syncthreads();
  const bool last = pass + 1 == p.passes;
  const uint32_t *kin = pass ? p.key[(pass - 1) & 1] : nullptr, *pin = pass ? p.pos[(pass - 1) & 1] : nullptr;
  uint32_t *kout = last ? p.sorted_key : p.key[pass & 1], *pout = last ? p.sorted_pos : p.pos[pass & 1];
  uint32_t k[Items], o[Items], digit[Items], place[Items];
  bool live[Items];
#pragma unroll
  for (int j = 0; j < Items; ++j) {
    const int64_t i = (int64_t)blockIdx.x * (kSortThreads * Items) + warp * 32 * Items + j * 32 + lane;
    live[j] = i < p.tokens;
    k[j] = live[j] ? (kin ? kin[i] : key_of(p, i)) : 0u;
    o[j] = live[j] ? (pin ? pin[i] : (uint32_t)i) : 0u;
    digit[j] = (k[j] >> (pass * kDigitBits)) & (kDigits - 1);
  }
  places<Items>(digit, live, count, base, place);
#pragma unroll
  for (int j = 0; j < Items; ++j) {
    if (live[j]) { kout[place[j]] = k[j]; pout[place[j]] = o[j]; }
    if (last) {  // one of a warp's equal rows is enough
      const unsigned same = __match_any_sync(0xffffffffu, live[j] ? k[j] : 0xffffffffu);
      if (live[j] && (same & ((1u << lane) - 1u)) == 0) touch(p, k[j]);
    }
  }
}

// ---- gradient: sums ----
struct SumArgs {
  const uint32_t *key, *pos;  // sorted
  int64_t tokens, vocab;
  int chunk;                  // sorted tokens per block
  int dim;
  const void* grad;
  int64_t ld_grad;
  void* table;
  int64_t ld_table;
  float scale;
  int accumulate;
  float* part;                // [chunks][2][pitch]: sums of the runs that began before the chunk, and that go on behind it
  int64_t pitch;
  uint32_t slabs, sum_blocks; // pieces of 128 threads in a row; blocks that sum
  int fill_rows;              // rows that each of the other blocks looks after
  const uint32_t* touched;
  FillArgs fill;
};
template <class T, bool Vec>
__device__ __forceinline__ void finish_row(const SumArgs& p, uint32_t row, int col, float* f) {
  constexpr int N = Piece<T>::N;
  T* dst = static_cast<T*>(p.table) + row * p.ld_table + col;
  const int left = p.dim - col;
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] *= p.scale;
  if (p.accumulate) {
    float old[N];
    get_values<T, Vec>(dst, left, old);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] += old[i];
  }
  put_values<T, Vec>(dst, left, f);
}
// Rows v0 .. v0 + rows - 1 but for those that have a token, a warp each.
__device__ void zero_untouched(const SumArgs& p, int64_t v0, int rows) {
  for (int64_t r = v0 + (threadIdx.x >> 5); r < v0 + rows; r += 4)
    if (!(p.touched[r / 32] >> (r % 32) & 1u)) zero_bytes(p.fill.table + r * p.fill.pitch_bytes, p.fill.row_bytes, threadIdx.x & 31, 32);
}
// The first p.sum_blocks blocks: a chunk's sums for 128 pieces of a row's columns, each thread its piece over the chunk's tokens in
// order.  The others: zeros.
template <class T, bool Vec>
__global__ void __launch_bounds__(128) sum_kernel(const SumArgs p) {
  tck::chain_wait();
  constexpr int N = Piece<T>::N;
  extern __shared__ uint32_t list[];  // [chunk] rows, [chunk] tokens
  if (blockIdx.x >= p.sum_blocks) {
    const int64_t v0 = p.fill.early + (int64_t)(blockIdx.x - p.sum_blocks) * p.fill_rows;
    zero_untouched(p, v0, (int)min((int64_t)p.fill_rows, p.fill.rows - v0));
    return;
  }
  const int64_t me = blockIdx.x / p.slabs, first = me * p.chunk;
  const int slab = blockIdx.x % p.slabs;
  const int n = (int)min((int64_t)p.chunk, p.tokens - first);
  for (int i = threadIdx.x; i < n; i += 128) { list[i] = p.key[first + i]; list[p.chunk + i] = p.pos[first + i]; }
  __syncthreads();
  const int col = (slab * 128 + threadIdx.x) * N, left = p.dim - col;
  if (left <= 0) return;
  const T* grad = static_cast<const T*>(p.grad) + col;
  const uint32_t none = (uint32_t)p.vocab;
  const uint32_t prev = first > 0 ? p.key[first - 1] : none, next = first + n < p.tokens ? p.key[first + n] : none;
  float sum[N] = {};
  int begin = 0;  // of the run
  constexpr int U = 8;
  for (int i0 = 0; i0 < n; i0 += U) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < n && list[i0 + u] != none) get_values<T, Vec>(grad + (int64_t)list[p.chunk + i0 + u] * p.ld_grad, left, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      const uint32_t row = list[i];
      if (row == none) break;  // sorted: nothing but tokens without a row from here on
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k] += v[u][k];
      const uint32_t after = i + 1 < n ? list[i + 1] : next;
      if (i + 1 < n && after == row) continue;
      const bool goes_on = i + 1 == n && after == row, came = begin == 0 && prev == row;
      if (!goes_on && !came) {
        finish_row<T, Vec>(p, row, col, sum);
      } else {
        float* dst = p.part + (me * 2 + (came ? 0 : 1)) * p.pitch + col;
#pragma unroll
        for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(dst + k) = make_float4(sum[k], sum[k + 1], sum[k + 2], sum[k + 3]);
      }
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k] = 0.f;
      begin = i + 1;
    }
  }
}
// Runs over several chunks: the block of the chunk in which one begins adds up its parts in order.
template <class T, bool Vec>
__global__ void __launch_bounds__(128) join_kernel(const SumArgs p) {
  tck::chain_wait();
  constexpr int N = Piece<T>::N, U = 8;
  const int64_t chunks = (p.tokens + p.chunk - 1) / p.chunk, me = blockIdx.x / p.slabs;
  const int slab = blockIdx.x % p.slabs;
  if (me + 1 >= chunks) return;
  const int64_t first = me * p.chunk, end = first + p.chunk;
  const uint32_t row = p.key[end - 1], none = (uint32_t)p.vocab;
  if (row == none || p.key[end] != row) return;
  if (first > 0 && p.key[first] == row && p.key[first - 1] == row) return;  // began in an earlier chunk
  // the last chunk that the run reaches: sorted, so it reaches those whose first token is the row's; every warp looks at 32 at a time
  int64_t last = me;
  for (int64_t c = me + 1;; c += 32) {
    const int64_t mine = c + (threadIdx.x & 31);
    const unsigned reached = __ballot_sync(0xffffffffu, mine < chunks && p.key[min(mine, chunks - 1) * p.chunk] == row);
    last += __popc(reached);
    if (reached != 0xffffffffu) break;
  }
  const int col = (slab * 128 + threadIdx.x) * N;
  if (p.dim - col <= 0) return;
  float sum[N];
  const float* part = p.part + col;
#pragma unroll
  for (int k = 0; k < N; ++k) sum[k] = part[(me * 2 + 1) * p.pitch + k];
  for (int64_t c0 = me + 1; c0 <= last; c0 += U) {
    float4 v[U][N / 4];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u <= last)
#pragma unroll
        for (int k = 0; k < N / 4; ++k) v[u][k] = *reinterpret_cast<const float4*>(part + (c0 + u) * 2 * p.pitch + 4 * k);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u <= last)
#pragma unroll
        for (int k = 0; k < N / 4; ++k) { sum[4 * k] += v[u][k].x; sum[4 * k + 1] += v[u][k].y; sum[4 * k + 2] += v[u][k].z; sum[4 * k + 3] += v[u][k].w; }
  }
  finish_row<T, Vec>(p, row, col, sum);
}

// ---- host ----
// Short chunks where there are few tokens, for the sake of blocks; longer ones for the sake of partial sums.
int chunk_of(int64_t tokens) { return tokens <= 8192 ? 16 : tokens <= 65536 ? 32 : tokens <= 262144 ? 64 : 256; }
int passes_of(int64_t vocab) {
  int bits = 1;
  while ((int64_t(1) << bits) <= vocab) ++bits;  // keys are 0 .. vocab
  return (bits + kDigitBits - 1) / kDigitBits;
}
int64_t part_pitch(int64_t dim) { return (dim + 7) / 8 * 8; }

struct Buffers {
  uint32_t *key[2], *pos[2], *sorted_key, *sorted_pos, *hist, *touched;
  float* part;
};
size_t carve(const TcOpShape& p, char* base, Buffers* b) {
  TcCarver c{base};
  const int64_t t = p.tokens;
  const bool passes = t > kOneBlock;
  for (int i = 0; i < 2; ++i) {
    b->key[i] = c.take<uint32_t>(passes ? t : 0);
    b->pos[i] = c.take<uint32_t>(passes ? t : 0);
  }
  b->sorted_key = c.take<uint32_t>(t);
  b->sorted_pos = c.take<uint32_t>(t);
  b->hist = c.take<uint32_t>(passes ? std::max((t + 4 * kSortThreads - 1) / (4 * kSortThreads), (std::min(t, kShortPasses) + kSortThreads - 1) / kSortThreads) * kDigits : 0);
  b->touched = c.take<uint32_t>((p.vocab + 31) / 32);
  // calls with fewer tokens may cut them into shorter chunks, of which there are at most these
  const int64_t chunks = std::max((t + chunk_of(t) - 1) / chunk_of(t), std::min<int64_t>((t + 15) / 16, 4096));
  b->part = c.take<float>(chunks * 2 * part_pitch(p.dim));
  return c.used;
}

bool vec16(const void* p, int64_t ld, int64_t dim, int es) { return !(reinterpret_cast<uintptr_t>(p) & 15) && ld * es % 16 == 0 && dim * es % 16 == 0; }

template <class T>
int lookup(const tc_op_plan& p, void* out, int64_t ld_out, const void* table, int64_t ld_table, const void* ids, int wide, int64_t tokens, cudaStream_t stream) {
  const int es = sizeof(T);
  const bool vec = vec16(out, ld_out, p.dim, es) && vec16(table, ld_table, p.dim, es);
  const int64_t pieces = tokens * ((p.dim + (vec ? 16 / es : 1) - 1) / (vec ? 16 / es : 1));
  const unsigned grid = (unsigned)std::min<int64_t>((pieces + 255) / 256, (int64_t)p.sms * 32);
  TC_CUDA_OK(tck::launch_chained(true, vec ? lookup_kernel<T, true> : lookup_kernel<T, false>, dim3(grid), 256u, 0, stream, static_cast<T*>(out), ld_out,
                                 static_cast<const T*>(table), ld_table, ids, wide, tokens, p.vocab, (int)p.dim, (float)p.scale));
  return TC_OK;
}

template <class T>
int table_grad(const tc_op_plan& p, const Buffers& b, void* dtable, int64_t ld_table, const void* grad, int64_t ld_grad, const void* ids, int wide, int64_t tokens,
               int accumulate, cudaStream_t stream) {
  const int es = sizeof(T);
  // What the sorting kernels zero meanwhile takes about as long as they do; the summing kernel does the rest.
  FillArgs fill{accumulate ? nullptr : static_cast<char*>(dtable), p.vocab, ld_table * es, p.dim * es, 0};
  const int64_t bytes = p.vocab * p.dim * es;
  const bool one_block = tokens <= kOneBlock;
  if (!accumulate) fill.early = tokens == 0 ? p.vocab : std::min<int64_t>(p.vocab, (int64_t)(p.vocab * std::min(1.0, kEarlyBytes * (one_block ? 4 : 2 * passes_of(p.vocab)) / bytes)));
  const int early_blocks = (int)std::min<int64_t>(p.sms - 1, (fill.early * p.dim * es + 32767) / 32768);
  SortArgs s{ids, wide, tokens, p.vocab, passes_of(p.vocab), {b.key[0], b.key[1]}, {b.pos[0], b.pos[1]}, b.sorted_key, b.sorted_pos, b.hist, b.touched, fill};
  if (one_block) {
    const int items = tokens <= kSortThreads ? 1 : kOneBlockItems;
    TC_CUDA_OK(tck::launch_chained(true, items == 1 ? sort_one_kernel<1> : sort_one_kernel<kOneBlockItems>, dim3(1 + early_blocks),
                                   (unsigned)kSortThreads, one_block_smem(items), stream, s));
  } else {
    const bool few = tokens <= kShortPasses;
    const int per = kSortThreads * (few ? 1 : 4), blocks = (int)((tokens + per - 1) / per), parts = 2 * s.passes;
    for (int pass = 0; pass < s.passes; ++pass) {
      TC_CUDA_OK(tck::launch_chained(true, few ? sort_count_kernel<1> : sort_count_kernel<4>, dim3(blocks + early_blocks), (unsigned)kSortThreads, 0, stream, s, pass, blocks, 2 * pass, parts));
      TC_CUDA_OK(tck::launch_chained(true, few ? sort_place_kernel<1> : sort_place_kernel<4>, dim3(blocks + early_blocks), (unsigned)kSortThreads, 0, stream, s, pass, blocks, 2 * pass + 1, parts));
    }
  }
  if (tokens == 0) return TC_OK;
  const int chunk = chunk_of(tokens);
  const int64_t chunks = (tokens + chunk - 1) / chunk, slabs = (p.dim + 128 * Piece<T>::N - 1) / (128 * Piece<T>::N);
  const int fill_rows = (int)std::min<int64_t>(1024, std::max<int64_t>(1, 131072 / (p.dim * es)));
  const int64_t fill_blocks = accumulate ? 0 : (p.vocab - fill.early + fill_rows - 1) / fill_rows;
  if (chunks * slabs + fill_blocks > INT32_MAX) return TC_ERR_UNSUPPORTED;
  const SumArgs a{b.sorted_key, b.sorted_pos, tokens, p.vocab, chunk, (int)p.dim, grad, ld_grad, dtable, ld_table, (float)p.scale, accumulate, b.part, part_pitch(p.dim),
                  (uint32_t)slabs, (uint32_t)(chunks * slabs), fill_rows, b.touched, fill};
  const bool vec = vec16(dtable, ld_table, p.dim, es) && vec16(grad, ld_grad, p.dim, es);
  TC_CUDA_OK(tck::launch_chained(true, vec ? sum_kernel<T, true> : sum_kernel<T, false>, dim3((unsigned)(chunks * slabs + fill_blocks)), 128u, (size_t)chunk * 8, stream, a));
  if (chunks > 1)
    TC_CUDA_OK(tck::launch_chained(true, vec ? join_kernel<T, true> : join_kernel<T, false>, dim3((unsigned)(chunks * slabs)), 128u, 0, stream, a));
  return TC_OK;
}

bool odd_address(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace

size_t tc_embed_workspace(const TcOpShape& p) {
  Buffers b;
  return carve(p, nullptr, &b);
}

int tc_embed_prepare() {
  TC_CUDA_OK(cudaFuncSetAttribute(sort_one_kernel<kOneBlockItems>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)one_block_smem(kOneBlockItems)));
  return TC_OK;
}

std::string tc_embed_json(const TcOpShape& p) {
  return "{\"operator\":\"embedding\",\"dtype\":\"" + std::string(p.dtype == TC_BF16 ? "bf16" : p.dtype == TC_F16 ? "f16" : "f32") +
         "\",\"tokens\":" + std::to_string(p.tokens) + ",\"vocab\":" + std::to_string(p.vocab) + ",\"dim\":" + std::to_string(p.dim) +
         ",\"workspace_bytes\":" + std::to_string(tc_embed_workspace(p)) + "}";
}

// a: what is written, whose rows may not overlap; b: what is read.  Without tokens there is nothing to point at.
static int check(const tc_op_plan* p, const void* a, int64_t ld_a, const void* b, int64_t ld_b, const void* ids, int index_dtype, int64_t tokens) {
  if (!p || p->kind != TC_OP_EMBEDDING || (tokens && (!a || !b || !ids)) || (index_dtype != TC_I32 && index_dtype != TC_I64)) return TC_ERR_INVALID_ARG;
  if (tokens < 0 || tokens > p->tokens || ld_a < p->dim || ld_b < 0) return TC_ERR_EXTENT;
  const int es = tc_elem_bytes(p->dtype);
  if (odd_address(a, es) || odd_address(b, es) || odd_address(ids, index_dtype == TC_I64 ? 8 : 4)) return TC_ERR_ALIGNMENT;
  return TC_OK;
}

extern "C" int tc_embedding_execute(tc_op_plan* p, void* out, int64_t ld_out, const void* table, int64_t ld_table, const void* ids, int index_dtype,
                                    int64_t tokens, void* stream) {
  int st = check(p, out, ld_out, table, ld_table, ids, index_dtype, tokens);
  if (st == TC_OK) st = tc_op_commit_for(p, static_cast<cudaStream_t>(stream));
  if (st != TC_OK || tokens == 0) return st;
  int dev = 0;
  TC_CUDA_OK(cudaGetDevice(&dev));
  if (dev != p->device) return TC_ERR_STATE;
  const int wide = index_dtype == TC_I64;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case TC_F32: return lookup<float>(*p, out, ld_out, table, ld_table, ids, wide, tokens, s);
    case TC_BF16: return lookup<__nv_bfloat16>(*p, out, ld_out, table, ld_table, ids, wide, tokens, s);
    default: return lookup<__half>(*p, out, ld_out, table, ld_table, ids, wide, tokens, s);
  }
}

extern "C" int tc_embedding_execute_grad(tc_op_plan* p, void* dtable, int64_t ld_dtable, const void* grad, int64_t ld_grad, const void* ids, int index_dtype,
                                         int64_t tokens, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check(p, dtable, ld_dtable, grad, ld_grad, ids, index_dtype, tokens);
  if (st == TC_OK && !dtable) st = TC_ERR_INVALID_ARG;
  if (st != TC_OK) return st;
  TcScratch scratch;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = scratch.open(p, TC_OP_EMBEDDING, workspace, workspace_bytes, s);
  if (st != TC_OK || (tokens == 0 && accumulate)) return st;
  Buffers b;
  carve(*p, scratch.base, &b);
  const int wide = index_dtype == TC_I64, add = accumulate != 0;
  switch (p->dtype) {
    case TC_F32: return scratch.close(table_grad<float>(*p, b, dtable, ld_dtable, grad, ld_grad, ids, wide, tokens, add, s));
    case TC_BF16: return scratch.close(table_grad<__nv_bfloat16>(*p, b, dtable, ld_dtable, grad, ld_grad, ids, wide, tokens, add, s));
    default: return scratch.close(table_grad<__half>(*p, b, dtable, ld_dtable, grad, ld_grad, ids, wide, tokens, add, s));
  }
}

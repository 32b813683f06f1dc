// Persistent matrix product of 16-bit operands on tcgen05 (kind::f16, fp32 accumulators in tensor memory) whose result never
// leaves the chip as it is: an epilogue type turns each accumulator tile into what the operator around it keeps.
//
//   D[m, n] = sum_k A[m, k] * B[n, k]        A, B both bf16 or both fp16, each with either index the fastest
//
//   CG = 2   256 x 256 tiles on pairs of CTAs (cta_group::2): each CTA fetches 128 rows of A and 128 of B per stage and
//            both are multiplied by the first CTA's one MMA thread, so an operand byte fetched from L2 serves 256 rows.
//   CG = 1   128 x BN tiles, one CTA each, for problems that would leave most pairs without a tile.
//
//   warps 0-7  EPILOGUE  a thread holds one row of its CTA's 128 x BN part, half of its columns; two accumulators, so a tile's
//                        epilogue runs under the next tile's products
//   warps 8, 10  LOADERS  for A and for B: tiled TMA boxes of 64 k by 128 rows (128-byte swizzle), or of 64 rows
//                        by BK k where the row index is the fastest: the layouts the MMA's descriptors name K-major and MN-major.
//                        What a loader and the MMA's warp do per stage -- wait, announce, issue, commit -- is what bounds the
//                        loop: one loader for both operands was 5 % slower on 8192 x 2048 x 131072, stages of 64 k instead of
//                        128 20 %, a condition on each MMA 10 %; loops that one lane goes through by itself 2 % on 4096 x 2048 x
//                        8192 and 12 % on 777 x 555 x 1023.
//   warp 9     MMA       (of the pair's first CTA)
//
// A stage is full when both CTAs' boxes have landed: both signal the first CTA's barrier.  Items (tile, slice of K, matrix of
// the batch) are dealt out in order, tiles of 16 rows of tiles at a time so that what runs together shares operands in L2.
// Every wait is bounded and reports through args.status.
//
// Measured on one B200: the statistics of 2048 rows, K = 1024, 32768 columns 91 us (1510 TFLOP/s, 0.93 of the measured burst rate); of 7782
// rows, K = 2048, 131072 columns 2.9 ms (1440 TFLOP/s); gradients by the logits there 3.3 ms and both products with them 6.6 ms (1270
// TFLOP/s): the rate a library product sustains under the power cap is 1368.  Small sums and few tiles are bound by the chain
// load, products, epilogue of one tile, about 5 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "tc_elem.cuh"
#include "tc_wd_kernel.cuh"
#include "tc_wm.h"

namespace tck {

template <int CG_, int BN_, int BK_>
struct WmCfg {
  static constexpr int CG = CG_, BN = BN_, BM = 128 * CG_, BK = BK_;  // BK: 64 or 128
  static constexpr int BROWS = BN / CG;                        // rows of B a CTA fetches
  static constexpr int A_BYTES = 128 * BK * 2, B_BYTES = BROWS * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = BK == 128 ? 3 : CG == 2 ? 6 : 5;  // five leave room for the next kernel's first blocks
  static constexpr int COLS = BN / 2;                          // columns of an epilogue thread
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int EPI_WARPS = 8, THREADS = 352;
  static constexpr int OUT_BYTES = 4096;                       // per epilogue warp: 32 rows of 128 bytes
  static constexpr int NBARS = 2 * STAGES + 5;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * OUT_BYTES + NBARS * 8 + 16;
  static_assert(SMEM_BYTES <= 232448 && BROWS % 64 == 0 && COLS % 32 == 0 && TMEM_COLS <= 512, "tile");
};

// ---- instructions ----
// Shared-memory descriptor with the 128-byte swizzle.  K-major: rows of 64 k (128 bytes), 8 rows per 1024-byte atom, `sbo` to
// the next 8 rows.  MN-major: rows of 64 m (or n), one per k, 8 of them per atom, `sbo` to the next 8 k and `lbo` to the next 64 m.
__device__ __forceinline__ uint64_t wm_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) | ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) |
         (2ull << 61);
}
// kind::f16, fp32 accumulators; bf: both operands bf16, else both fp16.
__host__ __device__ constexpr uint32_t wm_idesc(int m, int n, bool bf, bool a_mn, bool b_mn) {
  return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void wm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void wm_commit(uint64_t* bar) {
  if constexpr (CG == 2) tc05_pair_commit(bar);
  else tc05_commit(bar);
}
// Box at (c0, c1) of matrix c2 into this CTA's shared memory; the bytes count on `bar` of the pair's first CTA.
template <int CG>
__device__ __forceinline__ void wm_load(void* dst, const TcTensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  if constexpr (CG == 2)  // bit 24 of a shared::cluster address tells the pair's CTAs apart
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
                     smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar) & 0xFEFFFFFFu)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void wm_store(const TcTensorMap* map, const void* src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void wm_reduce(const TcTensorMap* map, const void* src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];\n" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void wm_ld32(uint32_t taddr, float* v) {
  tc05_ld16(taddr, v);
  tc05_ld16(taddr + 16, v + 16);
  tc05_wait_ld();
}
__device__ __forceinline__ uint32_t wm_pack(float a, float b, bool bf) {  // round to nearest
  uint32_t r;
  if (bf) asm("cvt.rn.bf16x2.f32 %0, %2, %1;\n" : "=r"(r) : "f"(a), "f"(b));
  else asm("cvt.rn.f16x2.f32 %0, %2, %1;\n" : "=r"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 wm_unpack(uint32_t v, bool bf) {
  if (bf) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// Sum of eight squares: in fp32, or in fp64 where one might have passed fp32's range on either side (or there is nothing but zeros).
__device__ __forceinline__ double wm_squares8(const float* f) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s = fmaf(f[k], f[k], s);
  if (s > 1e-30f && s < INFINITY) return (double)s;  // squares lost below 2^-149 are far below such a sum's own rounding
  double d = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) d = fma((double)f[k], (double)f[k], d);
  return d;
}
__device__ __forceinline__ float wm_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}

// One lane of a warp, the same each time.
__device__ __forceinline__ bool wm_elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one)::"memory");
  return one != 0;
}
// The same of a barrier that the pair's other CTA arrives on.
__device__ __forceinline__ bool wm_wait_cluster(uint64_t* bar, uint32_t parity, int* status, int code, uint32_t limit) {
  return __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, status, code, limit));
}

// ---- what an epilogue warp has; COLS: columns of a thread ----
struct WmPlace {
  uint32_t row0, col0;  // first row and column of the item's part that this CTA holds
  uint32_t M, N;        // of the problem
  int z, slice;
  bool empty;           // no k: the accumulator was not written and stands for zeros
  bool mirror;          // also store the transposed tile
  bool second;          // of the launch's second product
};
// 32 rows of 128 bytes: 16-byte piece c of row r at c ^ (r % 8), the layout of a box with the 128-byte swizzle.
__device__ __forceinline__ void wm_stage16(unsigned char* out, int lane, int piece, uint4 v) {
  *reinterpret_cast<uint4*>(out + lane * 128 + ((piece ^ (lane & 7)) << 4)) = v;
}
__device__ __forceinline__ void wm_out_free() {  // the copy before has read the staging area
  asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void wm_out_written() {
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void wm_out_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }

// 64 columns of 32 rows, packed in pairs, to their place: one box where a tensor map describes the output, else element by
// element along whichever index is contiguous.
__device__ __forceinline__ void wm_put_tile(const WmOut& o, const TcTensorMap* map, unsigned char* out, int lane, uint32_t row, uint32_t col,
                                            const WmPlace& at, const uint32_t (&p)[32]) {
  wm_out_free();
#pragma unroll
  for (int i = 0; i < 8; ++i) wm_stage16(out, lane, i, make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]));
  if (o.boxes) {
    wm_out_written();
    if (lane == 0 && row < at.M && col < at.N) wm_store(map, out, (int)col, (int)row, at.z);
    wm_out_commit();
    return;
  }
  __syncwarp();
  uint16_t* base = static_cast<uint16_t*>(o.ptr) + at.z * o.batch_stride;
  auto value = [&](int r, int c) { return *reinterpret_cast<const uint16_t*>(out + r * 128 + ((((c >> 3) ^ (r & 7)) << 4) | ((c & 7) << 1))); };
  const int rows = (int)min(32u, at.M > row ? at.M - row : 0u), cols = (int)min(64u, at.N > col ? at.N - col : 0u);
  if (o.col_stride != 1 && o.row_stride == 1) {
    if (lane < rows)
      for (int c = 0; c < cols; ++c) base[(int64_t)row + lane + (int64_t)(col + c) * o.col_stride] = value(lane, c);
  } else if (o.col_stride == 1) {  // two neighbouring elements per lane, from the row's first 4-byte boundary on
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      uint16_t* dst = base + (int64_t)(row + r) * o.row_stride + col;
      const uint32_t odd = (uint32_t)(reinterpret_cast<uintptr_t>(dst) >> 1) & 1u;
      const uint32_t mine = *reinterpret_cast<const uint32_t*>(out + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));  // 2 lane, 2 lane + 1
      const uint32_t next = __shfl_down_sync(0xffffffffu, mine, 1), pair = odd ? mine >> 16 | next << 16 : mine;
      const int c = 2 * lane + (int)odd;
      if (c + 1 < cols) *reinterpret_cast<uint32_t*>(dst + c) = pair;
      else if (c < cols) dst[c] = (uint16_t)pair;
      if (odd && lane == 0) dst[0] = (uint16_t)mine;
    }
  } else {
    for (int r = 0; r < rows; ++r)
      for (int c = lane; c < cols; c += 32) base[(int64_t)(row + r) * o.row_stride + (int64_t)(col + c) * o.col_stride] = value(r, c);
  }
  __syncwarp();
}

// Softmax statistics: each thread's largest logit and sum of exponentials over its columns, and its target's logit.
struct WmStats {
  static constexpr bool kAMn = false, kBMn = false, kSymmetric = false, kAdds = false, kTwo = false, kTerms = false, kSum = false;
  template <class CF, int COLS>
  __device__ static void run(const WmArgs& p, const WmPlace& at, uint32_t taddr, unsigned char*, int warp, int lane, uint4 (&)[8]) {
    constexpr float kLog2e = 1.4426950408889634f;
    const uint32_t row = at.row0 + 32 * (warp & 3) + lane, first = at.col0 + (warp >> 2) * COLS;
    const bool live = row < at.M;
    const int64_t target = !live ? -1 : p.stats.wide ? static_cast<const int64_t*>(p.stats.target)[row] : static_cast<const int32_t*>(p.stats.target)[row];
    const int64_t want = target >= 0 ? target - p.stats.first : -1;
    float top = -INFINITY, sum = 0.f;
    for (int c = 0; c < COLS; c += 32) {
      float v[32];
      wm_ld32(taddr + c, v);
      const uint32_t col = first + c;
      if (col >= at.N) break;  // the same for the whole warp
      if (want >= (int64_t)col && want < (int64_t)col + 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (want == (int64_t)col + i) p.stats.hit[row] = v[i];
      }
      if (col + 32 > at.N) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (col + i >= at.N) v[i] = -INFINITY;
      }
      float m = v[0];  // fmaxf drops NaN; the sum below keeps it
#pragma unroll
      for (int i = 1; i < 32; ++i) m = fmaxf(m, v[i]);
      m = fmaxf(m, top);
      const float shift = m == -INFINITY ? 0.f : m * kLog2e;  // nothing but -inf so far: exponentials are zeros, not NaN
      float s[4] = {sum * wm_exp2(top * kLog2e - shift), 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 32; ++i) s[i & 3] += wm_exp2(fmaf(v[i], kLog2e, -shift));
      sum = (s[0] + s[1]) + (s[2] + s[3]);
      top = m;
    }
    if (live) p.stats.part[(size_t)(p.stats.part0 + at.col0 / CF::BN * 2 + (warp >> 2)) * p.stats.pitch + row] = make_float2(top, sum);
  }
};

// The loss's gradient with respect to a piece's logits: (exp(l - lse) - [target]) * weight of the row, rounded once to the
// operands' type for the two products that follow.
struct WmProb {
  static constexpr bool kAMn = false, kBMn = false, kSymmetric = false, kAdds = false, kTwo = false, kTerms = false, kSum = false;
  template <class CF, int COLS>
  __device__ static void run(const WmArgs& p, const WmPlace& at, uint32_t taddr, unsigned char* out, int warp, int lane, uint4 (&)[8]) {
    constexpr float kLog2e = 1.4426950408889634f;
    const uint32_t row0 = at.row0 + 32 * (warp & 3), row = row0 + lane;
    const bool live = row < at.M;
    // rows of the tile that no token fills are zeros: they are k of the product for the table's gradient
    const WmRow r = live ? p.prob.rows[row] : WmRow{0.f, 0.f, -1};
    const int64_t want = live ? r.target - p.prob.first : -1;
    const bool bf = p.bf16 != 0;
    const uint32_t padded = (at.M + p.prob.pad - 1) / p.prob.pad * p.prob.pad;  // rows up to the end of a stage of k are written too
    WmPlace put = at;
    put.M = min(padded, p.prob.rows_most);
    for (int c = 0; c < COLS; c += 64) {
      const uint32_t col = at.col0 + (warp >> 2) * COLS + c;
      if (col >= at.N) break;
      uint32_t packed[32];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        wm_ld32(taddr + c + 32 * h, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = wm_exp2(fmaf(v[i], kLog2e, -r.lse2));
        const int64_t rel = want - (int64_t)(col + 32 * h);
        if (rel >= 0 && rel < 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (rel == i) v[i] -= 1.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[16 * h + i] = live ? wm_pack(v[2 * i] * r.weight, v[2 * i + 1] * r.weight, bf) : 0u;
      }
      wm_put_tile(p.out, &p.map_d, out, lane, row0, col, put, packed);
    }
  }
};

// Two products.  First: fp32 partial results, stored or added to what earlier pieces left.  Second: the product itself, scaled and
// rounded once.
struct WmGrads {
  static constexpr bool kAMn = false, kBMn = true, kSymmetric = false, kAdds = false, kTwo = true, kTerms = false, kSum = false;
  template <class CF, int COLS>
  __device__ static void run(const WmArgs& p, const WmPlace& at, uint32_t taddr, unsigned char* out, int warp, int lane, uint4 (&)[8]) {
    const uint32_t row = at.row0 + 32 * (warp & 3);
    if (at.second) {
      const float scale = *p.grads.scale;
      const bool bf = p.out.bf16 != 0;
      for (int c = 0; c < COLS; c += 64) {
        const uint32_t col = at.col0 + (warp >> 2) * COLS + c;
        if (col >= at.N) break;
        uint32_t packed[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[32];
          wm_ld32(taddr + c + 32 * h, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) packed[16 * h + i] = at.empty ? 0u : wm_pack(v[2 * i] * scale, v[2 * i + 1] * scale, bf);
        }
        wm_put_tile(p.out, &p.second.map_d, out, lane, row, col, at, packed);
      }
      return;
    }
    for (int c = 0; c < COLS; c += 32) {
      const uint32_t col = at.col0 + (warp >> 2) * COLS + c;
      if (col >= at.N) break;
      float v[32];
      wm_ld32(taddr + c, v);
      wm_out_free();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float4 f = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        if (at.empty) f = make_float4(0.f, 0.f, 0.f, 0.f);
        wm_stage16(out, lane, i, *reinterpret_cast<uint4*>(&f));
      }
      wm_out_written();
      if (lane == 0 && row < at.M) {
        if (p.grads.add) wm_reduce(&p.map_d, out, (int)col, (int)row, at.slice);
        else wm_store(&p.map_d, out, (int)col, (int)row, at.slice);
      }
      wm_out_commit();
    }
  }
};

// alpha * product + beta * (a matrix of the same place), fp16 in between and in the output's type at the end.  kSym: the result
// is symmetric, tiles above the diagonal only, each stored a second time transposed.
//
// Terms: operands, intermediate results and what is added are sums of two fp16 numbers, v = hi + lo (hi is v rounded, lo the rest:
// about 18 bits of entries near 2^-8, 22 of larger ones), in two planes, and the product is hi hi + lo hi + hi lo in one accumulator:
// three times the products.  terms 1: both operands have hi only; 2: hi hi + lo hi (B has hi only); 3: all three.
template <bool Sym, bool BMn, bool Terms>
struct WmAffine {
  static constexpr bool kAMn = false, kBMn = BMn, kSymmetric = Sym, kAdds = true, kTwo = false, kTerms = Terms, kSum = false;
  // 64 columns of a row of the matrix that the product is added to; rows are padded to 8 elements
  template <int N>
  __device__ static void fetch(const WmArgs& p, const WmPlace& at, int warp, int lane, uint32_t col, uint4 (&old)[N], int plane = 0) {
    const WmAffineArgs& f = p.affine;
    const uint32_t row = at.row0 + 32 * (warp & 3) + lane;
    const uint16_t* add = static_cast<const uint16_t*>(f.add) + (Terms ? 2 * at.z + plane : at.z) * f.add_batch + (int64_t)row * f.add_pitch + col;
#pragma unroll
    for (int i = 0; i < N; ++i) old[i] = f.add && row < at.M && col + 8 * i < at.N ? *reinterpret_cast<const uint4*>(add + 8 * i) : make_uint4(0, 0, 0, 0);
  }
  template <class CF, int COLS>
  __device__ static void run(const WmArgs& p, const WmPlace& at, uint32_t taddr, unsigned char* out, int warp, int lane, uint4 (&old)[8]) {
    const WmAffineArgs& f = p.affine;
    const float s = f.scale ? f.scale[at.z] : 1.f;
    const float alpha = f.alpha * (f.scale_power == 2 ? s * s : f.scale_power == 1 ? s : 1.f), beta = f.beta * (f.scale_power == 1 ? s : 1.f);
    const bool bf = p.out.bf16 != 0;
    for (int c = 0; c < COLS; c += 64) {
      const uint32_t col = at.col0 + (warp >> 2) * COLS + c;
      if (col >= at.N) break;
      if (c > 0) fetch(p, at, warp, lane, col, old);
      uint32_t packed[32], rest[Terms ? 32 : 1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        uint4 low[4];
        if constexpr (Terms) fetch(p, at, warp, lane, col + 32 * h, low, 1);
        wm_ld32(taddr + c + 32 * h, v);
        float shift = 0.f;
        int diagonal = -1;
        if (Sym && !at.mirror && f.shift != 0.f) {
          shift = f.shift;
          diagonal = (int)(at.row0 + 32 * (warp & 3) + lane) - (int)(col + 32 * h);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2 o = wm_unpack((&old[4 * h + (i >> 2)].x)[i & 3], false);
          if constexpr (Terms) {
            const float2 l = wm_unpack((&low[i >> 2].x)[i & 3], false);
            o.x += l.x;
            o.y += l.y;
          }
          float a = fmaf(alpha, v[2 * i], beta * o.x), b = fmaf(alpha, v[2 * i + 1], beta * o.y);
          if (Sym) {
            if (diagonal == 2 * i) a -= shift;
            if (diagonal == 2 * i + 1) b -= shift;
          }
          packed[16 * h + i] = wm_pack(a, b, bf);
          if constexpr (Terms) {
            const float2 hi = wm_unpack(packed[16 * h + i], false);
            rest[16 * h + i] = wm_pack(a - hi.x, b - hi.y, false);
          }
        }
      }
      if (Terms && p.out.planes == 2) {
        WmPlace plane = at;
        plane.z = 2 * at.z;
        put(p, out, warp, lane, col, plane, packed);
        ++plane.z;
        if constexpr (Terms) put(p, out, warp, lane, col, plane, rest);
      } else {
        put(p, out, warp, lane, col, at, packed);
      }
    }
  }
  __device__ static void put(const WmArgs& p, unsigned char* out, int warp, int lane, uint32_t col, const WmPlace& at, const uint32_t (&packed)[32]) {
    const uint32_t row0 = at.row0 + 32 * (warp & 3);
    wm_put_tile(p.out, &p.map_d, out, lane, row0, col, at, packed);
    if (Sym && at.mirror) {  // 64 rows of 32 columns, dense
      wm_out_free();
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        *reinterpret_cast<uint16_t*>(out + (2 * i) * 64 + lane * 2) = (uint16_t)packed[i];
        *reinterpret_cast<uint16_t*>(out + (2 * i + 1) * 64 + lane * 2) = (uint16_t)(packed[i] >> 16);
      }
      wm_out_written();
      if (lane == 0 && row0 < at.M && col < at.N) wm_store(&p.map_t, out, (int)row0, (int)col, at.z);
      wm_out_commit();
    }
  }
};

// A weight's gradient, out[n, m], both operands with k the slowest: 16 or 32 bits, stored or added to what is there; or fp32 slices for
// a later sum.  Neighbouring lanes hold neighbours of a row of the result, so stores need neither staging nor alignment.
// A may be the sum of two matrices (p.weight.terms): each step of k is taken with the first, then with the second.
struct WmWeight {
  static constexpr bool kAMn = true, kBMn = true, kSymmetric = false, kAdds = false, kTwo = false, kTerms = false, kSum = true;
  template <class CF, int COLS>
  __device__ static void run(const WmArgs& p, const WmPlace& at, uint32_t taddr, unsigned char*, int warp, int lane, uint4 (&)[8]) {
    const WmWeightArgs& f = p.weight;
    const uint32_t row = at.row0 + 32 * (warp & 3) + lane;
    for (int c = 0; c < COLS; c += 32) {
      const uint32_t col = at.col0 + (warp >> 2) * COLS + c;
      if (col >= at.N) break;
      float v[32];
      wm_ld32(taddr + c, v);
      const int cols = row < at.M ? (int)min(32u, at.N - col) : 0;
      auto put = [&](auto* out, bool add) {
        using T = std::remove_reference_t<decltype(*out)>;
        out += (int64_t)col * f.ld + row;
        if (cols == 32 && !add) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            *out = Elem<T>::put(v[i]);
            out += f.ld;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i < cols) *out = Elem<T>::put(add ? Elem<T>::get(*out) + v[i] : v[i]);
            out += f.ld;
          }
        }
      };
      if (f.type == TC_F32) put(static_cast<float*>(f.out) + at.slice * f.slice_stride, f.add != 0);
      else if (f.type == TC_BF16) put(static_cast<__nv_bfloat16*>(f.out), f.add != 0);
      else put(static_cast<__half*>(f.out), f.add != 0);
    }
  }
};

template <class CF, class EPI>
__global__ void __cluster_dims__(CF::CG, 1, 1) __launch_bounds__(CF::THREADS, 1) tc_wm_kernel(const __grid_constant__ WmArgs p) {
  constexpr int CG = CF::CG, BK = CF::BK, STAGES = CF::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* stages = smem_raw;
  unsigned char* outs = stages + STAGES * CF::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(outs + CF::EPI_WARPS * CF::OUT_BYTES);  // [STAGES] (first CTA) both CTAs' boxes have landed
  uint64_t* empty = full + STAGES;         // [STAGES] the MMAs that read them have completed
  uint64_t* acc_full = empty + STAGES;     // [2] an accumulator holds a finished tile
  uint64_t* acc_free = acc_full + 2;       // [2] (first CTA) both CTAs' epilogues have read it
  uint64_t* drained = acc_full + 4;        // the MMAs of a role that gave up have completed
  uint32_t* slot = reinterpret_cast<uint32_t*>(full + CF::NBARS);

  // `warp` is the same for the whole warp, and known to be: loaders and the MMA's warp go through their loops together and one lane issues, so
  // that what the instructions take is worked out once for the warp, in the registers that they take it from.
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_free + i, CG * CF::EPI_WARPS); }
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&p.map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&p.map_b)) : "memory");
  }
  if (warp == 9) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(slot)), "r"(CF::TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      tmem_alloc(slot, CF::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc05_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc05_fence_after();
  const uint32_t tmem = *slot;
  chain_wait();

  const uint32_t count = p.count ? (uint32_t)max(*p.count - p.count_first, 0) : 0u;
  const uint32_t M = p.count ? min(count, p.M) : p.M, N = p.N, K = p.K;
  const uint32_t tiles_m = (M + CF::BM - 1) / CF::BM, tiles_n = (N + CF::BN - 1) / CF::BN;
  const uint32_t tiles = EPI::kSymmetric ? tiles_n * (tiles_n + 1) / 2 : tiles_m * tiles_n;  // symmetric tiles are square
  const uint32_t terms = EPI::kSum ? (uint32_t)p.weight.terms : 1u;  // 1 or 2
  const uint32_t kblocks = (K + BK - 1) / BK * terms, slices = p.slices;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
  const uint32_t items1 = tiles * slices * p.batch;
  // The second product's items follow the first's, whose are longer: they fill up the last round.
  const uint32_t M2 = EPI::kTwo ? p.second.M : 0u, N2 = EPI::kTwo ? p.second.N : 0u, K2 = EPI::kTwo ? min(count, p.second.K) : 0u;
  const uint32_t tiles_m2 = (M2 + CF::BM - 1) / CF::BM, tiles_n2 = (N2 + CF::BN - 1) / CF::BN, kblocks2 = (K2 + BK - 1) / BK;
  const uint32_t total = items1 + tiles_m2 * tiles_n2;
  struct Item { uint32_t tm, tn, k0, k1, slice, z; bool second; };
  // 16 rows of tiles at a time, column by column
  auto grouped = [](uint32_t t, uint32_t all_m, uint32_t all_n, Item& it) {
    const uint32_t group = 16u * all_n, g = t / group, rows = min(16u, all_m - 16u * g), l = t % group;
    it.tm = 16u * g + l % rows;
    it.tn = l / rows;
  };
  auto item_of = [&](uint32_t i) {
    Item it;
    it.second = EPI::kTwo && i >= items1;
    if (it.second) {
      it.slice = it.z = it.k0 = 0;
      it.k1 = kblocks2;
      grouped(i - items1, tiles_m2, tiles_n2, it);
      return it;
    }
    uint32_t t = i % tiles;
    i /= tiles;
    it.slice = i % slices;
    it.z = i / slices;
    it.k0 = (uint32_t)((uint64_t)kblocks * it.slice / slices);
    it.k1 = EPI::kTerms ? kblocks * (uint32_t)p.terms : (uint32_t)((uint64_t)kblocks * (it.slice + 1) / slices);
    if constexpr (EPI::kSymmetric) {  // column tn has the tiles 0 .. tn
      uint32_t tn = (uint32_t)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
      while (tn * (tn + 1) / 2 > t) --tn;
      while ((tn + 1) * (tn + 2) / 2 <= t) ++tn;
      it.tn = tn;
      it.tm = t - tn * (tn + 1) / 2;
    } else {
      grouped(t, tiles_m, tiles_n, it);
    }
    return it;
  };
  const uint32_t limit = p.spin_limit;

  if (warp < CF::EPI_WARPS) {
    uint32_t n = 0;
    for (uint32_t i = first; i < total; i += step, ++n) {
      const uint32_t acc = n & 1u;
      const Item it = item_of(i);
      WmPlace at;
      at.row0 = it.tm * CF::BM + rank * 128;
      at.col0 = it.tn * CF::BN;
      at.M = it.second ? M2 : M;
      at.N = it.second ? N2 : N;
      at.second = it.second;
      at.z = (int)it.z;
      at.slice = (int)it.slice;
      at.empty = it.k0 == it.k1;
      at.mirror = EPI::kSymmetric && it.tm != it.tn;
      uint4 old[8];
      if constexpr (EPI::kAdds) EPI::fetch(p, at, warp, lane, at.col0 + (warp >> 2) * CF::COLS, old);  // under the tile's products
      if (!mbar_wait_warp(acc_full + acc, (n >> 1) & 1u, p.status, 20, limit)) break;
      tc05_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + acc * CF::BN;
      unsigned char* out = outs + warp * CF::OUT_BYTES;
      EPI::template run<CF, CF::COLS>(p, at, taddr + (warp >> 2) * CF::COLS, out, warp, lane, old);
      tc05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_first(acc_free + acc);
        else mbar_arrive(acc_free + acc);
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
  } else if (warp == 8 || warp == 10) {
    const bool loads_a = warp == 8, issues = wm_elect();
    uint32_t g = 0;
    bool alive = true;
    // which product is a constant of the loop over k: as a variable it cost 11 % on a large vocabulary
    auto fill = [&](const Item& it, auto second) {
      constexpr bool kSecond = decltype(second)::value;
      const TcTensorMap *ma = kSecond ? &p.second.map_a : &p.map_a, *mb = kSecond ? &p.second.map_b : &p.map_b;
      const int m0 = (int)(it.tm * CF::BM + rank * 128), n0 = (int)(it.tn * CF::BN + rank * CF::BROWS);
      int z = (int)it.z * (EPI::kTerms ? 2 : 1);  // of this loader's operand: hi hi, lo hi, hi lo
      uint32_t left = kblocks, term = 0;
      uint32_t kb = it.k0;
      for (uint32_t n = it.k1 - it.k0; n > 0; --n, ++kb, ++g) {
        if constexpr (EPI::kTerms) {
          if (left == 0) {
            left = kblocks;
            kb = 0;
            ++term;
            z = 2 * (int)it.z + (term == (loads_a ? 1u : 2u));
          }
          --left;
        }
        const uint32_t s = g % STAGES;
        if (g >= (uint32_t)STAGES && !mbar_wait_warp(empty + s, ((g / STAGES) - 1) & 1u, p.status, 21, limit)) { alive = false; break; }
        // tests only: one stage is left unannounced, so that the waits on it run out
        if (p.test_fault == 1 && blockIdx.x < CG && g == 1) continue;
        unsigned char* as = stages + s * CF::STAGE_BYTES;
        unsigned char* bs = as + CF::A_BYTES;
        const int k0 = (int)((EPI::kSum ? kb >> (terms - 1) : kb) * BK);
        if constexpr (EPI::kSum) z = loads_a ? (int)(kb & (terms - 1)) : 0;
        if (issues) {
          if (loads_a) {
            if (rank == 0) mbar_arrive_expect_tx(full + s, CG * CF::STAGE_BYTES);  // of both operands
            if constexpr (kSecond || EPI::kAMn) {
              wm_load<CG>(as, ma, m0, k0, z, full + s);
              wm_load<CG>(as + 128 * BK, ma, m0 + 64, k0, z, full + s);
            } else {
              wm_load<CG>(as, ma, k0, m0, z, full + s);
              if (BK == 128) wm_load<CG>(as + 16384, ma, k0 + 64, m0, z, full + s);
            }
          } else if constexpr (EPI::kBMn) {
#pragma unroll
            for (int h = 0; h < CF::BROWS; h += 64) wm_load<CG>(bs + h * 2 * BK, mb, n0 + h, k0, z, full + s);
          } else {
            wm_load<CG>(bs, mb, k0, n0, z, full + s);
            if (BK == 128) wm_load<CG>(bs + CF::BROWS * 128, mb, k0 + 64, n0, z, full + s);
          }
        }
        __syncwarp();
      }
    };
    for (uint32_t i = first; alive && i < total; i += step) {
      const Item it = item_of(i);
      if constexpr (EPI::kTwo) {
        if (it.second) fill(it, std::true_type());
        else fill(it, std::false_type());
      } else {
        fill(it, std::false_type());
      }
    }
    if (loads_a) chain_release();  // the next kernel may set itself up under the last tiles
    // A loader that gave up waits (with a limit) for the boxes that are under way; the first CTA's barriers count both CTAs'.
    if (!alive && rank == 0)
      for (uint32_t q = g > (uint32_t)STAGES ? g - STAGES : 0u; q < g; ++q)
        if (!(p.test_fault == 1 && blockIdx.x < CG && q == 1)) mbar_wait_warp(full + q % STAGES, (q / STAGES) & 1u, p.status, 21, limit);
  } else if (warp == 9 && rank == 0) {
    const bool issues = wm_elect();
    const uint32_t base = smem_u32(stages);
    uint32_t g = 0, n = 0;
    bool alive = true;
    auto multiply = [&](const Item& it, auto second) {
      constexpr bool kAMn = decltype(second)::value || EPI::kAMn;
      constexpr uint32_t idesc_mn = wm_idesc(CF::BM, CF::BN, false, kAMn, EPI::kBMn);
      const uint32_t idesc = idesc_mn | (p.bf16 ? (1u << 7) | (1u << 10) : 0u);
      const uint32_t acc = n & 1u, d = tmem + acc * CF::BN;
      if (n >= 2 && !wm_wait_cluster(acc_free + acc, ((n >> 1) - 1) & 1u, p.status, 22, limit)) { alive = false; return; }
      tc05_fence_after();
      for (uint32_t kb = it.k0; kb < it.k1; ++kb, ++g) {
        const uint32_t s = g % STAGES;
        if (!wm_wait_cluster(full + s, (g / STAGES) & 1u, p.status, 23, limit)) { alive = false; break; }
        tc05_fence_after();
        const uint64_t a = wm_desc(base + s * CF::STAGE_BYTES, kAMn ? 128 * BK : 16, 1024);
        const uint64_t b = wm_desc(base + s * CF::STAGE_BYTES + CF::A_BYTES, EPI::kBMn ? 128 * BK : 16, 1024);
        // a K step of 16: 32 bytes on in rows of 64 k, 64 k a box on; two groups of 8 k, 2048 bytes, where rows are one k each
        if (issues) {
#pragma unroll
          for (uint32_t k = 0; k < BK / 16; ++k) {
            const uint32_t a_at = kAMn ? k * 128u : (k >> 2) * (128 * 128 / 16) + (k & 3) * 2u;
            const uint32_t b_at = EPI::kBMn ? k * 128u : (k >> 2) * (CF::BROWS * 128 / 16) + (k & 3) * 2u;
            wm_mma<CG>(d, a + a_at, b + b_at, idesc, (kb > it.k0 || k > 0) ? 1u : 0u);
          }
          wm_commit<CG>(empty + s);
        }
        __syncwarp();
      }
      if (alive && issues) wm_commit<CG>(acc_full + acc);
      __syncwarp();
    };
    for (uint32_t i = first; alive && i < total; i += step, ++n) {
      const Item it = item_of(i);
      if constexpr (EPI::kTwo) {
        if (it.second) multiply(it, std::true_type());
        else multiply(it, std::false_type());
      } else {
        multiply(it, std::false_type());
      }
    }
    if (!alive) {  // what is under way must not outlive the memory it works on
      if (issues) wm_commit<CG>(drained);
      __syncwarp();
      mbar_wait_warp(drained, 0u, p.status, 23, limit);
    }
  }
  __syncwarp();
  tc05_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // neither CTA leaves while the other still reads its memory
  tc05_fence_after();
  if (warp == 9) {
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(CF::TMEM_COLS) : "memory");
    else
      tmem_dealloc(tmem, CF::TMEM_COLS);
  }
}

}  // namespace tck

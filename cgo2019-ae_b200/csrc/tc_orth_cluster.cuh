// The whole Newton-Schulz iteration of a matrix of up to 128 rows in one launch: a cluster of CTAs per matrix, nothing but the
// input and the result in global memory.
//
// Each CTA holds up to 512 columns of X in shared memory as fp16, in 64-column boxes of 64 or 128 rows with the 128-byte swizzle.  That
// one image is the K-major operand of A = X X^T (k: columns) and the MN-major one of B X (n: columns), so X is never laid out twice.
// Per step and CTA:
//   the CTA's part of A over its columns, 128 x 128 in tensor memory; its rows are dealt out over the cluster (each CTA sums
//   its share of the rows of all parts, in the CTAs' order), and every CTA gets all of A as fp16
//   A A and B = b A + c A A, by every CTA for itself: at most 8 MMAs, less than fetching it would take
//   B X over the CTA's columns, up to 128 x 512 in tensor memory; a X + B X rounded in place
// Terms: X, A and B are sums of two fp16 numbers in two images each (at most 192 columns of 128 rows per CTA then), products of
// them three.
// Two cluster barriers per step.  What bounds it is the chain of these small phases (each a few hundred cycles of MMAs between
// a barrier and a pass through registers), not bytes or products: twelve of 64 x 128 20 us for 5 steps, a 121 x 3357 batch of 7 72,
// of which a step's exchange of A's parts is half.
#pragma once
#include "tc_wm_kernel.cuh"

namespace tck {

struct OrthClusterArgs {
  const void* x;
  int64_t x_batch, x_row, x_col;        // strides of the orientation with fewer rows
  void* out;
  int64_t out_batch, out_row, out_col;
  int rows, cols, dtype, out_bf16, steps;
  int x_vec, out_vec;                   // eight columns of a row are aligned 16 (or 32) bytes
  int slab;                             // columns per CTA, a multiple of 64
  int tmem_cols;
  float4 coef[16];                      // per step: of x, of A x, of A A x, and what is subtracted from A's diagonal before
  double eps;
  int* status;
  uint32_t spin_limit;
  int test_fault;
};

constexpr int kOrthSlab = 512, kOrthThreads = 512, kOrthWarps = 16, kOrthGuard = 6;
// Images have 64 or 128 rows.  (The MMA's 128 rows of a first operand reach into what lies behind an image of 64: rows of the
// result that nobody reads.)
inline int orth_rows(int64_t m) { return m <= 64 ? 64 : 128; }
inline int orth_most_columns(int rows, bool terms) { return rows == 128 && terms ? 192 : kOrthSlab; }
inline int orth_cluster_smem(int slab, int rows, bool terms) { return (slab / 64 + rows / 64) * (terms ? 2 : 1) * rows * 128 + rows * 512 + 512; }

template <int Rows>
__device__ __forceinline__ int box_at(int r, int c) { return (c >> 6) * (Rows * 128) + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2; }
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster16(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <bool Terms, int Rows>
__global__ void __launch_bounds__(kOrthThreads, 1) orth_cluster_kernel(const __grid_constant__ OrthClusterArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int nbox = p.slab / 64;
  unsigned char* ximg = smem_raw;                // nbox boxes (per term)
  constexpr int T = Terms ? 2 : 1, kBox = Rows * 128, kSquare = Rows / 64;  // bytes of 64 columns; boxes of A and B
  unsigned char* aimg = ximg + T * nbox * kBox;  // kSquare boxes (per term)
  unsigned char* bimg = aimg + T * kSquare * kBox;  // as many ...
  const int xrest = nbox * kBox;                 // from a first term's image to the second's
  constexpr int rest2 = kSquare * kBox;          // ... A's and B's
  constexpr int kProducts = Terms ? 3 : 1;           // hi hi, lo hi, hi lo
  float* parts = reinterpret_cast<float*>(bimg);     // ... over this CTA's part of A, [Rows][128]
  double* sums = reinterpret_cast<double*>(bimg + Rows * 512);  // [8] the cluster's parts of the norm, [16] this block's warps'
  uint64_t* done = reinterpret_cast<uint64_t*>(sums + 8 + kOrthWarps);
  uint64_t* drained = done + 1;  // the MMAs of a CTA that gave up have completed
  uint32_t* slot = reinterpret_cast<uint32_t*>(drained + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t C = cluster_size(), rank = cluster_rank();
  const int z = blockIdx.x / C, m = p.rows, col0 = (int)rank * p.slab, n = min(p.slab, max(0, p.cols - col0));  // this CTA's columns
  if (tid == 0) {
    mbar_init(done, 1);
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    tmem_alloc(slot, p.tmem_cols);
    tmem_relinquish();
  }
  for (int i = tid; i < T * (nbox + kSquare) * kBox / 16; i += kOrthThreads) reinterpret_cast<uint4*>(ximg)[i] = make_uint4(0, 0, 0, 0);  // X and A
  chain_wait();

  // ---- the norm, then X as fp16 times the power of two that brings it to [2^5, 2^6) ----
  const int es = p.dtype == TC_F32 ? 4 : 2;
  const char* x = static_cast<const char*>(p.x) + (z * p.x_batch + col0 * p.x_col) * es;
  // A thread takes eight columns of a row at a time; neighbouring threads walk whichever index is contiguous.
  const bool turn = p.x_col != 1 && p.x_row == 1;
  const int per = (n + 7) / 8, pieces = m * per;
  auto place = [&](bool by_rows, int j, int* r, int* c) {
    const int q = j / (by_rows ? m : per), rest = j - q * (by_rows ? m : per);
    *r = by_rows ? rest : q;
    *c = 8 * (by_rows ? q : rest);
  };
  auto load32 = [&](int j, float* f) {
    int r, c;
    place(turn, j, &r, &c);
    const float* from = reinterpret_cast<const float*>(x) + r * p.x_row + c * p.x_col;
    if (p.x_vec) {
      const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = c + k < n ? from[k * p.x_col] : 0.f;
    }
  };
  auto load16 = [&](int j) {
    int r, c;
    place(turn, j, &r, &c);
    const uint16_t* from = reinterpret_cast<const uint16_t*>(x) + r * p.x_row + c * p.x_col;
    if (p.x_vec) return *reinterpret_cast<const uint4*>(from);
    uint32_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < n ? from[k * p.x_col] : 0u;
    return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  };
  auto unpack = [&](uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { const float2 t = wm_unpack(w[k], p.dtype == TC_BF16); f[2 * k] = t.x; f[2 * k + 1] = t.y; }
  };
  auto image = [&](int j) {  // where a piece goes
    int r, c;
    place(turn, j, &r, &c);
    return reinterpret_cast<uint4*>(ximg + box_at<Rows>(r, c));
  };
  double sum = 0;
  if (p.dtype == TC_F32) {
    constexpr int kBatch = 4;  // pieces under way
    for (int j0 = tid; j0 < pieces; j0 += kBatch * kOrthThreads) {
      float f[kBatch][8];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (j0 + u * kOrthThreads < pieces) load32(j0 + u * kOrthThreads, f[u]);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (j0 + u * kOrthThreads < pieces) sum += wm_squares8(f[u]);
    }
  } else {  // 16 bits: kept where X goes meanwhile
    constexpr int kBatch = 8;
    __syncthreads();  // the zeros are there
    for (int j0 = tid; j0 < pieces; j0 += kBatch * kOrthThreads) {
      uint4 v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (j0 + u * kOrthThreads < pieces) v[u] = load16(j0 + u * kOrthThreads);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (j0 + u * kOrthThreads >= pieces) break;
        float f[8];
        unpack(v[u], f);
        sum += wm_squares8(f);
        *image(j0 + u * kOrthThreads) = v[u];
      }
    }
  }
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) sums[8 + warp] = sum;
  __syncthreads();
  cluster_sync();  // every CTA of the cluster runs: its shared memory may be written
  if (tid < (int)C) {
    double all = 0;
    for (int w = 0; w < kOrthWarps; ++w) all += sums[8 + w];
    const uint32_t to = map_rank(smem_u32(sums + rank), tid);
    asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(to), "d"(all) : "memory");
  }
  cluster_sync();
  double square = 0;
  for (uint32_t c = 0; c < C; ++c) square += sums[c];
  const double norm = sqrt(square);
  int e = 0;
  const bool finite = norm < INFINITY;
  if (norm > 0 && finite) frexp(norm, &e);
  e = min(max(kOrthGuard - e, -126), 126);
  const float factor = ldexpf(1.f, e), rest = finite ? (float)(ldexp(1.0, -e) / (norm + p.eps)) : NAN;
  // Eight values to an image, the rest of their rounding to the second term's.
  auto put8 = [&](unsigned char* at, int to_rest, const float* f, bool bf = false) {
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = wm_pack(f[2 * k], f[2 * k + 1], bf);
    *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (Terms) {
      uint32_t l[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 got = wm_unpack(h[k], false);
        l[k] = wm_pack(f[2 * k] - got.x, f[2 * k + 1] - got.y, false);
      }
      *reinterpret_cast<uint4*>(at + to_rest) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  };
  // Eight values of an image, both terms.
  auto get8 = [&](const unsigned char* at, int to_rest, float* f) {
    const uint4 a = *reinterpret_cast<const uint4*>(at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { const float2 t = wm_unpack(w[k], false); f[2 * k] = t.x; f[2 * k + 1] = t.y; }
    if constexpr (Terms) {
      const uint4 b = *reinterpret_cast<const uint4*>(at + to_rest);
      const uint32_t v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) { const float2 t = wm_unpack(v[k], false); f[2 * k] += t.x; f[2 * k + 1] += t.y; }
    }
  };
  auto put_scaled = [&](unsigned char* at, float* f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= factor;
    put8(at, xrest, f);
  };
  if (p.dtype == TC_F32) {
    constexpr int kBatch = 4;
    for (int j0 = tid; j0 < pieces; j0 += kBatch * kOrthThreads) {
      float f[kBatch][8];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (j0 + u * kOrthThreads < pieces) load32(j0 + u * kOrthThreads, f[u]);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (j0 + u * kOrthThreads < pieces) put_scaled(reinterpret_cast<unsigned char*>(image(j0 + u * kOrthThreads)), f[u]);
    }
  } else {
#pragma unroll 2
    for (int j = tid; j < pieces; j += kOrthThreads) {  // this thread's own pieces
      float f[8];
      uint4* at = image(j);
      unpack(*at, f);
      put_scaled(reinterpret_cast<unsigned char*>(at), f);
    }
  }
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  tc05_fence_before();
  __syncthreads();
  tc05_fence_after();

  // ---- steps ----
  const uint32_t tmem = *slot, tlane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
  const int row = 32 * (warp & 3) + lane, quarter = warp >> 2;  // a thread's row of 128; it takes every fourth 32 columns
  const bool has_rows = 32 * (warp & 3) < Rows;                   // this warp's rows
  const int ksteps = (m + 15) / 16, units = (m + 31) / 32;       // of A and B: k in steps of 16, columns in 32s; the rest is zeros
  const uint32_t idesc_sq = wm_idesc(128, 16 * ksteps, false, false, false);
  uint32_t phase = 0;
  // All threads.  A warp whose wait gave up, which leaves its code, waits for nothing more and touches neither images nor accumulators, under
  // which MMAs may still be at work; it takes part in the barriers that are left.  Without its first warp a CTA issues no more MMAs.
  bool alive = true;
  auto wait_done = [&] {
    if (alive) alive = __all_sync(0xffffffffu, mbar_wait(done, phase & 1u, p.status, 24, p.spin_limit));
    ++phase;
    tc05_fence_after();
  };
  const int own_rows = (m + (int)C - 1) / (int)C;
  for (int step = 0; step < p.steps; ++step) {
    const bool first = step == 0, last = step + 1 == p.steps;
    const float4 coef = p.coef[step];
    const float ca = coef.x, cb = coef.y, cc = coef.z, shift = coef.w;
    // A's part
    if (tid == 0 && alive) {
      for (int q = 0; q < kProducts; ++q)
        for (int k = 0; k < nbox * 4; ++k) {
          const uint32_t at = smem_u32(ximg) + (k >> 2) * kBox + (k & 3) * 32;
          wm_mma<1>(tmem, wm_desc(at + (q == 1 ? xrest : 0), 16, 1024), wm_desc(at + (q == 2 ? xrest : 0), 16, 1024), idesc_sq, q > 0 || k > 0);
        }
      if (!(p.test_fault == 1 && blockIdx.x == 0 && first)) tc05_commit(done);
    }
    wait_done();
    const float alpha = first ? rest * rest : 1.f / (float)(1 << (2 * kOrthGuard));
    if (C == 1) {
      if (quarter < units && has_rows && alive) {
        float v[32];
        wm_ld32(tlane + 32 * quarter, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= alpha;
        if (shift != 0.f && (warp & 3) == quarter) {  // the diagonal
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (lane == i) v[i] -= shift;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) put8(aimg + box_at<Rows>(row, 32 * quarter + i), rest2, v + i);
      }
    } else {
      // Parts and rows of A are fetched from the CTAs that have them, whole lines by neighbouring lanes: written to their
      // readers instead, 16 bytes of a row per lane, the exchange took 12 000 cycles at eight CTAs.
      if (quarter < units && has_rows && alive) {  // over this CTA's B, which its own MMAs have read
        float v[32];
        wm_ld32(tlane + 32 * quarter, v);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(parts + row * 128 + 4 * (8 * quarter + ((i / 4 ^ row) & 7))) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
      cluster_sync();
      const int mine = min(own_rows, m - (int)rank * own_rows);  // rows that this CTA adds up; none or less: nothing to do
      for (int i = tid; i < mine * 8 * units && alive; i += kOrthThreads) {
        const int r = (int)rank * own_rows + i / (8 * units), piece = i % (8 * units);
        const uint32_t from = smem_u32(parts + r * 128 + 4 * ((piece & ~7) | ((piece ^ r) & 7)));
        float4 v[8], s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c)
          if (c < C) v[c] = ld_cluster16(map_rank(from, c));
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c)
          if (c < C) { s.x += v[c].x; s.y += v[c].y; s.z += v[c].z; s.w += v[c].w; }
        s = make_float4(alpha * s.x, alpha * s.y, alpha * s.z, alpha * s.w);
        const int diagonal = r - 4 * piece;
        if (diagonal == 0) s.x -= shift;
        if (diagonal == 1) s.y -= shift;
        if (diagonal == 2) s.z -= shift;
        if (diagonal == 3) s.w -= shift;
        const uint2 hi = make_uint2(wm_pack(s.x, s.y, false), wm_pack(s.z, s.w, false));
        *reinterpret_cast<uint2*>(aimg + box_at<Rows>(r, 4 * piece)) = hi;
        if constexpr (Terms) {
          const float2 a = wm_unpack(hi.x, false), b = wm_unpack(hi.y, false);
          *reinterpret_cast<uint2*>(aimg + rest2 + box_at<Rows>(r, 4 * piece)) =
              make_uint2(wm_pack(s.x - a.x, s.y - a.y, false), wm_pack(s.z - b.x, s.w - b.y, false));
        }
      }
      cluster_sync();
      for (int term = 0; term < T; ++term) {  // 16 bytes each, a box's rows one after the other; at most four per thread, all under way at once
        float4 v[4];
        unsigned char* at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = tid + u * kOrthThreads, box = i >= m * 8, j = i - box * m * 8, r = j >> 3, owner = r / own_rows;
          at[u] = alive && i < (units + 1) / 2 * m * 8 && owner != (int)rank ? aimg + term * rest2 + box * kBox + r * 128 + (j & 7) * 16 : nullptr;
          if (at[u]) v[u] = ld_cluster16(map_rank(smem_u32(at[u]), owner));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (at[u]) *reinterpret_cast<float4*>(at[u]) = v[u];
      }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    tc05_fence_before();
    __syncthreads();
    tc05_fence_after();
    // A A
    if (tid == 0 && alive) {
      for (int q = 0; q < kProducts; ++q)
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t at = smem_u32(aimg) + (k >> 2) * kBox + (k & 3) * 32;
          wm_mma<1>(tmem, wm_desc(at + (q == 1 ? rest2 : 0), 16, 1024), wm_desc(at + (q == 2 ? rest2 : 0), 16, 1024), idesc_sq, q > 0 || k > 0);
        }
      tc05_commit(done);
    }
    wait_done();
    if (quarter < units && has_rows && alive) {
      float v[32];
      wm_ld32(tlane + 32 * quarter, v);
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const int at = box_at<Rows>(row, 32 * quarter + i);
        float f[8];
        get8(aimg + at, rest2, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = fmaf(cc, v[i + k], cb * f[k]);
        put8(bimg + at, rest2, f);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    tc05_fence_before();
    __syncthreads();
    tc05_fence_after();
    // B X over 256 columns at a time
    if (tid == 0 && alive) {
      for (int b = 0; b < nbox; b += 4) {
        const int boxes = min(4, nbox - b);
        const uint32_t idesc = wm_idesc(128, 64 * boxes, false, false, true);
        for (int q = 0; q < kProducts; ++q)
          for (int k = 0; k < ksteps; ++k)
            wm_mma<1>(tmem + 64 * b, wm_desc(smem_u32(bimg) + (q == 1 ? rest2 : 0) + (k >> 2) * kBox + (k & 3) * 32, 16, 1024),
                      wm_desc(smem_u32(ximg) + (q == 2 ? xrest : 0) + b * kBox + k * 2048, kBox, 1024), idesc, q > 0 || k > 0);
      }
      tc05_commit(done);
    }
    wait_done();
    const float held = (first ? rest : 1.f / (float)(1 << kOrthGuard)) * (last ? 1.f : (float)(1 << kOrthGuard));
    const bool bf = last && p.out_bf16;
    for (int u = quarter; u < 2 * nbox && has_rows && alive; u += 4) {
      float v[32];
      wm_ld32(tlane + 32 * u, v);
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        unsigned char* at = ximg + box_at<Rows>(row, 32 * u + i);
        float f[8];
        get8(at, xrest, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = held * fmaf(ca, f[k], v[i + k]);
        put8(at, xrest, f, bf);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    tc05_fence_before();
    __syncthreads();
    tc05_fence_after();
  }

  // ---- the result, which the last step left as bits of the output's type ----
  uint16_t* out = static_cast<uint16_t*>(p.out) + z * p.out_batch + col0 * p.out_col;
  const bool by_rows = p.out_col != 1 && p.out_row == 1;
#pragma unroll 2
  for (int j = tid; j < pieces; j += kOrthThreads) {
    int r, c;
    place(by_rows, j, &r, &c);
    const uint4 v = *reinterpret_cast<const uint4*>(ximg + box_at<Rows>(r, c));
    uint16_t* to = out + r * p.out_row + c * p.out_col;
    if (p.out_vec) {
      *reinterpret_cast<uint4*>(to) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < n) to[k * p.out_col] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
  }
  if (tid == 0 && !alive) {  // what is under way must not outlive the memory it works on
    tc05_commit(drained);
    mbar_wait(drained, 0u, p.status, 24, p.spin_limit);
  }
  if (C > 1) cluster_sync();  // no CTA leaves while another may still read from it
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, p.tmem_cols);
}

}  // namespace tck

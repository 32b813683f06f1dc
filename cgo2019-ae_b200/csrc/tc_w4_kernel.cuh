// Persistent product of two matrices of microscaled 4-bit numbers on tcgen05 (kind::mxf4, fp32 accumulators in tensor memory).
//
//   out[n, m] = sum_k A[m, k] B[n, k]      A: 128 CG rows a tile (a layer's weights), B: BN rows (its tokens), k the fastest
//
// The tensor cores multiply e2m1 elements 64 k at a time and take both blocks' powers of two from tensor memory; products of two
// blocks are exact and are added up in fp32.
//
//   CG = 2   256 x 256 tiles on pairs of CTAs: each fetches 128 rows of A and 128 of B a stage, and the scales of its own rows of A
//            and of all of B's.
//   CG = 1   128 x BN tiles, one CTA each: BN down to 16, for few tokens.
//
//   warps 0-7   EPILOGUE  a thread has one m and half of the tile's n.  Neighbouring lanes hold neighbours of a row of the result, so
//                         stores need neither staging nor alignment.  A tile of 256 columns fills its accumulators' half of tensor
//                         memory: it is read into registers at once and free for the next tile before anything is stored.
//   warps 8, 10 LOADERS   one thread each: A and its scales, B and its scales.  Tiled TMA boxes of 256 k, 128 bytes with the 128-byte
//                         swizzle; of scales two pieces, 512 bytes for 128 rows of 128 k in the order tensor memory takes them.
//                         Behind the last row or k boxes are zeros, scales among them.
//   warp 9      MMA       one thread: per stage the scales to tensor memory (columns of the stage's own, so that nothing waits for
//                         the products that read them) and four MMAs.
//
// Where there are few tiles (CG = 1) a cluster of up to eight CTAs takes one, a slice of K each: the partial tiles go to shared memory,
// where the stages were, and each CTA adds up its share of them in order, through the cluster's shared memory.  Every wait is
// bounded and reports through args.status.
#pragma once
#include "tc_elem.cuh"
#include "tc_wm_kernel.cuh"

struct W4Args {
  TcTensorMap map_a, map_b, map_sa, map_sb;
  uint32_t M, N, K;
  uint32_t slices;        // CG = 1: of K, the cluster's CTAs
  void* out;
  int64_t ld_out;
  int* status;
  uint32_t spin_limit;
  int32_t test_fault, out_type, add;
};

namespace tck {

template <int CG_, int BN_>
struct W4Cfg {
  static constexpr int CG = CG_, BN = BN_, BM = 128 * CG, BROWS = BN / CG, BK = 256;  // k of a stage: 128 bytes
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BROWS * 128, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int B_PIECES = BN > 128 ? 2 : 1;                     // pieces of 128 rows of B's scales
  static constexpr int SCALE_BYTES = 1024 * (1 + B_PIECES);             // of a stage: two pieces of 128 k each
  static constexpr int STAGES = BN == 256 ? (CG == 2 ? 6 : 4) : BN == 128 ? 6 : BN == 64 ? 8 : 10;
  static constexpr int ACCS = BN == 256 ? 1 : 2;
  static constexpr int COLS = BN / 2;                                   // of an epilogue thread
  static constexpr int SCALE_COL = 256, STAGE_COLS = 8 * (1 + B_PIECES);
  static constexpr int THREADS = 352, EPI_WARPS = 8;
  static constexpr int NBARS = 2 * STAGES + 5;
  static constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + SCALE_BYTES) + NBARS * 8 + 16;
  static_assert(SMEM_BYTES <= 232448 && ACCS * BN <= SCALE_COL && SCALE_COL + STAGES * STAGE_COLS <= 512 && STAGE_BYTES % 1024 == 0, "tile");
};

// kind::mxf4: e2m1 by e2m1, scales ue8m0 of 32 k; `half`: which 64 k of a piece of 128 the scales are taken from.
__host__ __device__ constexpr uint32_t w4_idesc(int m, int n, int half) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)(2 * half) << 29) | ((uint32_t)(2 * half) << 4);
}
template <int CG>
__device__ __forceinline__ void w4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
}
// 512 bytes of scales to four columns of tensor memory: 32 rows of 16 bytes, to each of the four groups of 32 lanes.
template <int CG>
__device__ __forceinline__ void w4_scales(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = (uint64_t)((saddr >> 4) & 0x3FFF) | (8ull << 32) | (1ull << 46);  // no swizzle, 128 bytes from 8 rows to the next
  if constexpr (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
}
// Box at (c0, c1); its bytes count on `bar` of the pair's first CTA.
template <int CG>
__device__ __forceinline__ void w4_load(void* dst, const TcTensorMap* map, int c0, int c1, uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar) & 0xFEFFFFFFu)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
                 : "memory");
}
// One value of the result; `old`: where it is added to what is there.
template <class T>
__device__ __forceinline__ void w4_put(T* to, float v, bool add) { *to = Elem<T>::put(add ? Elem<T>::get(*to) + v : v); }

template <class F>
__device__ __forceinline__ void w4_typed(const W4Args& p, F put) {
  if (p.out_type == TC_F32) put(static_cast<float*>(p.out));
  else if (p.out_type == TC_BF16) put(static_cast<__nv_bfloat16*>(p.out));
  else put(static_cast<__half*>(p.out));
}
__device__ __forceinline__ float w4_of(uint32_t saddr, uint32_t rank) {  // of another CTA's shared memory
  float v;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}\n" : "=f"(v) : "r"(saddr), "r"(rank) : "memory");
  return v;
}

template <class CF>
__global__ void __launch_bounds__(CF::THREADS, 1) tc_w4_kernel(const __grid_constant__ W4Args p) {
  constexpr int CG = CF::CG, STAGES = CF::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* stages = smem_raw;
  unsigned char* scales = stages + STAGES * CF::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + STAGES * CF::SCALE_BYTES);  // [STAGES] (first CTA) what both CTAs fetched has landed
  uint64_t* empty = full + STAGES;         // [STAGES] the MMAs that read them have completed
  uint64_t* acc_full = empty + STAGES;     // [2] an accumulator holds a finished tile
  uint64_t* acc_free = acc_full + 2;       // [2] (first CTA) both CTAs' epilogues have read it
  uint64_t* drained = acc_free + 2;        // the MMAs of a role that gave up have completed
  uint32_t* slot = reinterpret_cast<uint32_t*>(full + CF::NBARS);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      tmem_alloc(slot, 512);
      tmem_relinquish();
    }
  }
  tc05_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc05_fence_after();
  const uint32_t tmem = *slot;
  chain_wait();

  const uint32_t M = p.M, N = p.N, K = p.K;
  const uint32_t tiles_m = (M + CF::BM - 1) / CF::BM, tiles_n = (N + CF::BN - 1) / CF::BN, tiles = tiles_m * tiles_n;
  const uint32_t kblocks = (K + CF::BK - 1) / CF::BK, per = CG == 2 ? 2u : p.slices;
  const uint32_t slice = CG == 2 || p.slices == 1 ? 0u : cluster_rank();
  const uint32_t kb0 = (uint32_t)((uint64_t)kblocks * slice / (CG == 2 ? 1u : p.slices)), kb1 = (uint32_t)((uint64_t)kblocks * (slice + 1) / (CG == 2 ? 1u : p.slices));
  const uint32_t first = blockIdx.x / per, step = gridDim.x / per, limit = p.spin_limit;
  struct Item { uint32_t tm, tn; };
  auto item_of = [&](uint32_t i) {  // 16 rows of tiles at a time, column by column: what runs together shares operands in L2
    const uint32_t group = 16u * tiles_n, q = i / group, rows = min(16u, tiles_m - 16u * q), l = i % group;
    return Item{16u * q + l % rows, l / rows};
  };

  if (warp < CF::EPI_WARPS) {
    uint32_t n = 0;
    for (uint32_t i = first; i < tiles; i += step, ++n) {
      const uint32_t acc = CF::ACCS == 2 ? n & 1u : 0u, use = CF::ACCS == 2 ? n >> 1 : n;
      const Item it = item_of(i);
      if (!mbar_wait(acc_full + acc, use & 1u, p.status, 30, limit)) break;
      tc05_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + acc * CF::BN + (warp >> 2) * CF::COLS;
      constexpr int kAtOnce = CF::COLS >= 16 ? CF::COLS : 8;
      float v[kAtOnce];
      if constexpr (CF::COLS >= 16) {
#pragma unroll
        for (int c = 0; c < CF::COLS; c += 16) tc05_ld16(taddr + c, v + c);
      } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "r"(taddr)
                     : "memory");
      }
      tc05_wait_ld();
      tc05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_first(acc_free + acc);
        else mbar_arrive(acc_free + acc);
      }
      const uint32_t in_tile = rank * 128 + 32 * (warp & 3) + lane, m = it.tm * CF::BM + in_tile, col = it.tn * CF::BN + (warp >> 2) * CF::COLS;
      if (CG == 1 && p.slices > 1) {
        float* to = reinterpret_cast<float*>(stages) + (warp >> 2) * CF::COLS * 128 + in_tile;  // no MMA reads a stage any more
#pragma unroll
        for (int c = 0; c < CF::COLS; ++c) to[c * 128] = v[c];
      } else if (m < M) {
        w4_typed(p, [&](auto* out) {
          out += m + (int64_t)col * p.ld_out;
#pragma unroll
          for (int c = 0; c < CF::COLS; ++c) {
            if (col + c < N) w4_put(out, v[c], p.add != 0);
            out += p.ld_out;
          }
        });
      }
    }
  } else if ((warp == 8 || warp == 10) && lane == 0) {
    const bool loads_a = warp == 8;
    uint32_t g = 0;
    bool alive = true;
    for (uint32_t i = first; alive && i < tiles; i += step) {
      const Item it = item_of(i);
      const int m0 = (int)(it.tm * CF::BM + rank * 128), n0 = (int)(it.tn * CF::BN);
      for (uint32_t kb = kb0; kb < kb1; ++kb, ++g) {
        const uint32_t s = g % STAGES;
        if (g >= (uint32_t)STAGES && !mbar_wait(empty + s, ((g / STAGES) - 1) & 1u, p.status, 31, limit)) { alive = false; break; }
        // tests only: one stage is left unannounced, so that the waits on it run out
        if (p.test_fault == 1 && blockIdx.x < CG && g == 1) continue;
        unsigned char* as = stages + s * CF::STAGE_BYTES;
        unsigned char* ss = scales + s * CF::SCALE_BYTES;
        const int k0 = (int)(kb * 128), p0 = (int)(kb * 256);  // bytes of codes, words of scales
        if (loads_a) {
          if (rank == 0) mbar_arrive_expect_tx(full + s, CG * (CF::STAGE_BYTES + CF::SCALE_BYTES));  // of both operands
          w4_load<CG>(as, &p.map_a, k0, m0, full + s);
          w4_load<CG>(ss, &p.map_sa, p0, m0 >> 7, full + s);
        } else {
          w4_load<CG>(as + CF::A_BYTES, &p.map_b, k0, n0 + (int)rank * CF::BROWS, full + s);
#pragma unroll
          for (int j = 0; j < CF::B_PIECES; ++j) w4_load<CG>(ss + 1024 * (1 + j), &p.map_sb, p0, (n0 >> 7) + j, full + s);
        }
      }
    }
    if (loads_a) chain_release();  // the next kernel may set itself up under the last tiles
    // A loader that gave up waits (with a limit) for what is under way; the first CTA's barriers count both CTAs'.
    if (!alive && rank == 0)
      for (uint32_t q = g > (uint32_t)STAGES ? g - STAGES : 0u; q < g; ++q)
        if (!(p.test_fault == 1 && blockIdx.x < CG && q == 1)) mbar_wait(full + q % STAGES, (q / STAGES) & 1u, p.status, 31, limit);
  } else if (warp == 9 && lane == 0 && rank == 0) {
    const uint32_t base = smem_u32(stages), sbase = smem_u32(scales);
    uint32_t g = 0, n = 0;
    bool alive = true;
    for (uint32_t i = first; alive && i < tiles; i += step, ++n) {
      const Item it = item_of(i);
      const uint32_t acc = CF::ACCS == 2 ? n & 1u : 0u, use = CF::ACCS == 2 ? n >> 1 : n, d = tmem + acc * CF::BN;
      if (use >= 1 && !mbar_wait_cluster(acc_free + acc, (use - 1) & 1u, p.status, 32, limit)) { alive = false; break; }
      tc05_fence_after();
      for (uint32_t kb = kb0; kb < kb1; ++kb, ++g) {
        const uint32_t s = g % STAGES;
        if (!mbar_wait_cluster(full + s, (g / STAGES) & 1u, p.status, 33, limit)) { alive = false; break; }
        tc05_fence_after();
        const uint32_t steps = min(4u, (K - kb * CF::BK + 63) / 64);  // of 64 k; what lies behind the last has no scales
        const uint32_t cols = tmem + CF::SCALE_COL + s * CF::STAGE_COLS, from = sbase + s * CF::SCALE_BYTES;
        const uint64_t a = wm_desc(base + s * CF::STAGE_BYTES, 16, 1024), b = wm_desc(base + s * CF::STAGE_BYTES + CF::A_BYTES, 16, 1024);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          if (2 * h >= steps) break;
          w4_scales<CG>(cols + 4 * h, from + 512 * h);
#pragma unroll
          for (uint32_t j = 0; j < (uint32_t)CF::B_PIECES; ++j) w4_scales<CG>(cols + 8 + 4 * (h * CF::B_PIECES + j), from + 1024 * (1 + j) + 512 * h);
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if (k >= steps) break;
          w4_mma<CG>(d, a + 2 * k, b + 2 * k, w4_idesc(CF::BM, CF::BN, k & 1), cols + 4 * (k >> 1), cols + 8 + 4 * CF::B_PIECES * (k >> 1), (kb > kb0 || k > 0) ? 1u : 0u);
        }
        wm_commit<CG>(empty + s);
      }
      if (alive) wm_commit<CG>(acc_full + acc);
    }
    if (!alive) {  // what is under way must not outlive the memory it works on
      wm_commit<CG>(drained);
      mbar_wait(drained, 0u, p.status, 33, limit);
    }
  }
  __syncwarp();
  tc05_fence_before();
  __syncthreads();
  if (CG == 1 && p.slices > 1) {
    cluster_sync();
    const Item it = item_of(first);
    const uint32_t m0 = it.tm * CF::BM, n0 = it.tn * CF::BN, cols = min((uint32_t)CF::BN, N - n0);
    w4_typed(p, [&](auto* out) {
      for (uint32_t at = slice * 256 + tid; tid < 256 && at < cols * 128; at += p.slices * 256) {
        float s = 0.f;
        for (uint32_t r = 0; r < p.slices; ++r) s += w4_of(smem_u32(stages) + at * 4, r);
        const uint32_t m = m0 + (at & 127);
        if (m < M) w4_put(out + m + (int64_t)(n0 + (at >> 7)) * p.ld_out, s, p.add != 0);
      }
    });
  }
  if (CG == 2 || p.slices > 1) cluster_sync();  // no CTA leaves while another still reads its memory
  tc05_fence_after();
  if (warp == 9) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    else tmem_dealloc(tmem, 512);
  }
}

}  // namespace tck

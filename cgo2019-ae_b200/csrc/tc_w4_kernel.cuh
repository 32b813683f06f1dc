// Persistent product of two matrices of microscaled 4-bit numbers on tcgen05 (kind::mxf4, fp32 accumulators in tensor memory).
//
//   out[n, m] = sum_k A[m, k] B[n, k]      A: 128 rows a tile (a layer's weights), B: BN rows (its tokens), k the fastest
//
// The tensor cores multiply e2m1 elements 64 k at a time and take both blocks' powers of two from tensor memory; products of two
// blocks are exact and are added up in fp32.  128 x BN tiles, one CTA each, BN from 256 down to 16 for few tokens.
//
//   warps 0-7    EPILOGUE  a thread has one m and half of the tile's n.  Neighbouring lanes hold neighbours of a row of the result, so
//                          stores need neither staging nor alignment.  A tile of 256 columns fills its accumulators' half of tensor
//                          memory: it is read into registers at once and free for the next tile before anything is stored.  Whole
//                          tiles are stored without a condition on each value (2048 x 2048 x 2048 12.7 -> 8.3 us).
//   warps 8, 10, 11  LOADERS   A, B, both scales.  Tiled TMA boxes of 256 k, 128 bytes with the 128-byte swizzle; of
//                          scales two pieces, 512 bytes for 128 rows of 128 k.  Behind the last row or k boxes are zeros, scales among them.
//   warp 9       MMA       four a stage.  Like the loaders the warp goes through its loop together and one lane issues, so that what the
//                          instructions take is worked out once for the warp, in the registers they take it from.
//   warps 12-15  SCALES    from shared to tensor memory, a copy for each of its four groups of lanes, to columns of the stage's own:
//                          nothing waits for the products that read them.  By tcgen05.cp the same copies stand in line with the
//                          products: 8192 x 8192 x 4096 139 us, so 131.
//
// One B200: 8192 x 8192 x 4096 115 us (4.8 PFLOP/s) in short runs, 133 in long ones under the board's power cap (1.49 GHz); with zeros for
// operands, which take less power, 100.  Of that the MMAs alone take 70, the loads alone 82, and both, which share the ports of shared memory,
// more than either; the rest is a tile's accumulators being read out.  4096 x 4096 x 4096 30.6 us, 1 x 4096 x 4096 5.6 (a launch 2.5).
//
// Where there are few tiles a cluster of up to eight CTAs takes one, a slice of K each: the partial tiles go to shared memory, where the
// stages were, and each CTA adds up its share of them in order, through the cluster's shared memory.  Every wait is bounded and
// reports through args.status.
#pragma once
#include "tc_elem.cuh"
#include "tc_wm_kernel.cuh"

struct W4Args {
  TcTensorMap map_a, map_b, map_sa, map_sb;
  uint32_t M, N, K;
  uint32_t slices;        // of K, the cluster's CTAs
  void* out;
  int64_t ld_out;
  int* status;
  uint32_t spin_limit;
  int32_t test_fault, out_type, add;
};

namespace tck {

template <int BN_>
struct W4Cfg {
  static constexpr int BN = BN_, BM = 128, BK = 256;                    // k of a stage: 128 bytes
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int B_PIECES = BN > 128 ? 2 : 1;                     // pieces of 128 rows of B's scales
  static constexpr int SCALE_BYTES = 1024 * (1 + B_PIECES);             // of a stage: two pieces of 128 k each
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : BN == 64 ? 8 : 10;
  static constexpr int ACCS = BN == 256 ? 1 : 2;
  static constexpr int COLS = BN / 2;                                   // of an epilogue thread
  static constexpr int SCALE_COL = 256, STAGE_COLS = 8 * (1 + B_PIECES);
  static constexpr int THREADS = 512, EPI_WARPS = 8, SCALE_WARPS = 4;
  static constexpr int NBARS = 4 * STAGES + 5;
  static constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + SCALE_BYTES) + NBARS * 8 + 16;
  static_assert(SMEM_BYTES <= 232448 && ACCS * BN <= SCALE_COL && SCALE_COL + STAGES * STAGE_COLS <= 512 && STAGE_BYTES % 1024 == 0, "tile");
  // 512 threads start with 128 registers; what the epilogue gains the other two warpgroups give up (checked against the built kernel before it
  // runs: with fewer the epilogue would wait for ever).
  static constexpr int LAUNCH_REGS = 128, EPILOGUE_REGS = 168, OTHER_REGS = 80;
  static_assert(256 * EPILOGUE_REGS + 256 * OTHER_REGS <= THREADS * LAUNCH_REGS, "register split");
};

// kind::mxf4: e2m1 by e2m1, scales ue8m0 of 32 k; `half`: which 64 k of a piece of 128 the scales are taken from.
__host__ __device__ constexpr uint32_t w4_idesc(int m, int n, int half) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)(2 * half) << 29) | ((uint32_t)(2 * half) << 4);
}
__device__ __forceinline__ void w4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
      : "memory");
}
// Two pieces of scales, 512 bytes each, to eight columns: row 32 j + i has its four bytes at byte 16 i + 4 j, so that a lane's 16 bytes are
// four columns.
__device__ __forceinline__ void w4_scales(uint32_t taddr, const unsigned char* p0, const unsigned char* p1, int lane) {
  const uint4 a = reinterpret_cast<const uint4*>(p0)[lane], b = reinterpret_cast<const uint4*>(p1)[lane];
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
               "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// Whether a phase has completed, without a wait.
__device__ __forceinline__ bool w4_landed(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

// One value of the result; `add`: onto what is there.
template <class T>
__device__ __forceinline__ void w4_put(T* to, float v, bool add) { *to = Elem<T>::put(add ? Elem<T>::get(*to) + v : v); }

template <class F>
__device__ __forceinline__ void w4_typed(const W4Args& p, F put) {
  if (p.out_type == TC_F32) put(static_cast<float*>(p.out));
  else if (p.out_type == TC_BF16) put(static_cast<__nv_bfloat16*>(p.out));
  else put(static_cast<__half*>(p.out));
}
__device__ __forceinline__ float4 w4_of(uint32_t saddr, uint32_t rank) {  // of another CTA's shared memory
  float4 v;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}\n"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(saddr), "r"(rank)
               : "memory");
  return v;
}

template <class CF>
__global__ void __launch_bounds__(CF::THREADS, 1) tc_w4_kernel(const __grid_constant__ W4Args p) {
  constexpr int STAGES = CF::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* stages = smem_raw;
  unsigned char* scales = stages + STAGES * CF::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + STAGES * CF::SCALE_BYTES);  // [STAGES] the operands' boxes have landed
  uint64_t* fetched = full + STAGES;       // [STAGES] the scales' boxes have
  uint64_t* scaled = fetched + STAGES;     // [STAGES] the scales are in tensor memory
  uint64_t* empty = scaled + STAGES;       // [STAGES] the MMAs that read all that have completed
  uint64_t* acc_full = empty + STAGES;     // [2] an accumulator holds a finished tile
  uint64_t* acc_free = acc_full + 2;       // [2] the epilogue has read it
  uint64_t* drained = acc_free + 2;        // the MMAs of a role that gave up have completed
  uint32_t* slot = reinterpret_cast<uint32_t*>(full + CF::NBARS);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // the same for the whole warp, and known to be
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(fetched + s, 1); mbar_init(scaled + s, CF::SCALE_WARPS); mbar_init(empty + s, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_free + i, CF::EPI_WARPS); }
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&p.map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&p.map_b)) : "memory");
  }
  if (warp == 9) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
  tc05_fence_before();
  __syncthreads();
  tc05_fence_after();
  const uint32_t tmem = *slot;
  chain_wait();

  const uint32_t M = p.M, N = p.N, K = p.K;
  const uint32_t tiles_m = (M + CF::BM - 1) / CF::BM, tiles_n = (N + CF::BN - 1) / CF::BN, tiles = tiles_m * tiles_n;
  const uint32_t kblocks = (K + CF::BK - 1) / CF::BK, slices = p.slices, slice = slices == 1 ? 0u : cluster_rank();
  const uint32_t kb0 = (uint32_t)((uint64_t)kblocks * slice / slices), kb1 = (uint32_t)((uint64_t)kblocks * (slice + 1) / slices);
  const uint32_t first = blockIdx.x / slices, step = gridDim.x / slices, limit = p.spin_limit;
  struct Item { uint32_t tm, tn; };
  auto item_of = [&](uint32_t i) {  // 16 rows of tiles at a time, column by column: what runs together shares operands in L2
    const uint32_t group = 16u * tiles_n, q = i / group, rows = min(16u, tiles_m - 16u * q), l = i % group;
    return Item{16u * q + l % rows, l / rows};
  };

  if (warp < CF::EPI_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(CF::EPILOGUE_REGS));
    uint32_t n = 0;
    for (uint32_t i = first; i < tiles; i += step, ++n) {
      const uint32_t acc = CF::ACCS == 2 ? n & 1u : 0u, use = CF::ACCS == 2 ? n >> 1 : n;
      const Item it = item_of(i);
      if (!mbar_wait_warp(acc_full + acc, use & 1u, p.status, 30, limit)) break;
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
      if (lane == 0) mbar_arrive(acc_free + acc);
      const uint32_t in_tile = 32 * (warp & 3) + lane, m = it.tm * CF::BM + in_tile, col = it.tn * CF::BN + (warp >> 2) * CF::COLS;
      if (slices > 1) {
        float* to = reinterpret_cast<float*>(stages) + (warp >> 2) * CF::COLS * 128 + in_tile;  // no MMA reads a stage any more
#pragma unroll
        for (int c = 0; c < CF::COLS; ++c) to[c * 128] = v[c];
      } else if (m < M) {
        w4_typed(p, [&](auto* out) {
          out += m + (int64_t)col * p.ld_out;
          if (!p.add && col + CF::COLS <= N) {
#pragma unroll
            for (int c = 0; c < CF::COLS; ++c) {
              w4_put(out, v[c], false);
              out += p.ld_out;
            }
          } else {
#pragma unroll
            for (int c = 0; c < CF::COLS; ++c) {
              if (col + c < N) w4_put(out, v[c], p.add != 0);
              out += p.ld_out;
            }
          }
        });
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(CF::OTHER_REGS));
    if (warp != 9 && warp < 12) {
      const bool loads_a = warp == 8, loads_scales = warp == 11, issues = wm_elect();
      uint32_t g = 0;
      bool alive = true;
      for (uint32_t i = first; alive && i < tiles; i += step) {
        const Item it = item_of(i);
        const int m0 = (int)(it.tm * CF::BM), n0 = (int)(it.tn * CF::BN);
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++g) {
          const uint32_t s = g % STAGES;
          if (g >= (uint32_t)STAGES && !mbar_wait_warp(empty + s, ((g / STAGES) - 1) & 1u, p.status, 31, limit)) { alive = false; break; }
          // tests only: one stage is left unannounced, so that the waits on it run out
          if (p.test_fault == 1 && blockIdx.x == 0 && g == 1) continue;
          unsigned char* as = stages + s * CF::STAGE_BYTES;
          unsigned char* ss = scales + s * CF::SCALE_BYTES;
          const int k0 = (int)(kb * 128), p0 = (int)(kb * 256);  // bytes of codes, words of scales
          if (issues) {
            if (loads_a) {
              mbar_arrive_expect_tx(full + s, CF::STAGE_BYTES);  // of both operands
              tma_load_2d(as, &p.map_a, k0, m0, full + s);
            } else if (loads_scales) {
              mbar_arrive_expect_tx(fetched + s, CF::SCALE_BYTES);
              tma_load_2d(ss, &p.map_sa, p0, m0 >> 7, fetched + s);
              tma_load_2d(ss + 1024, &p.map_sb, p0, n0 >> 7, fetched + s);
            } else {
              tma_load_2d(as + CF::A_BYTES, &p.map_b, k0, n0, full + s);
            }
          }
          __syncwarp();
        }
      }
      if (loads_a) chain_release();  // the next kernel may set itself up under the last tiles
      // A loader that gave up waits (with a limit) for what is under way.
      if (!alive)
        for (uint32_t q = g > (uint32_t)STAGES ? g - STAGES : 0u; q < g; ++q)
          if (!(p.test_fault == 1 && blockIdx.x == 0 && q == 1)) mbar_wait_warp((loads_scales ? fetched : full) + q % STAGES, (q / STAGES) & 1u, p.status, 31, limit);
    } else if (warp == 9) {
      // One lane by itself, which has to move every operand of an MMA into the warp's registers: 8192 x 8192 x 4096 131 us, so 116; 512 x 4096 x
      // 4096 11.3 and 8.6.
      const bool issues = wm_elect();
      const uint32_t base = smem_u32(stages);
      uint32_t g = 0, n = 0;
      bool alive = true;
      for (uint32_t i = first; alive && i < tiles; i += step, ++n) {
        const uint32_t acc = CF::ACCS == 2 ? n & 1u : 0u, use = CF::ACCS == 2 ? n >> 1 : n, d = tmem + acc * CF::BN;
        if (use >= 1 && !mbar_wait_warp(acc_free + acc, (use - 1) & 1u, p.status, 32, limit)) { alive = false; break; }
        tc05_fence_after();
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++g) {
          const uint32_t s = g % STAGES;
          if (!mbar_wait_warp(scaled + s, (g / STAGES) & 1u, p.status, 33, limit) || !mbar_wait_warp(full + s, (g / STAGES) & 1u, p.status, 34, limit)) { alive = false; break; }
          tc05_fence_after();
          const uint32_t left = K - kb * CF::BK, cols = tmem + CF::SCALE_COL + s * CF::STAGE_COLS;
          const uint64_t a = wm_desc(base + s * CF::STAGE_BYTES, 16, 1024), b = wm_desc(base + s * CF::STAGE_BYTES + CF::A_BYTES, 16, 1024);
          if (issues) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
              if (k == 0 || left > 64 * k)  // of 64 k; what lies behind the last is zeros
                w4_mma(d, a + 2 * k, b + 2 * k, w4_idesc(CF::BM, CF::BN, k & 1), cols + 4 * (k >> 1), cols + 8 + 4 * CF::B_PIECES * (k >> 1), (kb > kb0 || k > 0) ? 1u : 0u);
            tc05_commit(empty + s);
          }
          __syncwarp();
        }
        if (alive && issues) tc05_commit(acc_full + acc);
        __syncwarp();
      }
      if (!alive) {  // what is under way must not outlive the memory it works on
        if (issues) tc05_commit(drained);
        __syncwarp();
        mbar_wait_warp(drained, 0u, p.status, 33, limit);
      }
    } else if (warp >= 12) {
      const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + CF::SCALE_COL, items = first < tiles ? (tiles - first + step - 1) / step : 0u;
      const uint32_t all = items * (kb1 - kb0);
      // Stages that have landed meanwhile go together: a stage by itself takes about 600 cycles, most of them waits.
      for (uint32_t g = 0; g < all;) {
        // landed: the products that read these columns before have completed
        if (!mbar_wait_warp(fetched + g % STAGES, (g / STAGES) & 1u, p.status, 35, limit)) break;
        tc05_fence_after();
        uint32_t n = 0;
        do {
          const uint32_t s = (g + n) % STAGES, cols = lanes + s * CF::STAGE_COLS;
          const unsigned char* from = scales + s * CF::SCALE_BYTES;
          w4_scales(cols, from, from + 512, lane);
          if constexpr (CF::B_PIECES == 2) {  // columns by k first, then by piece of rows
            w4_scales(cols + 8, from + 1024, from + 2048, lane);
            w4_scales(cols + 16, from + 1536, from + 2560, lane);
          } else {
            w4_scales(cols + 8, from + 1024, from + 1536, lane);
          }
          ++n;
        } while (n < (uint32_t)STAGES && g + n < all && __all_sync(0xffffffffu, w4_landed(fetched + (g + n) % STAGES, ((g + n) / STAGES) & 1u)));
        tc05_wait_st();
        tc05_fence_before();
        __syncwarp();
        if (lane == 0)
          for (uint32_t i = 0; i < n; ++i) mbar_arrive(scaled + (g + i) % STAGES);
        g += n;
      }
    }
  }
  __syncwarp();
  tc05_fence_before();
  __syncthreads();
  tc05_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
  if (slices > 1) {
    cluster_sync();
    const Item it = item_of(first);
    const uint32_t m0 = it.tm * CF::BM, n0 = it.tn * CF::BN, end = min((uint32_t)CF::BN, N - n0) * 128, from = smem_u32(stages);
    w4_typed(p, [&](auto* out) {
      // four m of a column at a time; every part of them under way before the first is added
      constexpr int kAtOnce = CF::BN >= 64 ? 2 : 1;
      for (uint32_t at = slice * CF::THREADS + tid; at < end / 4; at += kAtOnce * slices * CF::THREADS) {
        float4 v[kAtOnce][8];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
          for (uint32_t r = 0; r < 8; ++r) {
            const uint32_t e = at + j * slices * CF::THREADS;
            v[j][r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < slices && e < end / 4) v[j][r] = w4_of(from + e * 16, r);
          }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const uint32_t e = at + j * slices * CF::THREADS, m = m0 + (e & 31) * 4;
          float4 s = v[j][0];
#pragma unroll
          for (int r = 1; r < 8; ++r) s = make_float4(s.x + v[j][r].x, s.y + v[j][r].y, s.z + v[j][r].z, s.w + v[j][r].w);
          if (e < end / 4) {
            auto* to = out + m + (int64_t)(n0 + (e >> 5)) * p.ld_out;
            if (m < M) w4_put(to, s.x, p.add != 0);
            if (m + 1 < M) w4_put(to + 1, s.y, p.add != 0);
            if (m + 2 < M) w4_put(to + 2, s.z, p.add != 0);
            if (m + 3 < M) w4_put(to + 3, s.w, p.add != 0);
          }
        }
      }
    });
    cluster_sync();  // no CTA leaves while another still reads its memory
  }
}

}  // namespace tck

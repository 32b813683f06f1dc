// Launches of the 16-bit matrix products (tc_wm_kernel.cuh).
#include "tc_wm.h"

#include <algorithm>
#include <cmath>

#include "tc_inst.cuh"
#include "tc_tensor_map.h"
#include "tc_wm_kernel.cuh"

namespace {

// [z][rows][cols] of es-byte elements, box box_c x box_r, of one z.
bool encode(TcTensorMap* out, const void* ptr, int64_t cols, int64_t rows, int64_t pitch, int64_t z, int64_t z_stride, uint32_t box_c, uint32_t box_r, int es,
            bool bf, CUtensorMapSwizzle swizzle) {
  const tc_encode_fn fn = tc_tensor_map_encoder();
  if (!fn || z > INT32_MAX || cols > INT32_MAX || rows > INT32_MAX) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)z};
  const cuuint64_t strides[2] = {(cuuint64_t)(pitch * es), (cuuint64_t)(z > 1 ? z_stride * es : pitch * es)};  // one matrix: any aligned stride
  const cuuint32_t box[3] = {box_c, box_r, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type = es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(reinterpret_cast<CUtensorMap*>(out), type, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BK> using Pair = tck::WmCfg<2, 256, BK>;
template <int BK> using Single = tck::WmCfg<1, 128, BK>;
typedef void (*Kernel)(WmArgs);
struct Built {
  Kernel kernel;
  int threads, smem;
};
template <class CF, class EPI>
Built built() { return Built{tck::tc_wm_kernel<CF, EPI>, CF::THREADS, CF::SMEM_BYTES}; }

template <int BK>
Built kernel_of(WmKind kind, bool pair, bool terms = false) {
  if (terms) {
    if (kind == WM_SYMMETRIC) return pair ? built<Pair<BK>, tck::WmAffine<true, false, true>>() : built<Single<BK>, tck::WmAffine<true, false, true>>();
    return pair ? built<Pair<BK>, tck::WmAffine<false, true, true>>() : built<Single<BK>, tck::WmAffine<false, true, true>>();
  }
  switch (kind) {
    case WM_STATS: return pair ? built<Pair<BK>, tck::WmStats>() : built<Single<BK>, tck::WmStats>();
    case WM_PROB: return pair ? built<Pair<BK>, tck::WmProb>() : built<Single<BK>, tck::WmProb>();
    case WM_GRADS: return pair ? built<Pair<BK>, tck::WmGrads>() : built<Single<BK>, tck::WmGrads>();
    case WM_SYMMETRIC: return pair ? built<Pair<BK>, tck::WmAffine<true, false, false>>() : built<Single<BK>, tck::WmAffine<true, false, false>>();
    case WM_UPDATE: return pair ? built<Pair<BK>, tck::WmAffine<false, true, false>>() : built<Single<BK>, tck::WmAffine<false, true, false>>();
    case WM_WEIGHT: return pair ? built<Pair<BK>, tck::WmWeight>() : built<Single<BK>, tck::WmWeight>();
  }
  return Built{nullptr, 0, 0};
}
// k of a stage.  128, half the waits and commits: a vocabulary of 131072 for 8192 tokens 15.5 -> 12.8 ms, four 1024 x 4096
// orthogonalised 416 -> 368 us, K = 768 of 50001 columns 64 -> 60.  64 where a last stage of 128 would be mostly empty (K = 72 of
// 36385 columns 14.0 us against 16.4, K = 777 of 50001 89.6 against 91.0).
// Single CTAs: from 1024 on, since three stages of 128 leave the SM no room for the kernel behind (36385 columns of K = 72 15.0 us
// against 17.5 with six stages of 64).
int stage_k(int64_t K, bool pair) { return (K + 127) / 128 * 128 - K <= K / 32 && (pair || K >= 1024) ? 128 : 64; }
// Two products: also 64 for fewer than 2048 tokens, k of the second.  Loss and gradients, us with 64 and by the rule above: 1023 tokens, 50001 rows
// of 768 346, 354; 32768 rows of 1024 with 512 tokens 164, 163, with 1280 345, 338, with 1792 450, 442, with 2048 494, 480, with 2560 647, 622;
// of 512 with 1792 276, 275, with 4096 550, 551.  What 1280 to 2047 tokens lose by it is 2 %.
int stage_k(int64_t K, int64_t K2, bool pair) { return K2 >= 2048 ? stage_k(K, pair) : 64; }

int64_t tiles_of(WmKind kind, int64_t M, int64_t N, int tile) {
  const int64_t tm = (M + wm_tile_m(tile) - 1) / wm_tile_m(tile), tn = (N + wm_tile_n(tile) - 1) / wm_tile_n(tile);
  return kind == WM_SYMMETRIC ? tn * (tn + 1) / 2 : tm * tn;
}

}  // namespace

void wm_choose(WmKind kind, int64_t M, int64_t N, int64_t K, int64_t batch, int slices_most, int sms, int* tile, int* slices) {
  const int64_t kblocks = std::max<int64_t>(1, (K + 63) / 64);
  double best = 0;
  *tile = WM_PAIR_256;
  *slices = 1;
  for (int t = 0; t < WM_TILES; ++t) {
    const int64_t workers = std::max(1, t == WM_PAIR_256 ? sms / 2 : sms), tiles = std::max<int64_t>(1, tiles_of(kind, M, N, t)) * batch;
    // cycles of 64 k of a tile, and of what an item costs besides
    const double block = t == WM_PAIR_256 ? 540 : 400, item = t == WM_PAIR_256 ? 900 : 600;
    for (int s = 1; s <= slices_most && s <= kblocks; ++s) {
      const int64_t rounds = (tiles * s + workers - 1) / workers;
      const double cost = rounds * (block * ((kblocks + s - 1) / s) + item) + 2500 + 300.0 * (s - 1);
      if (best == 0 || cost < best) {
        best = cost;
        *tile = t;
        *slices = s;
      }
    }
  }
}

void wm_choose_grads(int64_t M, int64_t N, int64_t K, int64_t M2, int64_t N2, int64_t K2, int slices_most, int sms, int* tile, int* slices) {
  const int64_t k1 = std::max<int64_t>(1, (K + 63) / 64), k2 = std::max<int64_t>(1, (K2 + 63) / 64);
  double best = 0;
  for (int t = 0; t < WM_TILES; ++t) {
    const double workers = std::max(1, t == WM_PAIR_256 ? sms / 2 : sms), block = t == WM_PAIR_256 ? 540 : 400, item = t == WM_PAIR_256 ? 900 : 600;
    const double n1 = (double)(M > 0 ? tiles_of(WM_GRADS, M, N, t) : 0), n2 = (double)(M2 > 0 ? tiles_of(WM_GRADS, M2, N2, t) : 0);
    for (int s = 1; s <= slices_most && s <= k1; ++s) {
      // long items first, the others fill up what they leave: all items' share of a worker, or the longest of a round
      const double c1 = block * ((k1 + s - 1) / s) + item, c2 = block * k2 + item, share = (n1 * s * c1 + n2 * c2) / workers;
      const double rounds1 = std::ceil(n1 * s / workers) * c1;
      const double cost = std::max(rounds1, share + 0.5 * (n2 > 0 ? c2 : c1)) + 2500 + 300.0 * (s - 1);
      if (best == 0 || cost < best) {
        best = cost;
        *tile = t;
        *slices = s;
      }
    }
  }
}

int wm_prepare(WmKind kind) {
  for (bool pair : {false, true})
    for (bool terms : {false, kind == WM_SYMMETRIC || kind == WM_UPDATE})
      for (const Built& k : {kernel_of<64>(kind, pair, terms), kernel_of<128>(kind, pair, terms)})
        TC_CUDA_OK(cudaFuncSetAttribute(k.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem));
  return TC_OK;
}

namespace {
int launch(WmKind kind, int tile, int bk, const WmArgs& p, int64_t items, int sms, cudaStream_t stream) {
  if (items <= 0) return TC_OK;
  if (items > UINT32_MAX / 2) return TC_ERR_UNSUPPORTED;
  const bool pair = tile == WM_PAIR_256;
  const int workers = std::max(1, pair ? sms / 2 : sms);
  const unsigned grid = (unsigned)std::min<int64_t>(items, workers) * (pair ? 2 : 1);
  const Built k = bk == 128 ? kernel_of<128>(kind, pair, p.terms > 0) : kernel_of<64>(kind, pair, p.terms > 0);
  TC_CUDA_OK(tck::launch_chained(true, k.kernel, dim3(grid), (unsigned)k.threads, (size_t)k.smem, stream, p));
  return TC_OK;
}
}  // namespace

int wm_launch(WmKind kind, int tile, WmArgs& p, const WmOperand& a, const WmOperand& b, int sms, cudaStream_t stream) {
  const int64_t M = p.M, N = p.N, K = p.K;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const bool bf = p.bf16 != 0;
  const int bk = stage_k(K, tile == WM_PAIR_256);
  // a slice without a stage would store what its accumulator happened to hold
  if (kind == WM_WEIGHT && p.slices > (uint64_t)((K + bk - 1) / bk * p.weight.terms)) return TC_ERR_UNSUPPORTED;
  const int64_t planes = (int64_t)p.batch * (p.terms ? 2 : 1), out_planes = (int64_t)p.batch * (p.out.planes == 2 ? 2 : 1);
  bool ok = kind == WM_WEIGHT ? encode(&p.map_a, a.ptr, M, K, a.pitch, p.weight.terms, a.batch_stride, 64, bk, 2, bf, sw)
                              : encode(&p.map_a, a.ptr, K, M, a.pitch, planes, a.batch_stride, 64, 128, 2, bf, sw);
  ok = ok && (kind == WM_UPDATE || kind == WM_WEIGHT ? encode(&p.map_b, b.ptr, N, K, b.pitch, planes, b.batch_stride, 64, bk, 2, bf, sw)
                                : encode(&p.map_b, b.ptr, K, N, b.pitch, planes, b.batch_stride, 64, 128, 2, bf, sw));
  if (kind != WM_STATS && kind != WM_WEIGHT && p.out.boxes) {
    const int64_t rows = kind == WM_PROB ? (int64_t)p.prob.rows_most : M;
    ok = ok && encode(&p.map_d, p.out.ptr, N, rows, p.out.row_stride, out_planes, p.out.batch_stride, 64, 32, 2, p.out.bf16 != 0, sw);
    if (kind == WM_SYMMETRIC)
      ok = ok && encode(&p.map_t, p.out.ptr, N, rows, p.out.row_stride, out_planes, p.out.batch_stride, 32, 64, 2, p.out.bf16 != 0, CU_TENSOR_MAP_SWIZZLE_NONE);
  }
  if (!ok) return TC_ERR_UNSUPPORTED;
  return launch(kind, tile, bk, p, tiles_of(kind, M, N, tile) * p.batch * p.slices, sms, stream);
}

int wm_weight_stage(int64_t K, int tile) { return stage_k(K, tile == WM_PAIR_256); }

int wm_grads_stage(int64_t K, int64_t K2, int tile) { return stage_k(K, K2, tile == WM_PAIR_256); }

int wm_launch_grads(int tile, WmArgs& p, const WmOperand& a, const WmOperand& b, float* slab, int64_t slab_rows, const WmOperand& a2, const WmOperand& b2, int sms,
                    cudaStream_t stream) {
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const bool bf = p.bf16 != 0;
  WmSecond& q = p.second;
  const int bk = wm_grads_stage(p.K, q.K, tile);
  const int64_t pitch = ((int64_t)p.N + 3) / 4 * 4;
  bool ok = true;
  if (p.M) {
    ok = ok && encode(&p.map_a, a.ptr, p.K, p.M, a.pitch, 1, 0, 64, 128, 2, bf, sw) && encode(&p.map_b, b.ptr, p.N, p.K, b.pitch, 1, 0, 64, bk, 2, bf, sw);
    ok = ok && encode(&p.map_d, slab, p.N, slab_rows, pitch, p.slices, slab_rows * pitch, 32, 32, 4, false, sw);
  }
  if (q.M) {
    ok = ok && encode(&q.map_a, a2.ptr, q.M, q.K, a2.pitch, 1, 0, 64, bk, 2, bf, sw) && encode(&q.map_b, b2.ptr, q.N, q.K, b2.pitch, 1, 0, 64, bk, 2, bf, sw);
    if (p.out.boxes) ok = ok && encode(&q.map_d, p.out.ptr, q.N, q.M, p.out.row_stride, 1, 0, 64, 32, 2, p.out.bf16 != 0, sw);
  }
  if (!ok) return TC_ERR_UNSUPPORTED;
  return launch(WM_GRADS, tile, bk, p, (p.M ? tiles_of(WM_GRADS, p.M, p.N, tile) * p.slices : 0) + (q.M ? tiles_of(WM_GRADS, q.M, q.N, tile) : 0), sms, stream);
}

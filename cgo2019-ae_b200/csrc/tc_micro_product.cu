// Products of matrices of microscaled 4-bit numbers (tc_micro_product_execute): tile, slices and launch of tc_w4_kernel.cuh.
#include <algorithm>

#include "tc_elem.cuh"
#include "tc_inst.cuh"
#include "tc_op.h"
#include "tc_tensor_map.h"
#include "tc_w4_kernel.cuh"

namespace {
using namespace tck;

enum Tile { k256, k128, k64, k32, k16, kTiles };
struct Built {
  void (*kernel)(W4Args);
  int bn, threads, smem;
};
template <int BN>
Built built() {
  using CF = W4Cfg<BN>;
  return Built{tc_w4_kernel<CF>, CF::BN, CF::THREADS, CF::SMEM_BYTES};
}
Built of(int tile) {
  switch (tile) {
    case k256: return built<256>();
    case k128: return built<128>();
    case k64: return built<64>();
    case k32: return built<32>();
    default: return built<16>();
  }
}
constexpr int kMostSlices = 8;  // CTAs of a cluster

struct Choice {
  int tile, slices;
};
// The least time by a model: rounds of tiles, each its stages of 256 k and what a tile costs besides; a cluster's sum over its slices.  The
// constants are times on one B200 (us): a stage .27 to .35, a tile of 16 columns .3 and of 256 1.5, a cluster 1.3 and 4.  By it 1 x 4096 x
// 4096 takes four slices (5.6; one 7.0, two 6.0), 512 x 4096 x 4096 128 columns (8.1; 256 9.7), 2048 x 2048 x 2048 256 (7.2; 128 8.4), 64 x
// 1000 x 1000 one slice (4.2; two 5.8).
Choice choose(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t kblocks = (K + 255) / 256;
  Choice best{k16, 1};
  double least = 0;
  for (int t = 0; t < kTiles; ++t) {
    const int bn = of(t).bn;
    if (bn < 128 && N > bn) continue;  // a tile's scales start with a piece of 128 rows
    const int64_t tiles = ((M + 127) / 128) * ((N + bn - 1) / bn);
    const double stage = 0.265 + 0.00032 * bn, item = 0.25 + 0.0048 * bn, cluster = 1.0 + 0.024 * bn;
    for (int s = 1; s <= kMostSlices && s <= kblocks; ++s) {
      if (s > 1 && tiles * s > sms) break;
      const double cost = (double)((tiles * s + sms - 1) / sms) * (stage * ((kblocks + s - 1) / s) + item) + (s > 1 ? cluster : 0);
      if (least == 0 || cost < least) {
        least = cost;
        best = Choice{t, s};
      }
    }
  }
  return best;
}

bool encode(TcTensorMap* out, const void* ptr, CUtensorMapDataType type, int64_t cols, int64_t rows, int64_t pitch_bytes, uint32_t box_c, uint32_t box_r, CUtensorMapSwizzle swizzle) {
  const tc_encode_fn fn = tc_tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch_bytes};
  const cuuint32_t box[2] = {box_c, box_r}, estr[2] = {1, 1};
  return fn(reinterpret_cast<CUtensorMap*>(out), type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int multiply(const tc_op_plan& p, void* out, int64_t ld_out, const void* a_codes, int64_t ld_a, const void* a_scales, const void* b_codes, int64_t ld_b,
             const void* b_scales, int64_t rows, int accumulate, cudaStream_t stream) {
  // the result's columns are the kernel's rows: neighbours of a row of the result lie in neighbouring lanes
  const int64_t M = p.outputs, N = rows, K = p.dim, bytes = (K + 31) / 32 * 16, words = (K + 127) / 128 * 128;
  const Choice c = choose(M, N, K, p.sms);
  const Built b = of(c.tile);
  W4Args a{};
  a.M = (uint32_t)M;
  a.N = (uint32_t)N;
  a.K = (uint32_t)K;
  a.slices = (uint32_t)c.slices;
  a.out = out;
  a.ld_out = ld_out;
  a.status = p.status;
  a.spin_limit = p.test_fault ? 1u << 14 : TC_SPIN_LIMIT;
  a.test_fault = p.test_fault;
  a.out_type = p.out_dtype;
  a.add = accumulate != 0;
  const bool ok = encode(&a.map_a, b_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, bytes, M, ld_b, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) &&
                  encode(&a.map_b, a_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, bytes, N, ld_a, 128, (uint32_t)b.bn, CU_TENSOR_MAP_SWIZZLE_128B) &&
                  encode(&a.map_sa, b_scales, CU_TENSOR_MAP_DATA_TYPE_INT32, words, (M + 127) / 128, words * 4, 256, 1, CU_TENSOR_MAP_SWIZZLE_NONE) &&
                  encode(&a.map_sb, a_scales, CU_TENSOR_MAP_DATA_TYPE_INT32, words, (N + 127) / 128, words * 4, 256, b.bn > 128 ? 2 : 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!ok) return TC_ERR_UNSUPPORTED;
  const int64_t tiles = ((M + 127) / 128) * ((N + b.bn - 1) / b.bn);
  if (tiles > UINT32_MAX / 2) return TC_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)std::min<int64_t>(tiles, std::max(1, p.sms / c.slices)) * c.slices;
  TC_CUDA_OK(launch_in_clusters(true, b.kernel, dim3(grid), (unsigned)b.threads, (size_t)b.smem, c.slices, stream, a));
  return TC_OK;
}

}  // namespace

size_t tc_micro_product_workspace(const TcOpShape&) { return 0; }

int tc_micro_product_prepare() {
  for (int t = 0; t < kTiles; ++t) {
    const Built b = of(t);
    cudaFuncAttributes built;
    TC_CUDA_OK(cudaFuncGetAttributes(&built, b.kernel));
    if (built.numRegs * b.threads < 256 * (W4Cfg<16>::EPILOGUE_REGS + W4Cfg<16>::OTHER_REGS)) return TC_ERR_UNSUPPORTED;
    TC_CUDA_OK(cudaFuncSetAttribute(b.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, b.smem));
  }
  return TC_OK;
}

std::string tc_micro_product_json(const TcOpShape& p) {
  const Choice c = choose(p.outputs, p.tokens, p.dim, p.sms);
  const Built b = of(c.tile);
  return "{\"operator\":\"micro_product\",\"out_dtype\":\"" + tc_type_name(p.out_dtype) + "\",\"rows\":" + std::to_string(p.tokens) + ",\"cols\":" + std::to_string(p.outputs) +
         ",\"inner\":" + std::to_string(p.dim) + ",\"tile\":[" + std::to_string(128) + "," + std::to_string(b.bn) + "],\"slices\":" + std::to_string(c.slices) +
         ",\"flops\":" + std::to_string(2.0 * p.tokens * p.outputs * p.dim) + ",\"workspace_bytes\":" + std::to_string(tc_micro_product_workspace(p)) + "}";
}

extern "C" int tc_micro_product_execute(tc_op_plan* p, void* out, int64_t ld_out, const void* a_codes, int64_t ld_a, const void* a_scales, const void* b_codes, int64_t ld_b,
                                        const void* b_scales, int64_t rows, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p || p->kind != TC_OP_MICRO_PRODUCT || (rows && (!out || !a_codes || !a_scales || !b_codes || !b_scales))) return TC_ERR_INVALID_ARG;
  const int64_t bytes = (p->dim + 31) / 32 * 16;
  if (rows < 0 || rows > p->tokens || ld_out < p->outputs || ld_a < bytes || ld_b < bytes) return TC_ERR_EXTENT;
  if (tc_odd_address(a_codes, 16) || tc_odd_address(a_scales, 16) || tc_odd_address(b_codes, 16) || tc_odd_address(b_scales, 16) || ld_a % 16 || ld_b % 16 ||
      tc_odd_address(out, tc_elem_bytes(p->out_dtype)))
    return TC_ERR_ALIGNMENT;
  const TcSpan spans[] = {{out, ld_out * tc_elem_bytes(p->out_dtype), p->outputs * tc_elem_bytes(p->out_dtype), rows, true},
                          {a_codes, ld_a, bytes, rows, false},
                          {a_scales, 0, rows ? tc_micro_scale_bytes(rows, p->dim) : 0, 1, false},
                          {b_codes, ld_b, bytes, p->outputs, false},
                          {b_scales, 0, tc_micro_scale_bytes(p->outputs, p->dim), 1, false}};
  if (tc_results_overlap(spans)) return TC_ERR_INVALID_ARG;
  if (ld_a >= int64_t(1) << 40 || ld_b >= int64_t(1) << 40) return TC_ERR_UNSUPPORTED;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  TcScratch scratch;
  const int st = scratch.open(p, TC_OP_MICRO_PRODUCT, workspace, workspace_bytes, s);
  if (st != TC_OK || rows == 0) return st;
  return scratch.close(multiply(*p, out, ld_out, a_codes, ld_a, a_scales, b_codes, ld_b, b_scales, rows, accumulate, s));
}

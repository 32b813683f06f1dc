// Matrix products of 16-bit operands on tcgen05 (tc_wm_kernel.cuh): arguments and launch.
#pragma once
#include <cuda_runtime.h>

#include "tc_internal.h"

// One token that takes part in the loss: log2(e) * logsumexp of its logits, the weight of its gradient, its target.
struct WmRow {
  float lse2, weight;
  int64_t target;
};

// A 16-bit output [batch][rows][cols]: boxes of a tensor map, or element by element (strides in elements).
struct WmOut {
  void* ptr;
  int64_t row_stride, col_stride, batch_stride;
  int32_t boxes, bf16;
  int32_t planes;         // 2: fp16 values as a sum of two, [batch][2][rows][cols]
};
struct WmStatsArgs {
  const void* target;     // per row, 64-bit where wide, else 32
  int32_t wide;
  float* hit;             // its target's logit
  float2* part;           // [2 per tile of columns][pitch]: largest logit, sum of exponentials relative to it
  uint32_t pitch, part0;
  int64_t first;          // vocabulary index of column 0
};
struct WmProbArgs {
  const WmRow* rows;
  int64_t first;
  uint32_t rows_most;     // rows of the output's buffer
  uint32_t pad;           // rows that there are no tokens for, up to a multiple of this, are zeros
};
struct WmGradsArgs {
  int32_t add;            // first product: added to what is there
  const float* scale;     // second product: device
};
struct WmAffineArgs {
  float alpha, beta;
  const float* scale;     // per matrix of the batch; alpha is multiplied by its scale_power-th power, beta by it where that is 1
  int32_t scale_power;
  const void* add;        // fp16, rows padded to 8 elements; two terms where the operands have
  int64_t add_pitch, add_batch;
  float shift;            // subtracted on a symmetric result's diagonal
};

// A second product of the same launch (WM_GRADS).
struct WmSecond {
  TcTensorMap map_a, map_b, map_d;
  uint32_t M, N, K;       // K: counted by `count`
};

struct WmArgs {
  TcTensorMap map_a, map_b, map_d, map_t;
  uint32_t M, N, K, batch, slices;
  const int32_t* count;   // device: how many rows there are (k of a second product), or null: all ...
  int32_t count_first;    // ... of which this launch has those from here on
  int32_t bf16;           // operands' type
  int32_t terms;          // two-term operands [batch][2][rows][k]: which products of terms (0: one-term operands), see WmAffine
  int* status;
  uint32_t spin_limit;
  int32_t test_fault;
  WmOut out;
  union {
    WmStatsArgs stats;
    WmProbArgs prob;
    WmGradsArgs grads;
    WmAffineArgs affine;
  };
  WmSecond second;
};

// stats, prob: A and B with k the fastest.  grads: two products, fp32 slices of one whose B has its row the fastest, and 16-bit
// results of one whose operands both have; either may have no rows.  symmetric: A and B k the fastest, the result symmetric.
// update: B with its row the fastest.
enum WmKind { WM_STATS, WM_PROB, WM_GRADS, WM_SYMMETRIC, WM_UPDATE };
enum WmTile { WM_PAIR_256 = 0, WM_128 = 1, WM_TILES = 2 };
inline int wm_tile_m(int tile) { return tile == WM_PAIR_256 ? 256 : 128; }
inline int wm_tile_n(int tile) { return tile == WM_PAIR_256 ? 256 : 128; }

// An operand [batch][rows][k], with two terms [batch][2][rows][k] and batch_stride between planes; pitch: elements between rows, or between k where the row index is the fastest.
struct WmOperand {
  const void* ptr;
  int64_t pitch, batch_stride;
};

// Whether boxes of a tensor map can address a matrix of es-byte elements.
inline bool wm_boxable(const void* ptr, int64_t pitch, int64_t batch_stride, int es) {
  return !(reinterpret_cast<uintptr_t>(ptr) & 15) && pitch > 0 && (pitch * es) % 16 == 0 && (batch_stride * es) % 16 == 0 && pitch * es < (int64_t(1) << 40) &&
         batch_stride * es < (int64_t(1) << 40);
}
// Whether boxes may be stored to a matrix of a caller's: a box whose row ends inside a 16-byte piece writes the whole piece
// (seen on B200; loads stop at the extent), so rows have to end with one.
inline bool wm_box_output(const void* ptr, int64_t cols, int64_t pitch, int64_t batch_stride) {
  return cols % 8 == 0 && wm_boxable(ptr, pitch, batch_stride, 2);
}
// Tile and slices of K that take the least time by the model beside it in tc_wm.cu; slices_most = 1: never sliced.
void wm_choose(WmKind kind, int64_t M, int64_t N, int64_t K, int64_t batch, int slices_most, int sms, int* tile, int* slices);
// k of a stage of the second product of WM_GRADS: rows of its operands are read up to a multiple of it.
int wm_grads_stage(int64_t K, int64_t K2, int tile);
// The same for WM_GRADS: slices of the first product.
void wm_choose_grads(int64_t M, int64_t N, int64_t K, int64_t M2, int64_t N2, int64_t K2, int slices_most, int sms, int* tile, int* slices);
// Opts the kernels of a kind in to their shared memory.
int wm_prepare(WmKind kind);
// Makes the maps of `args` (M, N, K, batch, slices, out and the kind's own arguments are set) and launches.
int wm_launch(WmKind kind, int tile, WmArgs& args, const WmOperand& a, const WmOperand& b, int sms, cudaStream_t stream);
// WM_GRADS: `slab` is the first product's fp32 output [slices][slab_rows][N], args.out the second's.
int wm_launch_grads(int tile, WmArgs& args, const WmOperand& a, const WmOperand& b, float* slab, int64_t slab_rows, const WmOperand& a2, const WmOperand& b2, int sms,
                    cudaStream_t stream);

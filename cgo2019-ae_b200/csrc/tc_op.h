// Plans of the operators around contractions: embedding, vocabulary loss, orthogonalised updates; microscaled 4-bit numbers and their
// products, activations kept in 8 bits, norms on the residual stream (tc_op.cu; tc_embed.cu, tc_loss.cu, tc_orth.cu; tc_micro.cu,
// tc_micro_product.cu, tc_checkpoint.cu, tc_norm.cu).
#pragma once
#include <cuda_runtime.h>

#include <mutex>
#include <string>
#include <vector>

#include "tc_internal.h"

enum TcOpKind {
  TC_OP_EMBEDDING = 0, TC_OP_VOCAB_LOSS = 1, TC_OP_ORTHOGONAL = 2, TC_OP_MICROSCALE = 3, TC_OP_MICRO_PRODUCT = 4, TC_OP_CHECKPOINT = 5, TC_OP_RESIDUAL_NORM = 6, TC_OP_KINDS = 7
};

// What a plan computes, and on how many multiprocessors.
struct TcOpShape {
  TcOpKind kind;
  int dtype = 0, out_dtype = 0;
  // embedding, vocabulary loss: the most tokens of a call, the table; the others: the most rows of a call and their elements
  int64_t tokens = 0, vocab = 0, dim = 0;
  double scale = 1.0;     // residual norm: of the residual stream
  int64_t outputs = 0;    // micro product
  int activation = 0, gated = 0, products = 0;  // checkpoint
  int gate = 0, weight_dtype = 0;        // residual norm (its eps below)
  // orthogonal
  int64_t batch = 0, rows = 0, cols = 0;
  int steps = 0;
  float coef[16][3] = {};
  double eps = 0;
  int sms = TC_DEFAULT_SMS;
};

struct tc_op_plan : TcOpShape {
  int ctas = 1;  // orthogonal: per matrix, where one launch runs the whole iteration (on commit)
  int test_fault = 0;
  bool committed = false;
  int device = -1;
  // The plan's memory: the status word, and from kOpHead bytes on the workspace of calls that bring none.
  size_t ws_bytes = 0;
  char* ws = nullptr;
  bool owns_ws = false;
  int* status = nullptr;
  // Calls that share the plan's workspace are ordered on the device, whichever streams they are on.
  std::mutex mu;
  cudaEvent_t done = nullptr;
  unsigned long long last = 0;  // id of that stream
  bool used = false;
  // The last call with a workspace of the caller's on each stream: its waits may still write the status word.
  struct Other {
    unsigned long long stream;  // its id, which no other stream ever has
    cudaEvent_t done;
  };
  std::vector<Other> others;
};

constexpr size_t kOpHead = 1024;

size_t tc_embed_workspace(const TcOpShape& p);
size_t tc_loss_workspace(const TcOpShape& p);
size_t tc_orth_workspace(const TcOpShape& p);
size_t tc_micro_product_workspace(const TcOpShape& p);
size_t tc_checkpoint_workspace(const TcOpShape& p);
size_t tc_norm_workspace(const TcOpShape& p);
// Once per device: the kernels' shared memory.
int tc_embed_prepare();
int tc_loss_prepare();
int tc_orth_prepare();
int tc_micro_product_prepare();
int tc_checkpoint_prepare();
int tc_norm_prepare();
int tc_orth_plan(tc_op_plan* p);  // on commit: what depends on the device
std::string tc_loss_json(const TcOpShape& p);
std::string tc_orth_json(const TcOpShape& p);
std::string tc_embed_json(const TcOpShape& p);
std::string tc_micro_json(const TcOpShape& p);
std::string tc_micro_product_json(const TcOpShape& p);
std::string tc_checkpoint_json(const TcOpShape& p);
std::string tc_norm_json(const TcOpShape& p);

// Commits a plan in its first call, which a stream capture cannot hold.
int tc_op_commit_for(tc_op_plan* p, cudaStream_t stream);

// The same, and that the plan is the current device's: for calls without a workspace.
int tc_op_ready(tc_op_plan* p, cudaStream_t stream);

inline std::string tc_type_name(int dtype) { return dtype == TC_BF16 ? "bf16" : dtype == TC_F16 ? "f16" : dtype == TC_F32 ? "f32" : "f64"; }
inline int tc_elem_bytes(int dtype) { return dtype == TC_F64 ? 8 : dtype == TC_F32 ? 4 : 2; }

// Memory of an argument: rows of `bytes` bytes that lie `pitch` bytes apart; none where ptr is null or a count is zero.
struct TcSpan {
  const void* ptr;
  int64_t pitch, bytes, rows;
  bool written;
};
// Whether two share a byte.  Rows may lie between each other's, as columns of one matrix do.
bool tc_spans_meet(const TcSpan& a, const TcSpan& b);
// Whether a result shares memory with an argument or with another result.  First by their first and last bytes: a pair costs a nanosecond, where
// looking at rows takes twenty.
template <int N>
bool tc_results_overlap(const TcSpan (&spans)[N]) {
  uintptr_t from[N], to[N];
  for (int i = 0; i < N; ++i) {
    const TcSpan& s = spans[i];
    int64_t length;
    from[i] = reinterpret_cast<uintptr_t>(s.ptr);
    const bool far = __builtin_mul_overflow(s.rows - 1, s.pitch, &length) || __builtin_add_overflow(length, s.bytes, &length);
    if (!s.ptr || s.rows < 1 || s.bytes < 1) to[i] = from[i] = 0;
    else if (far || __builtin_add_overflow(from[i], (uintptr_t)length, &to[i])) to[i] = UINTPTR_MAX;
  }
  for (int i = 0; i < N; ++i)
    for (int j = 0; spans[i].written && j < N; ++j)
      if (from[i] < to[j] && from[j] < to[i] && j != i && (j > i || !spans[j].written) && tc_spans_meet(spans[i], spans[j])) return true;
  return false;
}

// Scales of a microscaled 4-bit matrix: pieces of 512 bytes for 128 rows by 4 blocks.
inline int64_t tc_micro_scale_bytes(int64_t rows, int64_t cols) { return (rows + 127) / 128 * ((cols + 127) / 128) * 512; }

// Hands out pieces of a workspace, 1024-byte aligned; with base null it only counts.
struct TcCarver {
  char* base;
  size_t used = 0;
  template <class T>
  T* take(size_t count) {
    T* r = reinterpret_cast<T*>(base ? base + used : nullptr);
    used += (count * sizeof(T) + 1023) & ~size_t(1023);
    return r;
  }
};

// One call's hold on a workspace: the caller's, or the plan's behind the call that used it before.
class TcScratch {
 public:
  // Commits the plan where that is still to be done, and checks device and workspace.
  int open(tc_op_plan* p, TcOpKind kind, void* ws, size_t ws_bytes, cudaStream_t stream);
  // Marks the end of the call's work on the stream; what the call returns.
  int close(int status);
  char* base = nullptr;

 private:
  tc_op_plan* plan_ = nullptr;
  cudaStream_t stream_ = nullptr;
  unsigned long long last_ = 0;
  bool owned_ = false, captured_ = false;
  std::unique_lock<std::mutex> lock_;
};

// Plans of the operators around contractions: embedding, vocabulary loss, orthogonalised updates (tc_op.cu, tc_embed.cu,
// tc_loss.cu, tc_orth.cu).
#pragma once
#include <cuda_runtime.h>

#include <mutex>
#include <string>
#include <vector>

#include "tc_internal.h"

enum TcOpKind { TC_OP_EMBEDDING = 0, TC_OP_VOCAB_LOSS = 1, TC_OP_ORTHOGONAL = 2 };

// What a plan computes, and on how many multiprocessors.
struct TcOpShape {
  TcOpKind kind;
  int dtype = 0, out_dtype = 0;
  // embedding, vocabulary loss: the most tokens of a call, the table
  int64_t tokens = 0, vocab = 0, dim = 0;
  double scale = 1.0;
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
// Once per device: the kernels' shared memory.
int tc_embed_prepare();
int tc_loss_prepare();
int tc_orth_prepare();
int tc_orth_plan(tc_op_plan* p);  // on commit: what depends on the device
std::string tc_loss_json(const TcOpShape& p);
std::string tc_orth_json(const TcOpShape& p);
std::string tc_embed_json(const TcOpShape& p);

// Commits a plan in its first call, which a stream capture cannot hold.
int tc_op_commit_for(tc_op_plan* p, cudaStream_t stream);

inline int tc_elem_bytes(int dtype) { return dtype == TC_F64 ? 8 : dtype == TC_F32 ? 4 : 2; }

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

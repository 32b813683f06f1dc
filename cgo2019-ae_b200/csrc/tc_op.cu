// Plans of the operators around contractions: what they have in common.
#include "tc_op.h"

#include <string.h>

#include <algorithm>
#include <atomic>
#include <new>

namespace {
int new_plan(TcOpKind kind, tc_op_plan** out) {
  *out = new (std::nothrow) tc_op_plan;
  if (!*out) return TC_ERR_WORKSPACE;
  (*out)->kind = kind;
  return TC_OK;
}
bool half_type(int dtype) { return dtype == TC_BF16 || dtype == TC_F16; }
constexpr int64_t kMostExtent = int64_t(1) << 30;  // coordinates of tensor maps are 32 bits

std::atomic<uint64_t> g_prepared[TC_OP_KINDS];  // by kind: devices

struct Kind {
  size_t (*workspace)(const TcOpShape&);
  int (*prepare)();
  std::string (*json)(const TcOpShape&);
  bool products;  // on tensor cores, with waits that a test can let run out
};
size_t no_workspace(const TcOpShape&) { return 0; }
int no_preparation() { return TC_OK; }
const Kind kKinds[TC_OP_KINDS] = {{tc_embed_workspace, tc_embed_prepare, tc_embed_json, false},
                                  {tc_loss_workspace, tc_loss_prepare, tc_loss_json, true},
                                  {tc_orth_workspace, tc_orth_prepare, tc_orth_json, true},
                                  {no_workspace, no_preparation, tc_micro_json, false},
                                  {tc_micro_product_workspace, tc_micro_product_prepare, tc_micro_product_json, true},
                                  {tc_checkpoint_workspace, tc_checkpoint_prepare, tc_checkpoint_json, true},
                                  {tc_norm_workspace, tc_norm_prepare, tc_norm_json, false}};

size_t memory_of(const TcOpShape& p) {
  return kOpHead + kKinds[p.kind].workspace(p);
}

// Zero by the time this returns: no stream that a later call names is ordered behind the legacy one, on which it is written.
cudaError_t clear_word(int* word) {
  const cudaError_t e = cudaMemsetAsync(word, 0, sizeof(int), cudaStreamLegacy);
  return e != cudaSuccess ? e : cudaStreamSynchronize(cudaStreamLegacy);
}

int commit_locked(tc_op_plan* p, void* memory, size_t bytes) {
  if (p->committed) return TC_OK;
  int dev = 0;
  TC_CUDA_OK(cudaGetDevice(&dev));
  TC_CUDA_OK(cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, dev));
  if (dev >= 64 || !(g_prepared[p->kind].load() >> dev & 1)) {
    const int st = kKinds[p->kind].prepare();
    if (st != TC_OK) return st;
    if (dev < 64) g_prepared[p->kind].fetch_or(uint64_t(1) << dev);
  }
  if (p->kind == TC_OP_ORTHOGONAL) {
    const int st = tc_orth_plan(p);
    if (st != TC_OK) return st;
  }
  p->ws_bytes = memory_of(*p);
  if (!p->done) TC_CUDA_OK(cudaEventCreateWithFlags(&p->done, cudaEventDisableTiming));
  if (memory) {
    if (bytes < p->ws_bytes || (reinterpret_cast<uintptr_t>(memory) & 1023)) return TC_ERR_WORKSPACE;
    p->ws = static_cast<char*>(memory);
  } else {
    void* got = nullptr;
    TC_CUDA_OK(cudaMalloc(&got, p->ws_bytes));
    p->ws = static_cast<char*>(got);
    p->owns_ws = true;
  }
  p->status = reinterpret_cast<int*>(p->ws);
  const cudaError_t e = clear_word(p->status);
  if (e != cudaSuccess) {
    if (p->owns_ws) cudaFree(p->ws);
    p->ws = nullptr;
    p->status = nullptr;
    p->owns_ws = false;
    TC_CUDA_OK(e);
  }
  p->device = dev;
  p->committed = true;
  return TC_OK;
}
}  // namespace

namespace {
int commit_in_call(tc_op_plan* p, cudaStream_t stream) {
  if (p->committed) return TC_OK;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  TC_CUDA_OK(cudaStreamIsCapturing(stream, &capture));
  return capture != cudaStreamCaptureStatusNone ? TC_ERR_STATE : commit_locked(p, nullptr, 0);
}

// Marks the end of a call that brought its own workspace, under the plan's mutex.
cudaError_t note_other(tc_op_plan* p, cudaStream_t stream) {
  unsigned long long id = 0;
  cudaError_t e = cudaStreamGetId(stream, &id);
  if (e != cudaSuccess) return e;
  for (const auto& o : p->others)
    if (o.stream == id) return cudaEventRecord(o.done, stream);
  // a stream that has not been seen: the entry of one whose calls have all ended, where there are many
  if (p->others.size() >= 16) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // another thread may be capturing; these events are not its graph's
    const bool relaxed = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
    tc_op_plan::Other* ended = nullptr;
    for (auto& o : p->others)
      if (!ended && cudaEventQuery(o.done) == cudaSuccess) ended = &o;
    (void)cudaGetLastError();  // cudaErrorNotReady
    if (relaxed) cudaThreadExchangeStreamCaptureMode(&mode);
    if (ended) {
      ended->stream = id;
      return cudaEventRecord(ended->done, stream);
    }
  }
  cudaEvent_t made = nullptr;
  e = cudaEventCreateWithFlags(&made, cudaEventDisableTiming);
  if (e != cudaSuccess) return e;
  try {
    p->others.push_back({id, made});
  } catch (...) {
    cudaEventDestroy(made);
    return cudaErrorMemoryAllocation;
  }
  return cudaEventRecord(made, stream);
}
}  // namespace

int TcScratch::open(tc_op_plan* p, TcOpKind kind, void* ws, size_t ws_bytes, cudaStream_t stream) {
  if (!p || p->kind != kind) return TC_ERR_INVALID_ARG;
  lock_ = std::unique_lock<std::mutex>(p->mu);
  const int st = commit_in_call(p, stream);
  if (st != TC_OK) return st;
  int dev = 0;
  TC_CUDA_OK(cudaGetDevice(&dev));
  if (dev != p->device) return TC_ERR_STATE;
  if (ws && (ws_bytes < p->ws_bytes || (reinterpret_cast<uintptr_t>(ws) & 1023))) return TC_ERR_WORKSPACE;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  TC_CUDA_OK(cudaStreamIsCapturing(stream, &capture));
  captured_ = capture != cudaStreamCaptureStatusNone;
  plan_ = p;
  stream_ = stream;
  base = (ws ? static_cast<char*>(ws) : p->ws) + kOpHead;
  if (ws) {
    lock_.unlock();
    return TC_OK;
  }
  owned_ = true;
  if (captured_) return TC_OK;
  // Not by the handle: cudaStreamPerThread is one for all threads' streams, a destroyed stream's may be another's by now.  On the stream
  // of the call before the wait would order nothing and take 2 us, since kernels no longer begin under the end of the ones before.
  unsigned long long id = 0;
  TC_CUDA_OK(cudaStreamGetId(stream, &id));
  if (p->used && p->last != id) TC_CUDA_OK(cudaStreamWaitEvent(stream, p->done, 0));
  last_ = id;
  return TC_OK;
}

int TcScratch::close(int status) {
  if (captured_) return status;
  // also after a launch that failed: those before it may be under way
  cudaError_t e;
  if (owned_) {
    e = cudaEventRecord(plan_->done, stream_);
    plan_->last = last_;
    plan_->used = true;
  } else {
    lock_.lock();
    e = note_other(plan_, stream_);
    lock_.unlock();
    if (e != cudaSuccess) cudaStreamSynchronize(stream_);  // nothing that destroying the plan could wait for
  }
  if (status == TC_OK && e != cudaSuccess) {
    tc_note_cuda_error((int)e, "cudaEventRecord");
    return TC_ERR_CUDA;
  }
  return status;
}

bool tc_spans_meet(const TcSpan& a, const TcSpan& b) {
  typedef __int128 Wide;  // a caller's pitch may be anything
  struct Rows {
    Wide at, pitch, bytes, rows, end;
    explicit Rows(const TcSpan& s)
        : at((Wide)reinterpret_cast<uintptr_t>(s.ptr)), pitch(s.pitch), bytes(s.bytes), rows(s.pitch ? s.rows : 1), end(at + (rows - 1) * pitch + bytes) {}
    bool meets(Wide from, Wide to) const {  // the last row that begins before `to` reaches furthest
      if (to <= at) return false;
      const Wide last = rows == 1 ? 0 : std::min(rows - 1, (to - 1 - at) / pitch);
      return at + last * pitch + bytes > from;
    }
  };
  if (!a.ptr || !b.ptr || a.rows < 1 || b.rows < 1 || a.bytes < 1 || b.bytes < 1) return false;
  const Rows x(a), y(b);
  if (x.end <= y.at || y.end <= x.at) return false;
  const Rows &few = x.rows < y.rows ? x : y, &many = x.rows < y.rows ? y : x;
  if (few.rows > 1 && x.pitch == y.pitch) return many.meets(few.at, few.at + few.bytes) || few.meets(many.at, many.at + many.bytes);
  for (Wide i = 0; i < few.rows; ++i)
    if (many.meets(few.at + i * few.pitch, few.at + i * few.pitch + few.bytes)) return true;
  return false;
}

extern "C" int tc_op_create_embedding(int64_t tokens, int64_t vocab, int64_t dim, int dtype, double scale, tc_op_plan** out) {
  if (!out || (dtype != TC_F32 && !half_type(dtype)) || scale != scale) return TC_ERR_INVALID_ARG;
  if (tokens < 1 || vocab < 1 || dim < 1) return TC_ERR_EXTENT;
  if (tokens > kMostExtent || vocab > kMostExtent || dim > kMostExtent) return TC_ERR_UNSUPPORTED;
  const int st = new_plan(TC_OP_EMBEDDING, out);
  if (st != TC_OK) return st;
  (*out)->tokens = tokens;
  (*out)->vocab = vocab;
  (*out)->dim = dim;
  (*out)->dtype = dtype;
  (*out)->scale = scale;
  return TC_OK;
}

extern "C" int tc_op_create_vocab_loss(int64_t tokens, int64_t dim, int64_t vocab, int dtype, tc_op_plan** out) {
  if (!out) return TC_ERR_INVALID_ARG;
  if (!half_type(dtype)) return dtype == TC_F32 || dtype == TC_F64 ? TC_ERR_UNSUPPORTED : TC_ERR_INVALID_ARG;
  if (tokens < 1 || vocab < 1 || dim < 1) return TC_ERR_EXTENT;
  if (tokens > kMostExtent || vocab > kMostExtent || dim > kMostExtent) return TC_ERR_UNSUPPORTED;
  const int st = new_plan(TC_OP_VOCAB_LOSS, out);
  if (st != TC_OK) return st;
  (*out)->tokens = tokens;
  (*out)->vocab = vocab;
  (*out)->dim = dim;
  (*out)->dtype = dtype;
  return TC_OK;
}

extern "C" int tc_op_create_orthogonal(int64_t batch, int64_t rows, int64_t cols, int dtype, int out_dtype, int steps, const double* coefficients, double eps,
                                       tc_op_plan** out) {
  if (!out || !coefficients || (dtype != TC_F32 && !half_type(dtype)) || !half_type(out_dtype) || !(eps >= 0)) return TC_ERR_INVALID_ARG;
  if (batch < 1 || rows < 1 || cols < 1) return TC_ERR_EXTENT;
  if (steps < 1 || steps > 16 || batch > 65535 || rows > kMostExtent || cols > kMostExtent) return TC_ERR_UNSUPPORTED;
  for (int i = 0; i < 3 * steps; ++i)
    if (!(coefficients[i] - coefficients[i] == 0)) return TC_ERR_INVALID_ARG;
  const int st = new_plan(TC_OP_ORTHOGONAL, out);
  if (st != TC_OK) return st;
  (*out)->batch = batch;
  (*out)->rows = rows;
  (*out)->cols = cols;
  (*out)->dtype = dtype;
  (*out)->out_dtype = out_dtype;
  (*out)->steps = steps;
  for (int i = 0; i < steps; ++i)
    for (int j = 0; j < 3; ++j) (*out)->coef[i][j] = (float)coefficients[3 * i + j];
  (*out)->eps = eps;
  return TC_OK;
}

extern "C" int tc_op_create_microscale(int64_t rows, int64_t cols, int dtype, tc_op_plan** out) {
  if (!out || (dtype != TC_F32 && !half_type(dtype))) return TC_ERR_INVALID_ARG;
  if (rows < 1 || cols < 1) return TC_ERR_EXTENT;
  if (rows > kMostExtent || cols > kMostExtent) return TC_ERR_UNSUPPORTED;
  const int st = new_plan(TC_OP_MICROSCALE, out);
  if (st != TC_OK) return st;
  (*out)->tokens = rows;
  (*out)->dim = cols;
  (*out)->dtype = dtype;
  return TC_OK;
}

extern "C" int tc_op_create_micro_product(int64_t rows, int64_t cols, int64_t inner, int out_dtype, tc_op_plan** out) {
  if (!out || (out_dtype != TC_F32 && !half_type(out_dtype))) return TC_ERR_INVALID_ARG;
  if (rows < 1 || cols < 1 || inner < 1) return TC_ERR_EXTENT;
  if (rows > kMostExtent || cols > kMostExtent || inner > kMostExtent) return TC_ERR_UNSUPPORTED;
  const int st = new_plan(TC_OP_MICRO_PRODUCT, out);
  if (st != TC_OK) return st;
  (*out)->tokens = rows;
  (*out)->outputs = cols;
  (*out)->dim = inner;
  (*out)->dtype = (*out)->out_dtype = out_dtype;
  return TC_OK;
}

extern "C" int tc_op_create_checkpoint(int64_t tokens, int64_t dim, int dtype, int activation, int gated, int products, tc_op_plan** out) {
  if (!out || (dtype != TC_F32 && !half_type(dtype)) || activation < TC_ACT_NONE || activation > TC_ACT_GELU) return TC_ERR_INVALID_ARG;
  if (products && !half_type(dtype)) return TC_ERR_UNSUPPORTED;
  if (tokens < 1 || dim < 1) return TC_ERR_EXTENT;
  if (tokens > kMostExtent || dim > kMostExtent) return TC_ERR_UNSUPPORTED;
  const int st = new_plan(TC_OP_CHECKPOINT, out);
  if (st != TC_OK) return st;
  (*out)->tokens = tokens;
  (*out)->dim = dim;
  (*out)->dtype = dtype;
  (*out)->activation = activation;
  (*out)->gated = gated != 0;
  (*out)->products = products != 0;
  return TC_OK;
}

extern "C" int tc_op_create_residual_norm(int64_t tokens, int64_t dim, int dtype, int weight_dtype, int gate, double residual_scale, double eps, tc_op_plan** out) {
  if (!out || (dtype != TC_F32 && !half_type(dtype)) || (weight_dtype != TC_F32 && weight_dtype != dtype) || gate < TC_GATE_NONE || gate > TC_GATE_TOKEN) return TC_ERR_INVALID_ARG;
  const float scale = (float)residual_scale;
  // in 32 bits: a row of zeros has a finite norm
  if (!(scale - scale == 0) || !(eps >= 1e-30) || !(eps <= 1e30)) return TC_ERR_INVALID_ARG;
  if (tokens < 1 || dim < 1) return TC_ERR_EXTENT;
  if (tokens > kMostExtent || dim > kMostExtent) return TC_ERR_UNSUPPORTED;
  const int st = new_plan(TC_OP_RESIDUAL_NORM, out);
  if (st != TC_OK) return st;
  (*out)->tokens = tokens;
  (*out)->dim = dim;
  (*out)->dtype = dtype;
  (*out)->weight_dtype = weight_dtype;
  (*out)->gate = gate;
  (*out)->scale = residual_scale;
  (*out)->eps = eps;
  return TC_OK;
}

extern "C" int tc_op_commit(tc_op_plan* p) {
  if (!p) return TC_ERR_INVALID_ARG;
  std::lock_guard<std::mutex> hold(p->mu);
  return commit_locked(p, nullptr, 0);
}

int tc_op_commit_for(tc_op_plan* p, cudaStream_t stream) {
  std::lock_guard<std::mutex> hold(p->mu);
  return commit_in_call(p, stream);
}

int tc_op_ready(tc_op_plan* p, cudaStream_t stream) {
  const int st = tc_op_commit_for(p, stream);
  if (st != TC_OK) return st;
  int dev = 0;
  TC_CUDA_OK(cudaGetDevice(&dev));
  return dev != p->device ? TC_ERR_STATE : TC_OK;
}

extern "C" int tc_op_commit_in(tc_op_plan* p, void* memory, size_t bytes) {
  if (!p || !memory) return TC_ERR_INVALID_ARG;
  std::lock_guard<std::mutex> hold(p->mu);
  if (p->committed) return TC_ERR_STATE;
  return commit_locked(p, memory, bytes);
}

extern "C" int tc_op_set_test_fault(tc_op_plan* p, int fault) {
  if (!p || !kKinds[p->kind].products) return TC_ERR_INVALID_ARG;
  if (p->committed) return TC_ERR_STATE;
  p->test_fault = fault;
  return TC_OK;
}

extern "C" int tc_op_workspace_bytes(const tc_op_plan* p, size_t* bytes) {
  if (!p || !bytes) return TC_ERR_INVALID_ARG;
  if (p->committed) {
    *bytes = p->ws_bytes;
    return TC_OK;
  }
  TcOpShape sized(*p);
  int dev = 0;
  TC_CUDA_OK(cudaGetDevice(&dev));
  TC_CUDA_OK(cudaDeviceGetAttribute(&sized.sms, cudaDevAttrMultiProcessorCount, dev));
  *bytes = memory_of(sized);
  return TC_OK;
}

extern "C" int tc_op_describe(const tc_op_plan* p, char* buf, size_t cap) {
  if (!p || !buf || !cap) return TC_ERR_INVALID_ARG;
  std::string s;
  try {
    s = kKinds[p->kind].json(*p);
  } catch (...) {
    return TC_ERR_WORKSPACE;
  }
  strncpy(buf, s.c_str(), cap - 1);
  buf[cap - 1] = 0;
  return TC_OK;
}

extern "C" int tc_op_status(tc_op_plan* p, int* device_status) {
  if (!p || !device_status) return TC_ERR_INVALID_ARG;
  if (!p->committed) return TC_ERR_STATE;
  TC_CUDA_OK(cudaDeviceSynchronize());  // work on non-blocking streams too
  TC_CUDA_OK(cudaMemcpy(device_status, p->status, sizeof(int), cudaMemcpyDeviceToHost));
  return TC_OK;
}

extern "C" int tc_op_status_reset(tc_op_plan* p) {
  if (!p) return TC_ERR_INVALID_ARG;
  if (!p->committed) return TC_ERR_STATE;
  TC_CUDA_OK(cudaDeviceSynchronize());
  TC_CUDA_OK(clear_word(p->status));
  return TC_OK;
}

extern "C" void tc_op_destroy(tc_op_plan* p) {
  if (!p) return;
  // another thread may be capturing: waiting for these events and giving up this memory does not concern its graph
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  const bool relaxed = p->committed && cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
  // the memory's owner may use it again
  if (p->used) cudaEventSynchronize(p->done);
  for (const auto& o : p->others) {
    cudaEventSynchronize(o.done);
    cudaEventDestroy(o.done);
  }
  if (p->owns_ws) cudaFree(p->ws);
  if (p->done) cudaEventDestroy(p->done);
  if (relaxed) cudaThreadExchangeStreamCaptureMode(&mode);
  delete p;
}

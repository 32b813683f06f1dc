"""Host-side mirror of the contraction operator over the C-ABI library.

The reference is driven by one expression line per contraction
(``t3 [a,312,b,24,c,296] += sum(d,312) * t2 [d,c,a] * v2 [b,d];``,
cogent/input_strings/tccg/input_tccg_02.in:4) that ``tc_code_generator.py``
turns into a ``.cu`` file with the entry ``sd_t_d2_fusion_``
(cogent/src/codes/kernels/tc_interface.py:1444-1598).  Here the same line makes
a :class:`Plan`; ``Plan.execute`` enqueues the hand-written sm_100a kernels on
device tensors.  Everything numeric happens inside ``libtc_b200.so``; there is
no Python or CPU compute path, and a missing library is an error.
"""
import ctypes
import json
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libtc_b200.so")

F64, F32 = 0, 1
BF16, F16, I32, I64 = 2, 3, 4, 5  # the operators around contractions: EmbeddingPlan, VocabLossPlan, OrthogonalPlan
PATH_AUTO, PATH_DMMA, PATH_DFMA, PATH_FFMA, PATH_3XTF32, PATH_TCGEN05 = 0, 1, 2, 3, 4, 5
TENSOR_OUT, TENSOR_LEFT, TENSOR_RIGHT = 0, 1, 2

PROBES_PATH = os.path.join(_HERE, "probes", "libtc_probes.so")
PEAK_NAMES = {0: "dmma_m8n8k4", 1: "dmma_m16n8k4", 2: "dmma_m16n8k8", 3: "dmma_m16n8k16",
              4: "dfma", 5: "ffma", 6: "tf32_mma_sync", 7: "tf32_tcgen05"}


class TcError(RuntimeError):
    def __init__(self, status, where, detail=""):
        self.status = status
        msg = "%s failed: %s (status %d)" % (where, _status_string(status), status)
        if detail:
            msg += " -- " + detail
        super().__init__(msg)


class Options(ctypes.Structure):
    _fields_ = [("path", ctypes.c_int), ("tile_m", ctypes.c_int), ("tile_n", ctypes.c_int),
                ("split_k", ctypes.c_int), ("variant", ctypes.c_int), ("l2_prefetch", ctypes.c_int),
                ("c_path", ctypes.c_int), ("tma", ctypes.c_int), ("test_fault", ctypes.c_int)]


_lib = None

# name -> (restype, argtypes); every symbol include/tc_b200.h declares.
_SIGNATURES = {
    "tc_plan_create_sharded": (ctypes.c_int, [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int),
                                              ctypes.c_int, ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]),
    "tc_sharded_set_extents": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.POINTER(ctypes.c_char_p),
                                              ctypes.POINTER(ctypes.c_int64)]),
    "tc_sharded_describe": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]),
    "tc_sharded_commit": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_execute_sharded": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p),
                                          ctypes.POINTER(ctypes.c_void_p), ctypes.c_int]),
    "tc_sharded_synchronize": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_sharded_destroy": (None, [ctypes.c_void_p]),
    "tc_expr_describe": (ctypes.c_int, [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_size_t]),
    "tc_plan_create": (ctypes.c_int, [ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(Options),
                                      ctypes.POINTER(ctypes.c_void_p)]),
    "tc_plan_set_extents": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.POINTER(ctypes.c_char_p),
                                           ctypes.POINTER(ctypes.c_int64)]),
    "tc_plan_set_extents_ordered": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.POINTER(ctypes.c_int64)]),
    "tc_sd_t_d2_fusion": (ctypes.c_int, [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int),
                                         ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]),
    "tc_plan_set_strides": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_int,
                                           ctypes.POINTER(ctypes.c_int64)]),
    "tc_plan_commit": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_plan_destroy": (None, [ctypes.c_void_p]),
    "tc_plan_describe": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]),
    "tc_plan_cost": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_double),
                                    ctypes.POINTER(ctypes.c_double)]),
    "tc_plan_launches": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_plan_status": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]),
    "tc_plan_status_reset": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_plan_workspace_bytes": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]),
    "tc_execute": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                  ctypes.c_void_p]),
    "tc_execute_ws": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                     ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "tc_execute_noalloc": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                          ctypes.c_void_p]),
    "tc_plan_create_fused": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(ctypes.c_char_p), ctypes.c_int,
                                            ctypes.POINTER(ctypes.c_void_p)]),
    "tc_fused_set_extents": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.POINTER(ctypes.c_char_p),
                                            ctypes.POINTER(ctypes.c_int64)]),
    "tc_fused_commit": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_fused_describe": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]),
    "tc_fused_set_test_fault": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int]),
    "tc_fused_status": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]),
    "tc_fused_status_reset": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_execute_fused": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p),
                                        ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p]),
    "tc_fused_destroy": (None, [ctypes.c_void_p]),
    "tc_op_create_embedding": (ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_double,
                                              ctypes.POINTER(ctypes.c_void_p)]),
    "tc_op_create_vocab_loss": (ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.POINTER(ctypes.c_void_p)]),
    "tc_op_create_orthogonal": (ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                               ctypes.POINTER(ctypes.c_double), ctypes.c_double, ctypes.POINTER(ctypes.c_void_p)]),
    "tc_op_commit": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_op_commit_in": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t]),
    "tc_op_workspace_bytes": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]),
    "tc_op_describe": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]),
    "tc_op_status": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]),
    "tc_op_status_reset": (ctypes.c_int, [ctypes.c_void_p]),
    "tc_op_set_test_fault": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int]),
    "tc_op_destroy": (None, [ctypes.c_void_p]),
    "tc_embedding_execute": (ctypes.c_int, [ctypes.c_void_p] + [ctypes.c_void_p, ctypes.c_int64] * 2 + [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64,
                                                                                                       ctypes.c_void_p]),
    "tc_embedding_execute_grad": (ctypes.c_int, [ctypes.c_void_p] + [ctypes.c_void_p, ctypes.c_int64] * 2 +
                                  [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "tc_vocab_loss_execute": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_void_p, ctypes.c_int64] * 2 +
                              [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "tc_vocab_loss_execute_grad": (ctypes.c_int, [ctypes.c_void_p] + [ctypes.c_void_p, ctypes.c_int64] * 4 +
                                   [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                    ctypes.c_size_t, ctypes.c_void_p]),
    "tc_orthogonal_execute": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64), ctypes.c_void_p,
                                             ctypes.POINTER(ctypes.c_int64), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "tc_execute_host": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]),
    "tc_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "tc_last_cuda_error": (ctypes.c_char_p, []),
    "tc_version": (ctypes.c_char_p, []),
    "tc_fill_uniform": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_uint64,
                                       ctypes.c_int, ctypes.c_int64, ctypes.c_void_p]),
    "tc_axpy": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int,
                               ctypes.c_double, ctypes.c_void_p]),
}


def exported_symbols():
    return sorted(_SIGNATURES)


def lib():
    """The loaded C-ABI library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError("%s is missing: run `python %s` (or __graft_entry__.build()) first; "
                              "there is no fallback path" % (LIB_PATH, os.path.join(_HERE, "build.py")))
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def _status_string(status):
    try:
        return lib().tc_status_string(status).decode()
    except Exception:  # pragma: no cover - library missing
        return "?"


def _check(status, where):
    if status != 0:
        detail = lib().tc_last_cuda_error().decode() if status == 5 else ""
        raise TcError(status, where, detail)


def parse(expr):
    """Parsed form of one expression line (dict), or raises TcError(status 1 / 3)."""
    buf = ctypes.create_string_buffer(8192)
    st = lib().tc_expr_describe(expr.encode(), buf, len(buf))
    if st != 0:
        raise TcError(st, "tc_expr_describe", json.loads(buf.value.decode() or "{}").get("error", ""))
    return json.loads(buf.value.decode())


_raw_stream = None


def _current_stream(device_index):
    """Address of torch's current stream on a device (0: the legacy default stream)."""
    global _raw_stream
    if _raw_stream is None:
        import torch
        # the number itself where torch offers it: building a Stream object takes as long as the launch of a small kernel
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
    return _raw_stream(device_index)


def _stream(stream, *tensors):
    """cudaStream_t for a call: the caller's, else torch's current stream when the arguments are torch CUDA tensors
    (so that the launch is ordered with the surrounding torch work), else the legacy default stream."""
    if stream:
        return stream
    for t in tensors:
        if getattr(t, "is_cuda", False):
            return _current_stream(t.get_device()) or None
    return None


def _ptr(x):
    """Device/host address of a torch tensor, numpy array or raw int (ctypes converts it at the call)."""
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if x is None or isinstance(x, int):
        return x
    if hasattr(x, "ctypes"):
        return x.ctypes.data
    raise TypeError("expected a tensor, array or address, got %r" % type(x))


class Plan:
    """One contraction: expression + dtype (+ extents, strides, options)."""

    def __init__(self, expr, dtype=F64, path=PATH_AUTO, tile=None, split_k=0, extents=None, variant=0, l2_prefetch=0, c_path=0, tma=0,
                 test_fault=0):
        self._h = ctypes.c_void_p()
        opt = Options()
        opt.path = path
        if tile:
            opt.tile_m, opt.tile_n = tile
        opt.split_k = split_k
        opt.variant = variant
        opt.l2_prefetch = l2_prefetch
        opt.c_path = c_path
        opt.tma = tma
        opt.test_fault = test_fault
        self.expr = expr
        self.dtype = dtype
        _check(lib().tc_plan_create(expr.encode(), dtype, ctypes.byref(opt), ctypes.byref(self._h)), "tc_plan_create")
        if extents:
            self.set_extents(extents)

    def set_extents(self, extents):
        names = list(extents)
        arr_n = (ctypes.c_char_p * len(names))(*[n.encode() for n in names])
        arr_e = (ctypes.c_int64 * len(names))(*[int(extents[n]) for n in names])
        _check(lib().tc_plan_set_extents(self._h, len(names), arr_n, arr_e), "tc_plan_set_extents")
        return self

    def set_strides(self, tensor, strides):
        arr = (ctypes.c_int64 * len(strides))(*[int(s) for s in strides])
        _check(lib().tc_plan_set_strides(self._h, tensor, len(strides), arr), "tc_plan_set_strides")
        return self

    def commit(self):
        _check(lib().tc_plan_commit(self._h), "tc_plan_commit")
        return self

    def describe(self):
        buf = ctypes.create_string_buffer(16384)
        st = lib().tc_plan_describe(self._h, buf, len(buf))
        if st != 0:
            raise TcError(st, "tc_plan_describe", json.loads(buf.value.decode() or "{}").get("error", ""))
        return json.loads(buf.value.decode())

    def cost(self):
        f, b = ctypes.c_double(), ctypes.c_double()
        _check(lib().tc_plan_cost(self._h, ctypes.byref(f), ctypes.byref(b)), "tc_plan_cost")
        return f.value, b.value

    @property
    def launches(self):
        return lib().tc_plan_launches(self._h)

    def status(self):
        """Device status word (synchronises): 0 unless a bounded wait in a persistent kernel gave up."""
        v = ctypes.c_int()
        _check(lib().tc_plan_status(self._h, ctypes.byref(v)), "tc_plan_status")
        return v.value

    def status_reset(self):
        _check(lib().tc_plan_status_reset(self._h), "tc_plan_status_reset")

    def workspace_bytes(self):
        n = ctypes.c_size_t()
        _check(lib().tc_plan_workspace_bytes(self._h, ctypes.byref(n)), "tc_plan_workspace_bytes")
        return n.value

    def execute(self, C, A, B, stream=None, workspace=None):
        """Enqueue C (op)= sum A*B on device tensors (torch CUDA tensors or raw device addresses)."""
        s = _stream(stream, C)
        if workspace is None:
            st = _lib.tc_execute(self._h, _ptr(C), _ptr(A), _ptr(B), s)
            if st:
                _check(st, "tc_execute")
        else:
            nbytes = workspace.numel() * workspace.element_size()
            _check(lib().tc_execute_ws(self._h, _ptr(C), _ptr(A), _ptr(B), _ptr(workspace), nbytes, s), "tc_execute_ws")

    def execute_noalloc(self, C, A, B, stream=None):
        """tc_execute that takes K-slice scratch from the library's fixed array instead of allocated memory
        (for callers that cannot allocate); the plan must be committed and the scratch need must fit."""
        s = _stream(stream, C)
        _check(lib().tc_execute_noalloc(self._h, _ptr(C), _ptr(A), _ptr(B), s), "tc_execute_noalloc")

    def execute_host(self, C, A, B):
        """Blocking call on host arrays (numpy, C-contiguous 1-D storage in column-major element order)."""
        _check(lib().tc_execute_host(self._h, _ptr(C), _ptr(A), _ptr(B)), "tc_execute_host")

    def close(self):
        if self._h:
            lib().tc_plan_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


SHARD_EXTERNAL, SHARD_CONTRACTION, SHARD_C_IS_SLAB = 0, 1, 1


class ShardedPlan:
    """One contraction over several GPUs driven by this process (tc_plan_create_sharded): `kind` SHARD_EXTERNAL cuts
    an output index (no communication), SHARD_CONTRACTION a contraction index (NCCL reduce-scatter)."""

    def __init__(self, expr, dtype=F64, devices=(0,), kind=SHARD_EXTERNAL, index=None, extents=None):
        self._h = ctypes.c_void_p()
        self.devices = list(devices)
        ids = (ctypes.c_int * len(self.devices))(*self.devices)
        _check(lib().tc_plan_create_sharded(expr.encode(), dtype, len(self.devices), ids, kind,
                                            index.encode() if index else None, ctypes.byref(self._h)), "tc_plan_create_sharded")
        if extents:
            names = list(extents)
            an = (ctypes.c_char_p * len(names))(*[n.encode() for n in names])
            ae = (ctypes.c_int64 * len(names))(*[int(extents[n]) for n in names])
            _check(lib().tc_sharded_set_extents(self._h, len(names), an, ae), "tc_sharded_set_extents")

    def describe(self):
        buf = ctypes.create_string_buffer(1 << 16)
        st = lib().tc_sharded_describe(self._h, buf, len(buf))
        if st != 0:
            raise TcError(st, "tc_sharded_describe", json.loads(buf.value.decode() or "{}").get("error", ""))
        return json.loads(buf.value.decode())

    def commit(self):
        _check(lib().tc_sharded_commit(self._h), "tc_sharded_commit")
        return self

    def execute(self, Cs, As, Bs, c_is_slab=False):
        """Cs[d], As[d], Bs[d]: the tensors in device d's memory (torch CUDA tensors or device addresses)."""
        n = len(self.devices)
        if not (len(Cs) == len(As) == len(Bs) == n):
            raise ValueError("one output and two inputs per device")
        arr = lambda xs: (ctypes.c_void_p * n)(*[_ptr(x) for x in xs])
        _check(lib().tc_execute_sharded(self._h, arr(Cs), arr(As), arr(Bs), SHARD_C_IS_SLAB if c_is_slab else 0), "tc_execute_sharded")

    def synchronize(self):
        _check(lib().tc_sharded_synchronize(self._h), "tc_sharded_synchronize")

    def close(self):
        if self._h:
            lib().tc_sharded_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class FusedPlan:
    """Several contractions accumulated into one output in a single pass over it (e.g. the nine CCSD(T) terms
    of cogent/input_strings/ccsd_t/original-expressions/sd_t_d2.in); fp64."""

    def __init__(self, exprs, dtype=F64, extents=None, test_fault=0):
        self._h = ctypes.c_void_p()
        self.exprs = list(exprs)
        arr = (ctypes.c_char_p * len(self.exprs))(*[e.encode() for e in self.exprs])
        _check(lib().tc_plan_create_fused(len(self.exprs), arr, dtype, ctypes.byref(self._h)), "tc_plan_create_fused")
        if extents:
            names = list(extents)
            an = (ctypes.c_char_p * len(names))(*[n.encode() for n in names])
            ae = (ctypes.c_int64 * len(names))(*[int(extents[n]) for n in names])
            _check(lib().tc_fused_set_extents(self._h, len(names), an, ae), "tc_fused_set_extents")
        if test_fault:
            _check(lib().tc_fused_set_test_fault(self._h, test_fault), "tc_fused_set_test_fault")

    def status(self):
        """Status word (synchronises): 0 unless a bounded wait in one of this plan's launches gave up."""
        v = ctypes.c_int()
        _check(lib().tc_fused_status(self._h, ctypes.byref(v)), "tc_fused_status")
        return v.value

    def status_reset(self):
        _check(lib().tc_fused_status_reset(self._h), "tc_fused_status_reset")

    def commit(self):
        _check(lib().tc_fused_commit(self._h), "tc_fused_commit")
        return self

    def describe(self):
        buf = ctypes.create_string_buffer(8192)
        st = lib().tc_fused_describe(self._h, buf, len(buf))
        if st != 0:
            raise TcError(st, "tc_fused_describe", json.loads(buf.value.decode() or "{}").get("error", ""))
        return json.loads(buf.value.decode())

    def execute(self, C, As, Bs, stream=None):
        """C: the output; As[k], Bs[k]: left / right input of term k (torch CUDA tensors or device addresses)."""
        n = len(self.exprs)
        if len(As) != n or len(Bs) != n:
            raise ValueError("one left and one right input per term")
        pa = (ctypes.c_void_p * n)(*[_ptr(x) for x in As])
        pb = (ctypes.c_void_p * n)(*[_ptr(x) for x in Bs])
        _check(lib().tc_execute_fused(self._h, _ptr(C), pa, pb, _stream(stream, C)), "tc_execute_fused")

    def close(self):
        if self._h:
            lib().tc_fused_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class _OpPlan:
    """What the plans of the operators around contractions share.  Their tensors are torch CUDA tensors on one device."""

    def __init__(self):
        self._h = ctypes.c_void_p()
        self._device = self._memory = None
        self._committing = threading.Lock()

    def commit(self):
        """Takes the plan's workspace from torch's allocator on the current device and loads its kernels (else the first
        execute does).  Waits for what is queued on the current stream."""
        with self._committing:  # first calls of several threads may meet
            if self._device is None:
                import torch
                if torch.cuda.is_current_stream_capturing():
                    raise TcError(7, "commit", "commit the plan before the stream capture")
                size = self.workspace_bytes()
                memory = torch.empty(size + 1024, dtype=torch.uint8, device="cuda")
                # the allocator hands out memory that work queued on this stream still uses; the plan's calls may run on others
                torch.cuda.current_stream(memory.device).synchronize()
                _check(lib().tc_op_commit_in(self._h, memory.data_ptr() + -memory.data_ptr() % 1024, size), "tc_op_commit_in")
                self._memory, self._device = memory, memory.get_device()
        return self

    def _on(self, device):
        """A call's tensors are on the plan's device."""
        if self._device is None:
            self.commit()
        if device != self._device:
            raise ValueError("the plan is committed on device %d, the tensors are on device %d" % (self._device, device))

    def describe(self):
        buf = ctypes.create_string_buffer(4096)
        _check(lib().tc_op_describe(self._h, buf, len(buf)), "tc_op_describe")
        return json.loads(buf.value.decode())

    def workspace_bytes(self):
        n = ctypes.c_size_t()
        _check(lib().tc_op_workspace_bytes(self._h, ctypes.byref(n)), "tc_op_workspace_bytes")
        return n.value

    def status(self):
        """Status word (synchronises): 0 unless a bounded wait in one of this plan's launches gave up."""
        v = ctypes.c_int()
        _check(lib().tc_op_status(self._h, ctypes.byref(v)), "tc_op_status")
        return v.value

    def status_reset(self):
        _check(lib().tc_op_status_reset(self._h), "tc_op_status_reset")

    def close(self):
        if self._h:
            lib().tc_op_destroy(self._h)  # waits for the plan's calls: its memory goes back to the allocator
            self._h = ctypes.c_void_p()
            self._memory = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_codes, _index_types = None, ()  # torch type -> code; the types of token numbers


def _types(*codes):
    """The torch types of some codes."""
    global _codes, _index_types
    if _codes is None:
        import torch
        _codes = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.int32: I32, torch.int64: I64}
        _index_types = (torch.int32, torch.int64)
    return tuple(t for t, c in _codes.items() if c in codes)


def _tensor(t, name, types, shape, device):
    """Checks one argument: a CUDA tensor of one of the types and of the shape on the device (None: any), with its last index
    contiguous.  Returns its device index."""
    # the call itself takes as long as a small kernel's launch: what is right is found right by few look-ups
    try:
        if t.is_cuda and t.dtype in types and t.shape == shape:
            where = t.get_device()
            if (device is None or where == device) and (t.stride(-1) == 1 or shape[-1] <= 1 or len(shape) == 3):
                return where
    except AttributeError:
        pass
    if not getattr(t, "is_cuda", False):
        raise TypeError("%s: expected a torch CUDA tensor, got %r" % (name, type(t)))
    if t.dtype not in types:
        raise TypeError("%s: unexpected type %s" % (name, t.dtype))
    if t.shape != shape:
        raise ValueError("%s: expected shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    if device is not None and t.get_device() != device:
        raise ValueError("%s: on device %d, other arguments on %d" % (name, t.get_device(), device))
    raise ValueError("%s: its last index must be contiguous" % name)


def _tokens_of(t, name):
    """Checks a call's token numbers; returns (device, how many, code of their type)."""
    if getattr(t, "ndim", 1) != 1:
        raise ValueError("%s: expected one index, got shape %s" % (name, tuple(t.shape)))
    device = _tensor(t, name, _index_types, getattr(t, "shape", (0,)), None)
    return device, t.shape[0], _codes[t.dtype]


def _ld(t):
    """Element distance between the rows of a matrix (one row: any that holds it)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ld_out(t, name):
    """The same of an output, whose rows may not overlap."""
    ld = _ld(t)
    if ld < t.shape[1]:
        raise ValueError("%s: its rows overlap" % name)
    return ld


def _scratch(workspace, device):
    if workspace is None:
        return None, 0
    if not workspace.is_cuda or workspace.get_device() != device or not workspace.is_contiguous():
        raise ValueError("workspace: expected a contiguous CUDA tensor on device %d" % device)
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


class EmbeddingPlan(_OpPlan):
    """Rows of a table [vocab, dim] by token number, times `scale`, and the table's gradient: sums by sorted tokens, in fp32, in
    the tokens' order.  `tokens`: the most of a call.  Token numbers outside [0, vocab) stand for no token.  BF16, F16 or F32."""

    def __init__(self, tokens, vocab, dim, dtype=BF16, scale=1.0):
        super().__init__()
        self.tokens, self.vocab, self.dim, self.dtype, self.scale = tokens, vocab, dim, dtype, scale
        self._types, self._table = _types(dtype), (vocab, dim)
        _check(lib().tc_op_create_embedding(tokens, vocab, dim, dtype, scale, ctypes.byref(self._h)), "tc_op_create_embedding")

    def execute(self, out, table, ids, stream=None):
        """out[t] = scale * table[ids[t]]; a row of zeros where ids[t] is no token."""
        device, n, index = _tokens_of(ids, "ids")
        if device != self._device:
            self._on(device)
        _tensor(out, "out", self._types, (n, self.dim), device)
        _tensor(table, "table", self._types, self._table, device)
        st = _lib.tc_embedding_execute(self._h, out.data_ptr(), _ld_out(out, "out"), table.data_ptr(), _ld(table), ids.data_ptr(), index, n,
                                       _stream(stream, ids))
        if st:
            _check(st, "tc_embedding_execute")

    def execute_grad(self, dtable, grad, ids, accumulate=False, stream=None, workspace=None):
        """dtable[v] = scale * sum of grad[t] over the t with ids[t] = v (zeros where there is none); `accumulate`: added to
        what is there."""
        device, n, index = _tokens_of(ids, "ids")
        if device != self._device:
            self._on(device)
        _tensor(dtable, "dtable", self._types, self._table, device)
        _tensor(grad, "grad", self._types, (n, self.dim), device)
        ws, size = _scratch(workspace, device)
        st = _lib.tc_embedding_execute_grad(self._h, dtable.data_ptr(), _ld_out(dtable, "dtable"), grad.data_ptr(), _ld(grad), ids.data_ptr(), index, n,
                                            1 if accumulate else 0, ws, size, _stream(stream, ids))
        if st:
            _check(st, "tc_embedding_execute_grad")


class VocabLossPlan(_OpPlan):
    """Softmax cross entropy of hidden [tokens, dim] against a table [vocab, dim], in pieces of the vocabulary, without
    keeping the logits, and its gradients.  `tokens`: the most of a call.  Tokens whose target lies outside [0, vocab) take no
    part.  BF16 or F16."""

    def __init__(self, tokens, dim, vocab, dtype=BF16):
        super().__init__()
        self.tokens, self.dim, self.vocab, self.dtype = tokens, dim, vocab, dtype
        self._types, self._f32, self._table = _types(dtype), _types(F32), (vocab, dim)
        _check(lib().tc_op_create_vocab_loss(tokens, dim, vocab, dtype, ctypes.byref(self._h)), "tc_op_create_vocab_loss")

    def _inputs(self, hidden, weight, targets):
        device, n, index = _tokens_of(targets, "targets")
        if device != self._device:
            self._on(device)
        _tensor(hidden, "hidden", self._types, (n, self.dim), device)
        _tensor(weight, "weight", self._types, self._table, device)
        return device, n, index

    def execute(self, loss, lse, hidden, weight, targets, stream=None, workspace=None):
        """loss[t] and lse[t] (float32): the log of the sum of the exponentials of token t's logits, and that less its target's
        logit.  Zeros for tokens that take no part."""
        device, n, index = self._inputs(hidden, weight, targets)
        _tensor(loss, "loss", self._f32, (n,), device)
        _tensor(lse, "lse", self._f32, (n,), device)
        ws, size = _scratch(workspace, device)
        st = _lib.tc_vocab_loss_execute(self._h, loss.data_ptr(), lse.data_ptr(), hidden.data_ptr(), _ld(hidden), weight.data_ptr(), _ld(weight),
                                        targets.data_ptr(), index, n, ws, size, _stream(stream, targets))
        if st:
            _check(st, "tc_vocab_loss_execute")

    def execute_grad(self, dhidden, dweight, hidden, weight, targets, lse, grad, stream=None, workspace=None):
        """Gradients of sum_t grad[t] * loss[t] (grad, and lse as execute wrote it: float32) by hidden and by weight, in their
        type; either output may be None."""
        device, n, index = self._inputs(hidden, weight, targets)
        _tensor(lse, "lse", self._f32, (n,), device)
        _tensor(grad, "grad", self._f32, (n,), device)
        args = []
        for t, name, shape in ((dhidden, "dhidden", (n, self.dim)), (dweight, "dweight", self._table)):
            if t is not None:
                _tensor(t, name, self._types, shape, device)
            args += [None, self.dim] if t is None else [t.data_ptr(), _ld_out(t, name)]
        ws, size = _scratch(workspace, device)
        st = _lib.tc_vocab_loss_execute_grad(self._h, *args, hidden.data_ptr(), _ld(hidden), weight.data_ptr(), _ld(weight), targets.data_ptr(), index,
                                             lse.data_ptr(), grad.data_ptr(), n, ws, size, _stream(stream, targets))
        if st:
            _check(st, "tc_vocab_loss_execute_grad")


class OrthogonalPlan(_OpPlan):
    """Orthogonalised updates of `batch` matrices [rows, cols] by Newton-Schulz steps: x / (|x| + eps), then per step
    x <- a x + (b x x^T + c (x x^T)^2) x.  `coefficients`: (a, b, c), or one such triple per step.  Input BF16, F16 or F32, output
    BF16 or F16 (default: the input's type, BF16 for F32); F16 is within its own rounding of the exact result and takes about
    twice BF16's time."""

    def __init__(self, rows, cols, batch=1, dtype=BF16, out_dtype=None, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
        super().__init__()
        self.rows, self.cols, self.batch, self.dtype = rows, cols, batch, dtype
        self.out_dtype = (BF16 if dtype == F32 else dtype) if out_dtype is None else out_dtype
        triples = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else list(coefficients)
        if len(triples) != steps or any(len(t) != 3 for t in triples):
            raise ValueError("coefficients: three numbers, or three for each of the %d steps" % steps)
        flat = (ctypes.c_double * max(1, 3 * steps))(*[float(v) for t in triples for v in t])
        _check(lib().tc_op_create_orthogonal(batch, rows, cols, dtype, self.out_dtype, steps, flat, eps, ctypes.byref(self._h)),
               "tc_op_create_orthogonal")
        self._types, self._out_types, self._shape = _types(dtype), _types(self.out_dtype), (batch, rows, cols)

    def execute(self, out, x, stream=None, workspace=None):
        """out = the orthogonalised x; both [batch, rows, cols] (or [rows, cols] where batch is 1), with any strides."""
        if self.batch == 1:
            out, x = (t.unsqueeze(0) if getattr(t, "ndim", 0) == 2 else t for t in (out, x))
        device = _tensor(x, "x", self._types, self._shape, None)
        if device != self._device:
            self._on(device)
        _tensor(out, "out", self._out_types, self._shape, device)
        strides = [(ctypes.c_int64 * 3)(*t.stride()) for t in (out, x)]
        ws, size = _scratch(workspace, device)
        st = _lib.tc_orthogonal_execute(self._h, out.data_ptr(), strides[0], x.data_ptr(), strides[1], ws, size, _stream(stream, x))
        if st:
            _check(st, "tc_orthogonal_execute")


def sd_t_d2_fusion(expr, sizes, t3, t2, v2, dtype=F64):
    """The reference's generated entry for one expression: sizes in output-then-contraction order, numpy host arrays."""
    arr = (ctypes.c_int * len(sizes))(*[int(x) for x in sizes])
    _check(lib().tc_sd_t_d2_fusion(expr.encode(), dtype, len(sizes), arr, _ptr(t3), _ptr(t2), _ptr(v2)), "tc_sd_t_d2_fusion")


def fill_uniform(t, seed, tensor_id, first_index=0, stream=None):
    """Fills a CUDA tensor with the seeded uniform[-1,1) stream for (seed, tensor_id)."""
    import torch
    dt = F64 if t.dtype == torch.float64 else F32
    s = _stream(stream, t)
    _check(lib().tc_fill_uniform(_ptr(t), t.numel(), dt, seed, tensor_id, first_index, s), "tc_fill_uniform")
    return t


def axpy(y, x, alpha=1.0, stream=None):
    import torch
    dt = F64 if y.dtype == torch.float64 else F32
    s = _stream(stream, y)
    _check(lib().tc_axpy(_ptr(y), _ptr(x), y.numel(), dt, alpha, s), "tc_axpy")
    return y


_probes = None


def probes():
    """The bench-only probe library (pipe peaks, streaming read-modify-write); not part of the product ABI."""
    global _probes
    if _probes is None:
        if not os.path.exists(PROBES_PATH):
            raise ImportError("%s is missing: run build.py" % PROBES_PATH)
        h = ctypes.CDLL(PROBES_PATH)
        h.tc_peak_measure.restype = ctypes.c_int
        h.tc_peak_measure.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_double)]
        h.tc_peak_measure_rmw.restype = ctypes.c_int
        h.tc_peak_measure_rmw.argtypes = [ctypes.c_int64, ctypes.POINTER(ctypes.c_double)]
        _probes = h
    return _probes


def measure_peaks(which=(0, 4, 5), iters=4096, ctas_per_sm=2):
    """TFLOP/s of the arithmetic pipes (register-only loops; 7 = TF32 on tcgen05 from shared memory) on the current device."""
    out = {}
    for w in which:
        v = ctypes.c_double()
        _check(probes().tc_peak_measure(w, iters, ctas_per_sm, ctypes.byref(v)), "tc_peak_measure")
        out[PEAK_NAMES[w]] = v.value
    return out


def measure_rmw(nbytes=4 << 30):
    v = ctypes.c_double()
    _check(probes().tc_peak_measure_rmw(nbytes, ctypes.byref(v)), "tc_peak_measure_rmw")
    return v.value

"""ctypes binding of libadmm_hip.so (the C ABI declared in include/admm_hip.h).

Thin by design: every method is one C call.  There is no CPU implementation behind this module:
if the library is missing it raises at load time, and without a GPU the library's context
creation fails.
"""
import ctypes as C
import os
import struct

import numpy as np

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libadmm_hip.so")

# every symbol include/admm_hip.h declares
SYMBOLS = [
    "admm_last_error", "admm_abi_version", "admm_device_count", "admm_ctx_create", "admm_ctx_destroy", "admm_sync",
    "admm_timing_enable", "admm_timing_classes", "admm_timing_every", "admm_timing_reset", "admm_timing_get",
    "admm_vec_alloc", "admm_scratch_alloc", "admm_vec_free", "admm_vec_zero", "admm_vec_copy", "admm_vec_upload",
    "admm_vec_download",
    "admm_csr_upload", "admm_csr_synth", "admm_csr_shape", "admm_csr_download",
    "admm_csr_build_transposed", "admm_csr_relabel_by_frequency", "admm_csr_set_lean", "admm_synth_row_draws", "admm_csr_bytes", "admm_csr_layout_bytes", "admm_csr_layout_counts",
    "admm_csr_destroy",
    "admm_predict", "admm_metrics", "admm_auc_scores", "admm_tied_ranks", "admm_csr_copy_labels", "admm_ftrl_pass", "admm_ftrl_predict", "admm_ftrl_update", "admm_ftrl_pass_multi", "admm_logistic_fg", "admm_lbfgs_solve",
    "admm_payload", "admm_global_update", "admm_dual_update", "admm_consensus", "admm_consensus_static",
    "admm_comm_unique_id", "admm_comm_init", "admm_allreduce_sum_f32", "admm_comm_selftest",
    "admm_csr_bags", "admm_embed", "admm_embed_order_bytes", "admm_embed_order", "admm_embed_grad_workspace", "admm_embed_grad",
    "admm_softmax_loss_workspace", "admm_softmax_loss", "admm_sample_workspace", "admm_sample",
]

K_FORWARD, K_TRANSPOSED, K_FTRL_SEQ, K_ELEMENTWISE, K_FORWARD_EVAL, K_EMBED, K_SOFTMAX, K_SAMPLE = range(8)

# element types of matrices, ids and labels
F32, BF16, F16, I32, I64 = range(5)
_BYTES = (4, 2, 2, 4, 8)
# a context's stream: the device's default stream (None lets the library make one of its own)
DEFAULT_STREAM = 1


class AdmmError(RuntimeError):
    pass


class SynthSpec(C.Structure):
    _fields_ = [("nrows", C.c_uint64), ("dim", C.c_uint64), ("seed", C.c_uint64),
                ("model_seed", C.c_uint64), ("row_offset", C.c_uint64), ("mean_nnz", C.c_float), ("zipf_s", C.c_float),
                ("len_dist", C.c_int), ("tail_sigma", C.c_float), ("max_len", C.c_uint32),
                ("explicit_values", C.c_int)]


class LbfgsParams(C.Structure):
    _fields_ = [("m", C.c_int), ("max_iter", C.c_int), ("max_linesearch", C.c_int),
                ("epsilon", C.c_float), ("ftol", C.c_float), ("wolfe", C.c_float), ("linesearch", C.c_int)]


class LbfgsResult(C.Structure):
    _fields_ = [("f", C.c_double), ("evals", C.c_int), ("iters", C.c_int),
                ("forward_sweeps", C.c_int), ("transposed_sweeps", C.c_int)]


class MatStruct(C.Structure):
    _fields_ = [("data", C.c_void_p), ("rows", C.c_uint64), ("cols", C.c_uint64), ("stride", C.c_uint64), ("type", C.c_int)]


class BagsStruct(C.Structure):
    _fields_ = [("ids", C.c_void_p), ("rowptr", C.c_void_p), ("val", C.c_void_p), ("nrows", C.c_uint64),
                ("nnz", C.c_uint64), ("id_type", C.c_int)]


class SampleParamsStruct(C.Structure):
    _fields_ = [("temperature", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p), ("min_p", C.c_void_p)]


_lib = None


def load():
    """Load libadmm_hip.so; fails loudly when it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise AdmmError("%s not found: build it with `python -m admm_amd.build` "
                        "(there is no fallback implementation)" % LIB_PATH)
    L = C.CDLL(LIB_PATH)
    vp, u64, f32, i32 = C.c_void_p, C.c_uint64, C.c_float, C.c_int
    L.admm_last_error.restype = C.c_char_p
    L.admm_last_error.argtypes = []
    L.admm_abi_version.restype = i32
    sig = {
        "admm_device_count": [C.POINTER(i32)],
        "admm_ctx_create": [i32, vp, C.POINTER(vp)],
        "admm_ctx_destroy": [vp],
        "admm_sync": [vp],
        "admm_timing_enable": [vp, i32],
        "admm_timing_classes": [vp, C.c_uint32],
        "admm_timing_every": [vp, C.c_uint32],
        "admm_timing_reset": [vp],
        "admm_timing_get": [vp, i32, C.POINTER(C.c_double), C.POINTER(u64)],
        "admm_vec_alloc": [vp, u64, C.POINTER(vp)],
        "admm_scratch_alloc": [vp, u64, C.POINTER(vp)],
        "admm_vec_free": [vp, vp],
        "admm_vec_zero": [vp, vp, u64],
        "admm_vec_copy": [vp, vp, vp, u64],
        "admm_vec_upload": [vp, vp, vp, u64],
        "admm_vec_download": [vp, vp, vp, u64],
        "admm_csr_upload": [vp, vp, vp, vp, vp, u64, u64, u64, i32, C.POINTER(vp)],
        "admm_csr_synth": [vp, C.POINTER(SynthSpec), C.POINTER(vp)],
        "admm_csr_shape": [vp, C.POINTER(u64), C.POINTER(u64), C.POINTER(u64)],
        "admm_csr_download": [vp, vp, vp, vp, vp],
        "admm_csr_build_transposed": [vp, u64, C.c_uint32],
        "admm_csr_relabel_by_frequency": [vp],
        "admm_csr_bytes": [vp, C.POINTER(u64), C.POINTER(u64)],
        "admm_csr_set_lean": [vp, i32],
        "admm_synth_row_draws": [vp, vp, u64, C.POINTER(u64)],
        "admm_csr_layout_bytes": [vp, C.POINTER(u64)],
        "admm_csr_layout_counts": [vp, C.POINTER(u64)],
        "admm_csr_destroy": [vp],
        "admm_predict": [vp, C.POINTER(vp), i32, vp],
        "admm_metrics": [vp, C.POINTER(vp), i32, C.POINTER(C.c_double), C.POINTER(C.c_double),
                         C.POINTER(u64)],
        "admm_auc_scores": [vp, vp, vp, u64, C.POINTER(C.c_double)],
        "admm_tied_ranks": [vp, vp, u64, vp],
        "admm_csr_copy_labels": [vp, vp],
        "admm_ftrl_pass": [vp, vp, vp, vp, vp, vp, f32, f32, f32, f32, u64],
        "admm_ftrl_pass_multi": [vp, vp, vp, vp, vp, vp, C.c_int, f32, f32, f32, f32],
        "admm_ftrl_predict": [vp, vp, vp, C.c_uint32, vp, vp, vp, vp, vp, f32, f32, f32, f32, C.POINTER(C.c_float)],
        "admm_ftrl_update": [vp, vp, C.c_uint32, f32, f32, vp, vp, vp, f32],
        "admm_logistic_fg": [vp, vp, vp, vp, vp, f32, C.POINTER(C.c_double), vp],
        "admm_lbfgs_solve": [vp, vp, vp, vp, vp, f32, C.POINTER(LbfgsParams),
                             C.POINTER(LbfgsResult)],
        "admm_payload": [vp, vp, vp, f32, vp, u64],
        "admm_global_update": [vp, vp, i32, f32, f32, f32, vp, u64],
        "admm_dual_update": [vp, vp, vp, vp, f32, u64],
        "admm_consensus": [vp, vp, i32, f32, f32, f32, vp, vp, vp, u64, C.POINTER(C.c_double),
                           C.POINTER(C.c_double)],
        "admm_consensus_static": [vp, vp, i32, f32, f32, f32, vp, vp, vp, u64, vp],
        "admm_comm_unique_id": [vp],
        "admm_comm_init": [vp, i32, i32, vp],
        "admm_allreduce_sum_f32": [vp, vp, u64],
        "admm_comm_selftest": [vp],
        "admm_csr_bags": [vp, vp],
        "admm_embed": [vp, vp, vp, f32, vp],
        "admm_embed_order_bytes": [vp, u64, C.POINTER(u64)],
        "admm_embed_order": [vp, vp, u64, vp, u64],
        "admm_embed_grad_workspace": [vp, u64, C.POINTER(u64)],
        "admm_embed_grad": [vp, vp, vp, u64, vp, f32, i32, vp, vp, u64],
        "admm_softmax_loss_workspace": [u64, u64, C.POINTER(u64)],
        "admm_softmax_loss": [vp, vp, vp, i32, vp, f32, vp, vp, vp, vp, u64],
        "admm_sample_workspace": [u64, u64, C.POINTER(u64)],
        "admm_sample": [vp, vp, vp, vp, vp, vp, vp, u64],
    }
    for name, args in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = i32
    _lib = L
    return L


def _check(rc):
    if rc:
        raise AdmmError("libadmm_hip error %d: %s" % (rc, load().admm_last_error().decode()))


def _ptr(a):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


class DeviceVec:
    """dim floats in HBM."""

    def __init__(self, ctx, n):
        self.ctx, self.n = ctx, int(n)
        p = C.c_void_p()
        _check(ctx.L.admm_vec_alloc(ctx.h, self.n, C.byref(p)))
        self.ptr = p

    @classmethod
    def from_ptr(cls, ctx, ptr, n):
        """Wrap device memory owned by someone else (e.g. a torch tensor's data_ptr)."""
        v = cls.__new__(cls)
        v.ctx, v.n, v.ptr, v.borrowed = ctx, int(n), C.c_void_p(int(ptr)), True
        return v

    def upload(self, host):
        host = np.ascontiguousarray(host, np.float32)
        assert host.shape == (self.n,)
        _check(self.ctx.L.admm_vec_upload(self.ctx.h, self.ptr, _ptr(host), self.n))
        return self

    def download(self):
        out = np.empty(self.n, np.float32)
        _check(self.ctx.L.admm_vec_download(self.ctx.h, _ptr(out), self.ptr, self.n))
        return out

    def zero(self):
        _check(self.ctx.L.admm_vec_zero(self.ctx.h, self.ptr, self.n))
        return self

    def copy_from(self, other):
        _check(self.ctx.L.admm_vec_copy(self.ctx.h, self.ptr, other.ptr, self.n))
        return self

    def free(self):
        if getattr(self, "borrowed", False):
            self.ptr = None
        if self.ptr:
            _check(self.ctx.L.admm_vec_free(self.ctx.h, self.ptr))
            self.ptr = None


class DeviceBuf:
    """bytes in HBM (workspaces, orders, integer arrays); `type`: what elements they are (I32, I64, F32), where a call could take
    several for them"""

    type = None

    def __init__(self, ctx, nbytes, type=None):
        if type is not None and type not in range(len(_BYTES)):
            raise AdmmError("a buffer of elements of type %s" % (type,))
        self.vec = DeviceVec(ctx, max(1, (int(nbytes) + 3) // 4))
        self.nbytes, self.type = int(nbytes), type
        self.ptr = self.vec.ptr

    @classmethod
    def scratch(cls, ctx, nbytes):
        """of any contents; the calling thread's current device stays what it is (admm_scratch_alloc)"""
        b, v = cls.__new__(cls), DeviceVec.__new__(DeviceVec)
        b.nbytes = max(4, int(nbytes))
        p = C.c_void_p()
        _check(ctx.L.admm_scratch_alloc(ctx.h, b.nbytes, C.byref(p)))
        v.ctx, v.n, v.ptr = ctx, b.nbytes // 4, p
        b.vec, b.ptr = v, p
        return b

    def free(self):
        self.vec.free()
        self.ptr = None


class _Types(dict):
    """torch's element types to the library's; filled at the first look, so that this module does not need torch"""

    def __init__(self, *kinds):
        super().__init__()
        self.kinds = kinds

    def __missing__(self, dtype):
        import torch
        names = {"float32": F32, "bfloat16": BF16, "float16": F16, "int32": I32, "uint32": I32, "int64": I64, "uint64": I64}
        self.update({getattr(torch, n): k for n, k in names.items() if k in self.kinds and hasattr(torch, n)})
        if dtype not in self:
            raise KeyError(dtype)
        return self[dtype]


_FLOATS, _ARRAYS = _Types(F32, BF16, F16), _Types(F32, I32, I64)


# admm_mat and admm_bags as bytes, which a void pointer argument takes as they are: making a ctypes structure costs as much
# as the call itself
_MAT = struct.Struct("PQQQi4x").pack
_BAGS = struct.Struct("PPPQQi4x").pack


class DeviceMat:
    """A row-major matrix in HBM (admm_mat): from a pointer (`device`: the GPU it lies on, if calls are to check that), or `of` a
    torch tensor on the context's GPU"""

    __slots__ = ("rows", "cols", "packed", "device")

    def __init__(self, ptr, rows, cols, type=F32, stride=None, device=None):
        self.rows, self.cols, self.device = rows, cols, device
        self.packed = _MAT(ptr, rows, cols, cols if stride is None else stride, type)

    @classmethod
    def of(cls, ctx, m, name):
        if isinstance(m, DeviceMat):
            if m.device is not None and m.device != ctx.device:
                raise ctx._not_here(name, m.device)
            return m
        try:
            (rows, cols), (step, inner), kind = m.shape, m.stride(), _FLOATS[m.dtype]
        except Exception:
            raise _not_a_matrix(m, name) from None
        if m.get_device() != ctx.device:
            raise ctx._elsewhere(m, name)
        if inner != 1 and cols > 1:
            raise AdmmError("%s: the elements of a row lie %d apart: they have to be adjacent" % (name, inner))
        if step < cols:
            if rows > 1:
                raise AdmmError("%s: rows of %d elements lie %d apart" % (name, cols, step))
            step = cols
        return cls(m.data_ptr(), rows, cols, kind, step, ctx.device)


def _not_a_matrix(m, name):
    if not hasattr(m, "data_ptr"):
        return AdmmError("%s: a DeviceMat or a torch tensor is needed, not %s" % (name, m.__class__.__name__))
    if m.dim() != 2:
        return AdmmError("%s: a matrix is needed, not %d dimensions" % (name, m.dim()))
    return AdmmError("%s: float32, bfloat16 or float16 is needed, not %s" % (name, m.dtype))


class Bags:
    """Rows of ids (admm_bags); keeps the arrays alive, but for those of a sample set (`source`), which are asked for again at
    every call that reads them.  `device`: the GPU they lie on, where that is known"""

    __slots__ = ("nrows", "nnz", "keep", "packed", "source", "device")

    def __init__(self, ids, rowptr, val, nrows, nnz, id_type, keep=(), source=None, device=None):
        self.nrows, self.nnz, self.keep, self.source, self.device = nrows, nnz, keep, source, device
        self.packed = _BAGS(ids or 0, rowptr or 0, val or 0, nrows, nnz, id_type)


class Context:
    def __init__(self, device=0, stream=None):
        self.L = load()
        self.device = int(device)
        self._scratch, self._retired = None, []
        self._size = C.c_uint64()
        self._size_ref = C.byref(self._size)
        h = C.c_void_p()
        _check(self.L.admm_ctx_create(int(device), C.c_void_p(stream) if stream else None,
                                      C.byref(h)))
        self.h = h
        self.rank, self.world = 0, 1
        self.exchange = None

    def close(self):
        if self.h:
            for b in self._retired + ([self._scratch] if self._scratch is not None else []):
                b.free()
            self._scratch, self._retired = None, []
            self.L.admm_ctx_destroy(self.h)
            self.h = None

    def sync(self):
        _check(self.L.admm_sync(self.h))

    def vec(self, n, host=None):
        v = DeviceVec(self, n)
        if host is not None:
            v.upload(host)
        return v

    # timing -------------------------------------------------------------------------------
    def timing_enable(self, on=True, classes=None, every=1):
        """HIP-event timing of the library's kernels; `classes` (a list of K_* ids) restricts it, and of
        each class every `every`-th launch is timed"""
        mask = 0xFFFFFFFF if classes is None else sum(1 << k for k in classes)
        _check(self.L.admm_timing_classes(self.h, mask))
        _check(self.L.admm_timing_every(self.h, max(1, int(every))))
        _check(self.L.admm_timing_enable(self.h, 1 if on else 0))

    def timing_reset(self):
        _check(self.L.admm_timing_reset(self.h))

    def timing_get(self, kernel):
        ms, cnt = C.c_double(), C.c_uint64()
        _check(self.L.admm_timing_get(self.h, kernel, C.byref(ms), C.byref(cnt)))
        return ms.value, cnt.value

    # sample sets --------------------------------------------------------------------------
    def csr_upload(self, rowptr, col, val, label, dim, add_bias=True):
        rowptr = np.ascontiguousarray(rowptr, np.uint64)
        col = np.ascontiguousarray(col, np.uint32)
        val = None if val is None else np.ascontiguousarray(val, np.float32)
        label = np.ascontiguousarray(label, np.float32)
        nrows = rowptr.shape[0] - 1
        nnz = int(rowptr[-1])
        h = C.c_void_p()
        _check(self.L.admm_csr_upload(self.h, _ptr(rowptr), _ptr(col), _ptr(val), _ptr(label),
                                      nrows, nnz, int(dim), 1 if add_bias else 0, C.byref(h)))
        return SampleSet(self, h)

    def csr_synth(self, nrows, dim, mean_nnz, seed=20251111, row_offset=0, zipf_s=1.1,
                  len_dist=0, tail_sigma=1.0, max_len=None, model_seed=7, explicit_values=False):
        if max_len is None:
            max_len = int(min(1024, max(8, 4 * mean_nnz)))
        spec = SynthSpec(int(nrows), int(dim), int(seed), int(model_seed), int(row_offset), float(mean_nnz),
                         float(zipf_s), int(len_dist), float(tail_sigma), int(max_len),
                         1 if explicit_values else 0)
        h = C.c_void_p()
        _check(self.L.admm_csr_synth(self.h, C.byref(spec), C.byref(h)))
        return SampleSet(self, h)

    def synth_row_draws(self, nrows, dim, mean_nnz, block_rows, seed=20251111, row_offset=0, zipf_s=1.1, len_dist=0,
                        tail_sigma=1.0, max_len=None, model_seed=7, explicit_values=False):
        """entries the generator draws per block of block_rows rows (bias entry included), as a numpy array"""
        if max_len is None:
            max_len = int(min(1024, max(8, 4 * mean_nnz)))
        spec = SynthSpec(int(nrows), int(dim), int(seed), int(model_seed), int(row_offset), float(mean_nnz),
                         float(zipf_s), int(len_dist), float(tail_sigma), int(max_len), 1 if explicit_values else 0)
        nblocks = (int(nrows) + int(block_rows) - 1) // int(block_rows)
        out = np.zeros(max(nblocks, 1), np.uint64)
        _check(self.L.admm_synth_row_draws(self.h, C.byref(spec), int(block_rows), out.ctypes.data_as(C.POINTER(C.c_uint64))))
        return out[:nblocks]

    def ftrl_pass_multi(self, sets, w, z, n, offset, reg_offset, alpha, beta, l_1, l_2):
        """admm_ftrl_pass_multi: pass k runs sets[k] with state w[k], z[k], n[k]"""
        cnt = len(sets)
        assert all(len(v) == cnt for v in (w, z, n, offset, reg_offset))
        def arr(items, get):
            return (C.c_void_p * cnt)(*[getattr(get(i), "value", get(i)) for i in items])
        _check(self.L.admm_ftrl_pass_multi(arr(sets, lambda s: s.h), arr(w, lambda v: v.ptr), arr(z, lambda v: v.ptr),
                                           arr(n, lambda v: v.ptr), arr(offset, lambda v: v.ptr),
                                           arr(reg_offset, lambda v: v.ptr), cnt, alpha, beta, l_1, l_2))

    def ftrl_predict(self, index, value, w, z, n, offset, reg_offset, alpha, beta, l_1, l_2):
        """FtrlSolver::Predict (src/ftrl.cc:54-73) on one translated row held in host arrays (value None: all
        ones): refreshes w at the row's coordinates and returns P(y = 1)"""
        idx = np.ascontiguousarray(index, np.uint32)
        val = None if value is None else np.ascontiguousarray(value, np.float32)
        p = C.c_float()
        _check(self.L.admm_ftrl_predict(self.h, _ptr(idx), None if val is None else _ptr(val), idx.shape[0], w.ptr,
                                        z.ptr, n.ptr, offset.ptr, reg_offset.ptr, alpha, beta, l_1, l_2, C.byref(p)))
        return float(p.value)

    def ftrl_update(self, index, label, predict, w, z, n, alpha):
        """FtrlSolver::Update (src/ftrl.cc:75-88) on the same row"""
        idx = np.ascontiguousarray(index, np.uint32)
        _check(self.L.admm_ftrl_update(self.h, _ptr(idx), idx.shape[0], float(label), float(predict), w.ptr, z.ptr,
                                       n.ptr, alpha))

    # models with many classes or tokens -----------------------------------------------------
    # Matrices are torch tensors or DeviceMats, arrays are torch tensors, DeviceVecs (floats) or DeviceBufs (labels in one
    # need its type: buf(bytes, type=I64)); what they point to belongs to this context's GPU, and the work is queued on this
    # context's stream (make the context on the stream that the tensors are used on:
    # Context(device, stream=torch.cuda.current_stream().cuda_stream or DEFAULT_STREAM)).
    def _elsewhere(self, t, name):
        return AdmmError("%s is on %s, the context on GPU %d" % (name, t.device, self.device))

    def _not_here(self, name, device):
        return AdmmError("%s is on GPU %d, the context on GPU %d" % (name, device, self.device))

    def _array(self, a, name, count, kinds):
        """(pointer, type) of `count` adjacent elements of one of the types"""
        if a is None:
            return None, kinds[0]
        if hasattr(a, "data_ptr"):
            kind = _ARRAYS.get(a.dtype)
            if kind is None:
                try:
                    kind = _ARRAYS[a.dtype]
                except KeyError:
                    pass
            if kind not in kinds:
                raise AdmmError("%s: elements of type %s" % (name, a.dtype))
            if a.get_device() != self.device:
                raise self._elsewhere(a, name)
            if a.numel() < count or not a.is_contiguous():
                raise AdmmError("%s: %d adjacent elements are needed, it has %s with strides %s" %
                                (name, count, tuple(a.shape), tuple(a.stride())))
            return a.data_ptr(), kind
        if isinstance(a, DeviceVec):
            if F32 not in kinds or a.n < count:
                raise AdmmError("%s: %d floats do not do for %d elements" % (name, a.n, count))
            if a.ctx.device != self.device:
                raise self._not_here(name, a.ctx.device)
            if not a.ptr and count:
                raise AdmmError("%s was freed" % name)
            return a.ptr, F32
        if isinstance(a, DeviceBuf):
            if a.vec.ctx.device != self.device:
                raise self._not_here(name, a.vec.ctx.device)
            if not a.ptr:
                raise AdmmError("%s was freed" % name)
            kind = kinds[0] if a.type is None and len(kinds) == 1 else a.type
            if kind not in kinds:
                raise AdmmError("%s: %s" % (name, "a buffer that does not say its elements' type (buf(bytes, type=...))" if kind is None
                                            else "elements of type %d" % kind))
            if a.nbytes < count * _BYTES[kind]:
                raise AdmmError("%s: %d bytes do not do for %d elements" % (name, a.nbytes, count))
            return a.ptr, kind
        raise AdmmError("%s: a torch tensor, a DeviceVec or a DeviceBuf is needed, not %s" % (name, a.__class__.__name__))

    def _bytes(self, buf, name):
        if isinstance(buf, DeviceBuf):
            if buf.vec.ctx.device != self.device:
                raise self._not_here(name, buf.vec.ctx.device)
            if not buf.ptr:
                raise AdmmError("%s was freed" % name)
            return buf.ptr, buf.nbytes
        if not hasattr(buf, "data_ptr"):
            raise AdmmError("%s: a DeviceBuf or a torch tensor is needed, not %s" % (name, buf.__class__.__name__))
        if buf.get_device() != self.device:
            raise self._elsewhere(buf, name)
        if not buf.is_contiguous():
            raise AdmmError("%s: not contiguous" % name)
        return buf.data_ptr(), buf.nbytes

    def _workspace(self, given, size, *shape):
        """the caller's workspace, or one that the context keeps for calls without: it grows, and what it outgrew stays until
        close(), for graphs that were captured with it"""
        if given is not None:
            return self._bytes(given, "workspace")
        _check(size(*shape, self._size_ref))
        need = self._size.value
        if need == 0:
            return None, 0
        if self._scratch is None or self._scratch.nbytes < need:
            larger = DeviceBuf.scratch(self, (need + (need >> 2) + 4095) // 4096 * 4096)
            if self._scratch is not None:
                self._retired.append(self._scratch)
            self._scratch = larger
        return self._scratch.ptr, self._scratch.nbytes

    def buf(self, nbytes, type=None):
        return DeviceBuf(self, nbytes, type)

    def bags(self, ids, rowptr=None, val=None):
        """Rows of ids for embed / embed_grad: one per row, or with row pointers (nrows + 1 int64) and factors"""
        if not hasattr(ids, "data_ptr"):
            raise AdmmError("ids: a torch tensor is needed")
        nnz = ids.numel()
        p, kind = self._array(ids, "ids", nnz, (I32, I64))
        nrows, q, f = nnz, None, None
        if rowptr is not None:
            if not hasattr(rowptr, "data_ptr"):
                raise AdmmError("rowptr: a torch tensor is needed")
            nrows = rowptr.numel() - 1
            if nrows < 0:
                raise AdmmError("rowptr: no element")
            q, _ = self._array(rowptr, "rowptr", nrows + 1, (I64,))
        if val is not None:
            f, _ = self._array(val, "val", nnz, (F32,))
        return Bags(p, q, f, nrows, nnz, kind, (ids, rowptr, val), None, self.device)

    def _bags(self, bags, read=True):
        """what the library is told of the bags; `read`: it reads their arrays, not the counts alone"""
        if not isinstance(bags, Bags):
            raise AdmmError("bags: Context.bags() or SampleSet.bags() makes them, not %s" % bags.__class__.__name__)
        if bags.device != self.device and bags.device is not None:
            raise self._not_here("bags", bags.device)
        return bags.source._rows() if read and bags.source is not None else bags.packed

    def embed(self, bags, table, out, scale=1.0):
        """admm_embed: out[r] = scale * sum of val_e * table[id_e] over the entries of row r"""
        _check(self.L.admm_embed(self.h, self._bags(bags), DeviceMat.of(self, table, "table").packed, scale, DeviceMat.of(self, out, "out").packed))

    def embed_order_bytes(self, bags, table_rows):
        _check(self.L.admm_embed_order_bytes(self._bags(bags, False), int(table_rows), self._size_ref))
        return self._size.value

    def embed_order(self, bags, table_rows, order=None):
        """admm_embed_order: the entries sorted by id, into `order` (a DeviceBuf or a torch tensor of bytes; made if None, and then
        the caller's to free())"""
        rows = self._bags(bags)
        if order is None:
            order = DeviceBuf.scratch(self, self.embed_order_bytes(bags, table_rows))
        p, n = self._bytes(order, "order")
        _check(self.L.admm_embed_order(self.h, rows, int(table_rows), p, n))
        return order

    def embed_grad(self, bags, order, grad_out, grad_table, scale=1.0, accumulate=False, workspace=None):
        """admm_embed_grad: the gradient with respect to the table, written whole or added to"""
        src, to = DeviceMat.of(self, grad_out, "grad_out"), DeviceMat.of(self, grad_table, "grad_table")
        counts = self._bags(bags, False)
        p, n = self._bytes(order, "order")
        w, wn = self._workspace(workspace, self.L.admm_embed_grad_workspace, counts, src.cols)
        _check(self.L.admm_embed_grad(self.h, counts, p, n, src.packed, scale, 1 if accumulate else 0, to.packed, w, wn))

    def softmax_loss(self, logits, labels, loss, grad=None, lse=None, weight=None, grad_scale=1.0, workspace=None):
        """admm_softmax_loss: loss per row, and with `grad` (may be the logits) grad_scale times its gradient"""
        x = DeviceMat.of(self, logits, "logits")
        g = None if grad is None else DeviceMat.of(self, grad, "grad")
        rows = x.rows
        t, kind = self._array(labels, "labels", rows, (I32, I64, F32))
        w, _ = self._array(weight, "weight", rows, (F32,))
        o, _ = self._array(loss, "loss", rows, (F32,))
        e, _ = self._array(lse, "lse", rows, (F32,))
        ws, wn = self._workspace(workspace, self.L.admm_softmax_loss_workspace, rows, x.cols)
        _check(self.L.admm_softmax_loss(self.h, x.packed, t, kind, w, grad_scale, o, e, None if g is None else g.packed, ws, wn))

    def sample(self, logits, uniform, token, logprob=None, temperature=None, top_k=None, top_p=None, min_p=None, workspace=None):
        """admm_sample: a class per row into `token` (int32), the log of its probability into `logprob`"""
        x = DeviceMat.of(self, logits, "logits")
        rows = x.rows
        u, _ = self._array(uniform, "uniform", rows, (F32,))
        t, _ = self._array(token, "token", rows, (I32,))
        lp, _ = self._array(logprob, "logprob", rows, (F32,))
        f, _ = self._array(temperature, "temperature", rows, (F32,))
        k, _ = self._array(top_k, "top_k", rows, (I32,))
        p, _ = self._array(top_p, "top_p", rows, (F32,))
        m, _ = self._array(min_p, "min_p", rows, (F32,))
        params = SampleParamsStruct(f, k, p, m)
        ws, wn = self._workspace(workspace, self.L.admm_sample_workspace, rows, x.cols)
        _check(self.L.admm_sample(self.h, x.packed, C.byref(params), u, t, lp, ws, wn))

    # consensus algebra --------------------------------------------------------------------
    def payload(self, x, ydual, rho, out):
        _check(self.L.admm_payload(self.h, x.ptr, ydual.ptr, rho, out.ptr, x.n))

    def global_update(self, total, num_worker, rho, global_var, l1, z):
        _check(self.L.admm_global_update(self.h, total.ptr, num_worker, rho, global_var, l1,
                                         z.ptr, z.n))

    def dual_update(self, ydual, x, z, rho):
        _check(self.L.admm_dual_update(self.h, ydual.ptr, x.ptr, z.ptr, rho, x.n))

    def tied_ranks(self, scores, ranks, n=None):
        """Metrics::Sort (src/metrics.cc:14-46) of a device vector of scores into a device vector of ranks"""
        _check(self.L.admm_tied_ranks(self.h, scores.ptr, scores.n if n is None else int(n), ranks.ptr))

    def auc_scores(self, scores, labels, n):
        """tie-aware rank-sum AUC (src/metrics.cc:14-89) of n (score, label) pairs held in device vectors"""
        auc = C.c_double()
        _check(self.L.admm_auc_scores(self.h, scores.ptr, labels.ptr, int(n), C.byref(auc)))
        return auc.value

    def consensus(self, total, num_worker, rho, global_var, l1, x, ydual, z, want_residuals=True):
        r2, s2 = C.c_double(), C.c_double()
        _check(self.L.admm_consensus(self.h, total.ptr, num_worker, rho, global_var, l1, x.ptr,
                                     ydual.ptr, z.ptr, x.n,
                                     C.byref(r2) if want_residuals else None,
                                     C.byref(s2) if want_residuals else None))
        return (r2.value, s2.value) if want_residuals else None

    def consensus_static(self, total, num_worker, rho, global_var, l1, x, ydual, z, residuals=None, stream=None,
                         dim=None):
        """admm_consensus_static: the same step without a context, a host wait or an allocation, on `stream`
        (raw hipStream_t value, None = the default stream) of the current device; `residuals` is a device
        buffer of two doubles or None"""
        _check(self.L.admm_consensus_static(C.c_void_p(stream) if stream else None, total.ptr, num_worker, rho,
                                            global_var, l1, x.ptr, ydual.ptr, z.ptr, x.n if dim is None else int(dim),
                                            residuals.ptr if residuals is not None else None))

    def allreduce_sum(self, buf, n=None):
        """rabit::Allreduce<op::Sum> (src/admm_allreduce.cpp:69): in-place float sum over ranks on RCCL.
        `exchange` (set by a rehearsal in which several ranks share one GPU, where RCCL cannot run)
        replaces the library call by a caller-supplied function of (vector, count)."""
        cnt = buf.n if n is None else int(n)
        if self.exchange is not None:
            return self.exchange(buf, cnt)
        _check(self.L.admm_allreduce_sum_f32(self.h, buf.ptr, cnt))

    def comm_unique_id(self):
        """128 bytes that rank 0 hands to every rank (admm_comm_unique_id)"""
        buf = C.create_string_buffer(128)
        _check(self.L.admm_comm_unique_id(buf))
        return buf.raw

    def comm_init(self, rank, world, unique_id=None):
        self.rank, self.world = int(rank), int(world)
        _check(self.L.admm_comm_init(self.h, self.rank, self.world,
                                     C.create_string_buffer(unique_id, 128) if unique_id else None))

    def comm_selftest(self):
        _check(self.L.admm_comm_selftest(self.h))


class SampleSet:
    """One sample set resident in HBM (CSR, optionally with its column-block copy)."""

    def __init__(self, ctx, handle):
        self.ctx, self.h = ctx, handle
        a, b, c = C.c_uint64(), C.c_uint64(), C.c_uint64()
        _check(ctx.L.admm_csr_shape(self.h, C.byref(a), C.byref(b), C.byref(c)))
        self.nrows, self.nnz, self.dim = a.value, b.value, c.value
        self._bags = BagsStruct()
        self._bags_ref = C.byref(self._bags)

    def destroy(self):
        if self.h:
            self.ctx.L.admm_csr_destroy(self.h)
            self.h = None

    def download(self):
        rowptr = np.empty(self.nrows + 1, np.uint64)
        col = np.empty(max(self.nnz, 1), np.uint32)
        val = np.empty(max(self.nnz, 1), np.float32)
        label = np.empty(max(self.nrows, 1), np.float32)
        _check(self.ctx.L.admm_csr_download(self.h, _ptr(rowptr), _ptr(col), _ptr(val),
                                            _ptr(label)))
        return rowptr, col[:self.nnz], val[:self.nnz], label[:self.nrows]

    def _rows(self):
        """what admm_csr_bags says now, as a pointer to it"""
        if not self.h:
            raise AdmmError("bags: the sample set was destroyed")
        _check(self.ctx.L.admm_csr_bags(self.h, self._bags_ref))
        return self._bags_ref

    def bags(self):
        """the set's rows as bags for Context.embed / embed_grad (admm_csr_bags).  They are the set's arrays: once it is destroyed,
        relabelled, or lean and without its rows, calls that read them are refused (embed_grad takes only counts from them)"""
        self._rows()
        b = self._bags
        return Bags(b.ids, b.rowptr, b.val, b.nrows, b.nnz, b.id_type, source=self, device=self.ctx.device)

    def build_transposed(self, panel_rows=0, col_block=0):
        _check(self.ctx.L.admm_csr_build_transposed(self.h, int(panel_rows), int(col_block)))
        return self

    def set_lean(self, on=True):
        """whole-set sweeps only from here on: the builders free the row-major forms once their copies exist"""
        _check(self.ctx.L.admm_csr_set_lean(self.h, 1 if on else 0))
        return self

    def relabel_by_frequency(self):
        _check(self.ctx.L.admm_csr_relabel_by_frequency(self.h))
        return self

    def bytes(self):
        a, b = C.c_uint64(), C.c_uint64()
        _check(self.ctx.L.admm_csr_bytes(self.h, C.byref(a), C.byref(b)))
        return a.value, b.value

    def layout_bytes(self):
        """dict of HBM bytes by layout: row_major, forward_form, column_block_copy, row_vectors"""
        out = (C.c_uint64 * 4)()
        _check(self.ctx.L.admm_csr_layout_bytes(self.h, out))
        return dict(zip(("row_major", "forward_form", "column_block_copy", "row_vectors"), [int(v) for v in out]))

    def layout_counts(self):
        """dict of entry counts by layout (admm_csr_layout_counts)"""
        out = (C.c_uint64 * 6)()
        _check(self.ctx.L.admm_csr_layout_counts(self.h, out))
        return dict(zip(("mask_entries", "hot_stream_words", "list_entries", "column_stream_words", "cell_entries",
                         "cells"), [int(v) for v in out]))

    def _groups(self, groups):
        arr = (C.c_void_p * len(groups))(*[g.ptr.value for g in groups])
        return C.cast(arr, C.POINTER(C.c_void_p)), len(groups)

    def predict_into(self, groups, out):
        """per-row P(y=1|x) into a device vector of at least nrows floats"""
        arr, k = self._groups(groups)
        _check(self.ctx.L.admm_predict(self.h, arr, k, out.ptr))

    def copy_labels(self, out):
        _check(self.ctx.L.admm_csr_copy_labels(self.h, out.ptr))

    def predict(self, groups):
        out = DeviceVec(self.ctx, max(self.nrows, 1))
        arr, k = self._groups(groups)
        _check(self.ctx.L.admm_predict(self.h, arr, k, out.ptr))
        p = out.download()[:self.nrows]
        out.free()
        return p

    def metrics(self, groups, want_auc=True):
        arr, k = self._groups(groups)
        ll, auc, n = C.c_double(), C.c_double(), C.c_uint64()
        _check(self.ctx.L.admm_metrics(self.h, arr, k, C.byref(ll),
                                       C.byref(auc) if want_auc else None, C.byref(n)))
        return ll.value, (auc.value if want_auc else None), n.value

    def ftrl_pass(self, w, z, n, offset, reg_offset, alpha, beta, l1, l2, batch=1):
        _check(self.ctx.L.admm_ftrl_pass(self.h, w.ptr, z.ptr, n.ptr, offset.ptr, reg_offset.ptr,
                                         alpha, beta, l1, l2, int(batch)))

    def logistic_fg(self, x, g_out, offset=None, z=None, ydual=None, rho=0.0, want_f=True):
        f = C.c_double()
        _check(self.ctx.L.admm_logistic_fg(self.h, x.ptr, offset.ptr if offset else None,
                                           z.ptr if z else None, ydual.ptr if ydual else None,
                                           rho, C.byref(f) if want_f else None, g_out.ptr))
        return f.value if want_f else None

    def lbfgs_solve(self, x, offset=None, z=None, ydual=None, rho=0.0, **params):
        p = LbfgsParams(params.get("m", 6), params.get("max_iter", 10),
                        params.get("max_linesearch", 20), params.get("epsilon", 1e-5),
                        params.get("ftol", 1e-4), params.get("wolfe", 0.9), int(params.get("linesearch", 0)))
        res = LbfgsResult()
        _check(self.ctx.L.admm_lbfgs_solve(self.h, x.ptr, offset.ptr if offset else None,
                                           z.ptr if z else None, ydual.ptr if ydual else None,
                                           rho, C.byref(p), C.byref(res)))
        return dict(f=res.f, evals=res.evals, iters=res.iters, forward_sweeps=res.forward_sweeps,
                    transposed_sweeps=res.transposed_sweeps)

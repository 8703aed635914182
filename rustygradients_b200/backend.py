"""Host-side mirror of the reference's `Backend` trait (src/backend/mod.rs:130-227)
over the C ABI: same method names, argument meaning and error variants as
`CudaBackend` (src/backend/cuda.rs) so tests read like the reference's own."""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import numpy as np

from . import _lib
from ._lib import check


def _shape_arr(shape: Sequence[int]):
    return (C.c_size_t * max(1, len(shape)))(*[int(s) for s in shape])


_DTYPES = {"f32": _lib.RG_DTYPE_F32, "bf16": _lib.RG_DTYPE_BF16}
_DTYPE_NAMES = {v: k for k, v in _DTYPES.items()}
_FOREIGN = {"torch.float32": _lib.RG_DTYPE_F32, "float32": _lib.RG_DTYPE_F32, "torch.bfloat16": _lib.RG_DTYPE_BF16,
            "bfloat16": _lib.RG_DTYPE_BF16}
_SHAPES = [C.c_size_t * max(1, n) for n in range(9)]

# DLPack capsules: a consumer renames the capsule when it takes the tensor; one that nobody took is released with it
_capsule_new = C.pythonapi.PyCapsule_New
_capsule_new.restype, _capsule_new.argtypes = C.py_object, [C.c_void_p, C.c_char_p, C.c_void_p]
_capsule_valid = C.pythonapi.PyCapsule_IsValid
_capsule_valid.restype, _capsule_valid.argtypes = C.c_int, [C.c_void_p, C.c_char_p]
_capsule_ptr = C.pythonapi.PyCapsule_GetPointer
_capsule_ptr.restype, _capsule_ptr.argtypes = C.c_void_p, [C.c_void_p, C.c_char_p]
_DL_DELETER_OFFSET = 56   # DLManagedTensor: 48 bytes of DLTensor, manager_ctx, deleter


@C.PYFUNCTYPE(None, C.c_void_p)
def _capsule_gone(capsule):
    if _capsule_valid(capsule, b"dltensor"):
        m = _capsule_ptr(capsule, b"dltensor")
        C.CFUNCTYPE(None, C.c_void_p)(C.c_void_p.from_address(m + _DL_DELETER_OFFSET).value)(m)


_capsule_gone_ptr = C.cast(_capsule_gone, C.c_void_p).value


class Storage:
    """CudaStorage {data, shape, device} (src/backend/cuda.rs:29-33): an immutable
    device buffer owned by the library; freed when the Python object dies."""

    __slots__ = ("_backend", "_h", "_keep", "__weakref__")

    def __init__(self, backend: "B200Backend", handle: int, keep=None):
        self._backend = backend
        self._h = handle
        self._keep = keep     # the array whose memory this storage borrows

    @property
    def shape(self):
        lib = _lib.load()
        nd = C.c_int(0)
        buf = (C.c_size_t * 8)()
        check(lib.rg_shape(self._h, buf, 8, C.byref(nd)))
        return [int(buf[i]) for i in range(nd.value)]

    def __len__(self) -> int:
        return int(_lib.load().rg_storage_len(self._h))

    @property
    def dtype(self) -> str:
        """"f32" or "bf16"."""
        return _DTYPE_NAMES[_lib.load().rg_storage_dtype(self._h)]

    def to_dlpack(self):
        """A DLPack capsule that shares the buffer (`torch.utils.dlpack.from_dlpack(st.to_dlpack())`).  It is read in the
        order of the backend's stream; a storage of `from_device` cannot be exported."""
        m = C.c_void_p()
        status = self._backend._lib.rg_to_dlpack(self._h, C.byref(m))
        if status:
            check(status)
        return _capsule_new(m, b"dltensor", _capsule_gone_ptr)

    def __dlpack__(self, stream=None, *, max_version=None, dl_device=None, copy=None):
        """`torch.from_dlpack(st)`: for consumers on the backend's own stream (BufferError elsewhere).  The tensor shares the
        buffer: a copy, or another device, is a BufferError too.  Whatever `max_version` allows, the capsule is an unversioned
        one."""
        if copy:
            raise BufferError("the tensor shares the storage's buffer: copy it after the export (torch.from_dlpack(st).clone())")
        if dl_device is not None and tuple(int(v) for v in dl_device) != self.__dlpack_device__():
            raise BufferError(f"the storage is on CUDA device {self._backend.device_index} and is not moved by an export")
        mine = self._backend.stream or 1          # 1 is the name of the default stream in the protocol
        if stream != -1 and (stream or 1) != mine:
            raise BufferError("the storage is ordered on its backend's stream: make the backend on the consumer's stream")
        return self.to_dlpack()

    def __dlpack_device__(self):
        return (2, self._backend.device_index)

    def __del__(self):
        try:
            be = self._backend
            if self._h and be._ctx:
                be._free(self._h)
        except Exception:
            pass
        self._h = None


class B200Backend:
    """`CudaBackend::new(device_index)` (cuda.rs:87-125).  `stream`: a cudaStream_t (as an int, 0 for the default stream) of
    another owner of the GPU on which every call enqueues, instead of a stream of the backend's own."""

    def __init__(self, device_index: int = 0, stream: Optional[int] = None):
        lib = _lib.load()
        ctx = C.c_void_p()
        if stream is None:
            check(lib.rg_ctx_create(int(device_index), C.byref(ctx)))
        else:
            check(lib.rg_ctx_create_on_stream(int(device_index), C.c_void_p(int(stream)), C.byref(ctx)))
        self._ctx = ctx
        self._lib = lib
        self._free = lib.rg_storage_free
        self.device_index = device_index

    # -- CudaBackend::device_count / is_available (cuda.rs:127-135)
    @staticmethod
    def device_count() -> int:
        return int(_lib.load().rg_device_count())

    @staticmethod
    def is_available() -> bool:
        return B200Backend.device_count() > 0

    def device_type(self):
        return ("cuda", self.device_index)

    def synchronize(self) -> None:
        check(self._lib.rg_synchronize(self._ctx))

    @property
    def stream(self) -> int:
        return int(self._lib.rg_ctx_stream(self._ctx) or 0)

    @property
    def launch_count(self) -> int:
        return int(self._lib.rg_ctx_launch_count(self._ctx))

    def close(self) -> None:
        if self._ctx:
            check(self._lib.rg_ctx_destroy(self._ctx))
            self._ctx = None

    def __del__(self):
        # storages may outlive the backend object in GC order; keep the context
        # until the process exits rather than risk a use-after-free
        pass

    # -- memory operations
    def _wrap(self, h: C.c_void_p, keep=None) -> Storage:
        return Storage(self, h.value, keep)

    def zeros(self, shape) -> Storage:
        h = C.c_void_p()
        check(self._lib.rg_zeros(self._ctx, _shape_arr(shape), len(shape), C.byref(h)))
        return self._wrap(h)

    def ones(self, shape) -> Storage:
        h = C.c_void_p()
        check(self._lib.rg_ones(self._ctx, _shape_arr(shape), len(shape), C.byref(h)))
        return self._wrap(h)

    def from_slice(self, data, shape) -> Storage:
        a = np.ascontiguousarray(np.asarray(data, dtype=np.float32).reshape(-1))
        h = C.c_void_p()
        check(self._lib.rg_from_slice(self._ctx, a.ctypes.data_as(_lib._FP), a.size, _shape_arr(shape), len(shape),
                                      C.byref(h)))
        return self._wrap(h)

    def to_vec(self, st: Storage) -> np.ndarray:
        out = np.empty(len(st), dtype=np.float32)
        check(self._lib.rg_to_vec(self._ctx, st._h, out.ctypes.data_as(_lib._FP), out.size))
        return out

    def to_array(self, st: Storage) -> np.ndarray:
        return self.to_vec(st).reshape(st.shape)

    def shape(self, st: Storage):
        return st.shape

    def from_device(self, array) -> Storage:
        """A storage over a device array of another library (a torch tensor: f32 or bf16, contiguous, on this backend's GPU,
        its values ordered on this backend's stream).  Nothing is copied when it is 16-byte aligned; the storage keeps the
        array alive, and the array must not be written while work of this backend may still read it."""
        try:
            code = _FOREIGN.get(str(array.dtype))
            ptr, shape, dense = array.data_ptr(), array.shape, array.is_contiguous()
        except AttributeError:
            raise _lib.InvalidInput("from_device takes a device array with data_ptr(), shape, dtype and is_contiguous()") from None
        if code is None:
            raise _lib.Unsupported(f"from_device: dtype {array.dtype} is neither f32 nor bf16")
        if not dense:
            raise _lib.InvalidInput("from_device: the array is not contiguous")
        n = len(shape)
        if n > 8:
            raise _lib.DimensionError(f"storage rank {n} not in 0..8")
        h = C.c_void_p()
        status = self._lib.rg_from_device(self._ctx, ptr, code, _SHAPES[n](*shape), n, C.byref(h))
        if status:
            check(status)
        return Storage(self, h.value, array)

    def cast(self, a: Storage, dtype: str) -> Storage:
        """Values as "f32" or "bf16" (rounded to nearest even)."""
        if dtype not in _DTYPES:
            raise _lib.Unsupported(f"dtype {dtype!r} is neither 'f32' nor 'bf16'")
        h = C.c_void_p()
        check(self._lib.rg_cast(self._ctx, a._h, _DTYPES[dtype], C.byref(h)))
        return self._wrap(h, a._keep)

    # -- ops
    def _bin(self, fn, a, b):
        h = C.c_void_p()
        check(fn(self._ctx, a._h, b._h, C.byref(h)))
        return self._wrap(h)

    def _un(self, fn, a):
        h = C.c_void_p()
        check(fn(self._ctx, a._h, C.byref(h)))
        return self._wrap(h)

    def add(self, a, b): return self._bin(self._lib.rg_add, a, b)
    def sub(self, a, b): return self._bin(self._lib.rg_sub, a, b)
    def mul(self, a, b): return self._bin(self._lib.rg_mul, a, b)
    def matmul(self, a, b): return self._bin(self._lib.rg_matmul, a, b)
    def relu(self, a): return self._un(self._lib.rg_relu, a)
    def sigmoid(self, a): return self._un(self._lib.rg_sigmoid, a)
    def exp(self, a): return self._un(self._lib.rg_exp, a)
    def log(self, a): return self._un(self._lib.rg_log, a)
    def gelu(self, a): return self._un(self._lib.rg_gelu, a)
    def softmax(self, a): return self._un(self._lib.rg_softmax, a)
    def sum(self, a): return self._un(self._lib.rg_sum, a)
    def embedding(self, indices, weights): return self._bin(self._lib.rg_embedding, indices, weights)
    def sparse_cross_entropy(self, logits, targets): return self._bin(self._lib.rg_sparse_cross_entropy, logits, targets)

    def powf(self, a, power: float):
        h = C.c_void_p()
        check(self._lib.rg_powf(self._ctx, a._h, float(power), C.byref(h)))
        return self._wrap(h)

    def sum_axis(self, a, axis: int):
        h = C.c_void_p()
        check(self._lib.rg_sum_axis(self._ctx, a._h, int(axis), C.byref(h)))
        return self._wrap(h)

    def reshape(self, a, new_shape):
        h = C.c_void_p()
        check(self._lib.rg_reshape(self._ctx, a._h, _shape_arr(new_shape), len(new_shape), C.byref(h)))
        return self._wrap(h, a._keep)

    def transpose(self, a, axis1: int, axis2: int):
        h = C.c_void_p()
        check(self._lib.rg_transpose(self._ctx, a._h, int(axis1), int(axis2), C.byref(h)))
        return self._wrap(h)

    def layer_norm(self, x, gamma, beta, epsilon: float):
        h = C.c_void_p()
        check(self._lib.rg_layer_norm(self._ctx, x._h, gamma._h, beta._h, float(epsilon), C.byref(h)))
        return self._wrap(h)

    # -- training ops (the steps of WasmGptTrainer::train_step, src/wasm_api.rs:62-94, behind the last block)
    def layer_norm_fwd(self, x, gamma, beta, epsilon: float) -> Tuple[Storage, Storage, Storage]:
        """(y, mean, rstd): `layer_norm` of f32 or bf16 rows with the statistics that `layer_norm_bwd` needs."""
        y, mean, rstd = C.c_void_p(), C.c_void_p(), C.c_void_p()
        check(self._lib.rg_layer_norm_fwd(self._ctx, x._h, gamma._h, beta._h, float(epsilon), C.byref(y), C.byref(mean), C.byref(rstd)))
        return self._wrap(y), self._wrap(mean), self._wrap(rstd)

    def layer_norm_bwd(self, dy, x, gamma, mean, rstd) -> Tuple[Storage, Storage, Storage]:
        """(dx, dgamma, dbeta) of `layer_norm_fwd`."""
        dx, dg, db = C.c_void_p(), C.c_void_p(), C.c_void_p()
        check(self._lib.rg_layer_norm_bwd(self._ctx, dy._h, x._h, gamma._h, mean._h, rstd._h, C.byref(dx), C.byref(dg), C.byref(db)))
        return self._wrap(dx), self._wrap(dg), self._wrap(db)

    def linear_cross_entropy(self, x, w, bias, targets, ignore_index: int = -100) -> Tuple[Storage, Storage]:
        """(loss [1], lse [rows]): `sparse_cross_entropy` of x w + bias without the logits; rows whose target is
        `ignore_index` are left out.  `bias` may be None."""
        loss, lse = C.c_void_p(), C.c_void_p()
        check(self._lib.rg_linear_cross_entropy(self._ctx, x._h, w._h, bias._h if bias is not None else None, targets._h,
                                                int(ignore_index), C.byref(loss), C.byref(lse)))
        return self._wrap(loss), self._wrap(lse)

    def linear_cross_entropy_bwd(self, x, w, bias, targets, lse, dloss=None,
                                 ignore_index: int = -100) -> Tuple[Storage, Storage, Optional[Storage]]:
        """(dx, dw, dbias) of `linear_cross_entropy` for the upstream gradient `dloss` ([1]; None for 1); dbias is None
        when bias is."""
        dx, dw, db = C.c_void_p(), C.c_void_p(), C.c_void_p()
        check(self._lib.rg_linear_cross_entropy_bwd(self._ctx, x._h, w._h, bias._h if bias is not None else None, targets._h,
                                                    int(ignore_index), lse._h, dloss._h if dloss is not None else None,
                                                    C.byref(dx), C.byref(dw), C.byref(db) if bias is not None else None))
        return self._wrap(dx), self._wrap(dw), self._wrap(db) if bias is not None else None

    def clip_grad_norm(self, grads: Sequence[Storage], max_norm: float) -> Tuple[List[Storage], Storage]:
        """(clipped gradients, norm [1]): `clip_gradients` (src/wasm_api.rs:202-224) over all tensors at once."""
        n = len(grads)
        given, out, norm = (C.c_void_p * n)(*[g._h for g in grads]), (C.c_void_p * n)(), C.c_void_p()
        check(self._lib.rg_clip_grad_norm(self._ctx, given, n, float(max_norm), out, C.byref(norm)))
        return [Storage(self, h) for h in out], self._wrap(norm)

"""Host-side mirror of cutorch's tensor interface over the THC C API of libthcb200.so.

cutorch exposes the THC entry points as tensor methods through cwrap-generated stubs
(TensorMath.lua:429-438,552-2258: fetch ``cutorch._state``, check argument types, call
``TH<Type>Tensor_<name>(state, ...)``).  :class:`Tensor` plays the role of those stubs from
Python: ``z.cadd(x, 2.5, y)`` calls ``THCudaTensor_cadd(state, z, x, 2.5f, y)``.  Every method
goes through the C ABI of the shared library; there is no other implementation behind it.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib


class THCError(RuntimeError):
    """A THC call reported an error (THError / THArgCheck in cutorch)."""


class _Half(C.Structure):
    _fields_ = [("x", C.c_ushort)]


# kind -> (CReal infix of the symbol names, numpy dtype, ctypes `real`, ctypes `accreal`, thcb200 dtype)
KINDS = {
    "Byte": ("CudaByte", np.uint8, C.c_ubyte, C.c_long, _lib.U8),
    "Char": ("CudaChar", np.int8, C.c_byte, C.c_long, _lib.I8),
    "Short": ("CudaShort", np.int16, C.c_short, C.c_long, _lib.I16),
    "Int": ("CudaInt", np.int32, C.c_int, C.c_long, _lib.I32),
    "Long": ("CudaLong", np.int64, C.c_long, C.c_long, _lib.I64),
    "Half": ("CudaHalf", np.float16, _Half, C.c_float, _lib.F16),
    "Float": ("Cuda", np.float32, C.c_float, C.c_float, _lib.F32),
    "Double": ("CudaDouble", np.float64, C.c_double, C.c_double, _lib.F64),
}
KIND_OF_DTYPE = {np.dtype(v[1]): k for k, v in KINDS.items()}


class _THStorage(C.Structure):
    """torch7's CPU storage (lib/TH/generic/THStorage.h): the same fields for every element type."""
    _fields_ = [("data", C.c_void_p), ("size", C.c_ssize_t), ("refcount", C.c_int), ("flag", C.c_char),
                ("allocator", C.c_void_p), ("allocatorContext", C.c_void_p), ("view", C.c_void_p)]


class _THTensor(C.Structure):
    """torch7's CPU tensor (lib/TH/generic/THTensor.h)."""
    _fields_ = [("size", C.POINTER(C.c_long)), ("stride", C.POINTER(C.c_long)), ("nDimension", C.c_int),
                ("storage", C.POINTER(_THStorage)), ("storageOffset", C.c_ssize_t), ("refcount", C.c_int), ("flag", C.c_char)]


class CpuTensor:
    """A numpy array seen as a TH CPU tensor (TH<Type>Tensor): the argument of the copies between
    CPU and GPU tensors.  Any non-negative strides that are whole elements; the array is not copied."""

    def __init__(self, array: np.ndarray):
        if array.dtype not in KIND_OF_DTYPE:
            raise TypeError(f"no tensor type for {array.dtype}")
        if any(s < 0 or s % array.itemsize for s in array.strides):
            raise ValueError("strides must be non-negative multiples of the element size")
        self.array = array
        self.kind = KIND_OF_DTYPE[array.dtype]
        nd = array.ndim
        self._size = (C.c_long * max(nd, 1))(*array.shape)
        self._stride = (C.c_long * max(nd, 1))(*[s // array.itemsize for s in array.strides])
        extent = 1 + sum((n - 1) * (s // array.itemsize) for n, s in zip(array.shape, array.strides)) if array.size else 0
        self._storage = _THStorage(array.ctypes.data, extent, 1, b"\x00", None, None, None)
        self._tensor = _THTensor(self._size, self._stride, nd, C.pointer(self._storage), 0, 1, b"\x01")

    @property
    def ptr(self):
        return C.byref(self._tensor)
FLOATING = ("Half", "Float", "Double")
ACC_KIND = {"Half": "Float", "Float": "Float", "Double": "Double"}   # the tensor of a floating type's accreal

# Argument codes: T tensor of the receiver's type, L LongTensor, A tensor of the receiver's accreal (None: NULL), f accreal, C / M CPU Long / Byte tensor (CpuTensor), r real, l long, i int, S sizes.
# Return codes: v void, a accreal, R real, n int.
_UNARY = ["sigmoid", "log", "lgamma", "log1p", "exp", "cos", "acos", "cosh", "sin", "asin", "sinh", "tan", "atan",
          "tanh", "sqrt", "rsqrt", "ceil", "floor", "round", "trunc", "frac", "cinv", "neg", "abs", "sign"]
SIGNATURES = {name: ("v", "TT") for name in _UNARY}
SIGNATURES.update({
    "pow": ("v", "TTr"), "tpow": ("v", "TrT"), "atan2": ("v", "TTT"), "lerp": ("v", "TTTr"),
    "clamp": ("v", "TTrr"), "cross": ("v", "TTTi"),
    "cadd": ("v", "TTrT"), "csub": ("v", "TTrT"),
    "cmul": ("v", "TTT"), "cpow": ("v", "TTT"), "cdiv": ("v", "TTT"), "clshift": ("v", "TTT"), "crshift": ("v", "TTT"),
    "cmax": ("v", "TTT"), "cmin": ("v", "TTT"), "cfmod": ("v", "TTT"), "cremainder": ("v", "TTT"),
    "cmaxValue": ("v", "TTr"), "cminValue": ("v", "TTr"),
    "cbitand": ("v", "TTT"), "cbitor": ("v", "TTT"), "cbitxor": ("v", "TTT"),
    "addcmul": ("v", "TTrTT"), "addcdiv": ("v", "TTrTT"),
    "add": ("v", "TTr"), "sub": ("v", "TTr"), "mul": ("v", "TTr"), "div": ("v", "TTr"),
    "lshift": ("v", "TTr"), "rshift": ("v", "TTr"), "fmod": ("v", "TTr"), "remainder": ("v", "TTr"),
    "bitand": ("v", "TTr"), "bitor": ("v", "TTr"), "bitxor": ("v", "TTr"),
    "equal": ("n", "TT"),
    "sum": ("v", "TTli"), "prod": ("v", "TTli"), "mean": ("v", "TTli"), "norm": ("v", "TTrli"),
    "sumall": ("a", "T"), "prodall": ("a", "T"), "meanall": ("a", "T"),
    "min": ("v", "TLTli"), "max": ("v", "TLTli"), "minall": ("R", "T"), "maxall": ("R", "T"),
    "var": ("v", "TTlii"), "std": ("v", "TTlii"), "dist": ("a", "TTr"),
    "normall": ("a", "Tr"), "varall": ("a", "Ti"), "stdall": ("a", "Ti"),
    "fill": ("v", "Tr"), "zero": ("v", "T"), "copy": ("v", "TT"), "copyIgnoringOverlaps": ("v", "TT"),
    "resizeAs": ("v", "TT"),
    "tril": ("v", "TTl"), "triu": ("v", "TTl"), "renorm": ("v", "TTrlr"),
    "indexSelect": ("v", "TTiL"), "indexCopy": ("v", "TiLT"), "indexAdd": ("v", "TiLT"), "indexFill": ("v", "TiLr"),
    # thin callers of fill / copy / sumall; code S: a tuple of sizes passed as a THLongStorage
    "zeros": ("v", "TS"), "ones": ("v", "TS"), "zerosLike": ("v", "TT"), "onesLike": ("v", "TT"), "reshape": ("v", "TTS"),
    "numel": ("p", "T"), "nonzero": ("v", "LT"), "diag": ("v", "TTl"), "eye": ("v", "Tll"), "trace": ("a", "T"),
    # masks in a CPU ByteTensor (code M)
    "maskedFillByte": ("v", "TMr"), "maskedCopyByte": ("v", "TMT"), "maskedSelectByte": ("v", "TTM"),
    # the same with a CPU LongTensor of positions (code C)
    "indexSelect_long": ("v", "TTiC"), "indexCopy_long": ("v", "TiCT"), "indexAdd_long": ("v", "TiCT"),
    "indexFill_long": ("v", "TiCr"),
    "gather": ("v", "TTiL"), "scatter": ("v", "TiLT"), "scatterAdd": ("v", "TiLT"), "scatterFill": ("v", "TiLr"),
    "cumsum": ("v", "TTl"), "cumprod": ("v", "TTl"),
    # rows of an embedding table and their gradient, rows to the experts and back
    "embedding": ("v", "TTLf"), "embeddingAccGrad": ("v", "TTLfli"), "expertSort": ("v", "TTTTl"),
    "expertDispatch": ("v", "TTLA"), "expertCombine": ("v", "TTLA"), "expertCombineGrad": ("v", "TATTLA"),
    "maskedFill": ("v", "TBr"), "maskedCopy": ("v", "TBT"), "maskedSelect": ("v", "TTB"),
})
# comparisons: <op>Value / <op>Tensor write a Byte tensor ("B"), the ...T forms the operands' type
for _c in ("lt", "gt", "le", "ge", "eq", "ne"):
    SIGNATURES.update({_c + "Value": ("v", "BTr"), _c + "ValueT": ("v", "TTr"),
                       _c + "Tensor": ("v", "BTT"), _c + "TensorT": ("v", "TTT")})


def _half_from_float(v: float) -> _Half:
    return _Half(int(np.array(v, dtype=np.float16).view(np.uint16)))


def _half_to_float(h: _Half) -> float:
    return float(np.array(h.x, dtype=np.uint16).view(np.float16))


def _real_of(kind: str):
    """The conversion of a number to a tensor kind's C `real`."""
    creal = KINDS[kind][2]
    if kind == "Half":
        return lambda v: _half_from_float(float(v))
    if kind in FLOATING:
        return lambda v: creal(float(v))
    return lambda v: creal(int(v))


class State:
    """THCState: owns the per-device contexts; `stream` selects the current stream."""

    def __init__(self):
        self.lib = _lib.load_library()
        lib = self.lib
        self._failed = lib.THCB200_errorOccurred
        lib.THCState_alloc.restype = C.c_void_p
        lib.THCudaInit.argtypes = [C.c_void_p]
        lib.THCudaShutdown.argtypes = [C.c_void_p]
        lib.THCState_free.argtypes = [C.c_void_p]
        lib.THCB200_errorMessage.restype = C.c_char_p
        lib.THCB200_streamFromRaw.restype = C.c_void_p
        lib.THCB200_streamFromRaw.argtypes = [C.c_void_p, C.c_int]
        lib.THCState_setStream.argtypes = [C.c_void_p, C.c_void_p]
        lib.THCStream_free.argtypes = [C.c_void_p]
        lib.THCState_getCurrentStream.restype = C.c_void_p
        lib.THCState_getCurrentStream.argtypes = [C.c_void_p]
        lib.THCB200_currentContext.restype = C.c_void_p
        lib.THCB200_currentContext.argtypes = [C.c_void_p]
        self.ptr = C.c_void_p(lib.THCState_alloc())
        lib.THCB200_clearError()
        lib.THCudaInit(self.ptr)
        self.check()
        self._fn_cache = {}
        self._calls = {}

    def check(self):
        if self._failed():
            msg = self.lib.THCB200_errorMessage().decode()
            self.lib.THCB200_clearError()
            raise THCError(msg)

    def set_stream(self, raw_stream: int, device: int = 0):
        """Makes a stream created elsewhere (e.g. torch.cuda.Stream.cuda_stream) current."""
        s = self.lib.THCB200_streamFromRaw(C.c_void_p(raw_stream), device)
        self.lib.THCState_setStream(self.ptr, C.c_void_p(s))
        self.lib.THCStream_free(C.c_void_p(s))
        self.check()

    @property
    def stream(self) -> int:
        return self.lib.THCState_getCurrentStream(self.ptr) or 0

    @property
    def context(self) -> int:
        c = self.lib.THCB200_currentContext(self.ptr)
        self.check()
        return c

    def synchronize(self):
        _lib.check(self.lib.thcb200_stream_synchronize(C.c_void_p(self.stream)))

    def shutdown(self):
        if self.ptr:
            self.lib.THCudaShutdown(self.ptr)
            self.lib.THCState_free(self.ptr)
            self.ptr = None

    def fn(self, kind: str, name: str, prefix: str = "Tensor"):
        key = (kind, name, prefix)
        f = self._fn_cache.get(key)
        if f is None:
            # a private function object per symbol: ctypes caches attribute lookups, and the
            # argtypes set by one caller must not leak into another
            f = self.lib[f"TH{KINDS[kind][0]}{prefix}_{name}"]
            self._fn_cache[key] = f
        return f


class Tensor:
    """A THCuda<Kind>Tensor handle."""

    def __init__(self, state: State, kind: str, ptr: int):
        self.state, self.kind, self.ptr = state, kind, C.c_void_p(ptr)

    # ---- construction ------------------------------------------------------------------
    @classmethod
    def new(cls, state: State, kind: str = "Float", *sizes: int) -> "Tensor":
        f = state.fn(kind, "new")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p]
        t = cls(state, kind, f(state.ptr))
        if sizes:
            t.resize(*sizes)
        return t

    @classmethod
    def from_numpy(cls, state: State, arr: np.ndarray) -> "Tensor":
        """Clones a numpy array to the device with its exact sizes, strides and holes
        (cloneExactlyToGPUType, test/test.lua:348-361)."""
        kind = KIND_OF_DTYPE[arr.dtype]
        item = arr.dtype.itemsize
        if arr.ndim == 0:
            arr = arr.reshape(1)
        strides = [s // item for s in arr.strides]
        if any(s < 0 for s in strides):
            raise ValueError("negative strides are not representable as TH tensors")
        extent = 1 + sum((n - 1) * s for n, s in zip(arr.shape, strides)) if arr.size else 0
        t = cls.new(state, kind)
        if extent == 0:
            if arr.ndim:
                t.resize(*arr.shape)
            return t
        flat = np.lib.stride_tricks.as_strided(arr, shape=(extent,), strides=(item,))
        flat = np.ascontiguousarray(flat)
        st = state.fn(kind, "newWithSize", "Storage")
        st.restype = C.c_void_p
        st.argtypes = [C.c_void_p, C.c_ssize_t]
        storage = C.c_void_p(st(state.ptr, extent))
        state.check()
        data = state.fn(kind, "data", "Storage")
        data.restype = C.c_void_p
        data.argtypes = [C.c_void_p, C.c_void_p]
        dptr = data(state.ptr, storage)
        _lib.check(state.lib.thcb200_memcpy_h2d(C.c_void_p(dptr), flat.ctypes.data_as(C.c_void_p), flat.nbytes,
                                                 C.c_void_p(state.stream)))
        t._set_storage(storage, 0, arr.shape, strides)
        free = state.fn(kind, "free", "Storage")
        free.argtypes = [C.c_void_p, C.c_void_p]
        free(state.ptr, storage)
        return t

    @classmethod
    def wrap(cls, state: State, kind: str, device_ptr: int, sizes, strides=None, storage_elems=None) -> "Tensor":
        """A tensor over device memory owned by someone else (not freed, not resizable)."""
        sizes = list(sizes)
        if strides is None:
            strides, run = [], 1
            for n in reversed(sizes):
                strides.insert(0, run)
                run *= n
        if storage_elems is None:
            storage_elems = max(0, 1 + sum((n - 1) * s for n, s in zip(sizes, strides)))     # below 1 where a size is 0
        f = state.fn(kind, "newBorrowed")
        if f.argtypes is None:
            f.restype = C.c_void_p
            f.argtypes = [C.c_void_p, C.c_void_p, C.c_ssize_t, C.c_int, C.c_void_p, C.c_void_p]
        longs = C.c_long * len(sizes)
        p = f(state.ptr, device_ptr, storage_elems, len(sizes), longs(*sizes), longs(*strides))
        state.check()
        return cls(state, kind, p)

    @staticmethod
    def _long_storage(state, values):
        lib = state.lib
        lib.THLongStorage_newWithSize.restype = C.c_void_p
        lib.THLongStorage_newWithSize.argtypes = [C.c_ssize_t]
        lib.THLongStorage_set.argtypes = [C.c_void_p, C.c_ssize_t, C.c_long]
        lib.THLongStorage_free.argtypes = [C.c_void_p]
        s = C.c_void_p(lib.THLongStorage_newWithSize(len(values)))
        for k, v in enumerate(values):
            lib.THLongStorage_set(s, k, int(v))
        return s

    def _set_storage(self, storage, offset, sizes, strides):
        f = self.state.fn(self.kind, "setStorage")
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_ssize_t, C.c_void_p, C.c_void_p]
        sz, st = self._long_storage(self.state, sizes), self._long_storage(self.state, strides)
        f(self.state.ptr, self.ptr, storage, offset, sz, st)
        self.state.lib.THLongStorage_free(sz)
        self.state.lib.THLongStorage_free(st)
        self.state.check()

    def resize(self, *sizes):
        f = self.state.fn(self.kind, "resize")
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        sz = self._long_storage(self.state, sizes)
        f(self.state.ptr, self.ptr, sz, None)
        self.state.lib.THLongStorage_free(sz)
        self.state.check()
        return self

    def free(self):
        if self.ptr:
            f = self.state.fn(self.kind, "free")
            f.argtypes = [C.c_void_p, C.c_void_p]
            f(self.state.ptr, self.ptr)
            self.ptr = None

    # ---- views -------------------------------------------------------------------------
    def transpose(self, d1, d2) -> "Tensor":
        f = self.state.fn(self.kind, "newTranspose")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int]
        t = Tensor(self.state, self.kind, f(self.state.ptr, self.ptr, d1, d2))
        self.state.check()
        return t

    def expand(self, *sizes) -> "Tensor":
        """tensor:expand(sizes): a broadcast view (THCTensor_(newExpand))."""
        f = self.state.fn(self.kind, "newExpand")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        sz = self._long_storage(self.state, sizes)
        p = f(self.state.ptr, self.ptr, sz)
        self.state.lib.THLongStorage_free(sz)
        self.state.check()
        return Tensor(self.state, self.kind, p)

    def narrow(self, dim, first, size) -> "Tensor":
        f = self.state.fn(self.kind, "newNarrow")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_long, C.c_long]
        t = Tensor(self.state, self.kind, f(self.state.ptr, self.ptr, dim, first, size))
        self.state.check()
        return t

    def select(self, dim, index) -> "Tensor":
        f = self.state.fn(self.kind, "newSelect")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_long]
        t = Tensor(self.state, self.kind, f(self.state.ptr, self.ptr, dim, index))
        self.state.check()
        return t

    def contiguous(self) -> "Tensor":
        f = self.state.fn(self.kind, "newContiguous")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p, C.c_void_p]
        t = Tensor(self.state, self.kind, f(self.state.ptr, self.ptr))
        self.state.check()
        return t

    # ---- metadata ----------------------------------------------------------------------
    @property
    def ndim(self) -> int:
        f = self.state.fn(self.kind, "nDimension")
        f.argtypes = [C.c_void_p, C.c_void_p]
        return f(self.state.ptr, self.ptr)

    def _dims(self, name):
        f = self.state.fn(self.kind, name)
        f.restype = C.c_long
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_int]
        return [f(self.state.ptr, self.ptr, d) for d in range(self.ndim)]

    @property
    def sizes(self):
        return self._dims("size")

    @property
    def strides(self):
        return self._dims("stride")

    @property
    def nelement(self) -> int:
        f = self.state.fn(self.kind, "nElement")
        f.restype = C.c_ssize_t
        f.argtypes = [C.c_void_p, C.c_void_p]
        return f(self.state.ptr, self.ptr)

    @property
    def data_ptr(self) -> int:
        f = self.state.fn(self.kind, "data")
        f.restype = C.c_void_p
        f.argtypes = [C.c_void_p, C.c_void_p]
        return f(self.state.ptr, self.ptr) or 0

    @property
    def is_contiguous(self) -> bool:
        f = self.state.fn(self.kind, "isContiguous")
        f.argtypes = [C.c_void_p, C.c_void_p]
        return bool(f(self.state.ptr, self.ptr))

    def descriptor(self) -> _lib.TensorDesc:
        return _lib.make_desc(self.data_ptr, KINDS[self.kind][4], self.sizes, self.strides)

    def numpy(self) -> np.ndarray:
        """Copies the view back to the host as a dense array in logical order."""
        sizes, strides = self.sizes, self.strides
        dt = np.dtype(KINDS[self.kind][1])
        if not sizes or self.nelement == 0:
            return np.zeros(sizes, dtype=dt)
        if any(s < 0 for s in strides):
            raise ValueError("negative strides")
        extent = 1 + sum((n - 1) * s for n, s in zip(sizes, strides))
        flat = np.empty(extent, dtype=dt)
        self.state.synchronize()
        _lib.check(self.state.lib.thcb200_memcpy_d2h(flat.ctypes.data_as(C.c_void_p), C.c_void_p(self.data_ptr), flat.nbytes,
                                                      C.c_void_p(self.state.stream)))
        view = np.lib.stride_tricks.as_strided(flat, shape=sizes, strides=[s * dt.itemsize for s in strides])
        return np.array(view, copy=True)

    # ---- THC calls ---------------------------------------------------------------------
    def _prepare(self, name: str):
        """A call's function object with its C prototype, and per argument the kind a tensor has to be of, whether it may be
        missing, and the conversion of anything that is not a GPU tensor."""
        f = self.state.fn(self.kind, name)
        ret, spec = SIGNATURES[name]
        creal, cacc = KINDS[self.kind][2], KINDS[self.kind][3]
        codes = {"r": creal, "l": C.c_long, "f": cacc}
        f.argtypes = [C.c_void_p] + [codes.get(c, C.c_int if c == "i" else C.c_void_p) for c in spec]
        f.restype = {"v": None, "a": cacc, "R": creal, "n": C.c_int, "p": C.c_ssize_t}[ret]
        kinds = {"T": self.kind, "L": "Long", "B": "Byte", "A": ACC_KIND.get(self.kind)}

        def cpu(want):
            def convert(a):
                if not isinstance(a, CpuTensor) or a.kind != want:
                    raise TypeError(f"{name}: expected a CPU {want} tensor")
                return a.ptr
            return convert

        state = self.state
        converts = {"r": _real_of(self.kind), "l": int, "i": int, "f": float, "C": cpu("Long"), "M": cpu("Byte"),
                    "S": lambda a: Tensor._long_storage(state, tuple(a))}
        arguments = [(kinds.get(c), c == "A", converts.get(c)) for c in spec]
        storages = [k + 1 for k, c in enumerate(spec) if c == "S"]
        call = f, arguments, storages, ret == "R" and self.kind == "Half"
        state._calls[self.kind, name] = call
        return call

    def call(self, name: str, *args):
        """Calls TH<Kind>Tensor_<name>(state, ...) with `args` exactly in C order."""
        state = self.state
        try:
            f, arguments, storages, half = state._calls[self.kind, name]
        except KeyError:
            f, arguments, storages, half = self._prepare(name)
        if len(args) != len(arguments):
            spec = SIGNATURES[name][1]
            raise TypeError(f"{name} takes {len(spec)} arguments ({spec}), got {len(args)}")
        cargs = [state.ptr]
        for (kind, optional, convert), a in zip(arguments, args):
            if convert is not None:
                cargs.append(convert(a))
            elif isinstance(a, Tensor):
                if a.kind != kind:
                    raise TypeError(f"{name}: expected a {kind} tensor, got {a.kind}")
                cargs.append(a.ptr)
            elif optional and a is None:
                cargs.append(None)
            else:
                raise TypeError(f"{name}: expected a tensor")
        r = f(*cargs)
        for k in storages:
            state.lib.THLongStorage_free(cargs[k])
        state.check()
        return _half_to_float(r) if half else r

    def copy_from(self, src: "Tensor"):
        """self:copy(src) with type conversion (THCTensor_(copyCuda<Type>))."""
        if src.kind == self.kind:
            return self.call("copy", self, src)
        f = self.state.fn(self.kind, "copyCudaFloat" if src.kind == "Float" else "copy" + KINDS[src.kind][0])
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        f.restype = None
        f(self.state.ptr, self.ptr, src.ptr)
        self.state.check()

    def copy_from_cpu(self, cpu: "CpuTensor"):
        """self:copy(cpuTensor): THCuda<T>Tensor_copy<CpuType> (lib/THC/generic/THCTensorCopy.c:33-62)."""
        f = self.state.fn(self.kind, "copy" + cpu.kind)
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        f.restype = None
        f(self.state.ptr, self.ptr, cpu.ptr)
        self.state.check()

    def copy_to_cpu(self, cpu: "CpuTensor"):
        """cpuTensor:copy(self): TH<CpuType>Tensor_copyCuda<T> (lib/THC/generic/THCTensorCopy.c:66-110)."""
        f = getattr(self.state.lib, f"TH{cpu.kind}Tensor_copyCuda{self.kind}")
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        f.restype = None
        f(self.state.ptr, cpu.ptr, self.ptr)
        self.state.check()

    def copy_async_from_cpu(self, cpu: "CpuTensor"):
        """THCuda<T>Tensor_copyAsyncCPU (lib/THC/generic/THCTensorCopy.c:112-137): same element type, both
        contiguous, one asynchronous copy in the order of the current stream; the CPU side should be pinned."""
        f = self.state.fn(self.kind, "copyAsyncCPU")
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        f.restype = None
        f(self.state.ptr, self.ptr, cpu.ptr)
        self.state.check()

    def copy_async_to_cpu(self, cpu: "CpuTensor"):
        """TH<T>Tensor_copyAsyncCuda (lib/THC/generic/THCTensorCopy.c:139-164): the way back."""
        f = getattr(self.state.lib, f"TH{self.kind}Tensor_copyAsyncCuda")
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        f.restype = None
        f(self.state.ptr, cpu.ptr, self.ptr)
        self.state.check()

    def cat(self, inputs, dimension: int):
        """result:cat(inputs, dimension): THCTensor_(catArray) (lib/THC/generic/THCTensorMath.cu:84-260)."""
        f = self.state.fn(self.kind, "catArray")
        arr = (C.c_void_p * len(inputs))(*[t.ptr for t in inputs])
        f.argtypes = [C.c_void_p, C.c_void_p, C.POINTER(C.c_void_p), C.c_int, C.c_int]
        f.restype = None
        f(self.state.ptr, self.ptr, arr, len(inputs), dimension)
        self.state.check()

    def sumall_to_device(self, result_dev_ptr: int):
        f = self.state.fn(self.kind, "sumallToDevice")
        f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        f.restype = None
        f(self.state.ptr, self.ptr, C.c_void_p(result_dev_ptr))
        self.state.check()


_DIRECT = {        # per argument code: when an argument can go to C as it is, and what goes there
    "T": ("type({a}) is Tensor and {a}.kind == kind", "{a}.ptr"),
    "L": ("type({a}) is Tensor and {a}.kind == 'Long'", "{a}.ptr"),
    "B": ("type({a}) is Tensor and {a}.kind == 'Byte'", "{a}.ptr"),
    "A": ("({a} is None or type({a}) is Tensor and {a}.kind == ACC_KIND.get(kind))", "None if {a} is None else {a}.ptr"),
    "f": ("type({a}) is float", "{a}"),
    "l": ("type({a}) is int", "{a}"),
    "i": ("type({a}) is int", "{a}"),
}


def _method(name):
    """A tensor method in the Lua style: the receiver is the first C argument.  A step of small tensors is bound by what its
    calls take on the host, so arguments that need no conversion go to C from here (a lookup of one row 4.6 -> 4.0 us);
    everything else, refusals among it, goes through `call`."""
    ret, spec = SIGNATURES[name]

    def general(self, *args):
        return self.call(name, self, *args)

    general.__name__ = name
    if ret == "R" or spec[0] != "T" or any(c not in _DIRECT for c in spec):
        return general
    names = [f"a{k}" for k in range(1, len(spec))]
    fits = [_DIRECT[c][0].format(a=a) for c, a in zip(spec[1:], names)]
    passed = ["state.ptr", "self.ptr"] + [_DIRECT[c][1].format(a=a) for c, a in zip(spec[1:], names)]
    unpack = f"{', '.join(names)}, = args" if names else "pass"
    source = f"""
def {name}(self, *args):
    state, kind = self.state, self.kind
    f = ready.get(kind)
    if f is not None and len(args) == {len(names)}:
        {unpack}
        if {' and '.join(fits) or 'True'}:
            r = f({', '.join(passed)})
            if state._failed():
                state.check()
            return r
    r = self.call(name, self, *args)
    ready[kind] = state._calls[kind, name][0]
    return r
"""
    scope = {"Tensor": Tensor, "ACC_KIND": ACC_KIND, "ready": {}, "name": name}
    exec(source, scope)
    return scope[name]


for _name in SIGNATURES:
    if not hasattr(Tensor, _name):
        setattr(Tensor, _name, _method(_name))


class TensorList:
    """Handles of several tensors of one kind, as the calls over lists of tensors take them: an optimiser keeps one for its
    parameters, one for their gradients and one for each moment."""

    def __init__(self, tensors):
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("an empty list of tensors")
        self.state, self.kind = self.tensors[0].state, self.tensors[0].kind
        if any(t.kind != self.kind for t in self.tensors):
            raise TypeError("tensors of different kinds in one list")
        self.array = (C.c_void_p * len(self.tensors))(*[t.ptr for t in self.tensors])
        self.handles = C.c_void_p(C.addressof(self.array))

    def __len__(self):
        return len(self.tensors)

    def _call(self, name, lists, kinds, scalars=(), scalar_types=()):
        """`name` of these tensors and `lists`, which are of `kinds` (None: no list), and the scalars behind the count."""
        state, n = self.state, len(self.tensors)
        args = [state.ptr, self.handles]
        for what, want in zip(lists, kinds):
            if type(what) is TensorList and what.kind == want and len(what.tensors) == n:
                args.append(what.handles)
            elif what is None:
                args.append(None)
            elif not isinstance(what, TensorList):
                raise TypeError(f"{name}: expected a TensorList")
            elif what.kind != want:
                raise TypeError(f"{name}: expected {want} tensors, got {what.kind}")
            else:
                raise ValueError(f"{name}: lists of {n} and {len(what)} tensors")
        f = state._calls.get((self.kind, name, "list"))
        if f is None:
            f = state.fn(self.kind, name)
            f.argtypes = [C.c_void_p] * (2 + len(lists)) + [C.c_int, *scalar_types]
            f.restype = None
            state._calls[self.kind, name, "list"] = f          # other host threads find it there
        f(*args, n, *scalars)
        if state._failed():
            state.check()

    def adamw(self, grad, m, v, *, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, grad_scale=1.0, master=None):
        """One AdamW step of these parameters (THCTensor_(adamw)); m, v and master are of the parameters' accreal."""
        acc = ACC_KIND.get(self.kind)
        self._call("adamw", (grad, m, v, master), (self.kind, acc, acc, acc),
                   (step, lr, beta1, beta2, eps, weight_decay, grad_scale), _STEP_SCALARS)

    def adamw8bit(self, grad, m, v, m_unit, v_unit, *, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, grad_scale=1.0,
                  master=None):
        """The same with the moments in 8 bits (THCTensor_(adamw8bit)): Char and Byte codes, a float unit per 256 elements."""
        self._call("adamw8bit", (grad, m, v, m_unit, v_unit, master),
                   (self.kind, "Char", "Byte", "Float", "Float", ACC_KIND.get(self.kind)),
                   (step, lr, beta1, beta2, eps, weight_decay, grad_scale), _STEP_SCALARS)

    def adamwValues(self, v_value, m, v, m_unit, v_unit):
        """The floats that 8-bit moments stand for: these tensors receive the first moment's, v_value's the second's."""
        if self.kind != "Float":
            raise TypeError(f"adamwValues: expected Float tensors, got {self.kind}")
        self._call("adamwValues", (v_value, m, v, m_unit, v_unit), ("Float", "Char", "Byte", "Float", "Float"))


_STEP_SCALARS = (C.c_long, *[C.c_double] * 6)      # step, lr, beta1, beta2, eps, weight decay, scale of the gradients

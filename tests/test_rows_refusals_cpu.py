"""What the embedding, expert and AdamW calls refuse before they touch a context or a GPU, through the descriptor ABI."""
import ctypes as C

import numpy as np
import pytest

from cutorch_b200 import _lib
from cutorch_b200._lib import F16, F32, F64, I32, I64, make_desc

ARG, SIZE, UNSUPPORTED, LIMIT = -1, -3, -5, -7
HERE = np.zeros(4096, np.uint8)              # an address; nothing reads it


class Tensor(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("param", "grad", "m", "v", "m_unit", "v_unit", "master")] + [("numel", C.c_int64)]


class Args(C.Structure):
    _fields_ = [(n, C.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "grad_scale")] + [("step", C.c_int64)]


@pytest.fixture()
def lib():
    return _lib.load_library()


CONTEXT = C.c_void_p(HERE.ctypes.data)       # refused calls do not look at it


def view(dtype, *sizes, strides=None):
    if strides is None:
        strides, run = [], 1
        for n in reversed(sizes):
            strides.insert(0, run)
            run *= n
    return C.byref(make_desc(HERE.ctypes.data, dtype, sizes, strides))


def refused(lib, rc, want, text):
    lib.thcb200_last_error.restype = C.c_char_p
    assert rc == want, (rc, lib.thcb200_last_error())
    assert text in lib.thcb200_last_error().decode(), lib.thcb200_last_error()


def test_embedding(lib):
    f = lambda *a, ctx=CONTEXT: lib.thcb200_embedding(ctx, *a, C.c_double(1), None)  # noqa: E731
    w, ix, out = view(F32, 5, 8), view(I64, 3), view(F32, 3, 8)
    refused(lib, f(out, w, ix, ctx=None), ARG, "null context")
    refused(lib, f(out, view(I32, 5, 8), ix), ARG, "floating-point")
    refused(lib, f(out, view(F16, 5, 8), ix), ARG, "floating-point")
    refused(lib, f(out, w, view(I32, 3)), ARG, "I64")
    refused(lib, f(out, w, view(I64, 3, 1)), ARG, "vector")
    refused(lib, f(out, view(F32, 5), ix), ARG, "matrix")
    refused(lib, f(out, w, view(I64, 4)), SIZE, "sizes")
    refused(lib, f(view(F32, 3, 7), w, ix), SIZE, "sizes")
    refused(lib, f(view(F32, 3, 8, strides=(1, 3)), w, ix), ARG, "dense")
    refused(lib, f(view(F32, 3, 8, strides=(0, 1)), w, ix), ARG, "dense")


def test_embedding_grad(lib):
    def f(table, go, ix, padding=0):
        return lib.thcb200_embedding_grad(CONTEXT, table, go, ix, C.c_double(1), C.c_int64(padding), 0, None)
    table, go, ix = view(F32, 5, 8), view(F32, 3, 8), view(I64, 3)
    refused(lib, f(table, view(F64, 3, 8), ix), ARG, "floating-point")
    refused(lib, f(table, view(F32, 3, 9), ix), SIZE, "sizes")
    refused(lib, f(table, go, view(I64, 2)), SIZE, "sizes")
    refused(lib, f(table, go, ix, padding=6), ARG, "padding")
    refused(lib, f(table, go, ix, padding=-1), ARG, "padding")
    refused(lib, f(view(F32, 5, 8, strides=(0, 1)), go, ix), ARG, "dense")
    refused(lib, f(view(F32, 5, 8, strides=(4, 1)), go, ix), ARG, "dense")
    refused(lib, f(view(F32, 2 ** 31, 8), go, ix), LIMIT, "2^31")
    refused(lib, f(table, view(F32, 2 ** 31, 8), view(I64, 2 ** 31)), LIMIT, "2^31")


def test_experts(lib):
    sort = lambda *a: lib.thcb200_expert_sort(CONTEXT, *a, None)  # noqa: E731
    e, o = view(I64, 4, 2), view(I64, 8)
    refused(lib, sort(e, o, view(I64, 3), view(I32, 4, 2)), ARG, "I64")
    refused(lib, sort(e, o, view(I64, 3), view(I64, 4, 2, strides=(3, 1))), ARG, "contiguous")
    refused(lib, sort(e, view(I64, 7), view(I64, 3), e), SIZE, "sizes")
    refused(lib, sort(e, o, view(I64, 1), e), LIMIT, "experts")
    refused(lib, sort(e, o, view(I64, 2049), e), LIMIT, "experts")
    big = view(I64, 2 ** 31)
    refused(lib, sort(big, big, view(I64, 3), big), LIMIT, "2^31")
    for call, wide, narrow in ((lib.thcb200_expert_dispatch, (8, 6), (4, 6)), (lib.thcb200_expert_combine, (4, 6), (8, 6))):
        f = lambda *a: call(CONTEXT, *a, None)  # noqa: E731
        dst, src = view(F32, *wide), view(F32, *narrow)
        refused(lib, f(dst, view(F16, *narrow), e, None), ARG, "floating-point")
        refused(lib, f(dst, src, view(I64, 8), None), ARG, "matrix of I64")
        refused(lib, f(dst, src, e, view(F64, 4, 2)), ARG, "F32")
        refused(lib, f(view(F64, *wide), view(F64, *narrow), e, view(F32, 4, 2)), ARG, "F64")
        refused(lib, f(dst, src, e, view(F32, 2, 4)), SIZE, "differ")
        refused(lib, f(dst, src, view(I64, 5, 2), None), SIZE, "sizes")
        refused(lib, f(view(F32, wide[0], 5), src, e, None), SIZE, "sizes")
        refused(lib, f(view(F32, *wide, strides=(0, 1)), src, e, None), ARG, "dense")
        refused(lib, f(dst, src, view(I64, 2 ** 20, 2 ** 20), None), LIMIT, "2^31")
    f = lambda *a: lib.thcb200_expert_combine_grad(CONTEXT, *a, None)  # noqa: E731
    gr, gw, g, r = view(F32, 8, 6), view(F32, 4, 2), view(F32, 4, 6), view(F32, 8, 6)
    refused(lib, f(view(F32, 7, 6), gw, g, r, e, None), SIZE, "sizes")
    refused(lib, f(gr, gw, view(F32, 5, 6), r, e, None), SIZE, "sizes")
    refused(lib, f(gr, view(F64, 4, 2), g, r, e, None), ARG, "F32")
    refused(lib, f(view(F32, 8, 6, strides=(3, 1)), gw, g, r, e, None), ARG, "dense")


def test_adamw(lib):
    at = HERE.ctypes.data

    def f(dtype=F32, bits=32, tensors=None, n=1, **hyper):
        t = tensors or [Tensor(at, at + 1024, at + 256, at + 512, at + 768, at + 800, None, 4)]
        args = Args(**{**dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0, grad_scale=1, step=1), **hyper})
        return lib.thcb200_adamw(CONTEXT, dtype, bits, (Tensor * len(t))(*t), n, C.byref(args), None)

    refused(lib, f(dtype=I32), ARG, "floating-point")
    refused(lib, f(bits=16), ARG, "32 or 8")
    refused(lib, f(dtype=F64, bits=8), UNSUPPORTED, "half and float")
    refused(lib, f(n=-1), ARG, "null argument")
    nan = float("nan")
    for bad in (dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=nan), dict(eps=-1.0), dict(lr=nan), dict(lr=-1.0), dict(step=0)):
        refused(lib, f(**bad), ARG, "adamw")
    refused(lib, f(tensors=[Tensor(at, at + 1024, at + 256, None, None, None, None, 4)]), ARG, "null pointer")
    refused(lib, f(bits=8, tensors=[Tensor(at, at + 1024, at + 256, at + 512, None, None, None, 4)]), ARG, "null pointer")
    refused(lib, f(tensors=[Tensor(at, at + 1024, at + 256, at + 512, None, None, None, -4)]), SIZE, "negative")
    refused(lib, f(tensors=[Tensor(at, at + 1024, at + 256, at + 512, None, None, at + 700, 4)]), ARG, "half parameters")
    refused(lib, f(dtype=F16, n=2, tensors=[Tensor(at, at + 1024, at + 256, at + 512, None, None, at + 700, 4),
                                            Tensor(at + 2000, at + 1024, at + 2256, at + 2512, None, None, None, 4)]), ARG, "has no master")
    # the second moment ends inside the first; a tensor listed twice; in either order
    refused(lib, f(tensors=[Tensor(at, at + 1024, at + 256, at + 268, None, None, None, 4)]), ARG, "shares memory")
    one = Tensor(at, at + 1024, at + 256, at + 512, None, None, None, 4)
    for pair in ([one, Tensor(at, at + 1024, at + 2256, at + 2512, None, None, None, 4)],
                 [one, Tensor(at + 3000, at + 1024, at + 252, at + 2512, None, None, None, 4)]):
        refused(lib, f(tensors=pair, n=2), ARG, "shares memory")
        refused(lib, f(tensors=pair[::-1], n=2), ARG, "shares memory")


def test_adamw_gradients_apart_from_what_is_written(lib):
    """A gradient inside a written array is refused wherever the lists lie; gradients may share memory with one another."""
    at = HERE.ctypes.data

    def f(*tensors):
        args = Args(1e-3, 0.9, 0.99, 1e-8, 0, 1, 1)
        return lib.thcb200_adamw(CONTEXT, F32, 32, (Tensor * len(tensors))(*tensors), len(tensors), C.byref(args), None)

    for grad in (0, 8, 256, 264, 512, 524):
        refused(lib, f(Tensor(at, at + grad, at + 256, at + 512, None, None, None, 4)), ARG, "shares memory")
        refused(lib, f(Tensor(at, at + 1024, at + 256, at + 512, None, None, None, 4),
                       Tensor(at + 2048, at + grad, at + 2304, at + 2560, None, None, None, 4)), ARG, "shares memory")


def test_large_kernel_arguments_fit():
    """The list of an AdamW launch travels in the kernel's arguments, of which CUDA takes 32764 bytes."""
    entry = 9 * 8
    assert 8 + 320 * entry + 10 * 8 <= 32764


def test_list_calls_are_prepared_before_other_threads_see_them():
    """A function without its C prototype takes no numbers (ctypes.ArgumentError): it may not be in the table of prepared calls yet
    when its prototype is set, or another host thread's first step finds it there."""
    from cutorch_b200 import thc

    class Function:
        prepared = None

        def __setattr__(self, name, value):
            if name in ("argtypes", "restype"):
                assert not state._calls, f"{name} is set on a call that other threads may take"
            object.__setattr__(self, name, value)

        def __call__(self, *args):
            self.prepared = len(self.argtypes)

    class State:
        ptr, _calls, function = 1, {}, Function()

        def fn(self, kind, name):
            return self.function

        def _failed(self):
            return 0

    class Handle:
        def __init__(self, kind):
            self.state, self.kind, self.ptr = state, kind, 8

    state = State()
    lists = [thc.TensorList([Handle(k)]) for k in ("Float", "Float", "Char", "Byte", "Float", "Float")]
    lists[0].adamwValues(*lists[1:])
    assert state.function.prepared == 8 and list(state._calls.values()) == [state.function]
    lists[0].adamwValues(*lists[1:])

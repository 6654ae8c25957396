"""Tokens sorted by expert and back (THCudaLongTensor_expertSort, THCTensor_(expertDispatch), expertCombine,
expertCombineGrad) against plain implementations in 64 bits."""
import numpy as np
import pytest

from cutorch_b200 import thc
from common import FP_KINDS, NP_OF_KIND, assert_bit_equal, rng, to_device
from oracle import rows_oracle as ro
from test_embedding_gpu import U_ACC, U_OUT, take_errors

pytestmark = pytest.mark.gpu

ACC = {"Half": np.float32, "Float": np.float32, "Double": np.float64}


def sort(state, expert, experts):
    slot, order, offsets = (thc.Tensor.new(state, "Long") for _ in range(3))
    slot.expertSort(order, offsets, to_device(state, expert), experts)
    return slot, order, offsets


def check_sort(state, expert, experts):
    got = [t.numpy() for t in sort(state, expert, experts)]
    for g, w, what in zip(got, ro.expert_sort(expert, experts), ("slot", "order", "offsets")):
        assert_bit_equal(g, w, what)


# choices: the pair count, one CTA, and the tiled passes, at and around their borders
@pytest.mark.parametrize("tokens,chosen", [(1, 1), (1, 8), (32, 8), (257, 1), (33, 8), (512, 8), (4097, 1), (2048, 2), (3001, 7)])
@pytest.mark.parametrize("experts", [1, 2, 17, 128, 255, 256, 1000, 2047])
def test_sort(state, tokens, chosen, experts):
    check_sort(state, rng("sort", tokens, chosen, experts).integers(0, experts + 1, (tokens, chosen)), experts)


@pytest.mark.parametrize("tokens", [9, 300, 6000])
def test_sort_of_one_expert_none_and_bad_ones(state, tokens):
    take_errors(state)
    check_sort(state, np.full((tokens, 2), 3), 5)
    check_sort(state, np.zeros((tokens, 2), np.int64), 5)
    assert take_errors(state) == 0
    bad = rng("bad experts", tokens).integers(-2, 8, (tokens, 2))
    check_sort(state, bad, 5)
    assert take_errors(state) == int(((bad < 0) | (bad > 5)).sum())


def test_sort_without_choices_and_of_strided_tensors(state):
    dummy = to_device(state, np.zeros(1, np.int64))
    slot, order = (thc.Tensor.wrap(state, "Long", dummy.data_ptr, (0,)) for _ in range(2))
    offsets = thc.Tensor.new(state, "Long")
    slot.expertSort(order, offsets, thc.Tensor.wrap(state, "Long", dummy.data_ptr, (0,)), 4)
    assert_bit_equal(offsets.numpy(), np.zeros(5, np.int64))
    check_sort(state, rng("strided").integers(0, 6, (8, 90)).T, 5)
    # results that are views of larger tensors
    expert = rng("views").integers(0, 6, (30, 4))
    base = to_device(state, np.full((30, 6), -7, np.int64))
    order, offsets = thc.Tensor.new(state, "Long"), thc.Tensor.new(state, "Long")
    base.narrow(1, 1, 4).expertSort(order, offsets, to_device(state, expert), 5)
    want = np.full((30, 6), -7, np.int64)
    want[:, 1:5] = ro.expert_sort(expert, 5)[0]
    assert_bit_equal(base.numpy(), want)


def routed(r, tokens, chosen, experts, dropped=0.2):
    e = np.stack([r.permutation(experts)[:chosen] + 1 for _ in range(tokens)])
    e[r.random(e.shape) < dropped] = 0
    return e


CASES = [("Half", 1, 8, 8), ("Half", 37, 4, 64), ("Half", 50, 3, 1001), ("Float", 1, 1, 1), ("Float", 33, 5, 36), ("Float", 20, 9, 1021),
         ("Float", 300, 2, 2048), ("Double", 18, 6, 10), ("Double", 12, 2, 33), ("Half", 9, 2, 5000)]


@pytest.mark.parametrize("kind,tokens,chosen,width", CASES)
@pytest.mark.parametrize("weighted", [False, True])
def test_rows_to_the_experts_and_back(state, kind, tokens, chosen, width, weighted):
    r = rng("rows", kind, tokens, chosen, width)
    expert = routed(r, tokens, chosen, 16)
    slot, order, offsets = sort(state, expert, 16)
    s, o = slot.numpy(), order.numpy()
    live = int(offsets.numpy()[-1])
    x = r.standard_normal((tokens, width)).astype(NP_OF_KIND[kind])
    w = r.standard_normal((tokens, chosen)).astype(ACC[kind])
    dw = to_device(state, w) if weighted else None
    # dispatch: rows behind the last place are left as they were
    before = r.standard_normal((tokens * chosen + 2, width)).astype(NP_OF_KIND[kind])
    rows = to_device(state, before)
    rows.expertDispatch(to_device(state, x), slot, dw)
    want = before.copy()
    flat = o[:live] - 1
    moved = x[flat // chosen]
    if weighted:
        moved = (moved.astype(ACC[kind]) * w.reshape(-1)[flat, None]).astype(x.dtype)
    want[:live] = moved
    assert_bit_equal(rows.numpy(), want, "dispatched rows")
    # combine
    y = thc.Tensor.new(state, kind)
    answers = r.standard_normal((tokens * chosen, width)).astype(NP_OF_KIND[kind])
    y.expertCombine(to_device(state, answers), slot, dw)
    want, size = ro.combine(answers, s, w if weighted else None)
    # per addend a rounding of the product and one of the running sum (here and in the 64-bit sum), and one of the result
    tol = U_OUT[kind] * np.abs(want) + (chosen + 1) * (U_ACC[kind] + 2.0 ** -53) * size * 1.001 + (2.0 ** -25 if kind == "Half" else 0)
    assert (np.abs(y.numpy().astype(np.float64) - want) <= tol).all()


@pytest.mark.parametrize("kind,tokens,chosen,width", CASES)
@pytest.mark.parametrize("weighted", [False, True])
def test_gradients_of_combine(state, kind, tokens, chosen, width, weighted):
    r = rng("combine grad", kind, tokens, chosen, width)
    slot, order, offsets = sort(state, routed(r, tokens, chosen, 16), 16)
    s, live = slot.numpy(), int(offsets.numpy()[-1])
    g = r.standard_normal((tokens, width)).astype(NP_OF_KIND[kind])
    answers = r.standard_normal((tokens * chosen, width)).astype(NP_OF_KIND[kind])
    w = r.standard_normal((tokens, chosen)).astype(ACC[kind])
    before = r.standard_normal((tokens * chosen, width)).astype(NP_OF_KIND[kind])
    grad_rows, grad_weight = to_device(state, before), thc.Tensor.new(state, thc.ACC_KIND[kind])
    grad_rows.expertCombineGrad(grad_weight, to_device(state, g), to_device(state, answers), slot, to_device(state, w) if weighted else None)
    want = before.copy()
    flat = order.numpy()[:live] - 1
    scaled = g[flat // chosen]
    if weighted:
        scaled = (scaled.astype(ACC[kind]) * w.reshape(-1)[flat, None]).astype(g.dtype)
    want[:live] = scaled
    assert_bit_equal(grad_rows.numpy(), want, "rows")
    want, size = np.zeros((tokens, chosen)), np.zeros((tokens, chosen))
    for t, k in np.argwhere(s > 0):
        a, b = answers[s[t, k] - 1].astype(np.float64), g[t].astype(np.float64)
        want[t, k], size[t, k] = a @ b, np.abs(a) @ np.abs(b)
    # at most `width` products and additions, each rounded in the accumulator (and in the 64-bit product); the result is
    # rounded to the weights' type
    tol = np.finfo(ACC[kind]).eps / 2 * np.abs(want) + 2 * width * (U_ACC[kind] + 2.0 ** -53) * size
    assert (np.abs(grad_weight.numpy() - want) <= tol).all()


def test_only_one_of_the_gradients(state):
    r = rng("one gradient")
    slot, _, _ = sort(state, routed(r, 20, 3, 8), 8)
    g, a = (to_device(state, r.standard_normal(sh).astype(np.float32)) for sh in ((20, 32), (60, 32)))
    w = to_device(state, r.standard_normal((20, 3)).astype(np.float32))
    both_rows, both_weight = to_device(state, np.zeros((60, 32), np.float32)), thc.Tensor.new(state, "Float")
    both_rows.expertCombineGrad(both_weight, g, a, slot, w)
    rows = to_device(state, np.zeros((60, 32), np.float32))
    rows.expertCombineGrad(None, g, a, slot, w)
    assert_bit_equal(rows.numpy(), both_rows.numpy())
    weight = thc.Tensor.new(state, "Float")
    import ctypes as C
    f = state.fn("Float", "expertCombineGrad")
    f.argtypes, f.restype = [C.c_void_p] * 7, None
    f(state.ptr, None, weight.ptr, g.ptr, a.ptr, slot.ptr, w.ptr)
    state.check()
    assert_bit_equal(weight.numpy(), both_weight.numpy())


def test_layouts(state):
    """Broadcast, strided and transposed operands, and results that are windows."""
    r = rng("layouts")
    slot, order, offsets = sort(state, routed(r, 30, 3, 8), 8)
    s, live = slot.numpy(), int(offsets.numpy()[-1])
    token = (order.numpy()[:live] - 1) // 3
    for x, dx in (((lambda a: (a, to_device(state, a)))(r.standard_normal((24, 30)).astype(np.float32).T)),
                  ((lambda a: (a, to_device(state, a)))(r.standard_normal((30, 25)).astype(np.float32)[:, 1:])),
                  ((lambda a: (np.broadcast_to(a, (30, 24)), to_device(state, a).expand(30, 24)))(r.standard_normal((1, 24)).astype(np.float32))),
                  ((lambda a: (np.broadcast_to(a, (30, 24)), to_device(state, a).expand(30, 24)))(r.standard_normal((1, 1)).astype(np.float32)))):
        rows = thc.Tensor.new(state, "Float")
        rows.expertDispatch(dx, slot, None)
        assert_bit_equal(rows.numpy()[:live], np.ascontiguousarray(x[token]))
        y = thc.Tensor.new(state, "Float")
        y.expertCombine(rows, slot, None)
        # each addend is x itself: k of them add exactly up to one rounding
        want = (x.astype(np.float64) * (s > 0).sum(1)[:, None]).astype(np.float32)
        assert_bit_equal(y.numpy(), want)
        gw, gr = thc.Tensor.new(state, "Float"), to_device(state, np.zeros((90, 24), np.float32))
        gr.expertCombineGrad(gw, dx, rows, slot, None)
        assert_bit_equal(gr.numpy()[:live], np.ascontiguousarray(x[token]))
    base = to_device(state, np.full((90, 30), 3.0, np.float32))
    x = r.standard_normal((30, 24)).astype(np.float32)
    base.narrow(1, 5, 24).expertDispatch(to_device(state, x), slot, None)
    want = np.full((90, 30), 3.0, np.float32)
    want[:live, 5:29] = x[token]
    assert_bit_equal(base.numpy(), want)
    flipped = to_device(state, np.full((24, 90), 3.0, np.float32))
    flipped.transpose(0, 1).expertDispatch(to_device(state, x), slot, None)
    want = np.full((24, 90), 3.0, np.float32)
    want[:, :live] = x[token].T
    assert_bit_equal(flipped.numpy(), want)


def test_slots_beyond_the_rows_are_skipped_and_counted(state):
    x = np.arange(12, dtype=np.float32).reshape(3, 4)
    slot = to_device(state, np.array([[1, 9], [0, 2], [-4, 6]]))
    rows = to_device(state, np.full((6, 4), 8.0, np.float32))
    take_errors(state)
    rows.expertDispatch(to_device(state, x), slot, None)
    want = np.full((6, 4), 8.0, np.float32)
    want[0], want[1], want[5] = x[0], x[1], x[2]
    assert_bit_equal(rows.numpy(), want)
    assert take_errors(state) == 2
    y = thc.Tensor.new(state, "Float")
    y.expertCombine(rows, slot, None)
    assert_bit_equal(y.numpy(), x)
    assert take_errors(state) == 2
    gw, gr = thc.Tensor.new(state, "Float"), to_device(state, np.zeros((6, 4), np.float32))
    gr.expertCombineGrad(gw, to_device(state, x), rows, slot, None)
    assert take_errors(state) == 2
    assert_bit_equal(gw.numpy(), np.array([[x[0] @ x[0], 0], [0, x[1] @ x[1]], [0, x[2] @ x[2]]], np.float32))


def test_a_token_nobody_takes_gets_zeros_even_beside_infinities(state):
    rows = to_device(state, np.full((4, 8), np.inf, np.float16))
    y = to_device(state, np.full((2, 8), np.nan, np.float16))
    y.expertCombine(rows, to_device(state, np.zeros((2, 2), np.int64)), to_device(state, np.full((2, 2), np.nan, np.float32)))
    assert_bit_equal(y.numpy(), np.zeros((2, 8), np.float16))


def test_refusals(state):
    r = rng("refusals")
    f = lambda *sh: to_device(state, np.ones(sh, np.float32))  # noqa: E731
    slot = to_device(state, np.array([[1, 2], [3, 4]]))
    new = lambda: thc.Tensor.new(state, "Float")  # noqa: E731
    x = f(2, 8)
    with pytest.raises(thc.THCError, match="row for each row"):
        new().expertDispatch(f(3, 8), slot, None)
    with pytest.raises(thc.THCError, match="weight and slot"):
        new().expertDispatch(x, slot, f(2, 3))
    with pytest.raises(thc.THCError, match="weight and slot"):
        new().expertCombine(f(4, 8), slot, f(4))
    with pytest.raises(thc.THCError, match="vector or a matrix"):
        new().expertCombine(f(4, 8), to_device(state, np.ones((1, 2, 2), np.int64)), None)
    both = f(6, 8)
    with pytest.raises(thc.THCError, match="shares memory"):
        both.narrow(0, 0, 4).expertDispatch(both.narrow(0, 3, 2), slot, None)
    with pytest.raises(thc.THCError, match="shares memory"):
        both.narrow(0, 0, 2).expertCombine(both, slot, None)
    with pytest.raises(thc.THCError, match="shares memory"):
        both.expertCombineGrad(None, x, both, slot, None)
    with pytest.raises(thc.THCError, match="share memory"):
        f(1, 8).expand(4, 8).expertDispatch(x, slot, None)
    long = lambda: thc.Tensor.new(state, "Long")  # noqa: E731
    expert = to_device(state, r.integers(1, 4, (5, 2)))
    for n in (0, -1, 2048):
        with pytest.raises(thc.THCError, match="xperts"):
            long().expertSort(long(), long(), expert, n)
    with pytest.raises(thc.THCError, match="different tensors"):
        expert.expertSort(long(), long(), expert, 3)
    with pytest.raises(TypeError, match="Float"):
        thc.Tensor.new(state, "Half").expertCombine(to_device(state, np.ones((4, 8), np.float16)), slot, to_device(state, np.ones((2, 2))))


def test_a_result_that_is_an_argument_is_refused_as_it_was(state):
    a = np.arange(16, dtype=np.float32).reshape(2, 8)
    x, rows, w = to_device(state, a), to_device(state, np.ones((4, 8), np.float32)), to_device(state, np.ones((2, 2), np.float32))
    slot = to_device(state, np.array([[1, 2], [3, 4]]))
    for call in (lambda: x.expertDispatch(x, slot, None), lambda: w.expertDispatch(x, slot, w), lambda: rows.expertCombine(rows, slot, None),
                 lambda: w.expertCombine(rows, slot, w), lambda: x.expertCombineGrad(w, x, rows, slot, w),
                 lambda: rows.expertCombineGrad(None, x, rows, slot, w), lambda: thc.Tensor.new(state, "Float").expertCombineGrad(x, x, rows, slot, w)):
        with pytest.raises(thc.THCError, match="shares memory"):
            call()
    for t, want in ((x, a), (rows, np.ones((4, 8), np.float32)), (w, np.ones((2, 2), np.float32))):
        assert_bit_equal(t.numpy(), want)


@pytest.mark.parametrize("n", [4096, 4097, 8192, 8193, 16385, 32769, 65536, 65537])
@pytest.mark.parametrize("experts", [1, 2, 300, 511, 512])
def test_sort_at_its_borders(state, n, experts):
    expert = rng("sort borders", n, experts).integers(0, experts + 1, n)
    long = lambda: thc.Tensor.new(state, "Long")  # noqa: E731
    slot, order, offsets = long(), long(), long()
    slot.expertSort(order, offsets, to_device(state, expert), experts)
    routed = np.argsort(np.where(expert == 0, experts + 1, expert), kind="stable")[:np.count_nonzero(expert)]
    want = np.zeros(n, np.int64)
    want[routed] = np.arange(1, routed.size + 1)
    assert (slot.numpy() == want).all()
    assert (order.numpy() == np.concatenate([routed + 1, np.zeros(n - routed.size, np.int64)])).all()
    assert (offsets.numpy() == np.array([np.count_nonzero((expert > 0) & (expert <= e)) for e in range(experts + 1)])).all()


# rows of single elements: dispatch, combine and its gradient at the borders of a lane's elements, with strided token rows
@pytest.mark.parametrize("kind", ["Half", "Float", "Double"])
@pytest.mark.parametrize("width", [1, 31, 127, 129, 255, 257, 261, 515])
@pytest.mark.parametrize("chosen", [1, 3, 9])
def test_rows_of_single_elements(state, kind, width, chosen):
    r = rng("single rows", kind, width, chosen)
    dt, wt = {"Half": (np.float16, np.float32), "Float": (np.float32, np.float32), "Double": (np.float64, np.float64)}[kind]
    tokens = 11
    slot = r.permutation(tokens * chosen).reshape(tokens, chosen) + 1
    slot[r.random(slot.shape) < 0.2] = 0
    x, rows = r.integers(-4, 5, (tokens, 2 * width)).astype(dt), r.integers(-4, 5, (tokens * chosen, width)).astype(dt)
    weight = r.integers(1, 4, slot.shape).astype(wt)                       # small whole numbers: every product and sum is exact
    dslot, dweight = to_device(state, slot), to_device(state, weight)
    for how in ("narrow", "every other"):
        dx = to_device(state, x).narrow(1, 0, width) if how == "narrow" else to_device(state, x.reshape(tokens, width, 2)).select(2, 0)
        hx = x[:, :width] if how == "narrow" else x.reshape(tokens, width, 2)[:, :, 0]
        out = to_device(state, np.full_like(rows, 7))
        out.expertDispatch(dx, dslot, dweight)
        want = np.full_like(rows, 7)
        want[slot[slot > 0] - 1] = (hx[:, None, :] * weight[:, :, None].astype(dt))[slot > 0]
        assert (out.numpy() == want).all()
        gr, gw = to_device(state, np.full_like(rows, 7)), thc.Tensor.new(state, "Double" if kind == "Double" else "Float")
        gr.expertCombineGrad(gw, dx, to_device(state, rows), dslot, dweight)
        assert (gr.numpy() == want).all()
        full = rows[np.maximum(slot, 1) - 1].astype(np.float64) * (slot > 0)[:, :, None]
        assert (gw.numpy() == (full * hx[:, None, :].astype(np.float64)).sum(-1)).all()
    y = thc.Tensor.new(state, kind)
    y.expertCombine(to_device(state, rows), dslot, dweight)
    assert (y.numpy() == (full * weight[:, :, None]).sum(1)).all()

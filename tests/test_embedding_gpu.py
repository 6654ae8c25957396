"""Rows of an embedding table scaled on the way out, and the table's gradient (THCTensor_(embedding), embeddingAccGrad)
against a plain implementation in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from cutorch_b200 import thc
from common import FP_KINDS, NP_OF_KIND, assert_bit_equal, rng, to_device
from oracle import rows_oracle as ro

pytestmark = pytest.mark.gpu

U_OUT = {"Half": 2.0 ** -11, "Float": 2.0 ** -24, "Double": 2.0 ** -53}     # half a step of the element type
U_ACC = {"Half": 2.0 ** -24, "Float": 2.0 ** -53, "Double": 2.0 ** -53}     # half a step of its accumulator


def take_errors(state):
    count = C.c_int64()
    f = state.lib.thcb200_take_index_errors
    f.argtypes = [C.c_void_p, C.POINTER(C.c_int64), C.c_void_p]
    assert f(C.c_void_p(state.context), C.byref(count), C.c_void_p(state.stream)) == 0
    return count.value


def positions(r, n, rows, how):
    if how == "same":
        return np.full(n, rows, np.int64)
    if how == "two":
        return r.integers(1, 3, n).clip(1, rows)
    if how == "frequencies":
        return np.exp(r.random(n) * np.log(rows + 1)).astype(np.int64).clip(1, rows)
    return r.integers(1, rows + 1, n)


def check_grad(state, kind, rows, width, index, scale, padding, accumulate, go=None, table=None, device_go=None, device_table=None):
    r = rng("embedding grad", kind, rows, width, index.size)
    dt = NP_OF_KIND[kind]
    go = r.standard_normal(index.shape + (width,)).astype(dt) if go is None else go
    table = r.standard_normal((rows, width)).astype(dt) if table is None else table
    dgo = to_device(state, go) if device_go is None else device_go
    dtab = to_device(state, table) if device_table is None else device_table
    dix = to_device(state, index)
    take_errors(state)
    dtab.embeddingAccGrad(dgo, dix, scale, padding, accumulate)
    got = dtab.numpy()
    want, size, count = ro.embedding_grad(table, go, index, scale, padding, accumulate)
    # one rounding of the result; per addend a rounding of the running sum, three more for the scale (itself rounded to
    # the accumulator) and the join with what was there, and as many of the 64-bit sum this is compared with; half results
    # below the normal range are off by up to 2^-25
    tol = U_OUT[kind] * np.abs(want) + (count[:, None] + 3) * (U_ACC[kind] + 2.0 ** -53) * size * 1.001 + (2.0 ** -25 if kind == "Half" else 0)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (np.max(err - tol), np.argwhere(err > tol)[0])
    untouched = count == 0
    assert_bit_equal(got[untouched], table[untouched] if accumulate else np.zeros_like(table[untouched]), "rows no token names")
    bad = (index < 1) | (index > rows)
    assert take_errors(state) == int(bad.sum())
    return got


@pytest.mark.parametrize("kind", FP_KINDS)
@pytest.mark.parametrize("width", [1, 5, 8, 64, 1001, 2048])
@pytest.mark.parametrize("tokens", [1, 3, 100, 1025])
def test_rows_are_scaled_and_rounded_once(state, kind, width, tokens):
    r = rng("embedding", kind, width, tokens)
    w = r.standard_normal((77, width)).astype(NP_OF_KIND[kind])
    ix = r.integers(1, 78, tokens)
    out = thc.Tensor.new(state, kind)
    out.embedding(to_device(state, w), to_device(state, ix), 0.3)
    assert_bit_equal(out.numpy(), ro.embedding(w, ix, 0.3)[0])


def test_positions_of_any_shape_and_stride(state):
    r = rng("embedding shapes")
    w = r.standard_normal((40, 24)).astype(np.float32)
    for ix in (r.integers(1, 41, (3, 4)), r.integers(1, 41, (2, 3, 5)), r.integers(1, 41, 40)[::3], r.integers(1, 41, (6, 8)).T):
        out = thc.Tensor.new(state, "Float")
        out.embedding(to_device(state, w), to_device(state, ix), 2.0)
        assert out.sizes == list(ix.shape) + [24]
        assert_bit_equal(out.numpy(), ro.embedding(w, ix, 2.0)[0])


@pytest.mark.parametrize("layout", ["transposed", "padded", "offset", "expanded"])
def test_tables_of_other_layouts(state, layout):
    r = rng("embedding layouts", layout)
    ix = r.integers(1, 31, 50)
    if layout == "transposed":
        w = r.standard_normal((16, 30)).astype(np.float32).T
    elif layout == "padded":
        w = r.standard_normal((30, 21)).astype(np.float32)[:, :16]
    else:
        w = r.standard_normal((30, 17)).astype(np.float32)[:, 1:]
    dw = to_device(state, w)
    if layout == "expanded":
        w = np.broadcast_to(w[:1], w.shape)
        dw = to_device(state, np.ascontiguousarray(w[:1])).expand(30, 16)
    out = thc.Tensor.new(state, "Float")
    out.embedding(dw, to_device(state, ix), 1.5)
    assert_bit_equal(out.numpy(), ro.embedding(w, ix, 1.5)[0])


def test_result_view_keeps_its_layout_and_neighbours(state):
    r = rng("embedding result view")
    w, ix = r.standard_normal((9, 12)).astype(np.float32), r.integers(1, 10, 7)
    base = np.full((7, 20), 5.0, np.float32)
    for columns in (slice(4, 16), slice(3, 15)):
        dbase = to_device(state, base)
        view = dbase.narrow(1, columns.start, 12)
        view.embedding(to_device(state, w), to_device(state, ix), 1.0)
        want = base.copy()
        want[:, columns] = w[ix - 1]
        assert_bit_equal(dbase.numpy(), want)
    dbase = to_device(state, np.full((12, 7), 5.0, np.float32))
    dbase.transpose(0, 1).embedding(to_device(state, w), to_device(state, ix), 1.0)     # result columns, not rows, are dense
    assert_bit_equal(dbase.numpy(), w[ix - 1].T)


def test_positions_out_of_range_leave_their_rows(state):
    w = np.arange(12, dtype=np.float32).reshape(4, 3)
    out = to_device(state, np.full((5, 3), 9.0, np.float32))
    take_errors(state)
    out.embedding(to_device(state, w), to_device(state, np.array([1, 0, 5, -2 ** 62, 4])), 1.0)
    assert_bit_equal(out.numpy(), np.stack([w[0], [9] * 3, [9] * 3, [9] * 3, w[3]]).astype(np.float32))
    assert take_errors(state) == 3


def test_special_values_pass_through(state):
    w = np.array([[np.inf, -np.inf, np.nan, -0.0, 6e-8, 65504.0, 1, 2]], np.float16)
    out = thc.Tensor.new(state, "Half")
    out.embedding(to_device(state, w), to_device(state, np.array([1, 1])), 2.0)
    assert_bit_equal(out.numpy(), np.repeat((w.astype(np.float32) * 2).astype(np.float16), 2, 0))


# tokens: the pair count, one CTA's radix passes, and the tiled passes, at and around their borders
@pytest.mark.parametrize("tokens", [1, 2, 31, 256, 257, 1000, 4096, 4097, 9001])
@pytest.mark.parametrize("how", ["uniform", "same", "two", "frequencies"])
def test_gradient_sums_tokens_of_a_row(state, tokens, how):
    for kind, rows, width, accumulate in (("Float", 300, 8, 0), ("Half", 1000, 33, 1), ("Half", 70000, 16, 0)):
        ix = positions(rng("tokens", tokens, how, rows), tokens, rows, how)
        check_grad(state, kind, rows, width, ix, 0.75, 0, accumulate)


# rows with so many tokens that their partial sums are joined in sections, next to rows with few
@pytest.mark.parametrize("kind", FP_KINDS)
@pytest.mark.parametrize("width", [5, 72, 1040])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_gradient_of_rows_with_very_many_tokens(state, kind, width, accumulate):
    r = rng("sections", width, accumulate)
    ix = r.integers(1, 41, 12011)
    ix[r.random(ix.size) < 0.5] = 17
    ix[r.random(ix.size) < 0.2] = 18
    got = check_grad(state, kind, 40, width, ix, 1.5, 0, accumulate)
    assert_bit_equal(check_grad(state, kind, 40, width, ix, 1.5, 0, accumulate), got, "the same call again")


@pytest.mark.parametrize("kind", FP_KINDS)
@pytest.mark.parametrize("width", [1, 3, 64, 1001, 2056])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_gradient_widths_types_and_accumulation(state, kind, width, accumulate):
    ix = positions(rng("widths", width), 700, 90, "frequencies")
    check_grad(state, kind, 90, width, ix, -1.25, 3, accumulate)


def test_gradient_leaves_out_padding_and_positions_out_of_range(state):
    ix = rng("bad").integers(-3, 60, 5000)
    ix[7] = -2 ** 63
    ix[8] = 2 ** 63 - 1
    for padding in (0, 1, 17, 50):
        check_grad(state, "Float", 50, 12, ix, 1.0, padding, 1)
        check_grad(state, "Float", 50, 12, ix[:200], 1.0, padding, 0)
    check_grad(state, "Float", 50, 12, np.zeros(300, np.int64), 1.0, 0, 0)      # no token has a row
    check_grad(state, "Float", 50, 12, np.full(300, 4), 1.0, 4, 0)              # every token is padding


def test_gradient_without_tokens(state):
    for accumulate in (0, 1):
        table = to_device(state, np.ones((5, 8), np.float32))
        go = thc.Tensor.wrap(state, "Float", table.data_ptr, (0, 8))
        table.embeddingAccGrad(go, thc.Tensor.wrap(state, "Long", table.data_ptr, (0,)), 1.0, 0, accumulate)
        assert_bit_equal(table.numpy(), np.full((5, 8), float(accumulate), np.float32))


def test_gradient_of_broadcast_and_strided_output_gradients(state):
    r = rng("broadcast")
    ix = r.integers(1, 20, 600)
    row = r.standard_normal((1, 40)).astype(np.float32)
    check_grad(state, "Float", 20, 40, ix, 1.0, 0, 0, go=np.repeat(row, 600, 0), device_go=to_device(state, row).expand(600, 40))
    one = np.ones((1, 1), np.float32)
    check_grad(state, "Float", 20, 40, ix, 1.0, 0, 0, go=np.ones((600, 40), np.float32), device_go=to_device(state, one).expand(600, 40))
    check_grad(state, "Float", 20, 40, ix, 1.0, 0, 0, go=r.standard_normal((40, 600)).astype(np.float32).T)
    check_grad(state, "Float", 20, 40, ix.reshape(20, 30), 1.0, 0, 0, go=r.standard_normal((30, 20, 40)).astype(np.float32).transpose(1, 0, 2))
    # a table that is a window of a larger one, with rows off the 16-byte grid
    base = r.standard_normal((20, 47)).astype(np.float32)
    dbase = to_device(state, base)
    got = check_grad(state, "Float", 20, 40, ix, 1.0, 0, 1, table=base[:, 3:43].copy(), device_table=dbase.narrow(1, 3, 40))
    after = dbase.numpy()
    assert_bit_equal(after[:, 3:43], got)
    assert_bit_equal(after[:, :3], base[:, :3])
    assert_bit_equal(after[:, 43:], base[:, 43:])
    # a transposed table: its columns are dense
    base = r.standard_normal((40, 20)).astype(np.float32)
    check_grad(state, "Float", 20, 40, ix, 1.0, 0, 1, table=base.T.copy(), device_table=to_device(state, base).transpose(0, 1))


def test_gradient_repeats_bit_for_bit(state):
    r = rng("repeat")
    ix = positions(r, 20000, 5000, "frequencies")
    go = to_device(state, r.standard_normal((20000, 72)).astype(np.float16))
    dix = to_device(state, ix)
    first = None
    for _ in range(3):
        table = thc.Tensor.new(state, "Half", 5000, 72)
        table.embeddingAccGrad(go, dix, 1.0, 0, 0)
        first = table.numpy() if first is None else first
        assert_bit_equal(table.numpy(), first)


def test_gradient_matches_differences(state):
    """d/dw of sum(c * embedding(w)) by central differences: the forward is linear, so they are exact up to rounding."""
    r = rng("differences")
    w, ix = r.standard_normal((6, 3)), np.array([2, 2, 5, 1, 2])
    c = r.standard_normal((5, 3))
    table = to_device(state, np.zeros((6, 3)))
    table.embeddingAccGrad(to_device(state, c), to_device(state, ix), 0.7, 0, 0)
    got = table.numpy()
    dix = to_device(state, ix)

    def loss(x):
        out = thc.Tensor.new(state, "Double")
        out.embedding(to_device(state, x), dix, 0.7)
        return float((out.numpy() * c).sum())

    for i in range(6):
        for j in range(3):
            h = np.zeros((6, 3))
            h[i, j] = 0.5
            # twelve products and sums of numbers below 8, each rounded
            assert abs(loss(w + h) - loss(w - h) - got[i, j]) <= 64 * 8 * 2.0 ** -53


def test_refusals(state):
    w = to_device(state, np.ones((4, 6), np.float32))
    ix = to_device(state, np.array([1, 2, 3]))
    go = to_device(state, np.ones((3, 6), np.float32))
    out = thc.Tensor.new(state, "Float")
    with pytest.raises(thc.THCError, match="matrix of rows"):
        out.embedding(to_device(state, np.ones(4, np.float32)), ix, 1.0)
    with pytest.raises(thc.THCError, match="shares memory"):
        w.narrow(0, 0, 3).embedding(w, ix, 1.0)
    with pytest.raises(thc.THCError, match="sizes of index"):
        w.embeddingAccGrad(to_device(state, np.ones((2, 6), np.float32)), ix, 1.0, 0, 0)
    with pytest.raises(thc.THCError, match="sizes of index"):
        w.embeddingAccGrad(to_device(state, np.ones((3, 5), np.float32)), ix, 1.0, 0, 0)
    with pytest.raises(thc.THCError, match="paddingIndex"):
        w.embeddingAccGrad(go, ix, 1.0, 5, 0)
    with pytest.raises(thc.THCError, match="shares memory"):
        w.embeddingAccGrad(w.narrow(0, 0, 3), ix, 1.0, 0, 0)
    with pytest.raises(thc.THCError, match="share memory"):
        to_device(state, np.ones((1, 6), np.float32)).expand(4, 6).embeddingAccGrad(go, ix, 1.0, 0, 0)
    with pytest.raises(TypeError, match="Long"):
        out.embedding(w, go, 1.0)
    assert_bit_equal(w.numpy(), np.ones((4, 6), np.float32))


def test_a_result_that_is_the_table_is_refused_as_it_was(state):
    w = to_device(state, np.arange(24, dtype=np.float32).reshape(4, 6))
    with pytest.raises(thc.THCError, match="shares memory"):
        w.embedding(w, to_device(state, np.array([1, 2, 3, 4, 1])), 1.0)
    assert_bit_equal(w.numpy(), np.arange(24, dtype=np.float32).reshape(4, 6))


# the shares of one cluster's CTAs and the rounds they take, at their borders, and the first size beyond one cluster
@pytest.mark.parametrize("tokens", [4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769, 65536, 65537])
@pytest.mark.parametrize("rows", [300, 131072])
def test_gradient_at_the_borders_of_the_sort(state, tokens, rows):
    r = rng("borders", tokens, rows)
    ix = positions(r, tokens, rows, "frequencies")
    ix[::7] = 0                                        # no row: counted
    check_grad(state, "Float", rows, 4, ix, 1.0, 0, 0)
    check_grad(state, "Half", rows, 3, ix, 0.5, int(ix[1]), 1)


@pytest.mark.parametrize("tokens", [63, 64, 65])
@pytest.mark.parametrize("how", ["uniform", "same", "frequencies"])
@pytest.mark.parametrize("kind", FP_KINDS)
def test_gradient_of_few_tokens(state, tokens, how, kind):
    for width, accumulate in ((7, 0), (257, 1), (1024, 0)):
        check_grad(state, kind, 200, width, positions(rng("few", tokens, how), tokens, 200, how), 1.25, 3, accumulate)


# single elements: narrow teams of lanes, whole warps, columns apart
@pytest.mark.parametrize("kind", FP_KINDS)
@pytest.mark.parametrize("width", [1, 2, 15, 17, 31, 33, 63, 65, 127, 129, 255, 257, 515])
def test_lookup_of_single_elements(state, kind, width):
    r = rng("single", kind, width)
    w = r.standard_normal((50, 2 * width)).astype(NP_OF_KIND[kind])
    ix = r.integers(-1, 53, 77)
    bad = (ix < 1) | (ix > 50)
    rows = np.clip(ix, 1, 50) - 1
    apart = w.reshape(50, width, 2)
    for view, host in ((to_device(state, w).narrow(1, 1, width), w[:, 1:1 + width]), (to_device(state, apart).select(2, 1), apart[:, :, 1])):
        out = to_device(state, np.full((77, width), 5, host.dtype))
        take_errors(state)
        out.embedding(view, to_device(state, ix), 2.0)              # a product with a power of two is exact
        want = np.where(bad[:, None], np.array(5, host.dtype), host[rows] * host.dtype.type(2))
        assert_bit_equal(out.numpy(), want.astype(host.dtype))
        assert take_errors(state) == int(bad.sum())

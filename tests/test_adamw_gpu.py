"""One AdamW step over a list of tensors (THCTensor_(adamw), adamw8bit, adamwValues): the float form against the formula in
64 bits, the 8-bit moments bit for bit against the float arithmetic that defines their codes."""
import numpy as np
import pytest

from cutorch_b200 import thc
from common import FP_KINDS, NP_OF_KIND, assert_bit_equal, rng, to_device
from oracle import rows_oracle as ro

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, grad_scale=0.25)
ACC = {"Half": np.float32, "Float": np.float32, "Double": np.float64}
SIZES = [1, 7, 8, 9, 255, 256, 257, 2047, 2048, 2049, 5000]


def lists(state, *arrays):
    return [thc.TensorList([to_device(state, a) for a in group]) if group is not None else None for group in arrays]


def numpys(tensors):
    return [t.numpy() for t in tensors.tensors]


def inputs(r, kind, n, master=False):
    dt, acc = NP_OF_KIND[kind], ACC[kind]
    p, g = (r.standard_normal(n) * 0.5).astype(dt), (r.standard_normal(n) * 2).astype(dt)
    m, v = (r.standard_normal(n) * 0.3).astype(acc), (r.standard_normal(n) ** 2 * 0.1).astype(acc)
    return p, g, m, v, (p.astype(acc) + (r.standard_normal(n) * 1e-5).astype(acc)) if master else None


def check_param(got, start, g, m0, v0, step, kind, master=None, quotient=12):
    """The new parameter against the formula.  With u half a step of the arithmetic: the moments' sums have terms with at most
    four roundings (first) and six (second), the root halves its argument's relative error; with the scalars' own
    roundings the denominator is within 8 u, its quotient and product within 3 u more, and the two terms of the
    parameter are rounded twice and once more: 12 u for the quotient.  The 8-bit step takes the GPU's approximate root (2 u in
    place of 1) and quotient (2 units in the last place, 4 u, in place of 1): 16 u."""
    u = 2.0 ** -53 if kind == "Double" else 2.0 ** -24
    h = HYPER
    p, m, v, den = ro.adamw(start, g, m0, v0, step, **h)
    gs = np.abs(g.astype(np.float64)) * h["grad_scale"]
    m_size = np.abs(m0.astype(np.float64)) * h["beta1"] + (1 - h["beta1"]) * gs
    size = h["lr"] / (1 - h["beta1"] ** step)
    with np.errstate(invalid="ignore", divide="ignore"):
        tol = u * np.abs(p) + 2 * u * np.abs(start.astype(np.float64)) + size * (4 * u * m_size + quotient * u * np.abs(m)) / den
    tol = 1.01 * tol * (2 if kind == "Double" else 1)          # the formula's own roundings where it has as many bits
    if kind == "Half" and master is None:
        tol = tol + 2.0 ** -11 * (np.abs(p) + tol) + 2.0 ** -25
    err = np.abs(got.astype(np.float64) - p)
    if kind == "Half" and master is None:
        # a first moment over a second of zero can push a value beyond half's range: from 65520, the middle between the largest half
        # (65504) and the next power of two's grid, rounding gives the infinity of the value's sign
        beyond = np.abs(p) - tol >= 65520
        assert (got[beyond] == np.sign(p[beyond]) * np.inf).all()
        err[beyond] = 0
    worst = np.argmax(err - tol)
    assert (err <= tol).all(), (worst, err[worst], tol[worst], got[worst], p[worst])
    return m, v, m_size, u


@pytest.mark.parametrize("kind,master", [("Half", False), ("Half", True), ("Float", False), ("Double", False)])
@pytest.mark.parametrize("step", [1, 2, 1000])
def test_step_of_a_list(state, kind, master, step):
    r = rng("adamw", kind, master, step)
    data = [inputs(r, kind, n, master) for n in SIZES]
    p, g, m, v, w = lists(state, *[[d[k] for d in data] if k < 4 or master else None for k in range(5)])
    p.adamw(g, m, v, step=step, master=w, **HYPER)
    outs = [numpys(x) if x else [None] * len(data) for x in (p, m, v, w)]
    for (p0, g0, m0, v0, w0), p1, m1, v1, w1 in zip(data, *outs):
        start = w0 if master else p0
        mw, vw, m_size, u = check_param(w1 if master else p1, start, g0, m0, v0, step, kind, w0)
        if master:
            assert_bit_equal(p1, w1.astype(np.float16), "the parameter is its master's rounding")
        v_size = vw        # no term of the second moment is negative
        k = 2.02 if kind == "Double" else 1.01
        assert (np.abs(m1 - mw) <= k * 4 * u * m_size).all()
        assert (np.abs(v1 - vw) <= k * 6 * u * v_size).all()
    assert_bit_equal(numpys(g)[4], data[4][1], "gradients are left alone")


@pytest.mark.parametrize("count", [1, 16, 17, 320, 321, 700])
@pytest.mark.parametrize("bits", [32, 8])
def test_lists_of_every_length(state, count, bits):
    r = rng("lists", count)
    n = r.integers(1, 400, count)
    starts = np.concatenate([[0], np.cumsum(n)])
    total = int(starts[-1])
    p, g, m, v, _ = inputs(r, "Float", total)
    flat = {"p": p, "g": g, "m": m, "v": v}
    if bits == 8:
        blocks = -(-n // 256)
        bs = np.concatenate([[0], np.cumsum(blocks)])
        flat["m"], flat["v"] = r.integers(-127, 128, total).astype(np.int8), r.integers(0, 256, total).astype(np.uint8)
        flat["mu"], flat["vu"] = r.random(bs[-1]).astype(np.float32) * 1e-5, r.random(bs[-1]).astype(np.float32) * 1e-11
    dev = {k: to_device(state, a) for k, a in flat.items()}

    def pieces(name):
        at, size = (bs, blocks) if name in ("mu", "vu") else (starts, n)
        return thc.TensorList([dev[name].narrow(0, int(a), int(s)) for a, s in zip(at, size)])

    if bits == 32:
        pieces("p").adamw(pieces("g"), pieces("m"), pieces("v"), step=5, **HYPER)
        check_param(dev["p"].numpy(), p, g, m, v, 5, "Float")
        return
    pieces("p").adamw8bit(pieces("g"), pieces("m"), pieces("v"), pieces("mu"), pieces("vu"), step=5, **HYPER)
    got = {k: t.numpy() for k, t in dev.items()}
    for a, s, b, c in zip(starts, n, bs, blocks):
        w = ro.adamw8(p[a:a + s], g[a:a + s], flat["m"][a:a + s], flat["v"][a:a + s], flat["mu"][b:b + c], flat["vu"][b:b + c], 5, **HYPER)
        for name, want, sl in (("m", w[4], slice(a, a + s)), ("v", w[5], slice(a, a + s)), ("mu", w[6], slice(b, b + c)), ("vu", w[7], slice(b, b + c))):
            assert_bit_equal(got[name][sl], want, name)


@pytest.mark.parametrize("kind,master", [("Half", False), ("Half", True), ("Float", False)])
@pytest.mark.parametrize("step", [1, 77])
@pytest.mark.parametrize("start", ["zero", "random"])
def test_eight_bit_step(state, kind, master, step, start):
    r = rng("adamw8", kind, master, step, start)
    data = []
    for n in SIZES:
        p, g, _, _, w = inputs(r, kind, n, master)
        b = -(-n // 256)
        g[r.random(n) < 0.1] = 0
        if start == "zero":
            cm, cv, um, uv = np.zeros(n, np.int8), np.zeros(n, np.uint8), np.zeros(b, np.float32), np.zeros(b, np.float32)
        else:
            cm, cv = r.integers(-127, 128, n).astype(np.int8), r.integers(0, 256, n).astype(np.uint8)
            um, uv = (r.random(b) / 127 ** 2).astype(np.float32), (r.random(b) * 0.1 / 255 ** 4).astype(np.float32)
        data.append((p, g, cm, cv, um, uv, w))
    p, g, cm, cv, um, uv, w = lists(state, *[[d[k] for d in data] if k < 6 or master else None for k in range(7)])
    p.adamw8bit(g, cm, cv, um, uv, step=step, master=w, **HYPER)
    outs = [numpys(x) if x else [None] * len(data) for x in (p, cm, cv, um, uv, w)]
    mv, vv = (thc.TensorList([thc.Tensor.new(state, "Float") for _ in data]) for _ in range(2))
    mv.adamwValues(vv, cm, cv, um, uv)
    for (p0, g0, cm0, cv0, um0, uv0, w0), p1, cm1, cv1, um1, uv1, w1, mval, vval in zip(data, *outs, numpys(mv), numpys(vv)):
        m0, v0, m, v, km, kv, mu, vu = ro.adamw8(p0, g0, cm0, cv0, um0, uv0, step, **HYPER)
        check_param(w1 if master else p1, w0 if master else p0, g0, m0, v0, step, kind, w0, quotient=16)
        if master:
            assert_bit_equal(p1, w1.astype(np.float16))
        for got, want, what in ((um1, mu, "first unit"), (uv1, vu, "second unit"), (cm1, km, "first code"), (cv1, kv, "second code"),
                                (mval, ro.decode(km, mu, ro.first_value), "first value"), (vval, ro.decode(kv, vu, ro.second_value), "second value")):
            assert_bit_equal(got, want, what)
        # a code's value is one of the two that enclose the moment; one that is not zero stays so below the root
        unit = np.repeat(mu, 256)[:m.size].astype(np.float64)
        k = np.abs(km.astype(np.float64))
        assert (np.abs(mval.astype(np.float64) - m) <= (2 * k + 1.001) * unit).all()
        assert ((v > 0) == (kv > 0)).all()


def test_eight_bit_averages_do_not_stall_and_keep_their_expectation(state):
    """Gradients of constant size: the second moment has to climb from 1/100 of the block's largest to where the gradients put it,
    in steps of 0.1 %, far below the distance of two codes.  The dither's bits are as good as independent over 4096 elements
    and 3000 steps: the mean over the elements is held to five standard deviations of the rounding noise."""
    n, steps = 4096, 3000
    g = np.full(n, 0.5, np.float32)
    g[::256] = 2.0                                               # a block's largest value
    data = [np.zeros(n, np.float32), g, np.zeros(n, np.int8), np.zeros(n, np.uint8), np.zeros(n // 256, np.float32), np.zeros(n // 256, np.float32)]
    data[2][::256], data[3][::256] = 127, 255
    data[4][:], data[5][:] = 2.0 / 127 ** 2, 4.0 / 255.0 ** 4     # the largest are settled, the others start at zero
    p, dg, cm, cv, um, uv = lists(state, *[[d] for d in data])
    for step in range(1, steps + 1):
        p.adamw8bit(dg, cm, cv, um, uv, step=step, lr=0.0, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, grad_scale=1.0)
    mv, vv = (thc.TensorList([thc.Tensor.new(state, "Float")]) for _ in range(2))
    mv.adamwValues(vv, cm, cv, um, uv)
    rest = np.arange(n) % 256 != 0
    m, v = mv.tensors[0].numpy()[rest].astype(np.float64), vv.tensors[0].numpy()[rest].astype(np.float64)
    want_v = 0.25 * (1 - 0.999 ** steps)
    # rounding noise of one step is at most half the distance d of two codes (variance d^2 / 4 at most); an average that forgets
    # with factor b collects variance d^2 / 4 / (1 - b^2)
    code = (want_v / 4.0) ** 0.25 * 255
    d = ((code + 1) ** 4 - code ** 4) * 4.0 / 255 ** 4
    sigma_v = d / 2 / np.sqrt(1 - 0.999 ** 2) / np.sqrt(rest.sum())
    assert abs(v.mean() - want_v) <= 5 * sigma_v, (v.mean(), want_v, sigma_v)
    code = (0.5 / 2.0) ** 0.5 * 127
    d = (2 * code + 1) * 2.0 / 127 ** 2
    sigma_m = d / 2 / np.sqrt(1 - 0.9 ** 2) / np.sqrt(rest.sum())
    assert abs(m.mean() - 0.5) <= 5 * sigma_m, (m.mean(), sigma_m)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_off_the_vector_grid_and_strided_ones(state, bits):
    r = rng("off grid", bits)
    n = 1000
    p, g, m, v, _ = inputs(r, "Float", n)
    cm, cv = r.integers(-127, 128, n).astype(np.int8), r.integers(0, 256, n).astype(np.uint8)
    um, uv = (r.random(4) / 127 ** 2).astype(np.float32), (r.random(4) * 0.1 / 255 ** 4).astype(np.float32)
    states = (m, v) if bits == 32 else (cm, cv, um, uv)
    want = None
    for how in ("aligned", "param off by one", "state off by one", "strided", "transposed"):
        def place(a, this):
            if how == "transposed" and this and a.size == n:
                return to_device(state, a.reshape(40, 25).T.copy()).transpose(0, 1)
            if how == "strided" and this:
                big = np.full((a.size, 2), 9, a.dtype)
                big[:, 0] = a
                return to_device(state, big).select(1, 0)
            if "off by one" in how and this:
                return to_device(state, np.concatenate([[9], a, [9]]).astype(a.dtype)).narrow(0, 1, a.size)
            return to_device(state, a)
        dp, dg = place(p, "state" not in how), place(g, "state" not in how)
        ds = [place(a, "param" not in how) for a in states]
        one = [thc.TensorList([t]) for t in (dp, dg, *ds)]
        (one[0].adamw if bits == 32 else one[0].adamw8bit)(*one[1:], step=3, **HYPER)
        got = [t.numpy().reshape(-1) for t in (dp, *ds)]
        want = want or got
        for a, b in zip(got, want):
            assert_bit_equal(a, b, how)


def test_neighbours_of_a_tensor_are_left_alone(state):
    for n in (1, 100, 257, 2049):
        r = rng("neighbours", n)
        p, g, m, v, _ = inputs(r, "Half", n)
        base = [to_device(state, np.concatenate([np.full(16, 7), a, np.full(16, 7)]).astype(a.dtype)) for a in (p, m, v)]
        one = [thc.TensorList([b.narrow(0, 16, n)]) for b in base]
        one[0].adamw(thc.TensorList([to_device(state, g)]), one[1], one[2], step=1, **HYPER)
        for b in base:
            a = b.numpy()
            assert (a[:16] == 7).all() and (a[-16:] == 7).all()


def test_empty_tensors_in_a_list(state):
    r = rng("empty")
    p, g, m, v, _ = inputs(r, "Float", 10)
    full = [to_device(state, a) for a in (p, g, m, v)]
    hollow = [thc.Tensor.new(state, "Float") for _ in range(4)]
    each = [thc.TensorList([h, f, h]) for h, f in zip(hollow, full)]
    each[0].adamw(*each[1:], step=1, **HYPER)
    check_param(full[0].numpy(), p, g, m, v, 1, "Float")


def test_not_a_number_stays_where_it_is(state):
    r = rng("nan")
    p, g, m, v, _ = inputs(r, "Float", 600)
    g[3], g[300] = np.nan, np.inf
    one = lists(state, [p], [g], [m], [v])
    one[0].adamw(*one[1:], step=1, **HYPER)
    got = one[0].tensors[0].numpy()
    assert np.flatnonzero(~np.isfinite(got)).tolist() == [3, 300]
    # in 8 bits a block shares its unit: the block's moments are lost, the others' are not, nor this step's other parameters
    eight = lists(state, [p], [g], [np.zeros(600, np.int8)], [np.zeros(600, np.uint8)], [np.zeros(3, np.float32)], [np.zeros(3, np.float32)])
    eight[0].adamw8bit(*eight[1:], step=1, **HYPER)
    assert np.flatnonzero(~np.isfinite(eight[0].tensors[0].numpy())).tolist() == [3, 300]
    mv, vv = (thc.TensorList([thc.Tensor.new(state, "Float")]) for _ in range(2))
    mv.adamwValues(vv, *eight[2:])
    for values in (mv, vv):
        a = values.tensors[0].numpy()
        assert np.isfinite(a[512:]).all() and not np.isfinite(a[3]) and not np.isfinite(a[300])


def test_refusals(state):
    r = rng("refusals")
    p, g, m, v, _ = inputs(r, "Float", 20)
    P, G, M, V = lists(state, [p], [g], [m], [v])
    one = lambda *a: thc.TensorList(a)  # noqa: E731
    t = P.tensors[0]
    for bad, match in ((dict(step=0), "count from 1"), (dict(beta1=1.0), "beta1"), (dict(beta2=-0.1), "beta"), (dict(eps=-1.0), "eps"),
                       (dict(lr=float("nan")), "lr")):
        with pytest.raises(thc.THCError, match=match):
            P.adamw(G, M, V, **{**HYPER, "step": 1, **bad})
    with pytest.raises(thc.THCError, match="20 elements|has 19"):
        P.adamw(one(to_device(state, g[:19])), M, V, step=1, **HYPER)
    with pytest.raises(thc.THCError, match="shares? memory"):
        one(t, t).adamw(one(*G.tensors * 2), one(M.tensors[0], to_device(state, m)), one(V.tensors[0], to_device(state, v)), step=1, **HYPER)
    with pytest.raises(thc.THCError, match="shares? memory"):
        P.adamw(G, M, M, step=1, **HYPER)
    long = to_device(state, np.zeros(40, np.float32))
    with pytest.raises(thc.THCError, match="shares? memory"):
        one(long.narrow(0, 0, 20), long.narrow(0, 10, 20)).adamw(
            one(*G.tensors * 2), *[one(*(to_device(state, a) for _ in range(2))) for a in (m, v)], step=1, **HYPER)
    with pytest.raises(thc.THCError, match="masters go with half"):
        P.adamw(G, M, V, master=one(to_device(state, m)), step=1, **HYPER)
    with pytest.raises(thc.THCError, match="shares? memory"):
        one(to_device(state, np.zeros((1, 1), np.float32)).expand(4, 5)).adamw(G, M, V, step=1, **HYPER)
    d = [np.zeros(20), np.zeros(20), np.zeros(20, np.int8), np.zeros(20, np.uint8), np.zeros(1, np.float32), np.zeros(1, np.float32)]
    D = lists(state, *[[a] for a in d])
    with pytest.raises(thc.THCError, match="half and float"):
        D[0].adamw8bit(*D[1:], step=1, **HYPER)
    with pytest.raises(thc.THCError, match="expected 1"):
        P.adamw8bit(G, D[2], D[3], one(to_device(state, np.zeros(2, np.float32))), D[5], step=1, **HYPER)
    with pytest.raises(TypeError, match="Char"):
        P.adamw8bit(G, D[3], D[3], D[4], D[5], step=1, **HYPER)
    with pytest.raises(ValueError, match="lists of"):
        P.adamw(one(*G.tensors * 2), M, V, step=1, **HYPER)
    assert_bit_equal(t.numpy(), p)
    assert_bit_equal(M.tensors[0].numpy(), m)


def test_strided_tensors_of_one_matrix(state):
    """Strided tensors go to the step as copies: columns of one matrix beside one another are a list, the same column twice or
    two that meet are not, nor is a moment or a gradient inside the parameter."""
    r = rng("columns")
    mats = {k: r.standard_normal((33, 12)).astype(np.float32) ** (2 if k == "v" else 1) for k in "pgmv"}
    dev = {k: to_device(state, a) for k, a in mats.items()}
    one = lambda *a: thc.TensorList(a)  # noqa: E731
    column = lambda k, at, n: dev[k].narrow(1, at, n)  # noqa: E731
    split = lambda k: one(column(k, 7, 5), column(k, 0, 4), column(k, 4, 3))  # noqa: E731
    twice = lambda k, *at: one(*[column(k, a, 4) for a in at])  # noqa: E731
    dense = lambda k, n: one(*[to_device(state, mats[k][:, :4]) for _ in range(n)])  # noqa: E731
    own = dense("p", 1)
    for refused in (lambda: twice("p", 0, 0).adamw(dense("g", 2), dense("m", 2), dense("v", 2), step=1, **HYPER),
                    lambda: twice("p", 0, 3).adamw(dense("g", 2), dense("m", 2), dense("v", 2), step=1, **HYPER),
                    lambda: dense("p", 2).adamw(dense("g", 2), twice("m", 2, 5), dense("v", 2), step=1, **HYPER),
                    lambda: twice("p", 0).adamw(dense("g", 1), twice("p", 1), dense("v", 1), step=1, **HYPER),
                    lambda: twice("p", 0).adamw(twice("p", 0), dense("m", 1), dense("v", 1), step=1, **HYPER),
                    lambda: one(dev["p"]).adamw(one(dev["g"]), one(dev["m"]), one(dev["p"].transpose(0, 1)), step=1, **HYPER)):
        with pytest.raises(thc.THCError, match="shares memory"):
            refused()
    assert all((dev[k].numpy() == a).all() for k, a in mats.items())
    own.adamw(dense("g", 1), dense("m", 1), dense("v", 1), step=3, **HYPER)
    twice("p", 0).adamw(twice("g", 0), twice("m", 0), twice("v", 0), step=3, **HYPER)
    assert_bit_equal(dev["p"].numpy()[:, :4].copy(), own.tensors[0].numpy(), "one column list beside a contiguous one")
    dev = {k: to_device(state, a) for k, a in mats.items()}
    split("p").adamw(split("g"), split("m"), split("v"), step=3, **HYPER)
    check_param(dev["p"].numpy().ravel(), *(mats[k].ravel() for k in "pgmv"), 3, "Float")


@pytest.mark.parametrize("count", [79, 80, 81])
def test_tables_of_every_size(state, count):
    test_lists_of_every_length(state, count, 32)
    test_lists_of_every_length(state, count, 8)


def test_values_that_share_a_storage_which_grows(state):
    """The results are windows of one storage, a unit too, and the last of them has to grow: the memory moves, and every tensor of the
    call with it."""
    r = rng("values in one storage")
    sizes = (300, 5000)
    cm, cv = [r.integers(-127, 128, n).astype(np.int8) for n in sizes], [r.integers(0, 256, n).astype(np.uint8) for n in sizes]
    um, uv = ([(r.random(-(-n // 256)) * 1e-5).astype(np.float32) for n in sizes] for _ in range(2))
    m, v, mu, vu = lists(state, cm, cv, um, uv)
    base = to_device(state, np.concatenate([um[0], np.zeros(310, np.float32)]))
    firsts = base.narrow(0, 2, 300), base.narrow(0, 302, 10)
    seconds = [thc.Tensor.new(state, "Float") for _ in sizes]
    units = thc.TensorList([base.narrow(0, 0, 2), mu.tensors[1]])
    thc.TensorList(firsts).adamwValues(thc.TensorList(seconds), m, v, units, vu)
    for t, c, u, value in ((firsts[0], cm[0], um[0], ro.first_value), (firsts[1], cm[1], um[1], ro.first_value),
                           (seconds[0], cv[0], uv[0], ro.second_value), (seconds[1], cv[1], uv[1], ro.second_value)):
        assert_bit_equal(t.numpy(), ro.decode(c, u, value))
    assert_bit_equal(base.numpy()[:302], np.concatenate([um[0], ro.decode(cm[0], um[0], ro.first_value)]))


def test_values_over_an_argument_are_refused_as_it_was(state):
    r = rng("values refused")
    um, uv = (r.random(3).astype(np.float32) for _ in range(2))
    m, v, mu, vu = lists(state, [r.integers(-127, 128, 600).astype(np.int8)], [r.integers(0, 256, 600).astype(np.uint8)], [um], [uv])
    other = thc.TensorList([thc.Tensor.new(state, "Float")])
    for first, second in ((mu, other), (other, mu), (vu, other), (other, vu), (other, other)):
        with pytest.raises(thc.THCError, match="shares memory"):
            first.adamwValues(second, m, v, mu, vu)
    assert_bit_equal(mu.tensors[0].numpy(), um)
    assert_bit_equal(vu.tensors[0].numpy(), uv)
    assert other.tensors[0].numpy().ndim == 0, "an empty tensor still"


@pytest.mark.parametrize("kind", ["Half", "Float"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_whose_moments_are_not_finite_is_not_a_number(state, kind, bad):
    """A unit cannot stand beside an infinite moment: the whole block's moments become NaN, not infinities of either sign beside
    zeros.  Where only the square of a gradient is beyond float, the second moments do."""
    r = rng("not finite")
    n = 1300
    g = r.standard_normal(n).astype(NP_OF_KIND[kind])
    g[300], g[1290] = bad, bad                                  # a block of vectors, and the ragged last one
    if kind == "Float":
        g[600] = 1e25
    one = lists(state, [np.ones(n, g.dtype)], [g], [np.zeros(n, np.int8)], [np.zeros(n, np.uint8)], [np.zeros(6, np.float32)], [np.zeros(6, np.float32)])
    one[0].adamw8bit(*one[1:], step=1, **{**HYPER, "grad_scale": 1.0})
    mv, vv = (thc.TensorList([thc.Tensor.new(state, "Float")]) for _ in range(2))
    mv.adamwValues(vv, *one[2:])
    m, v = mv.tensors[0].numpy(), vv.tensors[0].numpy()
    lost = np.isin(np.arange(n) // 256, [1, 5])
    squares = lost | (np.arange(n) // 256 == 2) if kind == "Float" else lost
    assert np.isnan(m[lost]).all() and np.isfinite(m[~lost]).all()
    assert np.isnan(v[squares]).all() and np.isfinite(v[~squares]).all()
    w = ro.adamw8(np.ones(n, g.dtype), g, *(np.zeros(k, t) for k, t in ((n, np.int8), (n, np.uint8), (6, np.float32), (6, np.float32))), 1,
                  **{**HYPER, "grad_scale": 1.0})
    for got, want in ((one[4], w[6]), (one[5], w[7])):
        np.testing.assert_array_equal(got.tensors[0].numpy(), want)
    assert_bit_equal(one[2].tensors[0].numpy()[~lost], w[4][~lost])
    assert_bit_equal(one[3].tensors[0].numpy()[~squares], w[5][~squares])

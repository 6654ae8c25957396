"""Embedding, expert routing and AdamW used together: a small model's training steps against the same model in 64 bits, recorded
into graphs, on streams of their own, from several host threads, and at sizes whose offsets pass 32 bits."""
import ctypes as C
import threading

import numpy as np
import pytest

from cutorch_b200 import thc
from common import NP_OF_KIND, assert_bit_equal, rng, to_device
from oracle import rows_oracle as ro
from test_embedding_gpu import check_grad
from test_expert_gpu import check_sort

pytestmark = pytest.mark.gpu

V, D, E, K, T = 50, 24, 6, 2, 40
HYPER = dict(lr=5e-3, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.02, grad_scale=1.0)


class Model:
    """Rows of a table go to K of E experts, each of which scales its rows by a vector; the weighted answers are brought back
    and compared with a target: loss = sum of (y - target)^2 / 2.  Parameters: the table and the experts' vectors."""

    def __init__(self, state, kind="Float"):
        r = rng("model")
        self.state, self.kind = state, kind
        new = lambda *sizes: thc.Tensor.new(state, kind, *sizes)  # noqa: E731
        self.table0, self.scale0 = r.standard_normal((V, D)).astype(np.float32), r.standard_normal((E, D)).astype(np.float32)
        self.index, self.target = r.integers(1, V + 1, T), r.standard_normal((T, D)).astype(np.float32)
        self.index[5] = 3                                   # the padding row
        self.expert = np.stack([r.permutation(E)[:K] + 1 for _ in range(T)])
        self.expert[r.random((T, K)) < 0.15] = 0
        self.expert[7] = 0                                  # a token nobody takes
        self.weight = r.random((T, K)).astype(np.float32)
        put = lambda a: to_device(state, a)  # noqa: E731
        self.dindex, self.dexpert, self.dweight, self.dtarget = put(self.index), put(self.expert), put(self.weight), put(self.target)
        self.table, self.scale = put(self.table0), put(self.scale0)
        self.grad_table, self.grad_scale = put(np.zeros((V, D), np.float32)), put(np.zeros((E, D), np.float32))
        self.x, self.y = new(T, D), new(T, D)
        self.rows, self.answers, self.grad_answers, self.grad_rows = (put(np.zeros((T * K, D), np.float32)) for _ in range(4))
        self.grad_weight, self.grad_x, self.grad_y = new(T, K), new(T, D), new(T, D)
        self.slot, self.order, self.offsets = (thc.Tensor.new(state, "Long") for _ in range(3))
        zeros = lambda a: put(np.zeros_like(a))  # noqa: E731
        lists = [[self.table, self.scale], [self.grad_table, self.grad_scale], [zeros(self.table0), zeros(self.scale0)], [zeros(self.table0), zeros(self.scale0)]]
        self.param, self.grad, self.m, self.v = (thc.TensorList(x) for x in lists)
        self.work = put(np.zeros((T * K, D), np.float32))
        self.slot.expertSort(self.order, self.offsets, self.dexpert, E)      # routing is fixed: the offsets are known on the host
        self.at = self.offsets.numpy()
        self.pieces = [(e, int(self.at[e]), int(self.at[e + 1] - self.at[e])) for e in range(E) if self.at[e + 1] > self.at[e]]
        self.views = {k: [(e, t.narrow(0, a, n)) for e, a, n in self.pieces]
                      for k, t in (("rows", self.rows), ("answers", self.answers), ("grad_answers", self.grad_answers), ("grad_rows", self.grad_rows),
                                   ("work", self.work))}
        self.vectors = [self.scale.narrow(0, e, 1).expand(n, D) for e, a, n in self.pieces]
        self.grad_vectors = [self.grad_scale.narrow(0, e, 1) for e, a, n in self.pieces]

    def step(self, number):
        self.x.embedding(self.table, self.dindex, 1.5)
        self.slot.expertSort(self.order, self.offsets, self.dexpert, E)
        self.rows.expertDispatch(self.x, self.slot, None)
        for (_, r), (_, a), s in zip(self.views["rows"], self.views["answers"], self.vectors):
            a.cmul(r, s)
        self.y.expertCombine(self.answers, self.slot, self.dweight)
        self.grad_y.csub(self.y, 1.0, self.dtarget)
        self.grad_answers.expertCombineGrad(self.grad_weight, self.grad_y, self.answers, self.slot, self.dweight)
        for (_, ga), (_, gr), (_, r), (_, w), s, gs in zip(self.views["grad_answers"], self.views["grad_rows"], self.views["rows"], self.views["work"],
                                                          self.vectors, self.grad_vectors):
            gr.cmul(ga, s)
            w.cmul(ga, r)
            gs.sum(w, 0, 1)
        self.grad_x.expertCombine(self.grad_rows, self.slot, None)
        self.grad_table.embeddingAccGrad(self.grad_x, self.dindex, 1.5, 3, 0)
        self.param.adamw(self.grad, self.m, self.v, step=number, **HYPER)

    def wanted(self, steps):
        """The same in 64 bits with torch's automatic gradients: after `steps` steps the parameters, and the last gradients."""
        import torch
        f = lambda a: torch.tensor(a, dtype=torch.float64)  # noqa: E731
        table, scale, weight = f(self.table0).requires_grad_(), f(self.scale0).requires_grad_(), f(self.weight).requires_grad_()
        index, expert = torch.tensor(self.index), torch.tensor(self.expert)
        states = [[np.zeros(p.shape), np.zeros(p.shape)] for p in (table, scale)]
        for number in range(1, steps + 1):
            for p in (table, scale, weight):
                p.grad = None
            x = 1.5 * table[index - 1]
            padded = torch.where((index == 3)[:, None], x.detach(), x)       # no gradient reaches the padding row
            y = sum((expert[:, k:k + 1] > 0) * weight[:, k:k + 1] * scale[(expert[:, k] - 1).clamp(min=0)] * padded for k in range(K))
            ((y - f(self.target)) ** 2).sum().div(2).backward()
            grads = [p.grad.numpy().copy() for p in (table, scale, weight)]
            for p, g, s in zip((table, scale), grads, states):
                new, s[0], s[1], _ = ro.adamw(p.detach().numpy(), g, s[0], s[1], number, **HYPER)
                p.data = torch.from_numpy(new)
        return table.detach().numpy(), scale.detach().numpy(), grads


def close(got, want, what, rel):
    err = np.abs(got.astype(np.float64) - want)
    tol = rel * np.abs(want).max()
    assert (err <= tol).all(), (what, err.max(), tol)


def test_training_steps_against_the_model_in_64_bits(state):
    """Gradients after one step: sums of at most 40 products of four floats, each rounded once (2^-24) and added in double or, for the
    experts' vectors, in double by sum(): 8 roundings in a row per term and 40 terms of at most the largest one's size
    bound a relative error of the largest by 320 * 2^-24 = 2e-5.  A parameter moves by at most lr a step (a quotient of
    averages of at most 1, up to the first steps' 1 / (1 - beta)), so four steps keep it within 4 lr of the start, and what a
    gradient's relative error shifts a quotient by is of the order of that error where the gradient is not small itself; those
    below 1e-3 of the largest are held to the full length of a step."""
    model = Model(state)
    model.step(1)
    _, _, grads = model.wanted(1)
    for got, want, what in ((model.grad_table, grads[0], "table"), (model.grad_scale, grads[1], "vectors"), (model.grad_weight, grads[2], "weights")):
        close(got.numpy(), want, what, 2e-5)
    for number in (2, 3, 4):
        model.step(number)
    table, scale, grads = model.wanted(4)
    for got, want, g, what in ((model.table, table, grads[0], "table"), (model.scale, scale, grads[1], "vectors")):
        small = np.abs(g) < 1e-3 * np.abs(g).max()
        err = np.abs(got.numpy().astype(np.float64) - want)
        assert (err <= np.where(small & (g != 0), 2 * HYPER["lr"] * 4, 1e-4 * HYPER["lr"] * 4 + 4 * 2.0 ** -24 * np.abs(want))).all(), (what, err.max())
    assert np.array_equal(model.grad_table.numpy()[2], np.zeros(D, np.float32)), "the padding row has no gradient"


def test_steps_recorded_into_graphs_that_share_a_context(state):
    """A graph with the whole step replays like the calls; a second graph and eager calls on the same stream in between, and calls
    that need a larger workspace, leave its results alone."""
    import torch
    own = thc.State()
    side = torch.cuda.Stream()
    own.set_stream(side.cuda_stream, 0)
    plain, first, second = Model(own), Model(own), Model(own)
    big = rng("workspace").integers(1, 9, 30000)
    with torch.cuda.stream(side):
        for m in (first, second):
            m.step(1)                                       # kernels loaded, outputs and the workspace sized
        side.synchronize()
        graphs = []
        for m in (first, second):
            for t, a in ((m.table, m.table0), (m.scale, m.scale0)):
                t.copy_from(to_device(own, a))
            for s in (m.m, m.v):
                for t in s.tensors:
                    t.zero()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                m.step(1)
            graphs.append(g)
        plain.step(1)
        graphs[0].replay()
        # a gradient with a much larger workspace replaces the context's between the replays
        table = to_device(own, np.zeros((8, 600), np.float32))
        table.embeddingAccGrad(to_device(own, np.ones((30000, 600), np.float32)), to_device(own, big), 1.0, 0, 0)
        graphs[1].replay()
        side.synchronize()
        assert_bit_equal(table.numpy(), np.repeat(np.bincount(big, minlength=9)[1:, None], 600, 1).astype(np.float32))
        for m in (first, second):
            for a, b, what in ((m.table, plain.table, "table"), (m.scale, plain.scale, "vectors"), (m.grad_table, plain.grad_table, "gradient"),
                               (m.y, plain.y, "result"), (m.slot, plain.slot, "slots")):
                assert_bit_equal(a.numpy(), b.numpy(), what)
        # replays with other inputs
        other = rng("other index").integers(1, V + 1, T)
        for m in (plain, first):
            m.dindex.copy_from(to_device(own, other))
        plain.step(1)
        graphs[0].replay()
        side.synchronize()
        assert_bit_equal(first.table.numpy(), plain.table.numpy())
        assert_bit_equal(first.grad_table.numpy(), plain.grad_table.numpy())
    del graphs
    own.shutdown()


@pytest.mark.parametrize("tokens", [600, 70000])
def test_gradient_of_many_tokens_in_two_graphs_replayed_beside_one_another(state, tokens):
    """Two graphs captured in one context and replayed on two streams at once: each has a workspace of its own."""
    import torch
    own = thc.State()
    streams = [torch.cuda.Stream() for _ in range(3)]
    own.set_stream(streams[0].cuda_stream, 0)
    r = rng("two graphs", tokens)
    sets, graphs = [], []
    with torch.cuda.stream(streams[0]):
        for k in range(2):
            index = np.exp(r.random(tokens) * np.log(301)).astype(np.int64).clip(1, 300)
            go = r.standard_normal((tokens, 40)).astype(np.float32)
            table, plain = thc.Tensor.new(own, "Float", 300, 40), thc.Tensor.new(own, "Float", 300, 40)
            dgo, dindex = to_device(own, go), to_device(own, index)
            plain.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
            streams[0].synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[0]):
                table.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
            sets.append((table, plain, dgo, dindex))
            graphs.append(g)
        streams[0].synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams[1:]):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for table, plain, _, _ in sets:
        assert_bit_equal(table.numpy(), plain.numpy())
    del graphs
    own.shutdown()


def test_host_threads_with_a_stream_each():
    import torch
    own = thc.State()
    failures = []

    def work(k):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            own.set_stream(stream.cuda_stream, 0)
            r = rng("threads", k)
            index = r.integers(1, 400, 5000 + 1000 * k)
            go = r.standard_normal((index.size, 32)).astype(np.float32)
            dgo, dindex = to_device(own, go), to_device(own, index)
            first = None
            for _ in range(20):
                table = thc.Tensor.new(own, "Float", 400, 32)
                table.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
                slot, order, offsets = (thc.Tensor.new(own, "Long") for _ in range(3))
                slot.expertSort(order, offsets, dindex, 400)
                got = table.numpy(), slot.numpy(), order.numpy(), offsets.numpy()
                first = first or got
                for a, b in zip(got, first):
                    assert_bit_equal(a, b)
            total, size, count = ro.embedding_grad(np.zeros((400, 32), np.float32), go, index, 1.0, 0, 0)
            assert (np.abs(first[0] - total) <= 2.0 ** -24 * np.abs(total) + count[:, None] * 2.0 ** -52 * size).all()
            for a, b in zip(first[1:], ro.expert_sort(index, 400)):
                assert_bit_equal(a, b)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failures.append(f"thread {k}: {e!r}")

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    own.shutdown()


def test_host_threads_whose_gradients_need_different_shared_memory():
    """One kernel, rows of 4 floats on half of the threads and of 1024 on the others: 57856 and 49288 bytes of shared memory.  What a
    thread asks for must not take away what another is about to launch with."""
    import torch
    own = thc.State()
    failures = []
    ready = threading.Barrier(4)

    def work(k):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            own.set_stream(stream.cuda_stream, 0)
            r = rng("shared memory", k)
            width, tokens = (4, 3000) if k % 2 else (1024, 300)
            index = r.integers(1, 60, tokens)
            go = r.standard_normal((tokens, width)).astype(np.float32)
            dgo, dindex, table = to_device(own, go), to_device(own, index), to_device(own, np.zeros((60, width), np.float32))
            table.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
            first = table.numpy()
            ready.wait(60)
            for _ in range(3000):
                table.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
            assert_bit_equal(table.numpy(), first)
            total, size, count = ro.embedding_grad(np.zeros((60, width), np.float32), go, index, 1.0, 0, 0)
            assert (np.abs(first - total) <= 2.0 ** -24 * np.abs(total) + count[:, None] * 2.0 ** -52 * size).all()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failures.append(f"thread {k}: {e!r}")
            ready.abort()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    own.shutdown()


# one pass and three of the tiled sort, its first size and others
@pytest.mark.parametrize("tokens", [8193, 16385, 65536, 65537, 150001])
@pytest.mark.parametrize("rows", [200, 70000, 3000000])
def test_long_sorts(state, tokens, rows):
    r = rng("long sorts", tokens, rows)
    index = np.exp(r.random(tokens) * np.log(rows + 1)).astype(np.int64).clip(1, rows)
    index[r.integers(0, tokens, 50)] = rows
    index[r.integers(0, tokens, 50)] = rows + 1
    check_grad(state, "Float", rows, 4, index, 1.0, 2, 0)


@pytest.mark.parametrize("choices,experts", [(8193, 64), (65536, 500), (65537, 9), (70000, 2047), (300000, 128), (16384, 511), (16384, 512)])
def test_long_expert_sorts(state, choices, experts):
    check_sort(state, rng("long experts", choices, experts).integers(0, experts + 1, choices), experts)


@pytest.mark.parametrize("kind", ["Half", "Float", "Double"])
@pytest.mark.parametrize("width", [8, 7, 1])
def test_results_beside_their_sources_in_one_matrix(state, kind, width):
    """Neighbouring columns of one matrix share no memory, whatever the spans from their first to their last bytes: the calls take
    them, give what they give on tensors of their own and leave the other columns alone.  Windows that meet are refused."""
    r = rng("windows", kind, width)
    dt, wide = NP_OF_KIND[kind], np.float64 if kind == "Double" else np.float32
    T, K, E, V = 9, 2, 3, 12
    N, gap = T * K, 2                                           # rows of every matrix; columns between two windows
    index, expert = r.integers(1, V + 1, T), r.integers(0, E + 1, (T, K))
    slot = ro.expert_sort(expert, E)[0]
    data = {k: r.standard_normal((n, width)).astype(dt) for k, n in
            dict(table=V, x=T, grad_x=T, grad_table=V, rows=N, answers=N, y=T, grad_y=T, grad_answers=N).items()}
    weight, grad_weight = r.random((T, K)).astype(wide), np.zeros((T, K), wide)
    one = lambda a: to_device(state, a)  # noqa: E731
    dindex, dslot, dweight = one(index), one(slot), one(weight)

    calls = (
        (("x", "table"), lambda t: t["x"].embedding(t["table"], dindex, 1.5)),
        (("grad_table", "grad_x"), lambda t: t["grad_table"].embeddingAccGrad(t["grad_x"], dindex, 1.5, 0, 0)),
        (("grad_table", "grad_x"), lambda t: t["grad_table"].embeddingAccGrad(t["grad_x"], dindex, 1.5, 0, 1)),
        (("rows", "x"), lambda t: t["rows"].expertDispatch(t["x"], dslot, None)),
        (("rows", "x"), lambda t: t["rows"].expertDispatch(t["x"], dslot, dweight)),
        (("y", "answers"), lambda t: t["y"].expertCombine(t["answers"], dslot, dweight)),
        (("grad_answers", "grad_y", "answers"), lambda t: t["grad_answers"].expertCombineGrad(one(grad_weight), t["grad_y"], t["answers"], dslot, dweight)),
    )
    step = width + gap
    for names, call in calls:
        alone = {k: one(data[k]) for k in names}
        call(alone)
        wide_matrix = r.standard_normal((N, step * len(names))).astype(dt)
        for j, k in enumerate(names):
            wide_matrix[:len(data[k]), j * step:j * step + width] = data[k]
        matrix = one(wide_matrix)
        call({k: matrix.narrow(1, j * step, width).narrow(0, 0, len(data[k])) for j, k in enumerate(names)})
        want = wide_matrix.copy()
        want[:len(data[names[0]]), :width] = alone[names[0]].numpy().reshape(len(data[names[0]]), width)
        assert_bit_equal(matrix.numpy(), want, names)
        if width > 1:
            with pytest.raises(thc.THCError, match="shares memory"):
                call({k: matrix.narrow(1, min(j, 1) * (width - 1), width).narrow(0, 0, len(data[k])) for j, k in enumerate(names)})
            assert_bit_equal(matrix.numpy(), want, names)
    # weights beside their gradient, slots beside the experts they come from
    both = one(np.concatenate([grad_weight, weight], 1))
    alone = one(grad_weight)
    thc.Tensor.new(state, kind).expertCombineGrad(alone, one(data["grad_y"]), one(data["answers"]), dslot, dweight)
    thc.Tensor.new(state, kind).expertCombineGrad(both.narrow(1, 0, K), one(data["grad_y"]), one(data["answers"]), dslot, both.narrow(1, K, K))
    assert_bit_equal(both.numpy(), np.concatenate([alone.numpy(), weight], 1))
    longs = one(np.concatenate([expert, np.full((T, K), 7), np.full((T, 1), 9)], 1))
    longs.narrow(1, K, K).expertSort(thc.Tensor.new(state, "Long"), thc.Tensor.new(state, "Long"), longs.narrow(1, 0, K), E)
    assert_bit_equal(longs.numpy(), np.concatenate([expert, slot, np.full((T, 1), 9)], 1))
    with pytest.raises(thc.THCError, match="shares memory"):
        longs.narrow(1, 1, K).expertSort(thc.Tensor.new(state, "Long"), thc.Tensor.new(state, "Long"), longs.narrow(1, 0, K), E)


def test_captured_calls_over_strided_tensors(state):
    """Results and lists that go through copies for the length of a call: in a graph the copies are the graph's own, made anew from what
    the tensors hold at each replay."""
    import torch
    own = thc.State()
    side = torch.cuda.Stream()
    own.set_stream(side.cuda_stream, 0)
    r = rng("captured strided")
    T, K, E, V, W = 300, 2, 5, 40, 24
    data = dict(index=r.integers(1, V + 1, T), weight=r.random((K, T)).astype(np.float32), gw=np.zeros((K, T), np.float32),
                table=r.standard_normal((W, V)).astype(np.float32), x=np.zeros((W, T), np.float32), go=r.standard_normal((W, T)).astype(np.float32),
                grad=np.zeros((V, 2 * W), np.float32), rows=r.standard_normal((T * K, W)).astype(np.float32),
                grad_rows=np.zeros((W, T * K), np.float32), slot=ro.expert_sort(r.integers(0, E + 1, (T, K)), E)[0].T.copy(),
                m=np.zeros((V, 2 * W), np.float32), v=np.zeros((V, 2 * W), np.float32))

    class Set:
        def __init__(self):
            self.base = {k: to_device(own, a) for k, a in data.items()}
            flip = lambda k: self.base[k].transpose(0, 1)  # noqa: E731
            every_other = lambda k: self.base[k].narrow(1, 3, W)  # noqa: E731
            self.t = {k: flip(k) for k in ("weight", "gw", "table", "x", "go", "grad_rows", "slot")}
            self.t |= {k: every_other(k) for k in ("grad", "m", "v")}
            self.lists = [thc.TensorList([self.t[k]]) for k in ("table", "grad", "m", "v")]

        def run(self):
            t = self.t
            t["x"].embedding(t["table"], self.base["index"], 1.5)
            t["grad"].embeddingAccGrad(t["go"], self.base["index"], 1.0, 0, 1)
            t["grad_rows"].expertCombineGrad(t["gw"], t["x"], self.base["rows"], t["slot"], t["weight"])
            self.lists[0].adamw(*self.lists[1:], step=2, **HYPER)

        def check(self, other):
            for k in data:
                assert_bit_equal(self.base[k].numpy(), other.base[k].numpy(), k)

    plain, replayed = Set(), Set()
    with torch.cuda.stream(side):
        replayed.run()
        for k, a in data.items():
            replayed.base[k].copy_from(to_device(own, a))
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            replayed.run()
        replayed.check(plain)                               # capturing runs nothing
        for _ in range(3):
            graph.replay()
            plain.run()
            side.synchronize()
            replayed.check(plain)
    del graph
    own.shutdown()


def test_the_scratch_of_reductions_stays_where_it_is():
    """A gradient that needs hundreds of megabytes leaves the scratch of the context's other calls alone: its address is in the hands of
    captured reductions and of callers of THCState_getCurrentDeviceScratchSpace."""
    import torch
    own = thc.State()
    side = torch.cuda.Stream()
    own.set_stream(side.cuda_stream, 0)
    scratch = own.lib.THCState_getCurrentDeviceScratchSpace
    scratch.restype, scratch.argtypes = C.c_void_p, [C.c_void_p]
    r = rng("scratch")
    a = r.integers(-8, 9, (4, 200000)).astype(np.float32)
    x, out = to_device(own, a), to_device(own, np.zeros((4, 1), np.float32))
    with torch.cuda.stream(side):
        out.sum(x, 1, 1)
        before = scratch(own.ptr)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out.sum(x, 1, 1)
        index = r.integers(1, 9, 60000)
        table = to_device(own, np.zeros((8, 600), np.float32))
        table.embeddingAccGrad(to_device(own, np.ones((60000, 600), np.float32)), to_device(own, index), 1.0, 0, 0)
        assert scratch(own.ptr) == before
        out.copy_from(to_device(own, np.zeros((4, 1), np.float32)))
        graph.replay()
        side.synchronize()
    assert_bit_equal(out.numpy(), a.sum(1, keepdims=True))
    assert_bit_equal(table.numpy(), np.repeat(np.bincount(index, minlength=9)[1:, None], 600, 1).astype(np.float32))
    del graph
    own.shutdown()


def torch_handle(state, t, kind):
    w = thc.Tensor.wrap(state, kind, t.data_ptr(), tuple(t.shape), tuple(t.stride()))
    w.owner = t
    return w


def test_empty_windows_of_padded_rows(state):
    """An expert without tokens, a batch without words: views of no rows whose strides reach further than the other dims do."""
    import torch
    rows = torch.arange(50, device="cuda", dtype=torch.float32).view(5, 10)
    longs = torch.ones(5, 4, device="cuda", dtype=torch.int64)
    x, one, two = torch_handle(state, rows[5:, :8], "Float"), torch_handle(state, longs[5:, 0], "Long"), torch_handle(state, longs[5:, :2], "Long")
    table = to_device(state, np.ones((3, 8), np.float32))
    table.embeddingAccGrad(x, one, 1.0, 0, 1)
    assert_bit_equal(table.numpy(), np.ones((3, 8), np.float32))
    table.embeddingAccGrad(x, one, 1.0, 0, 0)
    assert_bit_equal(table.numpy(), np.zeros((3, 8), np.float32))
    x.embedding(table, one, 1.0)
    table.expertDispatch(x, two, None)
    x.expertCombine(table, two, None)
    slot, order, offsets = (thc.Tensor.new(state, "Long") for _ in range(3))
    slot.expertSort(order, offsets, two, 3)
    assert_bit_equal(offsets.numpy(), np.zeros(4, np.int64))
    state.synchronize()
    assert torch.equal(rows, torch.arange(50, device="cuda", dtype=torch.float32).view(5, 10))
    empty = torch_handle(state, rows[:, 10:], "Float")            # rows of no elements
    assert empty.numpy().shape == (5, 0)


def test_offsets_beyond_32_bits(state):
    """A table of 2^32 + elements: rows on both sides of the border, looked up, and their gradients added."""
    import torch
    rows, width = 70001, 65536
    table = torch.zeros(rows, width, device="cuda", dtype=torch.float16)      # 9.2 GB
    at = [1, 65536, 65537, 65538, 70001, 70001]
    values = torch.randn(len(at), width, device="cuda").half()
    h = torch_handle(state, table, "Half")
    index = to_device(state, np.array(at))
    h.embeddingAccGrad(torch_handle(state, values, "Half"), index, 1.0, 0, 1)
    torch.cuda.synchronize()
    for k, row in enumerate(at[:4]):
        assert torch.equal(table[row - 1], values[k])
    assert torch.equal(table[70000], (values[4].float() + values[5].float()).half())
    assert int(torch.count_nonzero(table[1:65535])) == 0
    out = torch.empty(len(at), width, device="cuda", dtype=torch.float16)
    torch_handle(state, out, "Half").embedding(h, index, 2.0)
    torch.cuda.synchronize()
    assert torch.equal(out[0], values[0] * 2) and torch.equal(out[3], values[3] * 2) and torch.equal(out[4], table[70000] * 2)
    # the same rows as sorted places
    slot = to_device(state, np.array([[1, 65536], [65537, 65538], [70001, 0]]))
    back = torch.empty(3, width, device="cuda", dtype=torch.float16)
    torch_handle(state, back, "Half").expertCombine(h, slot, None)
    torch.cuda.synchronize()
    assert torch.equal(back[1], (table[65536].float() + table[65537].float()).half()) and torch.equal(back[2], table[70000])


def test_adamw_of_more_than_2_31_elements(state):
    import torch
    n = 2 ** 31 + 1000
    p, g = (torch.ones(n, device="cuda", dtype=torch.float16) for _ in range(2))
    m, v = torch.zeros(n, device="cuda", dtype=torch.int8), torch.zeros(n, device="cuda", dtype=torch.uint8)
    units = [torch.zeros(-(-n // 256), device="cuda") for _ in range(2)]
    lists = [thc.TensorList([torch_handle(state, t, k)]) for t, k in ((p, "Half"), (g, "Half"), (m, "Char"), (v, "Byte"), (units[0], "Float"), (units[1], "Float"))]
    lists[0].adamw8bit(*lists[1:], step=1, lr=0.5, beta1=0.9, beta2=0.99, eps=0.0, weight_decay=0.0, grad_scale=1.0)
    torch.cuda.synchronize()
    for part in (slice(0, 5000), slice(2 ** 31 - 300, 2 ** 31 + 300), slice(n - 300, n)):
        assert bool((p[part] == 0.5).all()) and bool((m[part] == 127).all()) and bool((v[part] == 255).all())


def test_tensors_of_another_device_are_refused(state):
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    w = torch.zeros(4, 8, device="cuda:1")
    with pytest.raises(thc.THCError, match="different GPUs"):
        thc.Tensor.new(state, "Float").embedding(torch_handle(state, w, "Float"), to_device(state, np.array([1])), 1.0)


def test_a_failed_workspace_leaves_the_call_undone_and_the_state_usable():
    """The library's own allocation fails (injected on the host): the call reports it, its result is as it was, the next call works."""
    own = thc.State()
    index = rng("failed workspace").integers(1, 50, 20000)
    go = np.ones((20000, 40), np.float32)
    table, dgo, dindex = to_device(own, np.full((50, 40), 7, np.float32)), to_device(own, go), to_device(own, index)
    slot, order, offsets = (thc.Tensor.new(own, "Long") for _ in range(3))
    own.lib.thcb200_debug_fail_allocation(1)
    with pytest.raises(thc.THCError, match="workspace"):
        table.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
    assert_bit_equal(table.numpy(), np.full((50, 40), 7, np.float32))
    own.lib.thcb200_debug_fail_allocation(0)
    table.embeddingAccGrad(dgo, dindex, 1.0, 0, 0)
    assert_bit_equal(table.numpy(), np.repeat(np.bincount(index, minlength=51)[1:, None], 40, 1).astype(np.float32))
    slot.expertSort(order, offsets, dindex, 50)
    assert_bit_equal(offsets.numpy(), np.concatenate([[0], np.cumsum(np.bincount(index, minlength=51)[1:])]))
    own.shutdown()

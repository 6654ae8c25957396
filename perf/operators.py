"""Operators of language-model training and serving on THC tensors: what is timed, and on which inputs.

Three groups, used one after the other in a training step and the first two in serving:

* ``lookup`` / ``lookup_grad``: rows of an embedding table scaled on the way, and the table's gradient summed over the
  tokens that share a row.
* ``experts`` / ``experts_grad``: tokens sorted by the experts they are routed to, their rows laid out expert by expert,
  the experts' answers brought back with their weights, and the gradients of both moves.
* ``adamw``: one step over a list of tensors, with the two moments in 32 bits or in 8.

Positions are 1-based, as in every call of the library; 0 stands for "not routed" and for "no padding row".
"""
import math

import torch

own = False

_BLOCK = 256                      # elements that share a scale of the 8-bit moments
_HALF, _FLOAT, _DOUBLE = "half", "float", "double"
_DTYPE = {_HALF: torch.float16, _FLOAT: torch.float32, _DOUBLE: torch.float64}


def _wide(name):
    """The type plain forms compute in."""
    return torch.float64 if name == _DOUBLE else torch.float32


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence being served: the next token's row, scaled by the square root of the width
        {"name": "lookup, one token", "op": "lookup", "type": _HALF, "vocab": 32000, "width": 4096, "tokens": 1, "scale": 64.0},
        # the tokens of a large training batch
        {"name": "lookup, batch", "op": "lookup", "type": _HALF, "vocab": 131072, "width": 4096, "tokens": 32768, "scale": 64.0},
        # the table's gradient of such a batch, written whole; word frequencies fall off as 1 / rank
        {"name": "lookup gradient, batch", "op": "lookup_grad", "type": _HALF, "vocab": 131072, "width": 2048, "tokens": 65536,
         "scale": 1.0, "padding": 0, "accumulate": False},
        # a small batch added to a gradient that is there already, odd sizes, one row is padding
        {"name": "lookup gradient, odd, added", "op": "lookup_grad", "type": _FLOAT, "vocab": 50021, "width": 1001, "tokens": 5003,
         "scale": 0.5, "padding": 7, "accumulate": True},
        # one token being served by eight of 64 experts
        {"name": "experts, one token", "op": "experts", "type": _HALF, "tokens": 1, "chosen": 8, "experts": 64, "width": 2048, "dropped": 0.0},
        # a training batch over 128 experts
        {"name": "experts, batch", "op": "experts", "type": _HALF, "tokens": 16384, "chosen": 8, "experts": 128, "width": 2048, "dropped": 0.0},
        # odd everything, a tenth of the choices dropped by a capacity limit
        {"name": "experts, odd, dropped", "op": "experts", "type": _FLOAT, "tokens": 1003, "chosen": 3, "experts": 17, "width": 1021, "dropped": 0.1},
        # the backward of a training batch
        {"name": "experts gradient, batch", "op": "experts_grad", "type": _HALF, "tokens": 16384, "chosen": 4, "experts": 64, "width": 2048,
         "dropped": 0.05},
        # the few small tensors of a head or an adapter
        {"name": "adamw, small", "op": "adamw", "type": _FLOAT, "tensors": 12, "elements": 60000, "bits": 32, "master": False, "step": 3},
        # all tensors of a model that trains in single precision
        {"name": "adamw, model", "op": "adamw", "type": _FLOAT, "tensors": 290, "elements": 200000000, "bits": 32, "master": False, "step": 1000},
        # half parameters with single-precision masters
        {"name": "adamw, half with masters", "op": "adamw", "type": _HALF, "tensors": 150, "elements": 100000000, "bits": 32, "master": True,
         "step": 20},
        # the same model with its moments in 8 bits
        {"name": "adamw, 8 bits", "op": "adamw", "type": _FLOAT, "tensors": 290, "elements": 200000000, "bits": 8, "master": False, "step": 500},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    n = _spread(rng, low, high)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "experts", "experts_grad", "adamw", "adamw"])
    kind = rng.choice([_HALF, _HALF, _HALF, _FLOAT, _FLOAT, _FLOAT, _DOUBLE])
    size = {_HALF: 2, _FLOAT: 4, _DOUBLE: 8}[kind]
    if op in ("lookup", "lookup_grad"):
        width = _width(rng, 64, 8192)
        vocab = _spread(rng, 500, max(600, min(150000, 2 ** 29 // (width * size))))
        tokens = _spread(rng, 1, max(2, min(65536, 2 ** 28 // (width * size))))
        case = {"op": op, "type": kind, "vocab": vocab, "width": width, "tokens": tokens, "scale": rng.choice([1.0, 0.5, math.sqrt(width)])}
        if op == "lookup_grad":
            case["padding"] = rng.choice([0, 0, rng.randint(1, min(vocab, 50))])
            case["accumulate"] = rng.random() < 0.5
        return case
    if op in ("experts", "experts_grad"):
        width = _width(rng, 64, 6000)
        chosen = rng.choice([1, 2, 3, 4, 6, 8])
        experts = _spread(rng, max(4, chosen), 256)
        tokens = _spread(rng, 1, max(2, min(32768, 2 ** 29 // (width * size * chosen))))
        return {"op": op, "type": kind, "tokens": tokens, "chosen": chosen, "experts": experts, "width": width,
                "dropped": rng.choice([0.0, 0.0, 0.1, 0.4])}
    bits = rng.choice([32, 8])
    if bits == 8 and kind == _DOUBLE:
        kind = _FLOAT
    return {"op": "adamw", "type": kind, "tensors": _spread(rng, 1, 300), "elements": _spread(rng, 3000, 100000000), "bits": bits,
            "master": kind == _HALF and rng.random() < 0.5, "step": _spread(rng, 1, 5000)}


# ---- inputs --------------------------------------------------------------------------------------
def _sizes(case):
    """Element counts of the tensors of an optimiser's list: a few large ones, many small ones, odd counts among them."""
    n, total = case["tensors"], case["elements"]
    weight = [1.0 / (1 + k % 7) ** 3 for k in range(n)]
    share = total / sum(weight)
    return [max(1, int(w * share)) + (k % 3 if k % 2 else 0) for k, w in enumerate(weight)]


def _starts(sizes):
    """Where the tensors of a list lie in the flat buffers that hold them all, and those buffers' size: each tensor begins on a
    multiple of 256 elements, and the elements between two tensors are zero."""
    at = [0]
    for n in sizes:
        at.append(at[-1] + -(-n // _BLOCK) * _BLOCK)
    return at[:-1], at[-1]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev = torch.device("cuda")
    kind = _DTYPE[case["type"]]

    def normal(*shape, dtype=kind, by=1.0):
        return torch.randn(*shape, device=dev, generator=gen, dtype=dtype).mul_(by)

    op = case["op"]
    s = {"case": dict(case)}
    if op in ("lookup", "lookup_grad"):
        vocab, width, tokens = case["vocab"], case["width"], case["tokens"]
        u = torch.rand(tokens, device=dev, generator=gen, dtype=torch.float64)
        s["index"] = torch.exp(u * math.log(vocab + 1)).long().clamp_(1, vocab)     # frequencies fall off as 1 / rank
        if op == "lookup":
            s["weight"] = normal(vocab, width, by=0.02)
            s["result"] = torch.empty(tokens, width, device=dev, dtype=kind)
        else:
            s["grad_output"] = normal(tokens, width)
            s["grad_weight"] = normal(vocab, width) if case["accumulate"] else torch.empty(vocab, width, device=dev, dtype=kind)
    elif op in ("experts", "experts_grad"):
        tokens, chosen, experts, width = case["tokens"], case["chosen"], case["experts"], case["width"]
        score = torch.rand(tokens, experts, device=dev, generator=gen) + 0.3 * torch.rand(experts, device=dev, generator=gen)
        expert = score.topk(chosen, dim=1).indices + 1
        expert[torch.rand(tokens, chosen, device=dev, generator=gen) < case["dropped"]] = 0
        wide = _wide(case["type"])
        s["expert"] = expert.contiguous()
        s["weight"] = torch.softmax(normal(tokens, chosen, dtype=wide), dim=1)
        s["expert_rows"] = normal(tokens * chosen, width)           # what the experts answered, expert by expert
        if op == "experts":
            s["x"] = normal(tokens, width)
            s["slot"] = torch.empty(tokens, chosen, device=dev, dtype=torch.int64)
            s["order"] = torch.empty(tokens * chosen, device=dev, dtype=torch.int64)
            s["offsets"] = torch.empty(experts + 1, device=dev, dtype=torch.int64)
            s["rows"] = torch.zeros(tokens * chosen, width, device=dev, dtype=kind)
            s["y"] = torch.empty(tokens, width, device=dev, dtype=kind)
        else:
            s["grad_y"] = normal(tokens, width)
            s["grad_rows_in"] = normal(tokens * chosen, width)      # the gradient of the rows that went to the experts
            s["slot"] = _sort_plain(s["expert"], experts)[0]        # the forward pass left these
            s["grad_expert_rows"] = torch.zeros(tokens * chosen, width, device=dev, dtype=kind)
            s["grad_weight"] = torch.empty(tokens, chosen, device=dev, dtype=wide)
            s["grad_x"] = torch.empty(tokens, width, device=dev, dtype=kind)
    else:
        # the list's tensors are pieces of flat buffers, as getParameters() lays a model out
        sizes = _sizes(case)
        starts, room = _starts(sizes)
        wide = _wide(case["type"])
        blocks = room // _BLOCK
        begin = torch.tensor(starts, device=dev)
        owner = torch.searchsorted(begin, torch.arange(blocks, device=dev) * _BLOCK, right=True) - 1
        local = torch.arange(room, device=dev).view(blocks, _BLOCK) - begin[owner][:, None]
        inside = (local < torch.tensor(sizes, device=dev)[owner][:, None]).view(-1)
        s["sizes"], s["starts"] = sizes, starts

        def pieces(dtype, by):
            return normal(room, dtype=dtype, by=by).mul_(inside)

        s["param"] = pieces(kind, 0.05)
        s["grad"] = pieces(kind, 0.01)
        if case["master"]:
            s["master"] = s["param"].to(wide) + pieces(wide, 1e-6)
        if case["bits"] == 32:
            s["m"] = pieces(wide, 0.003)
            s["v"] = pieces(wide, 0.01).square_()
        else:
            s["place"] = local.to(torch.int32)                        # an element's place in its tensor
            s["m"] = torch.randint(-127, 128, (room,), device=dev, generator=gen, dtype=torch.int8).mul_(inside)
            s["v"] = torch.randint(1, 256, (room,), device=dev, generator=gen, dtype=torch.uint8).mul_(inside)
            s["m_unit"] = (torch.rand(blocks, device=dev, generator=gen) + 0.5) * (0.01 / 127 ** 2)
            s["v_unit"] = (torch.rand(blocks, device=dev, generator=gen) + 0.5) * (1e-4 / 255.0 ** 4)
            s["m_value"], s["v_value"] = torch.zeros(room, device=dev), torch.zeros(room, device=dev)
    if own:
        s["handles"] = _handles(s)
    return s


# ---- the library's calls -------------------------------------------------------------------------
_STATE = []


def _handles(s):
    """The tensor handles that a program of this library holds over its buffers."""
    from cutorch_b200 import thc

    if not _STATE:
        _STATE.append(thc.State())
    state = _STATE[0]
    kinds = {torch.float16: "Half", torch.float32: "Float", torch.float64: "Double", torch.int64: "Long", torch.int8: "Char",
             torch.uint8: "Byte"}

    def wrap(t):
        return thc.Tensor.wrap(state, kinds[t.dtype], t.data_ptr(), tuple(t.shape), tuple(t.stride()))

    if s["case"]["op"] != "adamw":
        return {k: wrap(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
    got = {}
    for k in ("param", "grad", "master", "m", "v", "m_value", "v_value", "m_unit", "v_unit"):
        by = _BLOCK if k.endswith("unit") else 1
        got[k] = thc.TensorList([wrap(s[k][at // by:at // by + -(-n // by)]) for at, n in zip(s["starts"], s["sizes"])]) if k in s else None
    return got


def _run_own(s):
    case, h = s["case"], s["handles"]
    op = case["op"]
    if op == "lookup":
        h["result"].embedding(h["weight"], h["index"], case["scale"])
        return s["result"]
    if op == "lookup_grad":
        h["grad_weight"].embeddingAccGrad(h["grad_output"], h["index"], case["scale"], case["padding"], case["accumulate"])
        return s["grad_weight"]
    if op == "experts":
        h["slot"].expertSort(h["order"], h["offsets"], h["expert"], case["experts"])
        h["rows"].expertDispatch(h["x"], h["slot"], None)
        h["y"].expertCombine(h["expert_rows"], h["slot"], h["weight"])
        return {k: s[k] for k in ("slot", "order", "offsets", "rows", "y")}
    if op == "experts_grad":
        h["grad_expert_rows"].expertCombineGrad(h["grad_weight"], h["grad_y"], h["expert_rows"], h["slot"], h["weight"])
        h["grad_x"].expertCombine(h["grad_rows_in"], h["slot"], None)
        return {k: s[k] for k in ("grad_expert_rows", "grad_weight", "grad_x")}
    step = dict(step=case["step"], lr=_LR, beta1=_BETA1, beta2=_BETA2, eps=_EPS, weight_decay=_DECAY, grad_scale=_GRAD_SCALE)
    if case["bits"] == 32:
        h["param"].adamw(h["grad"], h["m"], h["v"], master=h["master"], **step)
    else:
        h["param"].adamw8bit(h["grad"], h["m"], h["v"], h["m_unit"], h["v_unit"], master=h["master"], **step)
        # what the codes stand for, as a checkpoint stores it
        h["m_value"].adamwValues(h["v_value"], h["m"], h["v"], h["m_unit"], h["v_unit"])
    return _adamw_outputs(s)


# ---- plain forms ---------------------------------------------------------------------------------
_LR, _BETA1, _BETA2, _EPS, _DECAY, _GRAD_SCALE = 1e-3, 0.9, 0.999, 1e-8, 0.01, 0.5


def _lookup_plain(s):
    case = s["case"]
    return (s["weight"][s["index"] - 1].to(_wide(case["type"])) * case["scale"]).to(s["weight"].dtype)


def _lookup_grad_plain(s):
    case = s["case"]
    wide = _wide(case["type"])
    total = torch.zeros(case["vocab"], case["width"], device="cuda", dtype=wide)
    g = s["grad_output"].to(wide) * (s["index"] != case["padding"])[:, None]
    total.index_add_(0, s["index"] - 1, g)
    total *= case["scale"]
    if case["accumulate"]:
        total += s["grad_weight"]
    s["grad_weight"].copy_(total)
    return s["grad_weight"]


def _sort_plain(expert, experts):
    flat = expert.reshape(-1)
    key = torch.where((flat >= 1) & (flat <= experts), flat, experts + 1)
    key, order = torch.sort(key, stable=True)
    live = torch.sum(key <= experts)
    place = torch.arange(flat.numel(), device=flat.device)
    slot = torch.empty_like(flat)
    slot[order] = torch.where(place < live, place + 1, 0)
    order = torch.where(place < live, order + 1, 0)
    bins = torch.arange(experts + 1, device=flat.device) + 1
    offsets = torch.searchsorted(key, bins)
    return slot.view_as(expert), order, offsets


def _dispatch_plain(rows, x, slot):
    tokens, chosen = slot.shape
    token = torch.arange(tokens, device=slot.device).repeat_interleave(chosen)
    routed = slot.reshape(-1) > 0
    rows[slot.reshape(-1)[routed] - 1] = x[token[routed]]
    return rows


def _gathered(rows, slot, wide):
    return rows[(slot - 1).clamp(min=0).reshape(-1)].to(wide).view(*slot.shape, -1) * (slot > 0)[:, :, None]


def _combine_plain(rows, slot, weight, wide):
    g = _gathered(rows, slot, wide)
    return (g if weight is None else g * weight[:, :, None]).sum(1).to(rows.dtype)


def _combine_grad_plain(s):
    wide = _wide(s["case"]["type"])
    slot, g = s["slot"], s["grad_y"].to(wide)
    grad_weight = (_gathered(s["expert_rows"], slot, wide) * g[:, None, :]).sum(2)
    tokens, chosen = slot.shape
    routed = (slot > 0).reshape(-1)
    token = torch.arange(tokens, device=slot.device).repeat_interleave(chosen)[routed]
    s["grad_expert_rows"][slot.reshape(-1)[routed] - 1] = (g[token] * s["weight"].reshape(-1)[routed][:, None]).to(s["grad_y"].dtype)
    return s["grad_expert_rows"], grad_weight


# The 8-bit moments.  256 neighbours share a unit.  A code c of the first moment stands for c |c| unit, one of the second
# (0 to 255) for (c c)(c c) unit, so the values close to zero keep codes of their own; the largest magnitude of a block takes
# code 127 or 255.  A value between two codes takes the upper one with the probability that keeps its expectation, by a
# dither that is a hash of the element's place and the step: averages that move by less than a code's distance still move.
def _dither(place, step):
    h = place.long() * 0x9E3779B9 + (step * 0x7F4A7C15 & 0xFFFFFFFF) & 0xFFFFFFFF
    h = (h ^ h >> 16) * 0x9E3779B9 & 0xFFFFFFFF
    h = (h ^ h >> 15) * 0x9E3779B9 & 0xFFFFFFFF
    h = h ^ h >> 16
    return (h >> 16).float() * 2.0 ** -16, (h & 0xFFFF).float() * 2.0 ** -16


def _unit(magnitude, top, least):
    """The blocks' units, and their reciprocals."""
    most = magnitude.amax(1, keepdim=True)
    unit = torch.where(most >= least, most * torch.tensor(1.0 / top, device=most.device), 0.0)
    return unit, torch.where(unit > 0, 1.0 / unit, 0.0)


def _encode(x, dither, root, value, top):
    """The code of x units: the last one whose value is at most x, or by the dither the next."""
    k = root(x).floor().clamp(0, top)
    k = torch.where(value(k) > x, k - 1, k)
    k = torch.where((k < top) & (value(k + 1) <= x), k + 1, k)
    return k + ((k < top) & (dither * (value(k + 1) - value(k)) < x - value(k)))


def _square(k):
    return k * k


def _fourth(k):
    return (k * k) * (k * k)


def _fourth_root(x):
    return x.sqrt().sqrt()


def _adamw_outputs(s):
    m, v = ("m_value", "v_value") if s["case"]["bits"] == 8 else ("m", "v")
    return {k: s[n] for k, n in (("param", "param"), ("master", "master"), ("m", m), ("v", v)) if n in s}


def _adamw_plain(s):
    case = s["case"]
    wide = _wide(case["type"])
    step = case["step"]
    size = _LR / (1 - _BETA1 ** step)
    root = 1 / math.sqrt(1 - _BETA2 ** step)
    g = s["grad"].to(wide) * _GRAD_SCALE
    p = s["master"] if case["master"] else s["param"].to(wide)
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        cm, cv = s["m"].float().view(-1, _BLOCK), s["v"].float().view(-1, _BLOCK)
        m = (cm * cm.abs() * s["m_unit"][:, None]).view(-1)
        v = (_fourth(cv) * s["v_unit"][:, None]).view(-1)
    m = m * _BETA1 + g * (1 - _BETA1)
    v = v * _BETA2 + g * (1 - _BETA2) * g
    p = p * (1 - _LR * _DECAY) - size * (m / (v.sqrt() * root + _EPS))
    s["param"].copy_(p)
    if case["master"]:
        s["master"].copy_(p)
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _adamw_outputs(s)
    m, v = m.view(-1, _BLOCK), v.view(-1, _BLOCK)
    first, second = _dither(s["place"], step)
    unit, inverse = _unit(m.abs(), 127 ** 2, 1e-30)
    code = _encode(m.abs() * inverse, first, torch.sqrt, _square, 127)
    code = torch.where(m < 0, -code, code)
    s["m_unit"].copy_(unit.view(-1))
    s["m"].copy_(code.view(-1))
    s["m_value"].copy_((code * code.abs() * unit).view(-1))
    unit, inverse = _unit(v, 255.0 ** 4, 1e-28)
    code = _encode(v * inverse, second, _fourth_root, _fourth, 255)
    code = torch.where(v > 0, code.clamp(min=1), code)
    s["v_unit"].copy_(unit.view(-1))
    s["v"].copy_(code.view(-1))
    s["v_value"].copy_((_fourth(code) * unit).view(-1))
    return _adamw_outputs(s)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "lookup":
        return _lookup_plain(state)
    if op == "lookup_grad":
        return _lookup_grad_plain(state)
    wide = _wide(state["case"]["type"])
    if op == "experts":
        slot, order, offsets = _sort_plain(state["expert"], state["case"]["experts"])
        return {"slot": slot, "order": order, "offsets": offsets, "rows": _dispatch_plain(state["rows"], state["x"], slot),
                "y": _combine_plain(state["expert_rows"], slot, state["weight"], wide)}
    if op == "experts_grad":
        grad_rows, grad_weight = _combine_grad_plain(state)
        return {"grad_expert_rows": grad_rows, "grad_weight": grad_weight,
                "grad_x": _combine_plain(state["grad_rows_in"], state["slot"], None, wide)}
    return _adamw_plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    size = {_HALF: 2, _FLOAT: 4, _DOUBLE: 8}[case["type"]]
    wide = 8 if case["type"] == _DOUBLE else 4
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        row = case["width"] * size
        # different rows that such a batch is expected to name: sum over the ranks of 1 - (1 - p)^tokens
        n, top = case["tokens"], math.log(case["vocab"] + 1)
        used, r = 0.0, 1
        while r <= case["vocab"]:
            many = max(1, r // 64)                  # ranks of about the same frequency together
            many = min(many, case["vocab"] - r + 1)
            p = (math.log(r + many) - math.log(r)) / top / many
            used += many * -math.expm1(n * math.log1p(-min(p, 1 - 1e-12)))
            r += many
        if op == "lookup":
            return {"bytes": used * row + n * row + 8 * n, "flops": n * case["width"]}
        written = 2 * used * row if case["accumulate"] else case["vocab"] * row
        return {"bytes": n * row + 8 * n + written, "flops": 2 * n * case["width"]}
    if op in ("experts", "experts_grad"):
        pairs, row = case["tokens"] * case["chosen"], case["width"] * size
        live = pairs * (1 - case["dropped"])
        if op == "experts":
            # choices read; slots, order and offsets written; rows out and, weighted, back
            moved = 8 * (3 * pairs + case["experts"] + 1) + (case["tokens"] + live) * row + (live + case["tokens"]) * row + pairs * wide
            return {"bytes": moved, "flops": 2 * live * case["width"]}
        moved = 8 * pairs + (case["tokens"] + 2 * live) * row + 2 * pairs * wide + (live + case["tokens"]) * row
        return {"bytes": moved, "flops": 4 * live * case["width"]}
    n = sum(_sizes(case))
    each = 3 * size + (2 * wide if case["master"] else 0) - (size if case["master"] else 0)   # a master is read in the parameter's place
    each += 4 * wide if case["bits"] == 32 else 4 + 16 / _BLOCK + 8     # codes and units both ways, and the values they stand for
    return {"bytes": n * each, "flops": 16 * n}


# ---- from the definitions, in 64 bits ------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "lookup":
        return torch.index_select(s["weight"], 0, s["index"] - 1).to(f64).mul_(case["scale"])
    if op == "lookup_grad":
        g = s["grad_weight"].to(f64) if case["accumulate"] else torch.zeros(case["vocab"], case["width"], device="cuda", dtype=f64)
        keep = torch.nonzero(s["index"] != case["padding"])[:, 0]
        for part in keep.split(16384):
            g.index_put_((s["index"][part] - 1,), s["grad_output"][part].to(f64) * case["scale"], accumulate=True)
        return g
    if op in ("experts", "experts_grad"):
        experts, tokens, chosen = case["experts"], case["tokens"], case["chosen"]
        flat = s["expert"].reshape(-1)
        # the place of a pair: pairs of lower experts, then the earlier pairs of its own
        slot = torch.zeros_like(flat)
        offsets = [0]
        for e in range(1, experts + 1):
            mine = flat == e
            slot = torch.where(mine, torch.cumsum(mine, 0) + offsets[-1], slot)
            offsets.append(offsets[-1] + int(mine.sum()))
        slot = slot.view(tokens, chosen)

        def back(rows, weight):
            y = torch.zeros(tokens, case["width"], device="cuda", dtype=f64)
            for k in range(chosen):
                here = torch.nonzero(slot[:, k])[:, 0]
                part = rows[slot[here, k] - 1].to(f64)
                y[here] += part if weight is None else part * weight[here, k, None].to(f64)
            return y

        if op == "experts":
            order = torch.zeros_like(flat)
            rows = torch.zeros_like(s["rows"], dtype=f64)
            for k in range(chosen):
                here = torch.nonzero(slot[:, k])[:, 0]
                order[slot[here, k] - 1] = here * chosen + k + 1
                rows[slot[here, k] - 1] = s["x"][here].to(f64)
            return {"slot": slot, "order": order, "offsets": torch.tensor(offsets, device="cuda"), "rows": rows,
                    "y": back(s["expert_rows"], s["weight"])}
        grad_rows = torch.zeros_like(s["grad_expert_rows"], dtype=f64)
        grad_weight = torch.zeros(tokens, chosen, device="cuda", dtype=f64)
        for k in range(chosen):
            here = torch.nonzero(slot[:, k])[:, 0]
            at = slot[here, k] - 1
            g = s["grad_y"][here].to(f64)
            grad_weight[here, k] = torch.linalg.vecdot(s["expert_rows"][at].to(f64), g)
            grad_rows[at] = g * s["weight"][here, k, None].to(f64)
        return {"grad_expert_rows": grad_rows, "grad_weight": grad_weight, "grad_x": back(s["grad_rows_in"], None)}
    # the optimiser: its formulas over the flat buffers (the zeros between the tensors stay zeros)
    eight = case["bits"] == 8

    def moment(name, decode):
        if not eight:
            return s[name].to(f64)
        return decode(s[name].to(f64)).view(-1, _BLOCK).mul_(s[name + "_unit"].to(f64)[:, None]).view(-1)

    start = (s["master"] if case["master"] else s["param"]).to(f64)
    g = s["grad"].to(f64) / 2
    m = torch.lerp(g, moment("m", lambda c: c.abs() * c), _BETA1)
    v = torch.lerp(g.square(), moment("v", lambda c: c ** 4), _BETA2)
    t = case["step"]
    new = start - _LR * _DECAY * start - _LR * (m / (1 - _BETA1 ** t)) / ((v / (1 - _BETA2 ** t)).sqrt() + _EPS)
    out = {"param": new}
    if case["master"]:
        out["master"] = new
    # which code a value takes depends on its last bits: the 8-bit moments have no value in 64 bits
    out["m"], out["v"] = (None, None) if eight else (m, v)
    return out

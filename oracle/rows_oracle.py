"""TEST ONLY: numpy restatements of the embedding, expert-routing and AdamW calls, in 64 bits (the 8-bit codes in the
float arithmetic that defines them)."""
import numpy as np


def embedding(weight, index, scale):
    """scale * weight[index - 1], one rounding; rows whose position is out of range are NaN-marked through `valid`."""
    valid = (index >= 1) & (index <= weight.shape[0])
    rows = weight[np.where(valid, index, 1) - 1]
    math = np.float32 if weight.dtype == np.float16 else weight.dtype.type
    return (rows.astype(math) * math(scale)).astype(weight.dtype), valid


def embedding_grad(grad_weight, grad_output, index, scale, padding, accumulate):
    """(the sums in 64 bits, the sum of the addends' magnitudes, the number of addends of each row)."""
    v, d = grad_weight.shape
    flat = index.reshape(-1)
    g = grad_output.reshape(-1, d).astype(np.float64)
    keep = (flat >= 1) & (flat <= v) & (flat != (padding if padding else -1))
    total, size, count = np.zeros((v, d)), np.zeros((v, d)), np.zeros(v)
    np.add.at(total, flat[keep] - 1, g[keep])
    np.add.at(size, flat[keep] - 1, np.abs(g[keep]))
    np.add.at(count, flat[keep] - 1, 1)
    total, size = total * scale, size * abs(scale)
    if accumulate:
        total, size = total + grad_weight.astype(np.float64), size + np.abs(grad_weight.astype(np.float64))
    return total, size, count


def expert_sort(expert, experts):
    flat = expert.reshape(-1)
    slot = np.zeros(flat.size, np.int64)
    order = np.zeros(flat.size, np.int64)
    offsets = [0]
    place = 0
    for e in range(1, experts + 1):
        for i in np.flatnonzero(flat == e):
            order[place] = i + 1
            place += 1
            slot[i] = place
        offsets.append(place)
    return slot.reshape(expert.shape), order, np.array(offsets, np.int64)


def combine(rows, slot, weight):
    """(sums in 64 bits, sums of magnitudes)."""
    t, k = slot.shape
    out, size = np.zeros((t, rows.shape[1])), np.zeros((t, rows.shape[1]))
    for j in range(k):
        here = (slot[:, j] >= 1) & (slot[:, j] <= rows.shape[0])
        part = rows[slot[here, j] - 1].astype(np.float64)
        if weight is not None:
            part = part * weight[here, j, None].astype(np.float64)
        out[here] += part
        size[here] += np.abs(part)
    return out, size


def adamw(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay, grad_scale):
    p, g, m, v = (x.astype(np.float64) for x in (p, g, m, v))
    g = g * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    denominator = np.sqrt(v / (1 - beta2 ** step)) + eps
    with np.errstate(invalid="ignore", divide="ignore"):
        p = p * (1 - lr * weight_decay) - lr / (1 - beta1 ** step) * (m / denominator)
    return p, m, v, denominator


BLOCK = 256
_F = np.float32


def first_value(code):
    c = code.astype(np.int32)
    return (c * np.abs(c)).astype(_F)


def second_value(code):
    c = code.astype(np.int32)
    f = (c * c).astype(_F)
    return f * f


def decode(code, unit, value):
    return value(code) * np.repeat(unit, BLOCK)[:code.size]


def dither(n, step):
    """Two numbers in [0, 1) for each place, from a hash of the place and the step."""
    mask = np.uint64(0xFFFFFFFF)
    k = np.uint64(0x9E3779B9)
    h = (np.arange(n, dtype=np.uint64) * k + np.uint64(step * 0x7F4A7C15 & 0xFFFFFFFF)) & mask
    h = (h ^ (h >> np.uint64(16))) * k & mask
    h = (h ^ (h >> np.uint64(15))) * k & mask
    h = h ^ (h >> np.uint64(16))
    return (h >> np.uint64(16)).astype(_F) * _F(2.0 ** -16), (h & np.uint64(0xFFFF)).astype(_F) * _F(2.0 ** -16)


def _encode(x, dith, value, top):
    values = value(np.arange(top + 1))
    k = np.clip(np.searchsorted(values, x, side="right") - 1, 0, top)       # the last code whose value is at most x
    nxt = np.minimum(k + 1, top)
    up = (k < top) & (dith * (values[nxt] - values[k]) < x - values[k])
    return k + up


def adamw8(p, g, cm, cv, um, uv, step, lr, beta1, beta2, eps, weight_decay, grad_scale):
    """The float step: new moments, codes and units, bit for bit; the parameter in 64 bits from the decoded moments."""
    n = p.size
    gf = g.astype(_F) * _F(grad_scale)
    m0, v0 = decode(cm, um, first_value), decode(cv, uv, second_value)
    m = m0 * _F(beta1) + gf * _F(1 - beta1)
    v = v0 * _F(beta2) + gf * _F(1 - beta2) * gf
    out = []
    for x, top, value, least, dith in ((np.abs(m), 127, first_value, _F(1e-30), dither(n, step)[0]),
                                       (v, 255, second_value, _F(1e-28), dither(n, step)[1])):
        padded = np.zeros(-(-n // BLOCK) * BLOCK, _F)
        padded[:n] = x
        most = padded.reshape(-1, BLOCK).max(1)
        unit = np.where(most < least, _F(0), np.where(most <= np.finfo(_F).max, most * _F(1.0 / float(value(np.array([top]))[0])), _F(np.nan)))
        inverse = np.where(unit > 0, _F(1) / np.where(unit > 0, unit, _F(1)), _F(0))
        out.append((_encode(x * np.repeat(inverse, BLOCK)[:n], dith, value, top), unit))
    (km, nmu), (kv, nvu) = out
    kv = np.where((v > 0) & (kv == 0), 1, kv)
    return m0, v0, m, v, np.where(m < 0, -km, km).astype(np.int8), kv.astype(np.uint8), nmu, nvu

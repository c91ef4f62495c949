"""Plain float64 evaluations of the routed feed-forward operators."""
import numpy as np

LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
DIGITS = {"e4m3": (3, -6), "e5m2": (2, -14)}


def route(logits, k, renormalize):
    """(weights, ids) of float64 logits [tokens, experts]; -1 and 0 where
    fewer than k experts are above -inf."""
    t, e = logits.shape
    ids = np.full((t, k), -1)
    weights = np.zeros((t, k))
    for r in range(t):
        row = logits[r]
        if np.isnan(row).any():
            weights[r] = np.nan
        order = sorted((i for i in range(e) if row[i] > -np.inf), key=lambda i: (-row[i], i))[:k]
        ids[r, :len(order)] = order
        if not order or np.isnan(row).any():
            continue
        z = np.exp(row[order] - row[order[0]])
        total = z.sum() if renormalize else np.exp(row - row[order[0]]).sum()
        weights[r, :len(order)] = z / total
    return weights, ids


def sort(ids, experts):
    flat = ids.reshape(-1)
    rows = sorted((i for i in range(flat.size) if flat[i] >= 0), key=lambda i: (flat[i], i))
    source = np.full(flat.size, -1)
    source[:len(rows)] = rows
    position = np.full(flat.size, -1)
    position[rows] = np.arange(len(rows))
    offsets = np.array([sum(1 for v in flat if 0 <= v < e) for e in range(experts + 1)])
    return offsets, position.reshape(ids.shape), source


def spread(x, source, k, weights=None):
    out = np.zeros((source.size, x.shape[1]))
    for p, s in enumerate(source):
        if s >= 0:
            out[p] = x[s // k] * (1.0 if weights is None else weights.reshape(-1)[s])
    return out


def combine(ys, weights, position):
    t, k = position.shape
    y = np.zeros((t, ys.shape[1]))
    for i in range(t):
        for j in range(k):
            if position[i, j] >= 0:
                y[i] += weights[i, j] * ys[position[i, j]]
    return y


def scale(block, fmt):
    """The least power of two s >= 2^-126 with the block's largest finite
    magnitude / s within the format; 1 for a block of zeros."""
    finite = np.abs(block[np.isfinite(block)])
    top = finite.max() if finite.size else 0.0
    if top == 0.0:
        return 1.0
    s = 2.0 ** -126
    while top / s > LARGEST[fmt]:
        s *= 2.0
    return s


def round8(v, fmt):
    """Nearest number of the format, ties to even; infinities stay in e5m2 and
    are NaN in e4m3."""
    digits, least = DIGITS[fmt]
    out = np.array(v, dtype=np.float64)
    fin = np.isfinite(out)
    _, e = np.frexp(out[fin])
    step = np.ldexp(1.0, np.maximum(e - 1, least) - digits)
    out[fin] = np.rint(out[fin] / step) * step
    if fmt == "e4m3":
        out[~fin] = np.nan
    return out


def quantize(x, fmt, high):
    """Blocks of high x 128 of x [rows, cols]: (values of the data, scales
    [row blocks, column blocks])."""
    rows, cols = x.shape
    q = np.zeros_like(x)
    s = np.ones((-(-rows // high), -(-cols // 128)))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = (slice(i * high, (i + 1) * high), slice(j * 128, (j + 1) * 128))
            s[i, j] = scale(x[at], fmt)
            q[at] = round8(x[at] / s[i, j], fmt)
    return q, s


def values(q, s, high):
    """The numbers that quantize's result stands for."""
    return q * np.repeat(np.repeat(s, high, 0)[:q.shape[0]], 128, 1)[:, :q.shape[1]]


DIGITS16 = {"bf16": (7, -126), "f16": (10, -14)}
TOP16 = {"bf16": float(2.0 ** 128 - 2.0 ** 119), "f16": 65520.0}  # from here on a number rounds to infinity


def half_ulp(v, dtype):
    """Half the spacing of the type's numbers at v (0 for f32: its roundings
    are part of the bounds; 2^-149 so that subnormal results have one)."""
    if dtype == "f32":
        return np.full(np.shape(v), 2.0 ** -149)
    digits, least = DIGITS16[dtype]
    _, e = np.frexp(v)
    return np.ldexp(0.5, np.maximum(e - 1, least) - digits)


def outside(got, ref, bound, dtype):
    """Where got, of this type, is further from ref than the bound and half an
    ulp of the number that is rounded; beyond the type's range, where it is no
    infinity of ref's sign either."""
    limit = bound + half_ulp(np.abs(ref) + bound, dtype)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - ref) <= limit)
    if dtype in TOP16:
        bad &= ~((np.abs(ref) + bound >= TOP16[dtype]) & (got == np.copysign(np.inf, ref)))
    return bad

"""The block scales of the 8-bit products, in every kernel that applies them:
scales far from 1, whose product leaves f32 although the result does not, and
scales that are no powers of two.

The numbers are small integers times powers of two that are the same for a
whole row of the result, so every product, every block's sum and the result
are exact and the comparison is equality.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# rows, n, k (weight gradient: rows of the sum, n, k), experts, any_scales: the
# kernel for few rows, dense and by expert; one block of 128 at a time, whole
# and in parts; the tensor core's own scales, whole and in parts
FORWARD = [(3, 200, 640, None, False), (3, 200, 640, None, True), (5, 72, 384, 3, False), (140, 200, 640, None, False),
           (140, 200, 640, None, True), (150, 264, 640, 3, False), (140, 100, 2688, None, False),
           (2100, 1000, 4096, None, False), (1100, 1030, 8192, 4, False), (300, 1000, 19200, None, False)]
DINPUT = [(140, 200, 640, None, False), (140, 200, 640, None, True), (150, 264, 640, 3, False),
          (2100, 1000, 4096, None, False)]
WGRAD = [(700, 136, 200, None, False), (700, 136, 200, None, True), (900, 129, 72, 3, False), (2600, 128, 256, None, False),
         (4300, 1500, 1300, None, False), (60000, 520, 600, None, False)]
CASES = [("forward", *c) for c in FORWARD] + [("dinput", *c) for c in DINPUT] + [("dweight", *c) for c in WGRAD]

# exponents of a block's scales: (a's, b's)
FAR = [(0, 0), (100, -100), (-100, 100), (119, -119), (-119, 119), (60, -60)]


def _split(rows, experts):
    """Rows of each expert: the second has none, the last has some."""
    if experts is None:
        return [rows]
    last = rows // 3
    return [rows - last - (experts - 3), 0] + [1] * (experts - 3) + [last]


class Case:
    """Operands of one product as numpy: integers, scales and the layout that
    the entry takes; blocks[b] is block b's slice of the contraction."""

    def __init__(self, rng, form, rows, n, k, experts, any_scales):
        self.form, self.any_scales, self.n, self.k = form, any_scales, n, k
        self.counts = _split(rows, experts)
        self.experts = None if experts is None else len(self.counts)
        if form == "dweight":
            # places of 128 for each expert, as quantize8_transposed lays them out
            nb = -(-rows // 128) if experts is None else rows // 128 + self.experts
            self.m, self.nb, self.extent = n, nb, nb * 128
            used = np.zeros(self.extent, bool)
            at = 0
            self.starts = []
            for c in self.counts:
                self.starts.append(at)
                used[at * 128:at * 128 + c] = True
                at += -(-c // 128)
            self.starts.append(at)
            self.a = rng.integers(-3, 4, (n, self.extent)) * used
            self.b = rng.integers(-3, 4, (k, self.extent)) * used
            self.sb = np.zeros((nb, k), int)
        else:
            self.m, self.nb, self.extent = rows, -(-k // 128), k
            self.a = rng.integers(-3, 4, (rows, k))
            shape = (1 if experts is None else self.experts, n, k)
            self.b = rng.integers(-3, 4, shape if form == "forward" else (shape[0], k, n))
            self.sb = np.zeros((shape[0], -(-n // 128), self.nb) if form == "forward" else
                               (shape[0], self.nb, -(-n // 128)), int)
        self.sa = np.zeros((self.nb, self.m), int)
        self.factor_a, self.factor_b = np.ones(self.sa.shape), np.ones(self.sb.shape)

    def scale(self, block, a, b):
        """Exponents of one block of the contraction (all rows, all columns)."""
        self.sa[block] = a
        if self.form == "dweight":
            self.sb[block] = b
        elif self.form == "forward":
            self.sb[:, :, block] = b
        else:
            self.sb[:, block, :] = b

    def operands(self, cuda, formats=("e4m3", "e5m2")):
        import torch
        kinds = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}

        def put(v, fmt, scales, cols, blocks):
            ld = -(-cols // 16) * 16
            full = np.zeros((*v.shape[:-1], ld), np.float32)
            full[..., :cols] = v
            return cuda.Blocks8(torch.from_numpy(full).cuda().to(kinds[fmt]),
                                torch.from_numpy(scales.astype(np.float32)).cuda(), cols, blocks)
        sa = np.ldexp(1.0, self.sa) * self.factor_a
        sb = np.ldexp(1.0, self.sb) * self.factor_b
        a = put(self.a, formats[0], sa, self.extent, "rows")
        if self.form == "dweight":
            return a, put(self.b, formats[1], sb, self.extent, "rows")
        b, cols = self.b, self.k if self.form == "forward" else self.n
        if self.experts is None:
            b, sb = b[0], sb[0]
        return a, put(b, formats[1], sb, cols, "tiles")

    def offsets(self):
        import torch
        if self.experts is None:
            return None
        return torch.tensor(np.concatenate([[0], np.cumsum(self.counts)]), dtype=torch.int32, device="cuda")

    def run(self, cuda, operands=None):
        import torch
        a, b = operands or self.operands(cuda)
        if self.form == "dweight":
            y = cuda.matmul8_wgrad(a, b, self.offsets(), any_scales=self.any_scales)
        else:
            y = cuda.matmul8(a, b, self.form == "forward", self.offsets(), torch.float32, self.any_scales)
        torch.cuda.synchronize()
        return y.cpu().numpy().astype(np.float64)

    def reference(self):
        """float64: block sums times their two scales."""
        sa = np.ldexp(1.0, self.sa) * self.factor_a
        sb = np.ldexp(1.0, self.sb) * self.factor_b
        if self.form == "dweight":
            out = np.zeros((len(self.counts), self.n, self.k))
            for e in range(len(self.counts)):
                for b in range(self.starts[e], self.starts[e + 1]):
                    at = slice(b * 128, (b + 1) * 128)
                    out[e] += (self.a[:, at].astype(float) @ self.b[:, at].T.astype(float)) * sa[b][:, None] * sb[b][None]
            return out if self.experts is not None else out[0]
        out = np.zeros((self.m, self.n))
        row = 0
        for e, c in enumerate(self.counts):
            r = slice(row, row + c)
            for b in range(self.nb):
                at = slice(b * 128, min(self.k, (b + 1) * 128))
                w = self.b[e, :, at].T if self.form == "forward" else self.b[e, at]
                s = (sb[e, :, b] if self.form == "forward" else sb[e, b]).repeat(128)[:self.n]
                out[r] += (self.a[r, at].astype(float) @ w.astype(float)) * sa[b, r][:, None] * s[None]
            row += c
        return out


def _id(v):
    return "-".join(str(x) for x in v)


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_scales_far_from_one(cuda, case):
    """Blocks whose two scales are far apart and multiply to 1, so that one of
    them times the sum may leave f32 on the way to a small result."""
    c = Case(np.random.default_rng(1), *case)
    for b in range(c.nb):
        c.scale(b, *FAR[b % len(FAR)])
    c.a *= 8
    c.b *= 8  # sums up to 2^16
    assert (c.run(cuda) == c.reference()).all()
    cuda.device_status()


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_zero_sums_under_large_scales(cuda, case):
    """Every other block sums to zero (a has numbers in its first half, b in
    its second) under scales of 2^100 each, whose product is infinite."""
    c = Case(np.random.default_rng(2), *case)
    for b in range(0, c.nb, 2):
        c.scale(b, 100, 100)
        c.a[:, b * 128 + 64:(b + 1) * 128] = 0
        if c.form == "dinput":
            c.b[:, b * 128:b * 128 + 64] = 0
        else:
            c.b[..., b * 128:b * 128 + 64] = 0
    assert (c.run(cuda) == c.reference()).all()
    cuda.device_status()


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_large_sums_under_small_scales(cuda, case):
    """Numbers of 2^14 and more in e5m2 under scales of 2^-75 each: the product
    of the scales is zero in f32, the result is about 2^-110."""
    c = Case(np.random.default_rng(3), *case)
    for b in range(c.nb):
        c.scale(b, -75, -75)
    c.a *= 1 << 14
    c.b *= 1 << 14
    operands = c.operands(cuda, ("e5m2", "e5m2"))
    ref = c.reference()
    assert np.abs(ref).max() > 2.0 ** -120
    assert (c.run(cuda, operands) == ref).all()
    cuda.device_status()


BAD = {"1.5": 1.5, "zero": 0.0, "negative": -1.0, "inf": np.inf, "nan": np.nan, "subnormal": 2.0 ** -127}


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("side", ["a", "b"])
@pytest.mark.parametrize("case", [c for c in CASES if not c[-1]], ids=_id)
def test_a_scale_that_is_no_power_of_two(cuda, case, side, bad):
    """Whatever the size, the numbers under it are NaN, no others, and it is
    reported."""
    from chelis_b200 import lib as L
    c = Case(np.random.default_rng(4), *case)
    good = c.run(cuda)
    cuda.device_status()
    a, b = c.operands(cuda)
    hit = np.zeros(good.shape, bool)
    e = len(c.counts) - 1  # the last expert has rows
    if c.form == "dweight":
        block = c.starts[e]
        if side == "a":
            a.scales[block, 7] = BAD[bad]
            hit[..., 7, :][(e,) if c.experts else ()] = True
        else:
            b.scales[block, 9] = BAD[bad]
            hit[..., 9][(e,) if c.experts else ()] = True
    elif side == "a":
        a.scales[c.nb - 1, c.m - 1] = BAD[bad]
        hit[c.m - 1] = True
    else:
        at = (0, c.nb - 1) if c.form == "forward" else (c.nb - 1, 0)
        b.scales[(e, *at) if c.experts else at] = BAD[bad]
        hit[c.m - c.counts[e]:, :128] = True
    y = c.run(cuda, (a, b))
    with pytest.raises(L.ChelisCudaError, match="power of two"):
        cuda.device_status()
    assert np.isnan(y[hit]).all()
    assert (y[~hit] == good[~hit]).all()
    cuda.device_status()


@pytest.mark.parametrize("case", [c for c in CASES if c[0] != "dweight" and c[4] and not c[-1]], ids=_id)
def test_scales_under_no_numbers(cuda, case):
    """Those of an expert without rows, and of rows that no expert holds, are
    nobody's: whatever they are, nothing changes and nothing is reported."""
    c = Case(np.random.default_rng(6), *case)
    c.counts[-1] -= 1  # the last row is held by none
    good = c.run(cuda)
    a, b = c.operands(cuda)
    a.scales[:, -1] = float("nan")
    b.scales[1] = 1.5  # the second expert has no rows
    assert (c.run(cuda, (a, b)) == good).all()
    cuda.device_status()


@pytest.mark.parametrize("case", [c[:-1] + (True,) for c in CASES if c[1] < 3000], ids=_id)
def test_any_scales(cuda, case):
    """any_scales takes them all, in the gradients too: fractions, zeros,
    negative and subnormal ones."""
    rng = np.random.default_rng(5)
    c = Case(rng, *case)
    c.factor_a = rng.choice([0.75, 1.25, -1.5, 1.0, 0.0], c.factor_a.shape)
    c.factor_b = rng.choice([0.75, 1.25, -1.5, 1.0], c.factor_b.shape)
    for b in range(c.nb):
        c.scale(b, *[(0, 0), (-127, 127), (3, -3)][b % 3])
    assert (c.run(cuda) == c.reference()).all()
    cuda.device_status()

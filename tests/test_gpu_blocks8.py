"""8-bit matrices with a scale for each block of 128, and their products.

Quantising divides by a power of two and rounds once, so data and scales are
equal to the float64 evaluation.  A product of two 8-bit numbers is exact in
f32; a sum of k of them in f32, in any order and with truncation where the
tensor core truncates, is within (k + 2) 2^-23 of the sum of magnitudes,
which is the bound of the 16-bit products (tests/test_gpu_gemm.py) and covers
the scales (two f32 roundings a block); then half an ulp of the result's type
(_experts_ref.half_ulp).
"""
import numpy as np
import pytest

import _experts_ref as R

pytestmark = pytest.mark.gpu


def _dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _values(data):
    return data.float().cpu().double().numpy()


def _same(got, ref):
    assert got.shape == ref.shape
    assert ((got == ref) | (np.isnan(got) & np.isnan(ref))).all()


def _input(rng, shape, dtype):
    import torch
    v = rng.standard_normal(shape) * np.exp(rng.standard_normal((*shape[:-1], 1)) * 2)
    x = torch.from_numpy(v).to(_dtype(dtype))
    return x.cuda(), x.double().numpy()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,cols,dtype", [(1, 1, "f32"), (1, 128, "bf16"), (17, 100, "f16"),
                                             (33, 257, "f32"), (16, 1024, "bf16"), (130, 264, "bf16"),
                                             (5, 1000, "f16")])
def test_quantize_rows(cuda, rows, cols, dtype, fmt):
    rng = np.random.default_rng(rows + cols)
    x, xr = _input(rng, (rows, cols), dtype)
    b = cuda.quantize8(x, fmt)
    q, s = R.quantize(xr, fmt, 1)
    assert b.data.shape == (rows, -(-cols // 16) * 16)
    _same(_values(b.data)[:, :cols], q)
    assert not _values(b.data)[:, cols:].any()
    _same(b.scales.cpu().double().numpy(), s.T)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("batch,rows,cols,dtype", [(None, 1, 1, "f32"), (None, 128, 128, "bf16"),
                                                   (3, 130, 200, "f32"), (2, 5, 300, "f16")])
def test_quantize_tiles(cuda, batch, rows, cols, dtype, fmt):
    rng = np.random.default_rng(rows + cols)
    x, xr = _input(rng, (rows, cols) if batch is None else (batch, rows, cols), dtype)
    b = cuda.quantize8(x, fmt, "tiles")
    ref = [R.quantize(m, fmt, 128) for m in (xr[None] if batch is None else xr)]
    data, scales = _values(b.data), b.scales.cpu().double().numpy()
    if batch is None:
        data, scales = data[None], scales[None]
    _same(data[..., :cols], np.stack([q for q, _ in ref]))
    assert not data[..., cols:].any()
    _same(scales, np.stack([s for _, s in ref]))


def _turned(xr, counts, fmt, blocks):
    """Float64 form of quantize8_transposed."""
    rows, cols = xr.shape
    padded = np.zeros((blocks * 128, cols))
    at = row = 0
    for c in counts:
        padded[at:at + c] = xr[row:row + c]
        row += c
        at += -(-c // 128) * 128
    q, s = R.quantize(np.ascontiguousarray(padded.T), fmt, 1)
    return q, s.T


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("counts,loose,cols,dtype", [([1], 0, 1, "f32"), ([300], 0, 130, "bf16"),
                                                     ([5, 0, 128, 129], 0, 136, "f32"),
                                                     ([0, 0], 7, 40, "f16"), ([200, 1, 55], 3, 96, "bf16")])
def test_quantize_transposed(cuda, counts, loose, cols, dtype, fmt):
    import torch
    rng = np.random.default_rng(cols)
    rows = sum(counts) + loose  # loose rows belong to no expert
    x, xr = _input(rng, (rows, cols), dtype)
    if len(counts) == 1:
        b, blocks = cuda.quantize8_transposed(x, fmt), -(-rows // 128)
    else:
        off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
        b, blocks = cuda.quantize8_transposed(x, fmt, off), rows // 128 + len(counts)
    q, s = _turned(xr, counts, fmt, blocks)
    _same(_values(b.data), q)
    _same(b.scales.cpu().double().numpy(), s)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_special_values(cuda, fmt):
    import torch
    inf, nan = float("inf"), float("nan")
    big = torch.finfo(torch.float32).max
    x = torch.zeros((8, 128))
    x[1, :4] = torch.tensor([inf, -inf, nan, 3.0])
    x[2, :3] = torch.tensor([inf, nan, 0.0])
    x[3, :4] = torch.tensor([big, -big, 1.0, 2.0 ** -149])
    x[4, :3] = torch.tensor([2.0 ** -149, -2.0 ** -140, 2.0 ** -126])
    x[5, :4] = torch.tensor([448.0, 449.0, -57344.0, 57345.0])
    # ties to even, in steps of the block's largest binade
    x[6] = torch.arange(128) * 3.5
    x[7] = -(torch.arange(128) + 0.5) / 7
    for blocks in ("rows", "transposed"):
        if blocks == "rows":
            b = cuda.quantize8(x.cuda(), fmt)
            q, s = R.quantize(x.double().numpy(), fmt, 1)
            s = s.T
        else:
            b = cuda.quantize8_transposed(x.t().contiguous().cuda(), fmt)
            q, s = _turned(x.t().double().numpy(), [128], fmt, 1)
        _same(_values(b.data), q)
        _same(b.scales.cpu().double().numpy(), s)


def _counts(rng, rows, experts):
    c = rng.multinomial(rows, rng.dirichlet(np.ones(experts) * 0.7))
    c[rng.integers(experts)] = 0
    return c


def _offsets(counts):
    import torch
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def _near(got, ref, mag, k, dtype):
    assert not R.outside(got.double().cpu().numpy(), ref, (k + 2) * 2.0 ** -23 * mag, dtype).any()


def _operands(cuda, rng, rows, n, k, experts, trans_b, fa, fb):
    """a, b as Blocks8, and the numbers they stand for."""
    a, _ = _input(rng, (rows, k), "f32")
    a8 = cuda.quantize8(a, fa)
    shape = (n, k) if trans_b else (k, n)
    b, _ = _input(rng, shape if experts is None else (experts, *shape), "f32")
    b8 = cuda.quantize8(b, fb, "tiles")
    va = R.values(_values(a8.data)[:, :k], a8.scales.cpu().double().numpy().T, 1)
    data, s = _values(b8.data)[..., :b8.cols], b8.scales.cpu().double().numpy()
    vb = R.values(data, s, 128) if experts is None else np.stack([R.values(d, t, 128) for d, t in zip(data, s)])
    return a8, b8, va, vb if not trans_b else np.swapaxes(vb, -1, -2)


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("rows,n,k,fa,fb,dtype", [
    (1, 1, 1, "e4m3", "e4m3", "f32"), (1, 256, 512, "e4m3", "e4m3", "bf16"),
    (2, 130, 100, "e5m2", "e4m3", "f16"), (7, 129, 1000, "e4m3", "e5m2", "f32"),
    (16, 384, 2048, "e4m3", "e4m3", "f32"), (31, 100, 257, "e5m2", "e5m2", "bf16"),
    (33, 512, 640, "e4m3", "e4m3", "bf16"), (127, 72, 129, "e4m3", "e4m3", "f32"),
    (128, 256, 128, "e4m3", "e4m3", "f32"), (129, 257, 384, "e5m2", "e4m3", "f32"),
    (300, 520, 1100, "e4m3", "e4m3", "f16"), (257, 1024, 4096, "e4m3", "e4m3", "f32")])
def test_matmul8_dense(cuda, rows, n, k, fa, fb, dtype, trans_b):
    import torch
    rng = np.random.default_rng(rows * n + k)
    a8, b8, va, vb = _operands(cuda, rng, rows, n, k, None, trans_b, fa, fb)
    y = cuda.matmul8(a8, b8, trans_b, dtype=_dtype(dtype))
    _near(y, va @ vb, np.abs(va) @ np.abs(vb), k, dtype)
    assert torch.equal(y, cuda.matmul8(a8, b8, trans_b, dtype=_dtype(dtype)))
    cuda.device_status()


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("rows,loose,n,k,experts,dtype", [
    (3, 0, 64, 128, 2, "f32"), (16, 0, 256, 384, 8, "bf16"), (40, 5, 200, 520, 3, "f32"),
    (64, 0, 129, 130, 33, "f16"), (500, 0, 257, 300, 4, "f32"), (1000, 77, 384, 256, 5, "bf16"),
    (700, 3, 520, 1030, 2, "f32"), (2, 2, 1000, 64, 1000, "f32")])
def test_matmul8_by_expert(cuda, rows, loose, n, k, experts, dtype, trans_b):
    rng = np.random.default_rng(rows + n + k)
    counts = _counts(rng, rows, experts)
    a8, b8, va, vb = _operands(cuda, rng, rows + loose, n, k, experts, trans_b, "e4m3", "e4m3")
    y = cuda.matmul8(a8, b8, trans_b, _offsets(counts), _dtype(dtype))
    ref = np.zeros((rows + loose, n))
    mag = np.zeros((rows + loose, n))
    at = 0
    for e, c in enumerate(counts):
        ref[at:at + c] = va[at:at + c] @ vb[e]
        mag[at:at + c] = np.abs(va[at:at + c]) @ np.abs(vb[e])
        at += c
    _near(y, ref, mag, k, dtype)
    assert not y[rows:].any()
    cuda.device_status()


@pytest.mark.parametrize("counts,loose,n,k,fa,fb,dtype", [
    ([1], 0, 1, 1, "e4m3", "e4m3", "f32"), ([300], 0, 130, 260, "e5m2", "e4m3", "f32"),
    ([128], 0, 256, 512, "e4m3", "e4m3", "bf16"), ([5, 0, 128, 129], 0, 136, 100, "e5m2", "e4m3", "f32"),
    ([0, 0], 9, 40, 300, "e4m3", "e4m3", "f32"), ([700, 1, 55, 0, 400], 3, 257, 129, "e5m2", "e5m2", "f16")])
def test_matmul8_wgrad(cuda, counts, loose, n, k, fa, fb, dtype):
    rng = np.random.default_rng(n + k)
    rows = sum(counts) + loose
    dy, _ = _input(rng, (rows, n), "f32")
    x, _ = _input(rng, (rows, k), "f32")
    off = _offsets(counts) if len(counts) > 1 else None
    a8, b8 = cuda.quantize8_transposed(dy, fa, off), cuda.quantize8_transposed(x, fb, off)
    va = R.values(_values(a8.data), a8.scales.cpu().double().numpy().T, 1)
    vb = R.values(_values(b8.data), b8.scales.cpu().double().numpy().T, 1)
    got = cuda.matmul8_wgrad(a8, b8, off, _dtype(dtype))
    at = 0
    for e, c in enumerate(counts):
        end = at + -(-c // 128) * 128
        ref = va[:, at:end] @ vb[:, at:end].T
        mag = np.abs(va[:, at:end]) @ np.abs(vb[:, at:end]).T
        _near(got[e] if off is not None else got, ref, mag, c, dtype)
        at = end
    cuda.device_status()


def test_products_are_each_other_s_gradients(cuda):
    """<x W^T, dy> = <dy W, x> = <dy^T x, W> on the numbers that the operands
    stand for: x and dy take few enough values that every 8-bit form of them
    is exact, and the inner products differ by the products' f32 roundings."""
    import torch
    gen = torch.Generator().manual_seed(3)
    rows, n, k = 200, 144, 272
    x = torch.randint(-8, 9, (rows, k), generator=gen).float()
    dy = torch.randint(-4, 5, (rows, n), generator=gen).float()
    w = torch.randint(-8, 9, (n, k), generator=gen).float()
    w8 = cuda.quantize8(w.cuda(), "e4m3", "tiles")
    y = cuda.matmul8(cuda.quantize8(x.cuda()), w8, dtype=torch.float32).cpu()
    dx = cuda.matmul8(cuda.quantize8(dy.cuda(), "e5m2"), w8, trans_b=False, dtype=torch.float32).cpu()
    dw = cuda.matmul8_wgrad(cuda.quantize8_transposed(dy.cuda(), "e5m2"),
                            cuda.quantize8_transposed(x.cuda())).cpu()
    # small integers: every sum is below 2^24 and exact
    assert torch.equal(y, x @ w.t()) and torch.equal(dx, dy @ w) and torch.equal(dw, dy.t() @ x)
    inner = [(a.double() * b.double()).sum().item() for a, b in ((y, dy), (dx, x), (dw, w))]
    assert inner[0] == inner[1] == inner[2]


def test_matmul8_takes_any_scales(cuda):
    """Scales that are no powers of two, as another quantiser may choose them."""
    import torch
    rng = np.random.default_rng(9)
    a8, b8, _, _ = _operands(cuda, rng, 150, 200, 300, None, True, "e4m3", "e4m3")
    a8 = a8._replace(scales=torch.rand_like(a8.scales) + 0.5)
    b8 = b8._replace(scales=torch.rand_like(b8.scales) + 0.5)
    va = R.values(_values(a8.data)[:, :300], a8.scales.cpu().double().numpy().T, 1)
    vb = R.values(_values(b8.data)[:, :300], b8.scales.cpu().double().numpy(), 128).T
    for rows in (150, 4):
        part = a8._replace(data=a8.data[:rows].contiguous(), scales=a8.scales[:, :rows].contiguous())
        y = cuda.matmul8(part, b8, dtype=torch.float32, any_scales=True)
        _near(y, va[:rows] @ vb, np.abs(va[:rows]) @ np.abs(vb), 300, "f32")


@pytest.mark.parametrize("rows,n,k,counts,fa,fb,dtype,trans_b", [
    (2100, 1000, 4100, None, "e4m3", "e4m3", "f32", True), (2049, 4096, 1000, None, "e5m2", "e4m3", "bf16", True),
    (2100, 1000, 4100, None, "e5m2", "e4m3", "f32", False), (1500, 3001, 1500, None, "e4m3", "e5m2", "f16", True),
    (2200, 2040, 900, [1000, 0, 7, 513, 670], "e4m3", "e4m3", "f32", True),
    (4700, 520, 4200, [2500, 2190], "e4m3", "e4m3", "bf16", False),
    (1700, 2055, 1300, [0, 900, 800, 0], "e5m2", "e5m2", "f32", False)])
def test_matmul8_large(cuda, rows, n, k, counts, fa, fb, dtype, trans_b):
    """Enough work for the kernel that leaves the scales to the tensor core, in
    single blocks and in pairs, with ragged rows and columns."""
    import torch
    rng = np.random.default_rng(rows + n + k)
    a8, b8, va, vb = _operands(cuda, rng, rows, n, k, None if counts is None else len(counts), trans_b, fa, fb)
    off = None if counts is None else _offsets(counts)
    y = cuda.matmul8(a8, b8, trans_b, off, _dtype(dtype))
    at = 0
    for e, c in enumerate([rows] if counts is None else counts):
        w = vb if counts is None else vb[e]
        _near(y[at:at + c], va[at:at + c] @ w, np.abs(va[at:at + c]) @ np.abs(w), k, dtype)
        at += c
    assert not y[at:].any()
    assert torch.equal(y, cuda.matmul8(a8, b8, trans_b, off, _dtype(dtype)))
    cuda.device_status()


@pytest.mark.parametrize("counts,n,k,dtype", [([4300], 1500, 1300, "f32"), ([1700], 2000, 2300, "bf16"),
                                              ([3000, 0, 130, 5000, 1], 1100, 1030, "f32"),
                                              ([128, 640, 500, 700], 2048, 2048, "f16")])
def test_matmul8_wgrad_large(cuda, counts, n, k, dtype):
    rng = np.random.default_rng(n + k)
    rows = sum(counts)
    dy, _ = _input(rng, (rows, n), "f32")
    x, _ = _input(rng, (rows, k), "f32")
    off = _offsets(counts) if len(counts) > 1 else None
    a8, b8 = cuda.quantize8_transposed(dy, "e5m2", off), cuda.quantize8_transposed(x, "e4m3", off)
    va = R.values(_values(a8.data), a8.scales.cpu().double().numpy().T, 1)
    vb = R.values(_values(b8.data), b8.scales.cpu().double().numpy().T, 1)
    got = cuda.matmul8_wgrad(a8, b8, off, _dtype(dtype))
    at = 0
    for e, c in enumerate(counts):
        end = at + -(-c // 128) * 128
        _near(got[e] if off is not None else got, va[:, at:end] @ vb[:, at:end].T,
              np.abs(va[:, at:end]) @ np.abs(vb[:, at:end]).T, c, dtype)
        at = end
    cuda.device_status()


# Few tiles and long contractions, which are cut into parts: both kernels, last parts that are
# short, experts without rows, rows that no expert holds, results off 16 bytes.
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("rows,n,k,counts,any_scales,dtype", [
    (100, 300, 2600, None, False, "bf16"), (129, 40, 1400, None, True, "f32"), (70, 517, 4000, None, False, "f16"),
    (95, 129, 2100, [50, 0, 40], False, "f16"), (300, 1000, 19200, None, False, "f32"),
    (287, 1001, 9500, [100, 0, 180], False, "bf16")])
def test_matmul8_in_parts(cuda, rows, n, k, counts, any_scales, dtype, trans_b):
    import torch
    rng = np.random.default_rng(rows + n + k)
    a8, b8, va, vb = _operands(cuda, rng, rows, n, k, None if counts is None else len(counts), trans_b, "e4m3", "e5m2")
    off = None if counts is None else _offsets(counts)
    y = cuda.matmul8(a8, b8, trans_b, off, _dtype(dtype), any_scales=any_scales)
    at = 0
    for e, c in enumerate([rows] if counts is None else counts):
        w = vb if counts is None else vb[e]
        _near(y[at:at + c], va[at:at + c] @ w, np.abs(va[at:at + c]) @ np.abs(w), k, dtype)
        at += c
    assert not y[at:].any()
    assert torch.equal(y, cuda.matmul8(a8, b8, trans_b, off, _dtype(dtype), any_scales=any_scales))
    cuda.device_status()


@pytest.mark.parametrize("counts,n,k,any_scales,dtype", [
    ([9001], 77, 263, False, "f32"), ([3000, 0, 130, 5000, 1], 100, 300, False, "bf16"), ([2600], 128, 256, True, "f16"),
    ([60000], 520, 600, False, "f32"), ([40000, 0, 15000, 1], 301, 520, False, "f16")])
def test_matmul8_wgrad_in_parts(cuda, counts, n, k, any_scales, dtype):
    import torch
    rng = np.random.default_rng(n + k)
    rows = sum(counts)
    dy, _ = _input(rng, (rows, n), "f32")
    x, _ = _input(rng, (rows, k), "f32")
    off = _offsets(counts) if len(counts) > 1 else None
    a8, b8 = cuda.quantize8_transposed(dy, "e5m2", off), cuda.quantize8_transposed(x, "e4m3", off)
    va = R.values(_values(a8.data), a8.scales.cpu().double().numpy().T, 1)
    vb = R.values(_values(b8.data), b8.scales.cpu().double().numpy().T, 1)
    got = cuda.matmul8_wgrad(a8, b8, off, _dtype(dtype), any_scales=any_scales)
    at = 0
    for e, c in enumerate(counts):
        end = at + -(-c // 128) * 128
        _near(got[e] if off is not None else got, va[:, at:end] @ vb[:, at:end].T,
              np.abs(va[:, at:end]) @ np.abs(vb[:, at:end]).T, c, dtype)
        at = end
    assert torch.equal(got, cuda.matmul8_wgrad(a8, b8, off, _dtype(dtype), any_scales=any_scales))
    cuda.device_status()


def test_matmul8_reports_scales_that_are_no_powers_of_two(cuda):
    """Where the tensor core applies the scales it takes powers of two; another
    one makes the numbers under it NaN, is reported, and any_scales admits it."""
    import torch
    from chelis_b200 import lib as L
    a8 = cuda.quantize8(torch.ones((2048, 1024), device="cuda"))
    b8 = cuda.quantize8(torch.ones((4096, 1024), device="cuda"), "e4m3", "tiles")
    a8.scales[3, 77] *= 1.5
    y = cuda.matmul8(a8, b8)
    torch.cuda.synchronize()
    with pytest.raises(L.ChelisCudaError, match="power of two"):
        cuda.device_status()
    assert y[77].isnan().all() and not y[:77].isnan().any() and not y[78:].isnan().any()
    z = cuda.matmul8(a8, b8, any_scales=True)
    cuda.device_status()
    assert (z[77] == 1024 + 64).all() and (z[78:] == 1024).all()


def test_matmul8_keeps_nan_to_its_row(cuda):
    import torch
    for rows in (3, 140):
        x = torch.ones((rows, 256), device="cuda")
        x[1, 7] = float("nan")
        w8 = cuda.quantize8(torch.ones((64, 256), device="cuda"), "e4m3", "tiles")
        y = cuda.matmul8(cuda.quantize8(x), w8, dtype=torch.float32)
        assert y[1].isnan().all()
        assert (y[torch.arange(rows) != 1] == 256.0).all()


def test_refusals(cuda):
    import torch
    x = torch.zeros((4, 40), device="cuda")
    a8 = cuda.quantize8(x)
    w8 = cuda.quantize8(torch.zeros((6, 40), device="cuda"), "e4m3", "tiles")
    stack = cuda.quantize8(torch.zeros((2, 6, 40), device="cuda"), "e4m3", "tiles")
    off = torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda")
    for call in (lambda: cuda.quantize8(x, "e3m4"), lambda: cuda.quantize8(x, "e4m3", "columns"),
                 lambda: cuda.quantize8(x.double()), lambda: cuda.quantize8(x.t()),
                 lambda: cuda.quantize8(x.cpu()), lambda: cuda.quantize8(x[None]),
                 lambda: cuda.quantize8_transposed(x, "e4m3", off.long()),
                 lambda: cuda.matmul8(a8, a8), lambda: cuda.matmul8(w8, w8),
                 lambda: cuda.matmul8(a8, w8, trans_b=False), lambda: cuda.matmul8(a8, w8, offsets=off),
                 lambda: cuda.matmul8(a8, stack), lambda: cuda.matmul8(a8, stack, offsets=off[:2]),
                 lambda: cuda.matmul8(a8, w8, dtype=torch.float64),
                 lambda: cuda.matmul8(a8._replace(scales=a8.scales.double()), w8),
                 lambda: cuda.matmul8(a8._replace(scales=a8.scales.t()), w8),
                 lambda: cuda.matmul8(a8._replace(cols=41), w8),
                 lambda: cuda.matmul8_wgrad(a8, a8)):
        with pytest.raises(ValueError):
            call()
    # empty operands
    assert cuda.quantize8(torch.zeros((0, 40), device="cuda")).data.shape == (0, 48)
    assert cuda.matmul8(cuda.quantize8(torch.zeros((0, 40), device="cuda")), w8).shape == (0, 6)

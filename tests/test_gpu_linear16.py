"""The 16-bit product with bias, activation and residual, its gradients'
products, the activations' gradients and column sums, against float64.

Bounds are _sublayer_ref's; products of small whole numbers are equal, in every
layout, by every kernel (few rows; tiles of 128 and 256 columns; parts)."""
import numpy as np
import pytest

import _sublayer_ref as S

pytestmark = pytest.mark.gpu

DT = ["bf16", "f16"]


def _t(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _make(rng, shape, dtype, scale=1.0):
    import torch
    x = torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(_t(dtype))
    return x.cuda(), x.double().numpy()


def _operands(rng, m, n, k, ta, tb, dtype):
    """(a, b) on the device as they lie, and as [m, k] and [k, n] in float64."""
    a, fa = _make(rng, (k, m) if ta else (m, k), dtype)
    b, fb = _make(rng, (n, k) if tb else (k, n), dtype, 1.0 / np.sqrt(k))
    return a, b, fa.T if ta else fa, fb.T if tb else fb


# few rows (m <= 16, or little to read); tiles alone and many, ends of every kind; parts (a long k)
SHAPES = [(1, 1, 1), (1, 16, 8), (1, 4096, 1024), (3, 17, 33), (8, 1000, 264), (9, 65, 72), (17, 72, 512), (32, 200, 200),
          (33, 8, 16), (64, 128, 64), (128, 256, 128), (200, 136, 72), (257, 300, 100), (300, 257, 65), (129, 31, 70),
          (700, 1000, 264), (100, 264, 4160), (1500, 2600, 192), (50, 129, 40), (64, 1024, 72), (40, 3000, 4104), (20, 4104, 2056)]


@pytest.mark.parametrize("tb", [False, True])
@pytest.mark.parametrize("ta", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_whole_numbers_are_equal(cuda, m, n, k, ta, tb):
    import torch
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    for dtype in DT:
        a = torch.from_numpy(rng.integers(-4, 5, (k, m) if ta else (m, k))).to(_t(dtype)).cuda()
        b = torch.from_numpy(rng.integers(-4, 5, (n, k) if tb else (k, n))).to(_t(dtype)).cuda()
        bias = torch.from_numpy(rng.integers(-4, 5, n).astype(np.float32)).cuda()
        res = torch.from_numpy(rng.integers(-4, 5, (m, n)).astype(np.float32)).cuda()
        # |sums| <= 16 k + 8 < 2^24: f32 holds them and all on the way
        got = cuda.matmul16(a, b, ta, tb, bias=bias, residual=res, dtype=torch.float32)
        ref = (a.double().t() if ta else a.double()) @ (b.double().t() if tb else b.double()) + bias.double() + res.double()
        assert torch.equal(got.double(), ref)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k,ta,tb,activation,bias,residual,keep,out", [
    (1, 4096, 1024, False, False, "gelu", "bf16", False, False, None),
    (8, 1024, 512, False, True, "silu", "f32", True, True, None),
    (5, 33, 47, False, True, "relu", None, True, True, None),
    (20, 72, 100, False, False, "gelu", "f32", True, True, "f32"),
    (64, 128, 64, False, False, "gelu", "same", False, True, None),
    (130, 264, 200, False, True, "silu", "same", True, False, None),
    (130, 264, 200, True, False, None, "f32", True, True, None),
    (257, 200, 136, False, False, "relu", None, True, True, None),
    (300, 301, 99, True, True, "gelu", "same", True, True, None),
    (300, 302, 99, False, True, "silu", "f32", False, True, None),
    (260, 300, 64, False, False, "gelu", "same", True, True, "f32"),
    (260, 301, 64, False, False, None, "same", True, True, "f32"),
    (90, 264, 4160, False, False, "gelu", "same", True, True, None),   # parts
    (90, 263, 4160, False, True, "silu", "f32", True, True, "f32"),
    (3000, 1032, 192, False, False, "gelu", "same", True, True, None),  # more tiles than pairs
    (700, 3000, 136, False, False, "silu", "same", False, True, None),
])
def test_product_and_what_follows(cuda, m, n, k, ta, tb, activation, bias, residual, keep, out, dtype):
    import torch
    rng = np.random.default_rng(m + n + k)
    a, b, fa, fb = _operands(rng, m, n, k, ta, tb, dtype)
    bt = {"same": dtype, "bf16": dtype}.get(bias, bias)
    bv, fbias = _make(rng, (n,), bt, 0.5) if bias else (None, None)
    od = out or dtype
    rv, fres = _make(rng, (m, n), od) if residual else (None, None)
    got = cuda.matmul16(a, b, ta, tb, bias=bv, activation=activation, residual=rv, keep_pre=keep,
                        dtype=None if out is None else _t(out))
    y, bound, z, ez = S.linear(fa, fb, fbias, activation, fres)
    if keep:
        got, pre = got
        assert pre.dtype == got.dtype
        S.check(pre, z, ez, od)
    assert got.dtype == _t(od)
    S.check(got, y, bound, od)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k,activation,tb,out", [
    (4, 100, 64, "gelu", True, None), (31, 264, 72, "relu", False, None), (64, 128, 64, "silu", True, None),
    (257, 264, 136, "gelu", False, None), (257, 263, 100, "relu", True, None), (130, 264, 100, "silu", False, "f32"),
    (130, 261, 4160, "gelu", True, None), (2000, 1032, 72, "gelu", True, None)])
def test_gradient_through_an_activation(cuda, m, n, k, activation, tb, out, dtype):
    import torch
    rng = np.random.default_rng(m * n + k)
    a, b, fa, fb = _operands(rng, m, n, k, False, tb, dtype)
    od = out or dtype
    z, fz = _make(rng, (m, n), od, 2.0)
    z[:, ::7] = 0.0   # relu's slope at 0 is 0
    z[0, :1] = -0.0
    fz = z.double().cpu().numpy()
    got = cuda.matmul16(a, b, trans_b=tb, through=(z, activation), dtype=None if out is None else torch.float32)
    ref, bound = S.linear_through(fa, fb, fz, activation)
    S.check(got, ref, bound, od)


def _specials(dtype):
    import torch
    big = {"bf16": 3e38, "f16": 65504.0}[dtype]
    return torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), big, -big, 1e-7, -1e-7, -5.0, -13.0, 13.0,
                         17.0, -17.0, 90.0, -90.0], device="cuda")


@pytest.mark.parametrize("m", [4, 64])
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", DT)
def test_activations_of_special_numbers(cuda, dtype, activation, m):
    """By the bias of a product of zeros, whose z it is: infinities and NaN come
    out as the functions' limits; an f32 result is as close as the bounds say."""
    import torch
    v = _specials(dtype)
    n = v.numel()
    a = torch.zeros(m, 16, dtype=_t(dtype), device="cuda")
    b = torch.zeros(16, n, dtype=_t(dtype), device="cuda")
    z = v.double().cpu().numpy()
    ref, slope = S.act(z, activation)
    for out in (torch.float32, _t(dtype)):
        y, pre = cuda.matmul16(a, b, bias=v, activation=activation, keep_pre=True, dtype=out)
        if out == torch.float32:
            assert torch.equal(pre[0].nan_to_num(7.0), v.nan_to_num(7.0))
        y = y[m - 1].double().cpu().numpy()
        fin = np.isfinite(ref) & np.isfinite(y)
        assert (np.isnan(y) == np.isnan(ref)).all()
        assert (y[np.isinf(ref)] == ref[np.isinf(ref)]).all()
        if out == torch.float32:
            with np.errstate(invalid="ignore"):
                bound = S.act_error(z, activation) + 2 * S.U * np.abs(ref) + 2.0 ** -126
            assert (np.abs(y[fin] - ref[fin]) <= bound[fin]).all()
    # the slope of each, by the library's own gradient of 1 and by the product's
    if activation:
        zz = v.to(_t(dtype)).repeat(m, 1)
        fz = zz[0].double().cpu().numpy()
        slope = S.act(fz, activation)[1]
        g = cuda.activation16_bwd(torch.ones_like(zz), zz, activation)
        a[:, 0] = 1.0
        b[0] = 1.0
        for got in (g, cuda.matmul16(a, b, through=(zz, activation))):
            got = got[m - 1].double().cpu().numpy()
            want = np.where(np.isnan(fz), 0.0 if activation == "relu" else np.nan, slope)
            assert (np.isnan(got) == np.isnan(want)).all()
            ok = ~np.isnan(want)
            assert not S.R.outside(got[ok], want[ok], S.slope_error(want, activation)[ok] + 2 * S.U, dtype).any()


def test_infinities_in_the_operands(cuda):
    """An infinity or NaN of a row stays in that row, and past a ragged k nothing
    is multiplied."""
    import torch
    for m, k in ((3, 20), (70, 20), (70, 72)):
        a = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
        b = torch.ones(k, 24, dtype=torch.bfloat16, device="cuda")
        a[1, 3] = float("inf")
        a[2, k - 1] = float("nan")
        y = cuda.matmul16(a, b, activation="gelu").float()
        assert torch.isinf(y[1]).all() and (y[1] > 0).all() and torch.isnan(y[2]).all()
        assert (y[0] == k).all() and (y[3:] == k).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,n,k,tb,activation,wd", [(1, 40, 24, False, "gelu", "f32"), (37, 64, 136, True, None, "f32"),
                                                       (300, 200, 72, False, "silu", "same"), (515, 33, 65, True, "relu", "f32"),
                                                       (5000, 264, 72, False, "gelu", "f32")])
def test_gradients(cuda, rows, n, k, tb, activation, wd, dtype):
    rng = np.random.default_rng(rows + n)
    a, b, fa, fb = _operands(rng, rows, n, k, False, tb, dtype)
    dy, fdy = _make(rng, (rows, n), dtype, 0.1)
    z, fz = _make(rng, (rows, k), dtype)
    od = dtype if wd == "same" else wd
    da, db, dbias = cuda.matmul16_bwd(dy, a, b, tb, through=(z, activation) if activation else None, want_bias=True,
                                      weight_dtype=_t(od))
    if activation:
        ref, bound = S.linear_through(fdy, fb.T, fz, activation)
    else:
        ref, bound = S.product(fdy, fb.T)
    S.check(da, ref, bound, dtype)
    ref, bound = S.product(fa.T, fdy)
    S.check(db, ref.T if tb else ref, bound.T if tb else bound, od)
    assert db.shape == b.shape
    S.check(dbias, fdy.sum(0), rows * S.U * np.abs(fdy).sum(0), "f32")
    assert cuda.matmul16_bwd(dy, a, b, tb)[2] is None


def test_gradients_against_differences(cuda):
    """The directional derivative of sum(dy * (act(a . w1 + b1) . w2)) in float64
    by central differences, and by the calls' gradients: they differ by the 16-bit
    roundings of the hidden gradient and values (2^-9 each, three of them, of the
    terms' magnitudes)."""
    import torch
    rng = np.random.default_rng(11)
    x, fx = _make(rng, (40, 24), "bf16")
    w1, f1 = _make(rng, (24, 56), "bf16", 0.2)
    w2, f2 = _make(rng, (56, 16), "bf16", 0.2)
    b1, fb1 = _make(rng, (56,), "f32", 0.2)
    dy, fdy = _make(rng, (40, 16), "bf16")
    a, z = cuda.matmul16(x, w1, bias=b1, activation="gelu", keep_pre=True)
    dz, dw2, _ = cuda.matmul16_bwd(dy, a, w2, through=(z, "gelu"))
    dx, dw1, db1 = cuda.matmul16_bwd(dz, x, w1, want_bias=True)
    grads = [g.double().cpu().numpy() for g in (dx, dw1, dw2, db1)]

    def loss(x, w1, w2, b1):
        return float((fdy * (S.act(x @ w1 + b1, "gelu")[0] @ w2)).sum())

    at = [fx, f1, f2, fb1]
    fz = fx @ f1 + fb1
    # magnitudes of the terms that are summed
    hidden = np.abs(fdy) @ np.abs(f2).T * 1.13
    weight = [hidden @ np.abs(f1).T, np.abs(fx).T @ hidden, np.abs(S.act(fz, "gelu")[0]).T @ np.abs(fdy), hidden.sum(0)]
    for i in range(4):
        d = rng.standard_normal(at[i].shape)
        h = 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        numeric = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(numeric - float((grads[i] * d).sum())) <= 3 * 2.0 ** -9 * float((weight[i] * np.abs(d)).sum()) + 1e-6


@pytest.mark.parametrize("rows,cols", [(0, 5), (1, 1), (7, 33), (1000, 8), (4097, 264), (33, 5000)])
def test_column_sums(cuda, rows, cols):
    rng = np.random.default_rng(rows + cols)
    for dtype in DT:
        x, f = _make(rng, (rows, cols), dtype)
        S.check(cuda.column_sums16(x), f.sum(0), max(rows, 1) * S.U * np.abs(f).sum(0), "f32")


@pytest.mark.parametrize("count", [0, 1, 37, 8 * 300 * 3])
def test_activation_gradients(cuda, count):
    rng = np.random.default_rng(count)
    for dtype in DT:
        for activation in (None, "relu", "gelu", "silu"):
            g, fg = _make(rng, (count,), dtype)
            z, fz = _make(rng, (count,), dtype, 2.0)
            ref = fg * S.act(fz, activation)[1]
            bound = np.abs(fg) * (S.slope_error(fz, activation) + 2 * S.U * 1.13)
            S.check(cuda.activation16_bwd(g, z, activation), ref, bound, dtype)


def test_empty_products(cuda):
    import torch
    a = torch.zeros(40, 0, dtype=torch.float16, device="cuda")
    b = torch.zeros(0, 9, dtype=torch.float16, device="cuda")
    bias = torch.arange(9, dtype=torch.float32, device="cuda") - 4
    res = torch.ones(40, 9, dtype=torch.float16, device="cuda")
    y, z = cuda.matmul16(a, b, bias=bias, activation="relu", residual=res, keep_pre=True)
    assert torch.equal(y, (bias.clamp(min=0) + 1).half().expand(40, 9)) and torch.equal(z, bias.half().expand(40, 9))
    assert cuda.matmul16(b.t().contiguous(), a.t().contiguous()).shape == (9, 40)
    empty = torch.zeros(0, 16, dtype=torch.float16, device="cuda")
    w = torch.ones(16, 24, dtype=torch.float16, device="cuda")
    assert cuda.matmul16(empty, w, activation="gelu").shape == (0, 24)
    da, db, dbias = cuda.matmul16_bwd(torch.zeros(0, 24, dtype=torch.float16, device="cuda"), empty, w, want_bias=True)
    assert da.shape == (0, 16) and not db.any() and not dbias.any() and db.dtype == torch.float32


def test_unaligned_bases_and_neighbours(cuda):
    """Operands and results that start off 16 bytes, and nothing written around
    them: through the C entry, into the middle of a larger buffer."""
    import torch
    from chelis_b200 import lib as L
    rng = np.random.default_rng(5)
    for m, n, k in ((6, 40, 24), (70, 40, 24), (70, 264, 200)):
        for shift in (0, 1, 4, 8):
            whole = torch.from_numpy(rng.integers(-3, 4, shift + m * k)).bfloat16().cuda()
            a = whole[shift:].view(m, k)
            wb = torch.from_numpy(rng.integers(-3, 4, shift + k * n)).bfloat16().cuda()
            b = wb[shift:].view(k, n)
            out = torch.full((shift + m * n + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
            pre = torch.full_like(out, 9.0)
            y, z = out[shift:shift + m * n], pre[shift:shift + m * n]
            cuda._prepare(a, b)
            L.call("chelis_cuda_matmul16", L.DTYPE_BF16, 0, 0, m, n, k, a.data_ptr(), b.data_ptr(), None, 0, L.ACT_RELU,
                   None, None, z.data_ptr(), L.DTYPE_BF16, y.data_ptr())
            ref = a.double() @ b.double()
            assert torch.equal(z.view(m, n).double(), ref.bfloat16().double())
            assert torch.equal(y.view(m, n).double(), ref.clamp(min=0).bfloat16().double())
            for buf in (out, pre):
                assert (buf[:shift] == 9).all() and (buf[shift + m * n:] == 9).all()


def test_residual_may_be_the_result(cuda):
    import torch
    from chelis_b200 import lib as L
    rng = np.random.default_rng(6)
    for m, n in ((8, 64), (70, 264), (300, 263), (70, 264)):
        a, _ = _make(rng, (m, 136), "f16")
        b, _ = _make(rng, (136, n), "f16", 0.1)
        r, _ = _make(rng, (m, n), "f16")
        want = cuda.matmul16(a, b, activation="silu", residual=r)
        L.call("chelis_cuda_matmul16", L.DTYPE_F16, 0, 0, m, n, 136, a.data_ptr(), b.data_ptr(), None, 0, L.ACT_SILU,
               r.data_ptr(), None, None, L.DTYPE_F16, r.data_ptr())
        assert torch.equal(want, r)


def test_captured_and_on_other_streams(cuda):
    """Products with scratch (copies of unaligned operands, parts) in two graphs
    replayed at once, and eagerly on two streams at once, give the eager bits."""
    import torch
    rng = np.random.default_rng(8)
    sets = []
    for i in range(2):
        a, _ = _make(rng, (100, 4159 + i), "bf16")
        b, _ = _make(rng, (4159 + i, 201), "bf16", 0.02)
        sets.append((a, b, cuda.matmul16(a, b, activation="gelu"), cuda.matmul16_bwd(cuda.matmul16(a, b), a, b)[1]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for s, (a, b, *_) in zip(streams, sets):
        with torch.cuda.stream(s):
            cuda.matmul16(a, b)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append((cuda.matmul16(a, b, activation="gelu"), cuda.matmul16_bwd(cuda.matmul16(a, b), a, b)[1]))
            graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, y, w), (gy, gw) in zip(sets, outs):
            assert torch.equal(y, gy) and torch.equal(w, gw)
    eager = []
    for s, (a, b, *_) in zip(streams, sets):
        with torch.cuda.stream(s):
            eager.append([cuda.matmul16(a, b, activation="gelu") for _ in range(3)])
    torch.cuda.synchronize()
    for (_, _, y, _), got in zip(sets, eager):
        assert all(torch.equal(y, g) for g in got)
    cuda.device_status()


def test_offsets_past_32_bits(cuda):
    """Results, residuals and column sums of more than 2^31 numbers: the last rows
    are those of a small product."""
    import torch
    m, n = (1 << 19) + 300, 4104
    gen = torch.Generator(device="cuda").manual_seed(1)
    a = torch.randn((m, 16), generator=gen, device="cuda").bfloat16()
    b = torch.randn((16, n), generator=gen, device="cuda").bfloat16()
    res = torch.randn((m, n), device="cuda", dtype=torch.bfloat16)
    y, z = cuda.matmul16(a, b, activation="gelu", residual=res, keep_pre=True)
    for rows in (slice(0, 300), slice(m - 300, m)):
        sy, sz = cuda.matmul16(a[rows].contiguous(), b, activation="gelu", residual=res[rows].contiguous(), keep_pre=True)
        assert torch.equal(y[rows], sy) and torch.equal(z[rows], sz)
    g = cuda.activation16_bwd(y, z, "silu")
    assert torch.equal(g[-300:], cuda.activation16_bwd(sy, sz, "silu"))
    ones = torch.ones_like(res)
    assert torch.equal(cuda.column_sums16(ones), torch.full((n,), float(m), device="cuda"))
    w = cuda.matmul16(a, ones, trans_a=True, dtype=torch.float32)  # sums over all rows
    ref = a.double().sum(0)
    assert float((w.double() - ref[:, None]).abs().max()) <= (m + 2) * 2.0 ** -23 * float(a.double().abs().sum(0).max())


def test_refusals(cuda):
    import torch
    a = torch.zeros(8, 16, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(16, 24, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: cuda.matmul16(a, b.half()), lambda: cuda.matmul16(a.float(), b.float()),
                lambda: cuda.matmul16(a, b, trans_b=True), lambda: cuda.matmul16(a[0], b),
                lambda: cuda.matmul16(a, b, dtype=torch.float16), lambda: cuda.matmul16(a, b, activation="tanh"),
                lambda: cuda.matmul16(a, b, bias=torch.zeros(8, device="cuda")),
                lambda: cuda.matmul16(a, b, bias=torch.zeros(24, dtype=torch.float16, device="cuda")),
                lambda: cuda.matmul16(a, b, residual=torch.zeros(8, 24, device="cuda")),
                lambda: cuda.matmul16(a, b, through=(torch.zeros_like(a), "gelu")),
                lambda: cuda.matmul16(a, b, through=(torch.zeros(8, 24, dtype=a.dtype, device="cuda"), "gelu"), keep_pre=True),
                lambda: cuda.matmul16(a, b.t().contiguous().t()), lambda: cuda.matmul16(a, b.cpu()),
                lambda: cuda.matmul16_bwd(a, a, b), lambda: cuda.activation16_bwd(a, b, "gelu"),
                lambda: cuda.column_sums16(a.float())):
        with pytest.raises(ValueError):
            bad()


# f32 results by chunks of the contraction (k > 1024): tiles of 256 and 128 columns, and parts of more than a chunk
@pytest.mark.parametrize("m,n,k,ta,tb", [(300, 5000, 2200, False, False), (300, 2600, 2049, False, True), (513, 5001, 1100, True, False),
                                         (300, 5000, 1024, False, False), (300, 5000, 1025, True, True), (130, 1000, 20000, True, False),
                                         (1024, 4096, 16384, True, False)])
def test_long_contractions_are_added_up(cuda, m, n, k, ta, tb):
    """Whole numbers, whose sums f32 holds, with everything that may follow the sums."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)

    def whole(shape, dtype):
        return torch.randint(-4, 5, shape, generator=gen, device="cuda").to(dtype)

    for dtype in DT:
        a, b = whole((k, m) if ta else (m, k), _t(dtype)), whole((n, k) if tb else (k, n), _t(dtype))
        bias, res = whole((n,), torch.float32), whole((m, n), torch.float32)
        z = (a.double().t() if ta else a.double()) @ (b.double().t() if tb else b.double())
        assert torch.equal(cuda.matmul16(a, b, ta, tb, dtype=torch.float32).double(), z)
        y, pre = cuda.matmul16(a, b, ta, tb, bias=bias, residual=res, keep_pre=True, dtype=torch.float32)
        z += bias.double()
        assert torch.equal(pre.double(), z) and torch.equal(y.double(), z + res.double())


@pytest.mark.parametrize("m,n,k", [(512, 5000, 16384), (512, 5000, 65536), (512, 256, 65536)])
def test_long_sums_do_not_drift(cuda, m, n, k):
    """Sums of k positive products in f32 against float64.  An MMA adds 16 products to
    the sum and loses at most 2 units of its last place, 2^-22 of it; a chunk of 1024
    is 64 of them on a sum that grows evenly, 64 / 2 * 2^-22 = 2^-17 of the chunk, twice
    that for the unevenness; adding up k / 1024 chunks rounds by 2^-24 each."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(k)
    for dtype in DT:
        a = torch.randn((k, m), generator=gen, device="cuda").abs().to(_t(dtype))
        b = torch.randn((k, n), generator=gen, device="cuda").abs().to(_t(dtype))
        got = cuda.matmul16(a, b, trans_a=True, dtype=torch.float32)
        ref = a.double().t() @ b.double()
        assert float(((got.double() - ref).abs() / ref).max()) <= 2.0 ** -16 + k / 1024 * 2.0 ** -24


@pytest.mark.parametrize("m", [4, 64])
@pytest.mark.parametrize("dtype", DT)
def test_activations_of_far_negative_numbers(cuda, dtype, m):
    """Where e^-z and e^(-z^2/2) come to the ends of f32's range: silu keeps its
    digits down to -88.7, results of both widths as close as the bounds say."""
    import torch
    v = torch.tensor([-86.0, -87.3, -87.35, -87.4, -87.6, -88.0, -88.3, -88.5, -88.7, -89.0, -12.9, -13.1, -13.2, -13.3, -13.5, -14.4],
                     device="cuda")
    a = torch.zeros(m, 16, dtype=_t(dtype), device="cuda")
    b = torch.zeros(16, v.numel(), dtype=_t(dtype), device="cuda")
    z = v.double().cpu().numpy()
    for activation in ("silu", "gelu"):
        ref = S.act(z, activation)[0]
        bound = S.act_error(z, activation) + 2 * S.U * np.abs(ref)
        for out in ("f32", dtype):
            S.check(cuda.matmul16(a, b, bias=v, activation=activation, dtype=_t(out))[m - 1], ref, bound, out)


@pytest.mark.parametrize("count", [1, 37, 4096, 8 * 300 * 3, 5000000])
def test_activation_gradients_in_place(cuda, count):
    """dz may be dy, by the C entry."""
    import torch
    from chelis_b200 import lib as L
    for dtype, code in (("bf16", L.DTYPE_BF16), ("f16", L.DTYPE_F16)):
        gen = torch.Generator(device="cuda").manual_seed(count)
        dy, z = (torch.randn(count, generator=gen, device="cuda").to(_t(dtype)) for _ in range(2))
        for activation, act in (("gelu", L.ACT_GELU), ("silu", L.ACT_SILU), ("relu", L.ACT_RELU)):
            want, own = cuda.activation16_bwd(dy, z, activation), dy.clone()
            L.call("chelis_cuda_activation16_bwd", code, act, own.data_ptr(), z.data_ptr(), count, own.data_ptr())
            assert torch.equal(own, want)


@pytest.mark.parametrize("m,n,k,out", [(8, 64, 136, "f32"), (300, 264, 136, "f32"), (300, 263, 136, "f32"), (90, 264, 4160, None),
                                       (90, 263, 4160, "f32"), (300, 5000, 2200, "f32"), (300, 2604, 2200, "f32")])
def test_residual_may_be_the_result_in_f32_and_in_parts(cuda, m, n, k, out):
    import torch
    from chelis_b200 import lib as L
    rng = np.random.default_rng(m + n + k)
    for activation, act in ((None, L.ACT_NONE), ("silu", L.ACT_SILU)):
        a, _ = _make(rng, (m, k), "f16")
        b, _ = _make(rng, (k, n), "f16", 0.1)
        r, _ = _make(rng, (m, n), out or "f16")
        want = cuda.matmul16(a, b, activation=activation, residual=r, dtype=r.dtype)
        code = L.DTYPE_F32 if out else L.DTYPE_F16
        L.call("chelis_cuda_matmul16", L.DTYPE_F16, 0, 0, m, n, k, a.data_ptr(), b.data_ptr(), None, 0, act, r.data_ptr(), None,
               None, code, r.data_ptr())
        assert torch.equal(want, r)


@pytest.mark.parametrize("m,n,k,residual", [(512, 5000, 131072, False), (512, 5000, 131072, True), (300, 2600, 100001, True),
                                            (257, 5003, 40000, True)])
def test_long_sums_of_16_bits_do_not_drift(cuda, m, n, k, residual):
    """As above in chunks of 16384: 1024 MMAs on a sum that grows evenly, 1024 / 2 *
    2^-22 = 2^-13 of it, twice that for the unevenness, and half a step."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(k)
    for dtype in DT:
        a = torch.randn((k, m), generator=gen, device="cuda").abs().to(_t(dtype))
        b = (torch.randn((k, n), generator=gen, device="cuda").abs() * 0.25).to(_t(dtype))
        res = torch.randn((m, n), generator=gen, device="cuda").to(_t(dtype)) if residual else None
        got = cuda.matmul16(a, b, trans_a=True, residual=res)
        ref = a.double().t() @ b.double()
        bound = (2.0 ** -12 * ref).cpu().numpy()
        if residual:
            ref += res.double()
        S.check(got, ref.cpu().numpy(), bound, dtype)


@pytest.mark.parametrize("m,n,k", [(300, 5000, 17000), (300, 5003, 33000), (513, 2600, 16385)])
def test_long_contractions_of_16_bits_are_added_up(cuda, m, n, k):
    """Whole numbers with everything that may follow the sums; two numbers in a
    hundred are not 0, so that the results are whole in 16 bits nearly all."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(k)

    def whole(shape, dtype):
        x = torch.randint(-2, 3, shape, generator=gen, device="cuda")
        return (x * (torch.rand(shape, generator=gen, device="cuda") < 0.02)).to(_t(dtype))

    for dtype in DT:
        a, b, bias, res = whole((m, k), dtype), whole((k, n), dtype), whole((n,), dtype), whole((m, n), dtype)
        y, pre = cuda.matmul16(a, b, bias=bias, residual=res, keep_pre=True)
        z = a.double() @ b.double() + bias.double()
        assert torch.equal(pre, z.to(_t(dtype))) and torch.equal(y, (z + res.double()).to(_t(dtype)))

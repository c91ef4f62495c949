"""The norms around a block with its gate and residual scale, and their
gradients, against float64 (bounds: _sublayer_ref)."""
import numpy as np
import pytest

import _sublayer_ref as S

pytestmark = pytest.mark.gpu


def _t(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _rows(rng, shape, dtype, offset=0.0):
    import torch
    x = rng.standard_normal(shape) * np.exp(0.3 * rng.standard_normal(shape[:-1] + (1,))) + offset
    x = torch.from_numpy(x.astype(np.float32)).to(_t(dtype))
    return x.cuda(), x.double().numpy()


def _params(rng, hidden, kind, post, gate, pre, betas=True):
    """(keyword arguments on the device, the same in float64)."""
    import torch
    dev, ref = {}, {"scale": 0.5, "eps": 1e-5, "kind": kind}

    def put(name, v):
        v = v.astype(np.float32)
        dev[name] = torch.from_numpy(v).cuda()
        ref[name] = v.astype(np.float64)

    if post:
        put("post_gamma", 1 + 0.3 * rng.standard_normal(hidden))
        if betas:
            put("post_beta", 0.3 * rng.standard_normal(hidden))
    if gate:
        put("gate", 0.5 + 0.5 * rng.standard_normal(hidden if gate == 1 else (gate, hidden)))
    if pre:
        put("pre_gamma", 1 + 0.3 * rng.standard_normal(hidden))
        if betas:
            put("pre_beta", 0.3 * rng.standard_normal(hidden))
    dev.update(scale=0.5, eps=1e-5, kind=kind)
    return dev, ref


CASES = [  # rows, hidden, post, gate, pre: one row and many, ends inside packs, warps and teams, all widths of a team
    (1, 1, True, 1, True), (1, 8, True, 0, True), (3, 37, True, 1, True), (2, 64, False, 1, True), (5, 255, True, 0, False),
    (8, 256, True, 4, True), (4, 257, True, 1, True), (160, 264, True, 2, True), (7, 1000, False, 0, True),
    (300, 1000, True, 3, True), (6, 1024, True, 1, True), (400, 1024, True, 1, True), (4, 1031, True, 2, True),
    (200, 2048, True, 1, True), (3, 2056, False, 3, False), (170, 4096, True, 1, True), (2, 4097, True, 1, True),
    (160, 4104, True, 2, True), (3, 8192, True, 1, True), (151, 8192, True, 1, False), (2, 8191, True, 0, True),
    (1000, 72, True, 1000, True), (777, 16, True, 7, True)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,hidden,post,gate,pre", CASES)
def test_forward(cuda, rows, hidden, post, gate, pre, kind):
    rng = np.random.default_rng(rows * 5 + hidden)
    for dtype in ("f32", "bf16", "f16"):
        dev, ref = _params(rng, hidden, kind, post, gate, pre, betas=kind == "layer" or dtype == "f16")
        x, fx = _rows(rng, (rows, hidden), dtype)
        b, fb = _rows(rng, (rows, hidden), dtype, 0.5)
        y, h = cuda.residual_norm(x, b, **dev)
        ry, ey, rh, eh = S.join(fx, fb, ref)
        S.check(y, ry, ey, dtype)
        if pre:
            S.check(h, rh, eh, dtype)
        else:
            assert h is None


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,hidden,post,gate,pre", CASES)
def test_backward(cuda, rows, hidden, post, gate, pre, kind):
    rng = np.random.default_rng(rows * 7 + hidden)
    for i, dtype in enumerate(("f32", "bf16", "f16")):
        dev, ref = _params(rng, hidden, kind, post, gate, pre, betas=kind == "layer" or dtype == "f16")
        y, fy = _rows(rng, (rows, hidden), dtype)
        b, fb = _rows(rng, (rows, hidden), dtype, 0.5)
        dy, fdy = _rows(rng, (rows, hidden), dtype)
        dh, fdh = _rows(rng, (rows, hidden), dtype) if pre else (None, None)
        if pre and i == 0:
            dy, fdy = None, None  # nothing else reads y
        got = cuda.residual_norm_bwd(dy, dh, y, b, **dev)
        want = S.join_bwd(fdy, fdh, fy, fb, dict(ref, has_branch=True))
        for name, g in got._asdict().items():
            assert (g is None) == (name not in want), name
            if g is not None:
                S.check(g, *want[name], dtype if name in ("dx", "dbranch") else "f32")


@pytest.mark.parametrize("rows,hidden", [(1, 64), (9, 100), (500, 1024), (3, 5000)])
def test_second_norm_alone(cuda, rows, hidden):
    """branch None: the first norm of all, whose gradient joins the residual's."""
    rng = np.random.default_rng(rows + hidden)
    for dtype in ("f32", "bf16"):
        dev, ref = _params(rng, hidden, "layer", False, 0, True)
        dev["scale"] = ref["scale"] = 1.0
        x, fx = _rows(rng, (rows, hidden), dtype)
        same, h = cuda.residual_norm(x, None, **dev)
        assert same is x
        S.check(h, *S.join(fx, None, ref)[2:], dtype)
        dy, fdy = _rows(rng, (rows, hidden), dtype)
        dh, fdh = _rows(rng, (rows, hidden), dtype)
        got = cuda.residual_norm_bwd(dy, dh, x, None, **dev)
        want = S.join_bwd(fdy, fdh, fx, None, ref)
        assert got.dbranch is None and got.dgate is None and got.dpost_gamma is None
        for name in ("dx", "dpre_gamma", "dpre_beta"):
            S.check(getattr(got, name), *want[name], dtype if name == "dx" else "f32")


# rows, hidden, gate: one norm's gradients with more rows than there are teams of few values a thread; every width of
# a team, rows that end inside packs and teams, gates whose rows end inside a team's
MANY = [(2500, 264, 1), (1300, 512, 0), (1299, 504, 3), (700, 1000, 7), (640, 1024, 1), (330, 2048, 1), (322, 2056, 161),
        (170, 4096, 1), (163, 4104, 0), (100, 8192, 1), (102, 8184, 2)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,hidden,gate", MANY)
def test_one_norm_of_many_rows(cuda, rows, hidden, gate, kind):
    rng = np.random.default_rng(rows * 3 + hidden)
    for dtype in ("f32", "bf16", "f16"):
        y, fy = _rows(rng, (rows, hidden), dtype)
        b, fb = _rows(rng, (rows, hidden), dtype, 0.5)
        dy, fdy = _rows(rng, (rows, hidden), dtype)
        dh, fdh = _rows(rng, (rows, hidden), dtype)

        def compare(got, want):
            for name, g in got._asdict().items():
                assert (g is None) == (name not in want), name
                if g is not None:
                    S.check(g, *want[name], dtype if name in ("dx", "dbranch") else "f32")

        betas = kind == "layer"
        dev, ref = _params(rng, hidden, kind, False, 0, True, betas=betas)  # the second alone
        dev["scale"] = ref["scale"] = 1.0
        for d, fd in ((dy, fdy), (None, None)):
            want = S.join_bwd(fd, fdh, fy, None, ref)
            want.pop("dbranch", None)  # no branch
            compare(cuda.residual_norm_bwd(d, dh, y, None, **dev), want)
        dev, ref = _params(rng, hidden, kind, True, gate, False, betas=betas)  # the first alone
        compare(cuda.residual_norm_bwd(dy, None, y, b, **dev), S.join_bwd(fdy, None, fy, fb, dict(ref, has_branch=True)))
        if gate:  # a gate alone
            dev, ref = _params(rng, hidden, kind, False, gate, False)
            compare(cuda.residual_norm_bwd(dy, None, y, b, **dev), S.join_bwd(fdy, None, fy, fb, dict(ref, has_branch=True)))


@pytest.mark.parametrize("hidden", [40, 1024, 5000])
def test_mean_far_from_zero(cuda, hidden):
    """A mean of 1000 standard deviations costs the digits that the input's own
    rounding costs (its bound says so), not the variance."""
    rng = np.random.default_rng(hidden)
    dev, ref = _params(rng, hidden, "layer", True, 1, True)
    x, fx = _rows(rng, (5, hidden), "f32")
    b, fb = _rows(rng, (5, hidden), "f32", 1000.0)
    y, h = cuda.residual_norm(x, b, **dev)
    ry, ey, rh, eh = S.join(fx, fb, ref)
    S.check(y, ry, ey, "f32")
    S.check(h, rh, eh, "f32")
    # the normalised rows' variance is 1 within their bound's order
    n, _ = cuda.residual_norm(torch_zeros_like(x), b, post_gamma=torch_ones(hidden), scale=0.0)
    v = n.double().var(-1, unbiased=False).cpu().numpy()
    assert (np.abs(v - 1) < 1e-4).all()


def torch_zeros_like(x):
    import torch
    return torch.zeros_like(x)


def torch_ones(n):
    import torch
    return torch.ones(n, device="cuda")


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradients_against_differences(cuda, kind):
    """Directional derivatives of sum(dy y + dh h), central differences in
    float64, and the f32 gradients: within 2^-16 of the terms' magnitudes."""
    rng = np.random.default_rng(3)
    rows, hidden = 6, 48
    dev, ref = _params(rng, hidden, kind, True, 3, True)
    x, fx = _rows(rng, (rows, hidden), "f32")
    b, fb = _rows(rng, (rows, hidden), "f32", 0.3)
    dy, fdy = _rows(rng, (rows, hidden), "f32")
    dh, fdh = _rows(rng, (rows, hidden), "f32")
    y, _ = cuda.residual_norm(x, b, **dev)
    got = cuda.residual_norm_bwd(dy, dh, y, b, **dev)
    names = {"x": got.dx, "branch": got.dbranch, "post_gamma": got.dpost_gamma, "post_beta": got.dpost_beta,
             "gate": got.dgate, "pre_gamma": got.dpre_gamma, "pre_beta": got.dpre_beta}
    at = dict(ref, x=fx, branch=fb)

    def loss(v):
        y, _, h, _ = S.join(v["x"], v["branch"], v)
        return float((fdy * y + fdh * h).sum())

    for name, g in names.items():
        g = g.double().cpu().numpy()
        d = rng.standard_normal(g.shape)
        numeric = (loss(dict(at, **{name: at[name] + 1e-5 * d})) - loss(dict(at, **{name: at[name] - 1e-5 * d}))) / 2e-5
        assert abs(numeric - (g * d).sum()) <= 2.0 ** -16 * (np.abs(g * d).sum() + 10), name


def test_leading_axes_and_unaligned_rows(cuda):
    import torch
    rng = np.random.default_rng(4)
    x, fx = _rows(rng, (2, 3, 5, 72), "bf16")
    b, fb = _rows(rng, (2, 3, 5, 72), "bf16")
    dev, ref = _params(rng, 72, "layer", True, 6, True)
    y, h = cuda.residual_norm(x, b, **dev)
    assert y.shape == x.shape == h.shape
    y2, h2 = cuda.residual_norm(x.view(30, 72), b.view(30, 72), **dev)
    assert torch.equal(y.view(30, 72), y2) and torch.equal(h.view(30, 72), h2)
    # rows that start off 16 bytes
    flat = torch.zeros(30 * 72 + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.reshape(-1)
    y3, h3 = cuda.residual_norm(flat[1:].view(30, 72), b.view(30, 72), **dev)
    ry, ey, rh, eh = S.join(fx.reshape(30, 72), fb.reshape(30, 72), ref)
    S.check(y3, ry, ey, "bf16")
    S.check(h3, rh, eh, "bf16")


def test_special_rows(cuda):
    """An infinity or NaN of a row stays in that row; constant rows give beta."""
    import torch
    for hidden in (64, 100, 1024):
        x = torch.zeros(8, hidden, device="cuda")
        b = torch.randn(8, hidden, device="cuda")
        b[1, 3], b[2, 5], b[3] = float("inf"), float("nan"), 7.0
        ones, beta = torch.ones(hidden, device="cuda"), torch.full((hidden,), 0.25, device="cuda")
        y, h = cuda.residual_norm(x, b, post_gamma=ones, post_beta=beta, pre_gamma=ones)
        assert torch.isnan(y[2]).all() and torch.isnan(y[1]).any() and torch.isfinite(y[[0, 3, 4, 5, 6, 7]]).all()
        assert (y[3] == 0.25).all() and (h[3] == 0).all()
        g = cuda.residual_norm_bwd(x + 1, x + 1, y, b, post_gamma=ones, post_beta=beta, pre_gamma=ones)
        assert torch.isfinite(g.dx[[0, 3, 4, 5, 6, 7]]).all() and torch.isfinite(g.dbranch[[0, 3, 4, 5, 6, 7]]).all()


def test_empty_and_same_bits_twice(cuda):
    import torch
    dev, _ = _params(np.random.default_rng(1), 40, "layer", True, 1, True)
    e = torch.zeros(0, 40, device="cuda")
    y, h = cuda.residual_norm(e, e, **dev)
    assert y.shape == h.shape == (0, 40)
    g = cuda.residual_norm_bwd(e, e, e, e, **dev)
    assert g.dx.shape == (0, 40) and not g.dgate.any() and not g.dpost_gamma.any() and not g.dpre_beta.any()
    rng = np.random.default_rng(2)
    dev, _ = _params(rng, 1000, "layer", True, 5, True)
    t = [_rows(rng, (2000, 1000), "f16")[0] for _ in range(4)]
    first = cuda.residual_norm_bwd(*t, **dev)
    for _ in range(3):
        for a, b in zip(first, cuda.residual_norm_bwd(*t, **dev)):
            assert torch.equal(a, b)


def test_captured_on_two_streams(cuda):
    """Two graphs of the gradient (with scratch), replayed at once."""
    import torch
    rng = np.random.default_rng(9)
    dev, _ = _params(rng, 264, "rms", True, 4, True)
    runs = []
    for i in range(2):
        t = [_rows(rng, (800, 264), "bf16")[0] for _ in range(4)]
        want = cuda.residual_norm_bwd(*t, **dev)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = cuda.residual_norm_bwd(*t, **dev)
        runs.append((t, want, s, g, out))
    for _ in range(3):
        for _, _, s, g, _ in runs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, want, _, _, out in runs:
        for a, b in zip(want, out):
            assert (a is None and b is None) or torch.equal(a, b)
    cuda.device_status()


def test_offsets_past_32_bits(cuda):
    """Rows that begin past 2^31 numbers come out as they do alone."""
    import torch
    rows, hidden = (1 << 19) + 40, 4096
    rng = np.random.default_rng(5)
    dev, _ = _params(rng, hidden, "layer", True, 1, True)
    x, b = (torch.randn((rows, hidden), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    y, h = cuda.residual_norm(x, b, **dev)
    g = cuda.residual_norm_bwd(x, b, y, b, **dev)
    for at in (slice(0, 40), slice(rows - 40, rows)):
        part = [t[at].contiguous() for t in (x, b, y)]
        sy, sh = cuda.residual_norm(part[0], part[1], **dev)
        # a row's sums may be taken by another number of warps: a step of bf16 apart at most
        for got, want in ((y[at], sy), (h[at], sh)):
            assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-6).all()
        sg = cuda.residual_norm_bwd(part[0], part[1], part[2], part[1], **dev)
        for got, want in ((g.dx[at], sg.dx), (g.dbranch[at], sg.dbranch)):
            assert torch.equal(got, want)


def test_refusals(cuda):
    import torch
    x = torch.zeros(6, 40, device="cuda")
    g = torch.ones(40, device="cuda")
    for bad in (lambda: cuda.residual_norm(x, x.half()), lambda: cuda.residual_norm(x, x[:3]),
                lambda: cuda.residual_norm(x, x, kind="batch"), lambda: cuda.residual_norm(x, None),
                lambda: cuda.residual_norm(x, None, pre_gamma=g, scale=0.5), lambda: cuda.residual_norm(x, x, post_beta=g),
                lambda: cuda.residual_norm(x, x, gate=torch.ones(4, 40, device="cuda")),
                lambda: cuda.residual_norm(x, x, post_gamma=g.half()), lambda: cuda.residual_norm(x, x, pre_gamma=g[:8]),
                lambda: cuda.residual_norm(x.double(), x.double()), lambda: cuda.residual_norm(x[0], x[0]),
                lambda: cuda.residual_norm_bwd(x, x, x, x), lambda: cuda.residual_norm_bwd(None, None, x, x),
                lambda: cuda.residual_norm_bwd(x, None, x, x, pre_gamma=g),
                lambda: cuda.residual_norm_bwd(x, None, x, None, gate=g)):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros(1, 8200, device="cuda")
    with pytest.raises(Exception, match="8192"):
        cuda.residual_norm(wide, wide)


# values of at most 11 bits: f32 holds every sum of 8192 of them, so a row's mean is exact or its nearest f32
CONSTANT = {"f32": [7.5, 100.0, 1000.5, -30000.0], "bf16": [7.5, 100.0, 0.1015625], "f16": [7.5, 1000.5, 0.0999755859375]}


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("hidden", [1, 37, 40, 100, 264, 1000, 1024, 4104, 8192])
def test_constant_rows_give_beta(cuda, rows, hidden):
    """Whatever the constant: y is gate * beta and h beta, to the bit, and the
    gammas' gradients are 0; by parameters in shared memory, in registers and for
    each group's gate.  dbranch is r (w - mean w), a row's sum rounding by ROW."""
    import torch
    rng = np.random.default_rng(hidden)
    for dtype, values in CONSTANT.items():
        for i, c in enumerate(values):
            b = torch.full((rows, hidden), c, dtype=_t(dtype), device="cuda")
            assert float(b[0, 0]) == c
            ones = torch.ones(hidden, device="cuda")
            gate = torch.full((rows, hidden) if i % 2 else (hidden,), 1.5, device="cuda")
            p = dict(post_gamma=ones * 3, post_beta=ones * 0.25, gate=gate, pre_gamma=ones * 5)
            y, h = cuda.residual_norm(torch.zeros_like(b), b, pre_beta=ones * 0.125, **p)
            assert (y == 0.375).all() and (h == 0.125).all()
            _, h = cuda.residual_norm(b, None, pre_gamma=ones * 5, pre_beta=ones * 0.125)
            assert (h == 0.125).all()
            dy, fdy = _rows(rng, (rows, hidden), dtype)
            g = cuda.residual_norm_bwd(dy, dy, y, b, **p)
            assert not g.dpost_gamma.any() and not g.dpre_gamma.any()
            assert not cuda.residual_norm_bwd(dy, dy, b, None, pre_gamma=ones).dpre_gamma.any()
            g = cuda.residual_norm_bwd(dy, None, y, b, post_gamma=ones * 3, gate=gate)
            assert not g.dpost_gamma.any()
            w, r = fdy * 4.5, 1 / np.sqrt(1e-5)
            S.check(g.dbranch, r * (w - w.mean(-1, keepdims=True)),
                    2 * S.ROW * r * (np.abs(w) + np.abs(w).mean(-1, keepdims=True)), dtype)


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("hidden", [37, 40, 100, 1000, 1024, 4104, 8192])
def test_nearly_constant_rows(cuda, rows, hidden):
    """Rows of 1000.5 with a step of 0.5 here and there, whose sums f32 holds: the
    deviations are exact and the mean has twice f32's digits, so n is off by the
    root's ROW and eight roundings of its own, not by those of 1000.5 r."""
    import torch
    rng = np.random.default_rng(hidden + rows)
    fb = 1000.5 + 0.5 * rng.integers(0, 3, (rows, hidden)) * (rng.random((rows, hidden)) < 0.1)
    fb[:, 0] += 0.5
    b = torch.from_numpy(fb.astype(np.float32)).cuda()
    ones = torch.ones(hidden, device="cuda")
    n, r = S.stats(fb, "layer", 1e-5)
    en = (S.ROW + 8 * S.U) * np.abs(n)
    S.check(cuda.residual_norm(torch.zeros_like(b), b, post_gamma=ones)[0], n, en, "f32")
    S.check(cuda.residual_norm(b, None, pre_gamma=ones)[1], n, en, "f32")
    dy, fdy = _rows(rng, (rows, hidden), "f32")
    want, bound = S._through_norm(fdy, np.zeros_like(fdy), n, en, r, "layer")
    terms = np.abs(fdy) * en
    sums = (fdy * n).sum(0), terms.sum(0) + (rows + 64) * S.U * np.abs(fdy * n).sum(0)
    g = cuda.residual_norm_bwd(dy, None, b, b, post_gamma=ones)
    S.check(g.dbranch, want, bound, "f32")
    S.check(g.dpost_gamma, *sums, "f32")
    g = cuda.residual_norm_bwd(None, dy, b, None, pre_gamma=ones)
    S.check(g.dx, want, bound, "f32")
    S.check(g.dpre_gamma, *sums, "f32")


def test_two_threads_with_rows_of_different_lengths(cuda):
    """Calls of one kernel with different needs of shared memory, from two host
    threads that do little else, all launch and give their bits."""
    import threading

    import torch
    from chelis_b200 import lib as L
    lib = L.load()
    jobs = []
    for hidden in (1024, 264):
        rng = np.random.default_rng(hidden)
        x, b = (_rows(rng, (300, hidden), "bf16")[0] for _ in range(2))
        gamma = torch.ones(hidden, device="cuda")
        y, h, s = torch.empty_like(x), torch.empty_like(x), torch.cuda.Stream()
        args = cuda._residual_norm.pack(s.cuda_stream, L.DTYPE_BF16, L.NORM_LAYER, 300, hidden, x.data_ptr(), b.data_ptr(),
                                        gamma.data_ptr(), 0, 0, 1, 1.0, gamma.data_ptr(), 0, 1e-5, y.data_ptr(), h.data_ptr())
        jobs.append((args, s, y, h, cuda.residual_norm(x, b, post_gamma=gamma, pre_gamma=gamma), (x, b, gamma)))
    torch.cuda.synchronize()
    failed = []

    def work(args):
        for _ in range(30000):
            if lib.chelis_cuda_call_packed(L.PACKED_RESIDUAL_NORM, args):
                failed.append(L.last_error())
                return

    threads = [threading.Thread(target=work, args=(job[0],)) for job in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for _, _, y, h, want, _ in jobs:
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    cuda.device_status()


@pytest.mark.parametrize("betas", [False, True])
@pytest.mark.parametrize("hidden", [64, 100, 1024])
def test_infinite_gates(cuda, hidden, betas):
    """gate (n gamma + beta) with a gate of inf, -inf, NaN or one whose product with
    gamma leaves f32: the formula's infinities and NaN, and finite numbers elsewhere,
    by every way the parameters take."""
    import torch
    rng = np.random.default_rng(hidden)
    for kind in ("layer", "rms"):
        for post in (True, False):
            dev, ref = _params(rng, hidden, kind, post, 1, False, betas=betas and post)
            for p in (dev["gate"], ref["gate"]):
                p[3], p[5], p[7], p[9] = float("inf"), -float("inf"), float("nan"), 3e38
            if post:
                for p in (dev["post_gamma"], ref["post_gamma"]):
                    p[9] = 2.0 ** -20
                    p[11] = 3e38
                for p in (dev["gate"], ref["gate"]):
                    p[11] = 2.0 ** 20  # gate gamma leaves f32, (n gamma) gate does so too for |n| > 2^-20
            for rows in (9, 300):
                x, fx = _rows(rng, (rows, hidden), "f32")
                b, fb = _rows(rng, (rows, hidden), "f32")
                y, _ = cuda.residual_norm(x, b, **dev)
                with np.errstate(invalid="ignore", over="ignore"):
                    want, bound, _, _ = S.join(fx, fb, ref)
                    want[np.abs(want) > 3.5e38] *= np.inf
                y = y.double().cpu().numpy()
                assert (np.isnan(y) == np.isnan(want)).all()
                sure = ~np.isnan(want) & ~((np.abs(want) > 3.3e38) & np.isfinite(want))
                with np.errstate(invalid="ignore"):
                    same = (y == want) | (np.isfinite(want) & (np.abs(y - want) <= bound))
                assert same[sure].all()

"""The norm of all gradients and their clipping against float64.

The norm: a few squares at a time in f32 (at most 8 roundings, positive terms:
8 u of the sum), the rest in f64, a root and a rounding: 8 u / 2 + 2 u < 8 u.
A clipped number: the factor's rounding on that, the product's: 10 u, and half an
ulp of its type."""
import math

import numpy as np
import pytest

import _experts_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _t(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _make(sizes, dtypes, scale=1.0, seed=0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=gen, device="cuda") * scale).to(_t(d)) for n, d in zip(sizes, dtypes)]


def _norm(ts):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in ts))


def _name(t):
    import torch
    return {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[t.dtype]


def _check(got, src, factor):
    ref = src.double().cpu().numpy() * factor
    assert not R.outside(got.double().cpu().numpy(), ref, 10 * U * np.abs(ref), _name(got)).any()


LISTS = [[1], [0], [7, 0, 33], [32768], [32769, 1, 65536], [5] * 31, [5] * 33, [3] * 800, [100000, 3, 99999, 250001],
         list(range(1, 1700, 2)), [3000001]]


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "bf16"), ("mixed", "f16")])
def test_norm_and_clip(cuda, sizes, dtype, out):
    import torch
    kinds = [["f32", "bf16", "f16"][i % 3] if dtype == "mixed" else dtype for i in range(len(sizes))]
    g = _make(sizes, kinds, 0.5)
    ref = _norm(g)
    norm = cuda.grad_norm(g)
    assert abs(float(norm) - ref) <= 8 * U * ref
    for bound in (ref / 3 + 1e-3, ref * 2 + 1):
        factor = bound / ref if ref > bound else 1.0
        dst = [torch.full((n,), 9.0, dtype=_t(out), device="cuda") for n in sizes]
        assert torch.equal(cuda.clip_grads(g, bound, out=dst), norm)
        for a, b in zip(dst, g):
            _check(a, b, factor)
        own = [t.clone() for t in g]
        assert torch.equal(cuda.clip_grads(own, bound), norm)
        for a, b in zip(own, g):
            if factor == 1.0:
                assert torch.equal(a, b)
            else:
                _check(a, b, factor)


def test_empty_list(cuda):
    assert float(cuda.grad_norm([])) == 0 and float(cuda.clip_grads([], 1.0)) == 0


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e25, 3e37])
def test_squares_outside_f32(cuda, scale):
    import torch
    g = _make([1000, 70001], ["f32", "f32"], scale)
    g[0][3] = 0.0
    ref = _norm(g)
    if ref > 3.41e38:  # of 3e37: 8e39, which f32 does not hold; then nothing is changed either
        own = [t.clone() for t in g]
        assert float(cuda.clip_grads(own, 1.0)) == float("inf") and all(torch.equal(a, b) for a, b in zip(own, g))
    else:
        assert abs(float(cuda.grad_norm(g)) - ref) <= 8 * U * ref
    # one large number among many that vanish beside it, and denormal ones alone
    t = torch.full((5000,), 1e-25, device="cuda")
    t[4321] = 1e30
    assert float(cuda.grad_norm([t])) == float(np.float32(1e30))
    tiny = torch.full((64,), 1e-40, device="cuda")
    ref = math.sqrt(64) * float(tiny[0].double())
    assert abs(float(cuda.grad_norm([tiny])) - ref) <= 2.0 ** -149


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_norm_that_is_not_finite_changes_nothing(cuda, bad):
    import torch
    for dtype in ("f32", "f16"):
        g = _make([100, 5001], [dtype] * 2)
        g[1][77] = bad
        own = [t.clone() for t in g]
        norm = cuda.clip_grads(own, 0.1)
        assert not torch.isfinite(norm)
        for a, b in zip(own, g):
            assert torch.equal(a.nan_to_num(5.0, 6.0, 7.0), b.nan_to_num(5.0, 6.0, 7.0))


def test_unaligned_tensors_and_their_neighbours(cuda):
    import torch
    for dtype in ("f32", "bf16"):
        for out in ("f32", "bf16"):
            buf = _make([70000], [dtype])[0]
            pieces = [buf[1:2], buf[3:20], buf[21:33000], buf[33003:69999]]
            dst_buf = torch.full((70010,), 9.0, dtype=_t(out), device="cuda")
            dst = [dst_buf[2:3], dst_buf[5:22], dst_buf[24:33003], dst_buf[33010:70006]]
            ref = _norm(pieces)
            norm = cuda.clip_grads(pieces, ref / 2, out=dst)
            assert abs(float(norm) - ref) <= 8 * U * ref
            for a, b in zip(dst, pieces):
                _check(a, b, 0.5)
            rest = torch.ones(70010, dtype=torch.bool)
            for lo, hi in ((2, 3), (5, 22), (24, 33003), (33010, 70006)):
                rest[lo:hi] = False
            assert (dst_buf[rest.cuda()] == 9).all()
            keep = buf.clone()
            cuda.clip_grads(pieces, ref / 2)
            for lo, hi in ((0, 1), (2, 3), (20, 21), (33000, 33003), (69999, 70000)):
                assert torch.equal(buf[lo:hi], keep[lo:hi])


def test_flat_gradients_and_matrices(cuda):
    """The views of one flat buffer, as a data-parallel step has them."""
    import torch
    from chelis_b200 import dp
    flat = dp.FlatGrads({"w": (33, 70), "b": (70,), "g": (5,)}, "cuda")
    flat.flat.normal_()
    views = [flat[n] for n in ("w", "b", "g")]
    ref = _norm(views)
    src = [v.clone() for v in views]
    cuda.clip_grads(views, 1.0)
    for a, b in zip(views, src):
        _check(a.reshape(-1), b.reshape(-1), 1.0 / ref)


def test_same_bits_captured_and_on_two_streams(cuda):
    import torch
    runs = []
    for i in range(2):
        g = _make([100000, 7, 300001], ["f32", "bf16", "f16"], seed=i)
        out = [torch.empty_like(t) for t in g]
        want = [torch.empty_like(t) for t in g]
        norm = cuda.clip_grads(g, 3.0, out=want)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                n = cuda.clip_grads(g, 3.0, out=out)
        runs.append((s, graph, out, want, norm, n, g))  # a graph keeps no tensors alive
    for _ in range(3):
        for s, graph, *_ in runs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, want, norm, n, _ in runs:
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_offsets_past_32_bits(cuda):
    import torch
    n = (1 << 31) + 12345
    big = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    big[-5:] = 3.0
    small = torch.ones(7, device="cuda")
    ref = math.sqrt(0.25 * (n - 5) + 45 + 7)
    norm = cuda.clip_grads([small, big], ref / 2)
    assert abs(float(norm) - ref) <= 8 * U * ref
    assert (big[-5:] == 1.5).all() and (big[-100:-5] == 0.25).all() and (big[:100] == 0.25).all() and (small == 0.5).all()
    assert bool((big[(1 << 31) - 100:(1 << 31) + 100] == 0.25).all())


def test_refusals(cuda):
    import torch
    from chelis_b200 import lib as L
    a = torch.ones(100, device="cuda")
    for bad in (lambda: cuda.grad_norm([a.double()]), lambda: cuda.grad_norm([a.view(10, 10).t()]), lambda: cuda.grad_norm([a.cpu()]),
                lambda: cuda.clip_grads([a], 1.0, out=[a[:5].clone()]), lambda: cuda.clip_grads([a], 1.0, out=[])):
        with pytest.raises(ValueError):
            bad()
    b = torch.ones(100, device="cuda")
    for bad in (lambda: cuda.clip_grads([a, a], 1.0), lambda: cuda.clip_grads([a, a[50:]], 1.0),
                lambda: cuda.clip_grads([a, b], 1.0, out=[b, a]), lambda: cuda.clip_grads([a[:50]], 1.0, out=[a[10:60]]),
                lambda: cuda.clip_grads([a[:50]], 1.0, out=[a.view(torch.bfloat16)[:50]]),
                lambda: cuda.clip_grads([a], -1.0), lambda: cuda.clip_grads([a], float("nan"))):
        with pytest.raises(L.ChelisCudaError):
            bad()
    assert (a == 1).all() and (b == 1).all()


@pytest.mark.parametrize("sizes", [[1], [7, 0, 33], [1000, 24000, 1], [2000] * 32, [65536]])
def test_few_numbers_in_place_are_those_out_of_place(cuda, sizes):
    """One block reads the numbers for the norm and scales them in the same launch."""
    import torch
    for dtype in ("f32", "bf16", "f16"):
        g = _make(sizes, [dtype] * len(sizes))
        out = [torch.empty_like(t) for t in g]
        norm = cuda.clip_grads(g, 0.25, out=out)
        assert torch.equal(cuda.clip_grads(g, 0.25), norm) and all(torch.equal(a, b) for a, b in zip(g, out))


@pytest.mark.parametrize("sizes", [[1000, 33], [1000, 70001, 5]])
@pytest.mark.parametrize("scale,bound", [(1e25, 1.0), (1e25, 1e-3), (1e35, 1e-3), (1e35, 1e-8), (1e35, 1e-30), (1e35, 1e-44), (1e35, 0.0),
                                         (1.0, 1e-36), (1e-3, 1e-42)])
def test_clipping_by_a_factor_outside_f32(cuda, sizes, scale, bound):
    """A factor below 2^-126 keeps its digits: numbers of a finite norm come out
    as the formula says, with half a step of what they are where they vanish."""
    import torch
    bound = float(np.float32(bound))
    for out in ("f32", "bf16"):
        g = _make(sizes, ["f32", "bf16" if scale > 1e3 else "f32", "f32"][:len(sizes)], scale)
        ref = _norm(g)
        assert bound < ref < 3e38
        dst = [torch.full_like(t, 9.0, dtype=_t(out)) for t in g]
        norm = cuda.clip_grads(g, bound, out=dst)
        assert abs(float(norm) - ref) <= 8 * U * ref
        for a, b in zip(dst, g):
            _check(a, b, bound / ref)
        own = [t.clone() for t in g]
        cuda.clip_grads(own, bound)
        for a, b in zip(own, g):
            _check(a, b, bound / ref)

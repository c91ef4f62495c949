"""The router, the sort by expert, the rows there and back, and the routed
feed-forward layer, against plain float64 evaluations.

Bounds, with u = 2^-24 (an f32 rounding is at most u relative):
  router weights    the differences l - max (|.| <= 32: 32 u in the
                    exponent), exp within 4 u, a sum of at most 1024 positive
                    terms in 37 additions, the division: numerator and sum
                    together below 2 (32 + 4) u + 37 u + u = 110 u
  router gradient   p (g - inner): 110 u twice and 40 more roundings of terms
                    no larger than |g| + sum p |g|: 300 u of p (|g| + sum p|g|)
  sums of rows      k terms in order: k u of the sum of magnitudes
  dot products      hidden u of the sum of magnitudes, in any order
and half an ulp of the result's type (_experts_ref.half_ulp).
"""
import numpy as np
import pytest

import _experts_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _np(t):
    return t.double().cpu().numpy()


def _within(got, ref, bound, dtype="f32"):
    assert not R.outside(_np(got), ref, bound, dtype).any()


def _logits(rng, t, e, dtype):
    import torch
    x = torch.from_numpy(np.clip(rng.standard_normal((t, e)) * 3, -15, 15)).to(_dtype(dtype))
    return x.cuda(), x.double().numpy()


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("t,e,k,dtype", [(1, 1, 1, "f32"), (3, 7, 2, "f32"), (65, 32, 8, "bf16"),
                                         (33, 64, 8, "f32"), (17, 100, 3, "f16"), (9, 256, 32, "f32"),
                                         (5, 1000, 4, "bf16"), (1, 1024, 1, "f32")])
def test_route(cuda, t, e, k, dtype, renormalize):
    import torch
    rng = np.random.default_rng(t * e + k)
    x, l = _logits(rng, t, e, dtype)
    w, ids = cuda.expert_route(x, k, renormalize)
    ref_w, ref_ids = R.route(l, k, renormalize)
    assert (ids.cpu().numpy() == ref_ids).all()
    _within(w, ref_w, 110 * U * ref_w)
    g = torch.from_numpy(rng.standard_normal((t, k)).astype(np.float32))
    dl = cuda.expert_route_bwd(x, ids, g.cuda(), renormalize)
    p = np.zeros((t, e))
    if renormalize:
        np.put_along_axis(p, ref_ids, ref_w, 1)
    else:
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    gd = np.zeros((t, e))
    np.put_along_axis(gd, ref_ids, g.double().numpy(), 1)
    inner = (p * gd).sum(1, keepdims=True)
    bound = 300 * U * p * (np.abs(gd) + (p * np.abs(gd)).sum(1, keepdims=True))
    _within(dl, p * (gd - inner), bound, dtype)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient_is_the_difference(cuda, renormalize):
    """Central differences of f32 weights: with step h the third derivative
    leaves at most h^2 max|g| and the weights' rounding 110 u max|g| / h."""
    import torch
    rng = np.random.default_rng(5)
    t, e, k, h = 4, 12, 3, 2.0 ** -6
    x, _ = _logits(rng, t, e, "f32")
    g = torch.from_numpy(rng.standard_normal((t, k)).astype(np.float32)).cuda()
    _, ids = cuda.expert_route(x, k, renormalize)
    dl = _np(cuda.expert_route_bwd(x, ids, g, renormalize))
    top = float(g.abs().max())
    for i in range(e):
        v = []
        for s in (h, -h):
            y = x.clone()
            y[:, i] += s
            w, got = cuda.expert_route(y, k, renormalize)
            same = (got == ids).all(1)  # the choice does not change within the step
            v.append((_np(w * g).sum(1), same.cpu().numpy()))
        ok = v[0][1] & v[1][1]
        diff = (v[0][0] - v[1][0]) / (2 * h)
        assert (np.abs(diff - dl[:, i])[ok] <= (h * h + 110 * U / h) * top * k).all()


def test_route_special_rows(cuda):
    import torch
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[-inf, -inf, -inf, -inf],   # nothing to choose
                      [1.0, -inf, 3.0, -inf],     # fewer than k
                      [2.0, 2.0, 2.0, 2.0],       # ties
                      [0.0, -0.0, -0.0, 0.0],     # zeros of both signs tie
                      [low, low, low, -inf],      # the lowest finite value is a value
                      [1.0, nan, 2.0, 0.0],
                      [inf, 0.0, 1.0, 2.0]], device="cuda")
    for renormalize in (True, False):
        w, ids = cuda.expert_route(x, 3, renormalize)
        assert ids.cpu().tolist() == [[-1, -1, -1], [2, 0, -1], [0, 1, 2], [0, 1, 2], [0, 1, 2],
                                      [2, 0, 3], [0, 3, 2]]
        w = w.cpu()
        assert w[0].tolist() == [0.0] * 3 and w[1, 2] == 0.0
        assert abs(w[1, :2].sum().item() - 1.0) <= 110 * U
        third = 1 / 3 if renormalize else 1 / 4
        assert (w[2:4] - third).abs().max() <= 110 * U
        assert (w[4] - 1 / 3).abs().max() <= 110 * U
        assert w[5].isnan().all() and w[6, 0].isnan()
        dl = cuda.expert_route_bwd(x, ids, torch.ones_like(w).cuda(), renormalize).cpu()
        assert dl[0].tolist() == [0.0] * 4 and dl[1, 1] == 0.0 and dl[1, 3] == 0.0
        assert dl[5].isnan().all()
        assert not dl[:5].isnan().any()


def _ids(rng, t, k, experts, dropped=0.1):
    ids = np.stack([rng.permutation(experts)[:k] for _ in range(t)]) if t else np.zeros((0, k))
    ids[rng.random(ids.shape) < dropped] = -1
    return ids.astype(np.int32)


@pytest.mark.parametrize("t,k,experts", [(0, 2, 4), (1, 1, 1), (1, 1, 1024), (8, 2, 8), (100, 3, 5),
                                         (257, 8, 64), (1024, 2, 9), (1025, 2, 1000), (5000, 4, 4),
                                         (3000, 8, 300)])
def test_sort(cuda, t, k, experts):
    import torch
    rng = np.random.default_rng(t + k + experts)
    ids = _ids(rng, t, k, experts)
    order = cuda.expert_sort(torch.from_numpy(ids).cuda(), experts)
    for got, ref in zip(order, R.sort(ids, experts) if experts <= 64 else _fast_sort(ids, experts)):
        assert got.cpu().numpy().tolist() == ref.tolist()
    cuda.device_status()


# counts of segments that are added up in their own pass: just from there on, shares of one
# segment and of many, experts that a block of the pass is too wide for
@pytest.mark.parametrize("t,k,experts", [(8 * 1024, 1, 1024), (4099, 2, 1021), (8 * 1024 + 1, 8, 127), (300007, 3, 13),
                                         (131072, 8, 64), (1 << 20, 2, 4), (1 << 20, 8, 1)])
def test_sort_of_many_segments(cuda, t, k, experts):
    import torch
    rng = np.random.default_rng(t + experts)
    ids = rng.integers(-1, experts, size=(t, k), dtype=np.int32)
    order = cuda.expert_sort(torch.from_numpy(ids).cuda(), experts)
    for got, ref in zip(order, _fast_sort(ids, experts)):
        assert np.array_equal(got.cpu().numpy(), ref)
    cuda.device_status()


def _fast_sort(ids, experts):
    flat = ids.reshape(-1).astype(np.int64)
    key = np.where(flat < 0, experts, flat)
    order = np.argsort(key, kind="stable")
    n = int((flat >= 0).sum())
    source = np.where(np.arange(flat.size) < n, order, -1)
    position = np.full(flat.size, -1)
    position[order[:n]] = np.arange(n)
    return np.searchsorted(key[order], np.arange(experts + 1)), position.reshape(ids.shape), source


def test_sort_extremes_and_bad_ids(cuda):
    import torch
    one = torch.full((3000, 2), 6, dtype=torch.int32, device="cuda")
    order = cuda.expert_sort(one, 8)
    assert order.offsets.tolist() == [0] * 7 + [6000, 6000]
    assert order.source.tolist() == list(range(6000))
    none = torch.full((5, 2), -1, dtype=torch.int32, device="cuda")
    order = cuda.expert_sort(none, 3)
    assert order.offsets.tolist() == [0] * 4 and order.source.tolist() == [-1] * 10
    from chelis_b200 import lib as L
    for bad in (3, -2):
        ids = torch.tensor([[0, bad], [2, 1]], dtype=torch.int32, device="cuda")
        order = cuda.expert_sort(ids, 3)
        torch.cuda.synchronize()
        assert order.position.tolist() == [[0, -1], [2, 1]]
        with pytest.raises(L.ChelisCudaError):
            cuda.device_status()
        cuda.device_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,k,experts,hidden", [(1, 1, 1, 1), (1, 2, 3, 8), (8, 2, 8, 1024), (37, 3, 5, 100),
                                                (50, 8, 16, 257), (300, 2, 4, 72), (3, 2, 2, 5000)])
def test_rows_there_and_back(cuda, t, k, experts, hidden, dtype):
    import torch
    rng = np.random.default_rng(t * hidden + k)
    ids = _ids(rng, t, k, experts)
    _, position, source = R.sort(ids, experts)
    order = cuda.expert_sort(torch.from_numpy(ids).cuda(), experts)
    dt = _dtype(dtype)

    def make(rows):
        v = torch.from_numpy(rng.standard_normal((rows, hidden))).to(dt)
        return v.cuda(), v.double().numpy()

    x, xr = make(t)
    xs = cuda.expert_gather(x, order)
    assert (_np(xs) == R.spread(xr, source, k)).all()
    ys, yr = make(t * k)
    ones = np.ones((t, k))
    mag = R.combine(np.abs(yr), ones, position)
    _within(cuda.expert_gather_bwd(ys, order), R.combine(yr, ones, position), k * U * mag, dtype)
    w = torch.from_numpy(rng.random((t, k)).astype(np.float32)).cuda()
    wr = _np(w)
    mag = R.combine(np.abs(yr), wr, position)
    _within(cuda.expert_combine(ys, w, order), R.combine(yr, wr, position), k * U * mag, dtype)
    dy, dr = make(t)
    dys, dw = cuda.expert_combine_bwd(dy, ys, w, order)
    ref = R.spread(dr, source, k, wr)
    _within(dys, ref, U * np.abs(ref), dtype)
    dots = np.zeros((t, k))
    mags = np.zeros((t, k))
    for i in range(t):
        for j in range(k):
            if position[i, j] >= 0:
                dots[i, j] = dr[i] @ yr[position[i, j]]
                mags[i, j] = np.abs(dr[i]) @ np.abs(yr[position[i, j]])
    _within(dw, dots, hidden * U * mags)
    again = cuda.expert_combine_bwd(dy, ys, w, order)
    assert torch.equal(again[0], dys) and torch.equal(again[1], dw)


def test_rows_at_odd_addresses_and_on_another_stream(cuda):
    """A base that 16 bytes do not divide, and work queued on a side stream."""
    import torch
    rng = np.random.default_rng(0)
    ids = torch.from_numpy(_ids(rng, 40, 2, 4)).cuda()
    base = torch.randn(40 * 64 + 1, device="cuda").to(torch.bfloat16)
    x = base[1:].view(40, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        order = cuda.expert_sort(ids, 4)
        xs = cuda.expert_gather(x, order)
        dx = cuda.expert_gather_bwd(xs, order)
    torch.cuda.current_stream().wait_stream(side)
    _, position, source = R.sort(ids.cpu().numpy(), 4)
    assert (_np(xs) == R.spread(_np(x), source, 2)).all()
    kept = (position >= 0).sum(1)[:, None]
    assert (_np(dx) == _np(x) * kept).all()  # 0, 1 or 2 copies: exact


def test_refusals(cuda):
    import torch
    from chelis_b200 import lib as L
    x = torch.zeros((4, 8), device="cuda")
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    order = cuda.expert_sort(ids, 3)
    with pytest.raises(L.ChelisCudaError, match="DOMAIN"):
        cuda.expert_route(x, 9)
    with pytest.raises(L.ChelisCudaError, match="DOMAIN"):
        cuda.expert_route(x, 0)
    with pytest.raises(L.ChelisCudaError, match="UNSUPPORTED"):
        cuda.expert_route(torch.zeros((2, 1025), device="cuda"), 2)
    with pytest.raises(L.ChelisCudaError, match="UNSUPPORTED"):
        cuda.expert_route(torch.zeros((2, 64), device="cuda"), 33)
    with pytest.raises(ValueError):
        cuda.expert_route(x.double(), 2)
    with pytest.raises(ValueError):
        cuda.expert_route(x.t(), 2)
    with pytest.raises(ValueError):
        cuda.expert_sort(ids.long(), 3)
    with pytest.raises(L.ChelisCudaError, match="DOMAIN"):
        cuda.expert_sort(ids, 0)
    with pytest.raises(ValueError):
        cuda.expert_gather(x[:3], order)
    with pytest.raises(ValueError):
        cuda.expert_gather(x.to(torch.int32), order)
    with pytest.raises(ValueError):
        cuda.expert_combine(x, torch.zeros((4, 2), device="cuda"), order)
    ys = torch.zeros((8, 8), device="cuda")
    with pytest.raises(ValueError):
        cuda.expert_combine(ys, torch.zeros((4, 2), device="cuda").double(), order)
    with pytest.raises(ValueError):
        cuda.expert_combine_bwd(x.bfloat16(), ys, torch.zeros((4, 2), device="cuda"), order)


@pytest.mark.parametrize("tokens,d,ff,experts,k,renormalize", [(96, 128, 256, 4, 2, True),
                                                               (131, 72, 200, 5, 3, False)])
def test_feed_forward_against_float64(cuda, tokens, d, ff, experts, k, renormalize):
    """The whole layer and its gradients against float64 autograd of the layer
    without 8 bits: normwise (Frobenius) within 2^-3, the rounding of e5m2, of
    which errors of single numbers average to less; the router's part, which
    no 8-bit product precedes in the forward pass, chooses the same experts."""
    import torch
    from chelis_b200 import experts as X
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, d), generator=gen)
    router = torch.randn((d, experts), generator=gen) / d ** 0.5 * 2
    w1 = torch.randn((experts, ff, d), generator=gen) / d ** 0.5
    w2 = torch.randn((experts, d, ff), generator=gen) / ff ** 0.5
    dy = torch.randn((tokens, d), generator=gen)
    q1, q2 = (cuda.quantize8(w.cuda(), "e4m3", "tiles") for w in (w1, w2))
    y, saved = X.feed_forward(x.cuda(), router.cuda(), q1, q2, k, renormalize)
    grads = X.feed_forward_bwd(dy.cuda(), saved, router.cuda(), q1, q2, renormalize)
    torch.cuda.synchronize()
    cuda.device_status()
    p = [t.double().requires_grad_() for t in (x, router, w1, w2)]
    logits = p[0] @ p[1]
    ids = torch.argsort(-logits, dim=1, stable=True)[:, :k]
    assert (saved.experts.cpu() == ids).all()
    soft = torch.softmax(logits, 1).gather(1, ids)
    w = soft / soft.sum(1, keepdim=True) if renormalize else soft
    ref = torch.zeros((tokens, d), dtype=torch.float64)
    for j in range(k):
        h = torch.einsum("td,tfd->tf", p[0], p[2][ids[:, j]])
        ref = ref + w[:, j:j + 1] * torch.einsum("tf,tdf->td", torch.nn.functional.gelu(h), p[3][ids[:, j]])
    ref.backward(dy.double())
    pairs = [(y, ref.detach())] + [(grads[n], t.grad) for n, t in zip(("dx", "drouter", "dw1", "dw2"), p)]
    for got, want in pairs:
        assert (got.cpu().double() - want).norm() <= 2.0 ** -3 * want.norm()

"""The operators together: a dense feed-forward sublayer's training step in 16
bits, the routed layer's with the balance loss, their gradients clipped."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _reference(x, p, dy):
    """(y, gradients) of dense.feed_forward in float64 by autograd."""
    import torch
    leaves = {n: (None if getattr(p, n) is None else getattr(p, n).double().requires_grad_(True))
              for n in ("pre_gamma", "pre_beta", "w1", "b1", "w2", "b2", "post_gamma", "post_beta", "gate")}
    xx = x.double().requires_grad_(True)

    def norm(v, g, b):
        if p.kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / (v.square().mean(-1, keepdim=True) + p.eps).sqrt() * g
        return v if b is None else v + b

    h = norm(xx, leaves["pre_gamma"], leaves["pre_beta"])
    z = h @ leaves["w1"]
    if p.b1 is not None:
        z = z + leaves["b1"]
    a = {"gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z), "relu": lambda: z.clamp(min=0)}[p.activation]()
    f = a @ leaves["w2"]
    if p.b2 is not None:
        f = f + leaves["b2"]
    u = f if p.post_gamma is None else norm(f, leaves["post_gamma"], leaves["post_beta"])
    if p.gate is not None:
        g = leaves["gate"]
        u = u * (g if g.dim() == 1 else g.repeat_interleave(x.shape[0] // g.shape[0], 0))
    y = p.scale * xx + u
    y.backward(dy.double())
    grads = {n: v.grad for n, v in leaves.items() if v is not None}
    grads["dx"] = xx.grad
    return y.detach(), grads


def _sublayer(gen, d, ff, dt, full, kind, activation, gate):
    import torch
    from chelis_b200 import dense

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    layer = kind == "layer"
    return dense.Sublayer(
        pre_gamma=1 + 0.2 * randn(d), w1=(randn(d, ff) / math.sqrt(d)).to(dt), w2=(randn(ff, d) / math.sqrt(ff)).to(dt),
        pre_beta=0.2 * randn(d) if layer else None, b1=0.1 * randn(ff) if full else None, b2=(0.1 * randn(d)).to(dt) if full else None,
        post_gamma=1 + 0.2 * randn(d) if full else None, post_beta=0.1 * randn(d) if full and layer else None,
        gate=0.5 + 0.3 * randn(*gate) if gate else None, activation=activation, kind=kind, scale=0.75)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,d,ff,full,kind,activation,gate", [
    (8, 64, 256, True, "layer", "gelu", (64,)), (300, 72, 200, True, "rms", "silu", (3, 72)), (515, 128, 512, False, "layer", "relu", None),
    (2048, 256, 1024, True, "layer", "gelu", (8, 256)), (1, 40, 24, False, "rms", "gelu", None), (130, 33, 65, True, "layer", "silu", (33,))])
def test_dense_training_step(cuda, tokens, d, ff, full, kind, activation, gate, dtype):
    """Frobenius distances from float64.  h, a, f and y, dbranch, dz, dh and dx are
    each rounded to 16 bits, half a step e (2^-9, 2^-12) of each number at most,
    and each passes at most three factors of order one: 3 * 8 e, and four times
    that for what a norm's gradient takes away from it."""
    import torch
    from chelis_b200 import dense
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    e = torch.finfo(dt).eps / 2
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    p = _sublayer(gen, d, ff, dt, full, kind, activation, gate)
    x = torch.randn((tokens, d), generator=gen, device="cuda").to(dt)
    dy = torch.randn((tokens, d), generator=gen, device="cuda").to(dt)
    y, saved = dense.feed_forward(x, p)
    grads = dense.feed_forward_bwd(dy, saved, p)
    ry, want = _reference(x, p, dy)
    assert grads.keys() == want.keys()

    def near(a, b, limit):
        assert a.shape == b.shape and float((a.double() - b).norm()) <= limit * float(b.norm())

    near(y, ry, 24 * e)
    for name in want:
        near(grads[name], want[name], 96 * e)
    # the step's end: all gradients to one norm, f32 and 16 bits together
    whole = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    before = {n: g.clone() for n, g in grads.items()}
    norm = cuda.clip_grads(grads.values(), whole / 2)
    assert abs(float(norm) - whole) <= 1e-6 * whole
    for name, g in grads.items():
        near(g, before[name].double() / 2, e if g.dtype == dt else 1e-6)
    cuda.device_status()


def test_dense_step_captured(cuda):
    """The whole step with clipping in a graph, replayed on new inputs."""
    import torch
    from chelis_b200 import dense
    gen = torch.Generator(device="cuda").manual_seed(3)
    p = _sublayer(gen, 128, 264, torch.bfloat16, True, "layer", "gelu", (128,))
    x = torch.randn((600, 128), generator=gen, device="cuda").bfloat16()
    dy = torch.randn((600, 128), generator=gen, device="cuda").bfloat16()

    def step():
        y, s = dense.feed_forward(x, p)
        g = dense.feed_forward_bwd(dy, s, p)
        return y, list(g.values()), cuda.clip_grads(list(g.values()), 1.0)

    step()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y, grads, norm = step()
    for seed in range(3):
        x.copy_(torch.randn((600, 128), generator=gen, device="cuda"))
        dy.copy_(torch.randn((600, 128), generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        wy, wgrads, wnorm = step()
        assert torch.equal(y, wy) and torch.equal(norm, wnorm)
        for a, b in zip(grads, wgrads):
            assert torch.equal(a, b)


@pytest.mark.parametrize("masked", [False, True])
def test_routed_layer_with_the_balance_loss(cuda, masked):
    """Saved has the loss and the counts; the gradients of y are what they are
    without it, and the router's gets the loss's on top."""
    import torch
    from chelis_b200 import experts as X
    gen = torch.Generator(device="cuda").manual_seed(7)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    x, router, dy = randn(40, 64), randn(64, 6), randn(40, 64)
    w1, w2 = (cuda.quantize8(w, "e4m3", "tiles") for w in (randn(6, 96, 64), randn(6, 64, 96)))
    mask = torch.arange(40, device="cuda") < 31 if masked else None
    y0, s0 = X.feed_forward(x, router, w1, w2, 3)
    y1, s1 = X.feed_forward(x, router, w1, w2, 3, balance=0.25, mask=mask)
    assert torch.equal(y0, y1) and s0.loss is None
    loss, counts = cuda.expert_balance(s1.logits, s1.experts, mask)
    assert torch.equal(loss, s1.loss) and torch.equal(counts, s1.counts) and int(counts[-1]) == (31 if masked else 40)
    g0, g1 = X.feed_forward_bwd(dy, s0, router, w1, w2), X.feed_forward_bwd(dy, s1, router, w1, w2)
    assert torch.equal(g0["dw1"], g1["dw1"]) and torch.equal(g0["dw2"], g1["dw2"])
    # the loss's own gradient in float64
    l = (x.double() @ router.double()).requires_grad_(True)
    live = mask if masked else torch.ones(40, dtype=torch.bool, device="cuda")
    n = int(live.sum())
    p = torch.softmax(l[live], -1).sum(0)
    (0.25 * 6 / (3 * n * n) * (counts[:6].double() * p).sum()).backward()
    for name, extra in (("drouter", x.double().t() @ l.grad), ("dx", l.grad @ router.double().t())):
        diff = g1[name].double() - g0[name].double()
        # f32 sums of numbers as large as the gradients themselves
        assert float((diff - extra).abs().max()) <= 2e-6 * float(g0[name].abs().max()) + 1e-5 * float(extra.abs().max())
    norm = cuda.clip_grads([g1["dx"], g1["drouter"], g1["dw1"], g1["dw2"]], 1.0)
    assert float(norm) > 1 and abs(float(cuda.grad_norm([g1[n] for n in ("dx", "drouter", "dw1", "dw2")])) - 1) < 1e-5


def test_the_profiled_step_clips_the_parameters_alone(cuda, monkeypatch):
    """dx belongs to what comes before: neither in the norm nor scaled."""
    from chelis_b200 import profile_cases
    shapes, clip = [], cuda.clip_grads

    def recorded(grads, *args, **kw):
        grads = list(grads)
        shapes.extend(tuple(g.shape) for g in grads)
        return clip(grads, *args, **kw)

    monkeypatch.setattr(cuda, "clip_grads", recorded)
    profile_cases.run("sublayer")
    assert sorted(shapes) == sorted([(1024, 4096), (4096, 1024), (4096,)] + [(1024,)] * 6)

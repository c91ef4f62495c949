"""What is measured of the operators of a 16-bit training or serving step
around a feed-forward block: the matrix product with bias, activation and
residual in its epilogue, the norms before and after a block with its gate and
residual scale, the router's balance loss, the norm of all gradients and their
clipping.

`run` makes one pass through one operator on what `prepare` made: the plain
form (elementary torch operations in 32 bits) or, with `own` set, the calls of
chelis_b200.ops.  `exact` is the operator's definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
ACTIVATIONS = ["none", "relu", "gelu", "silu"]


# ------------------------------------------------------------------- cases

def listed():
    return [
        # serving: the first product of the feed-forward for eight sequences, one token each
        dict(name="linear_decode", op="linear", direction="forward", rows=8, n=4096, k=1024,
             trans_b=False, dtype="bf16", activation="gelu", bias=True, residual=False, keep_pre=False),
        # an odd batch through odd widths: rows that no 16 bytes divide
        dict(name="linear_ragged", op="linear", direction="forward", rows=1237, n=1000, k=999,
             trans_b=True, dtype="f16", activation="silu", bias=True, residual=True, keep_pre=False),
        # training: the first product over a batch of 8 x 2048 tokens, what gelu took kept
        dict(name="linear_up_train", op="linear", direction="forward", rows=16384, n=4096, k=1024,
             trans_b=False, dtype="bf16", activation="gelu", bias=True, residual=False, keep_pre=True),
        # training: the second product, added to the residual stream
        dict(name="linear_down_train", op="linear", direction="forward", rows=16384, n=1024, k=4096,
             trans_b=False, dtype="bf16", activation="none", bias=True, residual=True, keep_pre=False),
        # training: the second product's gradients, its input's on through gelu
        dict(name="linear_down_bwd", op="linear", direction="backward", rows=16384, n=1024, k=4096,
             trans_b=False, dtype="bf16", activation="gelu", bias=True, residual=False, keep_pre=False),
        # serving: what stands between two blocks, eight tokens
        dict(name="norm_decode", op="norm", direction="forward", rows=8, hidden=1024, dtype="bf16",
             kind="rms", post=True, gate=1, scale=1.0, pre=True),
        # training: the norm after a block, its gate, the residual and the next block's norm
        dict(name="norm_train", op="norm", direction="forward", rows=16384, hidden=1024, dtype="bf16",
             kind="layer", post=True, gate=1, scale=0.5, pre=True),
        # training in f32 on wide rows, a gate for each of eight samples: all gradients
        dict(name="norm_train_bwd", op="norm", direction="backward", rows=16384, hidden=4096,
             dtype="f32", kind="layer", post=True, gate=8, scale=0.5, pre=True),
        # a small step's router: 64 tokens, a quarter of them padding
        dict(name="balance_padded", op="balance", tokens=64, experts=8, k=2, dtype="f32",
             padding=0.25, backward=True),
        # a training step's router, with the gradient added to the router's own
        dict(name="balance_train", op="balance", tokens=16384, experts=64, k=8, dtype="f32",
             padding=0.0, backward=True),
        # a small model's gradients, where the launches are what counts
        dict(name="clip_small", op="clip", tensors=12, elements=20000, dtype="f32", out="f32", clip=True),
        # the gradients of a stack of blocks, 16 bits from the products, to f32 for the optimizer
        dict(name="clip_layers", op="clip", tensors=240, elements=100000000, dtype="bf16", out="f32",
             clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "balance", "clip"])
    if op == "linear":
        rows, n, k = _log(rng, 1, 16384), _log(rng, 16, 4096), _log(rng, 16, 4096)
        while rows * n * k > 16384 * 4096 * 1024:
            rows = max(1, rows // 2)
        forward = rng.random() < 0.7
        return dict(op=op, direction="forward" if forward else "backward", rows=rows, n=n, k=k,
                    trans_b=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16"]),
                    activation=rng.choice(ACTIVATIONS), bias=rng.random() < 0.7,
                    residual=forward and rng.random() < 0.4, keep_pre=forward and rng.random() < 0.4)
    if op == "norm":
        rows, hidden = _log(rng, 1, 16384), _log(rng, 16, 8192)
        while rows * hidden > 16384 * 4096:
            rows //= 2
        post, pre = rng.choice([(True, True), (True, False), (False, True)])
        gate = rng.choice([0, 1, 1, 4])
        if gate > 1:
            rows = max(1, rows // gate) * gate
        return dict(op=op, direction=rng.choice(["forward", "backward"]), rows=rows, hidden=hidden,
                    dtype=rng.choice(list(DTYPES)), kind=rng.choice(["layer", "rms"]), post=post,
                    gate=gate, scale=rng.choice([1.0, 0.5]), pre=pre)
    if op == "balance":
        experts = _log(rng, 2, 256)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=experts,
                    k=rng.randint(1, min(8, experts)), dtype=rng.choice(list(DTYPES)),
                    padding=rng.choice([0.0, 0.2]), backward=rng.random() < 0.7)
    dtype = rng.choice(list(DTYPES))
    elements = _log(rng, 1000, 100000000)
    return dict(op=op, tensors=_log(rng, 1, 400), elements=elements, dtype=dtype,
                out=rng.choice([dtype, "f32"]), clip=rng.random() < 0.7)


# ------------------------------------------------------------------ prepare

def _activations(gen, rows, cols, dtype):
    """Normal values with a scale for each row and a few large channels."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x *= torch.exp(torch.randn((rows, 1), generator=gen, device="cuda") * 0.3)
    x *= 1.0 + 3.0 * (torch.rand((1, cols), generator=gen, device="cuda") < 0.01).float()
    return x.to(dtype)


def _sizes(case):
    """The tensors' sizes: some large, some small, all of them case["elements"] about."""
    rng = random.Random(case["tensors"])
    share = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    total = sum(share)
    return [max(1, int(case["elements"] * v / total)) for v in share]


def _starts(case):
    """Where each tensor begins in the flat buffer, and the buffer's length."""
    starts = [0]
    for s in _sizes(case):
        starts.append(starts[-1] + (s + 63) // 64 * 64)
    return starts


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "linear":
        rows, n, k, dt = case["rows"], case["n"], case["k"], DTYPES[case["dtype"]]
        st["a"] = _activations(gen, rows, k, dt)
        w = normal(n, k) if case["trans_b"] else normal(k, n)
        st["b"] = (w / math.sqrt(k)).to(dt)
        if case["direction"] == "forward":
            st["bias_v"] = (normal(n) * 0.1).to(dt) if case["bias"] else None
            st["residual_v"] = _activations(gen, rows, n, dt) if case["residual"] else None
        else:
            st["dy"] = (normal(rows, n) * 0.1).to(dt)
            # what the activation before this product took: a is its value there
            st["through"] = _activations(gen, rows, k, dt) if case["activation"] != "none" else None
        return st
    if case["op"] == "norm":
        rows, hidden, dt = case["rows"], case["hidden"], DTYPES[case["dtype"]]
        beta = case["kind"] == "layer"
        st["x"] = _activations(gen, rows, hidden, dt)
        st["branch"] = _activations(gen, rows, hidden, dt)
        for name in ("post", "pre"):
            st[name + "_gamma"] = 1.0 + 0.2 * normal(hidden) if case[name] else None
            st[name + "_beta"] = 0.2 * normal(hidden) if case[name] and beta else None
        g = case["gate"]
        st["gate_v"] = (0.5 + 0.3 * (normal(hidden) if g == 1 else normal(g, hidden))) if g else None
        if case["direction"] == "backward":
            # y: the residual stream after this block, as the forward pass left it
            st["y"] = st.pop("x")
            st["dy"] = normal(rows, hidden).to(dt)
            st["dh"] = normal(rows, hidden).to(dt) if case["pre"] else None
        return st
    if case["op"] == "balance":
        t, e, k = case["tokens"], case["experts"], case["k"]
        popular = normal(1, e)
        st["logits"] = (normal(t, e) * 2 + popular).to(DTYPES[case["dtype"]])
        st["ids"] = st["logits"].float().topk(k, -1).indices.to(torch.int32).contiguous()
        st["mask"] = None
        if case["padding"]:
            st["mask"] = torch.rand((t,), generator=gen, device="cuda") >= case["padding"]
        # the gradient of a mean over the tokens; f16 training scales its loss
        scale = 0.01 * (t if case["dtype"] == "f16" else 1)
        st["router"] = (normal(t, e) * (scale / t)).to(DTYPES[case["dtype"]])
        st["dloss"] = torch.tensor(scale, device="cuda")
        return st
    dt, out = DTYPES[case["dtype"]], DTYPES[case["out"]]
    st["grads"] = [(normal(s) * 3e-3).to(dt) for s in _sizes(case)]
    if case["clip"]:
        # one flat buffer that the optimizer reads, each tensor from a multiple of 64 on
        starts = _starts(case)
        st["flat"] = torch.zeros(starts[-1], dtype=out, device="cuda")
        st["clipped"] = [st["flat"][at:at + g.numel()] for at, g in zip(starts, st["grads"])]
    st["max_norm"] = 0.25 if seed % 4 else 1e6   # one seed of four has nothing to clip
    return st


# -------------------------------------------------------------- plain forms

def _phi(z):
    """The normal distribution function."""
    return 0.5 * torch.erfc(z * -math.sqrt(0.5))


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return z * _phi(z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return _phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _run_linear(st):
    dt = DTYPES[st["dtype"]]
    a, b = st["a"].float(), st["b"].float()
    if st["direction"] == "forward":
        z = a @ (b.t() if st["trans_b"] else b)
        if st["bias_v"] is not None:
            z = z + st["bias_v"].float()
        y = _act(z, st["activation"])
        if st["residual_v"] is not None:
            y = y + st["residual_v"].float()
        out = {"y": y.to(dt)}
        if st["keep_pre"]:
            out["pre"] = z.to(dt)
        return out
    dy = st["dy"].float()
    da = dy @ (b if st["trans_b"] else b.t())
    if st["through"] is not None:
        da = da * _act_slope(st["through"].float(), st["activation"])
    db = dy.t() @ a if st["trans_b"] else a.t() @ dy
    out = {"da": da.to(dt), "db": db.to(dt)}
    if st["bias"]:
        out["dbias"] = dy.sum(0)
    return out


def _normalised(x, kind):
    """(x normalised along its rows, the reciprocal of what it was divided by)."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _affine(n, gamma, beta):
    n = n * gamma
    return n if beta is None else n + beta


def _gate_rows(gate, rows):
    """A gate [hidden] or [groups, hidden] for every row."""
    return gate if gate.dim() == 1 else gate.repeat_interleave(rows // gate.shape[0], 0)


def _norm_slope(g, n, r, kind):
    """The gradient through a norm, from that of its normalised rows n."""
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * r


def _run_norm(st):
    dt, kind, rows = DTYPES[st["dtype"]], st["kind"], st["rows"]
    branch = st["branch"].float()
    gate = None if st["gate_v"] is None else _gate_rows(st["gate_v"], rows)
    if st["post"]:
        n1, r1 = _normalised(branch, kind)
        u = _affine(n1, st["post_gamma"], st["post_beta"])
    else:
        u = branch
    if st["direction"] == "forward":
        y = st["scale"] * st["x"].float() + (u if gate is None else gate * u)
        out = {"y": y.to(dt)}
        if st["pre"]:
            out["h"] = _affine(_normalised(y, kind)[0], st["pre_gamma"], st["pre_beta"]).to(dt)
        return out
    dt_row = st["dy"].float()
    out = {}
    if st["pre"]:
        n2, r2 = _normalised(st["y"].float(), kind)
        dh = st["dh"].float()
        out["dpre_gamma"] = (dh * n2).sum(0)
        if kind == "layer":
            out["dpre_beta"] = dh.sum(0)
        dt_row = dt_row + _norm_slope(dh * st["pre_gamma"], n2, r2, kind)
    out["dx"] = (st["scale"] * dt_row).to(dt)
    du = dt_row if gate is None else dt_row * gate
    if gate is not None:
        dgate = dt_row * u
        if st["gate_v"].dim() == 1:
            out["dgate"] = dgate.sum(0)
        else:
            out["dgate"] = dgate.view(st["gate"], -1, st["hidden"]).sum(1)
    if st["post"]:
        out["dpost_gamma"] = (du * n1).sum(0)
        if kind == "layer":
            out["dpost_beta"] = du.sum(0)
        du = _norm_slope(du * st["post_gamma"], n1, r1, kind)
    out["dbranch"] = du.to(dt)
    return out


def _run_balance(st):
    t, e, k = st["tokens"], st["experts"], st["k"]
    l = st["logits"].float()
    p = torch.exp(l - l.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    live = torch.ones((t,), dtype=torch.bool, device=l.device) if st["mask"] is None else st["mask"]
    counts = torch.zeros((e + 1,), dtype=torch.int32, device=l.device)
    ids = torch.where(live[:, None], st["ids"].long(), torch.full_like(st["ids"], e).long()).reshape(-1)
    counts.scatter_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    counts[e] = live.sum().to(torch.int32)
    n = counts[e].float().clamp(min=1.0)
    c = counts[:e].float()
    per = e / (k * n * n)
    loss = per * (c * (p * live[:, None]).sum(0)).sum()
    out = {"loss": loss, "counts": counts}
    if st["backward"]:
        d = st["dloss"] * per * p * (c - (p * c).sum(-1, keepdim=True))
        out["dlogits"] = (st["router"].float() + d * live[:, None]).to(DTYPES[st["dtype"]])
    return out


def _run_clip(st):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in st["grads"]:
        f = g.float()
        total = total + (f * f).sum(dtype=torch.float64)
    norm = torch.sqrt(total)
    out = {"norm": norm.float()}
    if st["clip"]:
        c = torch.where(norm > st["max_norm"], st["max_norm"] / norm, torch.ones_like(norm)).float()
        for dst, g in zip(st["clipped"], st["grads"]):
            dst.copy_(g.float() * c)
        out["grads"] = st["flat"]
    return out


# ---------------------------------------------------------------------- run

def run(st):
    if own:
        return _run_own(st)
    return {"linear": _run_linear, "norm": _run_norm, "balance": _run_balance, "clip": _run_clip}[st["op"]](st)


def _run_own(st):
    from chelis_b200 import ops
    if st["op"] == "linear":
        act = None if st["activation"] == "none" else st["activation"]
        if st["direction"] == "forward":
            out = ops.matmul16(st["a"], st["b"], trans_b=st["trans_b"], bias=st["bias_v"], activation=act,
                               residual=st["residual_v"], keep_pre=st["keep_pre"])
            return {"y": out[0], "pre": out[1]} if st["keep_pre"] else {"y": out}
        through = None if act is None else (st["through"], act)
        da, db, dbias = ops.matmul16_bwd(st["dy"], st["a"], st["b"], trans_b=st["trans_b"], through=through,
                                         want_bias=st["bias"], weight_dtype=st["b"].dtype)
        out = {"da": da, "db": db}
        if st["bias"]:
            out["dbias"] = dbias
        return out
    if st["op"] == "norm":
        params = dict(post_gamma=st["post_gamma"], post_beta=st["post_beta"], gate=st["gate_v"],
                      scale=st["scale"], pre_gamma=st["pre_gamma"], pre_beta=st["pre_beta"], eps=EPS,
                      kind=st["kind"])
        if st["direction"] == "forward":
            y, h = ops.residual_norm(st["x"], st["branch"], **params)
            return {"y": y, "h": h} if st["pre"] else {"y": y}
        grads = ops.residual_norm_bwd(st["dy"], st["dh"], st["y"], st["branch"], **params)
        return {name: g for name, g in grads._asdict().items() if g is not None}
    if st["op"] == "balance":
        loss, counts = ops.expert_balance(st["logits"], st["ids"], mask=st["mask"])
        out = {"loss": loss, "counts": counts}
        if st["backward"]:
            out["dlogits"] = ops.expert_balance_bwd(st["logits"], counts, st["k"], dloss=st["dloss"],
                                                    mask=st["mask"], add=st["router"])
        return out
    if not st["clip"]:
        return {"norm": ops.grad_norm(st["grads"])}
    return {"norm": ops.clip_grads(st["grads"], st["max_norm"], out=st["clipped"]), "grads": st["flat"]}


# -------------------------------------------------------------------- exact

def _exact_linear(st):
    a, b = st["a"].double(), st["b"].double()
    if st["trans_b"]:
        b = b.t()

    def value(z):
        if st["activation"] == "none":
            return z
        if st["activation"] == "relu":
            return z.clamp(min=0)
        if st["activation"] == "silu":
            return z * torch.sigmoid(z)
        return z * torch.special.ndtr(z)

    if st["direction"] == "forward":
        z = torch.mm(a, b)
        if st["bias_v"] is not None:
            z += st["bias_v"].double()
        y = value(z)
        if st["residual_v"] is not None:
            y = y + st["residual_v"].double()
        return {"y": y, "pre": z} if st["keep_pre"] else {"y": y}
    dy = st["dy"].double()
    da = torch.mm(dy, b.t())
    if st["through"] is not None:
        z = st["through"].double().requires_grad_(True)
        value(z).backward(da)
        da = z.grad
    db = torch.mm(a.t(), dy)
    out = {"da": da, "db": db.t() if st["trans_b"] else db}
    if st["bias"]:
        out["dbias"] = dy.sum(0)
    return out


def _exact_join(x, branch, st, p):
    """(y, h) of the definition; p: the parameters in 64 bits."""
    def norm(v, name):
        if st["kind"] == "layer":
            var, mean = torch.var_mean(v, -1, unbiased=False, keepdim=True)
            v = (v - mean) / torch.sqrt(var + EPS)
        else:
            v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
        v = v * p[name + "_gamma"]
        return v + p[name + "_beta"] if p[name + "_beta"] is not None else v

    u = norm(branch, "post") if st["post"] else branch
    if p["gate"] is not None:
        g = p["gate"] if p["gate"].dim() == 1 else \
            p["gate"][:, None].expand(-1, st["rows"] // st["gate"], -1).reshape(u.shape)
        u = u * g
    y = u if x is None else st["scale"] * x + u
    return y, (norm(y, "pre") if st["pre"] else None), norm


def _exact_norm(st):
    def wide(v):
        return None if v is None else v.double().requires_grad_(st["direction"] == "backward")

    p = {name: wide(st[name]) for name in ("post_gamma", "post_beta", "pre_gamma", "pre_beta")}
    p["gate"] = wide(st["gate_v"])
    branch = wide(st["branch"])
    if st["direction"] == "forward":
        y, h, _ = _exact_join(st["x"].double(), branch, st, p)
        return {"y": y, "h": h} if st["pre"] else {"y": y}
    # the second norm at the given y, then the rest with what reaches y
    u, _, norm = _exact_join(None, branch, dict(st, pre=False), p)
    dy = st["dy"].double()
    if st["pre"]:
        y = st["y"].double().requires_grad_(True)
        norm(y, "pre").backward(st["dh"].double())
        dy = dy + y.grad
    if u.requires_grad:
        u.backward(dy)
    out = {"dx": st["scale"] * dy, "dbranch": branch.grad}
    for name, key in (("dpost_gamma", "post_gamma"), ("dpost_beta", "post_beta"), ("dgate", "gate"),
                      ("dpre_gamma", "pre_gamma"), ("dpre_beta", "pre_beta")):
        if p[key] is not None:
            out[name] = p[key].grad
    return out


def _exact_balance(st):
    l = st["logits"].double()
    t, e = l.shape
    keep = torch.arange(t, device=l.device) if st["mask"] is None else torch.nonzero(st["mask"]).reshape(-1)
    n = max(1, keep.numel())
    c = torch.bincount(st["ids"][keep].reshape(-1).long(), minlength=e).double()
    l.requires_grad_(True)
    p = torch.softmax(l[keep], -1)
    loss = e * torch.dot(c / (st["k"] * n), p.sum(0) / n)
    out = {"loss": loss.detach(), "counts": None}
    if st["backward"]:
        loss.backward()
        out["dlogits"] = st["router"].double() + st["dloss"].double() * l.grad
    return out


def _exact_clip(st):
    norm = math.sqrt(math.fsum(g.double().square().sum().item() for g in st["grads"]))
    out = {"norm": norm}
    if st["clip"]:
        c = st["max_norm"] / norm if norm > st["max_norm"] else 1.0
        out["grads"] = torch.zeros(st["flat"].shape, dtype=torch.float64, device="cuda")
        for at, g in zip(_starts(st), st["grads"]):
            out["grads"][at:at + g.numel()] = g.double() * c
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "balance": _exact_balance,
            "clip": _exact_clip}[case["op"]](st)


# --------------------------------------------------------------------- work

def work(case):
    op, w = case["op"], WIDTH[case["dtype"]]
    if op == "linear":
        r, n, k = case["rows"], case["n"], case["k"]
        if case["direction"] == "forward":
            wide = 1 + case["residual"] + case["keep_pre"]
            return {"bytes": w * (r * k + n * k + wide * r * n + case["bias"] * n), "flops": 2 * r * n * k}
        through = case["activation"] != "none"
        return {"bytes": w * (r * n + (2 + through) * r * k + 2 * n * k) + 4 * case["bias"] * n,
                "flops": 4 * r * n * k}
    if op == "norm":
        n, h = case["rows"] * case["hidden"], case["hidden"]
        params = 4 * h * ((case["post"] + case["pre"]) * (2 if case["kind"] == "layer" else 1) + case["gate"])
        if case["direction"] == "forward":
            return {"bytes": w * n * (3 + case["pre"]) + params, "flops": 14 * n}
        # dy, branch, dx, dbranch, and with the second norm y and dh; a branch that
        # is neither normed nor gated is not needed for its gradient
        reads = 1 + (case["post"] or case["gate"] > 0) + 2 * case["pre"]
        return {"bytes": w * n * (reads + 2) + 2 * params, "flops": 30 * n}
    if op == "balance":
        t, e, k = case["tokens"], case["experts"], case["k"]
        b, f = t * e * w + t * k * 4, 5 * t * e
        if case["backward"]:
            b, f = b + 2 * t * e * w, f + 5 * t * e
        return {"bytes": b, "flops": f}
    n = sum(_sizes(case))
    b = n * w
    if case["clip"]:
        b += n * WIDTH[case["out"]]
    return {"bytes": b, "flops": (3 if case["clip"] else 2) * n}

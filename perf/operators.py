"""What is measured of the routed feed-forward operators: the router, the sort
of tokens by expert, the weighted way back, the 8-bit block format and the
8-bit products.

`run` makes one pass through one operator on what `prepare` made: the plain
form (elementary torch operations in 32 bits) or, with `own` set, the calls of
chelis_b200.ops.  `exact` is the operator's definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 128
# largest finite value of each 8-bit format
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
FLOAT8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # the router of a serving step of eight sequences: one token each
        dict(name="route_8_tokens", op="route", tokens=8, experts=64, k=8, dtype="f32",
             renormalize=True, backward=False),
        # the router of a training step: a batch of 8 x 2048 tokens, with its gradient
        dict(name="route_train", op="route", tokens=16384, experts=64, k=8, dtype="f32",
             renormalize=False, backward=True),
        # serving: eight tokens to their two experts' rows, where the launches are what counts
        dict(name="gather_8_tokens", op="gather", tokens=8, experts=8, k=2, hidden=1024,
             dtype="bf16", dropped=0.0, backward=False),
        # training in f32 as the transformer block runs it: rows to 8 experts, and the gradient back
        dict(name="gather_train_f32", op="gather", tokens=16384, experts=8, k=2, hidden=1024,
             dtype="f32", dropped=0.0, backward=True),
        # an odd batch with rows that found no place at their expert
        dict(name="combine_ragged", op="combine", tokens=1237, experts=13, k=3, hidden=1000,
             dtype="f16", dropped=0.1, backward=True),
        # training with many small experts: the way back and both its gradients
        dict(name="combine_train", op="combine", tokens=16384, experts=64, k=8, hidden=1024,
             dtype="bf16", dropped=0.0, backward=True),
        # hidden activations of the feed-forward to 8 bits, a scale for each 128 of a row
        dict(name="quantize_rows", op="quantize", blocks="rows", rows=16384, cols=4096,
             experts=1, dtype="bf16", format="e4m3"),
        # gradients for the weight gradient: 128 rows of one expert a block, ragged experts, odd width
        dict(name="quantize_transposed_experts", op="quantize", blocks="transposed", rows=4099,
             cols=1000, experts=13, dtype="f32", format="e5m2"),
        # serving: 16 rows among 8 experts, bound by reading the experts' weights
        dict(name="matmul_decode_experts", op="matmul", form="forward", rows=16, n=4096, k=1024,
             experts=8, format_a="e4m3", format_b="e4m3", dtype="bf16"),
        # the first product of the feed-forward over a whole training batch, one matrix
        dict(name="matmul_dense", op="matmul", form="forward", rows=16384, n=4096, k=1024,
             experts=1, format_a="e4m3", format_b="e4m3", dtype="bf16"),
        # the input gradient of the experts' first product: the same weights, read the other way
        dict(name="matmul_dinput_experts", op="matmul", form="dinput", rows=32768, n=1024, k=4096,
             experts=8, format_a="e5m2", format_b="e4m3", dtype="bf16"),
        # the weight gradient of the experts' first product, in f32 for the optimizer
        dict(name="matmul_dweight_experts", op="matmul", form="dweight", rows=32768, n=4096,
             k=1024, experts=8, format_a="e5m2", format_b="e4m3", dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["route", "gather", "combine", "quantize", "matmul", "matmul", "matmul"])
    if op == "route":
        experts = _log(rng, 2, 256)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=experts,
                    k=rng.randint(1, min(8, experts)), dtype=rng.choice(list(DTYPES)),
                    renormalize=rng.random() < 0.5, backward=rng.random() < 0.5)
    if op in ("gather", "combine"):
        experts = _log(rng, 2, 128)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=experts,
                    k=rng.randint(1, min(8, experts)), hidden=_log(rng, 64, 2048),
                    dtype=rng.choice(list(DTYPES)), dropped=rng.choice([0.0, 0.1]),
                    backward=rng.random() < 0.5)
    if op == "quantize":
        blocks = rng.choice(["rows", "tiles", "transposed"])
        return dict(op=op, blocks=blocks, rows=_log(rng, 1, 16384), cols=_log(rng, 16, 4096),
                    experts=_log(rng, 1, 32), dtype=rng.choice(list(DTYPES)),
                    format=rng.choice(list(FLOAT8)))
    form = rng.choice(["forward", "forward", "dinput", "dweight"])
    rows, n, k = _log(rng, 1, 32768), _log(rng, 64, 4096), _log(rng, 64, 4096)
    while rows * n * k > 32768 * 4096 * 1024:
        rows = max(1, rows // 2)
    return dict(op="matmul", form=form, rows=rows, n=n, k=k, experts=_log(rng, 1, 32),
                format_a=rng.choice(list(FLOAT8)), format_b=rng.choice(list(FLOAT8)),
                dtype="f32" if form == "dweight" else rng.choice(list(DTYPES)))


# --------------------------------------------------- the 8-bit block format

def _ceil(a, b):
    return -(-a // b)


def _scale(amax, fmt):
    """The least power of two s with amax / s <= the format's largest value
    (2^-126 at the least, 1 for a block of zeros)."""
    top_f, top_e = math.frexp(LARGEST[fmt])
    f, e = torch.frexp(amax)
    e = (e - top_e + (f > top_f).to(e.dtype)).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(amax), e)
    return torch.where(amax == 0, torch.ones_like(s), s)


def _padded(x, rows, cols):
    out = torch.zeros((*x.shape[:-2], rows, cols), dtype=x.dtype, device=x.device)
    out[..., :x.shape[-2], :x.shape[-1]] = x
    return out


def _quantize_rows(x, fmt):
    """x[rows, cols] -> data [rows, cols rounded up to 16], scales [blocks, rows]."""
    rows, cols = x.shape
    kb = _ceil(cols, BLOCK)
    b = _padded(x.float(), rows, kb * BLOCK).view(rows, kb, BLOCK)
    s = _scale(b.abs().amax(-1), fmt)
    q = (b / s[..., None]).to(FLOAT8[fmt]).view(rows, kb * BLOCK)
    return q[:, :_ceil(cols, 16) * 16].contiguous(), s.t().contiguous()


def _quantize_tiles(w, fmt):
    """w[e, rows, cols] -> data [e, rows, cols rounded up to 16], scales [e, rows/128, cols/128]."""
    e, rows, cols = w.shape
    rb, kb = _ceil(rows, BLOCK), _ceil(cols, BLOCK)
    b = _padded(w.float(), rb * BLOCK, kb * BLOCK).view(e, rb, BLOCK, kb, BLOCK)
    s = _scale(b.abs().amax((2, 4)), fmt)
    q = (b / s[:, :, None, :, None]).to(FLOAT8[fmt]).view(e, rb * BLOCK, kb * BLOCK)
    return q[:, :rows, :_ceil(cols, 16) * 16].contiguous(), s.contiguous()


def _padded_rows(counts, rows, device):
    """For the transposed form: the row in each padded place (rows = none).
    Every expert's rows start on a block of 128; rows // 128 + experts blocks
    (of one expert no more than its rows take)."""
    blocks = rows // BLOCK + len(counts) if len(counts) > 1 else _ceil(rows, BLOCK)
    total = blocks * BLOCK
    place = torch.full((total,), rows, dtype=torch.int64, device=device)
    row, at = 0, 0
    for c in counts:
        place[at:at + c] = torch.arange(row, row + c, device=device)
        row += c
        at += _ceil(c, BLOCK) * BLOCK
    return place


def _quantize_transposed(x, fmt, place):
    """x[rows, cols] -> data [cols, padded rows], scales [padded rows / 128, cols]."""
    xp = torch.cat([x.float(), torch.zeros((1, x.shape[1]), device=x.device)])[place]
    b = xp.view(-1, BLOCK, x.shape[1])
    s = _scale(b.abs().amax(1), fmt)
    q = (b / s[:, None, :]).view(-1, x.shape[1]).t().contiguous().to(FLOAT8[fmt])
    return q, s.contiguous()


def _values_rows(q, s, cols):
    """The numbers that 8-bit rows stand for."""
    return q[:, :cols].float() * s.t().repeat_interleave(BLOCK, 1)[:, :cols]


def _values_tile(q, s, cols):
    full = s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
    return q[:, :cols].float() * full[:q.shape[0], :cols]


# ------------------------------------------------------------------ prepare

def _counts(rng, rows, experts):
    """Rows of each expert: a skewed share, some experts with none."""
    if experts == 1:
        return [rows]
    share = [rng.expovariate(1.0) if rng.random() > 0.1 else 0.0 for _ in range(experts)]
    total = sum(share) or 1.0
    counts = [int(rows * v / total) for v in share]
    for _ in range(rows - sum(counts)):
        counts[rng.randrange(experts)] += 1
    return counts


def _activations(gen, rows, cols, dtype):
    """Normal values with a scale for each row and a few large channels."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x *= torch.exp(torch.randn((rows, 1), generator=gen, device="cuda") * 0.5)
    x *= 1.0 + 7.0 * (torch.rand((1, cols), generator=gen, device="cuda") < 0.01).float()
    return x.to(dtype)


def _experts_of_tokens(gen, tokens, experts, k, dropped):
    """k distinct experts a token, some more popular; -1 where a row found no place."""
    popular = torch.randn((1, experts), generator=gen, device="cuda")
    score = popular + torch.randn((tokens, experts), generator=gen, device="cuda")
    ids = score.topk(k, -1).indices.to(torch.int32)
    if dropped:
        lost = torch.rand((tokens, k), generator=gen, device="cuda") < dropped
        ids = torch.where(lost, torch.full_like(ids, -1), ids)
    return ids.contiguous()


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(case)
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        st["logits"] = (torch.randn((t, e), generator=gen, device="cuda") * 2).to(DTYPES[case["dtype"]])
        st["dweights"] = torch.randn((t, k), generator=gen, device="cuda")
        return st
    if case["op"] in ("gather", "combine"):
        t, k, h = case["tokens"], case["k"], case["hidden"]
        dt = DTYPES[case["dtype"]]
        st["ids"] = _experts_of_tokens(gen, t, case["experts"], k, case["dropped"])
        if case["op"] == "gather":
            st["x"] = _activations(gen, t, h, dt)
            st["dxs"] = torch.randn((t * k, h), generator=gen, device="cuda").to(dt)
            return st
        st["ys"] = _activations(gen, t * k, h, dt)
        st["dy"] = torch.randn((t, h), generator=gen, device="cuda").to(dt)
        st["weights"] = torch.softmax(torch.randn((t, k), generator=gen, device="cuda"), -1)
        offsets, position, source = _sort(st["ids"], case["experts"])
        if own:
            from chelis_b200 import ops
            st["order"] = ops.ExpertOrder(offsets, position, source)
        else:
            st["order"] = (offsets, position, source)
        return st
    if case["op"] == "quantize":
        rows, cols, experts = case["rows"], case["cols"], case["experts"]
        dt = DTYPES[case["dtype"]]
        if case["blocks"] == "tiles":
            per = max(1, rows // experts)
            st["x"] = (torch.randn((experts, per, cols), generator=gen, device="cuda") / math.sqrt(cols)).to(dt)
            return st
        st["x"] = _activations(gen, rows, cols, dt)
        if case["blocks"] == "transposed":
            counts = _counts(rng, rows, experts)
            st["offsets"] = _offsets(counts) if experts > 1 else None
            st["place"] = _padded_rows(counts, rows, "cuda")
        return st
    rows, n, k, experts = case["rows"], case["n"], case["k"], case["experts"]
    counts = _counts(rng, rows, experts)
    st["counts"] = counts
    st["offsets"] = _offsets(counts) if experts > 1 else None
    if case["form"] == "dweight":
        place = _padded_rows(counts, rows, "cuda")
        dy = torch.randn((rows, n), generator=gen, device="cuda") * 1e-3
        st["a"] = _quantize_transposed(dy, case["format_a"], place)
        del dy
        st["b"] = _quantize_transposed(_activations(gen, rows, k, torch.bfloat16), case["format_b"], place)
    else:
        # forward: n outputs of k inputs; dinput: n outputs (the layer's inputs) of k (its outputs)
        st["a"] = _quantize_rows(_activations(gen, rows, k, torch.bfloat16), case["format_a"])
        shape = (experts, n, k) if case["form"] == "forward" else (experts, k, n)
        w = torch.randn(shape, generator=gen, device="cuda") / math.sqrt(k)
        st["b"] = _quantize_tiles(w, case["format_b"])
    if own:
        from chelis_b200 import ops
        if case["form"] == "dweight":
            st["a8"] = ops.Blocks8(st["a"][0], st["a"][1], st["a"][0].shape[1], "rows")
            st["b8"] = ops.Blocks8(st["b"][0], st["b"][1], st["b"][0].shape[1], "rows")
        else:
            st["a8"] = ops.Blocks8(st["a"][0], st["a"][1], k, "rows")
            # one matrix is passed as a matrix, several as a stack
            one = (lambda v: v[0]) if experts == 1 else (lambda v: v)
            st["b8"] = ops.Blocks8(one(st["b"][0]), one(st["b"][1]),
                                   k if case["form"] == "forward" else n, "tiles")
    return st


def _offsets(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


# -------------------------------------------------------------- plain forms

def _sort(ids, experts):
    """offsets, position, source of the stable order by expert; -1 stays out."""
    flat = ids.reshape(-1).long()
    n = flat.numel()
    key = torch.where(flat < 0, torch.full_like(flat, experts), flat)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(n, device=ids.device)
    position = torch.where(flat < 0, torch.full_like(place, -1), place).to(torch.int32).view(ids.shape)
    # the number of keys below each expert
    sorted_keys = key[order]
    offsets = torch.searchsorted(sorted_keys, torch.arange(experts + 1, device=ids.device)).to(torch.int32)
    source = torch.where(sorted_keys == experts, torch.full_like(order, -1), order).to(torch.int32)
    return offsets, position, source


def _route(logits, k, renormalize):
    l = logits.float()
    ids = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :k]
    e = torch.exp(l - l.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    w = p.gather(1, ids)
    if renormalize:
        c = e.gather(1, ids)
        w = c / c.sum(-1, keepdim=True)
    return w, ids, p


def _route_bwd(w, ids, p, g, renormalize):
    inner = (w * g).sum(-1, keepdim=True)
    if renormalize:
        return torch.zeros_like(p).scatter_(1, ids, w * (g - inner))
    return (-p * inner).scatter_add_(1, ids, w * g)


def _run_route(st):
    w, ids, p = _route(st["logits"], st["k"], st["renormalize"])
    out = {"weights": w, "experts": ids.to(torch.int32)}
    if st["backward"]:
        out["dlogits"] = _route_bwd(w, ids, p, st["dweights"], st["renormalize"])
    return out


def _sum_rows(rows, weights, position):
    """sum over slots of weights * rows[position], absent slots left out."""
    t, k = position.shape
    y = torch.zeros((t, rows.shape[1]), device=rows.device)
    for j in range(k):
        at = position[:, j].long()
        r = rows[at.clamp(min=0)].float()
        if weights is not None:
            r = r * weights[:, j:j + 1]
        y += torch.where(at[:, None] >= 0, r, torch.zeros_like(r))
    return y


def _spread(rows, source, k, weights):
    """out[p] = rows[source[p] / k] (times its weight), zero where there is none."""
    s = source.long().clamp(min=0)
    r = rows[s // k]
    if weights is not None:
        r = r * weights.reshape(-1)[s][:, None]
    return torch.where(source[:, None] >= 0, r, torch.zeros_like(r))


def _run_gather(st):
    offsets, position, source = _sort(st["ids"], st["experts"])
    out = {"offsets": offsets, "position": position, "source": source,
           "xs": _spread(st["x"].float(), source, st["k"], None)}
    if st["backward"]:
        out["dx"] = _sum_rows(st["dxs"], None, position)
    return out


def _run_combine(st):
    _, position, source = st["order"]
    k = st["k"]
    out = {"y": _sum_rows(st["ys"], st["weights"], position)}
    if st["backward"]:
        dy, w = st["dy"].float(), st["weights"]
        out["dys"] = _spread(dy, source, k, w)
        dw = torch.zeros_like(w)
        for j in range(k):
            at = position[:, j].long()
            d = (dy * st["ys"][at.clamp(min=0)].float()).sum(-1)
            dw[:, j] = torch.where(at >= 0, d, torch.zeros_like(d))
        out["dweights"] = dw
    return out


def _run_matmul(st, dtype):
    qa, sa = st["a"]
    qb, sb = st["b"]
    k, n = st["k"], st["n"]
    if st["form"] == "dweight":
        out = torch.zeros((st["experts"], n, k), device="cuda")
        at = 0
        for e, c in enumerate(st["counts"]):
            if c:
                end = at + _ceil(c, BLOCK) * BLOCK
                a = _values_rows(qa[:, at:end], sa[at // BLOCK:end // BLOCK], end - at)
                b = _values_rows(qb[:, at:end], sb[at // BLOCK:end // BLOCK], end - at)
                out[e] = a @ b.t()
                at = end
        out = out[0] if st["experts"] == 1 else out
        return {"dw": out.to(dtype)}
    out = torch.zeros((st["rows"], n), device="cuda")
    row = 0
    for e, c in enumerate(st["counts"]):
        if c:
            a = _values_rows(qa[row:row + c], sa[:, row:row + c], k)
            if st["form"] == "forward":
                out[row:row + c] = a @ _values_tile(qb[e], sb[e], k).t()
            else:
                out[row:row + c] = a @ _values_tile(qb[e], sb[e], n)
            row += c
    return {"y": out.to(dtype)}


# ---------------------------------------------------------------------- run

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    op, dt = st["op"], DTYPES[st.get("dtype", "f32")]
    if op == "route":
        out = _run_route(st)
        if "dlogits" in out:
            out["dlogits"] = out["dlogits"].to(dt)
        return out
    if op == "gather":
        out = _run_gather(st)
        return {key: v.to(dt) if key in ("xs", "dx") else v for key, v in out.items()}
    if op == "combine":
        out = _run_combine(st)
        return {key: v.to(dt) if key in ("y", "dys") else v for key, v in out.items()}
    if op == "quantize":
        if st["blocks"] == "rows":
            q, s = _quantize_rows(st["x"], st["format"])
        elif st["blocks"] == "tiles":
            q, s = _quantize_tiles(st["x"], st["format"])
        else:
            q, s = _quantize_transposed(st["x"], st["format"], st["place"])
        return {"data": q, "scales": s}
    return _run_matmul(st, dt)


def _run_own(st):
    from chelis_b200 import ops
    op = st["op"]
    if op == "route":
        w, ids = ops.expert_route(st["logits"], st["k"], st["renormalize"])
        out = {"weights": w, "experts": ids}
        if st["backward"]:
            out["dlogits"] = ops.expert_route_bwd(st["logits"], ids, st["dweights"], st["renormalize"])
        return out
    if op == "gather":
        order = ops.expert_sort(st["ids"], st["experts"])
        out = {"offsets": order.offsets, "position": order.position, "source": order.source,
               "xs": ops.expert_gather(st["x"], order)}
        if st["backward"]:
            out["dx"] = ops.expert_gather_bwd(st["dxs"], order)
        return out
    if op == "combine":
        out = {"y": ops.expert_combine(st["ys"], st["weights"], st["order"])}
        if st["backward"]:
            out["dys"], out["dweights"] = ops.expert_combine_bwd(st["dy"], st["ys"], st["weights"],
                                                                 st["order"])
        return out
    if op == "quantize":
        if st["blocks"] == "transposed":
            b = ops.quantize8_transposed(st["x"], st["format"], st["offsets"])
        else:
            b = ops.quantize8(st["x"], st["format"], st["blocks"])
        return {"data": b.data, "scales": b.scales}
    dt = DTYPES[st["dtype"]]
    if st["form"] == "dweight":
        return {"dw": ops.matmul8_wgrad(st["a8"], st["b8"], st["offsets"], dtype=dt)}
    return {"y": ops.matmul8(st["a8"], st["b8"], trans_b=st["form"] == "forward",
                             offsets=st["offsets"], dtype=dt)}


# -------------------------------------------------------------------- exact

def _exact_round8(v, fmt):
    """The nearest number of the 8-bit format, ties to even, in 64 bits."""
    digits, least = (3, -6) if fmt == "e4m3" else (2, -14)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=least) - digits)
    return torch.round(v / step) * step


def _exact_scale(amax, fmt):
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / LARGEST[fmt]))
    s = torch.exp2(e.clamp(min=-126))
    # log2 may round across a whole number: put the least power right
    s = torch.where(amax > s * LARGEST[fmt], s * 2, s)
    s = torch.where((amax <= s / 2 * LARGEST[fmt]) & (s > 2.0 ** -126), s / 2, s)
    return torch.where(amax > 0, s, torch.ones_like(s))


def _exact_quantize(st):
    x = st["x"].double()
    fmt = st["format"]
    if st["blocks"] == "transposed":
        cols = x.shape[1]
        xp = torch.cat([x, torch.zeros((1, cols), dtype=x.dtype, device=x.device)])[st["place"]]
        s = _exact_scale(xp.view(-1, BLOCK, cols).abs().amax(1), fmt)
        q = _exact_round8(xp / s.repeat_interleave(BLOCK, 0), fmt)
        return {"data": q.t().contiguous(), "scales": s}
    if st["blocks"] == "rows":
        x = x[None]
    e, rows, cols = x.shape
    high = 1 if st["blocks"] == "rows" else BLOCK
    rb, kb = _ceil(rows, high), _ceil(cols, BLOCK)
    xp = _padded(x, rb * high, kb * BLOCK)
    s = _exact_scale(xp.view(e, rb, high, kb, BLOCK).abs().amax((2, 4)), fmt)
    q = _exact_round8(xp / s.repeat_interleave(high, 1).repeat_interleave(BLOCK, 2), fmt)
    q = q[:, :rows, :_ceil(cols, 16) * 16]
    if st["blocks"] == "rows":
        return {"data": q[0].contiguous(), "scales": s[0].t().contiguous()}
    return {"data": q.contiguous(), "scales": s}


def _exact_route(st):
    l, k = st["logits"].double(), st["k"]
    order = torch.argsort(-l, dim=-1, stable=True)
    chosen = torch.zeros_like(l).scatter_(1, order[:, :k], 1.0)
    p = torch.softmax(l, -1) if not st["renormalize"] else \
        torch.softmax(torch.where(chosen > 0, l, torch.full_like(l, -math.inf)), -1)
    out = {"weights": p.gather(1, order[:, :k]), "experts": None}
    if st["backward"]:
        g = torch.zeros_like(l).scatter_(1, order[:, :k], st["dweights"].double())
        out["dlogits"] = p * (g - (p * g).sum(-1, keepdim=True))
    return out


def _exact_gather(st):
    ids = st["ids"].cpu()
    k, flat = st["k"], ids.reshape(-1).tolist()
    rows = sorted((i for i, e in enumerate(flat) if e >= 0), key=lambda i: (flat[i], i))
    x = st["x"].double()
    at = torch.tensor(rows, dtype=torch.int64, device=x.device)
    xs = torch.zeros((len(flat), x.shape[1]), dtype=x.dtype, device=x.device)
    xs[:len(rows)] = x.index_select(0, at // k)
    out = {"offsets": None, "position": None, "source": None, "xs": xs}
    if st["backward"]:
        out["dx"] = torch.zeros_like(x).index_add_(0, at // k, st["dxs"][:len(rows)].double())
    return out


def _exact_combine(st):
    _, _, source = st["order"]
    k = st["k"]
    p = torch.nonzero(source >= 0).reshape(-1)
    slot = source[p].long()
    w = st["weights"].double().reshape(-1)[slot][:, None]
    ys, dy = st["ys"].double(), st["dy"].double()
    out = {"y": torch.zeros_like(dy).index_add_(0, slot // k, ys[p] * w)}
    if st["backward"]:
        dys = torch.zeros_like(ys)
        dys[p] = dy[slot // k] * w
        dw = torch.zeros(st["weights"].numel(), dtype=ys.dtype, device=ys.device)
        dw[slot] = torch.einsum("ph,ph->p", dy[slot // k], ys[p])
        out["dys"], out["dweights"] = dys, dw.view(st["weights"].shape)
    return out


def _exact_matmul(st):
    """Block by block of the contraction: the scales times the sum of products."""
    (qa, sa), (qb, sb) = st["a"], st["b"]
    n, k, experts = st["n"], st["k"], st["experts"]
    if st["form"] == "dweight":
        out = torch.zeros((experts, n, k), dtype=torch.float64, device="cuda")
        block = 0
        for e, c in enumerate(st["counts"]):
            for b in range(block, block + _ceil(c, BLOCK)):
                at = slice(b * BLOCK, (b + 1) * BLOCK)
                part = qa[:, at].double() @ qb[:, at].double().t()
                out[e] += part * sa[b].double()[:, None] * sb[b].double()[None]
            block += _ceil(c, BLOCK)
        return {"dw": out[0] if experts == 1 else out}
    out = torch.zeros((st["rows"], n), dtype=torch.float64, device="cuda")
    row = 0
    for e, c in enumerate(st["counts"]):
        for b in range(_ceil(k, BLOCK)):
            at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            if st["form"] == "forward":
                part, s = qa[row:row + c, at].double() @ qb[e, :, at].double().t(), sb[e, :, b]
            else:
                part, s = qa[row:row + c, at].double() @ qb[e, at, :n].double(), sb[e, b]
            s = s.double().repeat_interleave(BLOCK)[:n]
            out[row:row + c] += part * sa[b, row:row + c].double()[:, None] * s[None]
        row += c
    return {"y": out}


def exact(case, seed):
    st = prepare(case, seed)
    return {"route": _exact_route, "gather": _exact_gather, "combine": _exact_combine,
            "quantize": _exact_quantize, "matmul": _exact_matmul}[case["op"]](st)


# --------------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "route":
        t, e, k, w = case["tokens"], case["experts"], case["k"], WIDTH[case["dtype"]]
        b, f = t * e * w + t * k * 8, t * e * 4 + t * k * 4
        if case["backward"]:
            b, f = b + t * e * w + t * k * 4, f + t * e * 3
        return {"bytes": b, "flops": f}
    if op in ("gather", "combine"):
        t, k, h, w = case["tokens"], case["k"], case["hidden"], WIDTH[case["dtype"]]
        one, many = t * h * w, t * k * h * w
        if op == "gather":
            b, f = one + many + t * k * 12 + case["experts"] * 4, 0
            if case["backward"]:
                b, f = b + one + many, t * k * h
            return {"bytes": b, "flops": f}
        b, f = one + many + t * k * 8, 2 * t * k * h
        if case["backward"]:
            b, f = b + one + many + t * k * 4, f + 3 * t * k * h
        return {"bytes": b, "flops": f}
    if op == "quantize":
        rows = case["rows"]
        if case["blocks"] == "tiles":
            rows = max(1, rows // case["experts"]) * case["experts"]
        n = rows * case["cols"]
        per = BLOCK * BLOCK if case["blocks"] == "tiles" else BLOCK
        return {"bytes": n * (WIDTH[case["dtype"]] + 1) + n // per * 4, "flops": 2 * n}
    rows, n, k, e, w = case["rows"], case["n"], case["k"], case["experts"], WIDTH[case["dtype"]]
    used = min(e, rows)
    if case["form"] == "dweight":
        b = rows * (n + k) + rows * (n + k) // BLOCK * 4 + e * n * k * w
    else:
        b = rows * k + rows * k // BLOCK * 4 + used * n * k + rows * n * w
    return {"bytes": b, "flops": 2 * rows * n * k}

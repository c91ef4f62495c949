"""The router's balance loss and the experts' counts, with the gradient.

Bounds, u = 2^-24: a probability is within 110 u relative (as the router's, of
logits that differ by at most 32); an expert's sum of T of them within
T u more; the loss is a sum of positive terms: (110 + T) u of it.  The gradient
p (c - sum p c) has two of them and 40 roundings more, of terms no larger than
p (c + sum p c): 300 u of that."""
import math

import numpy as np
import pytest

import _experts_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _t(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _ref(l, ids, live, k):
    """(loss, counts with N, p, per) in float64; l [tokens, experts]."""
    e = l.shape[1]
    c = np.bincount(ids[live].reshape(-1)[ids[live].reshape(-1) >= 0], minlength=e).astype(float)
    n = max(1, int(live.sum()))
    top = l.max(-1, keepdims=True)
    p = np.exp(l - np.where(np.isfinite(top), top, 0.0))
    z = p.sum(-1, keepdims=True)
    p = np.where(z > 0, p / np.where(z > 0, z, 1), 0.0)
    per = e / (k * float(n) * n)
    return per * float((c * p[live].sum(0)).sum()), np.append(c, live.sum()), p, per * c


def _case(rng, t, e, k, dtype, drop=0.2):
    import torch
    x = torch.from_numpy(np.clip(rng.standard_normal((t, e)) * 3, -15, 15)).to(_t(dtype))
    ids = np.argsort(-x.double().numpy(), axis=-1, kind="stable")[:, :k].astype(np.int32)
    ids[rng.random((t, k)) < drop] = -1
    return x.cuda(), x.double().numpy(), torch.from_numpy(ids).cuda(), ids


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("t,e,k,dtype", [(1, 1, 1, "f32"), (3, 7, 2, "f32"), (64, 8, 2, "bf16"), (128, 64, 8, "f32"), (129, 64, 8, "f32"),
                                         (65, 100, 3, "f16"), (300, 256, 32, "f32"), (33, 257, 4, "bf16"),
                                         (500, 1024, 1, "f32"), (20000, 33, 5, "bf16"), (5000, 64, 8, "f16")])
def test_loss_counts_and_gradient(cuda, t, e, k, dtype, masked):
    import torch
    rng = np.random.default_rng(t * 3 + e)
    x, l, ids, hids = _case(rng, t, e, k, dtype)
    live = rng.random(t) < 0.7 if masked else np.ones(t, dtype=bool)
    mask = torch.from_numpy(live).cuda() if masked else None
    if masked:  # what padding holds does not matter
        x[~mask] = float("nan")
        ids[~mask] = 10 ** 6
    loss, counts = cuda.expert_balance(x, ids, mask)
    ref, rc, p, pc = _ref(np.where(live[:, None], l, 0), hids, live, k)
    assert (counts.cpu().numpy() == rc).all()
    assert abs(float(loss) - ref) <= (110 + t + 8) * U * ref
    dloss = torch.tensor(0.5, device="cuda")
    add = torch.from_numpy(rng.standard_normal((t, e)) * 1e-3).to(_t(dtype)).cuda()
    for a in (None, add):
        got = cuda.expert_balance_bwd(x, counts, k, 2.0, dloss, mask, a)
        inner = (p * pc).sum(-1, keepdims=True)
        d = np.where(live[:, None], p * (pc - inner), 0.0)
        bound = np.where(live[:, None], 300 * U * p * (pc + inner), 0.0)
        if a is not None:
            d = d + a.double().cpu().numpy()
            bound = bound + U * np.abs(d)
        assert not R.outside(got.double().cpu().numpy(), d, bound, dtype).any()
    assert torch.equal(cuda.expert_balance(x, ids, mask)[0], loss)  # no order of atomics in it
    cuda.device_status()


def test_even_load_is_one_and_no_token_none(cuda):
    import torch
    x = torch.zeros(64, 8, device="cuda")
    ids = (torch.arange(128, device="cuda") % 8).int().view(64, 2)
    loss, counts = cuda.expert_balance(x, ids)
    assert abs(float(loss) - 1) < 1e-6 and counts.tolist() == [16] * 8 + [64]
    for m in (None, torch.zeros(0, dtype=torch.bool, device="cuda")):
        loss, counts = cuda.expert_balance(x[:0], ids[:0], m)
        assert float(loss) == 0 and counts.tolist() == [0] * 9
    off = torch.zeros(64, dtype=torch.bool, device="cuda")
    loss, counts = cuda.expert_balance(x, ids, off)
    assert float(loss) == 0 and counts.tolist() == [0] * 9
    assert not cuda.expert_balance_bwd(x, counts, 2, mask=off).any()


def test_experts_at_minus_infinity(cuda):
    import torch
    x = torch.zeros(70, 6, device="cuda")
    x[:, 2] = -float("inf")
    x[5] = -float("inf")  # no expert left: no probability, but it counts
    ids = torch.full((70, 1), 1, dtype=torch.int32, device="cuda")
    ids[5] = -1
    loss, counts = cuda.expert_balance(x, ids)
    assert counts.tolist() == [0, 69, 0, 0, 0, 0, 70]
    assert abs(float(loss) - 6 / 70 ** 2 * 69 * 69 / 5) < 1e-5
    g = cuda.expert_balance_bwd(x, counts, 1)
    assert not g[5].any() and not g[:, 2].any() and (g[0, 1] > 0) and torch.isfinite(g).all()
    x[7, 0] = float("nan")
    assert torch.isnan(cuda.expert_balance(x, ids)[0])


def test_gradient_against_differences(cuda):
    import torch
    rng = np.random.default_rng(1)
    x, l, ids, hids = _case(rng, 50, 9, 2, "f32")
    loss, counts = cuda.expert_balance(x, ids)
    g = cuda.expert_balance_bwd(x, counts, 2).double().cpu().numpy()
    d = rng.standard_normal(l.shape)
    live = np.ones(50, dtype=bool)
    numeric = (_ref(l + 1e-6 * d, hids, live, 2)[0] - _ref(l - 1e-6 * d, hids, live, 2)[0]) / 2e-6
    assert abs(numeric - (g * d).sum()) <= 1e-5 * np.abs(g * d).sum() + 1e-8


def test_offsets_past_32_bits(cuda):
    import torch
    t, e = (1 << 21) + 77, 1024
    x = torch.zeros(t, e, device="cuda", dtype=torch.bfloat16)
    x[-3:, 5] = 8.0
    ids = torch.zeros(t, 1, dtype=torch.int32, device="cuda")
    ids[-3:] = 5
    loss, counts = cuda.expert_balance(x, ids)
    assert int(counts[0]) == t - 3 and int(counts[5]) == 3 and int(counts[e]) == t
    g = cuda.expert_balance_bwd(x, counts, 1, float(t))
    p = math.exp(8) / (math.exp(8) + e - 1)
    q = 1 / (math.exp(8) + e - 1)
    want = e / t * p * (3 - (p * 3 + q * (t - 3)))
    assert abs(float(g[t - 1, 5]) - want) <= 2.0 ** -8 * abs(want) + 1e-4 * abs(want)
    assert abs(float(loss) - 1.0) < 1e-3


def test_bad_ids_are_reported(cuda):
    import torch
    from chelis_b200 import lib as L
    x = torch.zeros(40, 4, device="cuda")
    ids = torch.zeros(40, 2, dtype=torch.int32, device="cuda")
    ids[3, 1], ids[4, 0] = 4, -2
    _, counts = cuda.expert_balance(x, ids)
    assert counts.tolist() == [78, 0, 0, 0, 40]
    with pytest.raises(L.ChelisCudaError):
        cuda.device_status()


def test_captured(cuda):
    import torch
    rng = np.random.default_rng(2)
    x, l, ids, _ = _case(rng, 3000, 64, 4, "f32")
    want = cuda.expert_balance(x, ids)
    dwant = cuda.expert_balance_bwd(x, want[1], 4)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = cuda.expert_balance(x, ids)
            dgot = cuda.expert_balance_bwd(x, got[1], 4)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1]) and torch.equal(dwant, dgot)


def test_refusals(cuda):
    import torch
    x = torch.zeros(6, 4, device="cuda")
    ids = torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    c = torch.zeros(5, dtype=torch.int32, device="cuda")
    for bad in (lambda: cuda.expert_balance(x, ids.long()), lambda: cuda.expert_balance(x[:5], ids),
                lambda: cuda.expert_balance(x.double(), ids), lambda: cuda.expert_balance(x, ids, torch.ones(6, device="cuda")),
                lambda: cuda.expert_balance(x, ids, torch.ones(5, dtype=torch.bool, device="cuda")),
                lambda: cuda.expert_balance_bwd(x, c[:4], 2), lambda: cuda.expert_balance_bwd(x, c, 2, add=x.half()),
                lambda: cuda.expert_balance_bwd(x, c, 2, dloss=x), lambda: cuda.expert_balance(x.t(), ids)):
        with pytest.raises(ValueError):
            bad()

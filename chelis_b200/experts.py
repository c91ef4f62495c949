"""A routed feed-forward layer on the library's operators: forward and
vector-Jacobian product, the experts' products in 8 bits.

    y[t] = sum_j w[t, j] W2[e] gelu(W1[e] x[t]),  e = expert j of token t

x is f32 [tokens, d]; the router's matrix is f32 [d, experts]; the experts'
weights are 8-bit tiles (ops.quantize8(w, "e4m3", "tiles")), W1 [experts, ff,
d] and W2 [experts, d, ff].  Activations are quantised to e4m3 and gradients
to e5m2 where a product takes them; everything between is f32.  With a weight
for it, the loss that balances the experts' load joins in: Saved has it, and
the gradients are those of y's loss plus balance times it.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops
from .fused import External, FusedStep

_ADD = [FusedStep("add", External(0), External(1))]


class Saved(NamedTuple):
    """What feed_forward keeps for feed_forward_bwd."""
    x: torch.Tensor
    logits: torch.Tensor
    weights: torch.Tensor
    experts: torch.Tensor
    order: ops.ExpertOrder
    h: torch.Tensor   # before gelu
    ys: torch.Tensor  # the experts' rows
    renormalize: bool = True
    balance: float = 0.0                 # weight of the balance loss
    loss: torch.Tensor | None = None     # the loss itself (ops.expert_balance), with balance
    counts: torch.Tensor | None = None   # the experts' pairs, then the tokens that count
    mask: torch.Tensor | None = None


def feed_forward(x: torch.Tensor, router: torch.Tensor, w1: ops.Blocks8, w2: ops.Blocks8, k: int,
                 renormalize: bool = True, balance: float = 0.0, mask: torch.Tensor | None = None):
    """(y [tokens, d], Saved).  balance: the weight of the balance loss, over the
    tokens where mask (bool [tokens]) is true."""
    logits = ops.matmul(x, router)
    weights, chosen = ops.expert_route(logits, k, renormalize)
    order = ops.expert_sort(chosen, router.shape[1])
    x8 = ops.quantize8(ops.expert_gather(x, order))
    h = ops.matmul8(x8, w1, offsets=order.offsets, dtype=torch.float32)
    ys = ops.matmul8(ops.quantize8(ops.gelu(h)), w2, offsets=order.offsets, dtype=torch.float32)
    y = ops.expert_combine(ys, weights, order)
    loss, counts = ops.expert_balance(logits, chosen, mask) if balance else (None, None)
    return y, Saved(x, logits, weights, chosen, order, h, ys, bool(renormalize), float(balance), loss, counts, mask)


def feed_forward_bwd(dy: torch.Tensor, s: Saved, router: torch.Tensor, w1: ops.Blocks8,
                     w2: ops.Blocks8, renormalize: bool | None = None) -> dict:
    """The gradients of feed_forward: dx, drouter, dw1, dw2 (all f32).
    renormalize is the forward pass's, which s keeps; another one is refused."""
    if renormalize is not None and bool(renormalize) != s.renormalize:
        raise ValueError("feed_forward_bwd: renormalize is not the forward pass's")
    off = s.order.offsets
    dys, dweights = ops.expert_combine_bwd(dy, s.ys, s.weights, s.order)
    da = ops.matmul8(ops.quantize8(dys, "e5m2"), w2, trans_b=False, offsets=off, dtype=torch.float32)
    dw2 = ops.matmul8_wgrad(ops.quantize8_transposed(dys, "e5m2", off),
                            ops.quantize8_transposed(ops.gelu(s.h), "e4m3", off), off)
    dh = ops.gelu_adjoint(s.h, da)
    dxs = ops.matmul8(ops.quantize8(dh, "e5m2"), w1, trans_b=False, offsets=off, dtype=torch.float32)
    dw1 = ops.matmul8_wgrad(ops.quantize8_transposed(dh, "e5m2", off),
                            ops.quantize8_transposed(ops.expert_gather(s.x, s.order), "e4m3", off), off)
    dlogits = ops.expert_route_bwd(s.logits, s.experts, dweights, s.renormalize)
    if s.balance:
        dlogits = ops.expert_balance_bwd(s.logits, s.counts, s.experts.shape[1], s.balance, mask=s.mask, add=dlogits)
    dx = ops.fused_elementwise(_ADD, [ops.expert_gather_bwd(dxs, s.order),
                                      ops.matmul(dlogits, router, trans_b=True)])
    return {"dx": dx, "drouter": ops.matmul(s.x, dlogits, trans_a=True), "dw1": dw1, "dw2": dw2}

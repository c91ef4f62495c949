"""A dense feed-forward sublayer in 16 bits on the library's operators: forward
and vector-Jacobian product.

    h = N(x) pre_gamma + pre_beta
    f = act(h W1 + b1) W2 + b2
    y = scale x + gate (N(f) post_gamma + post_beta)

x and the matrices are bf16 or f16, W1 [d, ff] and W2 [ff, d]; norms, gate and
their gradients are f32, and so are the matrices' gradients.  The second norm,
the betas, the gate and the biases may be None.  Clip the parameters' gradients
of a whole step (all of feed_forward_bwd's but dx, which is the gradient of what
comes before) with ops.clip_grads, after dp.allreduce_sum where there are several
GPUs.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops


class Sublayer(NamedTuple):
    pre_gamma: torch.Tensor
    w1: torch.Tensor
    w2: torch.Tensor
    pre_beta: torch.Tensor | None = None
    b1: torch.Tensor | None = None
    b2: torch.Tensor | None = None
    post_gamma: torch.Tensor | None = None
    post_beta: torch.Tensor | None = None
    gate: torch.Tensor | None = None
    activation: str = "gelu"
    kind: str = "layer"
    scale: float = 1.0
    eps: float = 1e-5

    def _norms(self) -> dict:
        return dict(post_gamma=self.post_gamma, post_beta=self.post_beta, gate=self.gate, scale=self.scale,
                    eps=self.eps, kind=self.kind)


class Saved(NamedTuple):
    """What feed_forward keeps for feed_forward_bwd."""
    x: torch.Tensor
    h: torch.Tensor
    a: torch.Tensor   # the activation's value
    z: torch.Tensor   # what it was taken of
    f: torch.Tensor   # the branch
    y: torch.Tensor


def feed_forward(x: torch.Tensor, p: Sublayer):
    """(y [tokens, d], Saved)."""
    _, h = ops.residual_norm(x, None, pre_gamma=p.pre_gamma, pre_beta=p.pre_beta, eps=p.eps, kind=p.kind)
    a, z = ops.matmul16(h, p.w1, bias=p.b1, activation=p.activation, keep_pre=True)
    f = ops.matmul16(a, p.w2, bias=p.b2)
    y, _ = ops.residual_norm(x, f, **p._norms())
    return y, Saved(x, h, a, z, f, y)


def feed_forward_bwd(dy: torch.Tensor, s: Saved, p: Sublayer) -> dict:
    """The gradients of feed_forward: dx and, by their names, those of the
    parameters that there are."""
    out = ops.residual_norm_bwd(dy, None, s.y, s.f, **p._norms())
    dz, dw2, db2 = ops.matmul16_bwd(out.dbranch, s.a, p.w2, through=(s.z, p.activation),
                                    want_bias=p.b2 is not None)
    dh, dw1, db1 = ops.matmul16_bwd(dz, s.h, p.w1, want_bias=p.b1 is not None)
    inner = ops.residual_norm_bwd(out.dx, dh, s.x, None, pre_gamma=p.pre_gamma, pre_beta=p.pre_beta, eps=p.eps,
                                  kind=p.kind)
    grads = {"dx": inner.dx, "pre_gamma": inner.dpre_gamma, "pre_beta": inner.dpre_beta, "w1": dw1, "b1": db1,
             "w2": dw2, "b2": db2, "post_gamma": out.dpost_gamma, "post_beta": out.dpost_beta, "gate": out.dgate}
    return {name: g for name, g in grads.items() if g is not None}

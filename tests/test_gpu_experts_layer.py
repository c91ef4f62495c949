"""The routed feed-forward layer's gradients take the router's form from the
forward pass."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("renormalize", [True, False])
def test_gradients_follow_the_forward_pass(cuda, renormalize):
    import torch
    from chelis_b200 import experts as X
    gen = torch.Generator(device="cuda").manual_seed(7)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    x, router, dy = randn(40, 64), randn(64, 6), randn(40, 64)
    w1, w2 = (cuda.quantize8(w, "e4m3", "tiles") for w in (randn(6, 96, 64), randn(6, 64, 96)))
    _, saved = X.feed_forward(x, router, w1, w2, 3, renormalize)
    got = X.feed_forward_bwd(dy, saved, router, w1, w2)
    same = X.feed_forward_bwd(dy, saved, router, w1, w2, renormalize)
    # the router's gradient, from the weights' that the experts' rows give
    dweights = cuda.expert_combine_bwd(dy, saved.ys, saved.weights, saved.order)[1]
    dlogits = cuda.expert_route_bwd(saved.logits, saved.experts, dweights, renormalize)
    assert torch.equal(got["drouter"], cuda.matmul(x, dlogits, trans_a=True))
    for name in got:
        assert torch.equal(got[name], same[name])
    with pytest.raises(ValueError):
        X.feed_forward_bwd(dy, saved, router, w1, w2, not renormalize)

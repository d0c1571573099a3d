"""How exact the model-side operators are, each property with data that leaves
no room for anything else: weights of very different sizes.

Tolerances, derived here (U = 2^-24, half a step of f32):
  - a weight of a preference pair is computed in 64 bits, rounded once as the
    candidate's gradient, once with the factors and once in the row: 3 U, and
    one more for the mean's factor; an upstream weight of a score is rounded
    twice, and the sums lose 2^-48 of their largest weight at most.
"""
import math

import pytest
import torch

from test_gpu_head_ops import U, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fd(built):
    import flashtrie_device
    return flashtrie_device


# ------------------------------------------------------- weights of all sizes

def spiked(C):
    """Logits [1, 1, C + 1] of which the first takes all of the probability
    (the others have e^-60 of it), and a candidate for each of the others: its
    log-probability is -60 (off by 1e-23), its token no other's."""
    x = torch.zeros((1, 1, C + 1), device="cuda")
    x[..., 0] = 60.0
    toks = torch.arange(1, C + 1, device="cuda", dtype=torch.int32).view(1, C, 1)
    return x, toks, torch.ones((1, C), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("lo,hi,P,absent", [(25, 40, 1000, 0), (36, 50, 200, 0), (36, 60, 200, 0),
                                            (-5, 75, 1000, 0), (0, 40, 1, 0),
                                            (20, 30, 3, 200000)])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_pair_weights_of_any_margin(fd, lo, hi, P, absent, reduction):
    """Each pair's candidate gets the pair's own weight, however far apart the
    pair is, whatever other pairs there are."""
    beta = torch.tensor(0.1).item()
    x, toks, lens = spiked(P + 1)
    lens[0, P] = 0  # the other side of all pairs
    z = torch.linspace(lo, hi, P, dtype=torch.float64, device="cuda")
    ref = torch.zeros((1, P + 1), device="cuda")
    ref[0, :P] = (-60.0 - z / beta).float()
    z = beta * (-60.0 - ref[0, :P].double())
    c = torch.full((1, P + absent), -1, dtype=torch.int32, device="cuda")
    r = torch.full_like(c, P)
    at = torch.arange(P, device="cuda") * (1 + absent // P)
    c[0, at] = torch.arange(P, device="cuda", dtype=torch.int32)
    leaf = x.requires_grad_()
    loss, margin = fd.preference_loss(leaf, toks, lens, ref, c, r, beta=beta, reduction=reduction)
    assert bool(((margin[0, at].double() - z).abs() <= U * z.abs()).all())
    (dx,) = torch.autograd.grad(loss, leaf)
    want = -beta * torch.sigmoid(-z) / (P if reduction == "mean" else 1)
    # The softmax part of each entry: the row's whole weight times e^-60.
    tol = 4 * U * want.abs() + want.abs().sum() * 2 * math.exp(-60) + 2.0 ** -126
    err = (dx[0, 0, 1:P + 1].double() - want).abs()
    assert bool((err <= tol).all()), float((err / want.abs()).max())


@pytest.mark.parametrize("share", [1, 2, 50])
def test_token_weights_of_any_size(fd, share):
    """Weights 14 powers of ten apart in one row, `share` candidates of one
    size with each token: every token's sum is as exact as its own weights."""
    C = 1000
    x, toks, lens = spiked(C)
    toks = ((toks - 1) // share + 1).contiguous()
    size = 10.0 ** (-14 * torch.rand((C // share, 1), generator=gen(1), device="cuda", dtype=torch.float64))
    w = (size * (0.5 + torch.rand((C // share, share), generator=gen(2), device="cuda", dtype=torch.float64))).float()
    w *= torch.where(torch.rand(w.shape, generator=gen(3), device="cuda") < 0.5, -1.0, 1.0)
    leaf = x.requires_grad_()
    (dx,) = torch.autograd.grad(fd.sequence_logp(leaf, toks, lens), leaf, w.view(1, C))
    want = w.double().sum(1)
    tol = 3 * U * want.abs() + 2.0 ** -48 * w.double().abs().sum(1) + w.double().abs().sum() * 2 * math.exp(-60)
    err = (dx[0, 0, 1:C // share + 1].double() - want).abs()
    assert bool((err <= tol).all()), float((err / w.double().abs().sum(1)).max())

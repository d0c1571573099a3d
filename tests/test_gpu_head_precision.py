"""How exact the model-side operators are, each property with data that leaves
no room for anything else: weights of very different sizes,
low-rank values far from 1.

Tolerances, derived here (U = 2^-24, half a step of f32):
  - a weight of a preference pair is computed in 64 bits, rounded once as the
    candidate's gradient, once with the factors and once in the row: 3 U, and
    one more for the mean's factor; an upstream weight of a score is rounded
    twice, and the sums lose 2^-48 of their largest weight at most;
  - low-rank values: 2 (D + 2) U of their products' absolute sum, then what the
    16-bit parts lose (LOSS), then 2 (parts r + 2) U of sum |u b| for the second
    product.
"""
import math

import pytest
import torch

from test_gpu_head_ops import HALVES, U, gen, half_step, make_head

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


# ------------------------------------------------------------ low-rank values

# What the 16-bit parts of a low-rank value lose, relative, by (type, f32 out).
LOSS = {(torch.bfloat16, False): 2.0 ** -17, (torch.bfloat16, True): 2.0 ** -26,
        (torch.float16, False): 2.0 ** -23, (torch.float16, True): 2.0 ** -23}
# n, L, G: one request; requests of a few adapters; an adapter for every token.
FORMS = [(1, 5, 1), (6, 20, 3), (40, 1, 40)]


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,G", FORMS)
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 2.0 ** -9, 1.0, 1e5, 1e30])
@pytest.mark.parametrize("shared", [False, True])
def test_low_rank_values_of_any_size(fd, t, n, L, G, scale, shared):
    """The low-rank part beside a shared projection or alone: as exact where
    its values are tiny or beyond the type's largest as where they are near 1,
    and the same in every form that a batch may take."""
    D, V, r = 64, 300, 8
    h, w, ids, a, b, s = make_head(n, L, V, D, r, G, t, seed=7)
    ids = (torch.arange(n, device="cuda") % G).to(torch.int32)
    if not shared:
        w = torch.zeros_like(w)
    s = s * scale
    at = ids.long()
    hd, ad, bd = h.double(), a.double()[at], b.double()[at]
    u = (hd @ ad.transpose(1, 2)) * s.double()[at][:, None, None]
    y = hd @ w.double().T + u @ bd.transpose(1, 2)
    shared_mass = hd.abs() @ w.double().abs().T
    u_mass = (hd.abs() @ ad.abs().transpose(1, 2)) * s.double()[at][:, None, None] @ bd.abs().transpose(1, 2)
    mass = u.abs() @ bd.abs().transpose(1, 2)
    for out_t in (t, torch.float32):
        out = fd.adapter_logits(h, w, ids, a, b, s, out_dtype=out_t).double()
        parts = LOSS[t, out_t == torch.float32]
        tol = 2 * (D + 3 * r + 2) * U * (shared_mass + mass) + 2 * (D + 2) * U * u_mass + parts * mass
        if t == torch.float16:
            # Two f16 parts leave up to 2^-25 behind, absolute; tokens whose
            # largest value is below 2^-8 take no part in that.
            near = (u.abs().amax(-1) >= 2.0 ** -8)[..., None]
            tol = tol + near * 2.0 ** -25 * bd.abs().sum(-1)[:, None]
        tol = tol + half_step(out_t, y)
        beyond = y.abs() + tol > torch.finfo(out_t).max
        assert bool((torch.isfinite(out) | beyond).all())
        err = torch.where(beyond, 0.0, (out - y).abs())
        assert bool((err <= tol).all()), float((err / (mass + shared_mass)).max())
